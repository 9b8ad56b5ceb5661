// Shared by answers.hip (log probabilities) and distill.hip (distillation loss): how a row of logits is held, walked,
// reduced and ordered, and how its gradient is streamed.
#pragma once
#include <type_traits>

#include "common.h"
#include "wave.h"

namespace {

constexpr int AN_TOP_MAX = 128;     // alternatives / teacher answers per row
constexpr int AN_WAVE_C = 1024;     // classes up to which a row belongs to one wave
constexpr int AN_CAP = 1024;        // candidates for the top alternatives that fit in shared memory
constexpr float AN_NO_REST = 9.5367431640625e-07f;  // 2^-20: a smaller remainder of f32 log probabilities is rounding

constexpr double AN_LN2 = 0.69314718055994530942;
constexpr double AN_LOG2E = 1.44269504088896340736;

typedef unsigned long long u64;

// ---------------------------------------------------------------------------------------------
// Order of the alternatives: larger value first, then lower index; NaN above everything (as torch.topk has it)
// and the two zeros equal.
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ unsigned an_key(float x) {
  const unsigned u = __float_as_uint(x + 0.0f);   // -0 + 0 = +0
  const unsigned k = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return x != x ? 0xffffffffu : k;
}
__device__ __forceinline__ float an_unkey(unsigned k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
constexpr unsigned AN_KEY_MINF = 0x007fffffu;   // an_key(-inf): the lowest key of any value
__device__ __forceinline__ u64 an_pack(unsigned key, int idx) { return ((u64)key << 32) | (unsigned)~idx; }
__device__ __forceinline__ int an_index(u64 c) { return (int)~(unsigned)c; }

// exp(t) for t <= 0 to about 2^-40: t = k ln 2 + f with |f| <= ln 2 / 2, Taylor's polynomial of degree 10 in f
// (the first term left out is f^11 / 11! < 2^-41).  NaN stays NaN; below -700 the result is zero.
__device__ __forceinline__ double an_exp(double t) {
  const double c = t < -700.0 ? -700.0 : t;
  const double k = __builtin_rint(c * AN_LOG2E);
  const double f = fma(-k, AN_LN2, c);   // |k| < 1100: the constant's own rounding stays below 2^-42
  double p = 1.0 / 3628800.0;
  p = fma(p, f, 1.0 / 362880.0);
  p = fma(p, f, 1.0 / 40320.0);
  p = fma(p, f, 1.0 / 5040.0);
  p = fma(p, f, 1.0 / 720.0);
  p = fma(p, f, 1.0 / 120.0);
  p = fma(p, f, 1.0 / 24.0);
  p = fma(p, f, 1.0 / 6.0);
  p = fma(p, f, 0.5);
  p = fma(p, f, 1.0);
  p = fma(p, f, 1.0);
  return t < -700.0 ? 0.0 : ldexp(p, (int)k);
}

// the exponent's factor log2(e) / T: the nearest f32, how far off it is, and what is left of it as a second f32
struct AnTemp {
  float hi, lo;
  double inv_t;
  double delta;   // hi = log2(e) / T * (1 + delta)
};
inline AnTemp an_temp(double temperature) {
  AnTemp t;
  t.inv_t = 1.0 / temperature;
  const double c = AN_LOG2E * t.inv_t;
  t.hi = (float)c;
  t.lo = (float)(c - (double)t.hi);
  t.delta = (double)t.hi / c - 1.0;
  return t;
}
// (x - m) log2(e) / T with both terms, where no sum can take the first one's error out (the streamed gradients: they wait
// for memory anyway).  x = -inf gives -inf (the second term, of either sign, stays finite); NaN comes through the first.
__device__ __forceinline__ float an_arg(float x, float m, float hi, float lo) {
  const float d = x - m;
  return fmaf(d, hi, fmaxf(d, -3.402823466e38f) * lo);
}
__device__ __forceinline__ float an_exp2(float t) { return __builtin_amdgcn_exp2f(t); }
// the factor of e in the entropy's sum: finite where e is zero, so that 0 * t stays 0
__device__ __forceinline__ float an_floor(float t) { return fmaxf(t, -4096.f); }

// ---------------------------------------------------------------------------------------------
// A row cut into 16-byte pieces.
// ---------------------------------------------------------------------------------------------
template <bool BF16>
struct Piece {
  static constexpr int V = BF16 ? 8 : 4;
};
template <bool BF16>
__device__ __forceinline__ void an_unpack(const u32x4 r, float (&v)[Piece<BF16>::V]) {
  if constexpr (BF16) {
    v[0] = bf16_lo(r.x); v[1] = bf16_hi(r.x); v[2] = bf16_lo(r.y); v[3] = bf16_hi(r.y);
    v[4] = bf16_lo(r.z); v[5] = bf16_hi(r.z); v[6] = bf16_lo(r.w); v[7] = bf16_hi(r.w);
  } else {
    v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y);
    v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
  }
}

// Geometry of one row: its first element lies `shift` elements into piece 0.  A piece that reaches outside the memory of
// the whole matrix (at the very first or last row only) is read element by element.
struct Span {
  const unsigned char* first;   // address of piece 0
  int shift, pieces, C;
  int skip_lo, skip_hi;         // 1: piece 0 / the last piece reaches outside the matrix
};
template <bool BF16>
__device__ __forceinline__ Span an_span(const void* base, long ld, long row, long rows, int C) {
  constexpr int ES = BF16 ? 2 : 4;
  Span s;
  const unsigned char* b = reinterpret_cast<const unsigned char*>(base);
  const unsigned char* r = b + row * ld * ES;
  s.shift = (int)((reinterpret_cast<uintptr_t>(r) & 15u) / ES);
  s.first = r - s.shift * ES;
  s.pieces = (s.shift + C + Piece<BF16>::V - 1) / Piece<BF16>::V;
  s.C = C;
  s.skip_lo = s.first < b ? 1 : 0;
  s.skip_hi = s.first + (long)s.pieces * 16 > b + ((rows - 1) * ld + C) * ES ? 1 : 0;
  return s;
}
// The largest of two bf16 pairs as signed 16-bit integers: their order is that of the values as long as one of them is
// not negative (a negative result says that none was; NaN with a positive sign comes out above infinity).
typedef short s16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ unsigned an_pkmax(unsigned a, unsigned b) {
  return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(s16x2, a), __builtin_bit_cast(s16x2, b)));
}
// ... and where all are negative: the smallest as unsigned ones is the value nearest to zero
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ unsigned an_pkmin(unsigned a, unsigned b) {
  return __builtin_bit_cast(unsigned, __builtin_elementwise_min(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
__device__ __forceinline__ int an_pkmax1(unsigned a) {
  const int lo = (int)(short)a, hi = (int)a >> 16;
  return lo > hi ? lo : hi;
}
// Elements of piece c outside the row become -inf.  `el` = column of the piece's first element.
template <bool BF16>
__device__ __forceinline__ u32x4 an_mask(u32x4 r, int el, int C) {
  constexpr int V = Piece<BF16>::V;
  if (el < 0 || el + V > C) {
    unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const bool out = el + j < 0 || el + j >= C;
      if constexpr (BF16) {
        const unsigned keep = (j & 1) ? 0x0000ffffu : 0xffff0000u, put = (j & 1) ? 0xff800000u : 0x0000ff80u;
        w[j >> 1] = out ? ((w[j >> 1] & keep) | put) : w[j >> 1];
      } else {
        w[j] = out ? 0xff800000u : w[j];
      }
    }
    r = u32x4{w[0], w[1], w[2], w[3]};
  }
  return r;
}
// A piece that reaches outside the matrix, element by element.
template <bool BF16>
__device__ __forceinline__ u32x4 an_load_edge(const Span& s, int el) {
  constexpr int V = Piece<BF16>::V;
  const unsigned char* row = s.first + s.shift * (BF16 ? 2 : 4);
  unsigned w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (el + j >= 0 && el + j < s.C) {
      if constexpr (BF16) w[j >> 1] |= (unsigned)reinterpret_cast<const bf16_t*>(row)[el + j] << (16 * (j & 1));
      else w[j] = reinterpret_cast<const unsigned*>(row)[el + j];
    }
  }
  return u32x4{w[0], w[1], w[2], w[3]};
}

// The pieces id, id + NT, ... of a row, in registers (E > 0) or read again on every walk (E == 0).  The row belongs to a
// workgroup of NT threads, or (NT = 16) to sixteen lanes.
template <bool BF16, int NT, int E>
struct RowPieces {
  static constexpr int V = Piece<BF16>::V;
  Span s;
  u32x4 raw[E > 0 ? E : 1];

  static __device__ __forceinline__ int id() { return NT == 16 ? (int)threadIdx.x & 15 : (int)threadIdx.x; }
  // One piece.  A workgroup's rows have more than 1024 classes: pieces past the row, and those that reach outside the
  // matrix, read piece 1 instead, which lies inside the row.  Sixteen lanes' rows may be shorter: they read nothing then.
  __device__ __forceinline__ u32x4 fetch(int c) const {
    const bool safe = c >= s.skip_lo && c < s.pieces - s.skip_hi;
    if constexpr (NT == 16) {
      u32x4 r = {0, 0, 0, 0};
      if (safe) r = *reinterpret_cast<const u32x4*>(s.first + (size_t)((unsigned)c * 16u));
      return r;
    } else {
      return *reinterpret_cast<const u32x4*>(s.first + (size_t)(safe ? (unsigned)c * 16u : 16u));
    }
  }
  __device__ __forceinline__ u32x4 finish(u32x4 r, int c) const {
    const int el = c * V - s.shift;
    if (s.skip_lo + s.skip_hi != 0) {   // the first or the last row
      if ((c == 0 && s.skip_lo) || (c == s.pieces - 1 && s.skip_hi)) r = an_load_edge<BF16>(s, el);
    }
    return an_mask<BF16>(r, el, s.C);
  }
  __device__ __forceinline__ void load() {
    if constexpr (E > 0) {
#pragma unroll
      for (int i = 0; i < E; ++i) raw[i] = fetch(id() + i * NT);
#pragma unroll
      for (int i = 0; i < E; ++i) raw[i] = finish(raw[i], id() + i * NT);
    }
  }
  // The thread's largest value; NaN counts as the largest or not at all.
  __device__ __forceinline__ float max() const {
    return max_of([](const u32x4 r, int) { return r; });
  }
  // ... of the pieces as f(r, c) leaves them
  template <class F>
  __device__ __forceinline__ float max_of(F f) const {
    if constexpr (BF16) {
      unsigned k = 0x80008000u;   // the lowest pair
      walk_raw([&](const u32x4 p, int c, int) {
        const u32x4 r = f(p, c);
        k = an_pkmax(k, an_pkmax(an_pkmax(r.x, r.y), an_pkmax(r.z, r.w)));
      });
      const int b = an_pkmax1(k);
      if (b >= 0) return __uint_as_float((unsigned)b << 16);
      k = 0xff80ff80u;            // -inf
      walk_raw([&](const u32x4 p, int c, int) {
        const u32x4 r = f(p, c);
        k = an_pkmin(k, an_pkmin(an_pkmin(r.x, r.y), an_pkmin(r.z, r.w)));
      });
      return __uint_as_float(min(k & 0xffffu, k >> 16) << 16);
    } else {
      float m = -INFINITY;
      walk_raw([&](const u32x4 p, int c, int) {
        float v[V];
        an_unpack<BF16>(f(p, c), v);
#pragma unroll
        for (int j = 0; j < V; ++j) m = fmaxf(m, v[j]);
        if constexpr (E > 0) __builtin_amdgcn_sched_barrier(0);   // as in walk
      });
      return m;
    }
  }
  // whether a piece may hold a value of at least thr (it does, unless bf16 and thr <= 0)
  static __device__ __forceinline__ bool reaches(const u32x4 r, float thr) {
    if constexpr (BF16) {
      const int b = an_pkmax1(an_pkmax(an_pkmax(r.x, r.y), an_pkmax(r.z, r.w)));
      return !(thr > 0.f) || (b >= 0 && __uint_as_float((unsigned)b << 16) >= thr);
    } else {
      return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w))) >= thr;
    }
  }
  // f(v, el) for the pieces that may hold a value of at least thr, until it returns false: few, so they are read again
  // one by one (they are in the caches) rather than looked through in registers, which would unroll f for each of them
  template <class F>
  __device__ __forceinline__ void walk_reaching(float thr, F f) const {
    static_assert(E <= 64, "one bit for each piece");
    u64 hit = 0;
    if constexpr (E > 0) {
#pragma unroll
      for (int i = 0; i < E; ++i) hit |= reaches(raw[i], thr) ? 1ull << i : 0ull;
    }
    int c = id();
    while (E > 0 ? hit != 0 : c < s.pieces) {
      if (E > 0) {
        c = id() + (__ffsll((long long)hit) - 1) * NT;
        hit &= hit - 1;
      }
      const u32x4 r = c < s.pieces ? finish(fetch(c), c) : u32x4{0, 0, 0, 0};
      if (c < s.pieces && (E > 0 || reaches(r, thr))) {
        float v[V];
        an_unpack<BF16>(r, v);
        if (!f(v, c * V - s.shift)) break;
      }
      if (E == 0) c += NT;
    }
  }
  // Between two walks: the compiler sees the pieces as new, so that it unpacks them again (an instruction each) instead
  // of keeping the unpacked row, twice its size, alive from one walk to the next.
  __device__ __forceinline__ void renew() {
    if constexpr (E > 0) {
#pragma unroll
      for (int i = 0; i < E; ++i) asm volatile("" : "+v"(raw[i]));
    }
  }
  template <class F>
  __device__ __forceinline__ void walk_raw(F f) const {
    if constexpr (E > 0) {
#pragma unroll
      for (int i = 0; i < E; ++i) f(raw[i], id() + i * NT, (id() + i * NT) * V - s.shift);
    } else {
      for (int c = id(); c < s.pieces; c += NT) f(finish(fetch(c), c), c, c * V - s.shift);
    }
  }
  // f(v, c, el): the V values of piece c, the first of them in column el; columns outside [0, C) hold -inf
  template <class F>
  __device__ __forceinline__ void walk(F f) const {
    if constexpr (E > 0) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        float v[V];
        an_unpack<BF16>(raw[i], v);
        f(v, id() + i * NT, (id() + i * NT) * V - s.shift);
        __builtin_amdgcn_sched_barrier(0);   // one piece's temporaries at a time: other waves fill the gaps
      }
    } else {
      for (int c = id(); c < s.pieces; c += NT) {
        float v[V];
        an_unpack<BF16>(finish(fetch(c), c), v);
        f(v, c, c * V - s.shift);
      }
    }
  }
};

// whether the row holds a NaN (every thread of the workgroup calls; the row is read again)
template <bool BF16, int NT>
__device__ __forceinline__ bool an_block_nan(const Span& span) {
  constexpr int V = Piece<BF16>::V;
  RowPieces<BF16, NT, 0> row;
  row.s = span;
  int nan = 0;
  row.walk([&](const float (&v)[V], int, int) {
#pragma unroll
    for (int j = 0; j < V; ++j) nan |= v[j] != v[j] ? 1 : 0;
  });
  return __syncthreads_or(nan) != 0;
}

template <int V>
__device__ __forceinline__ float an_tree(const float (&v)[V]) {
  if constexpr (V == 8) return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
  else return (v[0] + v[1]) + (v[2] + v[3]);
}

template <bool BF16>
__device__ __forceinline__ float an_at(const void* row, long j) { return load1<BF16>(row, (size_t)j); }
template <bool BF16>
__device__ __forceinline__ const void* an_row(const void* base, long ld, long row) {
  return reinterpret_cast<const unsigned char*>(base) + row * ld * (BF16 ? 2 : 4);
}

// What a row's statistics give for one logit.  A row without a live entry (m = -inf) has log probability -inf
// everywhere; a NaN or +inf in the row makes all of it NaN.
__device__ __forceinline__ float an_logprob(float x, float m, double log_s, double inv_t) {
  if (m == -INFINITY) return -INFINITY;
  return (float)(((double)x - (double)m) * inv_t - log_s);
}

// rows of up to AN_WAVE_C classes: one wave per row, column lane + 64 i in register i
constexpr int AN_WAVES = 4;   // rows per workgroup

// maximum over the wave; NaN for a row that holds nothing else but -inf (the maximum leaves NaN out)
template <int E>
__device__ __forceinline__ float an_wave_row_max(const float (&v)[E], float m) {
  m = dpp_wave_max(m);
  if (m == -INFINITY) {
    bool nan = false;
#pragma unroll
    for (int i = 0; i < E; ++i) nan |= v[i] != v[i];
    if (__ballot(nan) != 0) m = NAN;
  }
  return m;
}

// ---------------------------------------------------------------------------------------------
// Gradients, streamed: the row's statistics are known, every logit is read once and its gradient written once.
// Entries of the row that something names (targets, alternatives, the teacher's answers) are written a second time,
// whole, after a barrier: a few 2- or 4-byte stores into lines that the workgroup has just written.  An entry named
// more than once is written by its first mention, which adds the others' terms in order.
// ---------------------------------------------------------------------------------------------
// the V gradients of a piece, into the row of the gradient that starts at the same place of its 16-byte grid
template <bool BF16>
__device__ __forceinline__ void an_store(unsigned char* grow, int el, int C, const float (&g)[Piece<BF16>::V]) {
  constexpr int V = Piece<BF16>::V;
  if (el >= 0 && el + V <= C) {
    u32x4 w;
    if constexpr (BF16) {
      w.x = pack_bf16x2(g[0], g[1]); w.y = pack_bf16x2(g[2], g[3]);
      w.z = pack_bf16x2(g[4], g[5]); w.w = pack_bf16x2(g[6], g[7]);
      *reinterpret_cast<u32x4*>(grow + (long)el * 2) = w;
    } else {
      w.x = __float_as_uint(g[0]); w.y = __float_as_uint(g[1]); w.z = __float_as_uint(g[2]); w.w = __float_as_uint(g[3]);
      *reinterpret_cast<u32x4*>(grow + (long)el * 4) = w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (el + j >= 0 && el + j < C) store1<BF16>(grow, (size_t)(el + j), g[j]);
  }
}

// Mentions in shared memory, `count` threads with number `id` share them: writes the entries in [from, to).  `repeats`:
// an entry may be named more than once.
template <bool BF16, class F, class G>
__device__ __forceinline__ void an_write_named(const int* idx, const float* add, int ns, bool repeats, int id, int count,
                                               int from, int to, const void* xr, unsigned char* grow, F base, G term) {
  for (int s = id; s < ns; s += count) {
    const int j = idx[s];
    if (j < from || j >= to) continue;
    bool first = true;
    float t = add[s];
    if (repeats) {
      t = 0.f;
      for (int o = 0; o < ns; ++o) {
        const bool same = idx[o] == j;
        if (same && o < s) first = false;
        if (same) t += add[o];
      }
    }
    if (first) store1<BF16>(grow, (size_t)j, base(an_at<BF16>(xr, j)) + term(t));
  }
}

constexpr int AN_ST = 256, AN_SP = 4;   // threads, pieces per thread of a streamed segment
constexpr int AN_NAMED = 2 * AN_TOP_MAX;

// A segment of 16 KB of a row for each workgroup.  Measured, 1001 x 50265 bf16: 37 us (5.5 TB/s read and written, the rate
// of a large copy); 511 x 50265 f32 with 100 named entries a row: 46 us (4.5 TB/s).
template <bool BF16, class OP>
__global__ __launch_bounds__(AN_ST) void answer_grad_block_kernel(const OP op, const void* x, long ld, long r0, long R, int C,
                                                                  int segments, void* grad, long ldg) {
  constexpr int V = Piece<BF16>::V;
  __shared__ int s_idx[AN_NAMED];
  __shared__ float s_add[AN_NAMED];
  if (op.done()) return;   // uniform
  const int in = (int)blockIdx.x / segments, seg = (int)blockIdx.x - in * segments, tid = threadIdx.x;
  const long r = r0 + in;
  RowPieces<BF16, AN_ST, 0> row;
  row.s = an_span<BF16>(x, ld, r, R, C);
  const int c0 = seg * (AN_ST * AN_SP);
  u32x4 raw[AN_SP];
#pragma unroll
  for (int i = 0; i < AN_SP; ++i) raw[i] = row.fetch(c0 + i * AN_ST + tid);
  const int ns = op.named();
  for (int s = tid; s < ns; s += AN_ST) op.mention(r, s, C, s_idx[s], s_add[s]);
  const typename OP::Row w = op.row(r, tid & 63, C);
  unsigned char* grow = reinterpret_cast<unsigned char*>(grad) + r * ldg * (BF16 ? 2 : 4);
#pragma unroll
  for (int i = 0; i < AN_SP; ++i) {
    const int c = c0 + i * AN_ST + tid, el = c * V - row.s.shift;
    if (c < row.s.pieces) {
      float v[V], g[V];
      an_unpack<BF16>(row.finish(raw[i], c), v);
#pragma unroll
      for (int j = 0; j < V; ++j) g[j] = OP::dense(w, v[j]);
      an_store<BF16>(grow, el, C, g);
    }
  }
  __syncthreads();
  const int from = c0 * V - row.s.shift;
  an_write_named<BF16>(s_idx, s_add, ns, ns > 1, tid, AN_ST, from < 0 ? 0 : from, min(C, from + AN_ST * AN_SP * V),
                       an_row<BF16>(x, ld, r), grow, [&](float v) { return OP::base(w, v); },
                       [&](float t) { return OP::term(w, t); });
}

// A wave to a row of up to 1024 classes.  Measured, log probabilities of 25000 x 430: bf16 21 us (2.0 TB/s: two bytes a lane),
// f32 18 us (4.8 TB/s).
template <bool BF16, int E, class OP>
__global__ __launch_bounds__(64 * AN_WAVES) void answer_grad_wave_kernel(const OP op, const void* x, long ld, long r0, long R,
                                                                         int C, void* grad, long ldg) {
  __shared__ int s_idx[AN_WAVES][AN_NAMED];
  __shared__ float s_add[AN_WAVES][AN_NAMED];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long r = r0 + (long)blockIdx.x * AN_WAVES + wave;
  if (r >= R || op.done()) return;   // no barrier below: a wave keeps to its own row
  const void* xr = an_row<BF16>(x, ld, r);
  float v[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int c = lane + 64 * i;
    v[i] = c < C ? an_at<BF16>(xr, c) : 0.f;
  }
  const int ns = op.named();
  for (int s = lane; s < ns; s += 64) op.mention(r, s, C, s_idx[wave][s], s_add[wave][s]);
  const typename OP::Row w = op.row(r, lane, C);
  unsigned char* grow = reinterpret_cast<unsigned char*>(grad) + r * ldg * (BF16 ? 2 : 4);
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int c = lane + 64 * i;
    if (c < C) store1<BF16>(grow, (size_t)c, OP::dense(w, v[i]));
  }
  __threadfence_block();
  __builtin_amdgcn_wave_barrier();
  an_write_named<BF16>(s_idx[wave], s_add[wave], ns, ns > 1, lane, 64, 0, C, xr, grow, [&](float u) { return OP::base(w, u); },
                       [&](float t) { return OP::term(w, t); });
}

// ---------------------------------------------------------------------------------------------
// Which kernel a row length takes
// ---------------------------------------------------------------------------------------------
// A launch may have fewer than 2^32 threads: calls f(first row, how many) for as many launches as the rows take, with
// `threads` for each row.
template <class F>
void an_by_launch(long R, long threads, F f) {
  const long most = (1L << 31) / threads;   // (a multiple of AN_WAVES)
  for (long r0 = 0; r0 < R; r0 += most) f(r0, R - r0 < most ? R - r0 : most);
}
// calls f(E) with the registers a lane needs for C classes, one wave per row
template <class F>
bool an_by_wave(int C, F f) {
  const int e = (C + 63) / 64;
  if (e <= 1) f(std::integral_constant<int, 1>());
  else if (e <= 2) f(std::integral_constant<int, 2>());
  else if (e <= 3) f(std::integral_constant<int, 3>());
  else if (e <= 4) f(std::integral_constant<int, 4>());
  else if (e <= 5) f(std::integral_constant<int, 5>());
  else if (e <= 6) f(std::integral_constant<int, 6>());
  else if (e <= 7) f(std::integral_constant<int, 7>());
  else if (e <= 8) f(std::integral_constant<int, 8>());
  else if (e <= 10) f(std::integral_constant<int, 10>());
  else if (e <= 12) f(std::integral_constant<int, 12>());
  else f(std::integral_constant<int, 16>());
  return true;
}
// calls f(NT, E) with the workgroup and pieces per thread that hold C classes wherever the row starts (a piece more
// than it fills when aligned); E = 0: the row is read again for every use
template <bool BF16, class F>
void an_by_block(int C, F f) {
  const int pieces = (C + Piece<BF16>::V - 1) / Piece<BF16>::V + 1;
#define AN_FIT(NT, E) if (pieces <= NT * E) return f(std::integral_constant<int, NT>(), std::integral_constant<int, E>())
  if constexpr (BF16) {
    AN_FIT(256, 2); AN_FIT(256, 4); AN_FIT(256, 8); AN_FIT(256, 12); AN_FIT(256, 16); AN_FIT(256, 20); AN_FIT(256, 25); AN_FIT(256, 33);
  } else {
    AN_FIT(256, 4); AN_FIT(256, 8); AN_FIT(256, 16); AN_FIT(256, 24); AN_FIT(256, 32); AN_FIT(256, 40); AN_FIT(256, 50); AN_FIT(512, 33);
  }
#undef AN_FIT
  return f(std::integral_constant<int, 1024>(), std::integral_constant<int, 0>());
}

// waves per SIMD to compile for: the pieces in registers and about 40 more
constexpr int an_waves(int e) {
  const int regs = 4 * e + 40, w = 512 / ((regs + 7) / 8 * 8);
  return w < 1 ? 1 : w > 8 ? 8 : w;
}

bool an_shape_ok(long ld, int R, int C, int K, double temperature) {
  // (temperatures between 2^-20 and 2^20: their factors stay far inside f32)
  return R > 0 && C > 0 && C <= (1 << 28) && ld >= 0 && K >= 0 && K <= AN_TOP_MAX && K <= C && temperature >= 9.5367431640625e-07 &&
         temperature <= 1048576.0;
}
// The gradient's rows have to lie on their 16-byte grid as the logits' do.
bool an_grad_layout_ok(const void* x, long ld, const void* g, long ldg, int C, int dtype) {
  const long es = (long)vqaf_esize(dtype);
  return ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(g)) & 15u) == 0 && ((ld - ldg) * es) % 16 == 0 && ldg >= C;
}
bool an_element_aligned(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % vqaf_esize(dtype) == 0; }

template <class OP>
int an_launch_grad(const OP& op, const void* x, long ld, int R, int C, int dtype, void* grad, long ldg, hipStream_t st) {
  if (C <= AN_WAVE_C) {
    an_by_wave(C, [&](auto e) {
      constexpr int E = decltype(e)::value;
      an_by_launch(R, 64, [&](long r0, long n) {
        const dim3 grid((unsigned)((n + AN_WAVES - 1) / AN_WAVES)), block(64 * AN_WAVES);
        if (dtype == VQAF_BF16) hipLaunchKernelGGL((answer_grad_wave_kernel<true, E, OP>), grid, block, 0, st, op, x, ld, r0, (long)R, C, grad, ldg);
        else hipLaunchKernelGGL((answer_grad_wave_kernel<false, E, OP>), grid, block, 0, st, op, x, ld, r0, (long)R, C, grad, ldg);
      });
    });
  } else {
    const int V = dtype == VQAF_BF16 ? 8 : 4;
    const long segments = ((long)C + V - 1 + (V - 1)) / V / (AN_ST * AN_SP) + 1;   // at most 2^16 (C <= 2^28)
    an_by_launch(R, AN_ST * segments, [&](long r0, long n) {
      const dim3 grid((unsigned)(segments * n));
      if (dtype == VQAF_BF16) hipLaunchKernelGGL((answer_grad_block_kernel<true, OP>), grid, dim3(AN_ST), 0, st, op, x, ld, r0, (long)R, C, (int)segments, grad, ldg);
      else hipLaunchKernelGGL((answer_grad_block_kernel<false, OP>), grid, dim3(AN_ST), 0, st, op, x, ld, r0, (long)R, C, (int)segments, grad, ldg);
    });
  }
  VQAF_LAUNCH_CHECK();
}

}  // namespace
