// What a model answers with: log probabilities of given tokens, the entropy of the answer distribution and its top
// alternatives (forward and backward), and the distillation loss against a teacher's top answers with its gradient.
// They score the answers for the membership attacks (attack/metric_src.py:302-426 reads a loss and a maximum per
// sample; these are the finer scores) and train a student on them in place of hard labels (utils/src.py:96).
//
// With z = x / T, m = max z, e_j = exp(z_j - m), S = sum_j e_j, p_j = e_j / S:
//   log p_t = z_t - m - log S            H = log S - sum_j e_j (z_j - m) / S
//   d log p_t / dx_j = (1{j = t} - p_j) / T            dH / dx_j = -p_j (log p_j + H) / T
// and for a teacher's answers i_k with probabilities q_k (rest r, held by no answer of the list):
//   L = T^2 [ sum_k q_k (log q_k - log p_{i_k}) + r (log r - log P) ],     P = sum of p_j outside the list
//   dL / dx_j = T [ p_j (sum q + r) - sum_{k: i_k = j} q_k ] on the list,  T p_j [ sum q + r - r / P ] elsewhere.
//
// All of it is bound by the row of logits: read once (and its gradient written once).  A row therefore stays in
// registers from its one read to its last use: rows of up to 1024 classes in one wave (four rows to a workgroup),
// longer ones in a workgroup of 256 to 1024 threads, which covers 65536 classes; longer rows are read again for each
// use.  Loads are whole 16-byte pieces on 16-byte addresses, whatever the row's own alignment (a vocabulary of 50265
// puts every second bf16 row on an odd address): the row is cut at the pieces' borders and what lies outside it is
// masked in registers.
//
// Precision.  The divergence of two close distributions is a small difference of large terms, so the normaliser, the
// entropy's sum and the loss are carried in 64 bits: sums of eight in f32, sums of those in f64; the exponent
// (x - m) log2(e) / T is formed with the two-term constant, because the rounding of a single one would shift every
// term of a row the same way.  Rows of one wave, whose few terms do not average their rounding out, take the
// exponential itself in f64 (a Taylor polynomial after range reduction; the f64 vector rate of this chip is the f32
// one).  Probabilities, and with them the gradients, are f32 and rounded once into their type.

#include <type_traits>

#include "common.h"

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

// ---------------------------------------------------------------------------------------------
// Wave reductions through DPP; the result is in every lane (read from lane 63).
// ---------------------------------------------------------------------------------------------
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned an_dpp(unsigned idle, unsigned x) {
  return (unsigned)__builtin_amdgcn_update_dpp((int)idle, (int)x, CTRL, ROWS, 0xf, false);
}
template <class F>
__device__ __forceinline__ unsigned an_wave_u32(unsigned x, unsigned idle, F f) {
  x = f(x, an_dpp<0x111, 0xf>(idle, x));
  x = f(x, an_dpp<0x112, 0xf>(idle, x));
  x = f(x, an_dpp<0x114, 0xf>(idle, x));
  x = f(x, an_dpp<0x118, 0xf>(idle, x));
  x = f(x, an_dpp<0x142, 0xa>(idle, x));
  x = f(x, an_dpp<0x143, 0xc>(idle, x));
  return (unsigned)__builtin_amdgcn_readlane((int)x, 63);
}
__device__ __forceinline__ float an_wave_max(float v) {
  return __uint_as_float(an_wave_u32(__float_as_uint(v), 0xff800000u, [](unsigned a, unsigned b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}
__device__ __forceinline__ unsigned an_wave_umax(unsigned v) {
  return an_wave_u32(v, 0u, [](unsigned a, unsigned b) { return a > b ? a : b; });
}
__device__ __forceinline__ unsigned an_wave_umin(unsigned v) {
  return an_wave_u32(v, 0xffffffffu, [](unsigned a, unsigned b) { return a < b ? a : b; });
}
__device__ __forceinline__ unsigned an_wave_uadd(unsigned v) {
  return an_wave_u32(v, 0u, [](unsigned a, unsigned b) { return a + b; });
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double an_dadd(double x) {
  const u64 u = __builtin_bit_cast(u64, x);
  const u64 o = ((u64)an_dpp<CTRL, ROWS>(0u, (unsigned)(u >> 32)) << 32) | an_dpp<CTRL, ROWS>(0u, (unsigned)u);
  return x + __builtin_bit_cast(double, o);   // idle lanes contribute +0
}
__device__ __forceinline__ double an_wave_sum(double x) {
  x = an_dadd<0x111, 0xf>(x);
  x = an_dadd<0x112, 0xf>(x);
  x = an_dadd<0x114, 0xf>(x);
  x = an_dadd<0x118, 0xf>(x);
  x = an_dadd<0x142, 0xa>(x);
  x = an_dadd<0x143, 0xc>(x);
  const u64 u = __builtin_bit_cast(u64, x);
  const u64 r = ((u64)(unsigned)__builtin_amdgcn_readlane((int)(u >> 32), 63) << 32) |
                (unsigned)__builtin_amdgcn_readlane((int)(unsigned)u, 63);
  return __builtin_bit_cast(double, r);
}

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

// the exponent's factor log2(e) / T in two f32 terms
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
// (x - m) log2(e) / T.  x = -inf gives -inf (the second term, of either sign, stays finite); NaN comes through the first.
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

// The pieces tid, tid + NT, ... of a row, in registers (E > 0) or read again on every walk (E == 0).
template <bool BF16, int NT, int E>
struct RowPieces {
  static constexpr int V = Piece<BF16>::V;
  Span s;
  u32x4 raw[E > 0 ? E : 1];

  // One piece.  Pieces past the row, and those that reach outside the matrix, read piece 1 instead, which lies inside
  // the row (rows here have more than 1024 classes).
  __device__ __forceinline__ u32x4 fetch(int c) const {
    const bool safe = c >= s.skip_lo && c < s.pieces - s.skip_hi;
    return *reinterpret_cast<const u32x4*>(s.first + (size_t)(safe ? (unsigned)c * 16u : 16u));
  }
  __device__ __forceinline__ u32x4 finish(u32x4 r, int c) const {
    const int el = c * V - s.shift;
    if (s.skip_lo + s.skip_hi != 0) {   // uniform
      if ((c == 0 && s.skip_lo) || (c == s.pieces - 1 && s.skip_hi)) r = an_load_edge<BF16>(s, el);
    }
    return an_mask<BF16>(r, el, s.C);
  }
  __device__ __forceinline__ void load() {
    if constexpr (E > 0) {
#pragma unroll
      for (int i = 0; i < E; ++i) raw[i] = fetch((int)threadIdx.x + i * NT);
#pragma unroll
      for (int i = 0; i < E; ++i) raw[i] = finish(raw[i], (int)threadIdx.x + i * NT);
    }
  }
  // The thread's largest value; NaN counts as the largest or not at all.
  __device__ __forceinline__ float max() const {
    if constexpr (BF16) {
      unsigned k = 0x80008000u;   // the lowest pair
      walk_raw([&](const u32x4 r, int, int) { k = an_pkmax(k, an_pkmax(an_pkmax(r.x, r.y), an_pkmax(r.z, r.w))); });
      const int b = an_pkmax1(k);
      if (b >= 0) return __uint_as_float((unsigned)b << 16);
      k = 0xff80ff80u;            // -inf
      walk_raw([&](const u32x4 r, int, int) { k = an_pkmin(k, an_pkmin(an_pkmin(r.x, r.y), an_pkmin(r.z, r.w))); });
      return __uint_as_float(min(k & 0xffffu, k >> 16) << 16);
    } else {
      float m = -INFINITY;
      walk([&](const float (&v)[V], int, int) {
#pragma unroll
        for (int j = 0; j < V; ++j) m = fmaxf(m, v[j]);
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
  // f(v, el) for the pieces that may hold a value of at least thr: few, so they are read again one by one (they are in
  // the caches) rather than looked through in registers, which would unroll f once for each of them
  template <class F>
  __device__ __forceinline__ void walk_reaching(float thr, F f) const {
    static_assert(E <= 64, "one bit for each piece");
    u64 hit = 0;
    if constexpr (E > 0) {
#pragma unroll
      for (int i = 0; i < E; ++i) hit |= reaches(raw[i], thr) ? 1ull << i : 0ull;
    }
    int c = threadIdx.x;
    while (E > 0 ? hit != 0 : c < s.pieces) {
      if (E > 0) {
        c = (int)threadIdx.x + (__ffsll((long long)hit) - 1) * NT;
        hit &= hit - 1;
      }
      const u32x4 r = c < s.pieces ? finish(fetch(c), c) : u32x4{0, 0, 0, 0};
      if (c < s.pieces && (E > 0 || reaches(r, thr))) {
        float v[V];
        an_unpack<BF16>(r, v);
        f(v, c * V - s.shift);
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
      for (int i = 0; i < E; ++i) f(raw[i], (int)threadIdx.x + i * NT, ((int)threadIdx.x + i * NT) * V - s.shift);
    } else {
      for (int c = threadIdx.x; c < s.pieces; c += NT) f(finish(fetch(c), c), c, c * V - s.shift);
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
        f(v, (int)threadIdx.x + i * NT, ((int)threadIdx.x + i * NT) * V - s.shift);
        __builtin_amdgcn_sched_barrier(0);   // one piece's temporaries at a time: other waves fill the gaps
      }
    } else {
      for (int c = threadIdx.x; c < s.pieces; c += NT) {
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

// ---------------------------------------------------------------------------------------------
// Log probabilities: one workgroup per row
// ---------------------------------------------------------------------------------------------
struct LogprobArgs {
  const void* x;
  const int64_t* targets;
  float* logprobs;
  float* entropy;
  float* top_logprobs;
  int64_t* top_indices;
  float* stats;   // (R,2): m, S
  long ld, R;
  int C, T, K;
  AnTemp temp;
};

template <int NT>
struct TopShared {
  float tmax[NT];
  u64 cand[AN_CAP];
  int rank[AN_CAP];
  int n;
  float thr;
  int cnt[2];
};

// how many of the workgroup's elements pass `f` (all threads call; two barriers)
template <int NT, class ROW, class F>
__device__ __forceinline__ int an_block_count(const ROW& row, int* cnt, F f) {
  constexpr int V = ROW::V;
  __syncthreads();
  if (threadIdx.x == 0) cnt[0] = 0;
  __syncthreads();
  unsigned n = 0;
  row.walk([&](const float (&v)[V], int, int el) {
#pragma unroll
    for (int j = 0; j < V; ++j) n += (el + j >= 0 && el + j < row.s.C && f(v[j], el + j)) ? 1u : 0u;
  });
  n = an_wave_uadd(n);
  if ((threadIdx.x & 63) == 0) atomicAdd(&cnt[0], (int)n);
  __syncthreads();
  return cnt[0];
}

// The K best of a row into sh.cand, by counting alone: the K-th key bit by bit, then the index up to which elements
// equal to it belong.  For rows whose candidates overflow the list (long ties: a masked row has nothing but) and rows
// with NaN; 63 passes at most.
template <bool BF16, int NT>
__device__ __forceinline__ void an_top_by_counting(const Span& span, TopShared<NT>& sh, int K) {
  constexpr int V = Piece<BF16>::V;
  RowPieces<BF16, NT, 0> row;   // reads the row again: the common path's registers stay its own
  row.s = span;
  unsigned t = 0;
  for (int b = 31; b >= 0; --b) {
    const unsigned mid = t | (1u << b);
    if (an_block_count<NT>(row, sh.cnt, [&](float x, int) { return an_key(x) >= mid; }) >= K) t = mid;
  }
  const int above = an_block_count<NT>(row, sh.cnt, [&](float x, int) { return an_key(x) > t; });
  const int need = K - above;   // of the elements equal to t, >= 1
  int last = 0;                 // the lowest index bound that admits `need` of them: [0, last]
  {
    int lo = 0, hi = row.s.C - 1;
    while (lo < hi) {
      const int mid = lo + ((hi - lo) >> 1);
      if (an_block_count<NT>(row, sh.cnt, [&](float x, int j) { return an_key(x) == t && j <= mid; }) >= need) hi = mid;
      else lo = mid + 1;
    }
    last = lo;
  }
  __syncthreads();
  if (threadIdx.x == 0) sh.n = 0;
  __syncthreads();
  row.walk([&](const float (&v)[V], int, int el) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int col = el + j;
      if (col < 0 || col >= row.s.C) continue;
      const unsigned k = an_key(v[j]);
      if (k > t || (k == t && col <= last)) sh.cand[atomicAdd(&sh.n, 1) & (AN_CAP - 1)] = an_pack(k, col);
    }
  });
  __syncthreads();
}

// Wave 0: a value that at least K, and not many more than K, of the threads' maxima reach.  At least K elements of the
// row reach it then, and the elements that do lie with few threads.
template <int NT>
__device__ __forceinline__ float an_threshold(const float* tmax, int threads_with_data, int K) {
  constexpr int PER = NT / 64;
  const int lane = threadIdx.x & 63;
  unsigned k[PER];
  unsigned lo = 0xffffffffu, hi = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int t = i * 64 + lane;
    k[i] = t < threads_with_data ? an_key(tmax[t]) : 0u;
  }
  unsigned best = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) best = k[i] > best ? k[i] : best;
  hi = an_wave_umax(best);
  lo = an_wave_umin(best);                      // 64 maxima reach it if every lane has one
  if (K > 64 || lo < AN_KEY_MINF) lo = AN_KEY_MINF;
  const int most = K + (K >> 1) + 16;
  // invariant: at least K maxima are >= lo; fewer than K are >= hi + 1
  unsigned up = hi;
  while (lo < up) {
    const unsigned mid = lo + ((up - lo) >> 1) + 1;
    int c = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) c += __popcll(__ballot(k[i] >= mid));
    if (c >= K) {
      lo = mid;
      if (c <= most) break;
    } else {
      up = mid - 1;
    }
  }
  return an_unkey(lo);
}

template <bool BF16, int NT, int E, int W>
__global__ __launch_bounds__(NT, W) void logprob_block_kernel(const LogprobArgs a) {
  constexpr int V = Piece<BF16>::V, NW = NT / 64;
  __shared__ TopShared<NT> sh;
  __shared__ float s_max[NW];
  __shared__ double s_sum[2][NW];
  const long r = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  RowPieces<BF16, NT, E> row;
  row.s = an_span<BF16>(a.x, a.ld, r, a.R, a.C);
  row.load();

  float m = row.max();
  row.renew();
  if (a.K > 0) {
    sh.tmax[tid] = m;
    if (tid == 0) sh.n = 0;
    for (int i = tid; i < AN_CAP; i += NT) sh.rank[i] = 0;
  }
  m = an_wave_max(m);
  if (lane == 0) s_max[wave] = m;
  __syncthreads();
  m = s_max[0];
#pragma unroll
  for (int i = 1; i < NW; ++i) m = fmaxf(m, s_max[i]);
  if (m == -INFINITY && an_block_nan<BF16, NT>(row.s)) m = NAN;   // (the maximum may leave NaN out)

  // one factor only: what its rounding shifts is taken out of log S below, to first order
  double S = 0.0, Wt = 0.0;
  const float hi = a.temp.hi;
  row.walk([&](const float (&v)[V], int, int) {
    float e[V], w[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float t = (v[j] - m) * hi;
      e[j] = an_exp2(t);
      w[j] = e[j] * an_floor(t);
    }
    S += (double)an_tree<V>(e);
    Wt += (double)an_tree<V>(w);
  });
  S = an_wave_sum(S);
  Wt = an_wave_sum(Wt);
  if (lane == 0) {
    s_sum[0][wave] = S;
    s_sum[1][wave] = Wt;
  }
  if (a.K > 0 && wave == 0) {
    const float t = an_threshold<NT>(sh.tmax, row.s.pieces < NT ? row.s.pieces : NT, a.K);
    if (lane == 0) sh.thr = t;
  }
  __syncthreads();
  S = s_sum[0][0];
  Wt = s_sum[1][0];
#pragma unroll
  for (int i = 1; i < NW; ++i) {
    S += s_sum[0][i];
    Wt += s_sum[1][i];
  }
  const bool empty = m == -INFINITY;
  const bool broken = !empty && !(S == S);   // a NaN or +inf in the row
  const double mean_t = AN_LN2 * (Wt / S);
  const double log_s = empty ? -INFINITY : log(S) - a.temp.delta * mean_t;
  const void* xr = an_row<BF16>(a.x, a.ld, r);
  if (tid == 0) {
    if (a.entropy != nullptr) a.entropy[r] = empty ? 0.f : (float)(log_s - mean_t * (1.0 - a.temp.delta));
    if (a.stats != nullptr) {
      a.stats[2 * r] = m;
      a.stats[2 * r + 1] = empty ? 1.f : (float)(S * (1.0 - a.temp.delta * mean_t));
    }
  }
  for (int i = tid; i < a.T; i += NT) {
    const int64_t t = a.targets[r * a.T + i];
    float lp = 0.f;                                         // a negative target is none
    if (t >= a.C) lp = NAN;
    else if (t >= 0) lp = an_logprob(an_at<BF16>(xr, t), m, log_s, a.temp.inv_t);
    a.logprobs[r * a.T + i] = lp;
  }
  if (a.K == 0) return;

  // candidates: what reaches the threshold
  row.renew();
  bool counted = broken;
  if (!broken) {
    const float thr = sh.thr;
    if (sh.tmax[tid] >= thr) {
      row.walk_reaching(thr, [&](const float (&v)[V], int el) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (v[j] >= thr && el + j >= 0 && el + j < a.C) {
            const int at = atomicAdd(&sh.n, 1);
            if (at < AN_CAP) sh.cand[at] = an_pack(an_key(v[j]), el + j);
          }
        }
      });
    }
    __syncthreads();
    counted = sh.n > AN_CAP;   // uniform
  }
  if (counted) an_top_by_counting<BF16, NT>(row.s, sh, a.K);
  const int n = sh.n;
  // rank of each candidate: how many are before it.  The list is cut among the threads left over.
  int npad = 64;
  while (npad < n) npad <<= 1;
  if (npad <= NT) {
    const int parts = NT / npad, i = tid & (npad - 1), p = tid / npad;
    if (i < n) {
      const u64 mine = sh.cand[i];
      int before = 0;
      for (int j = p; j < n; j += parts) before += sh.cand[j] > mine ? 1 : 0;
      if (before > 0) atomicAdd(&sh.rank[i], before);
    }
  } else {
    for (int i = tid; i < n; i += NT) {
      const u64 mine = sh.cand[i];
      int before = 0;
      for (int j = 0; j < n; ++j) before += sh.cand[j] > mine ? 1 : 0;
      sh.rank[i] = before;
    }
  }
  __syncthreads();
  for (int i = tid; i < n; i += NT) {
    const int k = sh.rank[i];
    if (k < a.K) {
      const int j = an_index(sh.cand[i]);
      a.top_indices[r * a.K + k] = j;
      a.top_logprobs[r * a.K + k] = an_logprob(an_at<BF16>(xr, j), m, log_s, a.temp.inv_t);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Log probabilities: one wave per row of up to 1024 classes, column lane + 64 i in register i
// ---------------------------------------------------------------------------------------------
constexpr int AN_WAVES = 4;   // rows per workgroup

// maximum over the wave; NaN for a row that holds nothing else but -inf (the maximum leaves NaN out)
template <int E>
__device__ __forceinline__ float an_wave_row_max(const float (&v)[E], float m) {
  m = an_wave_max(m);
  if (m == -INFINITY) {
    bool nan = false;
#pragma unroll
    for (int i = 0; i < E; ++i) nan |= v[i] != v[i];
    if (__ballot(nan) != 0) m = NAN;
  }
  return m;
}

constexpr int AN_WCAP = 256;   // candidates a wave lists

// Exactly the K best of a row of keys (0: none), by bisection over the keys and then in the order of the index, into
// cand[0..K).  From `low`, which at least K keys reach.
template <int E>
__device__ __forceinline__ void an_wave_select(const unsigned (&key)[E], unsigned low, int K, u64* cand) {
  const int lane = threadIdx.x & 63;
  unsigned best = key[0];
#pragma unroll
  for (int i = 1; i < E; ++i) best = key[i] > best ? key[i] : best;
  unsigned up = an_wave_umax(best);
  while (low < up) {
    const unsigned mid = low + ((up - low) >> 1) + 1;
    int c = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) c += __popcll(__ballot(key[i] >= mid));
    if (c >= K) {
      low = mid;
      if (c == K) break;
    } else {
      up = mid - 1;
    }
  }
  int n = 0, above = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) above += __popcll(__ballot(key[i] > low));
  int ties = K - above;   // of those equal to it, the first (all of them where the count was exact)
  const u64 below_lane = (1ull << lane) - 1ull;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const u64 eq = __ballot(key[i] == low);
    const bool take = key[i] > low || (key[i] == low && __popcll(eq & below_lane) < ties);
    const u64 who = __ballot(take);
    if (take) cand[n + __popcll(who & below_lane)] = an_pack(key[i], lane + 64 * i);
    n += __popcll(who);
    ties -= __popcll(eq);
    ties = ties < 0 ? 0 : ties;
  }
}

template <bool BF16, int E>
__global__ __launch_bounds__(64 * AN_WAVES) void logprob_wave_kernel(const LogprobArgs a) {
  __shared__ u64 s_cand[AN_WAVES][AN_WCAP];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long r = (long)blockIdx.x * AN_WAVES + wave;
  if (r >= a.R) return;   // no barrier below: a wave keeps to its own row
  const void* xr = an_row<BF16>(a.x, a.ld, r);
  float v[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int c = lane + 64 * i;
    v[i] = c < a.C ? an_at<BF16>(xr, c) : -INFINITY;
  }
  int64_t t = -1;
  if (lane < a.T) t = a.targets[r * a.T + lane];   // the first 64; more are read below
  float best = -INFINITY;
#pragma unroll
  for (int i = 0; i < E; ++i) best = fmaxf(best, v[i]);
  const float m = an_wave_row_max<E>(v, best);
  const bool empty = m == -INFINITY;
  double S = 0.0, Wt = 0.0;
  const float hi = a.temp.hi;
#pragma unroll
  for (int i0 = 0; i0 < E; i0 += 8) {   // eight at a time in f32, as in the longer rows
    float es = 0.f, ws = 0.f;
#pragma unroll
    for (int i = i0; i < E && i < i0 + 8; ++i) {
      const float u = (v[i] - m) * hi, e = an_exp2(u);
      es += e;
      ws = fmaf(e, an_floor(u), ws);
    }
    S += (double)es;
    Wt += (double)ws;
  }
  S = an_wave_sum(S);
  Wt = an_wave_sum(Wt);
  const double mean_t = AN_LN2 * (Wt / S);
  const double log_s = empty ? -INFINITY : log(S) - a.temp.delta * mean_t;
  if (lane == 0) {
    if (a.entropy != nullptr) a.entropy[r] = empty ? 0.f : (float)(log_s - mean_t * (1.0 - a.temp.delta));
    if (a.stats != nullptr) {
      a.stats[2 * r] = m;
      a.stats[2 * r + 1] = empty ? 1.f : (float)(S * (1.0 - a.temp.delta * mean_t));
    }
  }
  for (int i = lane; i < a.T; i += 64) {
    if (i >= 64) t = a.targets[r * a.T + i];
    float lp = 0.f;
    if (t >= a.C) lp = NAN;
    else if (t >= 0) lp = an_logprob(an_at<BF16>(xr, t), m, log_s, a.temp.inv_t);
    a.logprobs[r * a.T + i] = lp;
  }
  if (a.K == 0) return;

  // What the K-th largest of the lanes' maxima reaches is a short list that holds the K best.  Long ties, NaN and
  // longer lists go by the keys of all elements.
  u64* cand = s_cand[wave];
  const bool broken = !empty && !(S == S);
  int n = AN_WCAP + 1;
  if (a.K <= 64 && !broken) {
    const unsigned mine = lane < a.C ? an_key(best) : 0u;   // (lanes past a short row have none)
    unsigned up = an_wave_umax(mine), low = an_wave_umin(mine);
    if (low < AN_KEY_MINF) low = AN_KEY_MINF;
    while (low < up) {
      const unsigned mid = low + ((up - low) >> 1) + 1;
      const int c = __popcll(__ballot(mine >= mid));
      if (c >= a.K) {
        low = mid;
        if (c == a.K) break;
      } else {
        up = mid - 1;
      }
    }
    const float thr = an_unkey(low);
    n = 0;
    const u64 below_lane = (1ull << lane) - 1ull;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const bool take = v[i] >= thr && lane + 64 * i < a.C;
      const u64 who = __ballot(take);
      if (who != 0) {
        const int at = n + __popcll(who & below_lane);
        if (take && at < AN_WCAP) cand[at] = an_pack(an_key(v[i]), lane + 64 * i);
        n += __popcll(who);
      }
    }
  }
  if (n > AN_WCAP) {
    unsigned key[E];
#pragma unroll
    for (int i = 0; i < E; ++i) key[i] = lane + 64 * i < a.C ? an_key(v[i]) : 0u;
    an_wave_select<E>(key, AN_KEY_MINF, a.K, cand);
    n = a.K;
  }
  __builtin_amdgcn_wave_barrier();
  __threadfence_block();
  for (int i = lane; i < n; i += 64) {
    const u64 mine = cand[i];
    int before = 0;
    for (int j = 0; j < n; ++j) before += cand[j] > mine ? 1 : 0;
    if (before < a.K) {
      a.top_indices[r * a.K + before] = an_index(mine);
      a.top_logprobs[r * a.K + before] = an_logprob(an_unkey((unsigned)(mine >> 32)), m, log_s, a.temp.inv_t);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Gradients, streamed: the row's statistics are known, every logit is read once and its gradient written once.
// Entries of the row that something names (targets, alternatives, the teacher's answers) are written a second time,
// whole, after a barrier: a few 2- or 4-byte stores into lines that the workgroup has just written.  An entry named
// more than once is written by its first mention, which adds the others' terms in order.
// ---------------------------------------------------------------------------------------------
struct LogprobGrad {
  const int64_t* targets;
  const int64_t* top_indices;
  const float* stats;
  const float* entropy;
  const float* g_lp;
  const float* g_ent;
  const float* g_top;
  int T, K;
  AnTemp temp;
  // of the row
  struct Row {
    float m, inv_s, log_s, A, h, H, hi, lo, inv_t;
    bool empty;
  };
  __device__ __forceinline__ bool done() const { return false; }
  __device__ __forceinline__ int named() const { return (g_lp != nullptr ? T : 0) + (g_top != nullptr ? K : 0); }
  __device__ __forceinline__ void mention(long r, int s, int C, int& idx, float& add) const {
    const int t = g_lp != nullptr ? T : 0;
    int64_t j;
    float g;
    if (s < t) {
      j = targets[r * T + s];
      g = g_lp[r * T + s];
      if (j < 0) g = 0.f;        // no target: no gradient
      if (j >= C) g = NAN;       // outside the classes: the row says so
    } else {
      j = top_indices[r * K + (s - t)];
      g = g_top[r * K + (s - t)];
    }
    idx = j >= 0 && j < C ? (int)j : -1;
    add = g;
  }
  __device__ __forceinline__ Row row(long r, int lane, int C) const {
    Row w;
    w.m = stats[2 * r];
    const float S = stats[2 * r + 1];
    w.inv_s = 1.0f / S;
    w.log_s = logf(S);
    w.H = entropy != nullptr ? entropy[r] : 0.f;
    w.h = g_ent != nullptr ? g_ent[r] : 0.f;
    double sum = 0.0;
    for (int s = lane; s < named(); s += 64) {
      int j;
      float g;
      mention(r, s, C, j, g);
      sum += (double)g;
    }
    w.A = (float)an_wave_sum(sum);
    w.hi = temp.hi;
    w.lo = temp.lo;
    w.inv_t = (float)temp.inv_t;
    w.empty = w.m == -INFINITY;
    return w;
  }
  static __device__ __forceinline__ float dense(const Row& w, float x) {
    if (w.empty) return 0.f;
    const float t = an_arg(x, w.m, w.hi, w.lo);
    const float p = an_exp2(t) * w.inv_s;
    const float lp = fmaf(an_floor(t), (float)AN_LN2, -w.log_s);
    return -w.inv_t * (p * fmaf(w.h, lp + w.H, w.A));
  }
  static __device__ __forceinline__ float base(const Row& w, float x) { return dense(w, x); }
  static __device__ __forceinline__ float term(const Row& w, float g) { return w.empty ? 0.f : w.inv_t * g; }
};

// (R,5) f64: m, S, mass = sum q + r, slope = mass - r / P, log Q (q_k = exp(v_k - log Q))
struct DistillStat {
  double m, S, mass, slope, log_q;
};

// a row that is all masked, or that no answer teaches (whatever its logits hold)
__device__ __forceinline__ bool an_no_gradient(const DistillStat& s) {
  return s.m == -INFINITY || (s.mass == 0.0 && s.slope == 0.0);
}

struct DistillGrad {
  const float* teacher;
  const int64_t* indices;
  const DistillStat* stats;
  const float* up;     // gradient of the loss, one per row (up_step 1) or one (0)
  int up_step, K, skip_unit;   // skip_unit: nothing is left to do where up[0] is 1 (the gradient is there already)
  float scale;         // T * (1 for a sum, 1 / R for a mean)
  AnTemp temp;
  struct Row {
    float m, mass, slope, hi, lo, g;
    double log_q;
    bool empty;
  };
  __device__ __forceinline__ bool done() const { return skip_unit && up[0] == 1.0f; }
  __device__ __forceinline__ int named() const { return K; }
  __device__ __forceinline__ void mention(long r, int s, int C, int& idx, float& add) const {
    const int64_t j = indices[r * K + s];
    idx = j >= 0 && j < C ? (int)j : -1;
    add = (float)an_exp((double)teacher[r * K + s] - stats[r].log_q);
  }
  __device__ __forceinline__ Row row(long r, int, int) const {
    Row w;
    const DistillStat s = stats[r];
    w.m = (float)s.m;
    w.empty = an_no_gradient(s);
    const double inv = w.empty ? 0.0 : 1.0 / s.S;
    w.mass = (float)(s.mass * inv);
    w.slope = (float)(s.slope * inv);
    w.hi = temp.hi;
    w.lo = temp.lo;
    w.g = scale * up[r * up_step];
    return w;
  }
  static __device__ __forceinline__ float dense(const Row& w, float x) {
    return w.empty ? 0.f : w.g * (an_exp2(an_arg(x, w.m, w.hi, w.lo)) * w.slope);
  }
  static __device__ __forceinline__ float base(const Row& w, float x) {
    return w.empty ? 0.f : w.g * (an_exp2(an_arg(x, w.m, w.hi, w.lo)) * w.mass);
  }
  static __device__ __forceinline__ float term(const Row& w, float q) { return w.empty ? 0.f : -w.g * q; }
};

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

template <bool BF16, class OP>
__global__ __launch_bounds__(AN_ST) void answer_grad_block_kernel(const OP op, const void* x, long ld, long R, int C, int segments,
                                                                  void* grad, long ldg) {
  constexpr int V = Piece<BF16>::V;
  __shared__ int s_idx[AN_NAMED];
  __shared__ float s_add[AN_NAMED];
  if (op.done()) return;   // uniform
  const long r = blockIdx.x / segments;
  const int seg = (int)(blockIdx.x - r * segments), tid = threadIdx.x;
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

template <bool BF16, int E, class OP>
__global__ __launch_bounds__(64 * AN_WAVES) void answer_grad_wave_kernel(const OP op, const void* x, long ld, long R, int C,
                                                                         void* grad, long ldg) {
  __shared__ int s_idx[AN_WAVES][AN_NAMED];
  __shared__ float s_add[AN_WAVES][AN_NAMED];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long r = (long)blockIdx.x * AN_WAVES + wave;
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
// Distillation loss, with the gradient of the sum (or mean) in the same pass
// ---------------------------------------------------------------------------------------------
struct DistillArgs {
  const void* x;
  const float* teacher;
  const int64_t* indices;
  float* row_loss;
  DistillStat* stats;   // or NULL
  void* grad;           // or NULL
  long ld, ldg, R;
  int C, K, tail;
  float scale;          // of the gradient: T * (1 or 1 / R)
  double t2;            // T^2
  AnTemp temp;
};

// A row's list of answers in shared memory: the teacher's log probability, the student's logit, the class (-1: none),
// whether an earlier entry names it too, and, in the end, the teacher's probability.
struct DistillList {
  float v[AN_TOP_MAX], x[AN_TOP_MAX], q[AN_TOP_MAX];
  int idx[AN_TOP_MAX], again[AN_TOP_MAX];
};

// One wave: the row's statistics and loss from the sum of e over the classes outside the list (s_out) or, without a tail,
// over all of them (s_all).  `all`: the list covers every class; `bad`: an answer lies past the classes.
// Short loops on purpose: the pieces of the row are alive around this.
__device__ __forceinline__ DistillStat an_distill_row(DistillList& list, int K, bool bad, float m, double s_all, double s_out,
                                                      bool all, bool tail, double inv_t, double& loss) {
  const int lane = threadIdx.x & 63;
  const bool empty = m == -INFINITY;
  DistillStat st;
  st.m = m;
  st.S = s_all;
  st.log_q = 0.0;
  bool some = true;
  if (tail) {
    double own = 0.0;
#pragma unroll 1
    for (int k = lane; k < K; k += 64)
      if (list.idx[k] >= 0 && !list.again[k]) own += an_exp(((double)list.x[k] - (double)m) * inv_t);
    st.S = s_out + an_wave_sum(own);
  } else {
    float vm = -INFINITY;
    bool nan = false;
#pragma unroll 1
    for (int k = lane; k < K; k += 64) {
      if (list.idx[k] < 0) continue;
      vm = fmaxf(vm, list.v[k]);
      nan |= list.v[k] != list.v[k];
    }
    vm = an_wave_max(vm);
    // (a NaN among the values is left out of the maximum and comes back through the sum)
    some = vm != -INFINITY || __ballot(nan) != 0;
    if (some) {
      double sum = 0.0;
#pragma unroll 1
      for (int k = lane; k < K; k += 64) sum += list.idx[k] >= 0 ? an_exp((double)list.v[k] - (double)vm) : 0.0;
      st.log_q = (double)vm + log(an_wave_sum(sum));
    }
  }
  const double log_s = log(st.S);
  double mass = 0.0, l = 0.0;
  bool any = false;
#pragma unroll 1
  for (int k = lane; k < K; k += 64) {
    const bool live = list.idx[k] >= 0;
    const double lq = (double)list.v[k] - st.log_q;
    const double q = live && some ? an_exp(lq) : 0.0;
    const double lp = empty ? -INFINITY : ((double)list.x[k] - (double)m) * inv_t - log_s;
    any |= live;
    mass += q;
    if (q != 0.0) l += q * (lq - lp);   // (NaN goes in)
    list.q[k] = (float)q;
  }
  mass = an_wave_sum(mass);
  l = an_wave_sum(l);
  double cut = 0.0;
  if (tail) {
    double rest = all || __ballot(any) == 0 ? 0.0 : 1.0 - mass;   // (a row without answers teaches nothing)
    if (!(rest > (double)AN_NO_REST)) rest = 0.0;
    mass += rest;
    if (rest > 0.0) {
      if (empty) {
        l += INFINITY;
      } else {
        const double P = s_out / st.S;
        l += rest * (log(rest) - log(P));
        cut = P > 0.0 ? rest / P : (P == 0.0 ? mass : P);
      }
    }
  } else if (some) {
    mass = mass / mass;   // 1, or NaN
  }
  if (bad) l = mass = NAN;
  st.mass = mass;
  st.slope = mass - cut;
  loss = l;
  return st;
}

template <int NT>
struct DistillShared {
  DistillList list;
  float s_max[NT / 64];
  double s_sum[NT / 64];
  int bad, repeats;
  DistillStat st;
};

// The elements of a piece whose bits are set become -inf.
template <bool BF16>
__device__ __forceinline__ u32x4 an_drop(u32x4 r, unsigned bits) {
  unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int j = 0; j < Piece<BF16>::V; ++j) {
    const bool out = (bits >> j) & 1u;
    if constexpr (BF16) {
      const unsigned keep = (j & 1) ? 0x0000ffffu : 0xffff0000u, put = (j & 1) ? 0xff800000u : 0x0000ff80u;
      w[j >> 1] = out ? ((w[j >> 1] & keep) | put) : w[j >> 1];
    } else {
      w[j] = out ? 0xff800000u : w[j];
    }
  }
  return u32x4{w[0], w[1], w[2], w[3]};
}

// One workgroup per row.  The classes of the list are marked in a bitmap (in units of pieces).  TAIL: their elements are
// taken out of the registers before the exponentials, so that the rest is summed by itself (1 - sum p would lose what is
// left of it where the student agrees with its teacher), and their own terms are added by the list.
// HOLD: the exponentials stay in registers for the gradient (f32: in the place of the logits; bf16: in twice the
// registers, where that still leaves two workgroups to a CU); otherwise they are formed again.
template <bool BF16, int NT, int E, bool TAIL, bool HOLD, int W>
__global__ __launch_bounds__(NT, W) void distill_block_kernel(const DistillArgs a) {
  constexpr int V = Piece<BF16>::V, NW = NT / 64;
  __shared__ DistillShared<NT> sh;
  extern __shared__ unsigned s_mark[];   // one bit per element of the pieces
  const long r = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  RowPieces<BF16, NT, E> row;
  row.s = an_span<BF16>(a.x, a.ld, r, a.R, a.C);
  row.load();
  const void* xr = an_row<BF16>(a.x, a.ld, r);
  for (int i = tid; i < (row.s.pieces * V + 31) / 32; i += NT) s_mark[i] = 0u;
  if (tid == 0) sh.bad = sh.repeats = 0;
  __syncthreads();
  if (tid < a.K) {
    const int64_t j = a.indices[r * a.K + tid];
    const bool live = j >= 0 && j < a.C;
    int again = 0;
    sh.list.idx[tid] = live ? (int)j : -1;
    sh.list.v[tid] = a.teacher[r * a.K + tid];
    sh.list.x[tid] = live ? an_at<BF16>(xr, j) : 0.f;
    if (j >= a.C) sh.bad = 1;
    if (live) {
      const int b = (int)j + row.s.shift;
      again = (atomicOr(&s_mark[b >> 5], 1u << (b & 31)) >> (b & 31)) & 1u;
      if (again) sh.repeats = 1;
    }
    sh.list.again[tid] = again;
  }
  float m = an_wave_max(row.max());
  row.renew();
  if (lane == 0) sh.s_max[wave] = m;
  __syncthreads();
  m = sh.s_max[0];
#pragma unroll
  for (int i = 1; i < NW; ++i) m = fmaxf(m, sh.s_max[i]);
  if (m == -INFINITY && an_block_nan<BF16, NT>(row.s)) m = NAN;

  double S = 0.0;   // TAIL: over the classes outside the list
  const float hi = a.temp.hi, lo = a.temp.lo;
  const auto marks = [&](int c) { return c < row.s.pieces ? s_mark[(c * V) >> 5] >> ((c * V) & 31) : 0u; };
  float held[HOLD ? E : 1][V];
  int at = tid;
  asm volatile("" : "+v"(at));   // the pieces' columns are computed again, not kept from the load
  if constexpr (E > 0) {
    if constexpr (TAIL) {
      constexpr unsigned all = (1u << V) - 1u;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const unsigned b = marks(at + i * NT) & all;
        if (b != 0) row.raw[i] = an_drop<BF16>(row.raw[i], b);
      }
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
      float e[V];
      an_unpack<BF16>(row.raw[i], e);
#pragma unroll
      for (int j = 0; j < V; ++j) e[j] = an_exp2(an_arg(e[j], m, hi, lo));
      S += (double)an_tree<V>(e);
      if constexpr (HOLD) {
#pragma unroll
        for (int j = 0; j < V; ++j) held[i][j] = e[j];
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  } else {
    row.walk_raw([&](const u32x4 p, int c, int) {
      float e[V];
      an_unpack<BF16>(TAIL ? an_drop<BF16>(p, marks(c)) : p, e);
#pragma unroll
      for (int j = 0; j < V; ++j) e[j] = an_exp2(an_arg(e[j], m, hi, lo));
      S += (double)an_tree<V>(e);
    });
  }
  S = an_wave_sum(S);
  if (lane == 0) sh.s_sum[wave] = S;
  __syncthreads();
  if (wave == 0) {
    S = 0.0;
#pragma unroll
    for (int i = 0; i < NW; ++i) S += sh.s_sum[i];
    double loss;
    // (more than 1024 classes and at most 128 answers: never all of them)
    const DistillStat st = an_distill_row(sh.list, a.K, sh.bad != 0, m, S, S, false, TAIL, a.temp.inv_t, loss);
    if (lane == 0) {
      sh.st = st;
      a.row_loss[r] = (float)(a.t2 * loss);
      if (a.stats != nullptr) a.stats[r] = st;
    }
  }
  if (a.grad == nullptr) return;   // uniform
  __syncthreads();
  const DistillStat st = sh.st;
  const bool none = an_no_gradient(st);
  const double inv = none ? 0.0 : 1.0 / st.S;
  const float mass = (float)(st.mass * inv), slope = (float)(st.slope * inv) * a.scale;
  unsigned char* grow = reinterpret_cast<unsigned char*>(a.grad) + r * a.ldg * (BF16 ? 2 : 4);
  asm volatile("" : "+v"(at));
  if constexpr (HOLD) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int c = at + i * NT;
      float g[V];
#pragma unroll
      for (int j = 0; j < V; ++j) g[j] = none ? 0.f : held[i][j] * slope;
      if (c < row.s.pieces) an_store<BF16>(grow, c * V - row.s.shift, a.C, g);
      __builtin_amdgcn_sched_barrier(0);
    }
  } else {
    row.renew();
    row.walk([&](const float (&v)[V], int c, int) {
      const int here = c - tid + at;
      if (here >= row.s.pieces) return;
      float g[V];
#pragma unroll
      for (int j = 0; j < V; ++j) g[j] = none ? 0.f : an_exp2(an_arg(v[j], m, hi, lo)) * slope;
      an_store<BF16>(grow, here * V - row.s.shift, a.C, g);
    });
  }
  __syncthreads();
  const float sc = a.scale;
  an_write_named<BF16>(sh.list.idx, sh.list.q, a.K, sh.repeats != 0, tid, NT, 0, a.C, xr, grow,
                       [&](float x) { return none ? 0.f : sc * (an_exp2(an_arg(x, m, hi, lo)) * mass); },
                       [&](float q) { return none ? 0.f : -sc * q; });
}

template <bool BF16, int E>
__global__ __launch_bounds__(64 * AN_WAVES) void distill_wave_kernel(const DistillArgs a) {
  __shared__ DistillList s_list[AN_WAVES];
  __shared__ unsigned s_mark[AN_WAVES][AN_WAVE_C / 32];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long r = (long)blockIdx.x * AN_WAVES + wave;
  if (r >= a.R) return;   // no barrier below: a wave keeps to its own row
  DistillList& list = s_list[wave];
  unsigned* mark = s_mark[wave];
  const void* xr = an_row<BF16>(a.x, a.ld, r);
  float v[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int c = lane + 64 * i;
    v[i] = c < a.C ? an_at<BF16>(xr, c) : -INFINITY;
  }
  if (lane < AN_WAVE_C / 32) mark[lane] = 0u;
  __builtin_amdgcn_wave_barrier();
  __threadfence_block();
  bool beyond = false, named_again = false;
  for (int k = lane; k < a.K; k += 64) {
    const int64_t j = a.indices[r * a.K + k];
    const bool live = j >= 0 && j < a.C;
    int again = 0;
    beyond |= j >= a.C;
    list.idx[k] = live ? (int)j : -1;
    list.v[k] = a.teacher[r * a.K + k];
    list.x[k] = live ? an_at<BF16>(xr, j) : 0.f;
    if (live) again = (atomicOr(&mark[j >> 5], 1u << (j & 31)) >> (j & 31)) & 1u;
    named_again |= again != 0;
    list.again[k] = again;
  }
  const bool bad = __ballot(beyond) != 0, repeats = __ballot(named_again) != 0;
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < E; ++i) m = fmaxf(m, v[i]);
  m = an_wave_row_max<E>(v, m);
  __builtin_amdgcn_wave_barrier();
  __threadfence_block();
  double S = 0.0;   // tail: over the classes outside the list
  int outside = 0;
  float e32[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int c = lane + 64 * i;
    const double e = an_exp(((double)v[i] - (double)m) * a.temp.inv_t);
    e32[i] = (float)e;
    const bool in = (mark[c >> 5] >> (c & 31)) & 1u;   // E <= 16: c < 1024
    S += a.tail && in ? 0.0 : e;
    outside += c < a.C && !in ? 1 : 0;
  }
  S = an_wave_sum(S);
  const bool all = __ballot(outside != 0) == 0;
  double loss;
  const DistillStat st = an_distill_row(list, a.K, bad, m, S, S, all, a.tail != 0, a.temp.inv_t, loss);
  if (lane == 0) {
    a.row_loss[r] = (float)(a.t2 * loss);
    if (a.stats != nullptr) a.stats[r] = st;
  }
  if (a.grad == nullptr) return;
  const bool none = an_no_gradient(st);
  const double inv = none ? 0.0 : 1.0 / st.S;
  const float mass = (float)(st.mass * inv), slope = (float)(st.slope * inv) * a.scale;
  unsigned char* grow = reinterpret_cast<unsigned char*>(a.grad) + r * a.ldg * (BF16 ? 2 : 4);
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int c = lane + 64 * i;
    if (c < a.C) store1<BF16>(grow, (size_t)c, none ? 0.f : e32[i] * slope);
  }
  __threadfence_block();
  __builtin_amdgcn_wave_barrier();
  const float sc = a.scale;
  an_write_named<BF16>(list.idx, list.q, a.K, repeats, lane, 64, 0, a.C, xr, grow,
                       [&](float x) { return none ? 0.f : sc * ((float)an_exp(((double)x - (double)m) * a.temp.inv_t) * mass); },
                       [&](float t) { return none ? 0.f : -sc * t; });
}

// out[0] = scale * sum of x[0..n): one workgroup, every thread adds its own in order, waves in order
__global__ __launch_bounds__(1024) void answer_sum_kernel(const float* x, long n, double scale, float* out) {
  __shared__ double s_part[16];
  double s = 0.0;
  for (long i = threadIdx.x; i < n; i += 1024) s += (double)x[i];
  s = an_wave_sum(s);
  if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = s_part[0];
    for (int w = 1; w < 16; ++w) s += s_part[w];
    out[0] = (float)(scale * s);
  }
}

// ---------------------------------------------------------------------------------------------
// Which kernel a row length takes
// ---------------------------------------------------------------------------------------------
// calls f(E) with the registers a lane needs for C classes, one wave per row
template <class F>
bool an_by_wave(int C, F f) {
  if (C <= 64) f(std::integral_constant<int, 1>());
  else if (C <= 128) f(std::integral_constant<int, 2>());
  else if (C <= 256) f(std::integral_constant<int, 4>());
  else if (C <= 512) f(std::integral_constant<int, 8>());
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
  return R > 0 && C > 0 && C < 0x7ffffff0 && ld >= 0 && K >= 0 && K <= AN_TOP_MAX && K <= C && temperature >= 9.5367431640625e-07 &&
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
    const dim3 grid((unsigned)((R + AN_WAVES - 1) / AN_WAVES));
    an_by_wave(C, [&](auto e) {
      constexpr int E = decltype(e)::value;
      if (dtype == VQAF_BF16) hipLaunchKernelGGL((answer_grad_wave_kernel<true, E, OP>), grid, dim3(64 * AN_WAVES), 0, st, op, x, ld, (long)R, C, grad, ldg);
      else hipLaunchKernelGGL((answer_grad_wave_kernel<false, E, OP>), grid, dim3(64 * AN_WAVES), 0, st, op, x, ld, (long)R, C, grad, ldg);
    });
  } else {
    const int V = dtype == VQAF_BF16 ? 8 : 4;
    const long segments = ((long)C + V - 1 + (V - 1)) / V / (AN_ST * AN_SP) + 1;
    VQAF_REQUIRE(segments * R < 0x7fffffffL, VQAF_E_SHAPE);
    const dim3 grid((unsigned)(segments * R));
    if (dtype == VQAF_BF16) hipLaunchKernelGGL((answer_grad_block_kernel<true, OP>), grid, dim3(AN_ST), 0, st, op, x, ld, (long)R, C, (int)segments, grad, ldg);
    else hipLaunchKernelGGL((answer_grad_block_kernel<false, OP>), grid, dim3(AN_ST), 0, st, op, x, ld, (long)R, C, (int)segments, grad, ldg);
  }
  VQAF_LAUNCH_CHECK();
}

template <bool BF16>
void an_launch_logprobs(const LogprobArgs& a, hipStream_t st) {
  if (a.C <= AN_WAVE_C) {
    an_by_wave(a.C, [&](auto e) {
      hipLaunchKernelGGL((logprob_wave_kernel<BF16, decltype(e)::value>), dim3((unsigned)((a.R + AN_WAVES - 1) / AN_WAVES)),
                         dim3(64 * AN_WAVES), 0, st, a);
    });
  } else {
    an_by_block<BF16>(a.C, [&](auto nt, auto e) {
      hipLaunchKernelGGL((logprob_block_kernel<BF16, decltype(nt)::value, decltype(e)::value, an_waves(decltype(e)::value)>), dim3((unsigned)a.R),
                         dim3(decltype(nt)::value), 0, st, a);
    });
  }
}

template <bool BF16>
int an_launch_distill(const DistillArgs& a, hipStream_t st) {
  if (a.C <= AN_WAVE_C) {
    an_by_wave(a.C, [&](auto e) {
      hipLaunchKernelGGL((distill_wave_kernel<BF16, decltype(e)::value>), dim3((unsigned)((a.R + AN_WAVES - 1) / AN_WAVES)),
                         dim3(64 * AN_WAVES), 0, st, a);
    });
  } else {
    const size_t mark = ((size_t)a.C + 2 * Piece<BF16>::V + 31) / 32 * 4;
    VQAF_REQUIRE(mark <= 49152, VQAF_E_SHAPE);   // 393 thousand classes
    an_by_block<BF16>(a.C, [&](auto nt, auto e) {
      constexpr int NT = decltype(nt)::value, E = decltype(e)::value;
      constexpr bool HOLD = E > 0 && (!BF16 || E <= 4);
      constexpr int W = an_waves(BF16 && HOLD ? 2 * E + 2 : E + 2);
      if (a.tail) hipLaunchKernelGGL((distill_block_kernel<BF16, NT, E, true, HOLD, W>), dim3((unsigned)a.R), dim3(NT), mark, st, a);
      else hipLaunchKernelGGL((distill_block_kernel<BF16, NT, E, false, HOLD, W>), dim3((unsigned)a.R), dim3(NT), mark, st, a);
    });
  }
  VQAF_LAUNCH_CHECK();
}

}  // namespace

extern "C" int vqaf_token_logprobs(const void* logits, long ld, const int64_t* targets, int R, int C, int T, int K, int dtype,
                                   double temperature, float* logprobs, float* entropy, float* top_logprobs,
                                   int64_t* top_indices, float* stats, vqaf_stream_t stream) {
  VQAF_ENTRY();
  VQAF_REQUIRE(logits != nullptr, VQAF_E_NULL);
  VQAF_REQUIRE(an_shape_ok(ld, R, C, K, temperature) && T >= 0 && T <= AN_TOP_MAX, VQAF_E_SHAPE);
  VQAF_REQUIRE(vqaf_dtype_ok(dtype), VQAF_E_DTYPE);
  VQAF_REQUIRE(T == 0 || (targets != nullptr && logprobs != nullptr), VQAF_E_NULL);
  VQAF_REQUIRE(K == 0 || (top_logprobs != nullptr && top_indices != nullptr), VQAF_E_NULL);
  VQAF_REQUIRE(an_element_aligned(logits, dtype), VQAF_E_ALIGN);
  LogprobArgs a;
  a.x = logits; a.targets = targets; a.logprobs = logprobs; a.entropy = entropy;
  a.top_logprobs = top_logprobs; a.top_indices = top_indices; a.stats = stats;
  a.ld = ld; a.R = R; a.C = C; a.T = T; a.K = K;
  a.temp = an_temp(temperature);
  if (dtype == VQAF_BF16) an_launch_logprobs<true>(a, (hipStream_t)stream);
  else an_launch_logprobs<false>(a, (hipStream_t)stream);
  VQAF_LAUNCH_CHECK();
}

extern "C" int vqaf_token_logprobs_bwd(const void* logits, long ld, const int64_t* targets, const int64_t* top_indices, int R,
                                       int C, int T, int K, int dtype, double temperature, const float* stats,
                                       const float* entropy, const float* g_logprobs, const float* g_entropy,
                                       const float* g_top, void* grad, long ld_grad, vqaf_stream_t stream) {
  VQAF_ENTRY();
  VQAF_REQUIRE(logits != nullptr && stats != nullptr && grad != nullptr, VQAF_E_NULL);
  VQAF_REQUIRE(an_shape_ok(ld, R, C, K, temperature) && T >= 0 && T <= AN_TOP_MAX, VQAF_E_SHAPE);
  VQAF_REQUIRE(vqaf_dtype_ok(dtype), VQAF_E_DTYPE);
  VQAF_REQUIRE(g_logprobs == nullptr || T == 0 || targets != nullptr, VQAF_E_NULL);
  VQAF_REQUIRE(g_top == nullptr || K == 0 || top_indices != nullptr, VQAF_E_NULL);
  VQAF_REQUIRE(g_entropy == nullptr || entropy != nullptr, VQAF_E_NULL);
  VQAF_REQUIRE(an_element_aligned(logits, dtype) && an_grad_layout_ok(logits, ld, grad, ld_grad, C, dtype), VQAF_E_ALIGN);
  LogprobGrad op;
  op.targets = targets; op.top_indices = top_indices; op.stats = stats; op.entropy = entropy;
  op.g_lp = T > 0 ? g_logprobs : nullptr; op.g_ent = g_entropy; op.g_top = K > 0 ? g_top : nullptr;
  op.T = T; op.K = K;
  op.temp = an_temp(temperature);
  return an_launch_grad(op, logits, ld, R, C, dtype, grad, ld_grad, (hipStream_t)stream);
}

extern "C" int vqaf_distill(const void* logits, long ld, const float* teacher, const int64_t* indices, int R, int C, int K,
                            int dtype, double temperature, int tail, float* row_loss, double* stats, void* grad,
                            long ld_grad, double scale, float* loss, vqaf_stream_t stream) {
  VQAF_ENTRY();
  VQAF_REQUIRE(logits && teacher && indices && row_loss, VQAF_E_NULL);
  VQAF_REQUIRE(an_shape_ok(ld, R, C, 0, temperature) && K >= 1 && K <= AN_TOP_MAX, VQAF_E_SHAPE);
  VQAF_REQUIRE(vqaf_dtype_ok(dtype), VQAF_E_DTYPE);
  VQAF_REQUIRE(an_element_aligned(logits, dtype), VQAF_E_ALIGN);
  VQAF_REQUIRE(grad == nullptr || an_grad_layout_ok(logits, ld, grad, ld_grad, C, dtype), VQAF_E_ALIGN);
  DistillArgs a;
  a.x = logits; a.teacher = teacher; a.indices = indices; a.row_loss = row_loss;
  a.stats = reinterpret_cast<DistillStat*>(stats); a.grad = grad;
  a.ld = ld; a.ldg = ld_grad; a.R = R; a.C = C; a.K = K; a.tail = tail != 0;
  a.scale = (float)(temperature * scale);
  a.t2 = temperature * temperature;
  a.temp = an_temp(temperature);
  const int rc = dtype == VQAF_BF16 ? an_launch_distill<true>(a, (hipStream_t)stream)
                                    : an_launch_distill<false>(a, (hipStream_t)stream);
  if (rc != VQAF_OK || loss == nullptr) return rc;
  hipLaunchKernelGGL(answer_sum_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, row_loss, (long)R, scale, loss);
  VQAF_LAUNCH_CHECK();
}

extern "C" int vqaf_distill_bwd(const void* logits, long ld, const float* teacher, const int64_t* indices, int R, int C, int K,
                                int dtype, double temperature, const double* stats, const float* up, int up_step, int skip_unit,
                                double scale, void* grad, long ld_grad, vqaf_stream_t stream) {
  VQAF_ENTRY();
  VQAF_REQUIRE(logits && teacher && indices && stats && up && grad, VQAF_E_NULL);
  VQAF_REQUIRE(an_shape_ok(ld, R, C, 0, temperature) && K >= 1 && K <= AN_TOP_MAX && (up_step == 0 || up_step == 1), VQAF_E_SHAPE);
  VQAF_REQUIRE(vqaf_dtype_ok(dtype), VQAF_E_DTYPE);
  VQAF_REQUIRE(an_element_aligned(logits, dtype) && an_grad_layout_ok(logits, ld, grad, ld_grad, C, dtype), VQAF_E_ALIGN);
  DistillGrad op;
  op.teacher = teacher; op.indices = indices; op.stats = reinterpret_cast<const DistillStat*>(stats); op.up = up;
  op.up_step = up_step; op.K = K; op.scale = (float)(temperature * scale);
  op.skip_unit = skip_unit != 0 && up_step == 0;
  op.temp = an_temp(temperature);
  return an_launch_grad(op, logits, ld, R, C, dtype, grad, ld_grad, (hipStream_t)stream);
}
