// The distillation loss against a teacher's top answers, with its gradient: a student trained on what a model answers
// with in place of hard labels (utils/src.py:96).  For the answers i_k with the teacher's probabilities q_k and the rest
// r that no answer of the list holds, z = x / T, e_j = exp(z_j - max z), S = sum_j e_j, p_j = e_j / S:
//   L = T^2 [ sum_k q_k (log q_k - log p_{i_k}) + r (log r - log P) ],     P = sum of p_j outside the list
//   dL / dx_j = T [ p_j (sum q + r) - sum_{k: i_k = j} q_k ] on the list,  T p_j [ sum q + r - r / P ] elsewhere.
// P may lie below every number where the student leaves next to nothing outside the list (a mask of -500, a small
// temperature), and r / P above, so neither is formed: with e'_j = exp(z_j - m'), m' the largest z outside the list and S'
// the sum of e' there,
//   log P = m' - max z + log S' - log S,     dL / dx_j = T e'_j [ (sum q + r) exp(m' - max z) / S - r / S' ]  elsewhere,
// where S and S' are at least 1 and the bracket lies between -1 and 1.
// Rows are held and walked as in answers.hip; the gradient for an incoming gradient of 1 leaves from the same read.
//
// Precision.  The divergence of two close distributions is a small difference of large terms, so the list's terms, the
// logarithms and the loss are f64, and the sums over the row as in answers.hip (the factor's error taken out through
// sum e t).  Rows of one wave, whose few terms do not average their rounding out, take the exponential itself in f64 (a
// Taylor polynomial after range reduction; the f64 vector rate of this chip is the f32 one).

#include "answers.h"

namespace {

// ---------------------------------------------------------------------------------------------
// Distillation loss, with the gradient of the sum (or mean) in the same pass
// ---------------------------------------------------------------------------------------------
// 40 bytes a row: the row's largest logit, the one that `slope` goes with (tail: the largest outside the list; 0 where that
// is -inf), S, mass = sum q + r, slope: the bracket above (no tail: mass / S), log Q (q_k = exp(v_k - log Q))
struct DistillStat {
  float m, m_out;
  double S, mass, slope, log_q;
};
static_assert(sizeof(DistillStat) == 40, "five f64 a row");

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
    float m, m_out, mass, slope, hi, lo, g;
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
    w.m = s.m;
    w.m_out = s.m_out;
    w.empty = an_no_gradient(s);
    w.mass = (float)(s.mass / s.S);
    w.slope = (float)s.slope;
    w.hi = temp.hi;
    w.lo = temp.lo;
    w.g = scale * up[r * up_step];
    return w;
  }
  static __device__ __forceinline__ float dense(const Row& w, float x) {
    return w.empty ? 0.f : w.g * (an_exp2(an_arg(x, w.m_out, w.hi, w.lo)) * w.slope);
  }
  static __device__ __forceinline__ float base(const Row& w, float x) {
    return w.empty ? 0.f : w.g * (an_exp2(an_arg(x, w.m, w.hi, w.lo)) * w.mass);
  }
  static __device__ __forceinline__ float term(const Row& w, float q) { return w.empty ? 0.f : -w.g * q; }
};

struct DistillArgs {
  const void* x;
  const float* teacher;
  const int64_t* indices;
  float* row_loss;
  DistillStat* stats;   // or NULL
  void* grad;           // or NULL
  long ld, ldg, R, r0;  // r0: the launch's first row
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

// One wave: the row's statistics and loss.  m_dense, s: the largest logit of the classes outside the list (tail) or of all
// of them, and the sum of exp((x - m_dense) / T) over those, relative to 0 where m_dense is -inf.  `all`: the list covers
// every class; `bad`: an answer lies past the classes.  Short loops on purpose: the pieces of the row are alive around this.
__device__ __forceinline__ DistillStat an_distill_row(DistillList& list, int K, bool bad, float m_dense, double s, bool all,
                                                      bool tail, double inv_t, double& loss) {
  const int lane = threadIdx.x & 63;
  DistillStat st;
  st.m = m_dense;
  st.m_out = m_dense;
  st.S = s;
  st.log_q = 0.0;
  double part = 1.0;   // exp((m_dense - m) / T)
  bool some = true;
  if (tail) {
    float top = -INFINITY;
    bool nan = false;
#pragma unroll 1
    for (int k = lane; k < K; k += 64) {
      if (list.idx[k] < 0) continue;
      top = fmaxf(top, list.x[k]);
      nan |= list.x[k] != list.x[k];
    }
    st.m = fmaxf(m_dense, dpp_wave_max(top));
    // (maxima leave NaN out: a row of nothing else but -inf is not empty)
    if (st.m == -INFINITY && (s != s || __ballot(nan) != 0)) st.m = NAN;
    if (m_dense == -INFINITY) st.m_out = 0.f;
    else part = an_exp(((double)m_dense - (double)st.m) * inv_t);
    double own = 0.0;
#pragma unroll 1
    for (int k = lane; k < K; k += 64)
      if (list.idx[k] >= 0 && !list.again[k]) own += an_exp(((double)list.x[k] - (double)st.m) * inv_t);
    st.S = s * part + dpp_wave_sum(own);
  } else {
    float vm = -INFINITY;
    bool nan = false;
#pragma unroll 1
    for (int k = lane; k < K; k += 64) {
      if (list.idx[k] < 0) continue;
      vm = fmaxf(vm, list.v[k]);
      nan |= list.v[k] != list.v[k];
    }
    vm = dpp_wave_max(vm);
    // (a NaN among the values is left out of the maximum and comes back through the sum)
    some = vm != -INFINITY || __ballot(nan) != 0;
    if (some) {
      double sum = 0.0;
#pragma unroll 1
      for (int k = lane; k < K; k += 64) sum += list.idx[k] >= 0 ? an_exp((double)list.v[k] - (double)vm) : 0.0;
      st.log_q = (double)vm + log(dpp_wave_sum(sum));
    }
  }
  const bool empty = st.m == -INFINITY;
  const double log_s = log(st.S);
  double mass = 0.0, l = 0.0;
  bool any = false;
#pragma unroll 1
  for (int k = lane; k < K; k += 64) {
    const bool live = list.idx[k] >= 0;
    const double lq = (double)list.v[k] - st.log_q;
    const double q = live && some ? an_exp(lq) : 0.0;
    const double lp = empty ? -INFINITY : ((double)list.x[k] - (double)st.m) * inv_t - log_s;
    any |= live;
    mass += q;
    if (q != 0.0) l += q * (lq - lp);   // (NaN goes in)
    list.q[k] = (float)q;
  }
  mass = dpp_wave_sum(mass);
  l = dpp_wave_sum(l);
  double cut = 0.0;   // r / S'
  if (tail) {
    double rest = all || __ballot(any) == 0 ? 0.0 : 1.0 - mass;   // (a row without answers teaches nothing)
    if (!(rest > (double)AN_NO_REST)) rest = 0.0;
    mass += rest;
    if (rest > 0.0) {
      if (empty || s == 0.0) {   // nothing outside: met with probability 0, and no logit there to change
        l += INFINITY;
      } else {
        l += rest * (log(rest) - (((double)st.m_out - (double)st.m) * inv_t + log(s) - log_s));
        cut = rest / s;
      }
    }
  } else if (some) {
    mass = mass / mass;   // 1, or NaN
  }
  if (bad) l = mass = NAN;
  st.mass = mass;
  st.slope = mass == 0.0 ? 0.0 : mass * part / st.S - cut;
  loss = l;
  return st;
}

template <int NT>
struct DistillShared {
  DistillList list;
  float s_max[NT / 64];
  double s_sum[2][NT / 64];
  int bad, repeats, none;
  float m, mass, slope;   // the row's maximum; over S; times the gradient's scale
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
// taken out of the registers before the maximum, so that the rest is summed by itself and relative to its own largest logit
// (1 - sum p would lose what is left of it where the student agrees with its teacher, exponentials relative to the row's
// maximum where it lies far above), and their own terms are added by the list.
// HOLD: the exponentials stay in registers for the gradient (f32: in the place of the logits; bf16: in twice the
// registers, only for short rows); otherwise they are formed again.
// Measured, 1920 rows of 30522 bf16 classes, 64 answers, with the rest as an event and the gradient: 65 us (3.6 TB/s read
// and written; 45 us without the gradient); 511 x 50265 f32, 100 answers, without a gradient: 37 us with the statistics for
// one, 31 without (2.8 and 3.3 TB/s: two workgroups to a CU hold all the rows at once, so that loads, sums and reductions
// of a row follow one another); 511 x 70001 bf16, read again, with the gradient: 49 us.  25 vector instructions a value take
// two thirds of the first.
template <bool BF16, int NT, int E, bool TAIL, bool HOLD, int W>
__global__ __launch_bounds__(NT, W) void distill_block_kernel(const DistillArgs a) {
  constexpr int V = Piece<BF16>::V, NW = NT / 64;
  __shared__ DistillShared<NT> sh;
  extern __shared__ unsigned s_mark[];   // one bit per element of the pieces
  const long r = a.r0 + blockIdx.x;
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
  const auto marks = [&](int c) { return c < row.s.pieces ? s_mark[(c * V) >> 5] >> ((c * V) & 31) : 0u; };
  const auto outside = [&](const u32x4 p, int c) { return TAIL ? an_drop<BF16>(p, marks(c)) : p; };
  int at = tid;
  asm volatile("" : "+v"(at));   // the pieces' columns are computed again, not kept from the load
  if constexpr (TAIL) {
    __syncthreads();
    if constexpr (E > 0) {
      constexpr unsigned all = (1u << V) - 1u;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const unsigned b = marks(at + i * NT) & all;
        if (b != 0) row.raw[i] = an_drop<BF16>(row.raw[i], b);
      }
    }
  }
  float m;   // TAIL: of the classes outside the list
  if constexpr (E > 0) m = row.max();
  else m = row.max_of(outside);
  m = dpp_wave_max(m);
  row.renew();
  if (lane == 0) sh.s_max[wave] = m;
  __syncthreads();
  m = sh.s_max[0];
#pragma unroll
  for (int i = 1; i < NW; ++i) m = fmaxf(m, sh.s_max[i]);
  if (!TAIL && m == -INFINITY && an_block_nan<BF16, NT>(row.s)) m = NAN;
  const float from = TAIL && m == -INFINITY ? 0.f : m;   // (NaN comes back through the sum)

  // Sums of e = 2^t and of e t.  One factor only: what its rounding shifts is taken out of the sum below, to first order.
  double S = 0.0, Wt = 0.0;
  const float hi = a.temp.hi;
  const auto add = [&](float (&e)[V]) {
    float w = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float t = (e[j] - from) * hi;
      e[j] = an_exp2(t);
      w = fmaf(e[j], an_floor(t), w);
    }
    S += (double)an_tree<V>(e);
    Wt += (double)w;
  };
  float held[HOLD ? E : 1][V];
  if constexpr (E > 0) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      float e[V];
      an_unpack<BF16>(row.raw[i], e);
      add(e);
      if constexpr (HOLD) {
#pragma unroll
        for (int j = 0; j < V; ++j) held[i][j] = e[j];
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  } else {
    row.walk_raw([&](const u32x4 p, int c, int) {
      float e[V];
      an_unpack<BF16>(outside(p, c), e);
      add(e);
    });
  }
  S = dpp_wave_sum(S);
  Wt = dpp_wave_sum(Wt);
  if (lane == 0) {
    sh.s_sum[0][wave] = S;
    sh.s_sum[1][wave] = Wt;
  }
  __syncthreads();
  if (wave == 0) {
    S = Wt = 0.0;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      S += sh.s_sum[0][i];
      Wt += sh.s_sum[1][i];
    }
    S -= a.temp.delta * AN_LN2 * Wt;
    double loss;
    // (more than 1024 classes and at most 128 answers: never all of them)
    const DistillStat st = an_distill_row(sh.list, a.K, sh.bad != 0, m, S, false, TAIL, a.temp.inv_t, loss);
    if (lane == 0) {
      a.row_loss[r] = (float)(a.t2 * loss);
      if (a.stats != nullptr) a.stats[r] = st;
      sh.none = an_no_gradient(st) ? 1 : 0;
      sh.m = st.m;
      sh.mass = (float)(st.mass / st.S);
      sh.slope = (float)st.slope * a.scale;
    }
  }
  if (a.grad == nullptr) return;   // uniform
  __syncthreads();
  const bool none = sh.none != 0;
  const float mass = sh.mass, slope = sh.slope;
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
      for (int j = 0; j < V; ++j) g[j] = none ? 0.f : an_exp2((v[j] - from) * hi) * slope;
      an_store<BF16>(grow, here * V - row.s.shift, a.C, g);
    });
  }
  __syncthreads();
  const float sc = a.scale, top = sh.m;
  an_write_named<BF16>(sh.list.idx, sh.list.q, a.K, sh.repeats != 0, tid, NT, 0, a.C, xr, grow,
                       [&](float x) { return none ? 0.f : sc * (an_exp2((x - top) * hi) * mass); },
                       [&](float q) { return none ? 0.f : -sc * q; });
}

// One wave per row of up to 1024 classes.  Measured with the gradient, 64 x 430 bf16 8 us and 1024 x 430 f32 9 us, a chain of
// reductions and f64 logarithms; 25000 x 430 bf16 46 us, with the rest as an event 50 us: f64 arithmetic, 0.9 TB/s.
template <bool BF16, int E>
__global__ __launch_bounds__(64 * AN_WAVES) void distill_wave_kernel(const DistillArgs a) {
  __shared__ DistillList s_list[AN_WAVES];
  __shared__ unsigned s_mark[AN_WAVES][AN_WAVE_C / 32];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long r = a.r0 + (long)blockIdx.x * AN_WAVES + wave;
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
  __builtin_amdgcn_wave_barrier();
  __threadfence_block();
  int outside = 0;
  float m = -INFINITY;   // tail: of the classes outside the list
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int c = lane + 64 * i;
    const bool in = (mark[c >> 5] >> (c & 31)) & 1u;   // E <= 16: c < 1024
    outside += c < a.C && !in ? 1 : 0;
    if (a.tail && in) v[i] = -INFINITY;   // (their gradients are written by name)
    m = fmaxf(m, v[i]);
  }
  m = a.tail ? dpp_wave_max(m) : an_wave_row_max<E>(v, m);
  const double from = a.tail && m == -INFINITY ? 0.0 : (double)m;
  double S = 0.0;
  float e32[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const double e = an_exp(((double)v[i] - from) * a.temp.inv_t);
    e32[i] = (float)e;
    S += e;
  }
  S = dpp_wave_sum(S);
  const bool all = __ballot(outside != 0) == 0;
  double loss;
  const DistillStat st = an_distill_row(list, a.K, bad, m, S, all, a.tail != 0, a.temp.inv_t, loss);
  if (lane == 0) {
    a.row_loss[r] = (float)(a.t2 * loss);
    if (a.stats != nullptr) a.stats[r] = st;
  }
  if (a.grad == nullptr) return;
  const bool none = an_no_gradient(st);
  const float mass = (float)(st.mass / st.S), slope = (float)st.slope * a.scale;
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
                       [&](float x) { return none ? 0.f : sc * ((float)an_exp(((double)x - (double)st.m) * a.temp.inv_t) * mass); },
                       [&](float t) { return none ? 0.f : -sc * t; });
}

// out[0] = scale * sum of x[0..n): one workgroup, every thread adds its own in order, waves in order
__global__ __launch_bounds__(1024) void answer_sum_kernel(const float* x, long n, double scale, float* out) {
  __shared__ double s_part[16];
  double s = 0.0;
  for (long i = threadIdx.x; i < n; i += 1024) s += (double)x[i];
  s = dpp_wave_sum(s);
  if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = s_part[0];
    for (int w = 1; w < 16; ++w) s += s_part[w];
    out[0] = (float)(scale * s);
  }
}

template <bool BF16>
int an_launch_distill(DistillArgs a, hipStream_t st) {
  if (a.C <= AN_WAVE_C) {
    an_by_wave(a.C, [&](auto e) {
      an_by_launch(a.R, 64, [&](long r0, long n) {
        a.r0 = r0;
        hipLaunchKernelGGL((distill_wave_kernel<BF16, decltype(e)::value>), dim3((unsigned)((n + AN_WAVES - 1) / AN_WAVES)),
                           dim3(64 * AN_WAVES), 0, st, a);
      });
    });
  } else {
    const size_t mark = ((size_t)a.C + 2 * Piece<BF16>::V + 31) / 32 * 4;
    VQAF_REQUIRE(mark <= 49152, VQAF_E_SHAPE);   // 393 thousand classes
    an_by_block<BF16>(a.C, [&](auto nt, auto e) {
      constexpr int NT = decltype(nt)::value, E = decltype(e)::value;
      constexpr bool HOLD = E > 0 && (!BF16 || E <= 4);
      constexpr int W = an_waves(BF16 && HOLD ? 2 * E + 2 : E + 2);
      an_by_launch(a.R, NT, [&](long r0, long n) {
        a.r0 = r0;
        if (a.tail) hipLaunchKernelGGL((distill_block_kernel<BF16, NT, E, true, HOLD, W>), dim3((unsigned)n), dim3(NT), mark, st, a);
        else hipLaunchKernelGGL((distill_block_kernel<BF16, NT, E, false, HOLD, W>), dim3((unsigned)n), dim3(NT), mark, st, a);
      });
    });
  }
  VQAF_LAUNCH_CHECK();
}

}  // namespace

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
  a.ld = ld; a.ldg = ld_grad; a.R = R; a.r0 = 0; a.C = C; a.K = K; a.tail = tail != 0;
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
