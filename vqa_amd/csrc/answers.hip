// What a model answers with: log probabilities of given tokens, the entropy of the answer distribution and its top
// alternatives, forward and backward.  They score the answers for the membership attacks (attack/metric_src.py:302-426
// reads a loss and a maximum per sample; these are the finer scores) and label them for a student (distill.hip).
//
// With z = x / T, m = max z, e_j = exp(z_j - m), S = sum_j e_j, p_j = e_j / S:
//   log p_t = z_t - m - log S            H = log S - sum_j e_j (z_j - m) / S
//   d log p_t / dx_j = (1{j = t} - p_j) / T            dH / dx_j = -p_j (log p_j + H) / T
//
// All of it is bound by the row of logits, read once (and its gradient written once).  A row therefore stays in registers
// from its one read to its last use: rows of up to 1024 classes in one wave (many rows of up to 512 classes: four to a
// wave), longer ones in a workgroup of 256 threads with up to 50 pieces of 16 bytes each -- a row costs the fewest
// registers beside its own that way, so the most rows are in flight on a CU (30522 bf16 classes: five; with 512 threads it
// was three, with 1024 two) -- and past about 66000 classes the row is read again for each use.  Loads are whole 16-byte
// pieces on 16-byte addresses, whatever the row's own alignment (a vocabulary of 50265 puts every second bf16 row on an odd
// address): the row is cut at the pieces' borders and what lies outside it is masked in registers.
//
// Precision: sums of eight in f32, sums of those in f64, the logarithm in f64 (rows of one wave: f32 with the sum's
// rounding put back).  The exponent takes one f32 factor log2(e) / T (1 + delta); its rounding would shift every term the
// same way, so delta times the mean exponent, which the entropy needs anyway, is taken out of log S.  Probabilities and
// gradients are f32, rounded once into their type.

#include "answers.h"

namespace {

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
  long ld, R, r0;   // r0: the launch's first row
  int C, T, K;
  AnTemp temp;
};

// How many of cand[0..n) come before `mine`; sixteen of them a step, as broadcast 16-byte reads in flight together.
// The list is followed by sixteen zeros.
__device__ __forceinline__ int an_rank(const u64* cand, int n, u64 mine) {
  typedef u64 u64x2 __attribute__((ext_vector_type(2)));
  int before = 0;
  for (int j = 0; j < n; j += 16) {
    u64x2 c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = *reinterpret_cast<const u64x2*>(cand + j + 2 * i);
#pragma unroll
    for (int i = 0; i < 8; ++i) before += (c[i].x > mine ? 1 : 0) + (c[i].y > mine ? 1 : 0);
  }
  return before;
}

template <int NT>
struct TopShared {
  float tmax[NT];
  __attribute__((aligned(16))) u64 cand[AN_CAP + 16];   // and room for the ranking's last step
  int n;
  float thr;
  int cnt[1], round[2][NT / 64];
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
  n = dpp_wave_uadd(n);
  if ((threadIdx.x & 63) == 0) atomicAdd(&cnt[0], (int)n);
  __syncthreads();
  return cnt[0];
}

// The K best of a row into sh.cand, by counting: for rows whose candidates overflow the list (a long tie: a masked or
// padded row has nothing else) and rows with NaN.  `from`: a key that at least K elements reach.  The K-th key is that one
// if fewer than K lie above it, else it is found bit by bit; of the elements equal to it the first in the order of the
// index are taken, a round of pieces at a time.
template <bool BF16, int NT>
__device__ __forceinline__ void an_top_by_counting(const Span& span, TopShared<NT>& sh, int K, unsigned from) {
  constexpr int V = Piece<BF16>::V, NW = NT / 64;
  RowPieces<BF16, NT, 0> row;   // reads the row again: the common path's registers stay its own
  row.s = span;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  unsigned t = from;
  int above = an_block_count<NT>(row, sh.cnt, [&](float x, int) { return an_key(x) > t; });
  if (above >= K) {
    t = 0;
    for (int b = 31; b >= 0; --b) {
      const unsigned mid = t | (1u << b);
      if (an_block_count<NT>(row, sh.cnt, [&](float x, int) { return an_key(x) >= mid; }) >= K) t = mid;
    }
    above = an_block_count<NT>(row, sh.cnt, [&](float x, int) { return an_key(x) > t; });
  }
  const int need = K - above;   // of the elements equal to t, >= 1
  __syncthreads();
  if (tid == 0) sh.n = 0;
  __syncthreads();
  int taken = 0, higher = 0;    // of the equal ones and of the others, in the rounds so far
  for (int c0 = 0; c0 < row.s.pieces && (taken < need || higher < above); c0 += NT) {
    const int c = c0 + tid, el = c * V - row.s.shift;
    float v[V];
    int eq = 0, gt = 0;
    if (c < row.s.pieces) {
      an_unpack<BF16>(row.finish(row.fetch(c), c), v);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const bool in = el + j >= 0 && el + j < row.s.C;
        eq += in && an_key(v[j]) == t ? 1 : 0;
        gt += in && an_key(v[j]) > t ? 1 : 0;
      }
    }
    int upto = eq;              // equal elements up to this thread, first in its wave, then in the workgroup
    for (int o = 1; o < 64; o <<= 1) {
      const int left = __shfl_up(upto, o, 64);
      upto += lane >= o ? left : 0;
    }
    const int others = (int)dpp_wave_uadd((unsigned)gt);
    if (lane == 63) sh.round[0][wave] = upto;
    if (lane == 0) sh.round[1][wave] = others;
    __syncthreads();
    int before = taken + upto - eq;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      if (w < wave) before += sh.round[0][w];
      taken += sh.round[0][w];
      higher += sh.round[1][w];
    }
    if (eq + gt > 0) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (el + j < 0 || el + j >= row.s.C) continue;
        const unsigned k = an_key(v[j]);
        // (exactly K in all: `above` above t, `need` equal to it)
        if (k > t || (k == t && before++ < need)) sh.cand[atomicAdd(&sh.n, 1) & (AN_CAP - 1)] = an_pack(k, el + j);
      }
    }
    __syncthreads();
  }
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
  hi = dpp_wave_umax(best);
  lo = dpp_wave_umin(best);                      // 64 maxima reach it if every lane has one
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

// One read of the row into registers, its maximum (bf16: on packed pairs as integers), the sums of e and e t, and the
// alternatives.  Those reach the K-th largest of the threads' maxima, or very nearly only they do: the threads that hold
// such values look through their pieces once more, and the short list that results is ranked by counting.
// Measured, 1920 rows of 30522 bf16 classes: 28 us without alternatives (4.2 TB/s), 36 us with 20 (3.3 TB/s), 41 with 64;
// 1001 x 50265: 27 us without (3.7 TB/s); 511 x 70001, read again: 26 us without (2.8 TB/s), 33 with 20.  Half of the time is vector instructions (14 for each value, 7 of them for e and e t);
// 1920 rows are one and a half rounds of what fits on the chip.
template <bool BF16, int NT, int E, int W>
__global__ __launch_bounds__(NT, W) void logprob_block_kernel(const LogprobArgs a) {
  constexpr int V = Piece<BF16>::V, NW = NT / 64;
  __shared__ TopShared<NT> sh;
  __shared__ float s_max[NW];
  __shared__ double s_sum[2][NW], s_log;
  const long r = a.r0 + blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  RowPieces<BF16, NT, E> row;
  row.s = an_span<BF16>(a.x, a.ld, r, a.R, a.C);
  row.load();

  float m = row.max();
  row.renew();
  if (a.K > 0) {
    sh.tmax[tid] = m;
    if (tid == 0) sh.n = 0;
  }
  m = dpp_wave_max(m);
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
    float e[V], w = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float t = (v[j] - m) * hi;
      e[j] = an_exp2(t);
      w = fmaf(e[j], an_floor(t), w);
    }
    S += (double)an_tree<V>(e);
    Wt += (double)w;
  });
  S = dpp_wave_sum(S);
  Wt = dpp_wave_sum(Wt);
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
  const void* xr = an_row<BF16>(a.x, a.ld, r);
  if (wave == 0) {   // the row's results; the other waves only need log S, and only for the alternatives
    const double mean_t = AN_LN2 * (Wt / S);
    const double log_s = empty ? -INFINITY : log(S) - a.temp.delta * mean_t;
    if (lane == 0) {
      s_log = log_s;
      if (a.entropy != nullptr) a.entropy[r] = empty ? 0.f : (float)(log_s - mean_t * (1.0 - a.temp.delta));
      if (a.stats != nullptr) {
        a.stats[2 * r] = m;
        a.stats[2 * r + 1] = empty ? 1.f : (float)(S * (1.0 - a.temp.delta * mean_t));
      }
    }
    for (int i = lane; i < a.T; i += 64) {
      const int64_t t = a.targets[r * a.T + i];
      float lp = 0.f;                                         // a negative target is none
      if (t >= a.C) lp = NAN;
      else if (t >= 0) lp = an_logprob(an_at<BF16>(xr, t), m, log_s, a.temp.inv_t);
      a.logprobs[r * a.T + i] = lp;
    }
  }
  if (a.K == 0) return;

  // candidates: what reaches the threshold
  row.renew();
  bool counted = broken;
  if (!broken) {
    const float thr = sh.thr;
    if (sh.tmax[tid] >= thr) {
      row.walk_reaching(thr, [&](const float (&v)[V], int el) {
        int hits = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) hits += v[j] >= thr && el + j >= 0 && el + j < a.C ? 1 : 0;
        if (hits == 0) return true;
        int at = atomicAdd(&sh.n, hits);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (v[j] >= thr && el + j >= 0 && el + j < a.C) {
            if (at < AN_CAP) sh.cand[at] = an_pack(an_key(v[j]), el + j);
            ++at;
          }
        }
        return at <= AN_CAP;   // past the list's end there is no use in the rest
      });
    }
    __syncthreads();
    counted = sh.n > AN_CAP;   // uniform
  }
  if (counted) an_top_by_counting<BF16, NT>(row.s, sh, a.K, broken ? 0u : an_key(sh.thr));
  const int n = sh.n;
  if (tid < 16) sh.cand[n + tid] = 0;   // below every candidate
  __syncthreads();
  const double log_s = s_log;
  for (int i = tid; i < n; i += NT) {
    const u64 mine = sh.cand[i];
    const int k = an_rank(sh.cand, n, mine);
    if (k < a.K) {
      const int j = an_index(mine);
      a.top_indices[r * a.K + k] = j;
      a.top_logprobs[r * a.K + k] = an_logprob(an_unkey((unsigned)(mine >> 32)), m, log_s, a.temp.inv_t);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Log probabilities: one wave per row of up to 1024 classes, column lane + 64 i in register i
// ---------------------------------------------------------------------------------------------
constexpr int AN_WCAP = 256;   // candidates a wave lists

// Exactly the K best of a row of keys (0: none), by bisection over the keys and then in the order of the index, into
// cand[0..K).  From `low`, which at least K keys reach.
template <int E>
__device__ __forceinline__ void an_wave_select(const unsigned (&key)[E], unsigned low, int K, u64* cand) {
  const int lane = threadIdx.x & 63;
  unsigned best = key[0];
#pragma unroll
  for (int i = 1; i < E; ++i) best = key[i] > best ? key[i] : best;
  unsigned up = dpp_wave_umax(best);
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

// Measured, 430 f32 classes: 1024 rows with a target 3.4 us, with three alternatives 4.6, with 20 5.7 us; 25000 rows with a
// target and 20 alternatives 25 us, with 64 54 us: a row is some 300 instructions of one wave, most of them for the
// alternatives.
template <bool BF16, int E>
__global__ __launch_bounds__(64 * AN_WAVES, E <= 8 ? 8 : 5) void logprob_wave_kernel(const LogprobArgs a) {
  __shared__ __attribute__((aligned(16))) u64 s_cand[AN_WAVES][AN_WCAP + 16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long r = a.r0 + (long)blockIdx.x * AN_WAVES + wave;
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
  float xt = t >= 0 && t < a.C ? an_at<BF16>(xr, t) : 0.f;   // on its way under the exponentials
  double S = 0.0;
  float Wt = 0.f;
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
    Wt += ws;
  }
  S = dpp_wave_sum(S);
  const float w = dpp_wave_sum(Wt), s32 = (float)S;
  // log S: the f32 logarithm of the rounded sum and the rounding's share
  const float mean_t = (float)AN_LN2 * (w / s32);
  const double log_s = empty ? -INFINITY : (double)logf(s32) + (S - (double)s32) / s32 - a.temp.delta * mean_t;
  if (lane == 0) {
    if (a.entropy != nullptr) a.entropy[r] = empty ? 0.f : (float)(log_s - (double)mean_t);
    if (a.stats != nullptr) {
      a.stats[2 * r] = m;
      a.stats[2 * r + 1] = empty ? 1.f : s32 * (1.f - (float)a.temp.delta * mean_t);
    }
  }
  for (int i = lane; i < a.T; i += 64) {
    if (i >= 64) {
      t = a.targets[r * a.T + i];
      xt = t >= 0 && t < a.C ? an_at<BF16>(xr, t) : 0.f;
    }
    a.logprobs[r * a.T + i] = t < 0 ? 0.f : t >= a.C ? NAN : an_logprob(xt, m, log_s, a.temp.inv_t);   // (negative: none)
  }
  if (a.K == 0) return;

  // What the K-th largest of the lanes' maxima reaches is a list that holds the K best, short while K is; where it is too
  // long the bisection goes on over all elements.  Long ties and NaN go by the keys alone.
  u64* cand = s_cand[wave];
  const bool broken = !empty && !(S == S);
  int n = AN_WCAP + 1;
  if (!broken) {
    const unsigned mine = lane < a.C ? an_key(best) : 0u;   // (lanes past a short row have none)
    const unsigned most = dpp_wave_umax(mine);
    unsigned up = most, low = AN_KEY_MINF;
    if (a.K <= 8) {   // so few are found faster one by one: a reduction each, against some fifteen steps
      unsigned left = mine;
      low = most;
      for (int k = 1; k < a.K; ++k) {
        const u64 who = __ballot(left == low);
        left = lane == __ffsll((long long)who) - 1 ? 0u : left;
        low = dpp_wave_umax(left);
      }
      if (low < AN_KEY_MINF) low = AN_KEY_MINF;   // fewer lanes than answers: a short row, all of it
    } else if (a.K <= 64) {
      low = dpp_wave_umin(mine);
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
    }
    // what reaches thr into the list, as far as it goes; how many do
    const auto collect = [&](float thr) {
      const u64 below_lane = (1ull << lane) - 1ull;
      int c = 0;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const bool take = v[i] >= thr && lane + 64 * i < a.C;
        const u64 who = __ballot(take);
        if (who != 0) {
          const int at = c + __popcll(who & below_lane);
          if (take && at < AN_WCAP) cand[at] = an_pack(an_key(v[i]), lane + 64 * i);
          c += __popcll(who);
        }
      }
      return c;
    };
    n = collect(an_unkey(low));
    const int enough = a.K + (a.K >> 2) + 32;
    if (n > enough && low < most) {   // (ranking the list costs its length squared)
      up = most;
      while (n > enough && low < up) {
        const unsigned mid = low + ((up - low) >> 1) + 1;
        const float thr = an_unkey(mid);
        int c = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) c += __popcll(__ballot(v[i] >= thr && lane + 64 * i < a.C));
        if (c >= a.K) {
          low = mid;
          n = c;
        } else {
          up = mid - 1;
        }
      }
      n = collect(an_unkey(low));
    }
  }
  if (n > AN_WCAP) {
    unsigned key[E];
#pragma unroll
    for (int i = 0; i < E; ++i) key[i] = lane + 64 * i < a.C ? an_key(v[i]) : 0u;
    an_wave_select<E>(key, AN_KEY_MINF, a.K, cand);
    n = a.K;
  }
  if (lane < 16) cand[n + lane] = 0;
  __builtin_amdgcn_wave_barrier();
  __threadfence_block();
  for (int i = lane; i < n; i += 64) {
    const u64 mine = cand[i];
    const int before = an_rank(cand, n, mine);
    if (before < a.K) {
      a.top_indices[r * a.K + before] = an_index(mine);
      a.top_logprobs[r * a.K + before] = an_logprob(an_unkey((unsigned)(mine >> 32)), m, log_s, a.temp.inv_t);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Log probabilities: four rows of up to 512 classes per wave, a row to sixteen lanes
// ---------------------------------------------------------------------------------------------
// Taken from 8192 rows on, for up to eight alternatives.  With many rows the instructions of the reductions and of the
// alternatives count, and here four rows share them; with few the latency does, and a whole wave to a row has less of it.
// Measured (the shortest of many launches, both sides in one run), 430 f32 classes with a target and 0 / 3 / 8 alternatives: 25000 rows 11.2 / 15.4 / 18.2 us (3.8 TB/s without
// alternatives) against 13.1 / 19.6 / 23.0 with a wave to a row, 8192 rows 5.9 / 8.0 / 9.4 against 6.8 / 9.4 / 10.8, 4096
// rows 4.4 / 6.3 / 7.6 against 4.7 / 6.4 / 7.1, 1024 rows 3.4 / 5.3 / 6.4 against 2.8 / 4.1 / 4.4; 25000 rows of 430 bf16
// classes 10.3 / 14.8 / 17.4 against 15.6 / 21.4 / 24.5.  Loads are 16-byte pieces as in the longer rows: single elements
// of sixteen lanes cost the bf16 rows 19.5 us.
constexpr int AN_GROUP_FROM = 8192;
constexpr int AN_GROUP_C = 512, AN_GROUP_K = 8, AN_GROUP_ROWS = 16;   // classes, alternatives, rows per workgroup
constexpr int AN_GCAP = 48;                                           // candidates a row lists

// the sixteen bits of a ballot that belong to the lane's row
__device__ __forceinline__ unsigned an_group_bits(u64 who, int lane) {
  const unsigned half = lane & 32 ? (unsigned)(who >> 32) : (unsigned)who;
  return (half >> (lane & 16)) & 0xffffu;
}

template <bool BF16, int E>
__global__ __launch_bounds__(64 * AN_WAVES, E * (BF16 ? 2 : 1) <= 8 ? 8 : 7) void logprob_group_kernel(const LogprobArgs a) {
  constexpr int V = Piece<BF16>::V;
  __shared__ __attribute__((aligned(16))) u64 s_cand[AN_GROUP_ROWS][AN_GCAP + 16];
  const int lane = threadIdx.x & 63, l = lane & 15, group = threadIdx.x >> 4;
  const long rl = a.r0 + (long)blockIdx.x * AN_GROUP_ROWS + group;
  const bool live = rl < a.R;
  const long r = live ? rl : a.R - 1;   // (lanes without a row go along with the last one and write nothing)
  const void* xr = an_row<BF16>(a.x, a.ld, r);
  RowPieces<BF16, 16, E> row;
  row.s = an_span<BF16>(a.x, a.ld, r, a.R, a.C);
  row.load();
  int64_t t = -1;
  if (l < a.T) t = a.targets[r * a.T + l];   // the first 16; more are read below
  const float best = row.max();
  float m = dpp_row_max(best);
  if (__ballot(m == -INFINITY) != 0) {   // (the maximum may leave NaN out)
    bool nan = false;
    row.walk([&](const float (&v)[V], int, int) {
#pragma unroll
      for (int j = 0; j < V; ++j) nan |= v[j] != v[j];
    });
    if (an_group_bits(__ballot(nan), lane) != 0 && m == -INFINITY) m = NAN;
  }
  const bool empty = m == -INFINITY;
  float xt = t >= 0 && t < a.C ? an_at<BF16>(xr, t) : 0.f;   // on its way under the exponentials
  double S = 0.0;
  float Wt = 0.f;
  const float hi = a.temp.hi;
  row.renew();
  row.walk([&](const float (&v)[V], int, int) {
    float e[V], w = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float u = (v[j] - m) * hi;
      e[j] = an_exp2(u);
      w = fmaf(e[j], an_floor(u), w);
    }
    S += (double)an_tree<V>(e);
    Wt += w;
  });
  S = dpp_row_sum(S);
  const float w = dpp_row_sum(Wt), s32 = (float)S;
  // log S: the f32 logarithm of the rounded sum and the rounding's share
  const float mean_t = (float)AN_LN2 * (w / s32);
  const double log_s = empty ? -INFINITY
                             : (double)logf(s32) + (double)((float)(S - (double)s32) * __builtin_amdgcn_rcpf(s32)) - a.temp.delta * mean_t;
  if (l == 0 && live) {
    if (a.entropy != nullptr) a.entropy[r] = empty ? 0.f : (float)(log_s - (double)mean_t);
    if (a.stats != nullptr) {
      a.stats[2 * r] = m;
      a.stats[2 * r + 1] = empty ? 1.f : s32 * (1.f - (float)a.temp.delta * mean_t);
    }
  }
  for (int i = l; i < a.T; i += 16) {
    if (i >= 16) {
      t = a.targets[r * a.T + i];
      xt = t >= 0 && t < a.C ? an_at<BF16>(xr, t) : 0.f;
    }
    // (negative: none)
    if (live) a.logprobs[r * a.T + i] = t < 0 ? 0.f : t >= a.C ? NAN : an_logprob(xt, m, log_s, a.temp.inv_t);
  }
  if (a.K == 0) return;

  // what the K-th largest of the lanes' maxima reaches
  u64* cand = s_cand[group];
  unsigned left = l < row.s.pieces ? an_key(best) : 0u, low = dpp_row_umax(left);
  for (int k = 1; k < a.K; ++k) {
    const unsigned who = an_group_bits(__ballot(left == low), lane);
    left = l == __ffs((int)who) - 1 ? 0u : left;
    low = dpp_row_umax(left);
  }
  if (low < AN_KEY_MINF) low = AN_KEY_MINF;   // fewer lanes than answers: a short row, all of it
  const float thr = an_unkey(low);
  // which of the lane's values those are, their places in the list, and the values read again (there are few)
  unsigned hit[(E * V + 31) / 32] = {};
  row.renew();
  {
    int b = 0;
    row.walk([&](const float (&v)[V], int, int el) {
#pragma unroll
      for (int j = 0; j < V; ++j, ++b) hit[b / 32] |= v[j] >= thr && (thr > -INFINITY || (el + j >= 0 && el + j < a.C)) ? 1u << (b % 32) : 0u;
    });
  }
  int mine = 0;
#pragma unroll
  for (int i = 0; i < (E * V + 31) / 32; ++i) mine += __popc(hit[i]);
  int at = mine;
  at += (int)dpp_move<0x111, 0xf>(0u, (unsigned)at);   // sums over the lanes so far (row_shr)
  at += (int)dpp_move<0x112, 0xf>(0u, (unsigned)at);
  at += (int)dpp_move<0x114, 0xf>(0u, (unsigned)at);
  at += (int)dpp_move<0x118, 0xf>(0u, (unsigned)at);
  int n = __shfl(at, lane | 15, 64);
  at -= mine;
#pragma unroll
  for (int i = 0; i < (E * V + 31) / 32; ++i) {
    unsigned h = hit[i];
    while (h != 0 && at < AN_GCAP) {
      const int b = i * 32 + __ffs((int)h) - 1;
      h &= h - 1;
      const int col = (l + 16 * (b / V)) * V + b % V - row.s.shift;
      cand[at++] = an_pack(an_key(an_at<BF16>(xr, col)), col);
    }
  }
  // long ties and NaN: the whole wave takes the row by its keys, one such row after the other
  const bool broken = !empty && !(S == S);
  u64 over = __ballot(n > AN_GCAP || broken);
  while (over != 0) {
    constexpr int EW = (E * V + 3) / 4;
    const int of = (__ffsll((long long)over) - 1) & 48;   // first lane of that row
    const int in = (int)((threadIdx.x & ~63u) + of) / 16;
    const long which = a.r0 + (long)blockIdx.x * AN_GROUP_ROWS + in;
    const void* p = an_row<BF16>(a.x, a.ld, which < a.R ? which : a.R - 1);
    unsigned key[EW];
#pragma unroll
    for (int i = 0; i < EW; ++i) key[i] = lane + 64 * i < a.C ? an_key(an_at<BF16>(p, lane + 64 * i)) : 0u;
    an_wave_select<EW>(key, AN_KEY_MINF, a.K, s_cand[in]);
    if ((lane & 48) == of) n = a.K;
    over &= ~(0xffffull << of);
  }
  cand[n + l] = 0;
  __builtin_amdgcn_wave_barrier();
  __threadfence_block();
  for (int i = l; i < n; i += 16) {
    const u64 c = cand[i];
    int before = 0;
    for (int j = 0; j < n; j += 4)
#pragma unroll
      for (int o = 0; o < 4; ++o) before += cand[j + o] > c ? 1 : 0;
    if (before < a.K && live) {
      a.top_indices[r * a.K + before] = an_index(c);
      a.top_logprobs[r * a.K + before] = an_logprob(an_unkey((unsigned)(c >> 32)), m, log_s, a.temp.inv_t);
    }
  }
}

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
    w.A = (float)dpp_wave_sum(sum);
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

template <bool BF16>
void an_launch_logprobs(LogprobArgs a, hipStream_t st) {
  if (a.C <= AN_GROUP_C && a.K <= AN_GROUP_K && a.R >= AN_GROUP_FROM) {
    const auto go = [&](auto e) {
      an_by_launch(a.R, 16, [&](long r0, long n) {
        a.r0 = r0;
        hipLaunchKernelGGL((logprob_group_kernel<BF16, decltype(e)::value>), dim3((unsigned)((n + AN_GROUP_ROWS - 1) / AN_GROUP_ROWS)),
                           dim3(64 * AN_WAVES), 0, st, a);
      });
    };
    const int e = ((a.C + Piece<BF16>::V - 1) / Piece<BF16>::V + 1 + 15) / 16;   // (a piece more than an aligned row fills)
    if (e <= 1) go(std::integral_constant<int, 1>());
    else if (e <= 2) go(std::integral_constant<int, 2>());
    else if (e <= 3) go(std::integral_constant<int, 3>());
    else if (e <= 4) go(std::integral_constant<int, 4>());
    else if (BF16 || e <= 5) go(std::integral_constant<int, 5>());
    else if constexpr (!BF16) {
      if (e <= 6) go(std::integral_constant<int, 6>());
      else if (e <= 7) go(std::integral_constant<int, 7>());
      else go(std::integral_constant<int, 9>());
    }
  } else if (a.C <= AN_WAVE_C) {
    an_by_wave(a.C, [&](auto e) {
      an_by_launch(a.R, 64, [&](long r0, long n) {
        a.r0 = r0;
        hipLaunchKernelGGL((logprob_wave_kernel<BF16, decltype(e)::value>), dim3((unsigned)((n + AN_WAVES - 1) / AN_WAVES)),
                           dim3(64 * AN_WAVES), 0, st, a);
      });
    });
  } else {
    an_by_block<BF16>(a.C, [&](auto nt, auto e) {
      constexpr int NT = decltype(nt)::value, E = decltype(e)::value;
      an_by_launch(a.R, NT, [&](long r0, long n) {
        a.r0 = r0;
        hipLaunchKernelGGL((logprob_block_kernel<BF16, NT, E, an_waves(E)>), dim3((unsigned)n), dim3(NT), 0, st, a);
      });
    });
  }
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
  a.ld = ld; a.R = R; a.r0 = 0; a.C = C; a.T = T; a.K = K;
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
