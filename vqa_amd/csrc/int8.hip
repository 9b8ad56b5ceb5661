// Linear layers in eight-bit integers with a scale for each token and each output channel: the scoring and labelling
// passes of the encoders (model/vision_encoder.py:83-127, model/text_encoder.py:14-48 run these layers in f32).
//
//   s_m = max(max_k |x_mk| / 127, 2^-126),   q_mk = round-half-even(x_mk / s_m),   y_mn = (sum_k q_mk w_nk) s_m s_n + b_n
//
// The sum is exact in 32-bit integers (127^2 K < 2^31 for K up to 131072); the two scales, the bias and the rounding to
// the output type follow in f32, in the epilogue.  The quotient is rounded as if it were exact: next to a border the
// sign of x - (q +- 1/2) s, one fused multiply-add, decides.  A row with NaN or an infinity gets the scale NaN, which
// makes its outputs NaN.
//
// Three kernels.  Many tokens: one pass writes the rows as integers (bound by its bytes), and a matrix product on
// 32x32x32 integer MFMAs with the tile shape and LDS-DMA images of the bf16 Linear kernel: the 128-byte rows of a k-step
// hold 128 values instead of 64.  Up to 64 tokens: the product is bound by the weights' bytes and by latency, so a
// workgroup takes 16 output channels, its waves cut the contraction among themselves and read the weights straight into
// MFMA operands.  Up to a few tokens the workgroups also quantise the rows themselves and one launch does it all.

#include "common.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int I8_MAX_K = 131072;
constexpr int I8_BK = 128;   // bytes (values) of a row in one k-step

// ---------------------------------------------------------------------------------------------
// One value.  s is at least 2^-126 and |x| <= 127.00001 s.
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ int i8_round(float x, float s, float inv) {
  float q = rintf(x * inv);
  const float up = fmaf(-(q + 0.5f), s, x), down = fmaf(-(q - 0.5f), s, x);   // exact signs
  const bool odd = ((int)q) & 1;
  if (up > 0.f || (up == 0.f && odd)) q += 1.f;
  else if (down < 0.f || (down == 0.f && odd)) q -= 1.f;
  return (int)fminf(fmaxf(q, -127.f), 127.f);
}
__device__ __forceinline__ float i8_scale(float amax) { return fmaxf(__fdiv_rn(amax, 127.f), 1.17549435e-38f); }
__device__ __forceinline__ unsigned i8_pack(int a, int b, int c, int d) {
  return (unsigned)(a & 255) | (unsigned)(b & 255) << 8 | (unsigned)(c & 255) << 16 | (unsigned)(d & 255) << 24;
}

struct QuantArgs {
  const void* x;
  int8_t* q;
  float* scale;
  long ldx, ldq, M;
  int K;
};

// eight values of a row from column k on; columns past K read as zero
template <bool BF16, bool VEC>
__device__ __forceinline__ void i8_load8(const void* row, int k, int K, float (&v)[8]) {
  if (VEC && k + 8 <= K) {
    load8<BF16>(row, (size_t)k, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k + j < K ? load1<BF16>(row, (size_t)(k + j)) : 0.f;
  }
}
// maximum of |v| that carries NaN and infinity as NaN: `bad` collects them
__device__ __forceinline__ void i8_amax8(const float (&v)[8], float& amax, bool& bad) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float a = fabsf(v[j]);
    bad |= !(a < INFINITY);
    amax = fmaxf(amax, a);
  }
}
__device__ __forceinline__ u32x2 i8_quant8(const float (&v)[8], float s, float inv, bool bad) {
  int q[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) q[j] = bad ? 0 : i8_round(v[j], s, inv);
  return u32x2{i8_pack(q[0], q[1], q[2], q[3]), i8_pack(q[4], q[5], q[6], q[7])};
}

// One wave per row: E x 512 columns in registers, or (E = 0) the row read twice.  Writes zeros up to the row's pitch.
template <bool BF16, bool VEC, int E>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const QuantArgs a) {
  const int lane = threadIdx.x & 63;
  const long m = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (m >= a.M) return;
  const void* row = reinterpret_cast<const unsigned char*>(a.x) + m * a.ldx * (BF16 ? 2 : 4);
  int8_t* out = a.q + m * a.ldq;
  float amax = 0.f;
  bool bad = false;
  if constexpr (E > 0) {
    float v[E][8];
#pragma unroll
    for (int i = 0; i < E; ++i) i8_load8<BF16, VEC>(row, i * 512 + lane * 8, a.K, v[i]);
#pragma unroll
    for (int i = 0; i < E; ++i) i8_amax8(v[i], amax, bad);
    amax = wave_max(amax);
    bad = __ballot(bad) != 0;
    const float s = i8_scale(amax), inv = 1.0f / s;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int k = i * 512 + lane * 8;
      if (k < a.ldq) *reinterpret_cast<u32x2*>(out + k) = i8_quant8(v[i], s, inv, bad);
    }
    if (lane == 0) a.scale[m] = bad ? NAN : s;
  } else {
    for (int k = lane * 8; k < a.K; k += 512) {
      float v[8];
      i8_load8<BF16, VEC>(row, k, a.K, v);
      i8_amax8(v, amax, bad);
    }
    amax = wave_max(amax);
    bad = __ballot(bad) != 0;
    const float s = i8_scale(amax), inv = 1.0f / s;
    for (int k = lane * 8; k < a.ldq; k += 512) {
      float v[8];
      i8_load8<BF16, VEC>(row, k, a.K, v);
      *reinterpret_cast<u32x2*>(out + k) = i8_quant8(v, s, inv, bad);
    }
    if (lane == 0) a.scale[m] = bad ? NAN : s;
  }
}

// ---------------------------------------------------------------------------------------------
// Many tokens: 64 TM x 64 TN output tiles, four waves of 32 TM x 32 TN
// ---------------------------------------------------------------------------------------------
struct Int8Args {
  const int8_t* q;        // (M, ldq) with zeros from K to ldq, a multiple of I8_BK
  const int8_t* w;        // (N, ldw), K values in whole 16-byte pieces
  const float* x_scale;
  const float* w_scale;
  const void* bias;
  void* y;
  const unsigned int* zeros;
  long ldq, ldw, ldy;
  int M, N, K, bias_bf16, tiles_m, tiles_n, y_vec;
};

__device__ __forceinline__ void i8_glds16(const void* src, void* lds_dst) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                   (__attribute__((address_space(3))) void*)lds_dst, 16, 0, 0);
}
// piece c (16 values) of row r of a [rows][128] image lies at position c ^ i8_swz(r): the rows that one group of
// ds_read_b128 lanes touches then fall on distinct 16-byte slots of the bank row
__device__ __forceinline__ int i8_swz(int r) { return (r >> 1) & 7; }

__device__ __forceinline__ float i8_bias(const Int8Args& g, int n) {
  if (g.bias == nullptr) return 0.f;
  return g.bias_bf16 ? bf16_to_f32(reinterpret_cast<const bf16_t*>(g.bias)[n]) : reinterpret_cast<const float*>(g.bias)[n];
}

template <bool OUT_BF16, int TM, int TN>
__global__ __launch_bounds__(256) void int8_tile_kernel(const Int8Args g) {
  constexpr int BM = 64 * TM, BN = 64 * TN, XB = BM * I8_BK, WB = BN * I8_BK;
  constexpr int ES = OUT_BF16 ? 2 : 4;
  constexpr int PITCH = 32 * TN * ES + (OUT_BF16 ? 8 : 16);   // of a wave's image of 32 tokens x 32 TN channels
  constexpr int IMG = 4 * 32 * PITCH;
  __shared__ __attribute__((aligned(16))) unsigned char lds[XB + WB > IMG ? XB + WB : IMG];
  // each XCD gets a contiguous run of tiles, columns fastest (workgroup ids go round-robin over the 8 XCDs)
  const int nt = g.tiles_m * g.tiles_n;
  const int xcd = blockIdx.x & 7, share = nt >> 3, more = nt & 7;
  const int lin = (xcd < more ? xcd * (share + 1) : more * (share + 1) + (xcd - more) * share) + (blockIdx.x >> 3);
  const int tile_m = lin / g.tiles_n, tile_n = lin - tile_m * g.tiles_n;
  const int m0 = tile_m * BM, n0 = tile_n * BN;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1, half = lane >> 5;

  // LDS-DMA sources: piece j * 256 + tid -> (row piece / 8, position piece % 8)
  constexpr int XJ = 2 * TM, WJ = 2 * TN;
  const int8_t* xs[XJ];
  const int8_t* ws[WJ];
  int wk[WJ];
#pragma unroll
  for (int j = 0; j < XJ; ++j) {
    const int p = j * 256 + tid, row = p >> 3, c = (p & 7) ^ i8_swz(row);
    xs[j] = g.q + (long)min(m0 + row, g.M - 1) * g.ldq + c * 16;   // rows past the edge repeat the last one;
  }
#pragma unroll
  for (int j = 0; j < WJ; ++j) {
    const int p = j * 256 + tid, row = p >> 3, c = (p & 7) ^ i8_swz(row);
    ws[j] = g.w + (long)min(n0 + row, g.N - 1) * g.ldw + c * 16;   // their outputs are not stored
    wk[j] = c * 16;
  }
  unsigned char* const dma_x = lds + wave * 1024;
  unsigned char* const dma_w = lds + XB + wave * 1024;

  int xr[TM], wr[TN];
#pragma unroll
  for (int i = 0; i < TM; ++i) xr[i] = wm * 32 * TM + i * 32 + (lane & 31);
#pragma unroll
  for (int j = 0; j < TN; ++j) wr[j] = wn * 32 * TN + j * 32 + (lane & 31);

  i32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;

  const int T = (int)(g.ldq / I8_BK);
  for (int t = 0; t < T; ++t) {
    const int k0 = t * I8_BK;
#pragma unroll
    for (int j = 0; j < XJ; ++j) i8_glds16(xs[j] + k0, dma_x + j * 4096);
#pragma unroll
    for (int j = 0; j < WJ; ++j) {
      // pieces past the weights' row (the tokens' integers are zero there) come from the block of zeros
      const void* src = k0 + wk[j] < g.K ? (const void*)(ws[j] + k0) : (const void*)g.zeros;
      i8_glds16(src, dma_w + j * 4096);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      i32x4 xf[TM], wf[TN];
#pragma unroll
      for (int i = 0; i < TM; ++i)
        xf[i] = *reinterpret_cast<const i32x4*>(lds + xr[i] * I8_BK + (((2 * ks + half) ^ i8_swz(xr[i])) << 4));
#pragma unroll
      for (int j = 0; j < TN; ++j)
        wf[j] = *reinterpret_cast<const i32x4*>(lds + XB + wr[j] * I8_BK + (((2 * ks + half) ^ i8_swz(wr[j])) << 4));
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[j], xf[i], acc[i][j], 0, 0, 0);
    }
    __syncthreads();
  }

  // acc[i][j][e]: token wm 32 TM + 32 i + (lane & 31), channel wn 32 TN + 32 j + (e & 3) + 8 (e >> 2) + 4 half
  unsigned char* const img = lds + wave * (32 * PITCH);
  float sw[TN][16], bv[TN][16];
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int n = min(n0 + (wn * TN + j) * 32 + (e & 3) + 8 * (e >> 2) + 4 * half, g.N - 1);
      sw[j][e] = g.w_scale[n];
      bv[j][e] = i8_bias(g, n);
    }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const float sx = g.x_scale[min(m0 + xr[i], g.M - 1)];
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[e] = fmaf((float)acc[i][j][4 * r + e] * sx, sw[j][4 * r + e], bv[j][4 * r + e]);
        unsigned char* at = img + (lane & 31) * PITCH + (j * 32 + 8 * r + 4 * half) * ES;
        if constexpr (OUT_BF16) *reinterpret_cast<u32x2*>(at) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
        else *reinterpret_cast<f32x4*>(at) = f32x4{v[0], v[1], v[2], v[3]};
      }
    // the image is the wave's own, and its LDS operations complete in order
    constexpr int PER = 16 / ES, CH = 32 * TN / PER, ROWS = 64 / CH;   // pieces per row, rows per round
#pragma unroll
    for (int it = 0; it < 32 / ROWS; ++it) {
      const int ml = it * ROWS + lane / CH, c = lane % CH;
      const int m = m0 + (wm * TM + i) * 32 + ml, n = n0 + wn * 32 * TN + c * PER;
      const unsigned char* at = img + ml * PITCH + c * 16;
      const u32x2 lo = *reinterpret_cast<const u32x2*>(at), hi = *reinterpret_cast<const u32x2*>(at + 8);
      if (m < g.M && n < g.N) {
        unsigned char* yp = reinterpret_cast<unsigned char*>(g.y) + ((long)m * g.ldy + n) * ES;
        if (g.y_vec && n + PER <= g.N) {
          *reinterpret_cast<u32x4*>(yp) = u32x4{lo.x, lo.y, hi.x, hi.y};
        } else {
          const unsigned w[4] = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
          for (int e = 0; e < PER; ++e)
            if (n + e < g.N) {
              if constexpr (OUT_BF16) reinterpret_cast<bf16_t*>(yp)[e] = (bf16_t)(w[e >> 1] >> (16 * (e & 1)));
              else reinterpret_cast<unsigned*>(yp)[e] = w[e];
            }
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// ---------------------------------------------------------------------------------------------
// Few tokens: 16 output channels per workgroup, the contraction cut among its four waves
// ---------------------------------------------------------------------------------------------
constexpr int I8_SELF = 4;          // tokens whose rows the workgroups quantise themselves
constexpr int I8_SELF_K = 8192;     // and the columns up to which they do

// MT blocks of 16 tokens.  SELF: the tokens are x itself, quantised into shared memory (M <= I8_SELF, K <= I8_SELF_K).
template <bool X_BF16, bool OUT_BF16, int MT, bool SELF>
__global__ __launch_bounds__(256) void int8_few_kernel(const Int8Args g, const void* x, long ldx, int x_vec) {
  __shared__ __attribute__((aligned(16))) i32x4 s_part[4][MT][64];
  __shared__ float s_red[4];
  __shared__ int s_bad[4];
  __shared__ float s_scale[I8_SELF];
  extern __shared__ __attribute__((aligned(16))) unsigned char s_q[];   // SELF: (M, kp)
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n0 = blockIdx.x * 16;
  const int kp = (g.K + 63) & ~63;
  const int steps = kp >> 6, mine = (steps + 3) >> 2;   // 64 columns a step, a contiguous run for each wave
  const int s0 = min(steps, wave * mine), s1 = min(steps, s0 + mine);
  const int8_t* wrow = g.w + (long)min(n0 + (lane & 15), g.N - 1) * g.ldw;
  const int kl = (lane >> 4) * 16;

  if constexpr (SELF) {
    for (int m = 0; m < g.M; ++m) {
      const void* row = reinterpret_cast<const unsigned char*>(x) + m * ldx * (X_BF16 ? 2 : 4);
      float amax = 0.f;
      bool bad = false;
      for (int k = tid * 8; k < g.K; k += 2048) {
        float v[8];
        if (x_vec) i8_load8<X_BF16, true>(row, k, g.K, v);
        else i8_load8<X_BF16, false>(row, k, g.K, v);
        i8_amax8(v, amax, bad);
      }
      amax = wave_max(amax);
      bad = __ballot(bad) != 0;
      __syncthreads();
      if (lane == 0) {
        s_red[wave] = amax;
        s_bad[wave] = bad;
      }
      __syncthreads();
      amax = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
      bad = (s_bad[0] | s_bad[1] | s_bad[2] | s_bad[3]) != 0;
      const float s = i8_scale(amax), inv = 1.0f / s;
      for (int k = tid * 8; k < kp; k += 2048) {
        float v[8];
        if (x_vec) i8_load8<X_BF16, true>(row, k, g.K, v);
        else i8_load8<X_BF16, false>(row, k, g.K, v);
        *reinterpret_cast<u32x2*>(s_q + m * kp + k) = i8_quant8(v, s, inv, bad);
      }
      if (tid == 0) s_scale[m] = bad ? NAN : s;
    }
    __syncthreads();
  }

  i32x4 acc[MT];
#pragma unroll
  for (int b = 0; b < MT; ++b) acc[b] = i32x4{0, 0, 0, 0};
  for (int s = s0; s < s1; ++s) {
    const int k = s * 64 + kl;
    // (weights past K meet zeros; the piece that holds column K - 1 is whole, the next ones are not read)
    const i32x4 wf = k < g.K ? *reinterpret_cast<const i32x4*>(wrow + k) : i32x4{0, 0, 0, 0};
#pragma unroll
    for (int b = 0; b < MT; ++b) {
      const int m = b * 16 + (lane & 15);
      i32x4 xf = i32x4{0, 0, 0, 0};
      if constexpr (SELF) {
        if (m < g.M) xf = *reinterpret_cast<const i32x4*>(s_q + m * kp + k);
      } else {
        xf = *reinterpret_cast<const i32x4*>(g.q + (long)min(m, g.M - 1) * g.ldq + k);
      }
      acc[b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf, xf, acc[b], 0, 0, 0);
    }
  }
#pragma unroll
  for (int b = 0; b < MT; ++b) s_part[wave][b][lane] = acc[b];
  __syncthreads();
  // acc[b][e]: token 16 b + (lane & 15), channel 4 (lane >> 4) + e
  for (int b = wave; b < MT; b += 4) {
    i32x4 t = s_part[0][b][lane];
#pragma unroll
    for (int w = 1; w < 4; ++w) t += s_part[w][b][lane];
    const int m = b * 16 + (lane & 15);
    if (m < g.M) {
      const float sx = SELF ? s_scale[m < I8_SELF ? m : 0] : g.x_scale[m];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = n0 + 4 * (lane >> 4) + e;
        if (n < g.N) store1<OUT_BF16>(g.y, (size_t)m * g.ldy + n, fmaf((float)t[e] * sx, g.w_scale[n], i8_bias(g, n)));
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------
bool i8_self(int M, int K) { return M <= I8_SELF && K <= I8_SELF_K; }
constexpr int I8_FEW = 64;

long i8_pitch(int K) { return ((long)K + I8_BK - 1) / I8_BK * I8_BK; }
size_t i8_scale_offset(long M, int K) { return ((size_t)M * i8_pitch(K) + 255) / 256 * 256; }

template <bool BF16, bool VEC>
void i8_launch_quant(const QuantArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)((a.M + 3) / 4)), block(256);
  if (a.ldq <= 512) hipLaunchKernelGGL((quantize_rows_kernel<BF16, VEC, 1>), grid, block, 0, st, a);
  else if (a.ldq <= 1024) hipLaunchKernelGGL((quantize_rows_kernel<BF16, VEC, 2>), grid, block, 0, st, a);
  else if (a.ldq <= 2048) hipLaunchKernelGGL((quantize_rows_kernel<BF16, VEC, 4>), grid, block, 0, st, a);
  else if (a.ldq <= 4096) hipLaunchKernelGGL((quantize_rows_kernel<BF16, VEC, 8>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((quantize_rows_kernel<BF16, VEC, 0>), grid, block, 0, st, a);
}
bool i8_vec(const void* p, long ld, int dtype) { return vqaf_aligned16(p) && (ld * (long)vqaf_esize(dtype)) % 16 == 0; }

void i8_quant(const void* x, long ldx, int M, int K, int dtype, int8_t* q, long ldq, float* scale, hipStream_t st) {
  QuantArgs a;
  a.x = x; a.q = q; a.scale = scale; a.ldx = ldx; a.ldq = ldq; a.M = M; a.K = K;
  const bool vec = i8_vec(x, ldx, dtype);
  if (dtype == VQAF_BF16) vec ? i8_launch_quant<true, true>(a, st) : i8_launch_quant<true, false>(a, st);
  else vec ? i8_launch_quant<false, true>(a, st) : i8_launch_quant<false, false>(a, st);
}

template <bool XB, bool YB, bool SELF>
void i8_launch_few(const Int8Args& g, const void* x, long ldx, int x_vec, hipStream_t st) {
  const dim3 grid((unsigned)((g.N + 15) / 16)), block(256);
  if constexpr (SELF) {
    const size_t lds = (size_t)g.M * ((g.K + 63) / 64 * 64);
    hipLaunchKernelGGL((int8_few_kernel<XB, YB, 1, true>), grid, block, lds, st, g, x, ldx, x_vec);
  } else {
    if (g.M <= 16) hipLaunchKernelGGL((int8_few_kernel<true, YB, 1, false>), grid, block, 0, st, g, x, ldx, x_vec);
    else if (g.M <= 32) hipLaunchKernelGGL((int8_few_kernel<true, YB, 2, false>), grid, block, 0, st, g, x, ldx, x_vec);
    else hipLaunchKernelGGL((int8_few_kernel<true, YB, 4, false>), grid, block, 0, st, g, x, ldx, x_vec);
  }
}

template <bool YB>
void i8_launch_tiles(Int8Args& g, hipStream_t st) {
  const long big = (long)((g.M + 127) / 128) * ((g.N + 127) / 128);
  if (big >= 256) {
    g.tiles_m = (g.M + 127) / 128;
    g.tiles_n = (g.N + 127) / 128;
    hipLaunchKernelGGL((int8_tile_kernel<YB, 2, 2>), dim3((unsigned)(g.tiles_m * g.tiles_n)), dim3(256), 0, st, g);
  } else {
    g.tiles_m = (g.M + 63) / 64;
    g.tiles_n = (g.N + 63) / 64;
    hipLaunchKernelGGL((int8_tile_kernel<YB, 1, 1>), dim3((unsigned)(g.tiles_m * g.tiles_n)), dim3(256), 0, st, g);
  }
}

}  // namespace

extern "C" int vqaf_quantize_rows(const void* x, long ldx, int M, int K, int dtype, int8_t* q, long ldq, float* scale,
                                  vqaf_stream_t stream) {
  VQAF_ENTRY();
  VQAF_REQUIRE(x && q && scale, VQAF_E_NULL);
  VQAF_REQUIRE(M > 0 && K > 0 && ldx >= 0 && ldq >= K && ldq % 16 == 0 && ldq < 0x7ffff000L, VQAF_E_SHAPE);
  VQAF_REQUIRE(vqaf_dtype_ok(dtype), VQAF_E_DTYPE);
  VQAF_REQUIRE(vqaf_aligned16(q) && reinterpret_cast<uintptr_t>(x) % vqaf_esize(dtype) == 0, VQAF_E_ALIGN);
  i8_quant(x, ldx, M, K, dtype, q, ldq, scale, (hipStream_t)stream);
  VQAF_LAUNCH_CHECK();
}

extern "C" size_t vqaf_int8_linear_workspace_bytes(int M, int K) {
  if (M <= 0 || K <= 0 || i8_self(M, K)) return 0;
  return i8_scale_offset(M, K) + (size_t)M * sizeof(float);
}

extern "C" int vqaf_int8_linear(const void* x, long ldx, int x_dtype, const int8_t* w, long ldw, const float* w_scale,
                                const void* bias, int bias_dtype, int M, int N, int K, void* y, long ldy, int y_dtype,
                                void* workspace, size_t workspace_bytes, vqaf_stream_t stream) {
  VQAF_ENTRY();
  VQAF_REQUIRE(x && w && w_scale && y, VQAF_E_NULL);
  VQAF_REQUIRE(M > 0 && N > 0 && K > 0 && K <= I8_MAX_K && ldx >= 0 && ldw >= (K + 15) / 16 * 16 && ldw % 16 == 0 && ldy >= N,
               VQAF_E_SHAPE);
  VQAF_REQUIRE((long)((M + 63) / 64) * ((N + 63) / 64) < 0x7fffffffL, VQAF_E_SHAPE);
  VQAF_REQUIRE(vqaf_dtype_ok(x_dtype) && vqaf_dtype_ok(y_dtype) && (bias == nullptr || vqaf_dtype_ok(bias_dtype)), VQAF_E_DTYPE);
  VQAF_REQUIRE(vqaf_aligned16(w) && reinterpret_cast<uintptr_t>(x) % vqaf_esize(x_dtype) == 0 &&
               reinterpret_cast<uintptr_t>(y) % vqaf_esize(y_dtype) == 0 && reinterpret_cast<uintptr_t>(w_scale) % 4 == 0 &&
               (bias == nullptr || reinterpret_cast<uintptr_t>(bias) % vqaf_esize(bias_dtype) == 0), VQAF_E_ALIGN);
  const size_t need = vqaf_int8_linear_workspace_bytes(M, K);
  VQAF_REQUIRE(need == 0 || workspace != nullptr, VQAF_E_NULL);
  VQAF_REQUIRE(workspace_bytes >= need, VQAF_E_SHAPE);
  VQAF_REQUIRE(need == 0 || vqaf_aligned16(workspace), VQAF_E_ALIGN);
  hipStream_t st = (hipStream_t)stream;
  Int8Args g;
  g.w = w; g.w_scale = w_scale; g.bias = bias; g.bias_bf16 = bias_dtype == VQAF_BF16; g.y = y;
  g.q = nullptr; g.x_scale = nullptr; g.zeros = nullptr;
  g.ldw = ldw; g.ldy = ldy; g.ldq = i8_pitch(K);
  g.M = M; g.N = N; g.K = K; g.tiles_m = g.tiles_n = 0;
  g.y_vec = i8_vec(y, ldy, y_dtype);
  const bool xb = x_dtype == VQAF_BF16, yb = y_dtype == VQAF_BF16;
  if (i8_self(M, K)) {
    const int vec = i8_vec(x, ldx, x_dtype);
    if (xb && yb) i8_launch_few<true, true, true>(g, x, ldx, vec, st);
    else if (xb) i8_launch_few<true, false, true>(g, x, ldx, vec, st);
    else if (yb) i8_launch_few<false, true, true>(g, x, ldx, vec, st);
    else i8_launch_few<false, false, true>(g, x, ldx, vec, st);
    VQAF_LAUNCH_CHECK();
  }
  int8_t* q = reinterpret_cast<int8_t*>(workspace);
  float* s = reinterpret_cast<float*>(q + i8_scale_offset(M, K));
  i8_quant(x, ldx, M, K, x_dtype, q, g.ldq, s, st);
  g.q = q;
  g.x_scale = s;
  if (M <= I8_FEW) {
    yb ? i8_launch_few<true, true, false>(g, x, ldx, 0, st) : i8_launch_few<true, false, false>(g, x, ldx, 0, st);
  } else {
    VQAF_REQUIRE(vqaf_internal_zero_block(&g.zeros) == VQAF_OK, VQAF_E_LAUNCH);
    yb ? i8_launch_tiles<true>(g, st) : i8_launch_tiles<false>(g, st);
  }
  VQAF_LAUNCH_CHECK();
}
