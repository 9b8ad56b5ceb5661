// Linear layers in eight-bit integers with a scale for each token and each output channel: the scoring and labelling
// passes of the encoders (model/vision_encoder.py:83-127, model/text_encoder.py:14-48 run these layers in f32).
//
//   s_m = max(max_k |x_mk| / 127, 2^-126),   q_mk = round-half-even(x_mk / s_m),   y_mn = (sum_k q_mk w_nk) s_m s_n + b_n
//
// The sum is exact in 32-bit integers (127^2 K < 2^31 for K up to 131072); the two scales, the bias and the rounding to
// the output type follow in f32, in the epilogue, without leaving its range on the way where the result does not.  The
// quotient is rounded as if it were exact: next to a border the sign of x - (q +- 1/2) s, one fused multiply-add, decides.  A
// row with NaN or an infinity gets the scale NaN, which makes its outputs NaN.
//
// Many tokens: one pass writes the rows as integers, bound by its bytes, and a matrix product on 32x32x32 integer MFMAs
// reads them through a ring of stages in shared memory.  Up to 64 tokens: the product is bound by the weights' bytes and
// by latency, so a workgroup takes 16 output channels, its waves cut the contraction among themselves and read the weights
// straight into MFMA operands.  Up to four tokens the workgroups quantise the rows themselves and one launch does it all.

#include <mutex>
#include <type_traits>

#include "common.h"
#include "wave.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int I8_MAX_K = 131072;
constexpr int I8_ROW = 128;   // rows of quantised tokens are whole multiples of this many bytes

// ---------------------------------------------------------------------------------------------
// One value.  s is at least 2^-126 and |x| <= 127.00001 s, so the result stays in [-127, 127].
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ int i8_round(float x, float s, float inv) {
  float q = rintf(x * inv);
  if (s < 0x1p-100f) {   // half a step may be finer than f32's smallest number: both 2^64 times as large, exactly
    x *= 0x1p64f;
    s *= 0x1p64f;
  }
  const float up = fmaf(-(q + 0.5f), s, x), down = fmaf(-(q - 0.5f), s, x);   // exact signs
  const bool odd = ((int)q) & 1;
  if (up > 0.f || (up == 0.f && odd)) q += 1.f;
  else if (down < 0.f || (down == 0.f && odd)) q -= 1.f;
  return (int)q;
}
__device__ __forceinline__ float i8_scale(float amax) { return fmaxf(__fdiv_rn(amax, 127.f), 1.17549435e-38f); }
__device__ __forceinline__ unsigned i8_pack(int a, int b, int c, int d) {
  return (unsigned)(a & 255) | (unsigned)(b & 255) << 8 | (unsigned)(c & 255) << 16 | (unsigned)(d & 255) << 24;
}

struct QuantArgs {
  const void* x;
  int8_t* q;
  float* scale;
  long ldx, ldq, M, m0;   // m0: the launch's first row
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
// Maximum of |v| as bits: NaN lies above infinity, infinity above every number.
__device__ __forceinline__ unsigned i8_amax8(const float (&v)[8], unsigned amax) {
#pragma unroll
  for (int j = 0; j < 8; ++j) amax = max(amax, __float_as_uint(v[j]) & 0x7fffffffu);
  return amax;
}
__device__ __forceinline__ bool i8_bad(unsigned amax) { return amax >= 0x7f800000u; }
// x * inv is off by less than 2^-15 steps, so only a remainder that close to half a step leaves a doubt
__device__ __forceinline__ u32x2 i8_quant8(const float (&v)[8], float s, float inv, bool bad) {
  int q[8];
  bool doubt = false;
  const float near = 0.49996f * s;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float f = rintf(v[j] * inv);
    doubt |= fabsf(fmaf(-f, s, v[j])) > near;
    q[j] = (int)f;
  }
  if (doubt) {
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = i8_round(v[j], s, inv);
  }
  const u32x2 r = u32x2{i8_pack(q[0], q[1], q[2], q[3]), i8_pack(q[4], q[5], q[6], q[7])};
  return bad ? u32x2{0, 0} : r;
}

// The same eight values as they lie in memory (bf16 takes half the registers of f32).
template <bool BF16>
struct I8Raw {
  u32x4 r[BF16 ? 1 : 2];
};
template <bool BF16, bool VEC>
__device__ __forceinline__ I8Raw<BF16> i8_load8_raw(const void* row, int k, int K) {
  I8Raw<BF16> o;
  if (VEC && k + 8 <= K) {
    const u32x4* p = reinterpret_cast<const u32x4*>(reinterpret_cast<const unsigned char*>(row) + (size_t)k * (BF16 ? 2 : 4));
    o.r[0] = p[0];
    if constexpr (!BF16) o.r[1] = p[1];
  } else {
    unsigned w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k + j < K) {
        if constexpr (BF16) w[j >> 1] |= (unsigned)reinterpret_cast<const bf16_t*>(row)[k + j] << (16 * (j & 1));
        else w[j] = reinterpret_cast<const unsigned*>(row)[k + j];
      }
    o.r[0] = u32x4{w[0], w[1], w[2], w[3]};
    if constexpr (!BF16) o.r[1] = u32x4{w[4], w[5], w[6], w[7]};
  }
  return o;
}
template <bool BF16>
__device__ __forceinline__ void i8_unpack(const I8Raw<BF16>& o, float (&v)[8]) {
  if constexpr (BF16) {
    const u32x4 r = o.r[0];
    v[0] = bf16_lo(r.x); v[1] = bf16_hi(r.x); v[2] = bf16_lo(r.y); v[3] = bf16_hi(r.y);
    v[4] = bf16_lo(r.z); v[5] = bf16_hi(r.z); v[6] = bf16_lo(r.w); v[7] = bf16_hi(r.w);
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      v[4 * h] = __uint_as_float(o.r[h].x); v[4 * h + 1] = __uint_as_float(o.r[h].y);
      v[4 * h + 2] = __uint_as_float(o.r[h].z); v[4 * h + 3] = __uint_as_float(o.r[h].w);
    }
  }
}
// Running maximum of the magnitudes' bits: pairs of 16 (bf16) or one of 32.
typedef unsigned short i8_u16x2 __attribute__((ext_vector_type(2)));
template <bool BF16>
__device__ __forceinline__ unsigned i8_amax_raw(const I8Raw<BF16>& o, unsigned top) {
  if constexpr (BF16) {
    const unsigned w[4] = {o.r[0].x, o.r[0].y, o.r[0].z, o.r[0].w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      top = __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(i8_u16x2, top),
                                                                   __builtin_bit_cast(i8_u16x2, w[j] & 0x7fff7fffu)));
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const unsigned w[4] = {o.r[h].x, o.r[h].y, o.r[h].z, o.r[h].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) top = max(top, w[j] & 0x7fffffffu);
    }
  }
  return top;
}
template <bool BF16>
__device__ __forceinline__ unsigned i8_amax_bits(unsigned top) {   // as the bits of an f32
  return BF16 ? max(top << 16, top & 0xffff0000u) : top;
}

// One wave per row: E x 512 columns in registers, or (E = 0) the row read twice.  Writes zeros up to the row's pitch.
// Measured, bf16: 8191 x 4096 24 us (4.2 TB/s read and written), 12608 x 768 10 us (2.9 TB/s: a row is only 1.5 KB); f32:
// 38 us (4.4 TB/s), 10 us.
template <bool BF16, bool VEC, int E>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const QuantArgs a) {
  const int lane = threadIdx.x & 63;
  const long m = a.m0 + (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (m >= a.M) return;
  const void* row = reinterpret_cast<const unsigned char*>(a.x) + m * a.ldx * (BF16 ? 2 : 4);
  int8_t* out = a.q + m * a.ldq;
  unsigned top = 0;
  if constexpr (E > 0) {
    I8Raw<BF16> x[E];
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = i8_load8_raw<BF16, VEC>(row, i * 512 + lane * 8, a.K);
#pragma unroll
    for (int i = 0; i < E; ++i) top = i8_amax_raw<BF16>(x[i], top);
    top = dpp_wave_umax(i8_amax_bits<BF16>(top));
    const bool bad = i8_bad(top);
    const float s = i8_scale(__uint_as_float(top)), inv = 1.0f / s;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int k = i * 512 + lane * 8;
      float v[8];
      i8_unpack<BF16>(x[i], v);
      if (k < a.ldq) *reinterpret_cast<u32x2*>(out + k) = i8_quant8(v, s, inv, bad);
    }
    if (lane == 0) a.scale[m] = bad ? NAN : s;
  } else {
    for (int k = lane * 8; k < a.K; k += 512) {
      float v[8];
      i8_load8<BF16, VEC>(row, k, a.K, v);
      top = i8_amax8(v, top);
    }
    top = dpp_wave_umax(top);
    const bool bad = i8_bad(top);
    const float s = i8_scale(__uint_as_float(top)), inv = 1.0f / s;
    for (int k = lane * 8; k < a.ldq; k += 512) {
      float v[8];
      i8_load8<BF16, VEC>(row, k, a.K, v);
      *reinterpret_cast<u32x2*>(out + k) = i8_quant8(v, s, inv, bad);
    }
    if (lane == 0) a.scale[m] = bad ? NAN : s;
  }
}

// ---------------------------------------------------------------------------------------------
// Many tokens
// ---------------------------------------------------------------------------------------------
struct Int8Args {
  const int8_t* q;        // (M, ldq) with zeros from K to ldq, a multiple of I8_ROW
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
__device__ __forceinline__ float i8_bias(const Int8Args& g, int n) {
  if (g.bias == nullptr) return 0.f;
  return g.bias_bf16 ? bf16_to_f32(reinterpret_cast<const bf16_t*>(g.bias)[n]) : reinterpret_cast<const float*>(g.bias)[n];
}

// One output from its integer sum, (sum * token's scale) * channel's scale + bias with a rounding each.  A scale from 2^96
// on could carry the sum (below 2^31) past the f32 range before the channel's brings it back: of such a token 2^-64 goes
// through the products, and `back` is the 2^64 that is missing (1 of any other).
struct I8Token {
  float scale, back;
};
__device__ __forceinline__ I8Token i8_token(float scale) {
  const bool big = scale >= 0x1p96f;
  return I8Token{big ? scale * 0x1p-64f : scale, big ? 0x1p64f : 1.f};
}
__device__ __forceinline__ float i8_output(int sum, const I8Token t, float channel, float bias) {
  return fmaf((float)sum * t.scale * channel, t.back, bias);
}

// Scales and bias of a wave's tokens and channels, asked for before the product so that they are there after it: a lane
// has those of token 32 i + (lane & 31) and channel 32 j + (lane & 31).  The bias comes as its two halves, whatever its
// type, so that nothing is decided, and nothing awaited, before the product.
template <int TM, int TN>
struct I8Scales {
  float x[TM], w[TN];
  unsigned short lo[TN], hi[TN];
  __device__ __forceinline__ void load(const Int8Args& g, int m0, int n0, int lane) {
#pragma unroll
    for (int i = 0; i < TM; ++i) x[i] = g.x_scale[min(m0 + i * 32 + (lane & 31), g.M - 1)];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = min(n0 + j * 32 + (lane & 31), g.N - 1);
      w[j] = g.w_scale[n];
      const unsigned char* p = reinterpret_cast<const unsigned char*>(g.bias != nullptr ? g.bias : (const void*)g.zeros);
      const long at = g.bias == nullptr ? 0 : (long)n * (g.bias_bf16 ? 2 : 4);
      lo[j] = *reinterpret_cast<const unsigned short*>(p + at);
      hi[j] = *reinterpret_cast<const unsigned short*>(p + at + (g.bias_bf16 ? 0 : 2));
    }
  }
  __device__ __forceinline__ float bias(const Int8Args& g, int j) const {   // (bf16: both are the upper half)
    return __uint_as_float((unsigned)hi[j] << 16 | (g.bias_bf16 ? 0u : lo[j]));
  }
};

// A wave's 32 TM tokens x 32 TN channels from (m0, n0) on: scales, bias, rounding, and out through an image of 32 tokens
// in shared memory, so that stores are whole 16-byte pieces of rows.
// acc[i][j][e]: token 32 i + (lane & 31), channel 32 j + (e & 3) + 8 (e >> 2) + 4 (lane >> 5)
template <bool OUT_BF16, int TM, int TN>
__device__ __forceinline__ void i8_write_tile(const Int8Args& g, const I8Scales<TM, TN>& sc, i32x16 (&acc)[TM][TN], unsigned char* img,
                                              int m0, int n0, int lane) {
  constexpr int ES = OUT_BF16 ? 2 : 4;
  constexpr int PITCH = 32 * TN * ES + (OUT_BF16 ? 8 : 16);
  const int half = lane >> 5;
  float* chan = reinterpret_cast<float*>(img);   // the channels' scales and biases, from one lane each to all
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    chan[j * 64 + (lane & 31)] = sc.w[j];
    chan[j * 64 + 32 + (lane & 31)] = sc.bias(g, j);
  }
  asm volatile("" ::: "memory");
  I8Token token[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) token[i] = i8_token(sc.x[i]);
#pragma unroll
  for (int j = 0; j < TN; ++j) {   // in place: the sums become the outputs' bits
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const f32x4 sw = *reinterpret_cast<const f32x4*>(chan + j * 64 + 8 * r + 4 * half);
      const f32x4 bv = *reinterpret_cast<const f32x4*>(chan + j * 64 + 32 + 8 * r + 4 * half);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          acc[i][j][4 * r + e] = __float_as_int(i8_output(acc[i][j][4 * r + e], token[i], sw[e], bv[e]));
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  asm volatile("" ::: "memory");
#pragma unroll
  for (int i = 0; i < TM; ++i) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __int_as_float(acc[i][j][4 * r + e]);
        unsigned char* at = img + (lane & 31) * PITCH + (j * 32 + 8 * r + 4 * half) * ES;
        if constexpr (OUT_BF16) *reinterpret_cast<u32x2*>(at) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
        else *reinterpret_cast<f32x4*>(at) = f32x4{v[0], v[1], v[2], v[3]};
      }
    // the image is the wave's own, and its LDS operations complete in order
    constexpr int PER = 16 / ES, CH = 32 * TN / PER, ROWS = 64 / CH;   // pieces per row, rows per round
#pragma unroll
    for (int it = 0; it < 32 / ROWS; ++it) {
      const int ml = it * ROWS + lane / CH, c = lane % CH;
      const int m = m0 + i * 32 + ml, n = n0 + c * PER;
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

// The product: output tiles of 32 TM WM tokens x 32 TN WN channels, a workgroup of WM x WN waves of 32 TM x 32 TN each.
// k-steps of 64 values go through a ring of STAGES stages in shared memory, all but the one being read in flight, one
// barrier a step.  A wave reads the operands of a half step under the products of the half before.
// Measured: 8191 x 4096 x 4096 145 us on average and 133 to 157 from launch to launch (1.9 P operations/s), 8192 x 8192 x
// 8192 498 us (2.2 P; the library's product 2.1), where the chip's power sets the pace (1.8 GHz; the same with zeros 415 us
// at 2.3 GHz; matrix instructions alone, on random operands in registers, 3.5 P).  12608 x 768 x 2304 36 us (1.25 P: twelve
// k-steps, then 128 KB of output a workgroup that nothing overlaps, in two rounds of tiles of which the second is three
// quarters full; 43 us with f32 outputs), 1920 x 768 x 768 on 64 x 64 tiles 7.7 us, 500 x 4096 x 1024 12 us.  With each half
// step's operands awaited before its products they took 7 to 28 percent longer; scales and bias asked for after the
// product cost 4 us of the third.
constexpr int I8_BK = 64;

// piece c (16 values) of row r of a [rows][64] image lies at position c ^ i8_swz(r): sixteen rows on sixteen slots
__device__ __forceinline__ int i8_swz(int r) { return (r >> 2) & 3; }

// The operands of a wave's k32 step: TM token and TN channel fragments (blocks of 32 rows are 2048 bytes apart in the
// image and swizzled alike).
template <int TM, int TN>
struct I8Frag {
  i32x4 x[TM], w[TN];
};
// Inline assembly throughout: for a read that it can see, the compiler waits until every LDS-DMA has landed and would drain
// the ring.  Each block waits for its own reads, and ends with as many idle states as a reader of the last sum needs.
template <int TM, int TN>
__device__ __forceinline__ void i8_read(I8Frag<TM, TN>& n, unsigned xa, unsigned wa) {
  if constexpr (TM == 4 && TN == 2) {
    asm volatile("ds_read_b128 %4, %7\n\t"
                 "ds_read_b128 %5, %7 offset:2048\n\t"
                 "ds_read_b128 %0, %6\n\t"
                 "ds_read_b128 %1, %6 offset:2048\n\t"
                 "ds_read_b128 %2, %6 offset:4096\n\t"
                 "ds_read_b128 %3, %6 offset:6144\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(n.x[0]), "=&v"(n.x[1]), "=&v"(n.x[2]), "=&v"(n.x[3]), "=&v"(n.w[0]), "=&v"(n.w[1])
                 : "v"(xa), "v"(wa)
                 : "memory");
  } else if constexpr (TM == 2 && TN == 2) {
    asm volatile("ds_read_b128 %2, %5\n\t"
                 "ds_read_b128 %3, %5 offset:2048\n\t"
                 "ds_read_b128 %0, %4\n\t"
                 "ds_read_b128 %1, %4 offset:2048\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(n.x[0]), "=&v"(n.x[1]), "=&v"(n.w[0]), "=&v"(n.w[1])
                 : "v"(xa), "v"(wa)
                 : "memory");
  } else {
    static_assert(TM == 1 && TN == 1, "shapes with a block of their own");
    asm volatile("ds_read_b128 %1, %3\n\t"
                 "ds_read_b128 %0, %2\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(n.x[0]), "=&v"(n.w[0])
                 : "v"(xa), "v"(wa)
                 : "memory");
  }
}
// the products of c while the operands n of the next step arrive
template <int TM, int TN>
__device__ __forceinline__ void i8_step(i32x16 (&acc)[TM][TN], const I8Frag<TM, TN>& c, I8Frag<TM, TN>& n, unsigned xa, unsigned wa) {
  if constexpr (TM == 4 && TN == 2) {
    asm volatile("v_mfma_i32_32x32x32_i8 %0, %18, %14, %0\n\t"
                 "ds_read_b128 %12, %21\n\t"
                 "ds_read_b128 %8, %20\n\t"
                 "ds_read_b128 %13, %21 offset:2048\n\t"
                 "ds_read_b128 %9, %20 offset:2048\n\t"
                 "ds_read_b128 %10, %20 offset:4096\n\t"
                 "ds_read_b128 %11, %20 offset:6144\n\t"
                 "v_mfma_i32_32x32x32_i8 %1, %19, %14, %1\n\t"
                 "v_mfma_i32_32x32x32_i8 %2, %18, %15, %2\n\t"
                 "v_mfma_i32_32x32x32_i8 %3, %19, %15, %3\n\t"
                 "v_mfma_i32_32x32x32_i8 %4, %18, %16, %4\n\t"
                 "v_mfma_i32_32x32x32_i8 %5, %19, %16, %5\n\t"
                 "v_mfma_i32_32x32x32_i8 %6, %18, %17, %6\n\t"
                 "v_mfma_i32_32x32x32_i8 %7, %19, %17, %7\n\t"
                 "s_nop 11\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "+v"(acc[0][0]), "+v"(acc[0][1]), "+v"(acc[1][0]), "+v"(acc[1][1]), "+v"(acc[2][0]), "+v"(acc[2][1]), "+v"(acc[3][0]), "+v"(acc[3][1]), "=&v"(n.x[0]), "=&v"(n.x[1]), "=&v"(n.x[2]), "=&v"(n.x[3]), "=&v"(n.w[0]), "=&v"(n.w[1])
                 : "v"(c.x[0]), "v"(c.x[1]), "v"(c.x[2]), "v"(c.x[3]), "v"(c.w[0]), "v"(c.w[1]), "v"(xa), "v"(wa)
                 : "memory");
  } else if constexpr (TM == 2 && TN == 2) {
    asm volatile("v_mfma_i32_32x32x32_i8 %0, %10, %8, %0\n\t"
                 "ds_read_b128 %6, %13\n\t"
                 "ds_read_b128 %4, %12\n\t"
                 "ds_read_b128 %7, %13 offset:2048\n\t"
                 "ds_read_b128 %5, %12 offset:2048\n\t"
                 "v_mfma_i32_32x32x32_i8 %1, %11, %8, %1\n\t"
                 "v_mfma_i32_32x32x32_i8 %2, %10, %9, %2\n\t"
                 "v_mfma_i32_32x32x32_i8 %3, %11, %9, %3\n\t"
                 "s_nop 11\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "+v"(acc[0][0]), "+v"(acc[0][1]), "+v"(acc[1][0]), "+v"(acc[1][1]), "=&v"(n.x[0]), "=&v"(n.x[1]), "=&v"(n.w[0]), "=&v"(n.w[1])
                 : "v"(c.x[0]), "v"(c.x[1]), "v"(c.w[0]), "v"(c.w[1]), "v"(xa), "v"(wa)
                 : "memory");
  } else {
    static_assert(TM == 1 && TN == 1, "shapes with a block of their own");
    asm volatile("v_mfma_i32_32x32x32_i8 %0, %4, %3, %0\n\t"
                 "ds_read_b128 %2, %6\n\t"
                 "ds_read_b128 %1, %5\n\t"
                 "s_nop 11\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "+v"(acc[0][0]), "=&v"(n.x[0]), "=&v"(n.w[0])
                 : "v"(c.x[0]), "v"(c.w[0]), "v"(xa), "v"(wa)
                 : "memory");
  }
}
template <int TM, int TN>
__device__ __forceinline__ void i8_last(i32x16 (&acc)[TM][TN], const I8Frag<TM, TN>& c) {
  if constexpr (TM == 4 && TN == 2) {
    asm volatile("v_mfma_i32_32x32x32_i8 %0, %12, %8, %0\n\t"
                 "v_mfma_i32_32x32x32_i8 %1, %13, %8, %1\n\t"
                 "v_mfma_i32_32x32x32_i8 %2, %12, %9, %2\n\t"
                 "v_mfma_i32_32x32x32_i8 %3, %13, %9, %3\n\t"
                 "v_mfma_i32_32x32x32_i8 %4, %12, %10, %4\n\t"
                 "v_mfma_i32_32x32x32_i8 %5, %13, %10, %5\n\t"
                 "v_mfma_i32_32x32x32_i8 %6, %12, %11, %6\n\t"
                 "v_mfma_i32_32x32x32_i8 %7, %13, %11, %7\n\t"
                 "s_nop 15\n\t"
                 "s_nop 15"
                 : "+v"(acc[0][0]), "+v"(acc[0][1]), "+v"(acc[1][0]), "+v"(acc[1][1]), "+v"(acc[2][0]), "+v"(acc[2][1]), "+v"(acc[3][0]), "+v"(acc[3][1])
                 : "v"(c.x[0]), "v"(c.x[1]), "v"(c.x[2]), "v"(c.x[3]), "v"(c.w[0]), "v"(c.w[1]));
  } else if constexpr (TM == 2 && TN == 2) {
    asm volatile("v_mfma_i32_32x32x32_i8 %0, %6, %4, %0\n\t"
                 "v_mfma_i32_32x32x32_i8 %1, %7, %4, %1\n\t"
                 "v_mfma_i32_32x32x32_i8 %2, %6, %5, %2\n\t"
                 "v_mfma_i32_32x32x32_i8 %3, %7, %5, %3\n\t"
                 "s_nop 15\n\t"
                 "s_nop 15"
                 : "+v"(acc[0][0]), "+v"(acc[0][1]), "+v"(acc[1][0]), "+v"(acc[1][1])
                 : "v"(c.x[0]), "v"(c.x[1]), "v"(c.w[0]), "v"(c.w[1]));
  } else {
    static_assert(TM == 1 && TN == 1, "shapes with a block of their own");
    asm volatile("v_mfma_i32_32x32x32_i8 %0, %2, %1, %0\n\t"
                 "s_nop 15\n\t"
                 "s_nop 15"
                 : "+v"(acc[0][0])
                 : "v"(c.x[0]), "v"(c.w[0]));
  }
}

template <bool OUT_BF16, int TM, int TN, int WM, int WN, int STAGES, int OCC>
__global__ __launch_bounds__(64 * WM * WN, OCC) void int8_tile_kernel(const Int8Args g) {
  constexpr int THREADS = 64 * WM * WN, BM = 32 * TM * WM, BN = 32 * TN * WN;
  constexpr int XB = BM * I8_BK, STAGE = (BM + BN) * I8_BK;
  constexpr int XJ = BM * 4 / THREADS, WJ = BN * 4 / THREADS, D = XJ + WJ;   // LDS-DMA instructions a thread and stage
  constexpr int IMG = 32 * (32 * TN * (OUT_BF16 ? 2 : 4) + (OUT_BF16 ? 8 : 16));
  static_assert(XJ * THREADS == BM * 4 && WJ * THREADS == BN * 4, "whole rounds of LDS-DMA");
  static_assert(WM * WN * IMG <= STAGES * STAGE, "the output images fit the ring");
  extern __shared__ __attribute__((aligned(16))) unsigned char i8_lds[];   // STAGES * STAGE
  // each XCD gets a contiguous run of tiles (workgroup ids go round-robin over the 8 XCDs), in groups of four tile rows
  // with the columns slower within a group: what an XCD works on at a time shares operand rows both ways
  const int nt = g.tiles_m * g.tiles_n;
  const int xcd = blockIdx.x & 7, share = nt >> 3, more = nt & 7;
  const int lin = (xcd < more ? xcd * (share + 1) : more * (share + 1) + (xcd - more) * share) + (blockIdx.x >> 3);
  const int group = lin / (4 * g.tiles_n), first = group * 4, rows = min(4, g.tiles_m - first);
  const int in = lin - group * 4 * g.tiles_n, tile_n = in / rows, tile_m = first + in - tile_n * rows;
  const int m0 = tile_m * BM, n0 = tile_n * BN;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN, half = lane >> 5;

  I8Scales<TM, TN> scales;
  scales.load(g, m0 + wm * 32 * TM, n0 + wn * 32 * TN, lane);

  // LDS-DMA sources: piece j * THREADS + tid -> (row piece / 4, position piece % 4), as offsets from the tile's first rows;
  // rows past the edge repeat the last one, and their outputs are not stored
  const int8_t* xb = g.q + (long)m0 * g.ldq;
  const int8_t* wb = g.w + (long)n0 * g.ldw;
  unsigned xo[XJ];   // (tokens were laid out here: at most 256 rows of 128 KB)
  size_t wo[WJ];
  int wk[WJ];
#pragma unroll
  for (int j = 0; j < XJ; ++j) {
    const int p = j * THREADS + tid, row = p >> 2, c = (p & 3) ^ i8_swz(row);
    xo[j] = (unsigned)min(row, g.M - 1 - m0) * (unsigned)g.ldq + c * 16;
  }
#pragma unroll
  for (int j = 0; j < WJ; ++j) {
    const int p = j * THREADS + tid, row = p >> 2, c = (p & 3) ^ i8_swz(row);
    wo[j] = (size_t)min(row, g.N - 1 - n0) * (size_t)g.ldw + c * 16;
    wk[j] = c * 16;
  }
  const auto issue = [&](int t, int slot, bool whole) {
    unsigned char* st = i8_lds + slot * STAGE + wave * 1024;
    const int k0 = t * I8_BK;
    const int8_t* xk = xb + k0;
    const int8_t* wp = wb + k0;
#pragma unroll
    for (int j = 0; j < XJ; ++j) i8_glds16(xk + xo[j], st + j * (THREADS * 16));
    if (whole || k0 + I8_BK <= g.K) {
#pragma unroll
      for (int j = 0; j < WJ; ++j) i8_glds16(wp + wo[j], st + XB + j * (THREADS * 16));
    } else {   // pieces past the weights' row (the tokens are zero there) come from the block of zeros
#pragma unroll
      for (int j = 0; j < WJ; ++j)
        i8_glds16(k0 + wk[j] < g.K ? (const void*)(wp + wo[j]) : (const void*)g.zeros, st + XB + j * (THREADS * 16));
    }
  };

  const unsigned base = (unsigned)reinterpret_cast<size_t>((__attribute__((address_space(3))) unsigned char*)i8_lds);
  unsigned xa[2], wa[2];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    const int r = lane & 31;
    const unsigned at = base + (unsigned)(r * I8_BK + (((2 * ks + half) ^ i8_swz(r)) << 4));
    xa[ks] = at + wm * (32 * TM * I8_BK);
    wa[ks] = at + XB + wn * (32 * TN * I8_BK);
  }

  i32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;

  // Stages land in order: the oldest has when the instructions of the `behind` stages after it are all that is left.
  const auto landed = [&](int behind) {
    if (behind == STAGES - 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 1) * D) : "memory");
    else if (behind == STAGES - 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 2) * D) : "memory");
    else if (behind >= 2 && STAGES > 4) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * D) : "memory");
    else if (behind >= 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(D) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  };
  const int T = (int)(g.ldq / I8_BK);
#pragma unroll
  for (int s = 0; s < STAGES; ++s)
    if (s < T) issue(s, s, false);
  landed(min(T, STAGES) - 1);
  __builtin_amdgcn_s_barrier();
  I8Frag<TM, TN> even, odd;
  i8_read<TM, TN>(even, xa[0], wa[0]);
  int slot = 0, t = 0;
  // one stage: its second half is read under the first one's products, the next stage's first half under the second's
  const auto turn = [&](auto steady) {
    const unsigned st = (unsigned)(slot * STAGE);
    i8_step<TM, TN>(acc, even, odd, xa[1] + st, wa[1] + st);
    if constexpr (decltype(steady)::value) landed(STAGES - 2);
    else landed(min(T - 2 - t, STAGES - 2));
    __builtin_amdgcn_s_barrier();   // everyone's stage t + 1 has landed, and everyone has read stage t
    if constexpr (decltype(steady)::value) issue(t + STAGES, slot, true);
    else if (t + STAGES < T) issue(t + STAGES, slot, false);
    slot = slot == STAGES - 1 ? 0 : slot + 1;
    const unsigned sn = (unsigned)(slot * STAGE);
    i8_step<TM, TN>(acc, odd, even, xa[0] + sn, wa[0] + sn);
    ++t;
  };
  const int whole = g.K / I8_BK - STAGES;
  while (t < whole) turn(std::true_type());   // nothing to decide
  do turn(std::false_type()); while (t + 1 < T);   // T is at least 2: rows of tokens are whole multiples of two stages
  i8_step<TM, TN>(acc, even, odd, xa[1] + (unsigned)(slot * STAGE), wa[1] + (unsigned)(slot * STAGE));
  i8_last<TM, TN>(acc, odd);
  __syncthreads();   // the ring becomes the waves' output images
  i8_write_tile<OUT_BF16, TM, TN>(g, scales, acc, i8_lds + wave * IMG, m0 + wm * 32 * TM, n0 + wn * 32 * TN, lane);
}

// ---------------------------------------------------------------------------------------------
// Few tokens: 16 output channels per workgroup, the contraction cut among its four waves.  Measured: one token, 768 x 2304
// 5.0 us and 4096 x 4096 8.0 us (2.1 TB/s of weights), the quantiser and the launch included; 5, 16 and 64 tokens of 768 x 2304
// 4.0, 4.1 and 5.9 us behind a quantiser of 2.8, 3.4 and 4.3 us
// ---------------------------------------------------------------------------------------------
constexpr int I8_SELF = 4;          // tokens whose rows the workgroups quantise themselves
constexpr int I8_SELF_K = 8192;     // and the columns up to which they do

// MT blocks of 16 tokens.  SELF: the tokens are x itself, quantised into shared memory (M <= I8_SELF, K <= I8_SELF_K).
template <bool X_BF16, bool OUT_BF16, int MT, bool SELF>
__global__ __launch_bounds__(256) void int8_few_kernel(const Int8Args g, const void* x, long ldx, int x_vec) {
  __shared__ __attribute__((aligned(16))) i32x4 s_part[4][MT][64];
  __shared__ unsigned s_top[4];
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
      unsigned top = 0;
      for (int k = tid * 8; k < g.K; k += 2048) {
        float v[8];
        if (x_vec) i8_load8<X_BF16, true>(row, k, g.K, v);
        else i8_load8<X_BF16, false>(row, k, g.K, v);
        top = i8_amax8(v, top);
      }
      top = dpp_wave_umax(top);
      __syncthreads();
      if (lane == 0) s_top[wave] = top;
      __syncthreads();
      top = max(max(s_top[0], s_top[1]), max(s_top[2], s_top[3]));
      const bool bad = i8_bad(top);
      const float s = i8_scale(__uint_as_float(top)), inv = 1.0f / s;
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
  // the operands of four steps are requested together: the loop is all latency
  constexpr int U = 4;
  const int k_last = (g.K - 1) & ~15;
  for (int s = s0; s < s1; s += U) {
    i32x4 wf[U], xf[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // (weights past K meet zeros; the piece that holds column K - 1 is whole, the next ones are not read)
      const int k = (s + u) * 64 + kl;
      wf[u] = *reinterpret_cast<const i32x4*>(wrow + min(k, k_last));
      if constexpr (!SELF) {
#pragma unroll
        for (int b = 0; b < MT; ++b)
          xf[u][b] = *reinterpret_cast<const i32x4*>(g.q + (long)min(b * 16 + (lane & 15), g.M - 1) * g.ldq + min(k, kp - 16));
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (s + u) * 64 + kl;
      if (k >= g.K || s + u >= s1) wf[u] = i32x4{0, 0, 0, 0};
#pragma unroll
      for (int b = 0; b < MT; ++b) {
        if constexpr (SELF) {
          const int m = lane & 15;
          xf[u][b] = i32x4{0, 0, 0, 0};
          if (m < g.M && k < kp) xf[u][b] = *reinterpret_cast<const i32x4*>(s_q + m * kp + k);
        }
        acc[b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u], xf[u][b], acc[b], 0, 0, 0);
      }
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
      const I8Token token = i8_token(SELF ? s_scale[m < I8_SELF ? m : 0] : g.x_scale[m]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = n0 + 4 * (lane >> 4) + e;
        if (n < g.N) store1<OUT_BF16>(g.y, (size_t)m * g.ldy + n, i8_output(t[e], token, g.w_scale[n], i8_bias(g, n)));
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------
bool i8_self(int M, int K) { return M <= I8_SELF && K <= I8_SELF_K; }
constexpr int I8_FEW = 64;

long i8_pitch(int K) { return ((long)K + I8_ROW - 1) / I8_ROW * I8_ROW; }
size_t i8_scale_offset(long M, int K) { return ((size_t)M * i8_pitch(K) + 255) / 256 * 256; }

template <bool BF16, bool VEC>
void i8_launch_quant(const QuantArgs& a, long n, hipStream_t st) {
  const dim3 grid((unsigned)((n + 3) / 4)), block(256);
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
  // a launch may have fewer than 2^32 threads
  for (a.m0 = 0; a.m0 < M; a.m0 += 1L << 25) {
    const long n = M - a.m0 < (1L << 25) ? M - a.m0 : 1L << 25;
    if (dtype == VQAF_BF16) vec ? i8_launch_quant<true, true>(a, n, st) : i8_launch_quant<true, false>(a, n, st);
    else vec ? i8_launch_quant<false, true>(a, n, st) : i8_launch_quant<false, false>(a, n, st);
  }
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

template <bool YB, int TM, int TN, int WM, int WN, int STAGES, int OCC>
int i8_launch_tile(Int8Args& g, hipStream_t st) {
  constexpr int BM = 32 * TM * WM, BN = 32 * TN * WN, LDS = STAGES * (BM + BN) * I8_BK;
  const auto kernel = &int8_tile_kernel<YB, TM, TN, WM, WN, STAGES, OCC>;
  if constexpr (LDS > 65536) {
    // more dynamic LDS than 64 KB has to be asked for, once per kernel and device
    static std::mutex lock;
    static unsigned long long asked = 0;   // a bit for each of the first 64 devices
    int dev = 0;
    VQAF_REQUIRE(hipGetDevice(&dev) == hipSuccess && dev < 64, VQAF_E_LAUNCH);
    std::lock_guard<std::mutex> hold(lock);
    if (!(asked >> dev & 1ull)) {
      VQAF_REQUIRE(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                       LDS) == hipSuccess, VQAF_E_LAUNCH);
      asked |= 1ull << dev;
    }
  }
  g.tiles_m = (g.M + BM - 1) / BM;
  g.tiles_n = (g.N + BN - 1) / BN;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(g.tiles_m * g.tiles_n)), dim3(64 * WM * WN), LDS, st, g);
  return VQAF_OK;
}

template <bool YB>
int i8_launch_tiles(Int8Args& g, hipStream_t st) {
  // 256 x 256 tiles, one workgroup of eight waves per CU, once they nearly fill the chip (quantiser included, 12608 x 768 x
  // 2304: 450 tiles, 49 us against 52 on 128 x 128, and 8191 x 4096 x 4096 156 against 194; 2048 x 4096 x 4096: 128 tiles, 64
  // against 57 us); 128 x 128 tiles, two workgroups per CU, down to one for each CU (1920 x 768 x 2304: 270 tiles, 16.7 us
  // against 19.3 us on 64 x 64; 500 x 4096 x 1024: 32 tiles, 28 against 20 us); then 64 x 64 in a ring twice as deep, where
  // few workgroups have to hide the latency by themselves.  The channels that a tile lacks are not weighed: of 37000 tokens
  // of 768, 8 channels take 38 us on 256 x 256 against 32 on 64 x 64, 430 channels 80 against 68 on 128 x 128.
  const long t256 = (long)((g.M + 255) / 256) * ((g.N + 255) / 256), t128 = (long)((g.M + 127) / 128) * ((g.N + 127) / 128);
  if (t256 >= 144) return i8_launch_tile<YB, 4, 2, 2, 4, 4, 2>(g, st);
  if (t128 >= 256) return i8_launch_tile<YB, 2, 2, 2, 2, 4, 2>(g, st);
  return i8_launch_tile<YB, 1, 1, 2, 2, 8, 2>(g, st);
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
  VQAF_REQUIRE(N <= 1 << 27 && (long)((M + 63L) / 64) * ((N + 63) / 64) < 0x7fffffffL, VQAF_E_SHAPE);
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
    const int rc = yb ? i8_launch_tiles<true>(g, st) : i8_launch_tiles<false>(g, st);
    if (rc != VQAF_OK) return rc;
  }
  VQAF_LAUNCH_CHECK();
}
