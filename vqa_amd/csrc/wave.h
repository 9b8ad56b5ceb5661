// Reductions over a wave of 64 lanes.
#pragma once
#include <hip/hip_runtime.h>

namespace {

// ---------------------------------------------------------------------------------------------
// Wave reductions through DPP (six vector instructions instead of six trips through the LDS crossbar); the order is
// fixed and the result is in every lane (read from lane 63).
// ---------------------------------------------------------------------------------------------
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned dpp_move(unsigned idle, unsigned x) {
  return (unsigned)__builtin_amdgcn_update_dpp((int)idle, (int)x, CTRL, ROWS, 0xf, false);
}
template <class F>
__device__ __forceinline__ unsigned dpp_wave_u32(unsigned x, unsigned idle, F f) {
  x = f(x, dpp_move<0x111, 0xf>(idle, x));
  x = f(x, dpp_move<0x112, 0xf>(idle, x));
  x = f(x, dpp_move<0x114, 0xf>(idle, x));
  x = f(x, dpp_move<0x118, 0xf>(idle, x));
  x = f(x, dpp_move<0x142, 0xa>(idle, x));
  x = f(x, dpp_move<0x143, 0xc>(idle, x));
  return (unsigned)__builtin_amdgcn_readlane((int)x, 63);
}
__device__ __forceinline__ float dpp_wave_max(float v) {
  return __uint_as_float(dpp_wave_u32(__float_as_uint(v), 0xff800000u, [](unsigned a, unsigned b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}
__device__ __forceinline__ float dpp_wave_sum(float v) {
  return __uint_as_float(dpp_wave_u32(__float_as_uint(v), 0u, [](unsigned a, unsigned b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}
__device__ __forceinline__ unsigned dpp_wave_umax(unsigned v) {
  return dpp_wave_u32(v, 0u, [](unsigned a, unsigned b) { return a > b ? a : b; });
}
__device__ __forceinline__ unsigned dpp_wave_umin(unsigned v) {
  return dpp_wave_u32(v, 0xffffffffu, [](unsigned a, unsigned b) { return a < b ? a : b; });
}
__device__ __forceinline__ unsigned dpp_wave_uadd(unsigned v) {
  return dpp_wave_u32(v, 0u, [](unsigned a, unsigned b) { return a + b; });
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double x) {
  const unsigned long long u = __builtin_bit_cast(unsigned long long, x);
  const unsigned long long o = ((unsigned long long)dpp_move<CTRL, ROWS>(0u, (unsigned)(u >> 32)) << 32) | dpp_move<CTRL, ROWS>(0u, (unsigned)u);
  return x + __builtin_bit_cast(double, o);   // idle lanes contribute +0
}
__device__ __forceinline__ double dpp_wave_sum(double x) {
  x = dpp_add<0x111, 0xf>(x);
  x = dpp_add<0x112, 0xf>(x);
  x = dpp_add<0x114, 0xf>(x);
  x = dpp_add<0x118, 0xf>(x);
  x = dpp_add<0x142, 0xa>(x);
  x = dpp_add<0x143, 0xc>(x);
  const unsigned long long u = __builtin_bit_cast(unsigned long long, x);
  const unsigned long long r = ((unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(u >> 32), 63) << 32) |
                (unsigned)__builtin_amdgcn_readlane((int)(unsigned)u, 63);
  return __builtin_bit_cast(double, r);
}

// ---------------------------------------------------------------------------------------------
// The same over each row of sixteen lanes: four rotations, the result in every lane of the row.
// ---------------------------------------------------------------------------------------------
template <class F>
__device__ __forceinline__ unsigned dpp_row_u32(unsigned x, F f) {
  x = f(x, dpp_move<0x121, 0xf>(x, x));
  x = f(x, dpp_move<0x122, 0xf>(x, x));
  x = f(x, dpp_move<0x124, 0xf>(x, x));
  x = f(x, dpp_move<0x128, 0xf>(x, x));
  return x;
}
__device__ __forceinline__ float dpp_row_max(float v) {
  return __uint_as_float(dpp_row_u32(__float_as_uint(v), [](unsigned a, unsigned b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}
__device__ __forceinline__ float dpp_row_sum(float v) {
  return __uint_as_float(dpp_row_u32(__float_as_uint(v), [](unsigned a, unsigned b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}
__device__ __forceinline__ unsigned dpp_row_umax(unsigned v) {
  return dpp_row_u32(v, [](unsigned a, unsigned b) { return a > b ? a : b; });
}
__device__ __forceinline__ double dpp_row_sum(double x) {
  x = dpp_add<0x121, 0xf>(x);
  x = dpp_add<0x122, 0xf>(x);
  x = dpp_add<0x124, 0xf>(x);
  x = dpp_add<0x128, 0xf>(x);
  return x;
}

}  // namespace
