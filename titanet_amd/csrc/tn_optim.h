// titanet_amd — device side of the optimizer step: element access, reductions, and the 8-bit form of the moments.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

#include "../../include/titanet_amd.h"

// The tensor that chunk `chunk` of a launch belongs to: end[] ascends, what is not used holds the largest number.  One load per
// lane and a vote instead of a search: the wave waits for one round trip to the launch's arguments.
__device__ __forceinline__ int opt_find(const uint32_t* end, int count, uint32_t chunk) {
  const int lane = threadIdx.x & 63;
  int t = 0;
  for (int lo = 0; lo < count; lo += 64) {
    const bool past = lo + lane < count && end[lo + lane] <= chunk;
    t += __popcll(__ballot(past));
  }
  return __builtin_amdgcn_readfirstlane(t);
}

// four consecutive elements from i on, as floats; those from n on are 0 / not written.  The type's own alignment is enough.
template <typename T>
struct OptVec {
  typedef T type __attribute__((ext_vector_type(4), aligned(sizeof(T))));
};
template <typename T>
__device__ __forceinline__ void opt_load4(const T* p, int64_t i, int64_t n, float v[4]) {
  if (i + 4 <= n) {
    const typename OptVec<T>::type x = *reinterpret_cast<const typename OptVec<T>::type*>(p + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (float)x[j];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = i + j < n ? (float)p[i + j] : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void opt_store4(T* p, int64_t i, int64_t n, const float v[4]) {
  if (i + 4 <= n) {
    typename OptVec<T>::type x;
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = (T)v[j];
    *reinterpret_cast<typename OptVec<T>::type*>(p + i) = x;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j < n) p[i + j] = (T)v[j];
  }
}

// sum over a workgroup of 256, the same order every time; thread 0 has the result
__device__ __forceinline__ double opt_sum_workgroup(double s) {
  __shared__ double part[4];
#pragma unroll
  for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  return threadIdx.x == 0 ? (part[0] + part[1]) + (part[2] + part[3]) : 0.0;
}

__device__ __forceinline__ float opt_max_wave(float x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x = fmaxf(x, __shfl_xor(x, d, 64));
  return x;
}

// ---- 8-bit moments -------------------------------------------------------------------------------------------------------
// A block of 256 elements shares a 32-bit scale; a code stands for
//   exp_avg     sign (c / 127)^2 M     M = the block's largest |exp_avg|
//   exp_avg_sq       (c / 255)^4 V     V = the block's largest exp_avg_sq
// The second moment enters the step through its square root, whose code is the square of an 8-bit fraction like the first's:
// both then resolve what is small against the block's largest, 1 / 127^2 and 1 / 255^2 of it, at a relative step of 2 / c.  A
// second moment above 0 never becomes 0 (c >= 1): it would leave its first moment divided by eps alone.
// The nearest code is decided in 64 bits (vector double arithmetic runs at the rate of single here, and the kernels wait for
// memory): the code of a value is then a matter of the definition, not of a kernel's rounding.  The candidate c comes from a
// single-precision root, at most one below; one comparison with the border (c + 1/2) settles it, half way goes to the lower.
// The largest value is worth its scale exactly (16129 * fl(1 / 16129) = 1, 255^4 likewise), and opt_ema rounds each product and
// the sum as written: with b1 = 9/10 one new scale in a hundred lies half way between two floats, where a fused
// multiply-add would turn it the other way than the same formula computed elsewhere.
// A block that holds a NaN or an infinity gets the scale NaN: all its values are NaN then, and stay so.
__device__ __forceinline__ void opt_decode_first(uint32_t q, float scale, double x[4]) {
  const double s = (double)scale;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = (int8_t)(q >> (8 * j));
    x[j] = ((double)(c < 0 ? -c * c : c * c) * (1.0 / 16129.0)) * s;
  }
}
__device__ __forceinline__ void opt_decode_second(uint32_t q, float scale, double x[4]) {
  const double s = (double)scale;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t c = (q >> (8 * j)) & 255u;
    x[j] = ((double)(c * c * c * c) * (1.0 / 4228250625.0)) * s;      // 255^4, below 2^32
  }
}
__device__ __forceinline__ double opt_ema(double b, double x, double w, double y) {
#pragma clang fp contract(off)
  const double p = b * x, q = w * y;
  return p + q;
}
// all 64 lanes of the wave call these, each with four of the block's 256 values; *scale is that of the block, infinity or NaN
// if one of its values is
__device__ __forceinline__ float opt_scale_wave(const double x[4]) {
  float top = 0.f;
  bool bad = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = fabsf((float)x[j]);
    bad |= !(a < __builtin_huge_valf());
    top = fmaxf(top, a);
  }
  top = opt_max_wave(top);
  return __ballot(bad) ? __builtin_nanf("") : top;
}
__device__ __forceinline__ uint32_t opt_encode_first(const double x[4], float* scale) {
  const float top = opt_scale_wave(x);
  *scale = top;
  if (!(top > 0.f)) return 0u;
  const double inv = __builtin_amdgcn_rcp((double)top), border = (double)top * (1.0 / 64516.0);       // (2 * 127)^2
  uint32_t q = 0u;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const double a = fabs(x[j]);
    int c = (int)(127.f * __builtin_amdgcn_sqrtf((float)(a * inv)));
    c = c < 126 ? c : 126;
    c += a > (double)((2 * c + 1) * (2 * c + 1)) * border;
    q |= (uint32_t)(uint8_t)(int8_t)(x[j] < 0.0 ? -c : c) << (8 * j);
  }
  return q;
}
__device__ __forceinline__ uint32_t opt_encode_second(const double x[4], float* scale) {
  const float top = opt_scale_wave(x);
  *scale = top;
  if (!(top > 0.f)) return 0u;
  const double inv = __builtin_amdgcn_rcp((double)top), border = (double)top * (1.0 / 67652010000.0);     // (2 * 255)^4
  uint32_t q = 0u;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    int c = (int)(255.f * __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf((float)(x[j] * inv))));
    c = c < 254 ? c : 254;
    const double r = (double)((2 * c + 1) * (2 * c + 1));
    c += x[j] > r * r * border;
    c = x[j] > 0.0 && c == 0 ? 1 : c;
    q |= (uint32_t)c << (8 * j);
  }
  return q;
}
