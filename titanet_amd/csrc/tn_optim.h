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

// four consecutive elements from i on, as floats; those from n on are 0 / not written (WHOLE: none are).  The type's own alignment is enough.
template <typename T>
struct OptVec {
  typedef T type __attribute__((ext_vector_type(4), aligned(sizeof(T))));
};
// ONCE: nothing reads these lines again before the next step, they need not stay in a cache.
template <bool WHOLE = false, bool ONCE = false, typename T>
__device__ __forceinline__ void opt_load4(const T* p, int64_t i, int64_t n, float v[4]) {
  if (WHOLE || i + 4 <= n) {
    const typename OptVec<T>::type* at = reinterpret_cast<const typename OptVec<T>::type*>(p + i);
    const typename OptVec<T>::type x = ONCE ? __builtin_nontemporal_load(at) : *at;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (float)x[j];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = i + j < n ? (float)p[i + j] : 0.f;
  }
}
template <bool WHOLE = false, bool ONCE = false, typename T>
__device__ __forceinline__ void opt_store4(T* p, int64_t i, int64_t n, const float v[4]) {
  if (WHOLE || i + 4 <= n) {
    typename OptVec<T>::type x;
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = (T)v[j];
    typename OptVec<T>::type* at = reinterpret_cast<typename OptVec<T>::type*>(p + i);
    if constexpr (ONCE) __builtin_nontemporal_store(x, at);
    else *at = x;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j < n) p[i + j] = (T)v[j];
  }
}

// sum over a workgroup of WAVES waves, the same order every time; thread 0 has the result
template <int WAVES>
__device__ __forceinline__ double opt_sum_workgroup(double s) {
  __shared__ double part[WAVES];
#pragma unroll
  for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  double sum = 0.0;
  if (threadIdx.x == 0)
#pragma unroll
    for (int w = 0; w < WAVES; ++w) sum += part[w];
  return sum;
}

// largest of 64 lanes' numbers, the same in all lanes (a scalar)
__device__ __forceinline__ uint32_t opt_max_wave(uint32_t x) {
  auto up = [&](uint32_t y) { x = x > y ? x : y; };
  up(__builtin_amdgcn_update_dpp(0, x, 0xb1, 0xf, 0xf, false));       // lane ^ 1
  up(__builtin_amdgcn_update_dpp(0, x, 0x4e, 0xf, 0xf, false));       // lane ^ 2
  up(__builtin_amdgcn_update_dpp(0, x, 0x141, 0xf, 0xf, false));      // mirrored within 8
  up(__builtin_amdgcn_update_dpp(0, x, 0x140, 0xf, 0xf, false));      // mirrored within 16
  up(__builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));      // lane 15 of rows 0, 2 to rows 1, 3
  up(__builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));      // lane 31 to rows 2, 3: lane 63 has them all
  return __builtin_amdgcn_readlane(x, 63);
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
    const float c = (float)(int8_t)(q >> (8 * j));
    x[j] = ((double)(c * fabsf(c)) * (1.0 / 16129.0)) * s;             // 127^2
  }
}
__device__ __forceinline__ void opt_decode_second(uint32_t q, float scale, double x[4]) {
  const double s = (double)scale;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float c = (float)((q >> (8 * j)) & 255u);
    const double r = (double)(c * c);
    x[j] = ((r * r) * (1.0 / 4228250625.0)) * s;                       // 255^4
  }
}
__device__ __forceinline__ double opt_ema(double b, double x, double w, double y) {
#pragma clang fp contract(off)
  const double p = b * x, q = w * y;
  return p + q;
}
// All 64 lanes of the wave call these, each with four of the block's 256 values and the same rounded to 32 bits.  *scale becomes
// the block's; the bit pattern of a NaN or an infinity is above every finite one's, so the maximum finds them by itself.
__device__ __forceinline__ float opt_scale_wave(const float f[4]) {
  uint32_t top = 0u;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t b = __float_as_uint(f[j]) & 0x7fffffffu;
    top = top > b ? top : b;
  }
  top = opt_max_wave(top);
  return top < 0x7f800000u ? __uint_as_float(top) : __builtin_nanf("");
}
// x / scale to float accuracy, for candidates; a scale whose reciprocal a float cannot hold goes through 64 bits: below 2^-100, and from
// 2^125 on, since the hardware's reciprocal has no denormal results (1 / 2^127 is 0, and every code of the block would be 1 at most)
__device__ __forceinline__ void opt_ratio(const double x[4], const float f[4], float scale, float r[4]) {
  if (scale > 0x1p-100f && scale < 0x1p125f) {             // (uniform over the wave)
    const float inv = __builtin_amdgcn_rcpf(scale);
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = fabsf(f[j]) * inv;
  } else {
    const double inv = __builtin_amdgcn_rcp((double)scale);
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = (float)(fabs(x[j]) * inv);
  }
}
__device__ __forceinline__ uint32_t opt_encode_first(const double x[4], const float f[4], float* scale) {
  const float top = opt_scale_wave(f);
  *scale = top;
  if (!(top > 0.f)) return 0u;
  float ratio[4];
  opt_ratio(x, f, top, ratio);
  const double border = (double)top * (1.0 / 64516.0);                 // (2 * 127)^2
  uint32_t q = 0u;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float c = fminf(floorf(127.f * __builtin_amdgcn_sqrtf(ratio[j])), 126.f);
    const float e = fmaf(2.f, c, 1.f);
    c += fabs(x[j]) > (double)(e * e) * border ? 1.f : 0.f;
    q = __builtin_amdgcn_cvt_pk_u8_f32(c, j, q);
  }
  // negative values: two's complement of their byte, 0x80 - c with the top bit turned
  const uint32_t neg = (0x80808080u - q) ^ 0x80808080u;
  const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(f[1]), __float_as_uint(f[0]), 0x0c0c0b09u);      // 9, 11: a byte of sign bits
  const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(f[3]), __float_as_uint(f[2]), 0x0b090c0cu);
  const uint32_t mask = lo | hi;
  return (neg & mask) | (q & ~mask);
}
__device__ __forceinline__ uint32_t opt_encode_second(const double x[4], const float f[4], float* scale) {
  const float top = opt_scale_wave(f);
  *scale = top;
  if (!(top > 0.f)) return 0u;
  float ratio[4];
  opt_ratio(x, f, top, ratio);
  const double border = (double)top * (1.0 / 67652010000.0);           // (2 * 255)^4
  uint32_t q = 0u;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float c = fminf(floorf(255.f * __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(ratio[j]))), 254.f);
    const float e = fmaf(2.f, c, 1.f);
    const double r = (double)(e * e);
    c += x[j] > (r * r) * border ? 1.f : 0.f;
    c = fmaxf(c, x[j] > 0.0 ? 1.f : 0.f);
    q = __builtin_amdgcn_cvt_pk_u8_f32(c, j, q);
  }
  return q;
}

// m / (sqrt(v) root + eps) with the hardware's root and reciprocal (one step of 32 bits each) where they hold; a root of a denormal
// or a denominator of nothing goes the exact way
__device__ __forceinline__ float opt_update(float m, float v, float root, float eps) {
  const float d = fmaf(__builtin_amdgcn_sqrtf(v), root, eps);
  if (d > 1e-18f && d < 1e18f) return m * __builtin_amdgcn_rcpf(d);
  return m / (sqrtf(v) * root + eps);
}

struct OptStep {                       // what a step of one tensor needs besides its values
  double b1, b2, w1, w2, factor;       // w = 1 - b
  float rate, root, decay, eps;        // lr / (1 - b1^t), 1 / sqrt(1 - b2^t), 1 - lr wd
};

// One block of 256 elements, four to a lane, from element i0 of a tensor of n on
template <bool WHOLE, typename T>
__device__ __forceinline__ void opt_step8_block(const OptStep& h, T* p, const float g[4], int64_t i0, int64_t n, int64_t block, int8_t* exp_avg,
                                                uint8_t* exp_avg_sq, float* scale1, float* scale2) {
  const int lane = threadIdx.x & 63;
  const int64_t i = i0 + 4 * lane;
  float pv[4];
  opt_load4<WHOLE>(p, i, n, pv);
  uint32_t* q1 = reinterpret_cast<uint32_t*>(exp_avg + block * TN_OPT_BLOCK) + lane;
  uint32_t* q2 = reinterpret_cast<uint32_t*>(exp_avg_sq + block * TN_OPT_BLOCK) + lane;
  double m[4], v[4];
  float mf[4], vf[4];
  opt_decode_first(__builtin_nontemporal_load(q1), scale1[block], m);
  opt_decode_second(__builtin_nontemporal_load(q2), scale2[block], v);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const double gj = (double)g[j] * h.factor;
    m[j] = opt_ema(h.b1, m[j], h.w1, gj);
    v[j] = opt_ema(h.b2, v[j], h.w2, gj * gj);
    mf[j] = (float)m[j];
    vf[j] = (float)v[j];
    pv[j] = pv[j] * h.decay - h.rate * opt_update(mf[j], vf[j], h.root, h.eps);
  }
  opt_store4<WHOLE>(p, i, n, pv);
  float s1, s2;
  const uint32_t n1 = opt_encode_first(m, mf, &s1), n2 = opt_encode_second(v, vf, &s2);
  const bool bad = !(s1 < __builtin_huge_valf()) || !(s2 < __builtin_huge_valf());
  __builtin_nontemporal_store(bad ? 0u : n1, q1);
  __builtin_nontemporal_store(bad ? 0u : n2, q2);
  if (lane == 0) {
    scale1[block] = bad ? __builtin_nanf("") : s1;
    scale2[block] = bad ? __builtin_nanf("") : s2;
  }
}
template <bool WHOLE, typename T>
__device__ __forceinline__ void opt_step32(const OptStep& h, T* p, const float g[4], int64_t i, int64_t n, float* m, float* v) {
  const float b1 = (float)h.b1, b2 = (float)h.b2, w1 = (float)h.w1, w2 = (float)h.w2, factor = (float)h.factor;
  float pv[4], mv[4], vv[4], gf[4];
  opt_load4<WHOLE>(p, i, n, pv);
  opt_load4<WHOLE, true>(m, i, n, mv);              // (the padding of the last block is neither read nor written)
  opt_load4<WHOLE, true>(v, i, n, vv);
  if (fabsf(factor) < 0x1p-126f) {                  // (uniform; a clipping factor that 32 bits cannot hold to their precision)
#pragma unroll
    for (int j = 0; j < 4; ++j) gf[j] = (float)((double)g[j] * h.factor);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) gf[j] = g[j] * factor;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float gj = gf[j];
    mv[j] = b1 * mv[j] + w1 * gj;
    vv[j] = b2 * vv[j] + w2 * (gj * gj);
    pv[j] = pv[j] * h.decay - h.rate * opt_update(mv[j], vv[j], h.root, h.eps);
  }
  opt_store4<WHOLE>(p, i, n, pv);
  opt_store4<WHOLE, true>(m, i, n, mv);
  opt_store4<WHOLE, true>(v, i, n, vv);
}
