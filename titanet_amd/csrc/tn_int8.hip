// titanet_amd — matrix product in 8-bit integers with a scale for each row of both operands (token x channel).
//
//   y[m][n] = sa[m] sb[n] sum_k qa[m][k] qb[n][k] (+ bias[n])          the sum exact in 32 bits (K <= 131071)
//   q = x / s rounded to the nearest integer (even half way),  s = max(max |row| / 127, 2^-126), 0 for a row of zeros
//
// Layout: a row of codes takes a multiple of 64 bytes, what lies behind its K codes is 0 (and adds nothing to the sum), so that
// every fragment is a whole 16-byte load.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "../../include/titanet_amd.h"

namespace {

typedef __attribute__((ext_vector_type(4))) int i32x4_t;
typedef __attribute__((ext_vector_type(16))) int i32x16_t;

// nearest integer to x / s, even half way: the quotient's own rounding could move it across a border, the sign of the remainder
// against the border (one fused multiply-add, whose sign is exact) cannot
__device__ __forceinline__ int q8_code(float x, float s, float inv) {
  const float a = fabsf(x);
  float c = floorf(a * inv);
  c = fminf(c, 127.f);
  // the candidate is within one of the quotient: settle it between c - 1, c, c + 1
  c -= fmaf(-(c - 0.5f), s, a) < 0.f ? 1.f : 0.f;
  const float r = fmaf(-(c + 0.5f), s, a);
  const int k = (int)c;
  const int up = k + (r > 0.f || (r == 0.f && (k & 1)) ? 1 : 0);
  return x < 0.f ? -up : up;
}

__device__ __forceinline__ float q8_scale(float top) { return top > 0.f ? fmaxf(top / 127.f, 0x1p-126f) : 0.f; }

// one wave per row: maximum, then codes
template <typename T>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* __restrict__ x, int64_t rows, int cols, int64_t ldx, int8_t* __restrict__ q,
                                                            int64_t ldq, float* __restrict__ scales) {
  const int lane = threadIdx.x & 63;
  for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += (int64_t)gridDim.x * 4) {
    const T* row = x + r * ldx;
    float top = 0.f;
    bool bad = false;
    for (int k = lane; k < cols; k += 64) {
      const float a = fabsf((float)row[k]);
      bad |= !(a < __builtin_huge_valf());
      top = fmaxf(top, a);
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
    bad = __ballot(bad) != 0;
    const float s = q8_scale(top), inv = s > 0.f ? 1.f / s : 0.f;
    for (int64_t k = lane; k < ldq; k += 64) q[r * ldq + k] = !bad && s > 0.f && k < cols ? (int8_t)q8_code((float)row[k], s, inv) : (int8_t)0;
    if (lane == 0) scales[r] = bad ? __builtin_nanf("") : s;
  }
}

struct Int8Args {
  const int8_t *a, *b;
  const float *sa, *sb, *bias;
  void* y;
  int64_t lda, ldb, ldy, m, n;
  int k;                              // multiple of 64
};

// 128 x 128 outputs per workgroup, 64 x 64 per wave (2 x 2 matrix instructions of 32 x 32 x 32), K in steps of 64 bytes through LDS
template <typename T>
__global__ __launch_bounds__(256) void int8_matmul_kernel(Int8Args g, int tiles_n) {
  __shared__ __attribute__((aligned(16))) int8_t ta[128 * 80], tb[128 * 80];       // rows of 64 bytes, padded to 80
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1;
  const int64_t m0 = (int64_t)(blockIdx.x / tiles_n) * 128, n0 = (int64_t)(blockIdx.x % tiles_n) * 128;
  i32x16_t acc[2][2] = {};
  const int row = tid >> 1, part = (tid & 1) * 32;
  const int64_t ra = std::min<int64_t>(m0 + row, g.m - 1), rb = std::min<int64_t>(n0 + row, g.n - 1);
  const int8_t *pa = g.a + ra * g.lda + part, *pb = g.b + rb * g.ldb + part;
  const int fi = lane & 31, fh = lane >> 5;
  for (int k = 0; k < g.k; k += 64) {
    const i32x4_t a0 = *reinterpret_cast<const i32x4_t*>(pa + k), a1 = *reinterpret_cast<const i32x4_t*>(pa + k + 16);
    const i32x4_t b0 = *reinterpret_cast<const i32x4_t*>(pb + k), b1 = *reinterpret_cast<const i32x4_t*>(pb + k + 16);
    __syncthreads();
    *reinterpret_cast<i32x4_t*>(ta + row * 80 + part) = a0;
    *reinterpret_cast<i32x4_t*>(ta + row * 80 + part + 16) = a1;
    *reinterpret_cast<i32x4_t*>(tb + row * 80 + part) = b0;
    *reinterpret_cast<i32x4_t*>(tb + row * 80 + part + 16) = b1;
    __syncthreads();
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      i32x4_t af[2], bf[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        af[i] = *reinterpret_cast<const i32x4_t*>(ta + (wm * 64 + i * 32 + fi) * 80 + ks * 32 + fh * 16);
        bf[i] = *reinterpret_cast<const i32x4_t*>(tb + (wn * 64 + i * 32 + fi) * 80 + ks * 32 + fh * 16);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(af[i], bf[j], acc[i][j], 0, 0, 0);
    }
  }
  T* y = reinterpret_cast<T*>(g.y);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t col = n0 + wn * 64 + j * 32 + fi;
    const bool in = col < g.n;
    const float sb = in ? g.sb[col] : 0.f, bias = in && g.bias ? g.bias[col] : 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int64_t rw = m0 + wm * 64 + i * 32 + (r & 3) + 8 * (r >> 2) + 4 * fh;
        if (in && rw < g.m) y[rw * g.ldy + col] = (T)((float)acc[i][j][r] * g.sa[rw] * sb + bias);
      }
  }
}

template <typename F>
int q8_by_type(int dtype, F f) {
  if (dtype == TN_DTYPE_F32) return f((float*)nullptr);
  if (dtype == TN_DTYPE_BF16) return f((__bf16*)nullptr);
  if (dtype == TN_DTYPE_F16) return f((_Float16*)nullptr);
  return TN_E_UNSUPPORTED;
}

constexpr int64_t Q8_GRID = (1 << 24) - 1;

}  // namespace

extern "C" int tn_int8_quantize_rows(const void* x, int32_t dtype, int64_t rows, int64_t cols, int64_t ldx, void* codes, int64_t ld_codes,
                                     float* scales, void* stream) {
  if (rows < 0 || cols < 1 || ldx < 0 || ld_codes % 64 || ld_codes < cols || (rows > 0 && (!x || !codes || !scales))) return TN_E_BADARG;
  if (cols > TN_INT8_MAX_K || dtype < TN_DTYPE_F32 || dtype > TN_DTYPE_F16) return TN_E_UNSUPPORTED;
  if (!rows) return 0;
  return q8_by_type(dtype, [&](auto* kind) -> int {
    using T = std::remove_pointer_t<decltype(kind)>;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(quantize_rows_kernel<T>), dim3((unsigned)std::min<int64_t>((rows + 3) / 4, 1 << 20)), dim3(256), 0,
                       (hipStream_t)stream, (const T*)x, rows, (int)cols, ldx, (int8_t*)codes, ld_codes, scales);
    return (int)hipGetLastError();
  });
}

extern "C" int tn_int8_matmul(const void* a, const float* a_scales, int64_t lda, const void* b, const float* b_scales, int64_t ldb,
                              const float* bias, void* y, int32_t y_dtype, int64_t ldy, int64_t m, int64_t n, int64_t k, void* stream) {
  if (m < 0 || n < 0 || k < 1 || lda % 64 || ldb % 64 || lda < k || ldb < k || ldy < n) return TN_E_BADARG;
  if (m > 0 && n > 0 && (!a || !a_scales || !b || !b_scales || !y || ((uintptr_t)a | (uintptr_t)b) % 16)) return TN_E_BADARG;
  if (k > TN_INT8_MAX_K || y_dtype < TN_DTYPE_F32 || y_dtype > TN_DTYPE_F16) return TN_E_UNSUPPORTED;
  if (!m || !n) return 0;
  const int64_t tm = (m + 127) / 128, tn = (n + 127) / 128;
  if (tn > Q8_GRID || tm > Q8_GRID / tn) return TN_E_UNSUPPORTED;
  const Int8Args g = {(const int8_t*)a, (const int8_t*)b, a_scales, b_scales, bias, y, lda, ldb, ldy, m, n, (int)((k + 63) / 64 * 64)};
  return q8_by_type(y_dtype, [&](auto* kind) -> int {
    using T = std::remove_pointer_t<decltype(kind)>;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(int8_matmul_kernel<T>), dim3((unsigned)(tm * tn)), dim3(256), 0, (hipStream_t)stream, g, (int)tn);
    return (int)hipGetLastError();
  });
}
