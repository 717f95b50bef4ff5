// titanet_amd — AdamW over many tensors at once, its moments held in 32 bits or as 8-bit codes, and the global gradient norm.
//
//   m' = b1 m + (1 - b1) g        v' = b2 v + (1 - b2) g^2        (g: the gradient times the clipping factor)
//   p' = p (1 - lr wd) - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// Layout: the moments of all tensors lie in one buffer, every tensor beginning at a multiple of TN_OPT_BLOCK = 256 elements;
// parameters and gradients stay where the caller has them (any alignment their type has).  The step count t, the learning rate
// and the clipping factor are read from device memory, so that a captured step replays with the values of its time.
#include "tn_optim.h"

#include <algorithm>
#include <cmath>

namespace {

constexpr int OPT_CHUNK = 4096;        // elements of one workgroup of the step: 16 blocks of 256
constexpr int SUM_CHUNK = 16384;       // elements behind one partial sum of the norm
constexpr int OPT_LIST = 96;           // tensors one launch can name in its arguments
constexpr int64_t OPT_GRID = (1 << 24) - 1;      // workgroups of 256 in one launch: the grid is counted in 32 bits of threads

// ------------------------------------------------------------------------------------------------- global gradient norm
struct SumList {
  const void* g[OPT_LIST];
  int64_t numel[OPT_LIST];
  uint32_t end[OPT_LIST];              // chunks of this launch before the end of tensor i (ascending)
};

// One partial sum of squares per chunk of SUM_CHUNK elements, in 64 bits (no gradient of a 32-bit type overflows there, and the
// order of the sum is fixed: two runs give the same norm).
template <typename T>
__global__ __launch_bounds__(256) void grad_sumsq_kernel(SumList list, double* __restrict__ partials) {
  const int t = opt_find(list.end, OPT_LIST, blockIdx.x);
  const uint32_t before = t ? list.end[t - 1] : 0u;
  const int64_t lo = (int64_t)(blockIdx.x - before) * SUM_CHUNK, n = list.numel[t];
  const T* g = reinterpret_cast<const T*>(list.g[t]);
  double s = 0.0;
  for (int64_t i = lo + 4 * threadIdx.x; i < lo + SUM_CHUNK && i < n; i += 4 * 256) {
    float v[4];
    opt_load4(g, i, n, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) s = fma((double)v[j], (double)v[j], s);
  }
  s = opt_sum_workgroup(s);
  if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

// norm = |mult| sqrt(sum), ctl = {factor of the gradients, 1 if the step runs}: a norm that is no number stops the step
__global__ __launch_bounds__(256) void grad_norm_finish_kernel(const double* __restrict__ partials, int64_t count, double mult,
                                                               double max_norm, float* __restrict__ norm_out, double* __restrict__ ctl) {
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < count; i += 256) s += partials[i];
  s = opt_sum_workgroup(s);
  if (threadIdx.x == 0) {
    const double norm = sqrt(s) * fabs(mult);
    if (norm_out) *norm_out = (float)norm;
    if (ctl) {
      const bool ok = norm < __builtin_huge_val();      // false for NaN too
      const double c = max_norm / (norm + 1e-6);
      ctl[0] = ok ? mult * (c < 1.0 ? c : 1.0) : 0.0;
      ctl[1] = ok ? 1.0 : 0.0;
    }
  }
}

// -------------------------------------------------------------------------------------------------------------- the step
struct OptSlots {
  int32_t slot[256];
  int32_t count;
};

__device__ double opt_power(double b, int32_t t) {       // b^t by squaring: exact enough for 1 - b^t at every t
  double r = 1.0;
  while (t > 0) {
    if (t & 1) r *= b;
    b *= b;
    t >>= 1;
  }
  return r;
}

// steps[slot] += 1 and the four numbers of the step that depend on it: {step size, 1 / sqrt(1 - b2^t), 1 - lr wd, runs}
__global__ __launch_bounds__(256) void adamw_tick_kernel(OptSlots list, int32_t* __restrict__ steps, float* __restrict__ corr,
                                                         const double* __restrict__ ctl, double lr, const float* __restrict__ lr_dev,
                                                         double b1, double b2, double wd) {
  const int i = threadIdx.x;
  if (i >= list.count) return;
  const int s = list.slot[i];
  float* c = corr + 4 * (int64_t)s;
  if (ctl && ctl[1] == 0.0) {
    c[3] = 0.f;
    return;
  }
  const int32_t t = steps[s] + 1;
  steps[s] = t;
  if (lr_dev) lr = (double)*lr_dev;
  c[0] = (float)(lr / (1.0 - opt_power(b1, t)));
  c[1] = (float)(1.0 / sqrt(1.0 - opt_power(b2, t)));
  c[2] = (float)(1.0 - lr * wd);
  c[3] = 1.f;
}

struct OptList {
  void* p[OPT_LIST];
  const void* g[OPT_LIST];
  int64_t numel[OPT_LIST];
  uint32_t end[OPT_LIST];
  uint32_t first_block[OPT_LIST];
  uint32_t slot[OPT_LIST];
};

struct OptHyper {
  double b1, b2, w1, w2;               // w = 1 - b
  float eps;
  double mult;                         // factor of the gradients where ctl is null
};

template <typename T>
__global__ __launch_bounds__(256) void adamw32_kernel(OptList list, OptHyper h, float* __restrict__ exp_avg, float* __restrict__ exp_avg_sq,
                                                      const float* __restrict__ corr, const double* __restrict__ ctl) {
  const int t = opt_find(list.end, OPT_LIST, blockIdx.x);
  const float4 c = *reinterpret_cast<const float4*>(corr + 4 * (int64_t)list.slot[t]);
  if (c.w == 0.f) return;
  const float factor = (float)(ctl ? ctl[0] : h.mult);
  const float b1 = (float)h.b1, b2 = (float)h.b2, w1 = (float)h.w1, w2 = (float)h.w2;
  const uint32_t before = t ? list.end[t - 1] : 0u;
  const int64_t lo = (int64_t)(blockIdx.x - before) * OPT_CHUNK, n = list.numel[t];
  T* p = reinterpret_cast<T*>(list.p[t]);
  const T* g = reinterpret_cast<const T*>(list.g[t]);
  float* m = exp_avg + (int64_t)list.first_block[t] * TN_OPT_BLOCK;
  float* v = exp_avg_sq + (int64_t)list.first_block[t] * TN_OPT_BLOCK;
  for (int64_t i = lo + 4 * threadIdx.x; i < lo + OPT_CHUNK && i < n; i += 4 * 256) {
    float pv[4], gv[4], mv[4], vv[4];
    opt_load4(p, i, n, pv);
    opt_load4(g, i, n, gv);
    opt_load4(m, i, n, mv);            // (the padding of the last block is read and written as zeros)
    opt_load4(v, i, n, vv);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float gj = gv[j] * factor;
      mv[j] = b1 * mv[j] + w1 * gj;
      vv[j] = b2 * vv[j] + w2 * (gj * gj);
      pv[j] = pv[j] * c.z - c.x * (mv[j] / (sqrtf(vv[j]) * c.y + h.eps));
    }
    opt_store4(p, i, n, pv);
    opt_store4(m, i, n, mv);
    opt_store4(v, i, n, vv);
  }
}

// 8-bit moments: one wave holds one block of 256 elements, four to a lane, so that the block's maxima are a reduction over the
// wave and neither LDS nor a barrier is needed.
template <typename T>
__global__ __launch_bounds__(256) void adamw8_kernel(OptList list, OptHyper h, int8_t* __restrict__ exp_avg, uint8_t* __restrict__ exp_avg_sq,
                                                     float* __restrict__ scale1, float* __restrict__ scale2,
                                                     const float* __restrict__ corr, const double* __restrict__ ctl) {
  const int t = opt_find(list.end, OPT_LIST, blockIdx.x);
  const float4 c = *reinterpret_cast<const float4*>(corr + 4 * (int64_t)list.slot[t]);
  if (c.w == 0.f) return;
  const double factor = ctl ? ctl[0] : h.mult;
  const uint32_t before = t ? list.end[t - 1] : 0u;
  const int64_t lo = (int64_t)(blockIdx.x - before) * OPT_CHUNK, n = list.numel[t];
  T* p = reinterpret_cast<T*>(list.p[t]);
  const T* g = reinterpret_cast<const T*>(list.g[t]);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int k = wave; k < OPT_CHUNK / TN_OPT_BLOCK; k += 4) {
    const int64_t i0 = lo + (int64_t)k * TN_OPT_BLOCK, i = i0 + 4 * lane;
    if (i0 >= n) break;
    const int64_t block = (int64_t)list.first_block[t] + i0 / TN_OPT_BLOCK;
    float pv[4], gv[4];
    opt_load4(p, i, n, pv);
    opt_load4(g, i, n, gv);
    uint32_t* q1 = reinterpret_cast<uint32_t*>(exp_avg + block * TN_OPT_BLOCK) + lane;
    uint32_t* q2 = reinterpret_cast<uint32_t*>(exp_avg_sq + block * TN_OPT_BLOCK) + lane;
    double m[4], v[4];
    opt_decode_first(*q1, scale1[block], m);
    opt_decode_second(*q2, scale2[block], v);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double gj = (double)gv[j] * factor;
      m[j] = opt_ema(h.b1, m[j], h.w1, gj);
      v[j] = opt_ema(h.b2, v[j], h.w2, gj * gj);
      pv[j] = pv[j] * c.z - c.x * ((float)m[j] / (sqrtf((float)v[j]) * c.y + h.eps));
    }
    opt_store4(p, i, n, pv);
    float s1, s2;
    const uint32_t n1 = opt_encode_first(m, &s1), n2 = opt_encode_second(v, &s2);
    const bool bad = !(s1 < __builtin_huge_valf()) || !(s2 < __builtin_huge_valf());
    *q1 = n1;
    *q2 = n2;
    if (lane == 0) {
      scale1[block] = bad ? __builtin_nanf("") : s1;
      scale2[block] = bad ? __builtin_nanf("") : s2;
    }
  }
}

__global__ __launch_bounds__(256) void moments_decode_kernel(const int8_t* __restrict__ q1, const uint8_t* __restrict__ q2,
                                                             const float* __restrict__ scale1, const float* __restrict__ scale2,
                                                             float* __restrict__ m, float* __restrict__ v, int64_t blocks) {
  const int lane = threadIdx.x & 63;
  for (int64_t b = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); b < blocks; b += (int64_t)gridDim.x * 4) {
  double x[4];
  opt_decode_first(reinterpret_cast<const uint32_t*>(q1 + b * TN_OPT_BLOCK)[lane], scale1[b], x);
  reinterpret_cast<float4*>(m + b * TN_OPT_BLOCK)[lane] = make_float4((float)x[0], (float)x[1], (float)x[2], (float)x[3]);
  opt_decode_second(reinterpret_cast<const uint32_t*>(q2 + b * TN_OPT_BLOCK)[lane], scale2[b], x);
  reinterpret_cast<float4*>(v + b * TN_OPT_BLOCK)[lane] = make_float4((float)x[0], (float)x[1], (float)x[2], (float)x[3]);
  }
}

__global__ __launch_bounds__(256) void moments_encode_kernel(const float* __restrict__ m, const float* __restrict__ v, int8_t* __restrict__ q1,
                                                             uint8_t* __restrict__ q2, float* __restrict__ scale1,
                                                             float* __restrict__ scale2, int64_t blocks) {
  const int lane = threadIdx.x & 63;
  for (int64_t b = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); b < blocks; b += (int64_t)gridDim.x * 4) {
  const float4 a = reinterpret_cast<const float4*>(m + b * TN_OPT_BLOCK)[lane], c = reinterpret_cast<const float4*>(v + b * TN_OPT_BLOCK)[lane];
  const double x[4] = {a.x, a.y, a.z, a.w}, y[4] = {c.x, c.y, c.z, c.w};
  float s1, s2;
  const uint32_t n1 = opt_encode_first(x, &s1), n2 = opt_encode_second(y, &s2);
  const bool bad = !(s1 < __builtin_huge_valf()) || !(s2 < __builtin_huge_valf());
  reinterpret_cast<uint32_t*>(q1 + b * TN_OPT_BLOCK)[lane] = n1;
  reinterpret_cast<uint32_t*>(q2 + b * TN_OPT_BLOCK)[lane] = n2;
  if (lane == 0) {
    scale1[b] = bad ? __builtin_nanf("") : s1;
    scale2[b] = bad ? __builtin_nanf("") : s2;
  }
  }
}

// ------------------------------------------------------------------------------------------------------------- host side
size_t opt_size(int dtype) { return dtype == TN_DTYPE_F32 ? 4 : 2; }

// Tensors that follow one another in memory become one: a model whose parameters are views of one flat buffer is then a few
// long runs instead of hundreds of short ones.  Looked for anew in every call.
bool opt_follows(const void* a, int64_t numel, size_t size, const void* b) { return (const char*)a + (size_t)numel * size == (const char*)b; }

template <typename F>
int opt_by_type(int dtype, F f) {
  if (dtype == TN_DTYPE_F32) return f((float*)nullptr);
  if (dtype == TN_DTYPE_BF16) return f((__bf16*)nullptr);
  if (dtype == TN_DTYPE_F16) return f((_Float16*)nullptr);
  return TN_E_UNSUPPORTED;
}

}  // namespace

extern "C" int64_t tn_grad_sumsq_partials(int32_t count, const int64_t* numel) {
  if (count < 0 || (count > 0 && !numel)) return TN_E_BADARG;
  int64_t n = 0;
  for (int i = 0; i < count; ++i) {
    if (numel[i] < 0) return TN_E_BADARG;
    n += (numel[i] + SUM_CHUNK - 1) / SUM_CHUNK;
  }
  return n;
}

extern "C" int tn_grad_sumsq(int32_t count, const void* const* grads, const int64_t* numel, int32_t dtype, double* partials,
                             int64_t* written, void* stream) {
  if (count < 0 || (count > 0 && (!grads || !numel || !partials)) || !written) return TN_E_BADARG;
  if (dtype < TN_DTYPE_F32 || dtype > TN_DTYPE_F16) return TN_E_UNSUPPORTED;
  for (int i = 0; i < count; ++i)
    if (numel[i] < 0 || (numel[i] > 0 && !grads[i])) return TN_E_BADARG;
  *written = 0;
  SumList list;
  int used = 0;
  uint32_t chunks = 0;
  auto flush = [&]() -> int {
    if (!used) return 0;
    for (int i = used; i < OPT_LIST; ++i) list.end[i] = 0xffffffffu;
    const int rc = opt_by_type(dtype, [&](auto* kind) -> int {
      using T = std::remove_pointer_t<decltype(kind)>;
      hipLaunchKernelGGL(HIP_KERNEL_NAME(grad_sumsq_kernel<T>), dim3(chunks), dim3(256), 0, (hipStream_t)stream, list, partials + *written);
      return (int)hipGetLastError();
    });
    *written += chunks;
    used = 0;
    chunks = 0;
    return rc;
  };
  for (int i = 0; i < count;) {
    const void* g = grads[i];
    int64_t n = numel[i++];
    if (n == 0) continue;
    while (i < count && numel[i] > 0 && opt_follows(g, n, opt_size(dtype), grads[i])) n += numel[i++];
    const int64_t c = (n + SUM_CHUNK - 1) / SUM_CHUNK;
    if (c > OPT_GRID) return TN_E_UNSUPPORTED;
    if (used == OPT_LIST || (int64_t)chunks + c > OPT_GRID)
      if (const int rc = flush()) return rc;
    list.g[used] = g;
    list.numel[used] = n;
    chunks += (uint32_t)c;
    list.end[used++] = chunks;
  }
  return flush();
}

extern "C" int tn_grad_norm_finish(const double* partials, int64_t count, double grad_mult, double max_norm, float* norm, double* ctl,
                                   void* stream) {
  if (count < 0 || (count > 0 && !partials) || (!norm && !ctl) || (ctl && !(max_norm > 0.0))) return TN_E_BADARG;
  hipLaunchKernelGGL(grad_norm_finish_kernel, dim3(1), dim3(256), 0, (hipStream_t)stream, partials, count, grad_mult, max_norm, norm, ctl);
  return (int)hipGetLastError();
}

extern "C" int tn_adamw_tick(int32_t count, const int32_t* slots, int32_t* steps, float* corr, const double* ctl, double lr,
                             const float* lr_dev, double beta1, double beta2, double weight_decay, void* stream) {
  if (count < 0 || (count > 0 && (!slots || !steps || !corr))) return TN_E_BADARG;
  if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || (!lr_dev && !(lr >= 0.0)) || !(weight_decay >= 0.0)) return TN_E_BADARG;
  for (int lo = 0; lo < count; lo += 256) {
    OptSlots s;
    s.count = std::min(256, count - lo);
    for (int i = 0; i < s.count; ++i) {
      if (slots[lo + i] < 0) return TN_E_BADARG;
      s.slot[i] = slots[lo + i];
    }
    hipLaunchKernelGGL(adamw_tick_kernel, dim3(1), dim3(256), 0, (hipStream_t)stream, s, steps, corr, ctl, lr, lr_dev, beta1, beta2, weight_decay);
    if (const int rc = (int)hipGetLastError()) return rc;
  }
  return 0;
}

extern "C" int tn_adamw_apply(int32_t count, void* const* params, const void* const* grads, const int64_t* numel, const int64_t* first_block,
                              const int32_t* slots, int32_t dtype, int32_t state_bits, void* exp_avg, void* exp_avg_sq, float* scale1,
                              float* scale2, int64_t blocks, const float* corr, const double* ctl, double grad_mult, double beta1,
                              double beta2, double eps, void* stream) {
  if (count < 0 || (count > 0 && (!params || !grads || !numel || !first_block || !slots || !exp_avg || !exp_avg_sq || !corr))) return TN_E_BADARG;
  if (dtype < TN_DTYPE_F32 || dtype > TN_DTYPE_F16 || (state_bits != 8 && state_bits != 32)) return TN_E_UNSUPPORTED;
  if (count > 0 && state_bits == 8 && (!scale1 || !scale2)) return TN_E_BADARG;
  if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0)) return TN_E_BADARG;
  if (blocks < 0 || blocks > 0xffffffffll) return TN_E_UNSUPPORTED;
  for (int i = 0; i < count; ++i)
    if (numel[i] < 0 || (numel[i] > 0 && (!params[i] || !grads[i])) || slots[i] < 0 || first_block[i] < 0 ||
        first_block[i] + (numel[i] + TN_OPT_BLOCK - 1) / TN_OPT_BLOCK > blocks)
      return TN_E_BADARG;
  const OptHyper h = {beta1, beta2, 1.0 - beta1, 1.0 - beta2, (float)eps, grad_mult};
  const size_t size = opt_size(dtype);
  OptList list;
  int used = 0;
  uint32_t chunks = 0;
  auto flush = [&]() -> int {
    if (!used) return 0;
    for (int i = used; i < OPT_LIST; ++i) list.end[i] = 0xffffffffu;
    const int rc = opt_by_type(dtype, [&](auto* kind) -> int {
      using T = std::remove_pointer_t<decltype(kind)>;
      if (state_bits == 32)
        hipLaunchKernelGGL(HIP_KERNEL_NAME(adamw32_kernel<T>), dim3(chunks), dim3(256), 0, (hipStream_t)stream, list, h, (float*)exp_avg,
                           (float*)exp_avg_sq, corr, ctl);
      else
        hipLaunchKernelGGL(HIP_KERNEL_NAME(adamw8_kernel<T>), dim3(chunks), dim3(256), 0, (hipStream_t)stream, list, h, (int8_t*)exp_avg,
                           (uint8_t*)exp_avg_sq, scale1, scale2, corr, ctl);
      return (int)hipGetLastError();
    });
    used = 0;
    chunks = 0;
    return rc;
  };
  for (int i = 0; i < count;) {
    const int a = i++;
    int64_t n = numel[a];
    if (n == 0) continue;
    while (i < count && numel[i] > 0 && slots[i] == slots[a] && first_block[i] * TN_OPT_BLOCK == first_block[a] * TN_OPT_BLOCK + n &&
           opt_follows(params[a], n, size, params[i]) && opt_follows(grads[a], n, size, grads[i]))
      n += numel[i++];
    const int64_t c = (n + OPT_CHUNK - 1) / OPT_CHUNK;
    if (c > OPT_GRID) return TN_E_UNSUPPORTED;
    if (used == OPT_LIST || (int64_t)chunks + c > OPT_GRID)
      if (const int rc = flush()) return rc;
    list.p[used] = params[a];
    list.g[used] = grads[a];
    list.numel[used] = n;
    list.first_block[used] = (uint32_t)first_block[a];
    list.slot[used] = (uint32_t)slots[a];
    chunks += (uint32_t)c;
    list.end[used++] = chunks;
  }
  return flush();
}

extern "C" int tn_moments_decode(const void* exp_avg, const void* exp_avg_sq, const float* scale1, const float* scale2, float* out1,
                                 float* out2, int64_t blocks, void* stream) {
  if (blocks < 0 || (blocks > 0 && (!exp_avg || !exp_avg_sq || !scale1 || !scale2 || !out1 || !out2))) return TN_E_BADARG;
  if (!blocks) return 0;
  hipLaunchKernelGGL(moments_decode_kernel, dim3((unsigned)std::min<int64_t>((blocks + 3) / 4, 1 << 20)), dim3(256), 0, (hipStream_t)stream, (const int8_t*)exp_avg,
                     (const uint8_t*)exp_avg_sq, scale1, scale2, out1, out2, blocks);
  return (int)hipGetLastError();
}

extern "C" int tn_moments_encode(const float* in1, const float* in2, void* exp_avg, void* exp_avg_sq, float* scale1, float* scale2,
                                 int64_t blocks, void* stream) {
  if (blocks < 0 || (blocks > 0 && (!exp_avg || !exp_avg_sq || !scale1 || !scale2 || !in1 || !in2))) return TN_E_BADARG;
  if (!blocks) return 0;
  hipLaunchKernelGGL(moments_encode_kernel, dim3((unsigned)std::min<int64_t>((blocks + 3) / 4, 1 << 20)), dim3(256), 0, (hipStream_t)stream, in1, in2, (int8_t*)exp_avg,
                     (uint8_t*)exp_avg_sq, scale1, scale2, blocks);
  return (int)hipGetLastError();
}
