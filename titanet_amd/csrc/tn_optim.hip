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

// Elements of one workgroup of the step, 32- and 8-bit moments.  Timed at 1024 / 2048 / 4096 / 8192: 26.1 M elements fp32 and 32 bits
// 144.1 / 144.4 / 146.9 / 150.6 us, 6.2 M with their norm 45 / 42.2 / 44.5 / 46; 64 M elements and 8 bits 299 / 309 / 312 / 317 us.
constexpr int OPT_CHUNK32 = 2048, OPT_CHUNK8 = 1024;
constexpr int SUM_CHUNK = 8192;        // elements behind one partial sum of the norm
constexpr int SMALL_BLOCKS = 64;       // blocks of 256 that one workgroup steps by itself, norm and all
constexpr int OPT_LIST = 96;           // tensors one launch can name in its arguments
constexpr int64_t OPT_GRID = (1 << 24) - 1;      // workgroups of 256 in one launch: the grid is counted in 32 bits of threads

// ------------------------------------------------------------------------------------------------- global gradient norm
struct SumList {
  const void* g[OPT_LIST];
  int64_t numel[OPT_LIST];
  uint32_t end[OPT_LIST];              // chunks of this launch before the end of tensor i (ascending)
};

// One partial sum of squares per chunk of SUM_CHUNK elements, in 64 bits (no gradient of a 32-bit type overflows there).  The order of
// the sum is fixed: two runs over the same tensors give the same norm.  Tensors that lie next to each other are summed as one run, so
// another layout can end its chunks elsewhere and differ in the last places of 64 bits.  Bound by memory: all of a chunk's loads are
// asked for at once (6.2 M float gradients 7.2 us, 3.5 TB/s; with a loop over chunks twice as long 13 us).
template <typename T>
__global__ __launch_bounds__(256) void grad_sumsq_kernel(SumList list, double* __restrict__ partials) {
  const int t = opt_find(list.end, OPT_LIST, blockIdx.x);
  const uint32_t before = t ? list.end[t - 1] : 0u;
  const int64_t lo = (int64_t)(blockIdx.x - before) * SUM_CHUNK, n = list.numel[t];
  const T* g = reinterpret_cast<const T*>(list.g[t]);
  double s = 0.0;
  float v[SUM_CHUNK / 1024][4];        // all loads of the chunk on their way together
  if (lo + SUM_CHUNK <= n) {
#pragma unroll
    for (int k = 0; k < SUM_CHUNK / 1024; ++k) opt_load4<true>(g, lo + k * 1024 + 4 * threadIdx.x, n, v[k]);
  } else {
#pragma unroll
    for (int k = 0; k < SUM_CHUNK / 1024; ++k) opt_load4(g, lo + k * 1024 + 4 * threadIdx.x, n, v[k]);
  }
#pragma unroll
  for (int k = 0; k < SUM_CHUNK / 1024; ++k)
#pragma unroll
    for (int j = 0; j < 4; ++j) s = fma((double)v[k][j], (double)v[k][j], s);
  s = opt_sum_workgroup<4>(s);
  if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

struct NormArgs {
  const double* partials;
  int64_t count;
  double mult, max_norm;
  float* norm;                         // may be null
  double* ctl;                         // may be null
};

// norm = |mult| sqrt(sum), ctl = {factor of the gradients, 1 if the step runs}: a norm that is no number stops the step
__device__ void opt_finish_norm(const NormArgs& a, double sum, double ctl[2]) {
  const double norm = sqrt(sum) * fabs(a.mult);
  if (a.norm) *a.norm = (float)norm;
  const bool ok = norm < __builtin_huge_val();            // false for NaN too
  const double c = a.max_norm / (norm + 1e-6);
  ctl[0] = ok ? a.mult * (c < 1.0 ? c : 1.0) : 0.0;
  ctl[1] = ok ? 1.0 : 0.0;
}

__device__ double opt_power(double b, int32_t t) {       // b^t by squaring: exact enough for 1 - b^t at every t
  double r = 1.0;
  while (t > 0) {
    if (t & 1) r *= b;
    b *= b;
    t >>= 1;
  }
  return r;
}

constexpr int TICK_SLOTS = 512, SMALL_SLOTS = 256;     // slots that one launch can name in its arguments
template <int MOST>
struct OptSlots {
  int32_t slot[MOST];
  int32_t count;
};
struct TickArgs {
  int32_t* steps;
  float* corr;
  double lr;
  const float* lr_dev;
  double b1, b2, wd;
};

// steps[slot] += 1 and the four numbers of the step that depend on it: {step size, 1 / sqrt(1 - b2^t), 1 - lr wd, runs}
__device__ float4 opt_tick(const TickArgs& a, int slot, bool runs) {
  float4 c = make_float4(0.f, 0.f, 0.f, 0.f);
  if (runs) {
    const int32_t t = a.steps[slot] + 1;
    a.steps[slot] = t;
    const double lr = a.lr_dev ? (double)*a.lr_dev : a.lr;
    c = make_float4((float)(lr / (1.0 - opt_power(a.b1, t))), (float)(1.0 / sqrt(1.0 - opt_power(a.b2, t))), (float)(1.0 - lr * a.wd), 1.f);
  }
  reinterpret_cast<float4*>(a.corr)[slot] = c;
  return c;
}

// (the first four of the workgroup's WAVES waves add: the same order for every caller)
template <int WAVES>
__device__ double opt_sum_partials(const NormArgs& a) {
  double s = 0.0;
  if (threadIdx.x < 256)
    for (int64_t i = threadIdx.x; i < a.count; i += 256) s += a.partials[i];
  return opt_sum_workgroup<WAVES>(s);
}

__global__ __launch_bounds__(256) void grad_norm_finish_kernel(NormArgs a) {
  const double s = opt_sum_partials<4>(a);
  double ctl[2];
  if (threadIdx.x == 0) {
    opt_finish_norm(a, s, ctl);
    if (a.ctl) {
      a.ctl[0] = ctl[0];
      a.ctl[1] = ctl[1];
    }
  }
}

// The norm's end (first = true: from its partial sums; otherwise ctl has it) and the counts, in one launch
__global__ __launch_bounds__(TICK_SLOTS) void adamw_tick_kernel(OptSlots<TICK_SLOTS> list, TickArgs t, NormArgs a, bool first) {
  __shared__ double runs;
  if (first) {
    const double s = opt_sum_partials<TICK_SLOTS / 64>(a);
    double ctl[2];
    if (threadIdx.x == 0) {
      opt_finish_norm(a, s, ctl);
      a.ctl[0] = ctl[0];
      a.ctl[1] = ctl[1];
      runs = ctl[1];
    }
    __syncthreads();
  } else if (threadIdx.x == 0) {
    runs = a.ctl ? a.ctl[1] : 1.0;
  }
  __syncthreads();
  if ((int)threadIdx.x < list.count) opt_tick(t, list.slot[threadIdx.x], runs != 0.0);
}

// -------------------------------------------------------------------------------------------------------------- the step
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

__device__ __forceinline__ OptStep opt_step_of(const OptHyper& h, const float4& c, double factor) {
  return {h.b1, h.b2, h.w1, h.w2, factor, c.x, c.y, c.z, h.eps};
}

// 32-bit moments: four elements to a lane, 28 bytes of an element (float parameters) moved once.  Bound by HBM: 26.1 M elements in
// 130 us, 5.6 TB/s, where a large copy reaches 4.8; moments and gradients go past the caches (142 us with them left there).
// EACH: a run's tensors may be at different counts, every block of 256 elements (a wave's four times 64) has the numbers of its own.
template <typename T, bool EACH>
__global__ __launch_bounds__(256) void adamw32_kernel(OptList list, OptHyper h, float* __restrict__ exp_avg, float* __restrict__ exp_avg_sq,
                                                      const float* __restrict__ corr, const int32_t* __restrict__ owner,
                                                      const double* __restrict__ ctl) {
  const int t = opt_find(list.end, OPT_LIST, blockIdx.x);
  const float4* corrs = reinterpret_cast<const float4*>(corr);
  OptStep step;
  if constexpr (!EACH) {
    const float4 c = corrs[list.slot[t]];
    if (c.w == 0.f) return;
    step = opt_step_of(h, c, ctl ? ctl[0] : h.mult);
  } else if (ctl && ctl[1] == 0.0) {
    return;
  }
  const uint32_t before = t ? list.end[t - 1] : 0u;
  const int64_t lo = (int64_t)(blockIdx.x - before) * OPT_CHUNK32, n = list.numel[t];
  T* p = reinterpret_cast<T*>(list.p[t]);
  const T* g = reinterpret_cast<const T*>(list.g[t]);
  float* m = exp_avg + (int64_t)list.first_block[t] * TN_OPT_BLOCK;
  float* v = exp_avg_sq + (int64_t)list.first_block[t] * TN_OPT_BLOCK;
  if (lo + OPT_CHUNK32 <= n) {
#pragma unroll
    for (int k = 0; k < OPT_CHUNK32 / 1024; ++k) {
      const int64_t i = lo + k * 1024 + 4 * threadIdx.x;
      float gv[4];
      opt_load4<true, true>(g, i, n, gv);
      if constexpr (EACH) step = opt_step_of(h, corrs[owner[list.first_block[t] + i / TN_OPT_BLOCK]], ctl ? ctl[0] : h.mult);
      opt_step32<true>(step, p, gv, i, n, m, v);
    }
  } else {
    for (int64_t i = lo + 4 * threadIdx.x; i < n; i += 1024) {
      float gv[4];
      opt_load4(g, i, n, gv);
      if constexpr (EACH) step = opt_step_of(h, corrs[owner[list.first_block[t] + i / TN_OPT_BLOCK]], ctl ? ctl[0] : h.mult);
      opt_step32<false>(step, p, gv, i, n, m, v);
    }
  }
}

// 8-bit moments: one wave holds one block of 256 elements, four to a lane, so that the block's maxima are a reduction over the
// wave and neither LDS nor a barrier is needed.  16 bytes of an element (float parameters): 64 M elements in 187 us, 5.5 TB/s.  With
// 16-bit parameters (10 bytes) the vector pipe bounds it: some 450 instructions a block, a fifth of them in the 64 bits that
// decide every code (7.9 M bfloat16 elements in 26 us, 3.1 TB/s; 37 us with integer squares, 64-bit quotients and a shuffled maximum).
template <typename T, bool EACH>
__global__ __launch_bounds__(256) void adamw8_kernel(OptList list, OptHyper h, int8_t* __restrict__ exp_avg, uint8_t* __restrict__ exp_avg_sq,
                                                     float* __restrict__ scale1, float* __restrict__ scale2,
                                                     const float* __restrict__ corr, const int32_t* __restrict__ owner,
                                                     const double* __restrict__ ctl) {
  const int t = opt_find(list.end, OPT_LIST, blockIdx.x);
  const uint32_t before = t ? list.end[t - 1] : 0u;
  const int64_t lo = (int64_t)(blockIdx.x - before) * OPT_CHUNK8, n = list.numel[t];
  T* p = reinterpret_cast<T*>(list.p[t]);
  const T* g = reinterpret_cast<const T*>(list.g[t]);
  static_assert(OPT_CHUNK8 == 4 * TN_OPT_BLOCK, "a block to a wave");
  const int64_t i0 = lo + (threadIdx.x >> 6) * TN_OPT_BLOCK;
  if (i0 >= n) return;
  const int64_t i = i0 + 4 * (threadIdx.x & 63), block = (int64_t)list.first_block[t] + i0 / TN_OPT_BLOCK;
  const float4 c = reinterpret_cast<const float4*>(corr)[EACH ? (uint32_t)owner[block] : list.slot[t]];
  if (c.w == 0.f) return;
  const OptStep step = opt_step_of(h, c, ctl ? ctl[0] : h.mult);
  float gv[4];
  if (i0 + TN_OPT_BLOCK <= n) {
    opt_load4<true, true>(g, i, n, gv);
    opt_step8_block<true>(step, p, gv, i0, n, block, exp_avg, exp_avg_sq, scale1, scale2);
  } else {
    opt_load4(g, i, n, gv);
    opt_step8_block<false>(step, p, gv, i0, n, block, exp_avg, exp_avg_sq, scale1, scale2);
  }
}

// A few small tensors: one workgroup of 16 waves takes the norm, the counts and the step, a block of 256 elements to a wave and turn
// with its gradient kept in registers in between.  Nothing but latency: 7.8 us for 7 bfloat16 tensors of up to 1537 elements, where the
// three launches of the general way take 15 and the gaps between them; the call then waits for the host (11.7 us, was 22.9).
template <typename T, int BITS>
__global__ __launch_bounds__(1024) void adamw_small_kernel(OptList list, OptHyper h, OptSlots<SMALL_SLOTS> slots, TickArgs tick, NormArgs a, bool clip, void* exp_avg,
                                                           void* exp_avg_sq, float* scale1, float* scale2, const int32_t* owner) {
  constexpr int TURNS = SMALL_BLOCKS / 16;
  __shared__ double ctl[2];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  float g[TURNS][4];
  double s = 0.0;
#pragma unroll
  for (int k = 0; k < TURNS; ++k) {                 // (end counts blocks here)
    const uint32_t b = k * 16 + wave;
    const int t = opt_find(list.end, OPT_LIST, b);
    if (t >= OPT_LIST || list.end[t] == 0xffffffffu) continue;
    const int64_t i0 = (int64_t)(b - (t ? list.end[t - 1] : 0u)) * TN_OPT_BLOCK;
    opt_load4(reinterpret_cast<const T*>(list.g[t]), i0 + 4 * lane, list.numel[t], g[k]);
    if (clip)
#pragma unroll
      for (int j = 0; j < 4; ++j) s = fma((double)g[k][j], (double)g[k][j], s);
  }
  if (clip) {
    s = opt_sum_workgroup<16>(s);
    if (threadIdx.x == 0) opt_finish_norm(a, s, ctl);
  } else if (threadIdx.x == 0) {
    ctl[0] = h.mult;
    ctl[1] = 1.0;
  }
  __syncthreads();
  if ((int)threadIdx.x < slots.count) opt_tick(tick, slots.slot[threadIdx.x], ctl[1] != 0.0);
  __syncthreads();                                  // (corr is this workgroup's own writing: visible behind the barrier)
  if (ctl[1] == 0.0) return;
#pragma unroll
  for (int k = 0; k < TURNS; ++k) {
    const uint32_t b = k * 16 + wave;
    const int t = opt_find(list.end, OPT_LIST, b);
    if (t >= OPT_LIST || list.end[t] == 0xffffffffu) continue;
    const int64_t i0 = (int64_t)(b - (t ? list.end[t - 1] : 0u)) * TN_OPT_BLOCK, first = list.first_block[t];
    const float4 c = reinterpret_cast<const float4*>(tick.corr)[owner ? (uint32_t)owner[first + i0 / TN_OPT_BLOCK] : list.slot[t]];
    const OptStep step = opt_step_of(h, c, ctl[0]);
    T* p = reinterpret_cast<T*>(list.p[t]);
    if constexpr (BITS == 32)
      opt_step32<false>(step, p, g[k], i0 + 4 * lane, list.numel[t], (float*)exp_avg + first * TN_OPT_BLOCK, (float*)exp_avg_sq + first * TN_OPT_BLOCK);
    else
      opt_step8_block<false>(step, p, g[k], i0, list.numel[t], first + i0 / TN_OPT_BLOCK, (int8_t*)exp_avg, (uint8_t*)exp_avg_sq, scale1, scale2);
  }
}

// 10 bytes of an element, bound by HBM: 64 M elements in 100 us, 6.4 TB/s
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
  const float xf[4] = {a.x, a.y, a.z, a.w}, yf[4] = {c.x, c.y, c.z, c.w};
  const double x[4] = {a.x, a.y, a.z, a.w}, y[4] = {c.x, c.y, c.z, c.w};
  float s1, s2;
  const uint32_t n1 = opt_encode_first(x, xf, &s1), n2 = opt_encode_second(y, yf, &s2);
  const bool bad = !(s1 < __builtin_huge_valf()) || !(s2 < __builtin_huge_valf());
  reinterpret_cast<uint32_t*>(q1 + b * TN_OPT_BLOCK)[lane] = bad ? 0u : n1;
  reinterpret_cast<uint32_t*>(q2 + b * TN_OPT_BLOCK)[lane] = bad ? 0u : n2;
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
  const NormArgs a = {partials, count, grad_mult, max_norm, norm, ctl};
  hipLaunchKernelGGL(grad_norm_finish_kernel, dim3(1), dim3(256), 0, (hipStream_t)stream, a);
  return (int)hipGetLastError();
}

namespace {

bool hyper_ok(const tn_adamw_hyper* h) {
  return h && h->beta1 >= 0.0 && h->beta1 < 1.0 && h->beta2 >= 0.0 && h->beta2 < 1.0 && h->eps >= 0.0 && h->weight_decay >= 0.0 &&
         (h->lr_dev || h->lr >= 0.0);
}
OptHyper hyper_of(const tn_adamw_hyper* h, double mult) { return {h->beta1, h->beta2, 1.0 - h->beta1, 1.0 - h->beta2, (float)h->eps, mult}; }
TickArgs tick_of(const tn_adamw_hyper* h, int32_t* steps, float* corr) { return {steps, corr, h->lr, h->lr_dev, h->beta1, h->beta2, h->weight_decay}; }

int lists_ok(const tn_adamw_lists* l, const tn_adamw_state* s) {
  if (!l || !s || l->count < 0) return TN_E_BADARG;
  if (l->dtype < TN_DTYPE_F32 || l->dtype > TN_DTYPE_F16 || (s->bits != 8 && s->bits != 32)) return TN_E_UNSUPPORTED;
  if (s->blocks < 0 || s->blocks > 0xffffffffll) return TN_E_UNSUPPORTED;
  if (l->count == 0) return 0;
  if (!l->params || !l->grads || !l->numel || !l->first_block || !l->slots || !s->exp_avg || !s->exp_avg_sq || !s->corr) return TN_E_BADARG;
  if (s->bits == 8 && (!s->scale1 || !s->scale2)) return TN_E_BADARG;
  for (int i = 0; i < l->count; ++i)
    if (l->numel[i] < 0 || (l->numel[i] > 0 && (!l->params[i] || !l->grads[i])) || l->slots[i] < 0 || l->first_block[i] < 0 ||
        l->numel[i] > (s->blocks - l->first_block[i]) * TN_OPT_BLOCK)
      return TN_E_BADARG;
  return 0;
}

// Runs of the list, tensors that follow one another in parameters, gradients and moments joined (where each block knows its slot, whatever
// the slots): f(first of the run, elements).
template <typename F>
int each_run(const tn_adamw_lists* l, const tn_adamw_state* s, F f) {
  const size_t size = opt_size(l->dtype);
  for (int i = 0; i < l->count;) {
    const int a = i++;
    int64_t n = l->numel[a];
    if (n == 0) continue;
    while (i < l->count && l->numel[i] > 0 && (s->owner || l->slots[i] == l->slots[a]) &&
           l->first_block[i] * TN_OPT_BLOCK == l->first_block[a] * TN_OPT_BLOCK + n && opt_follows(l->params[a], n, size, l->params[i]) &&
           opt_follows(l->grads[a], n, size, l->grads[i]))
      n += l->numel[i++];
    if (const int rc = f(a, n)) return rc;
  }
  return 0;
}

void put_run(OptList& list, int at, const tn_adamw_lists* l, int a, int64_t n, uint32_t end) {
  list.p[at] = l->params[a];
  list.g[at] = l->grads[a];
  list.numel[at] = n;
  list.first_block[at] = (uint32_t)l->first_block[a];
  list.slot[at] = (uint32_t)l->slots[a];
  list.end[at] = end;
}

}  // namespace

extern "C" int tn_adamw_tick(int32_t count, const int32_t* slots, const tn_adamw_state* s, const tn_adamw_hyper* h, const double* partials,
                             int64_t n_partials, double grad_mult, double max_norm, float* norm, double* ctl, void* stream) {
  if (count < 0 || !s || !hyper_ok(h) || (count > 0 && (!slots || !s->steps || !s->corr))) return TN_E_BADARG;
  if (partials && (n_partials < 0 || !ctl || !(max_norm > 0.0))) return TN_E_BADARG;
  for (int i = 0; i < count; ++i)
    if (slots[i] < 0) return TN_E_BADARG;
  const NormArgs a = {partials, n_partials, grad_mult, max_norm, norm, ctl};
  for (int lo = 0; lo < count || (partials && lo == 0); lo += TICK_SLOTS) {      // (without slots the norm still ends)
    OptSlots<TICK_SLOTS> list;
    list.count = std::min(TICK_SLOTS, count - lo);
    for (int i = 0; i < list.count; ++i) list.slot[i] = slots[lo + i];
    hipLaunchKernelGGL(adamw_tick_kernel, dim3(1), dim3(TICK_SLOTS), 0, (hipStream_t)stream, list, tick_of(h, s->steps, s->corr), a, partials && lo == 0);
    if (const int rc = (int)hipGetLastError()) return rc;
  }
  return 0;
}

extern "C" int tn_adamw_apply(const tn_adamw_lists* l, const tn_adamw_state* s, const tn_adamw_hyper* h, double grad_mult, const double* ctl,
                              void* stream) {
  if (!hyper_ok(h)) return TN_E_BADARG;
  if (const int rc = lists_ok(l, s)) return rc;
  OptList list;
  int used = 0;
  uint32_t chunks = 0;
  auto flush = [&]() -> int {
    if (!used) return 0;
    for (int i = used; i < OPT_LIST; ++i) list.end[i] = 0xffffffffu;
    const int rc = opt_by_type(l->dtype, [&](auto* kind) -> int {
      using T = std::remove_pointer_t<decltype(kind)>;
      auto go = [&](auto each) {
        if (s->bits == 32)
          hipLaunchKernelGGL(HIP_KERNEL_NAME(adamw32_kernel<T, decltype(each)::value>), dim3(chunks), dim3(256), 0, (hipStream_t)stream, list,
                             hyper_of(h, grad_mult), (float*)s->exp_avg, (float*)s->exp_avg_sq, s->corr, s->owner, ctl);
        else
          hipLaunchKernelGGL(HIP_KERNEL_NAME(adamw8_kernel<T, decltype(each)::value>), dim3(chunks), dim3(256), 0, (hipStream_t)stream, list,
                             hyper_of(h, grad_mult), (int8_t*)s->exp_avg, (uint8_t*)s->exp_avg_sq, s->scale1, s->scale2, s->corr, s->owner, ctl);
      };
      s->owner ? go(std::true_type{}) : go(std::false_type{});
      return (int)hipGetLastError();
    });
    used = 0;
    chunks = 0;
    return rc;
  };
  const int rc = each_run(l, s, [&](int a, int64_t n) -> int {
    const int chunk = s->bits == 32 ? OPT_CHUNK32 : OPT_CHUNK8;
    const int64_t c = (n + chunk - 1) / chunk;
    if (c > OPT_GRID) return TN_E_UNSUPPORTED;
    if (used == OPT_LIST || (int64_t)chunks + c > OPT_GRID)
      if (const int e = flush()) return e;
    chunks += (uint32_t)c;
    put_run(list, used++, l, a, n, chunks);
    return 0;
  });
  return rc ? rc : flush();
}

extern "C" int tn_adamw_step_small(const tn_adamw_lists* l, const tn_adamw_state* s, const tn_adamw_hyper* h, int32_t n_slots, const int32_t* slots,
                                   double grad_mult, double max_norm, float* norm, void* stream) {
  if (!hyper_ok(h) || n_slots < 0 || (n_slots > 0 && !slots) || max_norm < 0.0) return TN_E_BADARG;
  if (const int rc = lists_ok(l, s)) return rc;
  if (!s->steps || n_slots > SMALL_SLOTS) return s->steps ? TN_E_UNSUPPORTED : TN_E_BADARG;
  OptSlots<SMALL_SLOTS> sl;
  sl.count = n_slots;
  for (int i = 0; i < n_slots; ++i) {
    if (slots[i] < 0) return TN_E_BADARG;
    sl.slot[i] = slots[i];
  }
  OptList list;
  int used = 0;
  uint32_t blocks = 0;
  const int rc = each_run(l, s, [&](int a, int64_t n) -> int {
    const int64_t c = (n + TN_OPT_BLOCK - 1) / TN_OPT_BLOCK;
    if (used == OPT_LIST || c > SMALL_BLOCKS || blocks + c > SMALL_BLOCKS) return TN_E_UNSUPPORTED;
    blocks += (uint32_t)c;
    put_run(list, used++, l, a, n, blocks);
    return 0;
  });
  if (rc) return rc;
  for (int i = used; i < OPT_LIST; ++i) list.end[i] = 0xffffffffu;
  const NormArgs a = {nullptr, 0, grad_mult, max_norm, norm, nullptr};
  return opt_by_type(l->dtype, [&](auto* kind) -> int {
    using T = std::remove_pointer_t<decltype(kind)>;
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, list, hyper_of(h, grad_mult), sl, tick_of(h, s->steps, s->corr), a,
                         max_norm > 0.0, s->exp_avg, s->exp_avg_sq, s->scale1, s->scale2, s->owner);
      return (int)hipGetLastError();
    };
    return s->bits == 32 ? go(adamw_small_kernel<T, 32>) : go(adamw_small_kernel<T, 8>);
  });
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
