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

// largest of an aligned group of GROUP lanes' numbers (none negative, so their bit patterns are ordered like them)
template <int GROUP>
__device__ __forceinline__ float q8_max_group(float f) {
  int x = __float_as_int(f);
  auto up = [&](int y) { x = x > y ? x : y; };
  up(__builtin_amdgcn_update_dpp(0, x, 0xb1, 0xf, 0xf, false));                       // lane ^ 1
  up(__builtin_amdgcn_update_dpp(0, x, 0x4e, 0xf, 0xf, false));                       // lane ^ 2
  up(__builtin_amdgcn_update_dpp(0, x, 0x141, 0xf, 0xf, false));                      // mirrored within 8
  if (GROUP >= 16) up(__builtin_amdgcn_update_dpp(0, x, 0x140, 0xf, 0xf, false));     // mirrored within 16
  if (GROUP >= 32) up(__shfl_xor(x, 16, 64));
  if (GROUP >= 64) up(__shfl_xor(x, 32, 64));
  return __int_as_float(x);
}

// eight consecutive elements from k on as floats, zeros behind the row's end; the type's own alignment is enough
template <typename T>
struct Q8Vec {
  typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};
template <typename T>
__device__ __forceinline__ void q8_load8(const T* row, int k, int cols, float v[8]) {
  if (k + 8 <= cols) {
    const typename Q8Vec<T>::type x = *reinterpret_cast<const typename Q8Vec<T>::type*>(row + k);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float)x[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k + j < cols ? (float)row[k + j] : 0.f;
  }
}
// largest |v|; bad where one of them is not finite (a maximum drops NaN)
__device__ __forceinline__ float q8_top8(const float v[8], float top, bool& bad) {
#pragma unroll
  for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(v[j]));
#pragma unroll
  for (int j = 0; j < 8; ++j) bad |= !(fabsf(v[j]) < __builtin_huge_valf());
  return top;
}
// Codes of eight values.  Adding 1.5 * 2^23 in one fused multiply-add leaves the nearest integer to x * inv in the sum's low byte
// (two's complement, even half way); inv itself is off by half a step, 127 * 2^-24 of a code at most, so only where the quotient
// comes within 2^-16 of half way the exact comparison has to decide.  5 instructions a value where the comparison alone takes 20:
// the quantiser is bound by memory instead of by the vector pipe.
__device__ __forceinline__ uint2 q8_pack8(const float v[8], float s, float inv) {
  constexpr float MAGIC = 12582912.f;
  float t[8], off = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    t[j] = fmaf(v[j], inv, MAGIC);
    off = fmaxf(off, fabsf(fmaf(v[j], inv, -(t[j] - MAGIC))));
  }
  if (off > 0.5f - 0x1p-16f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = __int_as_float(q8_code(v[j], s, inv));
  }
  auto four = [](const float* f) {
    const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(f[1]), __float_as_uint(f[0]), 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(f[3]), __float_as_uint(f[2]), 0x04000c0cu);
    return lo | hi;
  };
  return make_uint2(four(t), four(t + 4));
}

// Codes and scale of every row.  A row belongs to GROUP lanes of a wave, eight elements to a lane and pass, kept in registers
// between the maximum and the codes where PASSES of them hold the row (PASSES = 0: read twice).  One pass over memory and bound by
// it: 76800 x 1536 bfloat16 in 78 - 90 us, 3.9 - 4.5 TB/s (258 us element by element, 97 with 20 instructions a value).
template <typename T, int GROUP, int PASSES>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* __restrict__ x, int64_t rows, int cols, int64_t ldx, int8_t* __restrict__ q,
                                                            int64_t ldq, int padded, float* __restrict__ scales) {
  constexpr int PER = 64 / GROUP;                  // rows of a wave
  const int lane = threadIdx.x & 63, in = lane % GROUP;
  for (int64_t r0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * PER; r0 < rows; r0 += (int64_t)gridDim.x * 4 * PER) {
    const int64_t r = r0 + lane / GROUP < rows ? r0 + lane / GROUP : rows - 1;       // (the last row twice: the same codes)
    const T* row = x + r * ldx;
    float v[PASSES ? PASSES : 1][8];
    float top = 0.f;
    bool bad = false;
    if constexpr (PASSES > 0) {
#pragma unroll
      for (int p = 0; p < PASSES; ++p) q8_load8(row, (p * GROUP + in) * 8, cols, v[p]);
#pragma unroll
      for (int p = 0; p < PASSES; ++p) top = q8_top8(v[p], top, bad);
    } else {
      for (int k = in * 8; k < cols; k += GROUP * 8) {
        q8_load8(row, k, cols, v[0]);
        top = q8_top8(v[0], top, bad);
      }
    }
    top = q8_max_group<GROUP>(bad ? __builtin_huge_valf() : top);
    const bool finite = top < __builtin_huge_valf();
    const float s = finite ? q8_scale(top) : 0.f, inv = s > 0.f ? 1.f / s : 0.f;
    uint2* out = reinterpret_cast<uint2*>(q + r * ldq);
    if constexpr (PASSES > 0) {
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const int k = (p * GROUP + in) * 8;
        if (k < padded) out[k / 8] = s > 0.f ? q8_pack8(v[p], s, inv) : make_uint2(0u, 0u);
      }
    } else {
      for (int k = in * 8; k < padded; k += GROUP * 8) {
        q8_load8(row, k, cols, v[0]);
        out[k / 8] = s > 0.f ? q8_pack8(v[0], s, inv) : make_uint2(0u, 0u);
      }
    }
    if (in == 0) scales[r] = finite ? s : __builtin_nanf("");
  }
}

struct Int8Args {
  const int8_t *a, *b;
  const float *sa, *sb, *bias;
  void* y;
  int64_t lda, ldb, ldy, m, n;
  int k;                              // multiple of 64
};

// The sum times both scales.  The sum is a whole number below 2^32, so times a token scale below 2^96 it stays in range (and a small scale
// costs nothing: the product is a multiple of the scale's own last place).  A larger token scale (rows from 1e31 on) goes last: the sum
// times it could leave 32 bits where the product does not.
constexpr float Q8_FAR = 0x1p96f;
template <typename T, bool FAR>
__device__ __forceinline__ T q8_out(int acc, float sa, float sb, float bias) {
  if constexpr (!FAR) return (T)((float)acc * sa * sb + bias);
  const bool last = fabsf(sa) >= Q8_FAR;
  return (T)((float)acc * (last ? sb : sa) * (last ? sa : sb) + bias);
}

// ------------------------------------------------------------------------------------------------------- few rows (m <= 32)
// The weight is read once, straight from memory into matrix operands (a lane's 16 bytes of one weight row); the rows' codes are
// made by every workgroup for itself in LDS while the first weight loads are on their way, so one launch does it all.  NW waves
// share a tile of 32 channels by splitting K in KS parts (joined through LDS: integer sums, any order gives the same) or work on
// NW / KS tiles.  Bound by the latency of load - maximum - codes - product for small weights (1 x 7205 x 192 4.6 us, 16 x 192 x 1536 from
// float 6.3 us; quantised by a launch of its own and multiplied in tiles they took 8.4 and 28), by HBM for one row
// against a large one (1 x 100003 x 1536 34 us, 4.5 TB/s).  More rows make their codes anew in each of up to 2048 workgroups: 16 rows
// 43 us, 32 rows 75 (2.2 TB/s).
struct FewArgs {
  const void* x;                      // rows of X, or codes with scales sa
  Int8Args g;
  int64_t ldx;
  int cols;
};

template <typename X, typename Y, int NW, int KS>
__global__ __launch_bounds__(NW * 64) void int8_few_rows_kernel(FewArgs f) {
  constexpr int G = NW / KS, AHEAD = KS == 16 ? 3 : 6;      // weight loads on their way before the rows' codes are made
  extern __shared__ __attribute__((aligned(16))) int8_t smem[];
  const Int8Args& g = f.g;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fi = lane & 31, fh = lane >> 5;
  const int m = (int)g.m, pitch = g.k + 16;
  float* scales = reinterpret_cast<float*>(smem + (size_t)m * pitch);           // (pitch is a multiple of 16)
  int* part = reinterpret_cast<int*>(scales + 32);                              // [NW][m <= 32 rows: 16 x 64], used for KS > 1
  const int slice = wave % KS, steps = g.k / 32;
  const int lo = steps * slice / KS, hi = steps * (slice + 1) / KS;
  const int64_t tiles = (g.n + 31) / 32, stride = (int64_t)gridDim.x * G;
  int64_t tile = (int64_t)blockIdx.x * G + wave / KS;
  auto row_of = [&](int64_t t) {
    int64_t r = t * 32 + fi;
    r = r < g.n ? r : g.n - 1;
    return g.b + r * g.ldb + fh * 16;
  };
  i32x4_t first[AHEAD];
  {
    const int8_t* pb = row_of(tile < tiles ? tile : tiles - 1);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) first[i] = *reinterpret_cast<const i32x4_t*>(pb + (lo + i < steps ? lo + i : steps - 1) * 32);
  }
  // ---- codes of the rows
  if constexpr (std::is_same_v<X, int8_t>) {
    for (int i = threadIdx.x; i < m * (g.k / 16); i += NW * 64) {
      const int r = i / (g.k / 16), c = i % (g.k / 16);
      *reinterpret_cast<i32x4_t*>(smem + r * pitch + c * 16) = *reinterpret_cast<const i32x4_t*>(reinterpret_cast<const int8_t*>(f.x) + r * f.ldx + c * 16);
    }
    if (threadIdx.x < m) scales[threadIdx.x] = g.sa[threadIdx.x];
  } else {
    for (int r = wave; r < m; r += NW) {
      const X* row = reinterpret_cast<const X*>(f.x) + r * f.ldx;
      constexpr int HELD = 4;                      // a row of up to 64 * 8 * HELD elements is read once
      float v[HELD][8], top = 0.f;
      bool bad = false;
#pragma unroll
      for (int p = 0; p < HELD; ++p)
        if (p * 512 < f.cols) q8_load8(row, p * 512 + lane * 8, f.cols, v[p]);
#pragma unroll
      for (int p = 0; p < HELD; ++p)
        if (p * 512 < f.cols) top = q8_top8(v[p], top, bad);
      float w[8];
      for (int k = HELD * 512 + lane * 8; k < f.cols; k += 512) {
        q8_load8(row, k, f.cols, w);
        top = q8_top8(w, top, bad);
      }
      top = q8_max_group<64>(bad ? __builtin_huge_valf() : top);
      const bool finite = top < __builtin_huge_valf();
      const float s = finite ? q8_scale(top) : 0.f, inv = s > 0.f ? 1.f / s : 0.f;
      uint2* out = reinterpret_cast<uint2*>(smem + r * pitch);
#pragma unroll
      for (int p = 0; p < HELD; ++p) {
        const int k = p * 512 + lane * 8;
        if (k < g.k) out[k / 8] = s > 0.f ? q8_pack8(v[p], s, inv) : make_uint2(0u, 0u);
      }
      for (int k = HELD * 512 + lane * 8; k < g.k; k += 512) {
        q8_load8(row, k, f.cols, w);
        out[k / 8] = s > 0.f ? q8_pack8(w, s, inv) : make_uint2(0u, 0u);
      }
      if (lane == 0) scales[r] = finite ? s : __builtin_nanf("");
    }
  }
  __syncthreads();
  Y* y = reinterpret_cast<Y*>(g.y);
  const int8_t* pa = smem + (fi < m ? fi : m - 1) * pitch + fh * 16;
  auto store = [&](int64_t t, int r, int sum, float sb, float bias) {
    const int row = (r & 3) + 8 * (r >> 2) + 4 * fh;
    const int64_t col = t * 32 + fi;
    if (row < m && col < g.n) y[row * g.ldy + col] = q8_out<Y, true>(sum, scales[row], sb, bias);
  };
  bool held = true;
  for (int64_t base = (int64_t)blockIdx.x * G; base < tiles; base += stride, tile += stride) {      // uniform over the workgroup
    const bool live = tile < tiles;
    const int8_t* pb = row_of(live ? tile : tiles - 1);
    const int64_t col = tile * 32 + fi < g.n ? tile * 32 + fi : g.n - 1;
    const float sb = g.sb[col], bias = g.bias ? g.bias[col] : 0.f;
    i32x16_t acc = {};
    for (int ks = lo; ks < hi; ks += AHEAD) {
      i32x4_t bf[AHEAD];
      if (held) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) bf[i] = first[i];
        held = false;
      } else {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) bf[i] = *reinterpret_cast<const i32x4_t*>(pb + (ks + i < steps ? ks + i : steps - 1) * 32);
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (ks + i < hi) acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(*reinterpret_cast<const i32x4_t*>(pa + (ks + i) * 32), bf[i], acc, 0, 0, 0);
    }
    if constexpr (KS == 1) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (live) store(tile, r, acc[r], sb, bias);
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if ((r & 3) + 8 * (r >> 2) < m) part[(wave * 16 + r) * 64 + lane] = acc[r];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 16 / KS; ++i) {
        const int r = slice * (16 / KS) + i;
        if ((r & 3) + 8 * (r >> 2) < m) {
          int sum = 0;
#pragma unroll
          for (int k = 0; k < KS; ++k) sum += part[((wave - slice + k) * 16 + r) * 64 + lane];
          if (live) store(tile, r, sum, sb, bias);
        }
      }
      __syncthreads();
    }
  }
}

// ------------------------------------------------------------------------------------------------------------ tiles of rows
typedef __attribute__((address_space(3))) char q8_lds_char;

__device__ __forceinline__ i32x4_t q8_srd(const void* base, int64_t bytes) {
  const uint64_t b = (uint64_t)base;
  i32x4_t r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)b);
  r[1] = __builtin_amdgcn_readfirstlane((int)((uint32_t)(b >> 32) & 0xffffu));
  r[2] = __builtin_amdgcn_readfirstlane((int)(uint32_t)(bytes < 0x7fffffff ? (bytes > 0 ? bytes : 0) : 0x7fffffff));
  r[3] = 0x00020000;
  asm volatile("s_nop 4" : "+s"(r));                // (a descriptor written by the vector unit is not for the next five states' memory access)
  return r;
}
// 64 lanes x 16 bytes from descriptor + voff + soff into LDS at lds_addr + 16 * lane; zeros from the descriptor's end on.  The
// compiler does not see it: the kernel waits with its own counts.
__device__ __forceinline__ void q8_dma(unsigned voff, i32x4_t srd, unsigned soff, unsigned lds_addr) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %4\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "v"(voff), "s"(srd), "s"(soff), "s"(lds_addr) : "memory");
}
template <int N>
__device__ __forceinline__ void q8_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void q8_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// the same once this wave's LDS reads have returned: what they read may be overwritten behind it
__device__ __forceinline__ void q8_barrier_after_reads() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  q8_barrier();
}

// Workgroup b runs on XCD b % 8: each XCD takes a run of neighbouring tiles, so that the tiles of one row of tiles read their common
// operand rows through one L2.
__device__ __forceinline__ int q8_tile(int tiles) {
  const int per = tiles / 8, more = tiles % 8, xcd = blockIdx.x % 8;
  return xcd * per + (xcd < more ? xcd : more) + blockIdx.x / 8;
}

template <typename T>
struct Q8Pair {
  typedef T type __attribute__((ext_vector_type(2), aligned(sizeof(T))));
};
// TM x TN outputs per workgroup of 4 waves (2 x 2), operands through LDS in steps of STEP bytes of K, NS steps in flight, one tile to
// a workgroup: its stores drain while the next one on the compute unit multiplies (a persistent workgroup would wait for them with
// its next operands: loads and stores return in one order).  LDS image: rows of STEP bytes, chunk of 16 bytes ^= row / 2 & 7 (128) or
// row / 4 & 3 (64), applied to the source address of the LDS-DMA and undone by the fragment reads: sixteen rows of one chunk fall into
// sixteen different groups of the 64 banks.  Weight row 2 i + j of a wave's 64-column block lies at image row 32 j + i: a lane then owns
// two neighbouring columns and stores them together.
// Bound by stores for short sums (4708 x 50021 x 192 to float32: 221 us, 4.3 TB/s) and for long ones by the loop, which waits at two
// workgroup barriers and for its LDS reads in every step: at 76800 x 1536 x 1536 (241 - 290 us, 1.4 POP/s) the matrix pipe is busy in 36 %
// of the cycles, at a clock of 1.86 GHz; fed from registers alone it reaches 2.9 POP/s.  The library's product to 32-bit integers takes
// 268 us there; 76800 x 1024 x 1024 132 (library 148), 76800 x 512 x 512 41 - 48 (56), 2048 x 2048 x 2048 17 (21).  Built and not kept:
// tiles of 256 x 256 by 8 waves, persistent with LDS-DMA (267 us) or one to a workgroup through registers, one or two steps ahead
// (272 - 308, 288), 128 x 256 and 256 x 128 by 4 waves (278 - 297): within a tenth on the largest shape, behind on the others.
template <typename Y, int TM, int TN, int STEP, int NS>
__global__ __launch_bounds__(256, 2) void int8_tile_kernel(Int8Args g, int tiles_m, int tiles_n, bool down) {
  constexpr int STAGE = (TM + TN) * STEP, CPR = STEP / 16, RP = 64 / CPR, SH = STEP == 128 ? 1 : 2;
  constexpr int QA = TM / (4 * RP), QB = TN / (4 * RP);      // DMA instructions per wave and operand, RP rows each
  constexpr int WM = TM / 2, WN = TN / 2, MI = WM / 32, NJ = WN / 64;
  extern __shared__ __attribute__((aligned(16))) int8_t smem[];
  const unsigned lds0 = (unsigned)(uintptr_t)(q8_lds_char*)smem;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1;
  const int fi = lane & 31, fh = lane >> 5;
  const int tile = q8_tile(gridDim.x);
  const int64_t m0 = (int64_t)(down ? tile % tiles_m : tile / tiles_n) * TM, n0 = (int64_t)(down ? tile / tiles_m : tile % tiles_n) * TN;
  const int64_t rows_a = g.m - m0 < TM ? g.m - m0 : TM, rows_b = g.n - n0 < TN ? g.n - n0 : TN;
  const i32x4_t sa = q8_srd(g.a + m0 * g.lda, rows_a * g.lda), sb = q8_srd(g.b + n0 * g.ldb, rows_b * g.ldb);
  const int tr = (int)(threadIdx.x < rows_a ? threadIdx.x : rows_a - 1), tc = (int)(threadIdx.x < rows_b ? threadIdx.x : rows_b - 1);
  const float in_sa = g.sa[m0 + tr], in_sb = g.sb[n0 + tc], in_bias = g.bias ? g.bias[n0 + tc] : 0.f;
  const int chunk = (lane % CPR) ^ (((wave * RP + lane / CPR) >> SH) & (CPR - 1));      // (4 * RP rows further the same)
  unsigned offa[QA], offb[QB];
#pragma unroll
  for (int q = 0; q < QA; ++q) offa[q] = (unsigned)((q * 4 + wave) * RP + lane / CPR) * (unsigned)g.lda + chunk * 16;
#pragma unroll
  for (int q = 0; q < QB; ++q) {
    const int p = (q * 4 + wave) * RP + lane / CPR;
    offb[q] = (unsigned)((p & ~63) + 2 * (p & 31) + ((p >> 5) & 1)) * (unsigned)g.ldb + chunk * 16;
  }
  const int steps = (g.k + STEP - 1) / STEP;
  auto request = [&](int t, int stage) {
    if (t >= steps) return;
    const unsigned at = lds0 + stage * STAGE, soff = t * STEP, none = t * STEP + chunk * 16 < g.k ? 0u : 0x80000000u;
#pragma unroll
    for (int q = 0; q < QA; ++q) q8_dma(offa[q] | none, sa, soff, __builtin_amdgcn_readfirstlane(at + (q * 4 + wave) * 1024));
#pragma unroll
    for (int q = 0; q < QB; ++q) q8_dma(offb[q] | none, sb, soff, __builtin_amdgcn_readfirstlane(at + TM * STEP + (q * 4 + wave) * 1024));
  };
  i32x16_t acc[MI][NJ][2] = {};
#pragma unroll
  for (int t = 0; t < NS; ++t) request(t, t);
  int foff[STEP / 32];
#pragma unroll
  for (int ks = 0; ks < STEP / 32; ++ks) foff[ks] = fi * STEP + (((2 * ks + fh) ^ ((fi >> SH) & (CPR - 1))) << 4);
  int stage = 0;
  for (int t = 0; t < steps; ++t) {
    if (t + NS <= steps) q8_wait<(NS - 1) * (QA + QB)>();      // step t has landed; the later ones stay in flight
    else q8_wait<0>();
    q8_barrier();
    const int8_t* st = smem + stage * STAGE;
    const int8_t *pa = st + wm * WM * STEP, *pb = st + TM * STEP + wn * WN * STEP;
#pragma unroll
    for (int ks = 0; ks < STEP / 32; ++ks) {
      i32x4_t af[MI], bf[NJ][2];
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) bf[j][h] = *reinterpret_cast<const i32x4_t*>(pb + (j * 64 + h * 32) * STEP + foff[ks]);
#pragma unroll
      for (int i = 0; i < MI; ++i) af[i] = *reinterpret_cast<const i32x4_t*>(pa + i * 32 * STEP + foff[ks]);
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) acc[i][j][h] = __builtin_amdgcn_mfma_i32_32x32x32_i8(af[i], bf[j][h], acc[i][j][h], 0, 0, 0);
    }
    q8_barrier_after_reads();                       // everybody has read this stage
    request(t + NS, stage);
    stage = stage + 1 == NS ? 0 : stage + 1;
  }
  // ---- epilogue: scales and bias of the tile through LDS (a load per output row would be waited for row by row)
  float* sc = reinterpret_cast<float*>(smem);       // [TM] token scales, [TN] channel scales, [TN] bias, a wave's word each: a far token scale
  static_assert(TM <= 128 && (TM + 2 * TN + 2) * 4 <= STAGE, "token scales come from the first two waves");
  if (threadIdx.x < TM) sc[threadIdx.x] = in_sa;
  if (threadIdx.x < 128) sc[TM + 2 * TN + wave] = __ballot(fabsf(in_sa) >= Q8_FAR) ? 1.f : 0.f;
  if (threadIdx.x < TN) {
    sc[TM + threadIdx.x] = in_sb;
    sc[TM + TN + threadIdx.x] = in_bias;
  }
  __syncthreads();
  const bool far = sc[TM + 2 * TN] + sc[TM + 2 * TN + 1] != 0.f;
  Y* y = reinterpret_cast<Y*>(g.y);
  auto put = [&](auto whole, auto far) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int c = wn * WN + j * 64 + 2 * fi;
      const int64_t col = n0 + c;
      const bool two = whole || col + 1 < g.n;
      if (!whole && col >= g.n) continue;
      const float s0 = sc[TM + c], s1 = sc[TM + c + 1], b0 = sc[TM + TN + c], b1 = sc[TM + TN + c + 1];
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int rw = wm * WM + i * 32 + (r & 3) + 8 * (r >> 2) + 4 * fh;
          const int64_t row = m0 + rw;
          if (!whole && row >= g.m) continue;
          const float s = sc[rw];
          const Y y0 = q8_out<Y, far>(acc[i][j][0][r], s, s0, b0), y1 = q8_out<Y, far>(acc[i][j][1][r], s, s1, b1);
          if (two) {
            typename Q8Pair<Y>::type v;
            v[0] = y0;
            v[1] = y1;
            *reinterpret_cast<typename Q8Pair<Y>::type*>(y + row * g.ldy + col) = v;
          } else {
            y[row * g.ldy + col] = y0;
          }
        }
    }
  };
  if (far) put(std::false_type{}, std::true_type{});
  else if (rows_a == TM && rows_b == TN) put(std::true_type{}, std::false_type{});
  else put(std::false_type{}, std::false_type{});
}

template <typename F>
int q8_by_type(int dtype, F f) {
  if (dtype == TN_DTYPE_F32) return f((float*)nullptr);
  if (dtype == TN_DTYPE_BF16) return f((__bf16*)nullptr);
  if (dtype == TN_DTYPE_F16) return f((_Float16*)nullptr);
  return TN_E_UNSUPPORTED;
}

constexpr int64_t Q8_GRID = (1 << 24) - 1;
constexpr int64_t Q8_FEW = 32;                     // rows of the kernel that makes their codes itself
constexpr int64_t Q8_FEW_LDS = 64 * 1024;          // ... where these fit
constexpr int Q8_TILE = 128;                       // rows and columns of a tile
constexpr int64_t Q8_PITCH = 0x7fffffff / Q8_TILE; // most bytes from row to row of its operands: a descriptor spans 2^31 - 1 bytes, offsets are 32 bits

int64_t q8_padded(int64_t k) { return (k + 63) / 64 * 64; }
bool q8_few(int64_t m, int64_t k) { return m <= Q8_FEW && m * (q8_padded(k) + 16) <= Q8_FEW_LDS; }

// a launch that may need more than 64 KB of LDS
template <typename K, typename... A>
int q8_launch(K kernel, dim3 grid, int threads, size_t lds, void* stream, A... args) {
  if (lds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return (int)e;
  }
  hipLaunchKernelGGL(kernel, grid, dim3(threads), lds, (hipStream_t)stream, args...);
  return (int)hipGetLastError();
}

template <typename X, typename Y>
int q8_few_rows(const FewArgs& f, void* stream) {
  const int64_t tiles = (f.g.n + 31) / 32;
  const size_t base = (size_t)f.g.m * (f.g.k + 16) + 32 * 4;
  auto go = [&](auto nw, auto ks) {
    constexpr int NW = decltype(nw)::value, KS = decltype(ks)::value;
    const int64_t groups = (tiles + NW / KS - 1) / (NW / KS);
    return q8_launch(int8_few_rows_kernel<X, Y, NW, KS>, dim3((unsigned)std::min<int64_t>(groups, 2048)), NW * 64,
                     base + (KS > 1 ? (size_t)NW * 4096 : 0), stream, f);
  };
  // 32 channels to a workgroup while that leaves compute units idle, and more waves along K the fewer there are
  if (tiles <= 64 && f.g.k >= 512) return go(std::integral_constant<int, 16>{}, std::integral_constant<int, 16>{});
  if (tiles <= 1024 && f.g.k >= 128) return go(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{});
  return go(std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{});
}

template <typename Y>
int q8_tiles(const Int8Args& g, void* stream) {
  if (g.lda > Q8_PITCH || g.ldb > Q8_PITCH) return TN_E_UNSUPPORTED;
  auto go = [&](auto step, bool down) -> int {
    constexpr int T = Q8_TILE, STEP = decltype(step)::value, NS = 2;
    const int64_t a = (g.m + T - 1) / T, b = (g.n + T - 1) / T;
    if (b > Q8_GRID || a > Q8_GRID / b) return TN_E_UNSUPPORTED;
    return q8_launch(int8_tile_kernel<Y, T, T, STEP, NS>, dim3((unsigned)(a * b)), 256, (size_t)NS * 2 * T * STEP, stream, g, (int)a, (int)b, down);
  };
  // Up to 8 rows of tiles one after another share a column of weights (read once) before the next column; with more of them the
  // tiles run along the rows.  Rows / columns first: 250 x 100003 x 192 36.5 / 30.0 us, 1000 x 50000 x 192 52 / 41, but 4708 x 50021 x
  // 192 173 / 214 and 76800 x 1536 x 1536 291 / 314 (bf16 outputs).  Short sums of few rows are bound by their stores: steps of 64 bytes
  // leave room for twice the workgroups (250 x 100003 x 192 21.3 us, 1000 x 50000 x 192 30.1); everything else takes whole lines of
  // 128 (4708 x 50021 x 192 173 against 199 us, 76800 x 1536 x 1536 291 against 328, 2048 x 2048 x 2048 17 against 19).
  const bool down = g.m <= 8 * Q8_TILE;
  return down && g.k <= 512 ? go(std::integral_constant<int, 64>{}, down) : go(std::integral_constant<int, 128>{}, down);
}

bool q8_operands_ok(int64_t m, int64_t n, int64_t k, const void* b, const float* b_scales, int64_t ldb, const void* y, int64_t ldy) {
  if (m < 0 || n < 0 || k < 1 || ldb % 64 || ldb < k || ldy < n) return false;
  return !m || !n || (b && b_scales && y && (uintptr_t)b % 16 == 0);
}

}  // namespace

extern "C" int tn_int8_quantize_rows(const void* x, int32_t dtype, int64_t rows, int64_t cols, int64_t ldx, void* codes, int64_t ld_codes,
                                     float* scales, void* stream) {
  if (rows < 0 || cols < 1 || ldx < 0 || ld_codes % 64 || ld_codes < cols || (rows > 0 && (!x || !codes || !scales || (uintptr_t)codes % 16))) return TN_E_BADARG;
  if (cols > TN_INT8_MAX_K || dtype < TN_DTYPE_F32 || dtype > TN_DTYPE_F16) return TN_E_UNSUPPORTED;
  if (!rows) return 0;
  return q8_by_type(dtype, [&](auto* kind) -> int {
    using T = std::remove_pointer_t<decltype(kind)>;
    auto go = [&](auto group, auto passes) {
      constexpr int GROUP = decltype(group)::value, PASSES = decltype(passes)::value;
      const int64_t per = 4 * (64 / GROUP);
      return q8_launch(quantize_rows_kernel<T, GROUP, PASSES>, dim3((unsigned)std::min<int64_t>((rows + per - 1) / per, 1 << 20)), 256, 0, stream, (const T*)x,
                       rows, (int)cols, ldx, (int8_t*)codes, ld_codes, (int)q8_padded(cols), scales);
    };
    using std::integral_constant;
    // as few lanes as hold a row in one pass, so that short rows leave none idle; then more passes of a whole wave
    if (cols <= 64) return go(integral_constant<int, 8>{}, integral_constant<int, 1>{});
    if (cols <= 128) return go(integral_constant<int, 16>{}, integral_constant<int, 1>{});
    if (cols <= 256) return go(integral_constant<int, 32>{}, integral_constant<int, 1>{});
    if (cols <= 512) return go(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    if (cols <= 1024) return go(integral_constant<int, 64>{}, integral_constant<int, 2>{});
    if (cols <= 1536) return go(integral_constant<int, 64>{}, integral_constant<int, 3>{});
    if (cols <= 2048) return go(integral_constant<int, 64>{}, integral_constant<int, 4>{});
    if (cols <= 4096) return go(integral_constant<int, 64>{}, integral_constant<int, 8>{});
    return go(integral_constant<int, 64>{}, integral_constant<int, 0>{});
  });
}

extern "C" int tn_int8_matmul(const void* a, const float* a_scales, int64_t lda, const void* b, const float* b_scales, int64_t ldb,
                              const float* bias, void* y, int32_t y_dtype, int64_t ldy, int64_t m, int64_t n, int64_t k, void* stream) {
  if (!q8_operands_ok(m, n, k, b, b_scales, ldb, y, ldy) || lda % 64 || lda < k || (m > 0 && n > 0 && (!a || !a_scales || (uintptr_t)a % 16))) return TN_E_BADARG;
  if (k > TN_INT8_MAX_K || y_dtype < TN_DTYPE_F32 || y_dtype > TN_DTYPE_F16) return TN_E_UNSUPPORTED;
  if (!m || !n) return 0;
  const Int8Args g = {(const int8_t*)a, (const int8_t*)b, a_scales, b_scales, bias, y, lda, ldb, ldy, m, n, (int)q8_padded(k)};
  return q8_by_type(y_dtype, [&](auto* kind) -> int {
    using Y = std::remove_pointer_t<decltype(kind)>;
    if (q8_few(m, k)) return q8_few_rows<int8_t, Y>(FewArgs{a, g, lda, (int)k}, stream);
    return q8_tiles<Y>(g, stream);
  });
}

extern "C" int64_t tn_int8_linear_workspace(int64_t m, int64_t k) {
  if (m < 0 || k < 1 || k > TN_INT8_MAX_K) return TN_E_BADARG;
  return q8_few(m, k) ? 0 : m * q8_padded(k) + (m + 3) / 4 * 16;
}

extern "C" int tn_int8_linear(const void* x, int32_t x_dtype, int64_t ldx, const void* b, const float* b_scales, int64_t ldb, const float* bias,
                              void* y, int32_t y_dtype, int64_t ldy, int64_t m, int64_t n, int64_t k, void* workspace, int64_t workspace_bytes,
                              void* stream) {
  if (!q8_operands_ok(m, n, k, b, b_scales, ldb, y, ldy) || ldx < 0 || (m > 0 && n > 0 && !x)) return TN_E_BADARG;
  if (k > TN_INT8_MAX_K || y_dtype < TN_DTYPE_F32 || y_dtype > TN_DTYPE_F16 || x_dtype < TN_DTYPE_F32 || x_dtype > TN_DTYPE_F16) return TN_E_UNSUPPORTED;
  if (!m || !n) return 0;
  if (q8_few(m, k)) {
    const Int8Args g = {nullptr, (const int8_t*)b, nullptr, b_scales, bias, y, 0, ldb, ldy, m, n, (int)q8_padded(k)};
    return q8_by_type(x_dtype, [&](auto* kx) -> int {
      using X = std::remove_pointer_t<decltype(kx)>;
      return q8_by_type(y_dtype, [&](auto* ky) -> int { return q8_few_rows<X, std::remove_pointer_t<decltype(ky)>>(FewArgs{x, g, ldx, (int)k}, stream); });
    });
  }
  if (ldb > Q8_PITCH) return TN_E_UNSUPPORTED;
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < tn_int8_linear_workspace(m, k)) return TN_E_BADARG;
  const int64_t ld = q8_padded(k);
  float* scales = reinterpret_cast<float*>((char*)workspace + m * ld);
  if (const int rc = tn_int8_quantize_rows(x, x_dtype, m, k, ldx, workspace, ld, scales, stream)) return rc;
  return tn_int8_matmul(workspace, scales, ld, b, b_scales, ldb, bias, y, y_dtype, ldy, m, n, k, stream);
}
