// Layer norm of rows of any width, with its backward pass:
//   y = (x - mean) rstd w + b;   with xh = (x - mean) rstd and g = dy w:
//   dx = rstd (g - mean(g) - xh mean(g xh)) (+ d_sum),   dw = sum over rows of dy xh,   db = sum over rows of dy.
// Optionally x = rounded(a + residual), written as it is normalised.
//
// Bound by memory: a row is read once and stays in registers (16 bytes a load, a group of lanes per row wide enough for its
// chunks), so that the mean and then the centred sum of squares cost no second read; statistics and sums are fp32.  The
// backward pass keeps the columns' sums of the rows that a group walks in registers too, joins them per block in LDS and
// writes one line per block; a second launch adds the lines in order, so the weights' gradients do not depend on timing.
#include "common.h"
#include "../../include/ocean_hip.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// E values of T as floats <-> one load / store of E * sizeof(T) bytes at any alignment
template <typename T, int E> __device__ __forceinline__ void load_vec(const T* p, float (&f)[E]) {
  T x[E];
  __builtin_memcpy(x, p, sizeof(x));
#pragma unroll
  for (int e = 0; e < E; ++e) f[e] = (float)x[e];
}
template <typename T, int E> __device__ __forceinline__ void store_vec(T* p, const float (&f)[E]) {
  T x[E];
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = (T)f[e];
  __builtin_memcpy(p, x, sizeof(x));
}
// elements e0.. of a row of W, zeros past its end
template <typename T, int E> __device__ __forceinline__ void load_part(const T* row, int e0, int W, float (&f)[E]) {
  if (e0 + E <= W) load_vec<T, E>(row + e0, f);
  else
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = e0 + e < W ? (float)row[e0 + e] : 0.f;
}
template <typename T, int E> __device__ __forceinline__ void store_part(T* row, int e0, int W, const float (&f)[E]) {
  if (e0 + E <= W) store_vec<T, E>(row + e0, f);
  else
#pragma unroll
    for (int e = 0; e < E; ++e) if (e0 + e < W) row[e0 + e] = (T)f[e];
}

// the same unconverted
template <typename T, int E> __device__ __forceinline__ void raw_part(const T* row, int e0, int W, T (&x)[E]) {
  if (e0 + E <= W) __builtin_memcpy(x, row + e0, E * sizeof(T));
  else
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = e0 + e < W ? row[e0 + e] : (T)0.f;
}

// sum over the LPR threads of a row's group; LPR <= 64: lanes of a wave, else the whole block (red: one float a wave and value)
template <int LPR, int N> __device__ __forceinline__ void group_sum(float (&v)[N], float* red) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int o = (LPR < 64 ? LPR : 64) / 2; o > 0; o >>= 1) v[n] += __shfl_xor(v[n], o, 64);
  if (LPR > 64) {
    constexpr int kW = LPR / 64;
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int n = 0; n < N; ++n) red[n * kW + (threadIdx.x >> 6)] = v[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < kW; ++w) t += red[n * kW + w];
      v[n] = t;
    }
  }
}

struct LnP {
  const void* x; long ldx; const void* res; long ldr;
  const float* w; const float* b;
  void* y; void* sum; float* stats;              // y, sum: dense rows
  long rows; int W; float eps;
  long row0;                                     // forward: first row of the launch
  const void* dy; long lddy; const void* dsum; long ldds; void* dx; float* part; int blocks;
};

template <int LPR> struct Block { static constexpr int kThreads = LPR > 256 ? LPR : 256; };

// 4099 rows of 8192 fp32: 52 us = 5.2 TB/s, what a large copy reaches; 16384 of 768 bf16 with a residual: 21 us (101 MB, 4.8 TB/s).
template <typename T, int E, int LPR, int NC, bool RES> __global__ __launch_bounds__(Block<LPR>::kThreads) void fwd_kernel(const LnP p) {
  constexpr int kT = Block<LPR>::kThreads;
  __shared__ float red[LPR > 64 ? LPR / 64 : 1];
  const int lane = threadIdx.x % LPR;
  const long row = p.row0 + (long)blockIdx.x * (kT / LPR) + threadIdx.x / LPR;
  if (row >= p.rows) return;                     // LPR > 64: the block has one row (or kT == LPR rows apart), all threads agree
  float f[NC][E];
  float s[1] = {0.f};
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int e0 = (lane + n * LPR) * E;
    load_part<T, E>((const T*)p.x + row * p.ldx, e0, p.W, f[n]);
    if (RES) {
      float r[E];
      load_part<T, E>((const T*)p.res + row * p.ldr, e0, p.W, r);
#pragma unroll
      for (int e = 0; e < E; ++e) f[n][e] = (float)(T)(f[n][e] + r[e]);
      store_part<T, E>((T*)p.sum + row * p.W, e0, p.W, f[n]);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) s[0] += f[n][e];
  }
  group_sum<LPR, 1>(s, red);
  const float mean = s[0] / (float)p.W;
  s[0] = 0.f;
#pragma unroll
  for (int n = 0; n < NC; ++n)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      f[n][e] -= mean;
      if ((lane + n * LPR) * E + e < p.W) s[0] = fmaf(f[n][e], f[n][e], s[0]);
    }
  group_sum<LPR, 1>(s, red);
  const float rstd = 1.f / sqrtf(s[0] / (float)p.W + p.eps);
  if (p.stats && lane == 0) { p.stats[2 * row] = mean; p.stats[2 * row + 1] = rstd; }
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int e0 = (lane + n * LPR) * E;
    float w[E], b[E];
    if (p.w) load_part<float, E>(p.w, e0, p.W, w);
    if (p.b) load_part<float, E>(p.b, e0, p.W, b);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float v = f[n][e] * rstd;
      if (p.w) v *= w[e];
      if (p.b) v += b[e];
      f[n][e] = v;
    }
    store_part<T, E>((T*)p.y + row * p.W, e0, p.W, f[n]);
  }
}

// rows wider than a block's registers: the row is read three times, the second and third from cache
template <typename T, bool RES> __global__ __launch_bounds__(1024) void fwd_wide_kernel(const LnP p) {
  __shared__ float red[16];
  const long row = p.row0 + blockIdx.x;
  const T* x = (const T*)p.x + row * p.ldx;
  float s[1] = {0.f};
  for (long c = threadIdx.x; c < p.W; c += 1024) {
    float v = (float)x[c];
    if (RES) { v = (float)(T)(v + (float)((const T*)p.res)[row * p.ldr + c]); ((T*)p.sum)[row * p.W + c] = (T)v; }
    s[0] += v;
  }
  const T* from = RES ? (const T*)p.sum + row * p.W : x;   // each thread reads back what it wrote itself
  group_sum<1024, 1>(s, red);
  const float mean = s[0] / (float)p.W;
  s[0] = 0.f;
  for (long c = threadIdx.x; c < p.W; c += 1024) { const float v = (float)from[c] - mean; s[0] = fmaf(v, v, s[0]); }
  group_sum<1024, 1>(s, red);
  const float rstd = 1.f / sqrtf(s[0] / (float)p.W + p.eps);
  if (p.stats && threadIdx.x == 0) { p.stats[2 * row] = mean; p.stats[2 * row + 1] = rstd; }
  for (long c = threadIdx.x; c < p.W; c += 1024) {
    float v = ((float)from[c] - mean) * rstd;
    if (p.w) v *= p.w[c];
    if (p.b) v += p.b[c];
    ((T*)p.y)[row * p.W + c] = (T)v;
  }
}

// Rows that take a whole block: the next row is loaded before this one's sums, so that memory works while the block's waves meet
// (4099 rows of 8192 fp32: 106 us without, 84 with, 4.8 TB/s; 16384 of 768 bf16, one gradient more: 27 us, 3.7 TB/s).
template <typename T, int E, int LPR, int NC> __global__ __launch_bounds__(Block<LPR>::kThreads) void bwd_kernel(const LnP p) {
  constexpr int kT = Block<LPR>::kThreads, kG = kT / LPR;
  constexpr bool kNext = LPR >= 256;
  __shared__ float red[LPR > 64 ? 2 * LPR / 64 : 1];
  __shared__ float join[kG > 1 ? 2 * kG * LPR * NC * E : 1];
  const int lane = threadIdx.x % LPR, grp = threadIdx.x / LPR;
  float w[NC][E], sw[NC][E], sb[NC][E];
#pragma unroll
  for (int n = 0; n < NC; ++n) {
#pragma unroll
    for (int e = 0; e < E; ++e) { w[n][e] = 1.f; sw[n][e] = 0.f; sb[n][e] = 0.f; }
    if (p.w) load_part<float, E>(p.w, (lane + n * LPR) * E, p.W, w[n]);
  }
  const float inv_w = 1.f / (float)p.W;
  const long step = (long)gridDim.x * kG;
  T nx[NC][E], ng[NC][E];
  const auto fetch = [&](long row) {
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int e0 = (lane + n * LPR) * E;
      raw_part<T, E>((const T*)p.x + row * p.ldx, e0, p.W, nx[n]);
      raw_part<T, E>((const T*)p.dy + row * p.lddy, e0, p.W, ng[n]);
    }
  };
  long row = (long)blockIdx.x * kG + grp;
  if (kNext && row < p.rows) fetch(row);
  for (; row < p.rows; row += step) {
    const float mean = p.stats[2 * row], rstd = p.stats[2 * row + 1];
    if (!kNext) fetch(row);
    float xh[NC][E], g[NC][E], s[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int e0 = (lane + n * LPR) * E;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        xh[n][e] = e0 + e < p.W ? ((float)nx[n][e] - mean) * rstd : 0.f;
        const float d = (float)ng[n][e];
        sw[n][e] = fmaf(d, xh[n][e], sw[n][e]);
        sb[n][e] += d;
        g[n][e] = d * w[n][e];
        s[0] += g[n][e];
        s[1] = fmaf(g[n][e], xh[n][e], s[1]);
      }
    }
    if (kNext && row + step < p.rows) fetch(row + step);
    group_sum<LPR, 2>(s, red);
    const float mg = s[0] * inv_w, mgx = s[1] * inv_w;
    if (p.dx) {
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        const int e0 = (lane + n * LPR) * E;
        float d[E];
        if (p.dsum) load_part<T, E>((const T*)p.dsum + row * p.ldds, e0, p.W, d);
#pragma unroll
        for (int e = 0; e < E; ++e) g[n][e] = fmaf(rstd, g[n][e] - mg - xh[n][e] * mgx, p.dsum ? d[e] : 0.f);
        store_part<T, E>((T*)p.dx + row * p.W, e0, p.W, g[n]);
      }
    }
  }
  if (!p.part) return;
  float* pw = p.part + (long)blockIdx.x * 2 * p.W;
  if (kG > 1) {
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = (lane + n * LPR) * E + e;
        join[grp * LPR * NC * E + c] = sw[n][e];
        join[(kG + grp) * LPR * NC * E + c] = sb[n][e];
      }
    __syncthreads();
    for (int c = threadIdx.x; c < p.W; c += kT) {
      float a = 0.f, b = 0.f;
#pragma unroll
      for (int q = 0; q < kG; ++q) { a += join[q * LPR * NC * E + c]; b += join[(kG + q) * LPR * NC * E + c]; }
      pw[c] = a;
      pw[p.W + c] = b;
    }
  } else {
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      store_part<float, E>(pw, (lane + n * LPR) * E, p.W, sw[n]);
      store_part<float, E>(pw + p.W, (lane + n * LPR) * E, p.W, sb[n]);
    }
  }
}

// wide rows: the columns' sums live in the block's line of the workspace, which only this block writes.  Single values a load, and a
// read and a write of both sums for every row: 2048 rows of 16384 fp32 take 321 us, 1024 of 32768 336 us, 2048 of 32768 bf16 568 us,
// where x and dy read twice and dx written would be 131 us at a large copy's rate.
template <typename T> __global__ __launch_bounds__(1024) void bwd_wide_kernel(const LnP p) {
  __shared__ float red[32];
  float* pw = p.part ? p.part + (long)blockIdx.x * 2 * p.W : nullptr;
  if (pw) for (long c = threadIdx.x; c < 2L * p.W; c += 1024) pw[c] = 0.f;
  __syncthreads();
  for (long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const float mean = p.stats[2 * row], rstd = p.stats[2 * row + 1];
    const T* x = (const T*)p.x + row * p.ldx;
    const T* dy = (const T*)p.dy + row * p.lddy;
    float s[2] = {0.f, 0.f};
    for (long c = threadIdx.x; c < p.W; c += 1024) {
      const float xh = ((float)x[c] - mean) * rstd, d = (float)dy[c], g = p.w ? d * p.w[c] : d;
      s[0] += g;
      s[1] = fmaf(g, xh, s[1]);
      if (pw) { pw[c] = fmaf(d, xh, pw[c]); pw[p.W + c] += d; }
    }
    group_sum<1024, 2>(s, red);
    const float mg = s[0] / (float)p.W, mgx = s[1] / (float)p.W;
    if (p.dx)
      for (long c = threadIdx.x; c < p.W; c += 1024) {
        const float xh = ((float)x[c] - mean) * rstd, d = (float)dy[c], g = p.w ? d * p.w[c] : d;
        ((T*)p.dx)[row * p.W + c] = (T)fmaf(rstd, g - mg - xh * mgx, p.dsum ? (float)((const T*)p.dsum)[row * p.ldds + c] : 0.f);
      }
  }
}

// dw, db from the blocks' lines: 32 columns a block, 32 threads share a column's lines and meet in LDS
__global__ __launch_bounds__(1024) void join_kernel(const float* __restrict__ part, float* __restrict__ dw, float* __restrict__ db, int W, int lines) {
  __shared__ float red[32][33];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
  const long n = 2L * W, c = (long)blockIdx.x * 32 + cx;
  float t = 0.f;
  if (c < n) {
#pragma unroll 8
    for (int l = ry; l < lines; l += 32) t += part[l * n + c];
  }
  red[ry][cx] = t;
  __syncthreads();
  if (ry == 0 && c < n) {
    float a = 0.f;
#pragma unroll
    for (int q = 0; q < 32; ++q) a += red[q][cx];
    float* out = c < W ? dw : db;
    if (out) out[c < W ? c : c - W] = a;
  }
}

// Lanes per row and 16-byte chunks per lane, by the chunks of a row: a wave while its registers hold the row, then a block.  The
// backward kernel holds five values of every column (weight, both sums, xh, g), so it takes two chunks a lane.
#define LN_PICK_FWD(CALL)                              \
  do {                                                 \
    if (chunks <= 8) return CALL(8, 1);                \
    if (chunks <= 16) return CALL(16, 1);              \
    if (chunks <= 32) return CALL(32, 1);              \
    if (chunks <= 64) return CALL(64, 1);              \
    if (chunks <= 128) return CALL(64, 2);             \
    if (chunks <= 256) return CALL(64, 4);             \
    if (chunks <= 512) return CALL(256, 2);            \
    if (chunks <= 1024) return CALL(256, 4);           \
    if (chunks <= 2048) return CALL(512, 4);           \
    if (chunks <= 4096) return CALL(1024, 4);          \
  } while (0)
#define LN_PICK_BWD(CALL)                              \
  do {                                                 \
    if (chunks <= 8) return CALL(8, 1);                \
    if (chunks <= 16) return CALL(16, 1);              \
    if (chunks <= 32) return CALL(32, 1);              \
    if (chunks <= 64) return CALL(64, 1);              \
    if (chunks <= 128) return CALL(64, 2);             \
    if (chunks <= 512) return CALL(256, 2);            \
    if (chunks <= 1024) return CALL(512, 2);           \
    if (chunks <= 2048) return CALL(1024, 2);          \
  } while (0)

// A grid holds fewer than 2^32 threads (more wrap around, with no error, and leave rows out): many short rows take several launches.
constexpr long kMaxBlocks = 1L << 21;
template <typename K> int launch_rows(K kernel, const LnP& p, int rows_a_block, int threads, hipStream_t s) {
  LnP q = p;
  for (q.row0 = 0; q.row0 < p.rows; q.row0 += kMaxBlocks * rows_a_block) {
    const long blocks = (p.rows - q.row0 + rows_a_block - 1) / rows_a_block;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(blocks < kMaxBlocks ? blocks : kMaxBlocks)), dim3(threads), 0, s, q);
    OCEAN_LAUNCH_CHECK();
  }
  return OCEAN_OK;
}
template <typename T, int E, int LPR, int NC> int fwd_launch(const LnP& p, hipStream_t s) {
  constexpr int kT = Block<LPR>::kThreads;
  return launch_rows(p.res ? fwd_kernel<T, E, LPR, NC, true> : fwd_kernel<T, E, LPR, NC, false>, p, kT / LPR, kT, s);
}
template <typename T> int fwd_pick(const LnP& p, hipStream_t s) {
  constexpr int E = 16 / sizeof(T);
  const long chunks = (p.W + E - 1) / E;
#define LN_CALL(LPR, NC) fwd_launch<T, E, LPR, NC>(p, s)
  LN_PICK_FWD(LN_CALL);
#undef LN_CALL
  return launch_rows(p.res ? fwd_wide_kernel<T, true> : fwd_wide_kernel<T, false>, p, 1, 1024, s);
}
template <typename T, int E, int LPR, int NC> int bwd_launch(const LnP& p, hipStream_t s) {
  hipLaunchKernelGGL((bwd_kernel<T, E, LPR, NC>), dim3(p.blocks), dim3(Block<LPR>::kThreads), 0, s, p);
  OCEAN_LAUNCH_CHECK();
  return OCEAN_OK;
}
template <typename T> int bwd_pick(const LnP& p, hipStream_t s) {
  constexpr int E = 16 / sizeof(T);
  const long chunks = (p.W + E - 1) / E;
#define LN_CALL(LPR, NC) bwd_launch<T, E, LPR, NC>(p, s)
  LN_PICK_BWD(LN_CALL);
#undef LN_CALL
  hipLaunchKernelGGL((bwd_wide_kernel<T>), dim3(p.blocks), dim3(1024), 0, s, p);
  OCEAN_LAUNCH_CHECK();
  return OCEAN_OK;
}

// blocks (lines of the workspace) of the backward pass: what the chip holds at a time, the rows evenly among them
int bwd_blocks(long rows, int W, int type) {
  const int E = type == OCEAN_F32 ? 4 : 8;
  const long chunks = (W + E - 1) / E;
  const long groups = chunks <= 8 ? 32 : chunks <= 16 ? 16 : chunks <= 32 ? 8 : chunks <= 128 ? 4 : 1;   // rows of a block at a time
  const long fit = (1L << 24) / W, most = chunks <= 512 ? 768 : chunks <= 1024 ? 512 : fit > 256 ? 256 : fit > 16 ? fit : 16;
  const long sets = (rows + groups - 1) / groups, per = (sets + most - 1) / most;
  return (int)((sets + per - 1) / per);
}

int ln_check(const ocean_layer_norm_shape* s) {
  if (!s) return OCEAN_ERR_NULL;
  if (s->rows <= 0 || s->width <= 0 || s->x_stride < s->width || (s->dtype != OCEAN_F32 && s->dtype != OCEAN_BF16 && s->dtype != OCEAN_F16)) return OCEAN_ERR_BAD_SHAPE;
  if (s->rows > 0x7fffffffL || s->width > (1 << 24)) return OCEAN_ERR_UNSUPPORTED;
  return OCEAN_OK;
}

}  // namespace

extern "C" {

int ocean_layer_norm_fwd(const ocean_layer_norm_shape* s, const void* x, const void* residual, const float* weight, const float* bias, void* y,
                         void* sum, float* stats, void* stream) {
  OCEAN_TRY(ln_check(s));
  if (!x || !y || (residual && !sum)) return OCEAN_ERR_NULL;
  if (residual && s->residual_stride < s->width) return OCEAN_ERR_BAD_SHAPE;
  LnP p = {};
  p.x = x; p.ldx = s->x_stride; p.res = residual; p.ldr = s->residual_stride; p.w = weight; p.b = bias; p.y = y; p.sum = sum; p.stats = stats;
  p.rows = s->rows; p.W = s->width; p.eps = s->eps;
  hipStream_t st = (hipStream_t)stream;
  return s->dtype == OCEAN_F32 ? fwd_pick<float>(p, st) : s->dtype == OCEAN_BF16 ? fwd_pick<__bf16>(p, st) : fwd_pick<_Float16>(p, st);
}

size_t ocean_layer_norm_bwd_workspace(const ocean_layer_norm_shape* s) {
  return ln_check(s) == OCEAN_OK ? (size_t)bwd_blocks(s->rows, s->width, s->dtype) * 2 * s->width : 0;
}

int ocean_layer_norm_bwd(const ocean_layer_norm_shape* s, const void* x, const float* stats, const float* weight, const void* dy, const void* d_sum,
                         float* ws, size_t ws_floats, void* dx, float* dweight, float* dbias, void* stream) {
  OCEAN_TRY(ln_check(s));
  if (!x || !stats || !dy) return OCEAN_ERR_NULL;
  if (s->dy_stride < s->width || (d_sum && s->dsum_stride < s->width)) return OCEAN_ERR_BAD_SHAPE;
  const bool sums = dweight || dbias;
  if (sums && !ws) return OCEAN_ERR_NULL;
  if (sums && ws_floats < ocean_layer_norm_bwd_workspace(s)) return OCEAN_ERR_WORKSPACE;
  LnP p = {};
  p.x = x; p.ldx = s->x_stride; p.w = weight; p.stats = const_cast<float*>(stats); p.rows = s->rows; p.W = s->width; p.eps = s->eps;
  p.dy = dy; p.lddy = s->dy_stride; p.dsum = d_sum; p.ldds = s->dsum_stride; p.dx = dx; p.part = sums ? ws : nullptr;
  p.blocks = bwd_blocks(s->rows, s->width, s->dtype);
  hipStream_t st = (hipStream_t)stream;
  OCEAN_TRY(s->dtype == OCEAN_F32 ? bwd_pick<float>(p, st) : s->dtype == OCEAN_BF16 ? bwd_pick<__bf16>(p, st) : bwd_pick<_Float16>(p, st));
  if (sums) {
    hipLaunchKernelGGL(join_kernel, dim3((unsigned)((2L * p.W + 31) / 32)), dim3(1024), 0, st, ws, dweight, dbias, p.W, p.blocks);
    OCEAN_LAUNCH_CHECK();
  }
  return OCEAN_OK;
}

}  // extern "C"
