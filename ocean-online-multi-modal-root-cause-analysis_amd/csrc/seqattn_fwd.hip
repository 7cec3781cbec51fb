// Forward pass of attention without stored weights (seqattn.h): one pass over the keys with a running maximum and sum per row.
#include "seqattn.h"

namespace seqattn {
namespace {

constexpr int kRows = 128;           // queries of a block: four waves, 32 each

// running softmax state of one row, kept by both lanes that hold it (l: this lane's share of the sum)
struct RowState { float m, l; };

// Scores in, probabilities out (2^(t - m)); returns the factor that the accumulators take.  `mult` turns a score into its
// exponent t.  The maximum is only moved when it grows by more than 8 (a factor of 256, exact in fp32 sums): the factor is 1
// for almost every tile, and the accumulators need not be touched.
template <int N> __device__ __forceinline__ float softmax_step(f32x16 (&s)[N], float mult, RowState& st) {
  float mx = s[0][0];
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[n][r]);
  mx = other_half_max(mx) * mult;
  float f = 1.f;
  if (mx > st.m + 8.f || st.m == -INFINITY) {
    f = st.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st.m - mx);
    st.m = mx;
  }
  const float m = st.m == -INFINITY ? 0.f : st.m;
  float sum = 0.f;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float e = __builtin_amdgcn_exp2f(fmaf(s[n][r], mult, -m));
      s[n][r] = e;
      sum += e;
    }
  st.l = st.l * f + sum;
  return f;
}

// adds the bias and takes out the places that are not allowed, for keys j0..j0+31 and this lane's query
template <bool BIAS, bool MASK> __device__ __forceinline__ void adjust(const Params& p, f32x16& s, float mult, int j0, int pos, int pos0, int keys,
                                                                        const uint8_t* mrow, const float* lut, bool edge, int lane) {
  const int h4 = 4 * (lane >> 5);
  if (BIAS) {
    const f32x16 bias = block_bias<1>(p, lut, j0 + h4 - pos, j0 - pos0);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], mult, bias[r]);
  }
  if (MASK || edge) {
    const int end = (p.causal ? min(keys, pos + 1) : keys) - j0 - h4;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      uint32_t ok = 15u;
      if (MASK) ok = mrow ? mask4(p, mrow, j0 + 8 * g + h4, keys) : 15u;
#pragma unroll
      for (int e = 0; e < 4; ++e) if (8 * g + e >= end || (MASK && !((ok >> e) & 1u))) s[4 * g + e] = -INFINITY;
    }
  }
}

template <typename T, int D> struct FwdTile { static constexpr int kKeys = key_tile(sizeof(T) == 2); };

// joins a query tile's parts: a block takes a wave's 32 rows, its four waves the pieces in turn
template <typename T, int D> __global__ __launch_bounds__(256) void fwd_rows_join_kernel(const Params p) {
  const int unit = blockIdx.x >> 2, w = blockIdx.x & 3, lane = threadIdx.x & 63, r = lane & 31;
  const int tile = unit % p.q_tiles, bh = unit / p.q_tiles, b = bh / p.H, head = bh % p.H, i = tile * kRows + 32 * w + r;
  const int tiles = key_tiles<FwdTile<T, D>::kKeys>(p, tile, keys_of(p, b), start_of(p, b));
  if (tiles <= p.part_tiles || i >= p.Lq) return;
  const int parts = (tiles + p.part_tiles - 1) / p.part_tiles;
  const float* ml = p.part_ml + (long)unit * p.parts * 256 + 64 * w + r;
  float m = -INFINITY, l = 0.f;
  for (int s = 0; s < parts; ++s) m = fmaxf(m, ml[s * 256]);
  const float mref = m == -INFINITY ? 0.f : m;
  for (int s = 0; s < parts; ++s) l += __builtin_amdgcn_exp2f(ml[s * 256] - mref) * ml[s * 256 + 32];
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  const float* from = p.part_o + ((long)unit * p.parts * 4 + w) * 32 * D + lane * 4;
  T* out = (T*)p.o.p + b * p.o.b + head * p.o.h + (long)i * p.o.l;
  for (int n = threadIdx.x >> 6; n < D / 8; n += 4) {
    f32x4 t = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < parts; ++s) t += *reinterpret_cast<const f32x4*>(from + (long)s * 4 * 32 * D + n * 256) * __builtin_amdgcn_exp2f(ml[s * 256] - mref);
    store4<T>(out, part_feature(n, lane), p.d, t[0] * inv, t[1] * inv, t[2] * inv, t[3] * inv);
  }
  if (p.lse && threadIdx.x < 32) p.lse[((long)b * p.H + head) * p.Lq + i] = l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
}

// One block a query tile: the wave's 32 queries stay in registers as the right operand, keys and values pass through two LDS buffers,
// the next tile loading while this one is used.  Bound in bf16 by the turns of two waves a SIMD between matrix cores (busy 0.40 of
// the cycles), the softmax's vector instructions (0.42) and LDS (0.40, half of it bank conflicts).  Causal 16 heads (4 of keys) x 8192 x
// 128 bf16: 285 to 330 us (with the clock), 0.96 to 0.83 PFLOP/s of the pairs' 4 d, of 1.21 that a large product reaches; 2 x 16 heads x
// 4096: 171 us.  8 x 8 heads x 512 x 96 fp32, ragged: 67 us; short samples leave 1.07 waves a SIMD, which spend 0.69 of their cycles
// waiting for their turn, most of it for their own last matrix instruction (matrix cores busy 0.43).
template <typename T, int D, bool BIAS, bool MASK> __global__ __launch_bounds__(256, D * sizeof(T) > (MASK ? 128 : 256) ? 1 : 2) void fwd_rows_kernel(const Params p) {
  typedef Tile<T, D> TL;
  constexpr int BN = FwdTile<T, D>::kKeys, NS = BN / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int kBuf = BN * TL::kRowBytes;                  // two buffers of keys, two of values
  char* const kt = smem;
  char* const vt = smem + 2 * kBuf;
  float* const lut = reinterpret_cast<float*>(smem + 4 * BN * TL::kRowBytes);
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  int bh, tile, part;
  rows_work(p, blockIdx.x, gridDim.x, &bh, &tile, &part);
  const int b = bh / p.H, head = bh % p.H, kh = head / p.G;
  const int keys = keys_of(p, b), start = start_of(p, b);
  const int i0 = tile * kRows + 32 * w, i = i0 + (lane & 31), pos = start + i;
  if (BIAS) fill_bias(p, head, lut, tid, 256);
  const T* kb = (const T*)p.k.p + b * p.k.b + kh * p.k.h;
  const T* vb = (const T*)p.v.p + b * p.v.b + kh * p.v.h;
  const bool live = i < p.Lq;
  Keep kk;
  bool own = live;
  if (MASK) { kk = kept_keys(p, b, head); own = live && kept_queries(p, b, head).has(i); }
  RowRegs<T, D> q;
  q.load(own ? (const T*)p.q.p + b * p.q.b + head * p.q.h + (long)i * p.q.l : nullptr, p.d, lane);
  const uint8_t* mrow = MASK && live ? p.mask + b * p.mb + head * p.mh + (long)i * p.mi : nullptr;
  const int tiles = key_tiles<BN>(p, tile, keys, start), u0 = part * p.part_tiles, u1 = min(u0 + p.part_tiles, tiles);
  if (part > 0 && u0 >= u1) return;
  int wend = keys, wfull = keys;                            // keys that some query of the wave sees; that every one does
  if (p.causal) { wend = min(wend, start + min(i0 + 32, p.Lq)); wfull = min(wfull, start + i0 + 1); }
  const float c = p.scale * kLog2e;
  const float mult = BIAS ? 1.f : c;
  RowState st = {-INFINITY, 0.f};
  f32x16 acc[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db) acc[db] = f32x16{};
  const Async<T, D, BN, 256> kload(p.k.l, tid), vload(p.v.l, tid);
  if (u0 < u1) {
    kload.load(kt + (u0 & 1) * kBuf, kb, p.k.l, u0 * BN, keys, p.d, tid, kk);
    vload.load(vt + (u0 & 1) * kBuf, vb, p.v.l, u0 * BN, keys, p.d, tid, kk);
  }
  for (int t = u0; t < u1; ++t) {
    const int j0 = t * BN, cur = t & 1;
    wait_tiles();
    __syncthreads();
    if (t + 1 < u1) {
      kload.load(kt + (cur ^ 1) * kBuf, kb, p.k.l, j0 + BN, keys, p.d, tid, kk);
      vload.load(vt + (cur ^ 1) * kBuf, vb, p.v.l, j0 + BN, keys, p.d, tid, kk);
    }
    if (j0 < wend) {
      f32x16 s[NS];
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        s[n] = row_mma<T, D>(kt + cur * kBuf, 32 * n, lane, q, f32x16{});
        const int j = j0 + 32 * n;
        adjust<BIAS, MASK>(p, s[n], c, j, pos, start + i0, keys, mrow, lut, j + 32 > wfull, lane);
      }
      const float f = softmax_step<NS>(s, mult, st);
      if (__any(f != 1.f)) {
#pragma unroll
        for (int db = 0; db < D / 32; ++db) acc[db] *= f;
      }
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        PFrag<T> pf;
        pf.set(s[n]);
#pragma unroll
        for (int db = 0; db < D / 32; ++db) acc[db] = col_mma<D>(vt + cur * kBuf, 32 * n, db, lane, pf, acc[db]);
      }
    }
  }
  const float lsum = other_half_sum(st.l);
  if (tiles > p.part_tiles) {
    const long at = ((long)bh * p.q_tiles + tile) * p.parts + part;
    store_part<D>(p.part_o + (at * 4 + w) * 32 * D, acc, lane);
    if (lane < 32) {
      p.part_ml[at * 256 + 64 * w + lane] = st.m;
      p.part_ml[at * 256 + 64 * w + 32 + lane] = lsum;
    }
    return;
  }
  if (live) {
    const float l = lsum;
    store_row<T, D>((T*)p.o.p + b * p.o.b + head * p.o.h + (long)i * p.o.l, acc, l > 0.f || l != l ? 1.f / l : 0.f, p.d, lane);
    if (p.lse && lane < 32) p.lse[((long)b * p.H + head) * p.Lq + i] = l == 0.f ? INFINITY : st.m + __builtin_amdgcn_logf(l);
  }
}

// ---------------------------------------------------------------- few queries: the keys are split
// A block's 32 rows are the (query, head of the group) pairs of one key head (at most so many: launch plan), so a single token's G
// heads read the keys once; its four waves take 32-key tiles in turn, each through LDS of its own, and the blocks of a key head split
// the keys further.
// Bound by reading the keys and values once: 16 samples x 8 key heads x up to 16384 keys x 128 bf16, 698 MB, 138 us = 5.1 TB/s, what
// a large copy reaches; a short cache (257 keys) by latency, 8.0 us.  fp32, all 16384 keys: 265 us at 64 features (4.1 TB/s), 492 us at
// 128 (4.4 TB/s), where its registers (256 and 145 or more from 96 features on) leave one wave a SIMD to load ahead.
template <typename T, int D, bool BIAS, bool MASK> __global__ __launch_bounds__(256, D * sizeof(T) > 256 ? 1 : 2) void fwd_split_kernel(const Params p) {
  typedef Tile<T, D> TL;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  char* const kt = smem + w * 2 * 32 * TL::kRowBytes;
  char* const vt = kt + 32 * TL::kRowBytes;
  uint8_t* const bmap = reinterpret_cast<uint8_t*>(smem + 8 * 32 * TL::kRowBytes);
  const int split = blockIdx.x % p.splits, bk = blockIdx.x / p.splits, b = bk / p.Hk, kh = bk % p.Hk;
  const int keys = keys_of(p, b), start = start_of(p, b);
  const int m = lane & 31, i = m / p.G, head = kh * p.G + m % p.G, pos = start + i;
  const bool live = m < p.Lq * p.G;
  if (BIAS) {
    for (int x = tid; x <= 2 * p.max_dist; x += 256) bmap[x] = (uint8_t)bucket_of(p, x - p.max_dist);
    __syncthreads();
  }
  const T* kb = (const T*)p.k.p + b * p.k.b + kh * p.k.h;
  const T* vb = (const T*)p.v.p + b * p.v.b + kh * p.v.h;
  Keep kk;                                                  // (of all heads of the group)
  bool own = live;
  if (MASK) {
    if (p.mh == 0 || p.G == 1) kk = kept_keys(p, b, kh * p.G);
    own = live && kept_queries(p, b, head).has(i);
  }
  RowRegs<T, D> q;
  q.load(own ? (const T*)p.q.p + b * p.q.b + head * p.q.h + (long)i * p.q.l : nullptr, p.d, lane);
  const uint8_t* mrow = MASK && live ? p.mask + b * p.mb + head * p.mh + (long)i * p.mi : nullptr;
  const int end = p.causal ? min(keys, start + p.Lq) : keys;
  const int full = p.causal ? min(keys, start + 1) : keys;
  const int tiles = end > 0 ? (end + 31) / 32 : 0, per = (tiles + p.splits - 1) / p.splits;
  const int t1 = min(tiles, (split + 1) * per);
  const float c = p.scale * kLog2e, mult = BIAS ? 1.f : c;
  RowState st = {-INFINITY, 0.f};
  f32x16 acc[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db) acc[db] = f32x16{};
  Stage<T, D, 32, 64> ks, vs;
  int t = split * per + w;
  uint32_t kept = 1u;                                       // of the next tile's key that this lane (and lane + 32) asked about
  const auto ask = [&](int tile) {
    const int j = 32 * tile + (lane & 31);
    if (MASK && kk.at) kept = tile < t1 && j < keys ? kk.at[(long)j * kk.step] : 0u;
  };
  const auto fetch = [&](int tile) {
    if (MASK) {
      const KeepBits keep = {(uint32_t)__ballot(kept != 0u), 32 * tile};
      ks.fetch(kb, p.k.l, 32 * tile, keys, p.d, lane, keep);
      vs.fetch(vb, p.v.l, 32 * tile, keys, p.d, lane, keep);
    } else {
      ks.fetch(kb, p.k.l, 32 * tile, keys, p.d, lane, Keep{});
      vs.fetch(vb, p.v.l, 32 * tile, keys, p.d, lane, Keep{});
    }
    ask(tile + 4);
  };
  ask(t);
  if (t < t1) fetch(t);
  for (; t < t1; t += 4) {
    ks.put(kt, lane);
    vs.put(vt, lane);
    if (t + 4 < t1) fetch(t + 4);
    const int j0 = 32 * t;
    f32x16 bias;                                            // read in front of the fence: sixteen loads in flight, not one by one
    if (BIAS) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        bias[r] = p.table[(long)bmap[dist_slot(p, j0 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3) - pos)] * p.H + min(head, p.H - 1)];
    }
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
    f32x16 s[1];
    s[0] = row_mma<T, D>(kt, 0, lane, q, f32x16{});
    if (BIAS) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[0][r] = fmaf(s[0][r], c, bias[r] * kLog2e);
    }
    adjust<false, MASK>(p, s[0], c, j0, pos, 0, keys, mrow, nullptr, j0 + 32 > full, lane);
    const float f = softmax_step<1>(s, mult, st);
    if (__any(f != 1.f)) {
#pragma unroll
      for (int db = 0; db < D / 32; ++db) acc[db] *= f;
    }
    PFrag<T, true> pf;
    pf.set(s[0]);
#pragma unroll
    for (int db = 0; db < D / 32; ++db) acc[db] = col_mma<D>(vt, 0, db, lane, pf, acc[db]);
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  // the four waves' rows meet in LDS, [wave][feature][row]
  __syncthreads();
  float* const ob = reinterpret_cast<float*>(smem);
  float* const ml = ob + 4 * D * 32;                        // [wave][m, l][row]
  const float l = other_half_sum(st.l);
  if (lane < 32) { ml[(w * 2) * 32 + lane] = st.m; ml[(w * 2 + 1) * 32 + lane] = l; }
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) ob[(w * D + db * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3)) * 32 + (lane & 31)] = acc[db][r];
  __syncthreads();
  const int row = tid & 31;
  const int ir = row / p.G, hr = kh * p.G + row % p.G;
  float mx = -INFINITY;
#pragma unroll
  for (int v = 0; v < 4; ++v) mx = fmaxf(mx, ml[v * 64 + row]);
  float fw[4], lt = 0.f;
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    fw[v] = mx == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[v * 64 + row] - mx);
    lt += fw[v] * ml[v * 64 + 32 + row];
  }
  if (row >= p.Lq * p.G) return;
  const bool whole = p.splits == 1;
  const float inv = !whole ? 1.f : lt > 0.f || lt != lt ? 1.f / lt : 0.f;
  const long pr = ((long)bk * p.splits + split) * 32 + row;
  T* out = (T*)p.o.p + b * p.o.b + hr * p.o.h + (long)ir * p.o.l;
  for (int e0 = 4 * (tid >> 5); e0 < D; e0 += 32) {
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = 0.f;
#pragma unroll
      for (int v = 0; v < 4; ++v) x[e] += fw[v] * ob[(v * D + e0 + e) * 32 + row];
    }
    if (whole) store4<T>(out, e0, p.d, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
    else *reinterpret_cast<f32x4*>(p.part_o + pr * D + e0) = f32x4{x[0], x[1], x[2], x[3]};
  }
  if (tid < 32) {
    if (!whole) { p.part_ml[2 * pr] = mx; p.part_ml[2 * pr + 1] = lt; }
    else if (p.lse) p.lse[((long)b * p.H + hr) * p.Lq + ir] = lt == 0.f ? INFINITY : mx + __builtin_amdgcn_logf(lt);
  }
}

// joins the splits of a row: one wave a row
template <typename T, int D> __global__ __launch_bounds__(256) void fwd_join_kernel(const Params p) {
  const int lane = threadIdx.x & 63;
  const long rows = (long)p.B * p.Hk * p.Lq * p.G, n = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= rows) return;
  const int rg = p.Lq * p.G, m = (int)(n % rg), bk = (int)(n / rg), b = bk / p.Hk, kh = bk % p.Hk;
  const int i = m / p.G, head = kh * p.G + m % p.G;
  const long first = (long)bk * p.splits * 32 + m;
  float mx = -INFINITY;
  for (int s = lane; s < p.splits; s += 64) mx = fmaxf(mx, p.part_ml[2 * (first + (long)s * 32)]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
  const float mref = mx == -INFINITY ? 0.f : mx;
  float l = 0.f, x[(D + 63) / 64];
#pragma unroll
  for (int e = 0; e < (D + 63) / 64; ++e) x[e] = 0.f;
  for (int s = 0; s < p.splits; ++s) {
    const long at = first + (long)s * 32;
    const float f = __builtin_amdgcn_exp2f(p.part_ml[2 * at] - mref);
    l += f * p.part_ml[2 * at + 1];
#pragma unroll
    for (int e = 0; e < (D + 63) / 64; ++e) if (lane + 64 * e < D) x[e] += f * p.part_o[at * D + lane + 64 * e];
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  T* out = (T*)p.o.p + b * p.o.b + head * p.o.h + (long)i * p.o.l;
#pragma unroll
  for (int e = 0; e < (D + 63) / 64; ++e) if (lane + 64 * e < p.d) out[lane + 64 * e] = (T)(x[e] * inv);
  if (p.lse && lane == 0) p.lse[((long)b * p.H + head) * p.Lq + i] = l == 0.f ? INFINITY : mx + __builtin_amdgcn_logf(l);
}

template <typename T, int D, bool BIAS, bool MASK> int forward(const Params& p, hipStream_t s) {
  typedef Tile<T, D> TL;
  if (p.splits == 0) {
    const size_t lds = 4 * FwdTile<T, D>::kKeys * TL::kRowBytes + (BIAS ? (2 * p.max_dist + 1) * sizeof(float) : 0);
    OCEAN_TRY(set_lds(fwd_rows_kernel<T, D, BIAS, MASK>, lds));
    hipLaunchKernelGGL((fwd_rows_kernel<T, D, BIAS, MASK>), dim3((unsigned)((long)p.B * p.H * p.q_tiles * p.parts)), dim3(256), lds, s, p);
    OCEAN_LAUNCH_CHECK();
    if (p.parts > 1) {
      hipLaunchKernelGGL((fwd_rows_join_kernel<T, D>), dim3((unsigned)((long)p.B * p.H * p.q_tiles * 4)), dim3(256), 0, s, p);
      OCEAN_LAUNCH_CHECK();
    }
    return OCEAN_OK;
  }
  size_t lds = 8 * 32 * TL::kRowBytes + (BIAS ? 2 * p.max_dist + 1 : 0);
  const size_t meet = (size_t)(4 * D * 32 + 4 * 2 * 32) * sizeof(float);
  if (meet > lds) lds = meet;
  OCEAN_TRY(set_lds(fwd_split_kernel<T, D, BIAS, MASK>, lds));
  hipLaunchKernelGGL((fwd_split_kernel<T, D, BIAS, MASK>), dim3((unsigned)((long)p.B * p.Hk * p.splits)), dim3(256), lds, s, p);
  OCEAN_LAUNCH_CHECK();
  if (p.splits > 1) {
    hipLaunchKernelGGL((fwd_join_kernel<T, D>), dim3((unsigned)(((long)p.B * p.H * p.Lq + 3) / 4)), dim3(256), 0, s, p);
    OCEAN_LAUNCH_CHECK();
  }
  return OCEAN_OK;
}

template <typename T, int D> int forward_b(const Params& p, hipStream_t s) {
  if (p.mask) return p.table ? forward<T, D, true, true>(p, s) : forward<T, D, false, true>(p, s);
  return p.table ? forward<T, D, true, false>(p, s) : forward<T, D, false, false>(p, s);
}
template <typename T> int forward_d(const Params& p, hipStream_t s) {
  if (p.d <= 32) return forward_b<T, 32>(p, s);
  if (p.d <= 64) return forward_b<T, 64>(p, s);
  if (p.d <= 96) return forward_b<T, 96>(p, s);
  return forward_b<T, 128>(p, s);
}

}  // namespace

int launch_forward(const Params& p, int type, hipStream_t s) { return type == OCEAN_BF16 ? forward_d<__bf16>(p, s) : forward_d<float>(p, s); }

}  // namespace seqattn
