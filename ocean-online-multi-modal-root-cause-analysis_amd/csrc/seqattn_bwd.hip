// Backward pass of attention without stored weights (seqattn.h).  With the row's log-sum from the forward pass,
//   p_ij = 2^(s_ij - lse_i),  dp_ij = do_i . v_j,  ds_ij = p_ij (dp_ij - delta_i),  delta_i = do_i . o_i,
//   dq_i = scale sum_j ds_ij k_j,   dk_j = scale sum_i ds_ij q_i,   dv_j = sum_i p_ij do_i,   dbias(dist) = sum of ds over a diagonal.
// Two launches, each of which owns what it sums: one over queries (dq, delta), one over keys (dk, dv, with the heads that share
// a key head as more rows of the sum, and the bias).  The scores are formed in both - seven products instead of five - and in
// exchange no gradient is summed by atomics or through memory: results do not depend on the order of the blocks.
#include "seqattn.h"

namespace seqattn {
namespace {

constexpr int kRows = kKeyTile;      // queries (keys) of a block: four waves, 32 each

// p_ij for keys j0.. of this lane's query (at pos; the wave's first at pos0), from scores
template <bool BIAS, bool MASK> __device__ __forceinline__ void probabilities(const Params& p, f32x16& s, float c, float lse, int j0, int pos, int pos0, int keys,
                                                                              const uint8_t* mrow, const float* lut, bool edge, int lane) {
  const int h4 = 4 * (lane >> 5);
  f32x16 t;
  if (BIAS) {
    t = block_bias<1>(p, lut, j0 + h4 - pos, j0 - pos0);
#pragma unroll
    for (int r = 0; r < 16; ++r) t[r] -= lse;
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, BIAS ? t[r] : -lse));
  if (MASK || edge) {
    const int end = (p.causal ? min(keys, pos + 1) : keys) - j0 - h4;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      uint32_t ok = 15u;
      if (MASK) ok = mrow ? mask4(p, mrow, j0 + 8 * g + h4, keys) : 15u;
#pragma unroll
      for (int e = 0; e < 4; ++e) if (8 * g + e >= end || (MASK && !((ok >> e) & 1u))) s[4 * g + e] = 0.f;
    }
  }
}

// Sums of a wave's 32x32 block of ds (rows: queries, own columns: keys) over its 63 diagonals.  Eight rows make a chain: shifted by
// one lane before each row is added, so that lane l of the chain of rows 8c..8c+7 ends up with the diagonal key - query = l - 7 - 8c.
// The four chains are moved onto each other, lane l holding the diagonal l - 31, and added to the wave's own sums by distance: one
// lane owns one distance and blocks follow each other in order, so the sums come out the same in every run.  (16 x 12 heads x
// 512 x 64, launch over keys: 107 us through an LDS image of the block, 92 with LDS additions of the four chains, 71 this way; 57 is
// the launch without the sums.)
struct DiagSums {
  float* by_dist;                    // [2 max_dist + 1]
  float below, above;                // distances of -max_dist and less, max_dist and more
  static __device__ __forceinline__ float next_lane(float x) {      // lane l gets lane l - 1's, lane 0 gets 0
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x138, 0xf, 0xf, true));
  }
  __device__ __forceinline__ void add(const Params& p, const f32x16& ds, int d0, int lane) {
    if (d0 + 31 <= -p.max_dist || d0 - 31 >= p.max_dist) {
      float t = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) t += ds[r];
      if (d0 < 0) below += t; else above += t;
      return;
    }
    float chain[4];
    float hi[4][4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        // registers 4c + e: row 8c + e in the lower half, 8c + 4 + e in the upper one; both halves to lanes 0..31 over zeros
        const float x = ds[4 * c + e];
        const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), 0u, false, false);
        hi[c][e] = __builtin_bit_cast(float, (uint32_t)r[1]);
        const float lo = __builtin_bit_cast(float, (uint32_t)r[0]);
        chain[c] = e == 0 ? lo : next_lane(chain[c]) + lo;
      }
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int c = 0; c < 4; ++c) chain[c] = next_lane(chain[c]) + hi[c][e];
    float t = chain[3];
#pragma unroll
    for (int c = 0; c < 3; ++c)                             // chains are zero from lane 39 on, where the moves wrap to
      t += __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(4 * (lane - 8 * (3 - c)), __builtin_bit_cast(int, chain[c])));
    const int dist = d0 + lane - 31;
    if (dist <= -p.max_dist) below += t;
    else if (dist >= p.max_dist) above += t;
    else if (lane < 63) by_dist[dist + p.max_dist] += t;
    asm volatile("" ::: "memory");                          // the next block's lanes own other distances: its reads stay behind these writes
  }
};

// the block's sums by bucket (each bucket a run of distances), and the sums by distance back to zero for the next head
__device__ __forceinline__ void store_bias_sums(const Params& p, DiagSums& diag, float* dist_sums, float* part, int tid) {
  const int slots = 2 * p.max_dist + 1;
  float lo = diag.below, hi = diag.above;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) { lo += __shfl_xor(lo, o, 64); hi += __shfl_xor(hi, o, 64); }
  if ((tid & 63) == 0) { diag.by_dist[0] += lo; diag.by_dist[slots - 1] += hi; }
  diag.below = diag.above = 0.f;
  __syncthreads();
  for (int x = tid; x < slots; x += 256) dist_sums[x] = (dist_sums[x] + dist_sums[slots + x]) + (dist_sums[2 * slots + x] + dist_sums[3 * slots + x]);
  __syncthreads();
  // bucket k holds the distances of n0..n1 steps to one side: sixteen lanes add a bucket's
  const int sub = tid & 15;
  for (int k = tid >> 4; k < p.buckets; k += 16) {
    const int right = p.both && k >= p.side, f = right ? k - p.side : k;
    int n0 = f <= p.exact ? f : p.limits[f - p.exact - 1];
    const int n1 = f == p.side - 1 ? p.max_dist : f < p.exact ? f : p.limits[f - p.exact] - 1;
    int x0 = p.max_dist - n1, x1 = p.max_dist - n0;
    if (right) { n0 = max(n0, 1); x0 = p.max_dist + n0; x1 = p.max_dist + n1; }
    if (!p.both && f == 0) x1 = slots - 1;
    float t = 0.f;
    for (int x = x0 + sub; x <= x1; x += 16) t += dist_sums[x];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
    if (sub == 0) part[k] = t;
  }
  __syncthreads();
  for (int x = tid; x < 4 * slots; x += 256) dist_sums[x] = 0.f;
  __syncthreads();
}

template <typename T, int D> struct BwdTile {
  static constexpr int kRows = query_tile(D * sizeof(T));   // queries at a time of the launch over keys
  static constexpr int kKeys = key_tile(sizeof(T) == 2);    // keys at a time of the launch over queries
};

// Launch over queries, three products (s, dp, dq): the wave's 32 queries and their d_out in registers, keys and values through two
// LDS buffers each.  Bound by the turns of its two waves a SIMD between matrix cores (busy 0.45 of the cycles), vector units (0.37), LDS
// (0.45, half of it bank conflicts) and tiles (waiting 0.40); the registers hold no third wave and no second tile.  Causal 2 x 16
// heads (4 of keys) x 4096 x 128 bf16: 228 us = 0.90 PFLOP/s of the three products; 8 x 8 heads x 512 x 96 fp32, ragged: 96 us.
template <typename T, int D, bool BIAS, bool MASK> __global__ __launch_bounds__(256, D * sizeof(T) > (MASK ? 128 : 256) ? 1 : 2) void dq_kernel(const Params p) {
  typedef Tile<T, D> TL;
  constexpr int BN = BwdTile<T, D>::kKeys, NS = BN / 32;
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
  const bool live = i < p.Lq;
  if (BIAS) fill_bias(p, head, lut, tid, 256);
  const int tiles = key_tiles<BN>(p, tile, keys, start), u0 = part * p.part_tiles, u1 = min(u0 + p.part_tiles, tiles);
  if (part > 0 && u0 >= u1) return;
  const T* kb = (const T*)p.k.p + b * p.k.b + kh * p.k.h;
  const T* vb = (const T*)p.v.p + b * p.v.b + kh * p.v.h;
  Keep kk;
  bool own = live;
  if (MASK) { kk = kept_keys(p, b, head); own = live && kept_queries(p, b, head).has(i); }
  RowRegs<T, D> q, go;
  q.load(own ? (const T*)p.q.p + b * p.q.b + head * p.q.h + (long)i * p.q.l : nullptr, p.d, lane);
  go.load(own ? (const T*)p.go.p + b * p.go.b + head * p.go.h + (long)i * p.go.l : nullptr, p.d, lane);
  float delta = 0.f, lse = INFINITY;
  if (live) {
    RowRegs<T, D> o;
    o.load((const T*)p.o.p + b * p.o.b + head * p.o.h + (long)i * p.o.l, p.d, lane);
#pragma unroll
    for (int s = 0; s < RowRegs<T, D>::kSteps; ++s)
#pragma unroll
      for (int e = 0; e < Mm<T>::kEpc; ++e) delta = fmaf((float)go.f[s][e], (float)o.f[s][e], delta);
    lse = p.lse[((long)b * p.H + head) * p.Lq + i];
  }
  delta = other_half_sum(delta);
  float rest = 0.f;
  const uint8_t* mrow = MASK && live ? p.mask + b * p.mb + head * p.mh + (long)i * p.mi : nullptr;
  int wend = keys, wfull = keys;
  if (p.causal) { wend = min(wend, start + min(i0 + 32, p.Lq)); wfull = min(wfull, start + i0 + 1); }
  const float c = p.scale * kLog2e;
  f32x16 acc[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db) acc[db] = f32x16{};
  const Async<T, D, BN, 256> kload(p.k.l, tid), vload(p.v.l, tid);
  if (u0 < u1) {
    kload.load(kt + (u0 & 1) * kBuf, kb, p.k.l, u0 * BN, keys, p.d, tid, kk);
    vload.load(vt + (u0 & 1) * kBuf, vb, p.v.l, u0 * BN, keys, p.d, tid, kk);
  }
  // Up to two tiles of keys sit in the two buffers.  Rows of so few keys are where 16-bit rounding of `o` reaches dq through delta
  // (its share shrinks with the root of the number of keys that carry weight): their delta is formed from p and dp first
  // (a part has two tiles at least, so they are never split).
  const bool few = sizeof(T) == 2 && tiles <= 2;
  if (few && tiles == 2) {
    kload.load(kt + kBuf, kb, p.k.l, BN, keys, p.d, tid, kk);
    vload.load(vt + kBuf, vb, p.v.l, BN, keys, p.d, tid, kk);
  }
  if (few) {
    wait_tiles();
    __syncthreads();
    float sum = 0.f;
    for (int j = 0; j < wend; j += 32) {
      const int at = j / BN * kBuf, row = j % BN;
      f32x16 s = row_mma<T, D>(kt + at, row, lane, q, f32x16{});
      const f32x16 dp = row_mma<T, D>(vt + at, row, lane, go, f32x16{});
      probabilities<BIAS, MASK>(p, s, c, lse, j, pos, start + i0, keys, mrow, lut, j + 32 > wfull, lane);
#pragma unroll
      for (int r = 0; r < 16; ++r) sum = fmaf(s[r], dp[r], sum);
    }
    delta = other_half_sum(sum);
  }
  for (int t = u0; t < u1; ++t) {
    const int j0 = t * BN, cur = t & 1;
    if (!few) {
      wait_tiles();
      __syncthreads();
      if (t + 1 < u1) {
        kload.load(kt + (cur ^ 1) * kBuf, kb, p.k.l, j0 + BN, keys, p.d, tid, kk);
        vload.load(vt + (cur ^ 1) * kBuf, vb, p.v.l, j0 + BN, keys, p.d, tid, kk);
      }
    }
    if (j0 < wend) {
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        const int j = j0 + 32 * n;
        f32x16 s = row_mma<T, D>(kt + cur * kBuf, 32 * n, lane, q, f32x16{});
        const f32x16 dp = row_mma<T, D>(vt + cur * kBuf, 32 * n, lane, go, f32x16{});
        probabilities<BIAS, MASK>(p, s, c, lse, j, pos, start + i0, keys, mrow, lut, j + 32 > wfull, lane);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[r] *= dp[r] - delta;
          if (sizeof(T) == 2) rest += s[r];
        }
        PFrag<T> pf;
        pf.set(s);
#pragma unroll
        for (int db = 0; db < D / 32; ++db) acc[db] = col_mma<D>(kt + cur * kBuf, 32 * n, db, lane, pf, acc[db]);
      }
    }
  }
  if (tiles > p.part_tiles) {
    const long at = ((long)bh * p.q_tiles + tile) * p.parts + part;
    store_part<D>(p.part_o + (at * 4 + w) * 32 * D, acc, lane);
    if (sizeof(T) == 2) rest = other_half_sum(rest);
    if (lane < 32) {
      p.part_ml[at * 256 + 64 * w + lane] = delta;
      p.part_ml[at * 256 + 64 * w + 32 + lane] = rest;
    }
    return;
  }
  if (live && p.dq.p) store_row<T, D>((T*)p.dq.p + b * p.dq.b + head * p.dq.h + (long)i * p.dq.l, acc, p.scale, p.d, lane);
  // In 16 bits `o` was rounded, and so were the weights that formed it: delta is a few 1e-3 of |do| |o| off.  The row's ds sum to
  // what is missing, in fp32 and for one addition each; the launch over keys, and the bias with it, gets the exact delta.
  if (sizeof(T) == 2) delta += other_half_sum(rest);
  if (live && lane < 32) p.delta[((long)b * p.H + head) * p.Lq + i] = delta;
}

// a lane's sixteen rows' values from 32 consecutive ones (from its half's first on)
__device__ __forceinline__ f32x16 row_values(const float* at) {
  f32x16 x;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const f32x4 q = *reinterpret_cast<const f32x4*>(at + 8 * g);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[4 * g + e] = q[e];
  }
  return x;
}

// the tiles of BM queries that see some key of the tile: `tiles` from t0 on
template <int BM> __device__ __forceinline__ void query_tiles(const Params& p, int tile, int keys, int start, int* t0, int* tiles) {
  int first = p.causal ? min(max(tile * kRows - start, 0), p.Lq) : 0;
  if (tile * kRows >= keys) first = p.Lq;
  *t0 = first / BM;
  *tiles = first < p.Lq ? (p.Lq + BM - 1) / BM - *t0 : 0;
}

// What segment `seg` does of a key tile's list of query tiles (of all heads that share the key head): places u0..u1 - 1 of `all`; the
// list is in `pieces` segments, from first_seg on.  Without `causal` a segment is seg_tiles places.  With it a tile's list is
// shorter the later the tile, so tile t shares segments with tile k_tiles - 1 - t: the two lists behind one another, of about
// the same length for every pair, are cut into `segs` equal segments.
struct Span { int t0, tiles, all, u0, u1, first_seg, pieces; };
template <int BM> __device__ __forceinline__ Span span_of(const Params& p, int tile, int seg, int keys, int start) {
  Span s;
  query_tiles<BM>(p, tile, keys, start, &s.t0, &s.tiles);
  s.all = s.tiles * p.G;
  int per = p.seg_tiles, before = 0;
  if (p.causal) {
    const int other = p.k_tiles - 1 - tile;
    int t0, tiles = 0;
    if (other != tile) query_tiles<BM>(p, other, keys, start, &t0, &tiles);
    per = max(1, (s.all + tiles * p.G + p.segs - 1) / p.segs);
    if (tile > other) before = tiles * p.G;
  }
  s.u0 = min(max(seg * per - before, 0), s.all);
  s.u1 = min(max((seg + 1) * per - before, 0), s.all);
  s.first_seg = min(before / per, p.segs - 1);
  s.pieces = s.all > 0 ? (before + s.all - 1) / per - s.first_seg + 1 : 0;
  return s;
}

// A wave keeps its 32 keys' dk and dv in registers, and the keys as right operand; the values too where that leaves room for two
// waves on a SIMD, else they stay in LDS (VL): at 128 16-bit features the registers of both were 440, and half of the instructions
// moved accumulators between the two register files.  Four products (s, dp, dv, dk).  The 256 registers of two waves a SIMD still do
// not hold it at 96 and 128 16-bit features: 16 bytes a lane live in scratch memory at 128 (8 with a mask, 20 with a bias, 84 with both),
// 40 at 96 (28, 80, 152).  Causal 2 x 16 heads (4 of keys) x 4096 x 128 bf16: 419 us = 0.66 PFLOP/s of the four, bound by waiting for LDS
// and barriers with few waves (1.44 a SIMD, waiting 0.52 of their cycles; LDS busy 0.43 of the cycles, 0.19 in bank conflicts; matrix
// cores 0.31, vector 0.20).  16 x 12 heads x 512 x 64 with a bias, ragged: 77 us, waiting too (0.51, 1.2 waves a SIMD; matrix cores 0.11,
// vector 0.25).  8 x 8 heads x 512 x 96 fp32, ragged: 134 us, 0.7 waves a SIMD between their own matrix instructions (busy 0.45).
template <typename T, int D, bool BIAS, bool MASK> __global__ __launch_bounds__(256, D * sizeof(T) > 256 ? 1 : 2) void dkv_kernel(const Params p) {
  typedef Tile<T, D> TL;
  constexpr int BM = BwdTile<T, D>::kRows, NS = BM / 32;
  constexpr bool VL = values_in_lds(D * sizeof(T));
  // 16 bits: the products start at -lse in score units (4e-6 of a probability, far below its rounding); the bias, whose gradient is
  // summed in fp32, takes lse as it is
  constexpr bool FROM_LSE = sizeof(T) == 2 && !BIAS;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int kBuf = BM * TL::kRowBytes;                  // two buffers of queries, two of the outputs' gradients
  char* const qt = smem;
  char* const gt = smem + 2 * kBuf;
  char* const vt = smem + 4 * kBuf;                          // VL: the block's values
  float* const rowv = reinterpret_cast<float*>(vt + (VL ? kRows * TL::kRowBytes : 0));      // [2][lse, delta][BM]
  float* const lut = rowv + 4 * BM;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), h4 = 4 * (lane >> 5), slots = 2 * p.max_dist + 1;
  DiagSums diag;
  float* const dist_sums = lut + slots;                     // [wave][slots]
  const bool sum_bias = BIAS && p.dtable_part != nullptr;
  if (BIAS) {
    diag.by_dist = dist_sums + w * slots;
    diag.below = diag.above = 0.f;
    if (sum_bias) for (int x = tid; x < 4 * slots; x += 256) dist_sums[x] = 0.f;
  }
  // With `causal` a pair's segment lies in one tile or in the end of one and the beginning of the other: blocks for the longer part
  // of every segment come first, blocks for the rest fill the places that those with a rest leave early.
  const int k_tiles = p.k_tiles;
  int bk, place;
  work_of(p, blockIdx.x, gridDim.x, p.causal ? (k_tiles + 1) / 2 * 2 * p.segs : k_tiles * p.segs, &bk, &place);
  const int b = bk / p.Hk, kh = bk % p.Hk, head0 = kh * p.G, keys = keys_of(p, b), start = start_of(p, b);
  int tile = place % k_tiles, seg = place / k_tiles;
  Span span;
  if (p.causal) {
    const int pairs = (k_tiles + 1) / 2, second = place / (pairs * p.segs), r = place % (pairs * p.segs);
    seg = r / pairs;
    const int t1 = r % pairs, t2 = k_tiles - 1 - t1;
    if (t1 == t2 && second) return;
    const Span s1 = span_of<BM>(p, t1, seg, keys, start), s2 = span_of<BM>(p, t2, seg, keys, start);
    const bool take2 = t1 != t2 && (s2.u1 - s2.u0 > s1.u1 - s1.u0) != (second != 0);
    tile = take2 ? t2 : t1;
    span = take2 ? s2 : s1;
  } else {
    span = span_of<BM>(p, tile, seg, keys, start);
  }
  const int u0 = span.u0, u1 = span.u1, tiles = span.tiles, t0 = span.t0;
  if (sum_bias) {                                           // the heads that this segment does not reach
    const int g0 = u0 < u1 ? u0 / tiles : 0, g1 = u0 < u1 ? (u1 - 1) / tiles : -1;
    for (int x = tid; x < p.G * p.buckets; x += 256) {
      const int g = x / p.buckets;
      if (g < g0 || g > g1) p.dtable_part[((((long)(head0 + g) * p.B + b) * k_tiles + tile) * p.segs + seg) * p.buckets + x % p.buckets] = 0.f;
    }
  }
  if (u0 >= u1 && (span.all > 0 || seg != span.first_seg)) return;
  const T* vb = (const T*)p.v.p + b * p.v.b + kh * p.v.h;
  const float c = p.scale * kLog2e, row_unit = 1.f / c;
  const Async<T, D, BM, 256> qload(p.q.l, tid), gload(p.go.l, tid);
  const int j0 = tile * kRows + 32 * w, j = j0 + (lane & 31);
  Keep kk;                                                  // (of all heads of the group)
  if (MASK && (p.mh == 0 || p.G == 1)) kk = kept_keys(p, b, head0);
  const bool live = j < keys && kk.has(j);
  RowRegs<T, D> k, v;
  k.load(live ? (const T*)p.k.p + b * p.k.b + kh * p.k.h + (long)j * p.k.l : nullptr, p.d, lane);
  if (!VL) v.load(live ? vb + (long)j * p.v.l : nullptr, p.d, lane);
  f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db) { dk[db] = f32x16{}; dv[db] = f32x16{}; }
  // queries from wfirst on see some key of this wave; from wfull on every key
  int wfirst = 0, wfull = 0;
  if (p.causal) { wfirst = max(j0 - start, 0); wfull = j0 + 31 - start; }
  float rv = 0.f;                                           // threads 0..BM-1: -lse, BM..2BM-1: -delta
  const auto load = [&](int u, int buf) {
    const int head = head0 + u / tiles, r0 = (t0 + u % tiles) * BM;
    Keep kq;
    if (MASK) kq = kept_queries(p, b, head);
    if (tid < 2 * BM) {
      const int i = r0 + tid % BM;
      const float* from = tid < BM ? p.lse : p.delta;
      rv = i < p.Lq ? -from[((long)b * p.H + head) * p.Lq + i] : tid < BM ? -INFINITY : 0.f;
      if (FROM_LSE && tid < BM) rv *= row_unit;
    }
    qload.load(qt + buf * kBuf, (const T*)p.q.p + b * p.q.b + head * p.q.h, p.q.l, r0, p.Lq, p.d, tid, kq);
    gload.load(gt + buf * kBuf, (const T*)p.go.p + b * p.go.b + head * p.go.h, p.go.l, r0, p.Lq, p.d, tid, kq);
  };
  if (u0 < u1) {
    if (VL) Async<T, D, kRows, 256>(p.v.l, tid).load(vt, vb, p.v.l, tile * kRows, keys, p.d, tid, kk);
    load(u0, u0 & 1);
    if (BIAS) fill_bias(p, head0 + u0 / tiles, lut, tid, 256);
  }
  for (int u = u0; u < u1; ++u) {
    const int cur = u & 1, g = u / tiles, head = head0 + g, r0 = (t0 + u % tiles) * BM;
    if (tid < 2 * BM) rowv[cur * 2 * BM + tid] = rv;
    if (BIAS && u > u0 && u % tiles == 0) {
      __syncthreads();                                      // the last head's biases are still being read
      fill_bias(p, head, lut, tid, 256);
    }
    wait_tiles();
    __syncthreads();
    if (u + 1 < u1) load(u + 1, cur ^ 1);
    if (j0 < keys && r0 + BM > wfirst) {
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        const int i0 = r0 + 32 * n;
        const float* lr = rowv + cur * 2 * BM + 32 * n + h4;
        // the sums start at the row's -lse and -delta, read from LDS where they are needed
        f32x16 s = f32x16{};
        if (FROM_LSE) s = row_values(lr);
        s = row_mma<T, D>(qt + cur * kBuf, 32 * n, lane, k, s);
        f32x16 dp;
        const auto form_dp = [&] {
          dp = BIAS ? f32x16{} : row_values(lr + BM);
          if (VL) {
#pragma unroll
            for (int st = 0; st < RowRegs<T, D>::kSteps; ++st)
              dp = Mm<T>::mma(TL::row_frag(gt + cur * kBuf, 32 * n, st, lane), TL::row_frag(vt, 32 * w, st, lane), dp);
          } else {
            dp = row_mma<T, D>(gt + cur * kBuf, 32 * n, lane, v, dp);
          }
        };
        if (!VL) form_dp();
        f32x16 bias;
        if (BIAS) bias = block_bias<-1>(p, lut, j - (start + i0 + h4), j0 - (start + i0));
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int at = 8 * (r >> 2) + (r & 3);
          float t = FROM_LSE ? 0.f : lr[at];
          if (BIAS) t += bias[r];
          s[r] = __builtin_amdgcn_exp2f(FROM_LSE ? s[r] * c : fmaf(s[r], c, t));
        }
        if (MASK || j0 + 32 > keys || (p.causal && i0 < wfull)) {
          const uint8_t* mcol = MASK ? p.mask + b * p.mb + head * p.mh + (long)j * p.mj + (long)(i0 + h4) * p.mi : nullptr;
          const int from = live ? (p.causal ? j - start : 0) - i0 - h4 : 1 << 30;      // the first query that sees this key
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int i = 8 * (r >> 2) + (r & 3);
            bool ok = i >= from;
            if (MASK && ok && i0 + h4 + i < p.Lq) ok = mcol[(long)i * p.mi] != 0;
            if (!ok) s[r] = 0.f;
          }
        }
        PFrag<T> pf;
        pf.set(s);
        if (VL) __builtin_amdgcn_sched_barrier(0);          // one product at a time: the registers hold no more than its operands
#pragma unroll
        for (int db = 0; db < D / 32; ++db) dv[db] = col_mma<D>(gt + cur * kBuf, 32 * n, db, lane, pf, dv[db]);
        if (VL) {
          __builtin_amdgcn_sched_barrier(0);
          form_dp();
          __builtin_amdgcn_sched_barrier(0);
        }
        // With a bias dP is formed from zero and delta taken off after, by the steps of the launch over queries, whose sums delta comes
        // from: what the bf16 products' sums are off (to one side, on the average) then cancels over a row, and a row's ds add up to
        // zero.  Started at -delta, the bias's gradient over 16 x 12 heads x 512 x 512 was 1.0e-6 to 1.4e-6 of its norm off, 4e-7 this way.
        if (BIAS) dp += row_values(lr + BM);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= dp[r];
        if (sum_bias) diag.add(p, s, j0 - (start + i0), lane);
        pf.set(s);
#pragma unroll
        for (int db = 0; db < D / 32; ++db) dk[db] = col_mma<D>(qt + cur * kBuf, 32 * n, db, lane, pf, dk[db]);
      }
    }
    if (sum_bias && (u == u1 - 1 || u % tiles == tiles - 1))
      store_bias_sums(p, diag, dist_sums, p.dtable_part + ((((long)head * p.B + b) * k_tiles + tile) * p.segs + seg) * p.buckets, tid);
  }
  if (span.pieces > 1) {                                    // sums in the matrix instructions' layout
    float* part = p.part_o + ((((long)bk * k_tiles + tile) * p.segs + seg) * 4 + w) * (2 * 32 * D);
    store_part<D>(part, dk, lane);
    store_part<D>(part + 32 * D, dv, lane);
    return;
  }
  if (j < p.Lk) {                                           // keys past the sample's end get zeros
    if (p.dk.p) store_row<T, D>((T*)p.dk.p + b * p.dk.b + kh * p.dk.h + (long)j * p.dk.l, dk, p.scale, p.d, lane);
    if (p.dv.p) store_row<T, D>((T*)p.dv.p + b * p.dv.b + kh * p.dv.h + (long)j * p.dv.l, dv, 1.f, p.d, lane);
  }
}

// dq and delta of the query tiles whose keys were split: the parts' sums in their order
template <typename T, int D> __global__ __launch_bounds__(256) void dq_join_kernel(const Params p) {
  const int unit = blockIdx.x >> 2, w = blockIdx.x & 3, lane = threadIdx.x & 63, r = lane & 31;
  const int tile = unit % p.q_tiles, bh = unit / p.q_tiles, b = bh / p.H, head = bh % p.H, i = tile * kRows + 32 * w + r;
  const int tiles = key_tiles<BwdTile<T, D>::kKeys>(p, tile, keys_of(p, b), start_of(p, b));
  if (tiles <= p.part_tiles || i >= p.Lq) return;
  const int parts = (tiles + p.part_tiles - 1) / p.part_tiles;
  const float* from = p.part_o + ((long)unit * p.parts * 4 + w) * 32 * D + lane * 4;
  T* out = (T*)p.dq.p + b * p.dq.b + head * p.dq.h + (long)i * p.dq.l;
  if (p.dq.p)
    for (int n = threadIdx.x >> 6; n < D / 8; n += 4) {
      f32x4 t = {0.f, 0.f, 0.f, 0.f};
      for (int s = 0; s < parts; ++s) t += *reinterpret_cast<const f32x4*>(from + (long)s * 4 * 32 * D + n * 256);
      store4<T>(out, part_feature(n, lane), p.d, t[0] * p.scale, t[1] * p.scale, t[2] * p.scale, t[3] * p.scale);
    }
  if (threadIdx.x < 32) {
    const float* dr = p.part_ml + (long)unit * p.parts * 256 + 64 * w + r;
    float delta = dr[0];
    for (int s = 0; s < parts; ++s) delta += dr[s * 256 + 32];
    p.delta[((long)b * p.H + head) * p.Lq + i] = delta;
  }
}

// dk, dv of the key tiles whose queries were split: the segments' sums in their order.  A block joins a quarter of a wave's part.
template <typename T, int D> __global__ __launch_bounds__(256) void dkv_join_kernel(const Params p) {
  constexpr int BM = BwdTile<T, D>::kRows, kPieces = D / 8;  // 16-byte pieces a lane: D / 32 blocks x 4, of dk and of dv
  const int unit = blockIdx.x >> 2, w = blockIdx.x & 3, lane = threadIdx.x & 63;
  const int tile = unit % p.k_tiles, bk = unit / p.k_tiles, b = bk / p.Hk, kh = bk % p.Hk;
  const Span span = span_of<BM>(p, tile, 0, keys_of(p, b), start_of(p, b));
  if (span.pieces <= 1) return;
  const int j = tile * kRows + 32 * w + (lane & 31);
  const float* part = p.part_o + (((long)unit * p.segs + span.first_seg) * 4 + w) * (2 * 32 * D) + lane * 4;
  for (int n = threadIdx.x >> 6; n < 2 * kPieces; n += 4) {
    f32x4 t = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < span.pieces; ++s) t += *reinterpret_cast<const f32x4*>(part + (long)s * 4 * (2 * 32 * D) + n * 256);
    const bool value = n >= kPieces;
    const View& o = value ? p.dv : p.dk;
    const float f = value ? 1.f : p.scale;
    const int e = value ? n - kPieces : n;
    if (o.p && j < p.Lk) store4<T>((T*)o.p + b * o.b + kh * o.h + (long)j * o.l, part_feature(e, lane), p.d, t[0] * f, t[1] * f, t[2] * f, t[3] * f);
  }
}

// dtable[bucket][head]: the blocks' sums in their order, in 64 bits
__global__ __launch_bounds__(256) void dtable_kernel(const float* __restrict__ part, float* __restrict__ out, int blocks, int buckets, int H) {
  __shared__ double red[256];
  const int head = blockIdx.x, k = blockIdx.y;
  double t = 0.0;
  for (int n = threadIdx.x; n < blocks; n += 256) t += part[((long)head * blocks + n) * buckets + k];
  red[threadIdx.x] = t;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if (threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) out[(long)k * H + head] = (float)red[0];
}

template <typename T, int D, bool BIAS, bool MASK> int backward(const Params& p, float* dtable, hipStream_t s) {
  typedef Tile<T, D> TL;
  constexpr int BN = BwdTile<T, D>::kKeys, BM = BwdTile<T, D>::kRows;
  const size_t slots = 2 * p.max_dist + 1;
  size_t lds = 4 * BN * TL::kRowBytes;
  if (BIAS) lds += slots * sizeof(float);
  OCEAN_TRY(set_lds(dq_kernel<T, D, BIAS, MASK>, lds));
  hipLaunchKernelGGL((dq_kernel<T, D, BIAS, MASK>), dim3((unsigned)((long)p.B * p.H * p.q_tiles * p.parts)), dim3(256), lds, s, p);
  OCEAN_LAUNCH_CHECK();
  if (p.parts > 1) {
    hipLaunchKernelGGL((dq_join_kernel<T, D>), dim3((unsigned)((long)p.B * p.H * p.q_tiles * 4)), dim3(256), 0, s, p);
    OCEAN_LAUNCH_CHECK();
  }
  if (p.dk.p || p.dv.p || p.dtable_part) {
    lds = (4 * BM + (values_in_lds(D * sizeof(T)) ? kRows : 0)) * TL::kRowBytes + 4 * BM * sizeof(float) + (BIAS ? slots * sizeof(float) : 0);
    if (BIAS && p.dtable_part) lds += 4 * slots * sizeof(float);
    OCEAN_TRY(set_lds(dkv_kernel<T, D, BIAS, MASK>, lds));
    const long units = (long)p.B * p.Hk * p.k_tiles, blocks = (long)p.B * p.Hk * (p.causal ? (p.k_tiles + 1) / 2 * 2 : p.k_tiles) * p.segs;
    hipLaunchKernelGGL((dkv_kernel<T, D, BIAS, MASK>), dim3((unsigned)blocks), dim3(256), lds, s, p);
    OCEAN_LAUNCH_CHECK();
    if (p.segs > 1 && (p.dk.p || p.dv.p)) {
      hipLaunchKernelGGL((dkv_join_kernel<T, D>), dim3((unsigned)(units * 4)), dim3(256), 0, s, p);
      OCEAN_LAUNCH_CHECK();
    }
  }
  if (BIAS && p.dtable_part) {
    hipLaunchKernelGGL(dtable_kernel, dim3(p.H, p.buckets), dim3(256), 0, s, p.dtable_part, dtable, p.B * p.k_tiles * p.segs, p.buckets, p.H);
    OCEAN_LAUNCH_CHECK();
  }
  return OCEAN_OK;
}

template <typename T, int D> int backward_b(const Params& p, float* dtable, hipStream_t s) {
  if (p.mask) return p.table ? backward<T, D, true, true>(p, dtable, s) : backward<T, D, false, true>(p, dtable, s);
  return p.table ? backward<T, D, true, false>(p, dtable, s) : backward<T, D, false, false>(p, dtable, s);
}
template <typename T> int backward_d(const Params& p, float* dtable, hipStream_t s) {
  if (p.d <= 32) return backward_b<T, 32>(p, dtable, s);
  if (p.d <= 64) return backward_b<T, 64>(p, dtable, s);
  if (p.d <= 96) return backward_b<T, 96>(p, dtable, s);
  return backward_b<T, 128>(p, dtable, s);
}

}  // namespace

int launch_backward(const Params& p, int type, float* dtable, hipStream_t s) {
  return type == OCEAN_BF16 ? backward_d<__bf16>(p, dtable, s) : backward_d<float>(p, dtable, s);
}

}  // namespace seqattn
