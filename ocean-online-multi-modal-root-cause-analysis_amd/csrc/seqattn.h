// Attention without stored weights: what the forward and backward kernels share.
//
//   s_ij = scale * q_i . k_j (+ table[bucket(j - pos_i)][head]),  p_i = softmax of s_i over the places that are allowed,
//   o_i = sum_j p_ij v_j,  and a row with no allowed place is zero.
//
// Every product runs on 32x32 matrix instructions.  Their result layout puts one column (lane & 31) and the rows
// 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3), r = 0..15, into a lane.  The kernels form the scores transposed (rows: keys,
// columns: queries) where a wave owns queries, and plain where it owns keys, so that a lane's sixteen probabilities all belong
// to the wave's own row: row sums are in-lane, and the registers are, without any exchange between lanes, the right operand of
// the product that reduces over the other index.  That works because the order of a reduction index is free: the left
// operand is read from LDS in the same order (transposing LDS reads in 16 bits, plain column reads in 32).
#pragma once
#include "common.h"
#include "../../include/ocean_hip.h"
#include <math.h>

namespace seqattn {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kMaxDist = 1024;       // largest max_distance: a head's biases by distance, and four waves' sums of their gradients, stay in LDS
constexpr int kMaxBuckets = 128;

constexpr int kKeyTile = 128;        // keys of a block of the launch over keys
constexpr int query_tile(int row_bytes) { return row_bytes <= 192 ? 64 : 32; }       // and the queries it takes at a time
constexpr int key_tile(bool bits16) { return bits16 ? 64 : 32; }           // keys at a time of the launches over queries
constexpr bool values_in_lds(int row_bytes) { return row_bytes >= 256 && row_bytes < 512; }

struct View { const void* p; long b, h, l; };            // element strides of batch, head, position; the feature's is 1

struct Params {
  View q, k, v, o, go, dq, dk, dv;
  float* lse;                        // [B, H, Lq]: log2 of the row's sum of 2^(score * log2 e); +inf for an empty row
  float* delta;                      // [B, H, Lq]: sum_c do_ic o_ic
  int B, H, Hk, G, Lq, Lk, d;
  float scale;
  int causal, start0;
  const int* lengths;                // [B] or null: keys of each sample
  const int* starts;                 // [B] or null (start0): position of the first query among the keys
  const uint8_t* mask; long mb, mh, mi, mj;      // nonzero = allowed; strides may be 0
  const float* table;                // [buckets, H] or null
  int buckets, side, exact, both, max_dist;      // side: buckets of one side; exact: of them, one per distance
  int limits[kMaxBuckets];           // distances where the far buckets exact+1, exact+2, .. begin
  float* dtable_part;                // [H][B][key tiles][segments][buckets]
  int k_tiles, segs, seg_tiles;      // launch over keys: tiles of 128 keys, segments of their queries, query tiles (of all heads) a segment
  int splits; float* part_o; float* part_ml;     // partial results of split sums
  int q_tiles;                       // tiles of 128 queries
  int parts, part_tiles;             // launches over queries: parts a query tile's keys are split into, key tiles a part
};

// ---------------------------------------------------------------- types
template <typename T> struct Mm;
template <> struct Mm<__bf16> {
  typedef bf16x8 Frag;                                     // one 16-byte chunk: 8 values of the reduction index
  static constexpr int kEpc = 8;
  static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mm<float> {
  typedef f32x4 Frag;
  static constexpr int kEpc = 4;
  static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
};

// ---------------------------------------------------------------- LDS tiles [rows][D], 16-byte chunks permuted within a row
// so that eight lanes on eight consecutive rows (row operand) and four rows x 32 bytes (transposing read) meet all banks.
template <typename T, int D> struct Tile {
  static constexpr int kCh = D * (int)sizeof(T) / 16;      // chunks per row
  static constexpr int kRowBytes = kCh * 16;
  static __device__ __forceinline__ int swz(int row) {
    if (kCh % 8 == 0) return ((row & 3) << 1) | ((row >> 2) & 1);
    return (((row >> 1) & 1) << 1) | ((row >> 2) & 1);
  }
  static __device__ __forceinline__ int at(int row, int chunk) { return row * kRowBytes + ((chunk ^ swz(row)) << 4); }
  // row operand: chunk 2 * step + h of row (lane & 31)
  static __device__ __forceinline__ typename Mm<T>::Frag row_frag(const char* t, int row0, int step, int lane) {
    return *reinterpret_cast<const typename Mm<T>::Frag*>(t + at(row0 + (lane & 31), 2 * step + (lane >> 5)));
  }
};

// The 16 probabilities of a lane as the right operand of a product over the 32 rows they stand for.  The matrix instruction takes
// both operands in one type, so 16-bit inputs' probabilities are rounded to bf16: half a step, up to 2^-8 of each weight, where sums and
// statistics stay fp32.  FINE adds the product of what the rounding left, and 2^-16 remain: where the kernel waits for memory
// that is free (16 tokens over 16384 keys x 128: 139 -> 140 us), where it waits for matrix cores it is not (prompt of 8192: 298 -> 420 us,
// training step 2 x 4096: 756 -> 1028 us), and a bf16 output is 1.4 times as far from exact as its own rounding alone.
template <typename T, bool FINE = false> struct PFrag;
template <bool FINE> struct PFrag<__bf16, FINE> {
  bf16x8 f[2], rest[2];
  __device__ __forceinline__ void set(const f32x16& p) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[s][e] = (__bf16)p[8 * s + e];
        if (FINE) rest[s][e] = (__bf16)(p[8 * s + e] - (float)f[s][e]);
      }
  }
};
template <bool FINE> struct PFrag<float, FINE> {
  f32x16 f;
  __device__ __forceinline__ void set(const f32x16& p) { f = p; }
};

// acc[c][col] += sum over the 32 rows row0.. of tile[row][32 db + c] * p[row][col]
template <int D, bool FINE> __device__ __forceinline__ f32x16 col_mma(const char* t, int row0, int db, int lane, const PFrag<__bf16, FINE>& p, f32x16 acc) {
  typedef Tile<__bf16, D> TL;
  const int gl = lane & 15, grp = lane >> 4;
  const int chunk = db * 4 + 2 * (grp & 1) + ((gl & 3) >> 1), sub = (gl & 1) * 8;
  const int r0 = row0 + 4 * (grp >> 1) + (gl >> 2);
  typedef __attribute__((address_space(3))) s16x4* lds4;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(t + TL::at(r0 + 16 * s, chunk) + sub));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(t + TL::at(r0 + 16 * s + 8, chunk) + sub));
    const bf16x4 l4 = __builtin_bit_cast(bf16x4, lo), h4 = __builtin_bit_cast(bf16x4, hi);
    const bf16x8 a = __builtin_shufflevector(l4, h4, 0, 1, 2, 3, 4, 5, 6, 7);
    acc = Mm<__bf16>::mma(a, p.f[s], acc);
    if (FINE) acc = Mm<__bf16>::mma(a, p.rest[s], acc);
  }
  return acc;
}
template <int D, bool FINE> __device__ __forceinline__ f32x16 col_mma(const char* t, int row0, int db, int lane, const PFrag<float, FINE>& p, f32x16 acc) {
  typedef Tile<float, D> TL;
  const int c = db * 32 + (lane & 31), h = lane >> 5;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int row = row0 + 8 * (r >> 2) + 4 * h + (r & 3);
    const float a = *reinterpret_cast<const float*>(t + TL::at(row, c >> 2) + (c & 3) * 4);
    acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a, p.f[r], acc, 0, 0, 0);
  }
  return acc;
}

// Rows that a mask takes from everything: a key that no query of the sample and head sees (a mask without a query axis), a query
// that sees no key (one without a key axis).  They are not read, so whatever padding they hold reaches no sum.
struct Keep {
  const uint8_t* at = nullptr;
  long step = 0;
  __device__ __forceinline__ bool has(int row) const { return at == nullptr || at[(long)row * step] != 0; }
};

// The same of 32 keys from `first` on as bits, for a kernel that gathers them one tile ahead: a byte read in front of every 16 bytes of
// a cache doubles the time of a padded one (16 tokens over 16384 keys x 128 bf16: 435 us, 197 with the bits; 224 when such keys are read).
struct KeepBits {
  uint32_t bits;
  int first;
  __device__ __forceinline__ bool has(int row) const { return (bits >> (row - first)) & 1u; }
};

// ---------------------------------------------------------------- global memory, any alignment
// 16 bytes of a row of d features from feature e0 on; features past d are zero, memory past the row is not touched.
// A row's last, partial chunk is read as the 16 bytes that end with the row, shifted into place (d >= one chunk).
template <typename T> __device__ __forceinline__ u32x4 load_chunk(const T* row, int e0, int d) {
  constexpr int E = Mm<T>::kEpc;
  u32x4 x = {0u, 0u, 0u, 0u};
  if (e0 + E <= d) {
    __builtin_memcpy(&x, row + e0, 16);
  } else if (e0 < d) {
    __builtin_memcpy(&x, row + d - E, 16);
    const int drop = (E - (d - e0)) * (int)sizeof(T);      // bytes in front that belong to the chunk before
    uint64_t lo = (uint64_t)x[0] | ((uint64_t)x[1] << 32), hi = (uint64_t)x[2] | ((uint64_t)x[3] << 32);
    if (drop >= 8) { lo = hi; hi = 0; }
    const int sh = (drop & 7) * 8;
    if (sh) { lo = (lo >> sh) | (hi << (64 - sh)); hi >>= sh; }
    x = u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
  }
  return x;
}

// a [ROWS][D] tile by 64 * WAVES threads: global -> registers (fetch), registers -> LDS (put)
template <typename T, int D, int ROWS, int THREADS> struct Stage {
  typedef Tile<T, D> TL;
  static constexpr int kN = (ROWS * TL::kCh + THREADS - 1) / THREADS;
  u32x4 r[kN];
  // rows row0.. of a sequence; rows from `rows` on, and those that `keep` leaves out, are zero and not read
  template <typename K> __device__ __forceinline__ void fetch(const T* base, long stride, int row0, int rows, int d, int tid, K keep) {
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int id = tid + n * THREADS, row = id / TL::kCh, c = id % TL::kCh;
      u32x4 x = {0u, 0u, 0u, 0u};
      if (row < ROWS && row0 + row < rows && keep.has(row0 + row)) x = load_chunk<T>(base + (long)(row0 + row) * stride, c * Mm<T>::kEpc, d);
      r[n] = x;
    }
  }
  __device__ __forceinline__ void put(char* t, int tid) const {
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int id = tid + n * THREADS, row = id / TL::kCh, c = id % TL::kCh;
      if (row < ROWS) *reinterpret_cast<u32x4*>(t + TL::at(row, c)) = r[n];
    }
  }
};

// The same tile straight from global memory into LDS, 16 bytes a lane, in flight until wait_tiles(): no registers, no LDS
// writes.  A wave's 64 lanes fill 1024 consecutive bytes, so the permutation within a row is made on the global side.  Needs
// 16-byte aligned rows of whole chunks (the entry points copy other inputs into the workspace first); rows and features past the end come from a line of zeros.
static __device__ const u32x4 kZeros[1] = {{0u, 0u, 0u, 0u}};
template <typename T, int D, int ROWS, int THREADS> struct Async {
  typedef Tile<T, D> TL;
  static constexpr int kN = ROWS * TL::kCh / THREADS, E = Mm<T>::kEpc, kStep = THREADS / TL::kCh;
  static_assert(ROWS * TL::kCh % THREADS == 0, "a tile is whole rounds of the block");
  // every round kStep rows further at the same chunk, so that a lane has one offset and the rounds differ by a scalar
  static constexpr bool kEven = THREADS % TL::kCh == 0 && kStep % 8 == 0;
  long off[kEven ? 1 : kN];
  __device__ __forceinline__ Async(long stride, int tid) {
#pragma unroll
    for (int n = 0; n < (kEven ? 1 : kN); ++n) {
      const int id = tid + n * THREADS, row = id / TL::kCh;
      off[n] = (long)row * stride + ((id % TL::kCh) ^ TL::swz(row)) * E;
    }
  }
  __device__ __forceinline__ void load(char* t, const T* base, long stride, int row0, int rows, int d, int tid, Keep keep = Keep{}) const {
    char* const to = t + __builtin_amdgcn_readfirstlane(tid >> 6) * 1024;
    const T* const first = base + (long)row0 * stride;
    if (row0 + ROWS <= rows && d == D && keep.at == nullptr) {
#pragma unroll
      for (int n = 0; n < kN; ++n) issue(kEven ? first + (long)n * kStep * stride + off[0] : first + off[kEven ? 0 : n], to + n * THREADS * 16);
    } else {
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        const int id = tid + n * THREADS, row = id / TL::kCh, c = (id % TL::kCh) ^ TL::swz(row);
        const T* from = kEven ? first + (long)n * kStep * stride + off[0] : first + off[kEven ? 0 : n];
        if (row0 + row >= rows || c * E >= d || !keep.has(row0 + row)) from = reinterpret_cast<const T*>(kZeros);
        issue(from, to + n * THREADS * 16);
      }
    }
  }
  static __device__ __forceinline__ void issue(const T* from, char* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)to, 16, 0, 0);
  }
};
// every load into LDS of this wave has arrived (vmcnt 0; the other counters are left alone)
__device__ __forceinline__ void wait_tiles() { __builtin_amdgcn_s_waitcnt(0x0F70); }

// a wave's 32 rows as right operand: lane & 31 takes `row` (null: zeros)
template <typename T, int D> struct RowRegs {
  static constexpr int kSteps = D / (2 * Mm<T>::kEpc);
  typename Mm<T>::Frag f[kSteps];
  __device__ __forceinline__ void load(const T* row, int d, int lane) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      u32x4 x = {0u, 0u, 0u, 0u};
      if (row != nullptr) x = load_chunk<T>(row, (2 * s + (lane >> 5)) * Mm<T>::kEpc, d);
      f[s] = __builtin_bit_cast(typename Mm<T>::Frag, x);
    }
  }
};

// acc += rows row0..row0+31 of an LDS tile times a wave's own rows: [tile row][own row]
template <typename T, int D> __device__ __forceinline__ f32x16 row_mma(const char* t, int row0, int lane, const RowRegs<T, D>& own, f32x16 acc) {
#pragma unroll
  for (int s = 0; s < RowRegs<T, D>::kSteps; ++s) acc = Mm<T>::mma(Tile<T, D>::row_frag(t, row0, s, lane), own.f[s], acc);
  return acc;
}

// four features e0..e0+3 of a row, rounded once to the output's type
template <typename T> __device__ __forceinline__ void store4(T* row, int e0, int d, float a, float b, float c, float e) {
  T x[4] = {(T)a, (T)b, (T)c, (T)e};
  if (e0 + 4 <= d) __builtin_memcpy(row + e0, x, 4 * sizeof(T));
  else
#pragma unroll
    for (int n = 0; n < 4; ++n) if (e0 + n < d) row[e0 + n] = x[n];
}
// a product's transposed result [feature][own row]: lane & 31 stores its row
template <typename T, int D> __device__ __forceinline__ void store_row(T* row, const f32x16* acc, float f, int d, int lane) {
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      store4<T>(row, db * 32 + 8 * g + 4 * (lane >> 5), d, acc[db][4 * g] * f, acc[db][4 * g + 1] * f, acc[db][4 * g + 2] * f, acc[db][4 * g + 3] * f);
}

// ---------------------------------------------------------------- between the two halves of a wave
__device__ __forceinline__ float other_half_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float other_half_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}

// ---------------------------------------------------------------- places
__device__ __forceinline__ int keys_of(const Params& p, int b) { return p.lengths ? min(max(p.lengths[b], 0), p.Lk) : p.Lk; }
__device__ __forceinline__ int start_of(const Params& p, int b) { return p.starts ? min(max(p.starts[b], -(1 << 30)), 1 << 30) : p.start0; }

__device__ __forceinline__ Keep kept_keys(const Params& p, int b, int head) {
  return p.mask && p.mi == 0 ? Keep{p.mask + b * p.mb + head * p.mh, p.mj} : Keep{};
}
__device__ __forceinline__ Keep kept_queries(const Params& p, int b, int head) {
  return p.mask && p.mj == 0 ? Keep{p.mask + b * p.mb + head * p.mh, p.mi} : Keep{};
}

// bit e: mask[.., j + e] allows (row: the mask's row of this query; j + e < keys)
__device__ __forceinline__ uint32_t mask4(const Params& p, const uint8_t* row, int j, int keys) {
  uint32_t m = 0;
  if (p.mj == 1 && j + 4 <= keys) {
    uint32_t x;
    __builtin_memcpy(&x, row + j, 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) m |= ((x >> (8 * e)) & 255u) ? 1u << e : 0u;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) if (j + e < keys && row[(long)(j + e) * p.mj]) m |= 1u << e;
  }
  return m;
}

// ---------------------------------------------------------------- position buckets
// dist = key position - query position.  One-sided: only keys behind the query are told apart.  Both: half of the buckets for
// each side.  The first `exact` distances have a bucket each, the far ones begin at limits[], found by bisection.
__device__ __forceinline__ int bucket_of(const Params& p, int dist) {
  const int n = p.both ? abs(dist) : max(-dist, 0);
  int b = n;
  if (n >= p.exact) {
    int lo = 0, hi = p.side - p.exact - 1;                 // how many limits are <= n
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (p.limits[mid] <= n) lo = mid + 1; else hi = mid;
    }
    b = p.exact + lo;
  }
  return p.both && dist > 0 ? b + p.side : b;
}
// lut[x] = bias of distance x - max_dist for one head, times log2 e; beyond max_dist the bucket does not change
__device__ __forceinline__ void fill_bias(const Params& p, int head, float* lut, int tid, int threads) {
  for (int x = tid; x <= 2 * p.max_dist; x += threads) lut[x] = p.table[(long)bucket_of(p, x - p.max_dist) * p.H + head] * kLog2e;
}
__device__ __forceinline__ int dist_slot(const Params& p, int dist) { return min(max(dist, -p.max_dist), p.max_dist) + p.max_dist; }

// Block number -> work: consecutive blocks of one launch go to the eight dies in turn, so a die takes a contiguous run of the
// work list and the blocks that share keys and values share its L2.
__device__ __forceinline__ int die_order(int id, int n) {
  const int per = n >> 3, rem = n & 7, die = id & 7, k = id >> 3;
  return die * per + min(die, rem) + k;
}


// The biases of a lane's sixteen places of a 32x32 block, place r at distance first + step * (8 (r >> 2) + (r & 3)), where d0 is
// the distance at the block's corner (d0 - 31 .. d0 + 31 occur): beyond max_dist there is one bias for all, and a block inside needs no
// clamping, so its reads differ by constants.
template <int STEP> __device__ __forceinline__ f32x16 block_bias(const Params& p, const float* lut, int first, int d0) {
  f32x16 x;
  if (d0 + 31 <= -p.max_dist || d0 - 31 >= p.max_dist) {
    const float far = lut[d0 < 0 ? 0 : 2 * p.max_dist];
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = far;
  } else if (d0 - 31 >= -p.max_dist && d0 + 31 <= p.max_dist) {
    const float* at = lut + p.max_dist + first + (STEP < 0 ? 27 * STEP : 0);
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = at[(STEP < 0 ? -27 * STEP : 0) + STEP * (8 * (r >> 2) + (r & 3))];
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = lut[dist_slot(p, first + STEP * (8 * (r >> 2) + (r & 3)))];
  }
  return x;
}

// Block number -> (key head of a sample, place in its list of `inner` blocks).  A die takes every eighth key head, so that the blocks
// that share keys and values share an L2 and samples of unequal lengths spread over the dies.  With `causal` the lists go through place by place, over all key heads (of the die): they begin with the longest
// loops, and the short ones fill the end (16 heads x 4096: 280 us key head by key head, 236 this way).
__device__ __forceinline__ void work_of(const Params& p, int id, int blocks, int inner, int* bk, int* place) {
  const int groups = p.B * p.Hk;
  if (groups % 8 == 0) {
    const int per = groups / 8, r = id >> 3;
    *bk = (id & 7) + 8 * (p.causal ? r % per : r / inner);
    *place = p.causal ? r / per : r % inner;
  } else if (8 % groups == 0 && inner % (8 / groups) == 0) {
    *bk = (id & 7) % groups;                               // one, two or four key heads: several dies share one's list
    *place = (id >> 3) * (8 / groups) + (id & 7) / groups;
  } else if (p.causal) {
    *bk = id % groups;
    *place = id / groups;
  } else {
    const int r = die_order(id, blocks);
    *bk = r / inner;
    *place = r % inner;
  }
}
// launches over queries: the last query tiles have the most keys with `causal`
__device__ __forceinline__ void rows_work(const Params& p, int id, int blocks, int* bh, int* tile, int* part) {
  int bk, r;
  work_of(p, id, blocks, p.G * p.q_tiles * p.parts, &bk, &r);
  *tile = p.q_tiles - 1 - r / (p.G * p.parts);
  r %= p.G * p.parts;
  *bh = bk * p.G + r / p.parts;
  *part = r % p.parts;
}

// tiles of BN keys that some query of a tile may see
template <int BN> __device__ __forceinline__ int key_tiles(const Params& p, int tile, int keys, int start) {
  const int end = p.causal ? min(keys, start + min((tile + 1) * kKeyTile, p.Lq)) : keys;
  return end > 0 ? (end + BN - 1) / BN : 0;
}

// a wave's 32 rows of partial sums, in the matrix instructions' layout: 64 lanes x 16 bytes a piece, D / 8 pieces
template <int D> __device__ __forceinline__ void store_part(float* part, const f32x16* acc, int lane) {
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<f32x4*>(part + (db * 4 + g) * 256 + lane * 4) = f32x4{acc[db][4 * g], acc[db][4 * g + 1], acc[db][4 * g + 2], acc[db][4 * g + 3]};
}
// and where piece n of lane's row goes: features part_feature(..).. + 3
__device__ __forceinline__ int part_feature(int n, int lane) { return n / 4 * 32 + 8 * (n & 3) + 4 * (lane >> 5); }

// a launch with more than the default 64 KB of LDS has to say so
template <typename K> int set_lds(K kernel, size_t bytes) {
  if (bytes <= 65536) return OCEAN_OK;
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  return e == hipSuccess ? OCEAN_OK : OCEAN_ERR_HIP + (int)e;
}

int launch_forward(const Params& p, int type, hipStream_t s);
int launch_backward(const Params& p, int type, float* dtable, hipStream_t s);

}  // namespace seqattn
