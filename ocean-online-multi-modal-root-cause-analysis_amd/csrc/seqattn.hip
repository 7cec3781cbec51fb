// Entry points of attention without stored weights: argument checks, launch plan, workspaces.
#include "seqattn.h"

namespace {

using seqattn::Params;
using seqattn::View;
using seqattn::u32x4;

View view(const void* p, const long* st) { View v; v.p = p; v.b = st[0]; v.h = st[1]; v.l = st[2]; return v; }

// the buckets' limits in whole numbers: far bucket exact + k begins at the smallest n >= exact with
// (n / exact)^far >= (max_distance / exact)^k, that is far * ln(n / exact) >= k * ln(max_distance / exact).  In fp64 the two
// sides of an equality differ by a few 1e-16, two different ones by more than 1e-6 (n < 2^12): the slack decides ties.
void bucket_limits(Params& p) {
  const double span = log((double)p.max_dist / p.exact);
  const int far = p.side - p.exact;
  int n = p.exact;
  for (int k = 1; k < far; ++k) {
    while (n < p.max_dist && far * log((double)n / p.exact) < k * span - 1e-9) ++n;
    p.limits[k - 1] = n;
  }
}

// The tile loads of the kernels take 16-byte aligned rows of whole 16-byte chunks.  Inputs that are not (odd features or strides)
// are copied once into the workspace, rows padded with zeros: two passes over an input next to the products over pairs of rows.
template <typename T> __global__ __launch_bounds__(256) void pack_kernel(const View in, u32x4* __restrict__ out, int heads, int L, int d, int chunks, long n) {
  for (long x = (long)blockIdx.x * 256 + threadIdx.x; x < n; x += (long)gridDim.x * 256) {
    const int c = (int)(x % chunks);
    const long row = x / chunks, bh = row / L;
    const T* from = (const T*)in.p + bh / heads * in.b + bh % heads * in.h + row % L * in.l;
    out[x] = seqattn::load_chunk<T>(from, c * seqattn::Mm<T>::kEpc, d);
  }
}

bool loose(const ocean_attention_shape* s, const long* st, int bit) {
  const int E = s->dtype == OCEAN_F32 ? 4 : 8;
  return (s->unaligned >> bit & 1) || s->d % E || st[0] % E || st[1] % E || st[2] % E;
}
size_t packed_floats(const ocean_attention_shape* s, int heads, int L) {
  const int E = s->dtype == OCEAN_F32 ? 4 : 8;
  return (size_t)s->B * heads * L * ((s->d + E - 1) / E) * 4;
}
// copies `v` to *ws if it has to be (advancing *ws); a base that is less aligned than the caller said is refused
int pack(const ocean_attention_shape* s, View* v, const long* st, int bit, int heads, int L, float** ws, hipStream_t stream) {
  if (!loose(s, st, bit)) return reinterpret_cast<uintptr_t>(v->p) % 16 ? OCEAN_ERR_BAD_SHAPE : OCEAN_OK;
  const int E = s->dtype == OCEAN_F32 ? 4 : 8, chunks = (s->d + E - 1) / E;
  const long n = (long)s->B * heads * L * chunks;
  const unsigned blocks = (unsigned)(n < 256L * 4096 ? (n + 255) / 256 : 4096);
  u32x4* out = reinterpret_cast<u32x4*>(*ws);
  if (s->dtype == OCEAN_F32) hipLaunchKernelGGL(pack_kernel<float>, dim3(blocks), dim3(256), 0, stream, *v, out, heads, L, s->d, chunks, n);
  else hipLaunchKernelGGL(pack_kernel<__bf16>, dim3(blocks), dim3(256), 0, stream, *v, out, heads, L, s->d, chunks, n);
  OCEAN_LAUNCH_CHECK();
  *v = View{out, (long)heads * L * chunks * E, (long)L * chunks * E, (long)chunks * E};
  *ws += (size_t)n * 4;
  return OCEAN_OK;
}

// Into how many pieces the loop of every block is split.  A block holds its tile's result in registers, so with few tiles, or with
// `causal` (where one tile's loop is long and another's next to nothing), the chip waits for the longest block.  Pieces cost a round
// trip of fp32 partial sums and a launch that joins them.  The estimate counts both, in microseconds: `tile_us` for one step of the
// loop with the chip full, 4 TB/s for the partial sums.
void plan_pieces(long units, long steps, bool causal, double slots, double tile_us, double piece_bytes, int* pieces, int* per_piece) {
  double best = 1e30;
  *pieces = 1;
  for (int n = 1; n <= 16 && (n == 1 || n <= steps / 2); ++n) {
    const long per = (steps + n - 1) / n;
    double load = causal ? 0.5 * units * steps / slots : ceil(units * n / slots) * per;
    if (causal) load = load + 0.25 * per > per ? load + 0.25 * per : per;
    const double us = load * tile_us + (n > 1 ? 5.0 + 2.0 * units * n * piece_bytes / 4.0e6 : 0.0);
    if (us < best) { best = us; *pieces = n; }
  }
  *per_piece = (int)((steps + *pieces - 1) / *pieces);
}

// A grid holds fewer than 2^32 threads (more wrap around, with no error): no launch may have more blocks of 256 than this.
constexpr long kMaxBlocks = (1L << 24) - 1;

struct Plan { int parts, part_tiles, dq_parts, dq_part_tiles, segs, seg_tiles; size_t part_at, ml_at, packed; int D; int split; int splits; bool fwd_fits, bwd_fits; size_t fwd_floats, bwd_floats, delta_at, parts_at; };

int plan_of(const ocean_attention_shape* s, Plan* pl) {
  *pl = Plan{};
  if (!s) return OCEAN_ERR_NULL;
  if (s->B <= 0 || s->H <= 0 || s->Hk <= 0 || s->Lq <= 0 || s->Lk <= 0 || s->d <= 0 || s->H % s->Hk != 0) return OCEAN_ERR_BAD_SHAPE;
  if (s->dtype != OCEAN_F32 && s->dtype != OCEAN_BF16) return OCEAN_ERR_BAD_SHAPE;
  // within these, scale * log2 e and the log-sums over it (where the launch over keys starts its products) stay finite
  if (!(s->scale >= 1.0e-30f && s->scale <= 1.0e30f)) return OCEAN_ERR_BAD_SHAPE;
  if (s->d < (s->dtype == OCEAN_F32 ? 4 : 8) || s->d > 128) return OCEAN_ERR_UNSUPPORTED;
  if (s->Lq > (1 << 30) || s->Lk > (1 << 30) || s->query_start > (1 << 30) || s->query_start < -(1 << 30)) return OCEAN_ERR_UNSUPPORTED;
  const int G = s->H / s->Hk;
  if ((long)s->Lq * G > (1L << 30)) return OCEAN_ERR_UNSUPPORTED;
  if (s->num_buckets != 0) {
    const int side = s->bidirectional ? s->num_buckets / 2 : s->num_buckets;
    if (s->num_buckets < 0 || (s->bidirectional && s->num_buckets % 2) || side < 2 || s->max_distance <= side / 2) return OCEAN_ERR_BAD_SHAPE;
    if (s->num_buckets > seqattn::kMaxBuckets || s->max_distance > seqattn::kMaxDist) return OCEAN_ERR_UNSUPPORTED;
  }
  pl->D = (s->d + 31) / 32 * 32;
  const long q_tiles = (s->Lq + 127) / 128, blocks = (long)s->B * s->H * q_tiles;
  if (blocks > 0x7fffffffL / 16 || (long)s->B * s->Hk * ((s->Lk + 127) / 128) > 0x7fffffffL / 16) return OCEAN_ERR_UNSUPPORTED;
  // Few queries take the kernel that splits the keys over blocks and packs the heads of a group as one block's rows.
  pl->split = (long)s->Lq * G <= 32;
  const long base = (long)s->B * s->Hk;
  long want = (512 + base - 1) / base;
  const long most = (s->Lk + 511) / 512;
  if (want > most) want = most;
  pl->splits = (int)(want < 1 ? 1 : want);
  pl->fwd_floats = pl->split && pl->splits > 1 ? (size_t)base * pl->splits * 32 * (pl->D + 2) : 0;
  if (!pl->split) {
    if (loose(s, s->k_strides, 1)) pl->fwd_floats += packed_floats(s, s->Hk, s->Lk);
    if (loose(s, s->v_strides, 2)) pl->fwd_floats += packed_floats(s, s->Hk, s->Lk);
  }
  size_t at = 0;                                            // backward: packed inputs (the caller's first), delta, sums by bucket
  if (loose(s, s->q_strides, 0)) at += packed_floats(s, s->H, s->Lq);
  if (loose(s, s->k_strides, 1)) at += packed_floats(s, s->Hk, s->Lk);
  if (loose(s, s->v_strides, 2)) at += packed_floats(s, s->Hk, s->Lk);
  if (loose(s, s->go_strides, 3)) at += packed_floats(s, s->H, s->Lq);
  const size_t rows = (size_t)s->B * s->H * s->Lq;
  pl->delta_at = at;
  pl->parts_at = at + ((rows + 3) & ~size_t(3));
  // Rates measured with the chip full, at 96 and 128 features: a step is 64 (32 in fp32) keys or queries of a tile of 128.  Samples
  // count as Lk keys long, and the forward launch as two blocks a compute unit, also where its build (fp32 or a mask at 128) holds one.
  const bool b16 = s->dtype != OCEAN_F32;
  const int key_step = seqattn::key_tile(b16), row_bytes = pl->D * (b16 ? 2 : 4), query_step = seqattn::query_tile(row_bytes);
  const double wide = pl->D / 128.0, slots = row_bytes > 256 ? 256.0 : 512.0;
  const long key_steps = (s->Lk + key_step - 1) / key_step, query_steps = (long)G * ((s->Lq + query_step - 1) / query_step);
  plan_pieces(blocks, key_steps, s->causal, 512.0, (b16 ? 2.7 : 9.0) * wide, 128.0 * pl->D * 4, &pl->parts, &pl->part_tiles);
  plan_pieces(blocks, key_steps, s->causal, slots, (b16 ? 3.6 : 13.0 * slots / 512.0) * wide, 128.0 * pl->D * 4, &pl->dq_parts, &pl->dq_part_tiles);
  const long tiles_of_keys = (s->Lk + seqattn::kKeyTile - 1) / seqattn::kKeyTile;      // in pairs of equal work with `causal`
  plan_pieces((long)s->B * s->Hk * (s->causal ? (tiles_of_keys + 1) / 2 : tiles_of_keys), query_steps, false, slots,
              (b16 ? 2.9 * query_step / 32.0 : 17.0 * slots / 512.0) * wide, 128.0 * pl->D * 8, &pl->segs, &pl->seg_tiles);
  // the launches and, where there are several pieces, those that join them
  const long with_join = pl->parts > 4 ? pl->parts : pl->parts > 1 ? 4 : 1, dq_with_join = pl->dq_parts > 4 ? pl->dq_parts : pl->dq_parts > 1 ? 4 : 1;
  const long key_tiles = base * (s->causal ? (tiles_of_keys + 1) / 2 * 2 : tiles_of_keys), dkv_with_join = pl->segs > 4 ? pl->segs : pl->segs > 1 ? 4 : 1;
  pl->fwd_fits = (pl->split ? base * pl->splits : blocks * with_join) <= kMaxBlocks;
  pl->bwd_fits = blocks * dq_with_join <= kMaxBlocks && key_tiles * dkv_with_join <= kMaxBlocks;
  if (!pl->split && pl->parts > 1) {
    pl->ml_at = pl->fwd_floats + (size_t)blocks * pl->parts * 128 * pl->D;
    pl->packed = pl->fwd_floats;
    pl->fwd_floats = pl->ml_at + (size_t)blocks * pl->parts * 256;
  }
  const size_t k_tiles = (s->Lk + seqattn::kKeyTile - 1) / seqattn::kKeyTile;
  pl->part_at = pl->parts_at + (((size_t)s->B * s->H * k_tiles * pl->segs * (s->num_buckets > 0 ? s->num_buckets : 0) + 3) & ~size_t(3));
  // partial sums: the two launches use the same place one after the other
  const size_t over_keys = pl->segs > 1 ? (size_t)s->B * s->Hk * k_tiles * pl->segs * seqattn::kKeyTile * pl->D * 2 : 0;
  const size_t over_queries = pl->dq_parts > 1 ? (size_t)blocks * pl->dq_parts * (128 * pl->D + 256) : 0;
  pl->bwd_floats = pl->part_at + (over_keys > over_queries ? over_keys : over_queries);
  return OCEAN_OK;
}

int fill(const ocean_attention_shape* s, const Plan& pl, const void* q, const void* k, const void* v, const uint8_t* mask, const int* lengths,
         const int* starts, const float* table, Params* out) {
  if (!q || !k || !v) return OCEAN_ERR_NULL;
  if ((s->num_buckets > 0) != (table != nullptr)) return OCEAN_ERR_NULL;
  Params& p = *out;
  p = Params{};
  p.q = view(q, s->q_strides); p.k = view(k, s->k_strides); p.v = view(v, s->v_strides);
  p.B = s->B; p.H = s->H; p.Hk = s->Hk; p.G = s->H / s->Hk; p.Lq = s->Lq; p.Lk = s->Lk; p.d = s->d; p.scale = s->scale; p.causal = s->causal != 0;
  p.start0 = s->query_start; p.lengths = lengths; p.starts = starts;
  p.mask = mask; p.mb = s->mask_strides[0]; p.mh = s->mask_strides[1];
  // an axis of one place has no stride: kept_keys and kept_queries know a mask without queries or without keys by its zero there
  p.mi = s->Lq == 1 ? 0 : s->mask_strides[2]; p.mj = s->Lk == 1 ? 0 : s->mask_strides[3];
  p.table = table; p.buckets = s->num_buckets; p.both = s->bidirectional != 0; p.max_dist = s->max_distance;
  if (table) {
    p.side = p.both ? p.buckets / 2 : p.buckets;
    p.exact = p.side / 2;
    bucket_limits(p);
  }
  p.q_tiles = (s->Lq + 127) / 128;
  return OCEAN_OK;
}

}  // namespace

extern "C" {

size_t ocean_attention_fwd_workspace(const ocean_attention_shape* s) { Plan pl; return plan_of(s, &pl) == OCEAN_OK ? pl.fwd_floats : 0; }
size_t ocean_attention_bwd_workspace(const ocean_attention_shape* s) { Plan pl; return plan_of(s, &pl) == OCEAN_OK ? pl.bwd_floats : 0; }

int ocean_attention_fwd(const ocean_attention_shape* s, const void* q, const void* k, const void* v, const uint8_t* mask, const int* lengths,
                        const int* starts, const float* table, float* ws, size_t ws_floats, void* out, float* lse, void* stream) {
  Plan pl;
  Params p;
  OCEAN_TRY(plan_of(s, &pl));
  if (!pl.fwd_fits || (lse && !pl.bwd_fits)) return OCEAN_ERR_UNSUPPORTED;
  OCEAN_TRY(fill(s, pl, q, k, v, mask, lengths, starts, table, &p));
  if (!out || (pl.fwd_floats && !ws)) return OCEAN_ERR_NULL;
  if (ws_floats < pl.fwd_floats) return OCEAN_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(ws) % 16) return OCEAN_ERR_BAD_SHAPE;
  p.o = view(out, s->o_strides);
  p.lse = lse;
  if (pl.split) {
    p.splits = pl.splits;
    const size_t rows = (size_t)s->B * s->Hk * pl.splits * 32;
    p.part_o = ws;
    p.part_ml = ws + rows * pl.D;
  } else {
    p.parts = pl.parts;
    p.part_tiles = pl.part_tiles;
    p.part_o = ws + pl.packed;
    p.part_ml = ws + pl.ml_at;
    OCEAN_TRY(pack(s, &p.k, s->k_strides, 1, s->Hk, s->Lk, &ws, (hipStream_t)stream));
    OCEAN_TRY(pack(s, &p.v, s->v_strides, 2, s->Hk, s->Lk, &ws, (hipStream_t)stream));
  }
  return seqattn::launch_forward(p, s->dtype, (hipStream_t)stream);
}

int ocean_attention_bwd(const ocean_attention_shape* s, const void* q, const void* k, const void* v, const uint8_t* mask, const int* lengths,
                        const int* starts, const float* table, const void* out, const float* lse, const void* d_out, float* ws, size_t ws_floats,
                        void* dq, void* dk, void* dv, float* dtable, void* stream) {
  Plan pl;
  Params p;
  OCEAN_TRY(plan_of(s, &pl));
  if (!pl.bwd_fits) return OCEAN_ERR_UNSUPPORTED;
  OCEAN_TRY(fill(s, pl, q, k, v, mask, lengths, starts, table, &p));
  if (!out || !lse || !d_out || !ws || (dtable && !table)) return OCEAN_ERR_NULL;
  if (ws_floats < pl.bwd_floats) return OCEAN_ERR_WORKSPACE;
  p.o = view(out, s->o_strides); p.go = view(d_out, s->go_strides); p.lse = const_cast<float*>(lse);
  p.dq = view(dq, s->dq_strides); p.dk = view(dk, s->dk_strides); p.dv = view(dv, s->dv_strides);
  p.delta = ws + pl.delta_at;
  p.dtable_part = dtable ? ws + pl.parts_at : nullptr;
  p.part_o = ws + pl.part_at;
  p.part_ml = ws + pl.part_at + (size_t)s->B * s->H * p.q_tiles * pl.dq_parts * 128 * pl.D;
  p.parts = pl.dq_parts;
  p.part_tiles = pl.dq_part_tiles;
  p.k_tiles = (s->Lk + seqattn::kKeyTile - 1) / seqattn::kKeyTile;
  p.segs = pl.segs;
  p.seg_tiles = pl.seg_tiles;
  if (reinterpret_cast<uintptr_t>(ws) % 16) return OCEAN_ERR_BAD_SHAPE;
  OCEAN_TRY(pack(s, &p.q, s->q_strides, 0, s->H, s->Lq, &ws, (hipStream_t)stream));
  OCEAN_TRY(pack(s, &p.k, s->k_strides, 1, s->Hk, s->Lk, &ws, (hipStream_t)stream));
  OCEAN_TRY(pack(s, &p.v, s->v_strides, 2, s->Hk, s->Lk, &ws, (hipStream_t)stream));
  OCEAN_TRY(pack(s, &p.go, s->go_strides, 3, s->H, s->Lq, &ws, (hipStream_t)stream));
  return seqattn::launch_backward(p, s->dtype, dtable, (hipStream_t)stream);
}

}  // extern "C"
