// What the attentions over the quantised paged caches share on the host: how a batch is split between
// the decode kernel and the prompt kernel, the workspace, the checks, the launches, and the merge of both
// kernels' partials in one launch (two launches: 46.5 us a layer where one takes 43.5, 16 decode rows beside
// 512 prompt rows on 3000 cached, 12/2 heads of 128, 4 bits). The formats' kernels come in as a class
// `Kernels` with decode<D>(args, cus, stream) and prefill<D>(args, stream), kSplitBlocks, the blocks of a
// split, and kFinite, whether V's values are fp16 numbers (i8_result).
#pragma once

#include "prefill_int8.h"

namespace ts {

// Chunks that the decode kernel takes, in tiles of 16 rows each of which reads the sequence's codes
// anew. Us a call here and in the prefill kernel, D = 128, 12/2 heads:
//   rows per KV head up to kI8ShortRows (their splits are merged): 16 chunks of 8 tokens on 4096 cached
//   31.6 / 37.7, one of 21 on 8192 23.5 / 34.0, 16 of 21 on 4096 41.9 / 42.3; above it, one chunk of
//   42 on 4096 35.9 / 33.3, 16 of 32 57.4 / 46.9;
//   otherwise sequences up to kI8SmallSeq tokens, each tile's in one piece, of kI8SmallWork (tile, pair
//   of blocks) steps at most: 4 chunks of 128 on 2048 34.6 / 40.8, 16 of 128 on 512 35.4 / 41.5; above
//   them 16 of 64 on 2048 51.7 / 44.6, 4 of 512 on 1024 53.3 / 44.1, one of 64 on 4096 35.7 / 33.7.
// The same lines at other heads (of twelve shapes each, one is off by more than a tenth, the last here):
//   14/2 heads of 64: 16 chunks of 8 on 4096 23.4 / 24.0, 16 of 16 27.7 / 25.9, one of 16 on 8192 19.0 /
//   19.1, 4 of 128 on 2048 23.1 / 26.1; above them 16 of 32 on 4096 41.8 / 31.4, one of 64 25.5 / 18.2,
//   4 of 512 on 1024 43.3 / 36.5; 8/8 heads of 64: 16 of 16 on 4096 27.1 / 41.4; above them 4 of 512 on
//   1024 33.5 / 28.5; 16/4 heads of 32: 16 of 8 on 4096 19.0 / 24.4, 16 of 32 (128 rows) 33.7 / 26.9.
// And with the 4-bit cache (the last one is its worst miss):
//   12/2 heads of 128: 16 chunks of 8 on 4096 30.2 / 41.2, 16 of 21 43.3 / 44.2, 16 of 128 on 512 37.3 / 41.0,
//   one of 1000 29.7 / 34.9; above the lines one of 42 on 4096 39.9 / 32.6, 16 of 32 65.0 / 47.5, 4 of 512 on
//   1024 65.1 / 51.1; 14/2 heads of 64: 16 of 8 on 4096 25.6 / 27.5, 16 of 128 on 512 29.7 / 32.9, above one of
//   64 on 4096 30.9 / 21.7; 8/8 heads of 64: 16 of 21 on 4096 36.3 / 45.3; 28/4 heads of 128, above: 16 of 21
//   84.8 / 62.8; 14/2 heads of 64: one of 1000 26.4 / 23.6.
// The choice is one for the batch, by its largest chunk.
constexpr int kI8ShortRows = 128;
constexpr int kI8SmallSeq = 2048;
constexpr int64_t kI8SmallWork = 32768;

// Launch shape and scratch of a batch, from the host's bounds.
struct QuantPlan {
  int small;                             // sequences that the decode kernel takes: the first ones
  int row_slots, max_splits;             // a chunk's rows per KV head that are merged, splits of the longest
  int chunk_parts;                       // a chunk's partials per KV head
  int groups;                            // prefill: workgroups
  size_t dec_o, dec_ml, pre_o, pre_ml;   // offsets of the partials
  size_t joints;
  size_t bytes;
};

static size_t take(size_t& at, size_t bytes) {
  const size_t here = at;
  at += (bytes + 255) / 256 * 256;
  return here;
}

static QuantPlan quant_plan(int split_blocks, int num_seqs, int num_decode, int max_query_len, int max_seq_len,
                            int max_prefill_seq_len, int H, int KVH, int D, int cus) {
  QuantPlan pl = {};
  size_t at = 0;
  const int64_t nb = ((int64_t)(max_seq_len > 0 ? max_seq_len : 0) + kBlockSize - 1) / kBlockSize;
  const int G = H / KVH;
  const int64_t chunk_rows = (int64_t)(max_query_len > 0 ? max_query_len : 1) * G;
  const int64_t P = num_seqs - num_decode;
  const int seq = max_prefill_seq_len > 0 ? max_prefill_seq_len : max_seq_len > 0 ? max_seq_len : 1;
  // (sizes that no batch has may come as bounds: products of four in floating point)
  const double work = (double)P * KVH * ((chunk_rows + 15) / 16) * ((seq + 31) / 32);
  const bool all = P == 0 || chunk_rows <= kI8ShortRows || (seq <= kI8SmallSeq && work <= kI8SmallWork);
  pl.small = all ? num_seqs : num_decode;
  pl.row_slots = (int)(chunk_rows < kI8ShortRows ? chunk_rows : kI8ShortRows);
  if (pl.row_slots < G) pl.row_slots = G;
  pl.max_splits = i8_splits((int)nb, kI8MaxSplits, split_blocks);
  const int row_tiles = (pl.row_slots + 15) / 16;
  pl.chunk_parts = row_tiles == 1 ? pl.row_slots * pl.max_splits : 16 * (pl.max_splits + row_tiles);
  if (pl.chunk_parts < G * pl.max_splits) pl.chunk_parts = G * pl.max_splits;   // (chunks of one row)
  if (pl.small > 0 && pl.max_splits > 1) {
    const size_t rows = (size_t)num_decode * H * pl.max_splits +
                        (size_t)(pl.small - num_decode) * KVH * pl.chunk_parts;
    pl.dec_o = take(at, rows * D * sizeof(float));
    pl.dec_ml = take(at, rows * 2 * sizeof(float));
  }
  if (!all) {
    const int tile_rows = 32 * i8_prefill_waves(D);
    const double tiles = (double)P * KVH * ((chunk_rows + tile_rows - 1) / tile_rows);
    const double shares = tiles * ((seq - 1) / kI8Keys + 1 + kI8TileCost) / kI8MinShare;
    const int most = i8_prefill_groups(D) * cus;
    pl.groups = shares < most ? (shares < 1 ? 1 : (int)shares) : most;
    const size_t r = (size_t)2 * pl.groups * tile_rows;
    pl.pre_o = take(at, r * D * sizeof(float));
    pl.pre_ml = take(at, r * 2 * sizeof(float));
    pl.joints = take(at, pl.groups * sizeof(I8Joint));
  }
  pl.bytes = at;
  return pl;
}

// Work items of the decode kernel at most (splits of tiles of 16 rows), for one KV head. A chunk of one
// row has max_splits for each of its tiles, a longer one 64 over all of them, or one a tile.
static int64_t decode_items(const QuantPlan& pl, int num_decode, int64_t num_tokens, int G) {
  const int64_t row = (int64_t)pl.max_splits * ((G + 15) / 16), chunks = pl.small - num_decode;
  const int64_t split = pl.max_splits > 1 ? (row > kI8MaxSplits ? row : kI8MaxSplits) : 0;
  return num_decode * row + (chunks > 0 ? chunks * (split + 1) + num_tokens * G / 16 : 0);
}

// Rows that the decode kernel's merge goes over.
static int64_t merge_rows(const QuantPlan& pl, int num_decode, int H, int KVH) {
  return (int64_t)num_decode * H + (int64_t)(pl.small - num_decode) * KVH * pl.row_slots;
}

static bool quant_head_dim(int D) { return D == 16 || D == 32 || D == 64 || D == 128 || D == 256; }

// Arguments of an attention entry point.
struct QuantCall {
  const void* q;
  int64_t q_st, q_sh;
  void* out;
  int64_t out_st, num_tokens;
  const void *k_cache, *v_cache;
  const float *k_scale, *v_scale;        // (the 8-bit cache's)
  int64_t num_blocks;
  const int32_t* block_tables;
  int64_t bt_stride;
  int max_blocks;
  const int32_t *seq_lens, *query_start_loc;
  int num_seqs, num_decode, max_query_len, max_seq_len, max_prefill_seq_len, heads, kvh, head_dim;
  float scale;
  void* workspace;
  size_t workspace_bytes;
  void* stream;
};

template <class Kernels>
static size_t quant_workspace_bytes(int num_seqs, int num_decode, int max_query_len, int max_seq_len,
                                    int max_prefill_seq_len, int heads, int kvh, int head_dim, int cus) {
  if (num_seqs <= 0 || num_decode < 0 || num_decode > num_seqs || kvh <= 0 || heads < kvh || heads % kvh != 0 ||
      !quant_head_dim(head_dim))
    return 0;
  return quant_plan(Kernels::kSplitBlocks, num_seqs, num_decode, max_query_len, max_seq_len, max_prefill_seq_len,
                    heads, kvh, head_dim, cus > 0 ? cus : 256).bytes;
}

// The launches of a batch: `rows` rows for the decode kernel's merge (0: it has no sequences), prompts
// unless p.groups is 0.
template <class Kernels, int D>
static void quant_launch(const Int8DecodeArgs& a, int64_t rows, const Int8PrefillArgs& p, int cus, hipStream_t s) {
  constexpr int ROWS = 32 * i8_prefill_waves(D), EACH = Kernels::kSplitBlocks;
  constexpr bool FINITE = Kernels::kFinite;
  const unsigned row_groups = rows > 0 && a.max_splits > 1 ? (unsigned)((rows + kI8Waves - 1) / kI8Waves) : 0;
  const unsigned tile_groups = p.groups > 1 ? (unsigned)(p.groups - 1) * (ROWS / kI8MergeRows) : 0;
  if (rows > 0) Kernels::template decode<D>(a, cus, s);
  if (p.groups > 0) Kernels::template prefill<D>(p, s);
  if (row_groups > 0 && tile_groups > 0)
    int8_merge_kernel<D, ROWS, EACH, FINITE><<<tile_groups + row_groups, 256, 0, s>>>(a, p, (int)tile_groups);
  else if (row_groups > 0)
    decode_int8_merge_kernel<D, EACH, FINITE><<<row_groups, kI8Threads, 0, s>>>(a);
  else if (tile_groups > 0)
    prefill_int8_merge_kernel<D, ROWS, FINITE><<<tile_groups, 256, 0, s>>>(p);
}

template <class Kernels, bool SCALES>
static int quant_attention(const char* what, const QuantCall& c) {
  TS_REQUIRE(c.num_seqs >= 0 && c.num_decode >= 0 && c.num_decode <= c.num_seqs && c.num_decode <= c.num_tokens,
             TS_ERR_INVALID_ARG, "%s: num_seqs=%d num_decode=%d num_tokens=%lld", what, c.num_seqs, c.num_decode,
             (long long)c.num_tokens);
  if (c.num_seqs == 0 || c.num_tokens == 0) return TS_OK;
  TS_REQUIRE(c.q && c.out && c.k_cache && c.v_cache && (!SCALES || (c.k_scale && c.v_scale)) && c.block_tables &&
                 c.seq_lens && c.query_start_loc,
             TS_ERR_INVALID_ARG, "%s: null pointer argument", what);
  TS_REQUIRE(quant_head_dim(c.head_dim), TS_ERR_UNSUPPORTED, "%s: head_dim %d (16, 32, 64, 128, 256)", what,
             c.head_dim);
  TS_REQUIRE(c.kvh > 0 && c.heads > 0 && c.heads % c.kvh == 0, TS_ERR_INVALID_ARG, "%s: %d heads over %d KV heads",
             what, c.heads, c.kvh);
  // (a sequence's tokens are counted in 31 bits)
  TS_REQUIRE(c.num_blocks > 0 && c.max_blocks > 0 && c.max_blocks <= 1 << 26 && c.bt_stride >= c.max_blocks,
             TS_ERR_INVALID_ARG, "%s: num_blocks=%lld max_blocks_per_seq=%d bt_stride=%lld", what,
             (long long)c.num_blocks, c.max_blocks, (long long)c.bt_stride);
  TS_REQUIRE(c.q_st % 8 == 0 && c.q_sh % 8 == 0 && c.q_st >= 0 && c.q_sh >= 0 && c.out_st % 4 == 0 &&
                 c.out_st >= (int64_t)c.heads * c.head_dim && aligned(c.q, 16) && aligned(c.out, 8) &&
                 aligned(c.k_cache, 16) && aligned(c.v_cache, 16) &&
                 (!SCALES || (aligned(c.k_scale, 4) && aligned(c.v_scale, 4))),
             TS_ERR_INVALID_ARG, "%s: misaligned q / out / caches", what);
  TS_REQUIRE(c.scale > 0.f && c.scale < INFINITY, TS_ERR_INVALID_ARG, "%s: scale must be positive and finite", what);
  // The kernels count rows in 31 bits, and splits, of which a sequence has 64 for each tile of rows.
  TS_REQUIRE(c.num_seqs <= 1 << 20 && c.num_tokens < (1ll << 30) / (c.heads / c.kvh), TS_ERR_UNSUPPORTED,
             "%s: %lld tokens of %d sequences", what, (long long)c.num_tokens, c.num_seqs);
  const int group = c.heads / c.kvh;
  QuantPlan pl = quant_plan(Kernels::kSplitBlocks, c.num_seqs, c.num_decode, c.max_query_len, c.max_seq_len,
                            c.max_prefill_seq_len, c.heads, c.kvh, c.head_dim, 256);
  // ... and steps: those of at most `tiles` tiles, each of which sees what its table holds before the
  // chunk and the chunk (the last term: the rounded rate). (None of this hangs on the number of CUs.)
  const int tile_rows = 32 * i8_prefill_waves(c.head_dim);
  const int64_t one = c.num_tokens * group / tile_rows + 1, tiles = one + c.num_seqs - pl.small;
  const int64_t steps = kI8TileCost + 4 + (c.max_blocks + (c.num_tokens + 2 * tile_rows) / kBlockSize) /
                        kI8StepBlocks + one / 4096;
  TS_REQUIRE(merge_rows(pl, c.num_decode, c.heads, c.kvh) < (1ll << 30) &&
                 decode_items(pl, c.num_decode, c.num_tokens, group) * c.kvh < (1ll << 31) &&
                 (pl.small == c.num_seqs || tiles * steps * c.kvh < (1ll << 31)),
             TS_ERR_UNSUPPORTED, "%s: %lld tokens of %d sequences over tables of %d blocks", what,
             (long long)c.num_tokens, c.num_seqs, c.max_blocks);
  int cus = 0;
  int status = device_cu_count(c.stream, &cus);
  if (status != TS_OK) return status;
  pl = quant_plan(Kernels::kSplitBlocks, c.num_seqs, c.num_decode, c.max_query_len, c.max_seq_len,
                  c.max_prefill_seq_len, c.heads, c.kvh, c.head_dim, cus);
  TS_REQUIRE(pl.bytes == 0 || (c.workspace && c.workspace_bytes >= pl.bytes && aligned(c.workspace, 256)),
             TS_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", what, c.workspace_bytes, pl.bytes);
  char* ws = static_cast<char*>(c.workspace);
  const hipStream_t s = reinterpret_cast<hipStream_t>(c.stream);
  Int8DecodeArgs a = {};
  a.q = static_cast<const half_t*>(c.q), a.q_st = c.q_st, a.q_sh = c.q_sh;
  a.out = static_cast<half_t*>(c.out), a.out_st = c.out_st;
  a.kc = static_cast<const int8_t*>(c.k_cache), a.vc = static_cast<const int8_t*>(c.v_cache);
  a.ks = c.k_scale, a.vs = c.v_scale, a.num_blocks = c.num_blocks;
  a.block_tables = c.block_tables, a.bt_stride = c.bt_stride, a.max_blocks = c.max_blocks;
  a.seq_lens = c.seq_lens, a.heads = c.heads, a.kvh = c.kvh;
  a.by_kvh = I8Div::by(c.kvh), a.by_group = I8Div::by(group);
  a.group = group, a.qsl = c.query_start_loc, a.num_tokens = c.num_tokens;
  a.sl2 = c.scale * 1.44269504088896340736f;
  Int8PrefillArgs p = {};
  if (c.num_seqs > pl.small) {
    p.a = a;
    p.a.part_o = reinterpret_cast<float*>(ws + pl.pre_o);
    p.a.part_ml = reinterpret_cast<float*>(ws + pl.pre_ml);
    p.joints = reinterpret_cast<I8Joint*>(ws + pl.joints);
    p.num_seqs = c.num_seqs, p.first = pl.small, p.groups = pl.groups;
    p.rate = i8_rate(32 * i8_prefill_waves(c.head_dim), a.group);
  }
  int64_t rows = 0;
  if (pl.small > 0) {
    a.num_seqs = pl.small, a.num_decode = c.num_decode;
    a.row_slots = pl.row_slots, a.max_splits = pl.max_splits, a.chunk_parts = pl.chunk_parts;
    a.by_slots = I8Div::by(pl.row_slots);
    a.by_units = I8Div::by((int64_t)pl.small * c.kvh < 1 << 30 ? pl.small * c.kvh : 1);   // (not used above)
    a.part_o = reinterpret_cast<float*>(ws + pl.dec_o);
    a.part_ml = reinterpret_cast<float*>(ws + pl.dec_ml);
    rows = merge_rows(pl, c.num_decode, c.heads, c.kvh);
  }
  switch (c.head_dim) {
    case 16: quant_launch<Kernels, 16>(a, rows, p, cus, s); break;
    case 32: quant_launch<Kernels, 32>(a, rows, p, cus, s); break;
    case 64: quant_launch<Kernels, 64>(a, rows, p, cus, s); break;
    case 128: quant_launch<Kernels, 128>(a, rows, p, cus, s); break;
    default: quant_launch<Kernels, 256>(a, rows, p, cus, s); break;
  }
  return check_launch(what);
}

}  // namespace ts
