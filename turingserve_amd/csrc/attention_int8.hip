// Entry points of the attention over the 8-bit paged cache: decode rows, then prompt rows.
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
// The choice is one for the batch, by its largest chunk.
constexpr int kI8ShortRows = 128;
constexpr int kI8SmallSeq = 2048;
constexpr int64_t kI8SmallWork = 32768;

// Launch shape and scratch of a batch, from the host's bounds.
struct Int8Plan {
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

static Int8Plan int8_plan(int num_seqs, int num_decode, int max_query_len, int max_seq_len,
                          int max_prefill_seq_len, int H, int KVH, int D, int cus) {
  Int8Plan pl = {};
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
  pl.max_splits = i8_splits((int)nb, kI8MaxSplits);
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
static int64_t decode_items(const Int8Plan& pl, int num_decode, int64_t num_tokens, int G) {
  const int64_t row = (int64_t)pl.max_splits * ((G + 15) / 16), chunks = pl.small - num_decode;
  const int64_t split = pl.max_splits > 1 ? (row > kI8MaxSplits ? row : kI8MaxSplits) : 0;
  return num_decode * row + (chunks > 0 ? chunks * (split + 1) + num_tokens * G / 16 : 0);
}

// Rows that the decode kernel's merge goes over.
static int64_t merge_rows(const Int8Plan& pl, int num_decode, int H, int KVH) {
  return (int64_t)num_decode * H + (int64_t)(pl.small - num_decode) * KVH * pl.row_slots;
}

static bool int8_head_dim(int D) { return D == 16 || D == 32 || D == 64 || D == 128 || D == 256; }

template <int D>
static int launch_decode(const Int8DecodeArgs& a, int64_t rows, int cus, hipStream_t s) {
  // Every split of the batch, at most as many workgroups as the CUs hold; the rest go round.
  const int64_t most = a.num_seqs > a.num_decode ? INT32_MAX : (int64_t)a.num_decode * a.max_splits;
  const int64_t units = most * a.kvh * ((a.group + 15) / 16);
  const int64_t cap = (int64_t)i8_decode_groups(D) * cus;
  decode_int8_kernel<D><<<(unsigned)(units < cap ? units : cap), kI8Threads, 0, s>>>(a);
  if (a.max_splits > 1)
    decode_int8_merge_kernel<D><<<(unsigned)((rows + kI8Waves - 1) / kI8Waves), kI8Threads, 0, s>>>(a);
  return check_launch("paged_attention_int8");
}

template <int D>
static int launch_prefill(const Int8PrefillArgs& p, hipStream_t s) {
  constexpr int WAVES = i8_prefill_waves(D), ROWS = 32 * WAVES;
  prefill_int8_kernel<D><<<p.groups, WAVES * kWave, 0, s>>>(p);
  if (p.groups > 1)
    prefill_int8_merge_kernel<D, ROWS><<<(p.groups - 1) * (ROWS / kI8MergeRows), 256, 0, s>>>(p);
  return check_launch("paged_attention_int8");
}

}  // namespace ts

using namespace ts;

extern "C" size_t ts_paged_attention_int8_workspace_bytes(int32_t num_seqs, int32_t num_decode,
                                                          int32_t max_query_len, int32_t max_seq_len,
                                                          int32_t max_prefill_seq_len,
                                                          int32_t num_heads, int32_t num_kv_heads,
                                                          int32_t head_dim, int32_t cu_count) {
  if (num_seqs <= 0 || num_decode < 0 || num_decode > num_seqs || num_kv_heads <= 0 ||
      num_heads < num_kv_heads || num_heads % num_kv_heads != 0 || !int8_head_dim(head_dim))
    return 0;
  return int8_plan(num_seqs, num_decode, max_query_len, max_seq_len, max_prefill_seq_len, num_heads,
                   num_kv_heads, head_dim, cu_count > 0 ? cu_count : 256).bytes;
}

extern "C" int ts_paged_attention_int8(const void* q, int64_t q_stride_t, int64_t q_stride_h, void* out,
                                       int64_t out_stride_t, int64_t num_tokens, const void* k_cache,
                                       const void* v_cache, const float* k_scale, const float* v_scale,
                                       int64_t num_blocks, const int32_t* block_tables,
                                       int64_t bt_stride, int32_t max_blocks_per_seq,
                                       const int32_t* seq_lens, const int32_t* query_start_loc,
                                       int32_t num_seqs, int32_t num_decode, int32_t max_query_len,
                                       int32_t max_seq_len, int32_t max_prefill_seq_len,
                                       int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                       float scale, void* workspace, size_t workspace_bytes,
                                       void* stream) {
  ts::clear_error();
  TS_REQUIRE(num_seqs >= 0 && num_decode >= 0 && num_decode <= num_seqs && num_decode <= num_tokens,
             TS_ERR_INVALID_ARG, "paged_attention_int8: num_seqs=%d num_decode=%d num_tokens=%lld",
             num_seqs, num_decode, (long long)num_tokens);
  if (num_seqs == 0 || num_tokens == 0) return TS_OK;
  TS_REQUIRE(q && out && k_cache && v_cache && k_scale && v_scale && block_tables && seq_lens &&
                 query_start_loc,
             TS_ERR_INVALID_ARG, "paged_attention_int8: null pointer argument");
  TS_REQUIRE(int8_head_dim(head_dim), TS_ERR_UNSUPPORTED,
             "paged_attention_int8: head_dim %d (16, 32, 64, 128, 256)", head_dim);
  TS_REQUIRE(num_kv_heads > 0 && num_heads > 0 && num_heads % num_kv_heads == 0, TS_ERR_INVALID_ARG,
             "paged_attention_int8: %d heads over %d KV heads", num_heads, num_kv_heads);
  // (a sequence's tokens are counted in 31 bits)
  TS_REQUIRE(num_blocks > 0 && max_blocks_per_seq > 0 && max_blocks_per_seq <= 1 << 26 &&
                 bt_stride >= max_blocks_per_seq,
             TS_ERR_INVALID_ARG, "paged_attention_int8: num_blocks=%lld max_blocks_per_seq=%d bt_stride=%lld",
             (long long)num_blocks, max_blocks_per_seq, (long long)bt_stride);
  TS_REQUIRE(q_stride_t % 8 == 0 && q_stride_h % 8 == 0 && q_stride_t >= 0 && q_stride_h >= 0 &&
                 out_stride_t % 4 == 0 && out_stride_t >= (int64_t)num_heads * head_dim &&
                 aligned(q, 16) && aligned(out, 8) && aligned(k_cache, 16) && aligned(v_cache, 16) &&
                 aligned(k_scale, 4) && aligned(v_scale, 4),
             TS_ERR_INVALID_ARG, "paged_attention_int8: misaligned q / out / caches");
  TS_REQUIRE(scale > 0.f && scale < INFINITY, TS_ERR_INVALID_ARG,
             "paged_attention_int8: scale must be positive and finite");
  // The kernels count rows in 31 bits, and splits, of which a sequence has 64 for each tile of rows.
  TS_REQUIRE(num_seqs <= 1 << 20 && num_tokens < (1ll << 30) / (num_heads / num_kv_heads), TS_ERR_UNSUPPORTED,
             "paged_attention_int8: %lld tokens of %d sequences", (long long)num_tokens, num_seqs);
  const int group = num_heads / num_kv_heads;
  Int8Plan pl = int8_plan(num_seqs, num_decode, max_query_len, max_seq_len, max_prefill_seq_len, num_heads,
                          num_kv_heads, head_dim, 256);
  // ... and steps: those of at most `tiles` tiles, each of which sees what its table holds before the
  // chunk and the chunk (the last term: the rounded rate). (None of this hangs on the number of CUs.)
  const int tile_rows = 32 * i8_prefill_waves(head_dim);
  const int64_t one = num_tokens * group / tile_rows + 1, tiles = one + num_seqs - pl.small;
  const int64_t steps = kI8TileCost + 4 + (max_blocks_per_seq + (num_tokens + 2 * tile_rows) / kBlockSize) /
                        kI8StepBlocks + one / 4096;
  TS_REQUIRE(merge_rows(pl, num_decode, num_heads, num_kv_heads) < (1ll << 30) &&
                 decode_items(pl, num_decode, num_tokens, group) * num_kv_heads < (1ll << 31) &&
                 (pl.small == num_seqs || tiles * steps * num_kv_heads < (1ll << 31)),
             TS_ERR_UNSUPPORTED, "paged_attention_int8: %lld tokens of %d sequences over tables of %d blocks",
             (long long)num_tokens, num_seqs, max_blocks_per_seq);
  int cus = 0;
  int status = device_cu_count(stream, &cus);
  if (status != TS_OK) return status;
  pl = int8_plan(num_seqs, num_decode, max_query_len, max_seq_len, max_prefill_seq_len, num_heads,
                 num_kv_heads, head_dim, cus);
  TS_REQUIRE(pl.bytes == 0 || (workspace && workspace_bytes >= pl.bytes && aligned(workspace, 256)),
             TS_ERR_WORKSPACE, "paged_attention_int8: workspace of %zu bytes, %zu needed", workspace_bytes,
             pl.bytes);
  char* ws = static_cast<char*>(workspace);
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  Int8DecodeArgs a = {};
  a.q = static_cast<const half_t*>(q), a.q_st = q_stride_t, a.q_sh = q_stride_h;
  a.out = static_cast<half_t*>(out), a.out_st = out_stride_t;
  a.kc = static_cast<const int8_t*>(k_cache), a.vc = static_cast<const int8_t*>(v_cache);
  a.ks = k_scale, a.vs = v_scale, a.num_blocks = num_blocks;
  a.block_tables = block_tables, a.bt_stride = bt_stride, a.max_blocks = max_blocks_per_seq;
  a.seq_lens = seq_lens, a.heads = num_heads, a.kvh = num_kv_heads;
  a.by_kvh = I8Div::by(num_kv_heads), a.by_group = I8Div::by(group);
  a.group = group, a.qsl = query_start_loc, a.num_tokens = num_tokens;
  a.sl2 = scale * 1.44269504088896340736f;
  if (pl.small > 0) {
    a.num_seqs = pl.small, a.num_decode = num_decode;
    a.row_slots = pl.row_slots, a.max_splits = pl.max_splits, a.chunk_parts = pl.chunk_parts;
    a.by_slots = I8Div::by(pl.row_slots);
    a.part_o = reinterpret_cast<float*>(ws + pl.dec_o);
    a.part_ml = reinterpret_cast<float*>(ws + pl.dec_ml);
    const int64_t rows = merge_rows(pl, num_decode, num_heads, num_kv_heads);
    switch (head_dim) {
      case 16: status = launch_decode<16>(a, rows, cus, s); break;
      case 32: status = launch_decode<32>(a, rows, cus, s); break;
      case 64: status = launch_decode<64>(a, rows, cus, s); break;
      case 128: status = launch_decode<128>(a, rows, cus, s); break;
      default: status = launch_decode<256>(a, rows, cus, s); break;
    }
    if (status != TS_OK) return status;
  }
  if (num_seqs > pl.small) {
    Int8PrefillArgs p = {};
    p.a = a;
    p.a.part_o = reinterpret_cast<float*>(ws + pl.pre_o);
    p.a.part_ml = reinterpret_cast<float*>(ws + pl.pre_ml);
    p.joints = reinterpret_cast<I8Joint*>(ws + pl.joints);
    p.num_seqs = num_seqs, p.first = pl.small, p.groups = pl.groups;
    p.rate = i8_rate(32 * i8_prefill_waves(head_dim), a.group);
    switch (head_dim) {
      case 16: status = launch_prefill<16>(p, s); break;
      case 32: status = launch_prefill<32>(p, s); break;
      case 64: status = launch_prefill<64>(p, s); break;
      case 128: status = launch_prefill<128>(p, s); break;
      default: status = launch_prefill<256>(p, s); break;
    }
  }
  return status;
}
