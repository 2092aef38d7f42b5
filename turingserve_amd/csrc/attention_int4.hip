// Entry points of the attention over the 4-bit paged cache: decode rows, then prompt rows. Partials, splits
// and cut tiles are those of the 8-bit cache, and so is the kernel that merges the latter.
#include "prefill_int4.h"
#include "quant_attention.h"

namespace ts {

struct Int4Kernels {
  template <int D>
  static void decode(const Int8DecodeArgs& a, int64_t rows, int cus, void* split_map, hipStream_t s) {
    if (split_map) {
      const int per_slot = a.kvh * ((a.group + 15) / 16);
      const int64_t units = I4Map::entries(a.num_seqs, a.max_splits) * per_slot;
      const int64_t cap = (int64_t)i8_decode_groups(D) * cus;
      decode_int4_mapped_kernel<D><<<(unsigned)(units < cap ? units : cap), kI8Threads, 0, s>>>(
          a, I4Map{static_cast<int*>(split_map)}, I8Div::by(per_slot));
      return;
    }
    // Every split of the batch, at most as many workgroups as the CUs hold; the rest go round.
    const int64_t most = a.num_seqs > a.num_decode ? INT32_MAX : (int64_t)a.num_decode * a.max_splits;
    const int64_t units = most * a.kvh * ((a.group + 15) / 16);
    const int64_t cap = (int64_t)i8_decode_groups(D) * cus;
    decode_int4_kernel<D><<<(unsigned)(units < cap ? units : cap), kI8Threads, 0, s>>>(a);
    if (a.max_splits > 1)
      decode_int4_merge_kernel<D><<<(unsigned)((rows * (D / 4) + kI8Threads - 1) / kI8Threads), kI8Threads, 0, s>>>(a);
  }

  template <int D>
  static void prefill(const Int8PrefillArgs& p, hipStream_t s) {
    constexpr int WAVES = i8_prefill_waves(D), ROWS = 32 * WAVES;
    prefill_int4_kernel<D><<<p.groups, WAVES * kWave, 0, s>>>(p);
    if (p.groups > 1)
      prefill_int8_merge_kernel<D, ROWS><<<(p.groups - 1) * (ROWS / kI8MergeRows), 256, 0, s>>>(p);
  }
};

}  // namespace ts

using namespace ts;

extern "C" size_t ts_paged_attention_int4_workspace_bytes(int32_t num_seqs, int32_t num_decode,
                                                          int32_t max_query_len, int32_t max_seq_len,
                                                          int32_t max_prefill_seq_len,
                                                          int32_t num_heads, int32_t num_kv_heads,
                                                          int32_t head_dim, int32_t cu_count) {
  return quant_workspace_bytes(num_seqs, num_decode, max_query_len, max_seq_len, max_prefill_seq_len, num_heads,
                               num_kv_heads, head_dim, cu_count);
}

// Bytes of the map of a pure-decode step, 0 where it has none: nothing is split, or too many sequences.
static size_t map_bytes(int num_seqs, int heads, int kvh, int head_dim, int max_seq_len) {
  if (num_seqs <= 0 || num_seqs > I4Map::kMaxSeqs || kvh <= 0 || heads < kvh || heads % kvh != 0 ||
      !quant_head_dim(head_dim))
    return 0;
  const QuantPlan pl = quant_plan(num_seqs, num_seqs, 1, max_seq_len, 0, heads, kvh, head_dim, 256);
  return pl.max_splits > 1 ? I4Map::ints(num_seqs, pl.max_splits, kvh, heads / kvh) * sizeof(int) : 0;
}

extern "C" size_t ts_decode_split_map_int4_bytes(int32_t num_seqs, int32_t num_heads, int32_t num_kv_heads,
                                                 int32_t head_dim, int32_t max_seq_len) {
  return map_bytes(num_seqs, num_heads, num_kv_heads, head_dim, max_seq_len);
}

extern "C" int ts_decode_split_map_int4(const int32_t* block_tables, int64_t bt_stride, int32_t max_blocks_per_seq,
                                        int64_t num_blocks, const int32_t* seq_lens, int32_t num_seqs,
                                        int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                        int32_t max_seq_len, void* split_map, size_t split_map_bytes,
                                        void* stream) {
  ts::clear_error();
  TS_REQUIRE(num_seqs >= 0 && num_seqs <= I4Map::kMaxSeqs, TS_ERR_UNSUPPORTED,
             "decode_split_map_int4: %d sequences (0 .. %d; attend without a map)", num_seqs, I4Map::kMaxSeqs);
  if (num_seqs == 0) return TS_OK;
  TS_REQUIRE(num_kv_heads > 0 && num_heads > 0 && num_heads % num_kv_heads == 0, TS_ERR_INVALID_ARG,
             "decode_split_map_int4: %d heads over %d KV heads", num_heads, num_kv_heads);
  TS_REQUIRE(quant_head_dim(head_dim), TS_ERR_UNSUPPORTED, "decode_split_map_int4: head_dim %d (16, 32, 64, 128, 256)",
             head_dim);
  TS_REQUIRE(block_tables && seq_lens, TS_ERR_INVALID_ARG, "decode_split_map_int4: null pointer argument");
  TS_REQUIRE(num_blocks > 0 && max_blocks_per_seq > 0 && max_blocks_per_seq <= 1 << 26 &&
                 bt_stride >= max_blocks_per_seq,
             TS_ERR_INVALID_ARG, "decode_split_map_int4: num_blocks=%lld max_blocks_per_seq=%d bt_stride=%lld",
             (long long)num_blocks, max_blocks_per_seq, (long long)bt_stride);
  const size_t need = map_bytes(num_seqs, num_heads, num_kv_heads, head_dim, max_seq_len);
  if (need == 0) return TS_OK;                             // nothing is split: no map
  TS_REQUIRE(split_map && split_map_bytes >= need && aligned(split_map, 128), TS_ERR_WORKSPACE,
             "decode_split_map_int4: map of %zu bytes, %zu needed (128-byte aligned)", split_map_bytes, need);
  const QuantPlan pl = quant_plan(num_seqs, num_seqs, 1, max_seq_len, 0, num_heads, num_kv_heads, head_dim, 256);
  Int8DecodeArgs a = {};
  a.block_tables = block_tables, a.bt_stride = bt_stride, a.max_blocks = max_blocks_per_seq;
  a.num_blocks = num_blocks, a.seq_lens = seq_lens, a.num_seqs = a.num_decode = num_seqs, a.num_tokens = num_seqs;
  a.heads = num_heads, a.kvh = num_kv_heads, a.group = num_heads / num_kv_heads, a.max_splits = pl.max_splits;
  const int64_t entries = I4Map::entries(num_seqs, pl.max_splits);
  decode_int4_map_kernel<<<(unsigned)((entries + kI8Waves - 1) / kI8Waves), kI8Threads, 0,
                           reinterpret_cast<hipStream_t>(stream)>>>(a, I4Map{static_cast<int*>(split_map)});
  return check_launch("decode_split_map_int4");
}

extern "C" int ts_paged_attention_int4(const void* q, int64_t q_stride_t, int64_t q_stride_h, void* out,
                                       int64_t out_stride_t, int64_t num_tokens, const void* k_cache,
                                       const void* v_cache, int64_t num_blocks, const int32_t* block_tables,
                                       int64_t bt_stride, int32_t max_blocks_per_seq,
                                       const int32_t* seq_lens, const int32_t* query_start_loc,
                                       int32_t num_seqs, int32_t num_decode, int32_t max_query_len,
                                       int32_t max_seq_len, int32_t max_prefill_seq_len,
                                       int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                       float scale, void* workspace, size_t workspace_bytes,
                                       void* stream, void* split_map, size_t split_map_bytes) {
  ts::clear_error();
  if (split_map) {
    const size_t need = map_bytes(num_seqs, num_heads, num_kv_heads, head_dim, max_seq_len);
    TS_REQUIRE(num_decode == num_seqs, TS_ERR_INVALID_ARG,
               "paged_attention_int4: a split map is for steps of decode rows alone (%d of %d sequences)", num_decode,
               num_seqs);
    TS_REQUIRE(need == 0 || (split_map_bytes >= need && aligned(split_map, 128)), TS_ERR_INVALID_ARG,
               "paged_attention_int4: split map of %zu bytes, %zu needed (128-byte aligned)", split_map_bytes, need);
    if (need == 0) split_map = nullptr;
  }
  return quant_attention<Int4Kernels, false>(
      "paged_attention_int4",
      {q, q_stride_t, q_stride_h, out, out_stride_t, num_tokens, k_cache, v_cache, nullptr, nullptr, num_blocks,
       block_tables, bt_stride, max_blocks_per_seq, seq_lens, query_start_loc, num_seqs, num_decode, max_query_len,
       max_seq_len, max_prefill_seq_len, num_heads, num_kv_heads, head_dim, scale, workspace, workspace_bytes,
       stream, split_map});
}
