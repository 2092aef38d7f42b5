// Entry points of the attention over the 8-bit paged cache: decode rows, then prompt rows.
#include "quant_attention.h"

namespace ts {

struct Int8Kernels {
  static constexpr int kSplitBlocks = kI8SplitBlocks;
  static constexpr bool kFinite = false;                   // (a code times its scale may be any fp32 number)

  template <int D>
  static void decode(const Int8DecodeArgs& a, int cus, hipStream_t s) {
    // Every split of the batch, at most as many workgroups as the CUs hold; the rest go round.
    const int64_t most = a.num_seqs > a.num_decode ? INT32_MAX : (int64_t)a.num_decode * a.max_splits;
    const int64_t units = most * a.kvh * ((a.group + 15) / 16);
    const int64_t cap = (int64_t)i8_decode_groups(D) * cus;
    decode_int8_kernel<D><<<(unsigned)(units < cap ? units : cap), kI8Threads, 0, s>>>(a);
  }

  template <int D>
  static void prefill(const Int8PrefillArgs& p, hipStream_t s) {
    prefill_int8_kernel<D><<<p.groups, i8_prefill_waves(D) * kWave, 0, s>>>(p);
  }
};

}  // namespace ts

using namespace ts;

extern "C" size_t ts_paged_attention_int8_workspace_bytes(int32_t num_seqs, int32_t num_decode,
                                                          int32_t max_query_len, int32_t max_seq_len,
                                                          int32_t max_prefill_seq_len,
                                                          int32_t num_heads, int32_t num_kv_heads,
                                                          int32_t head_dim, int32_t cu_count) {
  return quant_workspace_bytes<Int8Kernels>(num_seqs, num_decode, max_query_len, max_seq_len, max_prefill_seq_len, num_heads,
                               num_kv_heads, head_dim, cu_count);
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
  return quant_attention<Int8Kernels, true>(
      "paged_attention_int8",
      {q, q_stride_t, q_stride_h, out, out_stride_t, num_tokens, k_cache, v_cache, k_scale, v_scale, num_blocks,
       block_tables, bt_stride, max_blocks_per_seq, seq_lens, query_start_loc, num_seqs, num_decode, max_query_len,
       max_seq_len, max_prefill_seq_len, num_heads, num_kv_heads, head_dim, scale, workspace, workspace_bytes,
       stream});
}
