// Entry points of the attention over the 4-bit paged cache: decode rows, then prompt rows. Partials, splits
// and cut tiles are those of the 8-bit cache, and so are the kernels that merge them.
#include "prefill_int4.h"
#include "quant_attention.h"

namespace ts {

struct Int4Kernels {
  static constexpr int kSplitBlocks = kI4SplitBlocks;
  static constexpr bool kFinite = true;

  template <int D>
  static void decode(const Int8DecodeArgs& a, int cus, hipStream_t s) {
    // Every split of the batch, at most as many workgroups as the CUs hold; the rest go round. Where all that the
    // host's bound allows fit at once, each knows its split without the lengths. Us a pass of four layers of 12/2
    // heads of 128 by events over replays, so and by the lookup: one sequence of 6000 tokens 34.5 / 38.4, four of
    // 8000 to 32768 62.5 / 64.8, eight of 500 to 4000 36.5 / 40.4, eight of 500 under a bound of 32768 36.2 / 38.1.
    // Beyond that those past a sequence's end take the others' places: 64 sequences of up to 4096 72 / 60. What the
    // lookup found is kept for up to 64 sequences, a lane each, so that a workgroup need not look up again to find
    // its next item or that there is none: those 64 (632 items in 1024 workgroups: none has a second) 58.4 where a
    // new lookup makes them 60.5, 48 rows beside a chunk of 512 (952 items) 88.5 / 91, 64 of 2000 to 8000 of 8/8
    // heads of 64 (two layers; several items a workgroup) 123 / 131. For up to 256, in LDS, it gained 3 % there and
    // lost as much below.
    const int64_t most = a.num_seqs > a.num_decode ? INT32_MAX : (int64_t)a.num_decode * a.max_splits;
    const int64_t units = most * a.kvh * ((a.group + 15) / 16), cap = (int64_t)i4_decode_groups(D) * cus;
    if (a.group <= 16 && units <= cap)
      decode_int4_direct_kernel<D><<<(unsigned)units, kI4Threads, 0, s>>>(a);
    else if (a.num_seqs <= kWave)
      decode_int4_kernel<D, true><<<(unsigned)(units < cap ? units : cap), kI4Threads, 0, s>>>(a);
    else
      decode_int4_kernel<D, false><<<(unsigned)(units < cap ? units : cap), kI4Threads, 0, s>>>(a);
  }

  template <int D>
  static void prefill(const Int8PrefillArgs& p, hipStream_t s) {
    prefill_int4_kernel<D><<<p.groups, i8_prefill_waves(D) * kWave, 0, s>>>(p);
  }
};

}  // namespace ts

using namespace ts;

extern "C" size_t ts_paged_attention_int4_workspace_bytes(int32_t num_seqs, int32_t num_decode,
                                                          int32_t max_query_len, int32_t max_seq_len,
                                                          int32_t max_prefill_seq_len,
                                                          int32_t num_heads, int32_t num_kv_heads,
                                                          int32_t head_dim, int32_t cu_count) {
  return quant_workspace_bytes<Int4Kernels>(num_seqs, num_decode, max_query_len, max_seq_len, max_prefill_seq_len,
                                            num_heads, num_kv_heads, head_dim, cu_count);
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
                                       void* stream) {
  ts::clear_error();
  return quant_attention<Int4Kernels, false>(
      "paged_attention_int4",
      {q, q_stride_t, q_stride_h, out, out_stride_t, num_tokens, k_cache, v_cache, nullptr, nullptr, num_blocks,
       block_tables, bt_stride, max_blocks_per_seq, seq_lens, query_start_loc, num_seqs, num_decode, max_query_len,
       max_seq_len, max_prefill_seq_len, num_heads, num_kv_heads, head_dim, scale, workspace, workspace_bytes,
       stream});
}
