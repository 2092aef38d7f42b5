// The quantising write of a step's new K/V rows into the 8-bit paged cache, with or without RoPE.
//
// For each block that new rows fall in, per KV head and for K and V apart:
//   scale' = max(scale of the rows already there, max|new rows| / 127)
//   code'  = rint(code * (scale / scale'))      rows already there, when the scale grew
//   code   = rint(row / scale')                 new rows
// A block whose row 0 is written starts anew: what its last owner left there has no say. Rows past
// the sequence's end keep their codes. A row that is not finite makes its block's scale NaN, so
// that whatever attends to the block comes out NaN and nothing finite is made up.
//
// One wavefront owns one (block, KV head, K or V): it holds the whole block in registers (four
// lanes a row), so the maximum, the scale and every row's rewrite need no other wavefront and the
// result does not depend on the order of anything. A sequence's blocks are found from the step's
// metadata (query_start_loc, seq_lens, block tables), not from slots: the rows of a block then lie
// together and its owner knows them without a search. The rest of the grid (RoPE form) rotates q.
#include <float.h>

#include "int8_kv.h"
#include "rope.h"

namespace ts {

constexpr int kWriteWaves = 4;

// A lane's share of a row: D / 4 elements in pieces of VEC, piece p at element (4 p + s) * VEC.
// The pieces of the first half of a row and their rotation partners in the second half belong to
// the same lane.
template <int D>
struct RowShare {
  static constexpr int VEC = D >= 64 ? 8 : D / 8;
  static constexpr int PIECES = D / (4 * VEC);
  typedef _Float16 Halves __attribute__((ext_vector_type(VEC)));
  typedef int8_t Codes __attribute__((ext_vector_type(VEC)));
  typedef float Floats __attribute__((ext_vector_type(VEC)));
};

struct Int8WriteArgs {
  const half_t *k, *v;                    // rows of the step (k, v heads)
  int64_t k_st, k_sh, v_st, v_sh;
  int8_t *kc, *vc;
  float *ks, *vs;
  int64_t num_blocks;
  const int32_t* block_tables;
  int64_t bt_stride;
  int max_blocks;
  const int32_t *seq_lens, *qsl;
  int num_seqs, num_decode, chunk_slots;  // slots (wavefront groups) of a sequence past num_decode
  int64_t num_tokens;
  int kvh;
  // RoPE form
  const half_t* q;
  int64_t q_st;
  half_t* q_out;
  const int64_t* positions;
  const float *cos_t, *sin_t;
  int64_t max_pos;
  int heads;
  int64_t kv_groups;                      // workgroups before the first q workgroup
};

// Rotation of a K row in 64 bits, rounded once to 32: a row's code is decided by the quotient's
// last bits, and the products (11 x 24 bits) are exact here.
template <int D, typename V>
__device__ __forceinline__ void rotate_k(V& lo, V& hi, const float* cp, const float* sp) {
#pragma unroll
  for (int e = 0; e < RowShare<D>::VEC; ++e) {
    const double c = cp[e], s = sp[e], a = lo[e], b = hi[e];
    lo[e] = (float)fma(-b, s, a * c);
    hi[e] = (float)fma(a, s, b * c);
  }
}

template <int D, bool ROPE, bool IS_K>
__device__ __forceinline__ void write_block(const Int8WriteArgs& a, int b, int j, int64_t blk, int first,
                                            int len, int64_t row0, int h) {
  typedef RowShare<D> R;
  const int lane = threadIdx.x % kWave, r = lane >> 2, s = lane & 3;
  const int lo = first > 16 * j ? first - 16 * j : 0;      // rows [0, lo) stand there already
  const int hi = min(len - 16 * j, 16);                    // rows [lo, hi) are new
  const bool fresh = r >= lo && r < hi, old = r < lo;
  const int64_t t = row0 + 16 * j + r;                     // flat row of a new row
  const int64_t unit = blk * a.kvh + h;
  int8_t* dst = (IS_K ? a.kc : a.vc) + (unit * kBlockSize + r) * D;
  float* scale = (IS_K ? a.ks : a.vs) + unit;

  typename R::Floats x[R::PIECES];
  typename R::Codes code[R::PIECES];
#pragma unroll
  for (int p = 0; p < R::PIECES; ++p)
#pragma unroll
    for (int e = 0; e < R::VEC; ++e) x[p][e] = 0.f;
  if (fresh) {
    const half_t* src = IS_K ? a.k + t * a.k_st + h * a.k_sh : a.v + t * a.v_st + h * a.v_sh;
#pragma unroll
    for (int p = 0; p < R::PIECES; ++p) {
      const typename R::Halves y = ld<typename R::Halves>(src + (4 * p + s) * R::VEC);
#pragma unroll
      for (int e = 0; e < R::VEC; ++e) x[p][e] = (float)y[e];
    }
    if (ROPE && IS_K) {
      const int64_t pos = rope_row(a.positions[t], a.max_pos) * (D / 2);
#pragma unroll
      for (int p = 0; p < R::PIECES / 2; ++p) {
        const int at = (4 * p + s) * R::VEC;
        rotate_k<D>(x[p], x[p + R::PIECES / 2], a.cos_t + pos + at, a.sin_t + pos + at);
      }
    }
  } else if (old) {
#pragma unroll
    for (int p = 0; p < R::PIECES; ++p) code[p] = ld<typename R::Codes>(dst + (4 * p + s) * R::VEC);
  }
  const float was = lo > 0 ? *scale : 0.f;

  float top = 0.f;
#pragma unroll
  for (int p = 0; p < R::PIECES; ++p)
#pragma unroll
    for (int e = 0; e < R::VEC; ++e) top = vmax(top, fabsf(x[p][e]));   // NaN stays NaN
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) top = vmax(top, shfl_xor(top, m));
  const float now = top <= FLT_MAX ? vmax(was, top / kCodeMax) : __builtin_nanf("");

  if (old && now > was) {                                  // false where the scale is NaN
    const float ratio = was / now;
#pragma unroll
    for (int p = 0; p < R::PIECES; ++p) {
#pragma unroll
      for (int e = 0; e < R::VEC; ++e) code[p][e] = (int8_t)(int)rintf((float)code[p][e] * ratio);
      st(dst + (4 * p + s) * R::VEC, code[p]);
    }
  }
  if (fresh) {
#pragma unroll
    for (int p = 0; p < R::PIECES; ++p) {
#pragma unroll
      for (int e = 0; e < R::VEC; ++e) {
        const float y = now > 0.f ? rintf(x[p][e] / now) : 0.f;
        code[p][e] = (int8_t)(int)fminf(fmaxf(y, -kCodeMax), kCodeMax);
      }
      st(dst + (4 * p + s) * R::VEC, code[p]);
    }
  }
  if (lane == 0) *scale = now;
}

// Grid: kv_groups workgroups for the K/V blocks (slot-major, units of one wavefront each: a
// sequence's first num_decode rows have one slot, the others chunk_slots), then, in the RoPE form,
// one per four (16-row tile, q head) pairs. A sequence with more blocks than slots goes through
// them in steps of its slots, so the host's bound on the rows decides the speed only.
template <int D, bool ROPE>
__global__ void __launch_bounds__(kWriteWaves * kWave) kv_write_int8_kernel(Int8WriteArgs a) {
  typedef RowShare<D> R;
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  if (!ROPE || blockIdx.x < a.kv_groups) {
    const int units = 2 * a.kvh;
    const int64_t u = (int64_t)blockIdx.x * kWriteWaves + wave;
    const int64_t slot = u / units;
    const int unit = (int)(u % units);
    int b, at, step;
    if (slot < a.num_decode) {
      b = (int)slot, at = 0, step = 1;
    } else {
      const int64_t rest = slot - a.num_decode;
      b = a.num_decode + (int)(rest / a.chunk_slots), at = (int)(rest % a.chunk_slots);
      step = a.chunk_slots;
    }
    if (b >= a.num_seqs) return;
    const int len = table_entry(a.seq_lens + b);
    const int64_t q0 = table_entry(a.qsl + b), q1 = table_entry(a.qsl + b + 1);
    if (len <= 0 || q0 < 0 || q1 <= q0 || q1 > a.num_tokens) return;
    const int64_t start = (int64_t)len - (q1 - q0);        // position of the sequence's row q0
    const int first = start > 0 ? (int)start : 0;
    for (int j = first / kBlockSize + at; j <= (len - 1) / kBlockSize && j < a.max_blocks; j += step) {
      const int64_t blk = table_entry(a.block_tables + b * a.bt_stride + j);
      if (blk < 0 || blk >= a.num_blocks) continue;
      if (unit < a.kvh)
        write_block<D, ROPE, true>(a, b, j, blk, first, len, q0 - start, unit);
      else
        write_block<D, ROPE, false>(a, b, j, blk, first, len, q0 - start, unit - a.kvh);
    }
  } else if constexpr (ROPE) {
    const int64_t u = ((int64_t)blockIdx.x - a.kv_groups) * kWriteWaves + wave;
    const int h = (int)(u % a.heads);
    const int64_t t = (u / a.heads) * 16 + (lane >> 2);
    if (t >= a.num_tokens) return;
    const int s = lane & 3;
    const int64_t pos = rope_row(a.positions[t], a.max_pos) * (D / 2);
    const half_t* src = a.q + t * a.q_st + (int64_t)h * D;
    half_t* dst = a.q_out + (t * a.heads + h) * D;
#pragma unroll
    for (int p = 0; p < R::PIECES / 2; ++p) {
      const int at = (4 * p + s) * R::VEC;
      typename R::Halves x = ld<typename R::Halves>(src + at), y = ld<typename R::Halves>(src + D / 2 + at);
#pragma unroll
      for (int e = 0; e < R::VEC; ++e) {                   // in fp32, rounded once
        const float c = a.cos_t[pos + at + e], n = a.sin_t[pos + at + e];
        const float f = (float)x[e], g = (float)y[e];
        x[e] = (half_t)fmaf(-g, n, f * c);
        y[e] = (half_t)fmaf(f, n, g * c);
      }
      st(dst + at, x);
      st(dst + D / 2 + at, y);
    }
  }
}

template <int D>
int launch_write(const Int8WriteArgs& a, bool rope, unsigned grid, hipStream_t s) {
  if (rope)
    kv_write_int8_kernel<D, true><<<grid, kWriteWaves * kWave, 0, s>>>(a);
  else
    kv_write_int8_kernel<D, false><<<grid, kWriteWaves * kWave, 0, s>>>(a);
  return check_launch(rope ? "rope_kv_write_int8" : "kv_write_int8");
}

static int write_int8(Int8WriteArgs a, bool rope, int D, int max_query_len, const char* what, void* stream) {
  TS_REQUIRE(a.num_tokens >= 0 && a.num_seqs >= 0 && a.num_decode >= 0 && a.num_decode <= a.num_seqs,
             TS_ERR_INVALID_ARG, "%s: num_tokens=%lld num_seqs=%d num_decode=%d", what,
             (long long)a.num_tokens, a.num_seqs, a.num_decode);
  if (a.num_tokens == 0) return TS_OK;
  TS_REQUIRE(a.k && a.v && a.kc && a.vc && a.ks && a.vs && a.block_tables && a.seq_lens && a.qsl,
             TS_ERR_INVALID_ARG, "%s: null pointer argument", what);
  TS_REQUIRE(a.kvh > 0 && a.num_blocks > 0 && a.max_blocks > 0 && a.bt_stride >= a.max_blocks &&
                 max_query_len >= 0,
             TS_ERR_INVALID_ARG, "%s: num_kv_heads=%d num_blocks=%lld max_blocks_per_seq=%d "
             "bt_stride=%lld max_query_len=%d", what, a.kvh, (long long)a.num_blocks, a.max_blocks,
             (long long)a.bt_stride, max_query_len);
  TS_REQUIRE(D == 16 || D == 32 || D == 64 || D == 128 || D == 256, TS_ERR_UNSUPPORTED,
             "%s: head_dim %d (16, 32, 64, 128, 256)", what, D);
  const int vec = D >= 64 ? 8 : D / 8;                     // elements of one load
  TS_REQUIRE(a.k_st >= 0 && a.k_sh >= 0 && a.v_st >= 0 && a.v_sh >= 0 && a.k_st % vec == 0 &&
                 a.k_sh % vec == 0 && a.v_st % vec == 0 && a.v_sh % vec == 0 &&
                 aligned(a.k, 2 * vec) && aligned(a.v, 2 * vec),
             TS_ERR_INVALID_ARG, "%s: k and v rows must be %d-byte aligned", what, 2 * vec);
  TS_REQUIRE(aligned(a.kc, 16) && aligned(a.vc, 16) && aligned(a.ks, 4) && aligned(a.vs, 4),
             TS_ERR_INVALID_ARG, "%s: caches must be 16-byte aligned", what);
  // One sequence of max_query_len rows falls in at most this many blocks.
  a.chunk_slots = (int)(((int64_t)max_query_len + 14) / kBlockSize + 1);
  const int64_t slots = a.num_decode + (int64_t)(a.num_seqs - a.num_decode) * a.chunk_slots;
  a.kv_groups = (slots * 2 * a.kvh + kWriteWaves - 1) / kWriteWaves;
  const int64_t q_units = rope ? (a.num_tokens + 15) / 16 * a.heads : 0;
  const int64_t grid = a.kv_groups + (q_units + kWriteWaves - 1) / kWriteWaves;
  if (grid == 0) return TS_OK;
  TS_REQUIRE(grid < (1ll << 31), TS_ERR_UNSUPPORTED, "%s: %lld workgroups", what, (long long)grid);
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  switch (D) {
    case 16: return launch_write<16>(a, rope, (unsigned)grid, s);
    case 32: return launch_write<32>(a, rope, (unsigned)grid, s);
    case 64: return launch_write<64>(a, rope, (unsigned)grid, s);
    case 128: return launch_write<128>(a, rope, (unsigned)grid, s);
    default: return launch_write<256>(a, rope, (unsigned)grid, s);
  }
}

}  // namespace ts

using namespace ts;

extern "C" int ts_kv_write_int8(const void* k, const void* v, int64_t k_stride_t, int64_t k_stride_h,
                                int64_t v_stride_t, int64_t v_stride_h, void* k_cache, void* v_cache,
                                float* k_scale, float* v_scale, int64_t num_blocks,
                                const int32_t* block_tables, int64_t bt_stride,
                                int32_t max_blocks_per_seq, const int32_t* seq_lens,
                                const int32_t* query_start_loc, int32_t num_seqs, int32_t num_decode,
                                int32_t max_query_len, int64_t num_tokens, int32_t num_kv_heads,
                                int32_t head_dim, void* stream) {
  ts::clear_error();
  Int8WriteArgs a = {};
  a.k = static_cast<const half_t*>(k), a.v = static_cast<const half_t*>(v);
  a.k_st = k_stride_t, a.k_sh = k_stride_h, a.v_st = v_stride_t, a.v_sh = v_stride_h;
  a.kc = static_cast<int8_t*>(k_cache), a.vc = static_cast<int8_t*>(v_cache);
  a.ks = k_scale, a.vs = v_scale, a.num_blocks = num_blocks;
  a.block_tables = block_tables, a.bt_stride = bt_stride, a.max_blocks = max_blocks_per_seq;
  a.seq_lens = seq_lens, a.qsl = query_start_loc, a.num_seqs = num_seqs, a.num_decode = num_decode;
  a.num_tokens = num_tokens, a.kvh = num_kv_heads;
  return write_int8(a, false, head_dim, max_query_len, "kv_write_int8", stream);
}

extern "C" int ts_rope_kv_write_int8(const void* qkv, int64_t qkv_stride, const int64_t* positions,
                                     const float* cos_table, const float* sin_table,
                                     int64_t max_position, void* q_out, void* k_cache, void* v_cache,
                                     float* k_scale, float* v_scale, int64_t num_blocks,
                                     const int32_t* block_tables, int64_t bt_stride,
                                     int32_t max_blocks_per_seq, const int32_t* seq_lens,
                                     const int32_t* query_start_loc, int32_t num_seqs,
                                     int32_t num_decode, int32_t max_query_len, int64_t num_tokens,
                                     int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                     void* stream) {
  ts::clear_error();
  TS_REQUIRE(num_heads > 0 && num_kv_heads > 0, TS_ERR_INVALID_ARG,
             "rope_kv_write_int8: num_heads=%d num_kv_heads=%d", num_heads, num_kv_heads);
  if (num_tokens > 0) {
    TS_REQUIRE(qkv && q_out && positions && cos_table && sin_table && max_position > 0,
               TS_ERR_INVALID_ARG, "rope_kv_write_int8: null pointer or empty table");
    TS_REQUIRE(qkv_stride >= (int64_t)(num_heads + 2 * num_kv_heads) * head_dim && qkv_stride % 8 == 0 &&
                   aligned(qkv, 16) && aligned(q_out, 16) && aligned(cos_table, 16) &&
                   aligned(sin_table, 16),
               TS_ERR_INVALID_ARG, "rope_kv_write_int8: qkv rows and tables must be 16-byte aligned");
  }
  Int8WriteArgs a = {};
  const half_t* row = static_cast<const half_t*>(qkv);
  a.k = row ? row + (int64_t)num_heads * head_dim : nullptr;
  a.v = row ? row + (int64_t)(num_heads + num_kv_heads) * head_dim : nullptr;
  a.k_st = a.v_st = qkv_stride, a.k_sh = a.v_sh = head_dim;
  a.kc = static_cast<int8_t*>(k_cache), a.vc = static_cast<int8_t*>(v_cache);
  a.ks = k_scale, a.vs = v_scale, a.num_blocks = num_blocks;
  a.block_tables = block_tables, a.bt_stride = bt_stride, a.max_blocks = max_blocks_per_seq;
  a.seq_lens = seq_lens, a.qsl = query_start_loc, a.num_seqs = num_seqs, a.num_decode = num_decode;
  a.num_tokens = num_tokens, a.kvh = num_kv_heads;
  a.q = row, a.q_st = qkv_stride, a.q_out = static_cast<half_t*>(q_out);
  a.positions = positions, a.cos_t = cos_table, a.sin_t = sin_table, a.max_pos = max_position;
  a.heads = num_heads;
  return write_int8(a, true, head_dim, max_query_len, "rope_kv_write_int8", stream);
}
