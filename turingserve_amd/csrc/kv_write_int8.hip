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
// One workgroup owns one (block, KV head, K or V): it holds the whole block in registers (sixteen
// lanes a row; a single new row spread over D / 2 threads gained nothing), so the maximum, the
// scale and every row's rewrite need no other workgroup and the result does not depend on the order
// of anything. A sequence's blocks are found from the step's metadata (query_start_loc, seq_lens,
// block tables), not from slots: the rows of a block then lie together and its owner knows them without
// a search. The rest of the grid (RoPE form) rotates q.
//
// A small launch is bound by its chain of dependent loads (lengths, then block id, then rows,
// positions, codes and scale, then angles), so each link asks for everything it can before it waits:
// 64 appended rows with RoPE, 12/2 heads of 128, 3.5 us (7.7 with a wavefront a block, four rows at a
// time and a division a code). Larger ones are bound by the rows in flight: a chunk of 2048 rows on 4096
// cached 6.5 us, 17 MB or 2.6 TB/s; 8192 rows of 32/8 heads 48 us, 185 MB or 3.8 TB/s, of a copy's 5.0.
// (Rows asked for ahead of the block id cost registers: 6 % there, and nothing gained at the small.)
#include <float.h>

#include "int8_kv.h"
#include "rope.h"

namespace ts {

constexpr int kWriteThreads = 256;

// A thread's share of a row: VEC elements of its first half and their rotation partners in the
// second. Sixteen lanes hold a row (eight at head_dim 16, the others then nothing).
template <int D>
struct RowShare {
  static constexpr int VEC = D >= 32 ? D / 32 : 1;
  static constexpr int LANES = D / (2 * VEC);
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
  int num_seqs, num_decode, chunk_slots;  // workgroups a unit for the blocks of sequences past num_decode
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

// Rotation of a pair of K in 64 bits, rounded once to 32: a row's code is decided by the quotient's
// last bits, and the products (11 x 24 bits) are exact here.
__device__ __forceinline__ void rotate_k(float& lo, float& hi, float cos, float sin) {
  const double c = cos, s = sin, a = lo, b = hi;
  lo = (float)fma(-b, s, a * c);
  hi = (float)fma(a, s, b * c);
}

// The largest |value| of the wavefront; a NaN's bits are above every number's.
__device__ __forceinline__ float largest(float x) { return i8_most(fabsf(x)); }
__device__ __forceinline__ float larger(float a, float b) {
  return __int_as_float(max(__float_as_int(fabsf(a)), __float_as_int(fabsf(b))));
}

// The block's new scale: NaN where a new value is not finite; one that is not finite stays so.
__device__ __forceinline__ float grown(float was, float top) {
  return top <= FLT_MAX ? vmax(was, top / kCodeMax) : __builtin_nanf("");
}

// rint(x / scale) for |x| <= 127 scale, by a reciprocal where that decides it: x * rcp is within
// 127 * 2^-22 of the quotient, so it rounds alike unless it lies that close to a half. `near` is set
// where the division has to be made. (Divisions alone: 24.9 us against 23.3 at 8192 rows, 8 heads of 128.)
__device__ __forceinline__ float code_of(float x, float rcp, bool& near) {
  const float y = x * rcp, c = rintf(y);
  near = near || fabsf(fabsf(y - c) - 0.5f) < 1.f / 16384.f;
  return c;
}
__device__ __forceinline__ float exact_code(float x, float scale) {
  return fminf(fmaxf(rintf(x / scale), -kCodeMax), kCodeMax);
}

// Both segments of a thread's share of row r of a block.
template <int D>
struct RowCodes {
  typedef RowShare<D> R;
  typename R::Codes a, b;
  __device__ __forceinline__ void load(const int8_t* block, int r, int s) {
    a = ld<typename R::Codes>(block + r * D + s * R::VEC);
    b = ld<typename R::Codes>(block + r * D + s * R::VEC + D / 2);
  }
  __device__ __forceinline__ void store(int8_t* block, int r, int s) const {
    st(block + r * D + s * R::VEC, a);
    st(block + r * D + s * R::VEC + D / 2, b);
  }
};

template <int D, bool ROPE, bool IS_K>
__device__ __forceinline__ void write_block(const Int8WriteArgs& a, int j, int64_t blk, int first, int len,
                                            int64_t row0, int h, float* s_top) {
  typedef RowShare<D> R;
  constexpr bool TURN = ROPE && IS_K;
  const int tid = threadIdx.x, r = tid >> 4, s = tid & 15;
  const bool lane = s < R::LANES;
  const int lo = first > 16 * j ? first - 16 * j : 0;      // rows [0, lo) stand there already
  const int hi = min(len - 16 * j, 16);                    // rows [lo, hi) are new
  const int64_t unit = blk * a.kvh + h;
  int8_t* block = (IS_K ? a.kc : a.vc) + unit * kBlockSize * D;
  float* scale = (IS_K ? a.ks : a.vs) + unit;
  const half_t* rows = IS_K ? a.k + h * a.k_sh : a.v + h * a.v_sh;
  const int64_t st_t = IS_K ? a.k_st : a.v_st;
  const bool old = lane && r < lo;
  const float was = lo > 0 ? *scale : 0.f;
  RowCodes<D> kept;
  if (old) kept.load(block, r, s);

  const bool fresh = lane && r >= lo && r < hi;
  RowCodes<D> code;
  typename R::Floats x, y;
  float top = 0.f;
  if (fresh) {
    const int64_t t = row0 + 16 * j + r;
    const typename R::Halves u = ld<typename R::Halves>(rows + t * st_t + s * R::VEC);
    const typename R::Halves v = ld<typename R::Halves>(rows + t * st_t + s * R::VEC + D / 2);
#pragma unroll
    for (int e = 0; e < R::VEC; ++e) x[e] = (float)u[e], y[e] = (float)v[e];
    if (TURN) {
      const int64_t pos = rope_row(a.positions[t], a.max_pos) * (D / 2) + s * R::VEC;
      const typename R::Floats c = ld<typename R::Floats>(a.cos_t + pos);
      const typename R::Floats n = ld<typename R::Floats>(a.sin_t + pos);
#pragma unroll
      for (int e = 0; e < R::VEC; ++e) {
        float f = x[e], g = y[e];
        rotate_k(f, g, c[e], n[e]);
        x[e] = f, y[e] = g;
      }
    }
#pragma unroll
    for (int e = 0; e < R::VEC; ++e) top = larger(top, larger(x[e], y[e]));
  }
  top = largest(top);
  if (tid % kWave == 0) s_top[tid / kWave] = top;
  __syncthreads();
  const float now = grown(was, larger(larger(s_top[0], s_top[1]), larger(s_top[2], s_top[3])));

  if (fresh) {
    const float rcp = now >= FLT_MIN ? 1.f / now : 0.f;    // (scales below the normal numbers divide)
    bool near = !(now >= FLT_MIN);
#pragma unroll
    for (int e = 0; e < R::VEC; ++e) {
      code.a[e] = (int8_t)(int)code_of(x[e], rcp, near);
      code.b[e] = (int8_t)(int)code_of(y[e], rcp, near);
    }
    if (near) {
#pragma unroll
      for (int e = 0; e < R::VEC; ++e) {
        code.a[e] = now > 0.f ? (int8_t)(int)exact_code(x[e], now) : (int8_t)0;
        code.b[e] = now > 0.f ? (int8_t)(int)exact_code(y[e], now) : (int8_t)0;
      }
    }
    code.store(block, r, s);
  }
  if (old && now > was) {                                  // (not where the scale is NaN)
    const float ratio = was / now;
#pragma unroll
    for (int e = 0; e < R::VEC; ++e) {
      kept.a[e] = (int8_t)(int)rintf((float)kept.a[e] * ratio);
      kept.b[e] = (int8_t)(int)rintf((float)kept.b[e] * ratio);
    }
    kept.store(block, r, s);
  }
  if (tid == 0) *scale = now;
}

// A sequence of the step: its rows' positions and the blocks that they fall in.
struct WriteSeq {
  int len, first;                         // tokens after the step, position of its first row in the cache
  int64_t row0;                           // flat row of position 0
  int j0, blocks;                         // its first block, blocks (0: nothing to write)
};

__device__ __forceinline__ WriteSeq write_seq(const Int8WriteArgs& a, int len, int64_t q0, int64_t q1) {
  WriteSeq s = {};
  if (len <= 0 || q0 < 0 || q1 <= q0 || q1 > a.num_tokens) return s;
  const int64_t start = (int64_t)len - (q1 - q0);          // position of row q0
  s.len = len, s.first = start > 0 ? (int)start : 0, s.row0 = q0 - start;
  s.j0 = s.first / kBlockSize;
  s.blocks = max(0, min((len - 1) / kBlockSize, a.max_blocks - 1) - s.j0 + 1);
  return s;
}

// Block `item` of the sequences past num_decode, numbered densely over them: every wavefront looks it
// up for itself, a sequence a lane, 64 at a time. (With as many workgroups a sequence as the longest
// chunk has blocks, 31 prompts of 100 tokens beside one of 8192 took 44 us, 128 of them 158.)
__device__ __forceinline__ bool write_find(const Int8WriteArgs& a, int item, int& b, int& j, WriteSeq& s) {
  const int lane = threadIdx.x % kWave;
  int base = 0;
  for (int first = a.num_decode; first < a.num_seqs; first += kWave) {
    WriteSeq x = {};
    int q0 = 0;
    if (first + lane < a.num_seqs) {
      q0 = a.qsl[first + lane];
      x = write_seq(a, a.seq_lens[first + lane], q0, a.qsl[first + lane + 1]);
    }
    const int sum = i8_scan(x.blocks);
    const uint64_t past = __ballot(base + sum > item);
    if (past) {
      const int i = __ffsll((unsigned long long)past) - 1;
      auto of = [&](int v) { return __builtin_amdgcn_readlane(v, i); };
      b = first + i;
      s.len = of(x.len), s.first = of(x.first), s.j0 = of(x.j0), s.blocks = of(x.blocks);
      s.row0 = (int64_t)of(q0) - of((int)(q0 - x.row0));   // (the start, an int)
      const int at = item - (base + of(sum) - s.blocks);
      j = s.j0 + at;
      return at >= 0 && at < s.blocks;
    }
    base += __builtin_amdgcn_readlane(sum, kWave - 1);
  }
  return false;
}

// Grid: kv_groups workgroups for the K/V blocks (2 KVH units a block: one a decode row, then
// chunk_slots for the blocks of the other sequences, in turn where they are more), then, in the RoPE
// form, one for every 16 rows of a q head. The host's bound on the rows decides the speed only.
template <int D, bool ROPE>
__global__ void __launch_bounds__(kWriteThreads) kv_write_int8_kernel(Int8WriteArgs a) {
  typedef RowShare<D> R;
  __shared__ float s_top[2][kWriteThreads / kWave];        // of two blocks in turn
  if (!ROPE || blockIdx.x < a.kv_groups) {
    const int units = 2 * a.kvh;
    const int slot = (int)(blockIdx.x / (unsigned)units), unit = (int)(blockIdx.x - slot * units);
    int turn = 0;
    auto write = [&](const WriteSeq& s, int b, int j) {
      const int64_t blk = table_entry(a.block_tables + b * a.bt_stride + j);
      if (blk < 0 || blk >= a.num_blocks) return;
      if (unit < a.kvh)
        write_block<D, ROPE, true>(a, j, blk, s.first, s.len, s.row0, unit, s_top[turn]);
      else
        write_block<D, ROPE, false>(a, j, blk, s.first, s.len, s.row0, unit - a.kvh, s_top[turn]);
      turn ^= 1;
    };
    if (slot < a.num_decode) {
      const WriteSeq s = write_seq(a, table_entry(a.seq_lens + slot), table_entry(a.qsl + slot),
                                   table_entry(a.qsl + slot + 1));
      for (int j = s.j0; j < s.j0 + s.blocks; ++j) write(s, slot, j);
    } else {
      WriteSeq s;
      int b, j;
      for (int64_t item = slot - a.num_decode; item <= INT32_MAX && write_find(a, (int)item, b, j, s);
           item += a.chunk_slots)
        write(s, b, j);
    }
  } else if constexpr (ROPE) {
    const int64_t u = blockIdx.x - a.kv_groups;
    const int64_t tile = u / a.heads;
    const int h = (int)(u - tile * a.heads), s = threadIdx.x & 15;
    const int64_t t = tile * 16 + (threadIdx.x >> 4);
    if (t >= a.num_tokens || s >= R::LANES) return;
    const int at = s * R::VEC;
    const half_t* src = a.q + t * a.q_st + (int64_t)h * D;
    half_t* dst = a.q_out + (t * a.heads + h) * D;
    typename R::Halves x = ld<typename R::Halves>(src + at), y = ld<typename R::Halves>(src + D / 2 + at);
    const int64_t pos = rope_row(a.positions[t], a.max_pos) * (D / 2) + at;
    const typename R::Floats c = ld<typename R::Floats>(a.cos_t + pos);
    const typename R::Floats n = ld<typename R::Floats>(a.sin_t + pos);
#pragma unroll
    for (int e = 0; e < R::VEC; ++e) {                     // in fp32, rounded once
      const float f = (float)x[e], g = (float)y[e];
      x[e] = (half_t)fmaf(-g, n[e], f * c[e]);
      y[e] = (half_t)fmaf(f, n[e], g * c[e]);
    }
    st(dst + at, x);
    st(dst + D / 2 + at, y);
  }
}

template <int D>
int launch_write(const Int8WriteArgs& a, bool rope, unsigned grid, hipStream_t s) {
  if (rope)
    kv_write_int8_kernel<D, true><<<grid, kWriteThreads, 0, s>>>(a);
  else
    kv_write_int8_kernel<D, false><<<grid, kWriteThreads, 0, s>>>(a);
  return check_launch(rope ? "rope_kv_write_int8" : "kv_write_int8");
}

static int write_int8(Int8WriteArgs a, bool rope, int D, int max_query_len, const char* what, void* stream) {
  TS_REQUIRE(a.num_tokens >= 0 && a.num_seqs >= 0 && a.num_decode >= 0 && a.num_decode <= a.num_seqs,
             TS_ERR_INVALID_ARG, "%s: num_tokens=%lld num_seqs=%d num_decode=%d", what,
             (long long)a.num_tokens, a.num_seqs, a.num_decode);
  if (a.num_tokens == 0) return TS_OK;
  TS_REQUIRE(a.k && a.v && a.kc && a.vc && a.ks && a.vs &&
                 (a.num_seqs == 0 || (a.block_tables && a.seq_lens && a.qsl)),
             TS_ERR_INVALID_ARG, "%s: null pointer argument", what);
  TS_REQUIRE(a.kvh > 0 && a.num_blocks > 0 && (a.num_seqs == 0 || a.max_blocks > 0) &&
                 a.bt_stride >= a.max_blocks && max_query_len >= 0,
             TS_ERR_INVALID_ARG, "%s: num_kv_heads=%d num_blocks=%lld max_blocks_per_seq=%d "
             "bt_stride=%lld max_query_len=%d", what, a.kvh, (long long)a.num_blocks, a.max_blocks,
             (long long)a.bt_stride, max_query_len);
  TS_REQUIRE(D == 16 || D == 32 || D == 64 || D == 128 || D == 256, TS_ERR_UNSUPPORTED,
             "%s: head_dim %d (16, 32, 64, 128, 256)", what, D);
  const int vec = D >= 32 ? D / 32 : 1;                    // elements of one load
  TS_REQUIRE(a.k_st >= 0 && a.k_sh >= 0 && a.v_st >= 0 && a.v_sh >= 0 && a.k_st % vec == 0 &&
                 a.k_sh % vec == 0 && a.v_st % vec == 0 && a.v_sh % vec == 0 &&
                 aligned(a.k, 2 * vec) && aligned(a.v, 2 * vec),
             TS_ERR_INVALID_ARG, "%s: k and v rows must be %d-byte aligned", what, 2 * vec);
  TS_REQUIRE(aligned(a.kc, 16) && aligned(a.vc, 16) && aligned(a.ks, 4) && aligned(a.vs, 4),
             TS_ERR_INVALID_ARG, "%s: caches must be 16-byte aligned", what);
  // n rows fall in at most (n + 14) / 16 + 1 blocks: less than n / 16 + 2.
  const int64_t chunks = a.num_seqs - a.num_decode, each = ((int64_t)max_query_len + 14) / kBlockSize + 1;
  const int64_t blocks = a.num_tokens / kBlockSize + 2 * chunks;
  const int64_t chunk_slots = chunks * each < blocks ? chunks * each : blocks;
  a.kv_groups = (a.num_decode + chunk_slots) * 2 * a.kvh;
  const int64_t grid = a.kv_groups + (rope ? (a.num_tokens + 15) / 16 * a.heads : 0);
  if (grid == 0) return TS_OK;
  TS_REQUIRE(grid < (1ll << 31), TS_ERR_UNSUPPORTED, "%s: %lld workgroups", what, (long long)grid);
  a.chunk_slots = (int)chunk_slots;
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
