// The quantising write of a step's new K/V rows into the 4-bit paged cache, with or without RoPE, and the
// reading of its blocks as fp16. For each row, KV head and group of 32 channels
//   low  = fp16(least value),  step = (largest value - low) / 15 in fp32, rounded towards zero to fp16,
//   code = rint((value - low) / step) within 0 .. 15 (0 where step is 0),
// fp32 throughout, divisions rounded correctly. The step is rounded towards zero so that no code stands for
// more than the largest value (the nearest one could leave the fp16 range at 65504); that costs the group's
// upper end at most 15 units in the step's last place: 0.015 of a normal step (2^-14 or more), where a code is
// off by half of one, and 15 * 2^-24 where the step is subnormal or 0, which may be all of a narrow group's
// span.
//
// A thread holds an octet of a row of K or of V, those of a (token, KV head) side by side in a wavefront: a
// group's extremes come over 4 neighbouring lanes, a rotation's partner from a second load, and whether
// the row is finite from a ballot. q (RoPE form) is rotated by the rest of the grid, two octets a thread.
//
// 12/2 heads of 128 with RoPE: 64 appended rows 3.7 us (2.3 at least, a launch's chain slot and position ->
// row and angles -> 64-bit products -> quotients), 2048 rows 6.5 us for 19.1 MB (2.9 TB/s, the same chain over
// five workgroups a CU; a thread loads 64 bytes of angles for its 16 of a row, anew for each of a token's 14
// rotated heads, and the other half of K a second time). With two octets of K and of V a thread, so that a rotation's pairs met in one, it
// took 6.8 and 10.9: a fourth of the threads, each with four times the chain. The correctly rounded divisions
// were most of the arithmetic; i4_word leaves all but the doubtful ones out.
#include "int4_kv.h"
#include "decode_int8.h"
#include "rope.h"

namespace ts {

constexpr int kI4WriteThreads = 256;

struct Int4WriteArgs {
  const half_t *k, *v;                    // rows of the step (k, v heads)
  int64_t k_st, k_sh, v_st, v_sh;
  uint8_t *kc, *vc;
  int64_t num_blocks;
  const int64_t* slots;
  int num_tokens, kvh;
  I8Div by_kvh;
  // RoPE form
  const half_t* q;
  int64_t q_st;
  half_t* q_out;
  const int64_t* positions;
  const float *cos_t, *sin_t;
  int64_t max_pos;
  int heads, kv_groups;                   // workgroups before the first of q
  I8Div by_heads;
};

struct I4Rotation {
  float4_t c[2], n[2];                    // cosines and sines of 8 pairs
  __device__ __forceinline__ void load(const Int4WriteArgs& a, int t, int half_dim, int at) {
    const int64_t pos = rope_row(a.positions[t], a.max_pos) * half_dim + at;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      c[i] = ld<float4_t>(a.cos_t + pos + 4 * i), n[i] = ld<float4_t>(a.sin_t + pos + 4 * i);
  }
};

// rint((x - low) / step) within 0 .. 15 of 8 channels, as an octet's word. By the reciprocal where that
// decides it: the quotient is below 31 (a subnormal step may be little more than half the span's fifteenth), the
// product with v_rcp_f32's result (one unit in the last place) within 31 * 1.5 * 2^-23 < 2^-17 of it, so it
// rounds alike unless it lies that close to a half; then the division is made.
__device__ __forceinline__ uint32_t i4_word(const float (&x)[8], float low, float step) {
  const float rcp = __builtin_amdgcn_rcpf(step);           // (steps are 2^-24 at least, or 0)
  uint32_t w = 0;
  float worst = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float y = (x[e] - low) * rcp, c = rintf(y);
    worst = fmaxf(worst, fabsf(y - c));
    w |= (uint32_t)(int)__builtin_amdgcn_fmed3f(c, 0.f, 15.f) << 4 * (e / 2 + 4 * (e % 2));
  }
  if (worst > 0.5f - 1.f / 65536.f) {
    w = 0;
#pragma unroll 1
    for (int e = 0; e < 8; ++e) {
      float v = x[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) v = i == e ? x[i] : v;
      const float c = fminf(fmaxf(rintf((v - low) / step), 0.f), 15.f);
      w |= (uint32_t)(int)c << 4 * (e / 2 + 4 * (e % 2));
    }
  }
  return step > 0.f ? w : 0;
}

template <int D, bool ROPE>
__device__ __forceinline__ void i4_write_kv(const Int4WriteArgs& a) {
  typedef I4Unit<D> U;
  constexpr int OCTETS = D / 8, LANES = U::GROUP / 8, PER = 2 * OCTETS;   // lanes of a group, of a (token, head)
  const int item = (int)(blockIdx.x * (kI4WriteThreads / PER) + threadIdx.x / PER), in = threadIdx.x % PER;
  const int t = a.by_kvh(item), h = item - t * a.kvh, side = in / OCTETS, octet = in % OCTETS;
  if (t >= a.num_tokens) return;                           // (all lanes of an item)
  const int64_t slot = a.slots[t];
  const half_t* row = side == 0 ? a.k + t * a.k_st + h * a.k_sh : a.v + t * a.v_st + h * a.v_sh;
  const half8_t own = ld<half8_t>(row + 8 * octet);
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (float)own[e];
  if (ROPE && side == 0) {
    // in 64 bits, where the products are exact, rounded once to 32: a quotient's last bits decide a code
    const half8_t other = ld<half8_t>(row + 8 * (octet ^ (OCTETS / 2)));
    I4Rotation r;
    r.load(a, t, D / 2, 8 * (octet % (OCTETS / 2)));
    const double sign = octet < OCTETS / 2 ? -1.0 : 1.0;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      x[e] = (float)fma((double)(float)other[e] * sign, (double)r.n[e / 4][e % 4],
                        (double)x[e] * (double)r.c[e / 4][e % 4]);
  }
  float lo = x[0], hi = x[0];
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    lo = fminf(lo, x[e]), hi = fmaxf(hi, x[e]);
    bad = bad || !(fabsf(x[e]) <= 65504.f);
  }
  if constexpr (LANES > 1) lo = fminf(lo, i8_lane<0xb1>(lo)), hi = fmaxf(hi, i8_lane<0xb1>(hi));   // 1 0 3 2
  if constexpr (LANES > 2) lo = fminf(lo, i8_lane<0x4e>(lo)), hi = fmaxf(hi, i8_lane<0x4e>(hi));   // 2 3 0 1
  const uint64_t lost = __ballot(bad), mine = PER == kWave ? ~0ull : ((1ull << PER % kWave) - 1)
                                                                       << (threadIdx.x % kWave / PER * PER);
  half_t low = (half_t)lo + (half_t)0.f;                   // (-0 as 0, also where a number rounds to it)
  const float span = fmaxf(hi - (float)low, 0.f) / 15.f;
  half_t step = (half_t)span;
  if ((float)step > span) step = __builtin_bit_cast(half_t, (uint16_t)(__builtin_bit_cast(uint16_t, step) - 1));
  uint32_t w = i4_word(x, (float)low, (float)step);
  if (lost & mine) w = 0, step = (half_t)0.f, low = (half_t)__builtin_nanf("");
  if (slot < 0 || slot >= a.num_blocks * kBlockSize) return;
  const int64_t unit = ((slot / kBlockSize) * a.kvh + h) * U::BYTES;
  const int at = (int)(slot % kBlockSize), group = octet / LANES;
  if (side == 0) {
    st<uint32_t>(a.kc + unit + U::k_word(at, octet), w);
    if (octet % LANES == 0) st<half2_t>(a.kc + unit + U::k_numbers(at, group), half2_t{step, low});
  } else {
    st<uint32_t>(a.vc + unit + U::v_word(at, octet), w);
    if (octet % LANES == 0) {
      st<half_t>(a.vc + unit + U::v_numbers(at, group), step);
      st<half_t>(a.vc + unit + U::v_numbers(at, group) + 8, low);
    }
  }
}

template <int D, bool ROPE>
__global__ void __launch_bounds__(kI4WriteThreads) kv_write_int4_kernel(Int4WriteArgs a) {
  if (!ROPE || (int)blockIdx.x < a.kv_groups) return i4_write_kv<D, ROPE>(a);
  if constexpr (ROPE) {
    constexpr int PER = D / 16;
    const int item = (int)((blockIdx.x - a.kv_groups) * (kI4WriteThreads / PER) + threadIdx.x / PER);
    const int t = a.by_heads(item), h = item - t * a.heads, at = 8 * (threadIdx.x % PER);
    if (t >= a.num_tokens) return;
    const half_t* src = a.q + t * a.q_st + (int64_t)h * D + at;
    half_t* dst = a.q_out + ((int64_t)t * a.heads + h) * D + at;
    const half8_t x = ld<half8_t>(src), y = ld<half8_t>(src + D / 2);
    I4Rotation r;
    r.load(a, t, D / 2, at);
    half8_t p, s;
#pragma unroll
    for (int e = 0; e < 8; ++e) {                          // in fp32, rounded once
      const float f = (float)x[e], g = (float)y[e], c = r.c[e / 4][e % 4], n = r.n[e / 4][e % 4];
      p[e] = (half_t)fmaf(-g, n, f * c);
      s[e] = (half_t)fmaf(f, n, g * c);
    }
    st(dst, p);
    st(dst + D / 2, s);
  }
}

struct Int4ReadArgs {
  const uint8_t* cache;
  const int32_t* blocks;
  half_t* out;
  int64_t num_blocks;
  int n, kvh, units;                      // blocks asked for; units of the result
  I8Div by_n, by_kvh;
};

// Sixteen bytes of a V unit are an octet of four rows, so a thread takes an octet of four rows: of K a word a
// row (consecutive lanes have consecutive words, and the rows of a request follow one another), of V all of
// them at once. D / 2 threads a unit; every store is 16 bytes, of whole rows. Bound by memory: 32 sequences
// of 14/2 heads of 64, 8 layers, 371 MB in 64.5 us (5.7 TB/s; 101 us with an octet of one row a thread, whose
// V words are 4 bytes in 64); a small call is its launch (94 blocks of 4 layers 3.6 us).
template <int D>
__global__ void __launch_bounds__(kI4WriteThreads) kv_read_int4_kernel(Int4ReadArgs a) {
  typedef I4Unit<D> U;
  constexpr int PER = D / 2, OCTETS = D / 8;
  const int unit = (int)(blockIdx.x * (kI4WriteThreads / PER) + threadIdx.x / PER), in = threadIdx.x % PER;
  if (unit >= a.units) return;
  const int lb = a.by_kvh(unit), h = unit - lb * a.kvh;    // (layer, K or V) and block; head
  const int side = a.by_n(lb);
  const int blk = clamp_block(a.blocks[lb - side * a.n], a.num_blocks);
  const uint8_t* src = a.cache + (((int64_t)side * a.num_blocks + blk) * a.kvh + h) * U::BYTES;
  half_t* dst = a.out + (int64_t)unit * (kBlockSize * D);
  const int quad = in / OCTETS, octet = in % OCTETS, group = 8 * octet / U::GROUP;
  const I4Bits k;
  uint32_t w[4], n[4];
  const bool is_v = side & 1;
  if (!is_v) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      w[r] = ld<uint32_t>(src + U::k_word(4 * r + quad, octet));
      n[r] = ld<uint32_t>(src + U::k_numbers(4 * r + quad, group));
    }
  } else {
    const uint4_t v = ld<uint4_t>(src + U::v_word(4 * quad, octet));
    const uint4_t m = ld<uint4_t>(src + U::v_numbers(4 * quad, group));
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      w[r] = v[r];
      n[r] = __builtin_amdgcn_perm(m[2 + r / 2], m[r / 2], r % 2 ? 0x07060302u : 0x05040100u);   // step, low
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
    st<half8_t>(dst + (is_v ? 4 * quad + r : 4 * r + quad) * D + 8 * octet, i4_octet(k, w[r], n[r]));
}

static bool int4_head_dim(int D) { return D == 16 || D == 32 || D == 64 || D == 128 || D == 256; }

template <int D>
static void launch_write(const Int4WriteArgs& a, bool rope, unsigned grid, hipStream_t s) {
  if (rope)
    kv_write_int4_kernel<D, true><<<grid, kI4WriteThreads, 0, s>>>(a);
  else
    kv_write_int4_kernel<D, false><<<grid, kI4WriteThreads, 0, s>>>(a);
}

static int write_int4(Int4WriteArgs a, bool rope, int64_t num_tokens, int D, const char* what, void* stream) {
  TS_REQUIRE(num_tokens >= 0, TS_ERR_INVALID_ARG, "%s: num_tokens=%lld", what, (long long)num_tokens);
  if (num_tokens == 0) return TS_OK;
  TS_REQUIRE(a.k && a.v && a.kc && a.vc && a.slots, TS_ERR_INVALID_ARG, "%s: null pointer argument", what);
  TS_REQUIRE(a.kvh > 0 && a.num_blocks > 0, TS_ERR_INVALID_ARG, "%s: num_kv_heads=%d num_blocks=%lld", what, a.kvh,
             (long long)a.num_blocks);
  TS_REQUIRE(int4_head_dim(D), TS_ERR_UNSUPPORTED, "%s: head_dim %d (16, 32, 64, 128, 256)", what, D);
  TS_REQUIRE(a.k_st >= 0 && a.k_sh >= 0 && a.v_st >= 0 && a.v_sh >= 0 && a.k_st % 8 == 0 && a.k_sh % 8 == 0 &&
                 a.v_st % 8 == 0 && a.v_sh % 8 == 0 && aligned(a.k, 16) && aligned(a.v, 16),
             TS_ERR_INVALID_ARG, "%s: k and v rows must be 16-byte aligned", what);
  TS_REQUIRE(aligned(a.kc, 16) && aligned(a.vc, 16), TS_ERR_INVALID_ARG, "%s: caches must be 16-byte aligned", what);
  const int64_t units = (rope ? (int64_t)a.heads : 0) + a.kvh;
  TS_REQUIRE(units < (1ll << 30) && num_tokens < (1ll << 30) / units, TS_ERR_UNSUPPORTED,
             "%s: %lld tokens of %lld heads", what, (long long)num_tokens, (long long)units);
  a.num_tokens = (int)num_tokens, a.by_kvh = I8Div::by(a.kvh);
  a.kv_groups = (int)((num_tokens * a.kvh * (D / 4) + kI4WriteThreads - 1) / kI4WriteThreads);
  int64_t grid = a.kv_groups;
  if (rope) {
    a.by_heads = I8Div::by(a.heads);
    grid += (num_tokens * a.heads * (D / 16) + kI4WriteThreads - 1) / kI4WriteThreads;
  }
  TS_REQUIRE(grid < (1ll << 31), TS_ERR_UNSUPPORTED, "%s: %lld workgroups", what, (long long)grid);
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  switch (D) {
    case 16: launch_write<16>(a, rope, (unsigned)grid, s); break;
    case 32: launch_write<32>(a, rope, (unsigned)grid, s); break;
    case 64: launch_write<64>(a, rope, (unsigned)grid, s); break;
    case 128: launch_write<128>(a, rope, (unsigned)grid, s); break;
    default: launch_write<256>(a, rope, (unsigned)grid, s); break;
  }
  return check_launch(what);
}

}  // namespace ts

using namespace ts;

extern "C" int ts_kv_write_int4(const void* k, const void* v, int64_t k_stride_t, int64_t k_stride_h,
                                int64_t v_stride_t, int64_t v_stride_h, void* k_cache, void* v_cache,
                                int64_t num_blocks, const int64_t* slot_mapping, int64_t num_tokens,
                                int32_t num_kv_heads, int32_t head_dim, void* stream) {
  ts::clear_error();
  Int4WriteArgs a = {};
  a.k = static_cast<const half_t*>(k), a.v = static_cast<const half_t*>(v);
  a.k_st = k_stride_t, a.k_sh = k_stride_h, a.v_st = v_stride_t, a.v_sh = v_stride_h;
  a.kc = static_cast<uint8_t*>(k_cache), a.vc = static_cast<uint8_t*>(v_cache);
  a.num_blocks = num_blocks, a.slots = slot_mapping, a.kvh = num_kv_heads;
  return write_int4(a, false, num_tokens, head_dim, "kv_write_int4", stream);
}

extern "C" int ts_rope_kv_write_int4(const void* qkv, int64_t qkv_stride, const int64_t* positions,
                                     const float* cos_table, const float* sin_table, int64_t max_position,
                                     void* q_out, void* k_cache, void* v_cache, int64_t num_blocks,
                                     const int64_t* slot_mapping, int64_t num_tokens, int32_t num_heads,
                                     int32_t num_kv_heads, int32_t head_dim, void* stream) {
  ts::clear_error();
  TS_REQUIRE(num_heads > 0 && num_kv_heads > 0, TS_ERR_INVALID_ARG,
             "rope_kv_write_int4: num_heads=%d num_kv_heads=%d", num_heads, num_kv_heads);
  if (num_tokens > 0) {
    TS_REQUIRE(qkv && q_out && positions && cos_table && sin_table && max_position > 0, TS_ERR_INVALID_ARG,
               "rope_kv_write_int4: null pointer or empty table");
    TS_REQUIRE(qkv_stride >= ((int64_t)num_heads + 2 * (int64_t)num_kv_heads) * head_dim && qkv_stride % 8 == 0 &&
                   aligned(qkv, 16) && aligned(q_out, 16) && aligned(cos_table, 16) && aligned(sin_table, 16),
               TS_ERR_INVALID_ARG, "rope_kv_write_int4: qkv rows and tables must be 16-byte aligned");
  }
  Int4WriteArgs a = {};
  const half_t* row = static_cast<const half_t*>(qkv);
  a.k = row ? row + (int64_t)num_heads * head_dim : nullptr;
  a.v = row ? row + ((int64_t)num_heads + num_kv_heads) * head_dim : nullptr;
  a.k_st = a.v_st = qkv_stride, a.k_sh = a.v_sh = head_dim;
  a.kc = static_cast<uint8_t*>(k_cache), a.vc = static_cast<uint8_t*>(v_cache);
  a.num_blocks = num_blocks, a.slots = slot_mapping, a.kvh = num_kv_heads;
  a.q = row, a.q_st = qkv_stride, a.q_out = static_cast<half_t*>(q_out);
  a.positions = positions, a.cos_t = cos_table, a.sin_t = sin_table, a.max_pos = max_position;
  a.heads = num_heads;
  return write_int4(a, true, num_tokens, head_dim, "rope_kv_write_int4", stream);
}

extern "C" int ts_kv_read_int4(const void* cache, int32_t num_layers, int64_t num_blocks, int32_t num_kv_heads,
                               int32_t head_dim, const int32_t* blocks, int32_t n, void* out, void* stream) {
  ts::clear_error();
  TS_REQUIRE(num_layers >= 0 && n >= 0, TS_ERR_INVALID_ARG, "kv_read_int4: num_layers=%d n=%d", num_layers, n);
  if (num_layers == 0 || n == 0) return TS_OK;
  TS_REQUIRE(cache && blocks && out, TS_ERR_INVALID_ARG, "kv_read_int4: null pointer argument");
  TS_REQUIRE(num_kv_heads > 0 && num_blocks > 0, TS_ERR_INVALID_ARG, "kv_read_int4: num_kv_heads=%d num_blocks=%lld",
             num_kv_heads, (long long)num_blocks);
  TS_REQUIRE(int4_head_dim(head_dim), TS_ERR_UNSUPPORTED, "kv_read_int4: head_dim %d (16, 32, 64, 128, 256)", head_dim);
  TS_REQUIRE(aligned(cache, 16) && aligned(out, 16), TS_ERR_INVALID_ARG,
             "kv_read_int4: cache and out must be 16-byte aligned");
  const double units = 2.0 * num_layers * n * num_kv_heads;
  TS_REQUIRE(units < (double)(1ll << 30), TS_ERR_UNSUPPORTED, "kv_read_int4: %d blocks of %d layers", n, num_layers);
  Int4ReadArgs a = {static_cast<const uint8_t*>(cache), blocks, static_cast<half_t*>(out), num_blocks, n,
                    num_kv_heads, (int)units, I8Div::by(n), I8Div::by(num_kv_heads)};
  const unsigned grid = (unsigned)(((int64_t)a.units * (head_dim / 2) + kI4WriteThreads - 1) / kI4WriteThreads);
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  switch (head_dim) {
    case 16: kv_read_int4_kernel<16><<<grid, kI4WriteThreads, 0, s>>>(a); break;
    case 32: kv_read_int4_kernel<32><<<grid, kI4WriteThreads, 0, s>>>(a); break;
    case 64: kv_read_int4_kernel<64><<<grid, kI4WriteThreads, 0, s>>>(a); break;
    case 128: kv_read_int4_kernel<128><<<grid, kI4WriteThreads, 0, s>>>(a); break;
    default: kv_read_int4_kernel<256><<<grid, kI4WriteThreads, 0, s>>>(a); break;
  }
  return check_launch("kv_read_int4");
}
