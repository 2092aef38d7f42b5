// The quantising write of a step's new K/V rows into the 4-bit paged cache, with or without RoPE, and the
// reading of its blocks as fp16. For each row, KV head and group of 32 channels
//   low  = fp16(least value),  step = (largest value - low) / 15 in fp32, rounded towards zero to fp16,
//   code = rint((value - low) / step) within 0 .. 15 (0 where step is 0),
// fp32 throughout, divisions rounded correctly. The step is rounded towards zero so that no code stands for
// more than the largest value (the nearest one could leave the fp16 range at 65504); that costs at most
// 15 units in the step's last place, 0.015 of a step, where a code is off by half of one.
//
// A thread holds the octets o and o + D / 16 of a row of K and of V, D / 16 threads a row: the rotation's
// pairs in one thread, the groups' extremes over 4 neighbouring lanes at most.
#include "int4_kv.h"
#include "decode_int8.h"
#include "rope.h"

namespace ts {

constexpr int kI4Threads = 256;

struct Int4WriteArgs {
  const half_t *k, *v;                    // rows of the step (k, v heads)
  int64_t k_st, k_sh, v_st, v_sh;
  uint8_t *kc, *vc;
  int64_t num_blocks;
  const int64_t* slots;
  int num_tokens, kvh, units;             // units a token: q heads in the RoPE form, then KV heads
  I8Div by_units;
  // RoPE form
  const half_t* q;
  int64_t q_st;
  half_t* q_out;
  const int64_t* positions;
  const float *cos_t, *sin_t;
  int64_t max_pos;
  int heads;
};

// Smallest and largest of a group: over the lane's octets that belong to it, then over its lanes.
struct I4Span {
  float lo, hi;
  __device__ __forceinline__ void add(float x) { lo = fminf(lo, x), hi = fmaxf(hi, x); }
  template <int MASK>
  __device__ __forceinline__ void meet() {
    lo = fminf(lo, shfl_xor(lo, MASK)), hi = fmaxf(hi, shfl_xor(hi, MASK));
  }
};

struct I4Numbers {
  half_t step, low;
};
__device__ __forceinline__ I4Numbers i4_numbers(const I4Span& s) {
  I4Numbers n;
  n.low = (half_t)(s.lo + 0.f);                            // (-0 as 0)
  const float span = fmaxf(s.hi - (float)n.low, 0.f) / 15.f;
  half_t step = (half_t)span;
  if ((float)step > span) step = __builtin_bit_cast(half_t, (uint16_t)(__builtin_bit_cast(uint16_t, step) - 1));
  n.step = step;
  return n;
}
__device__ __forceinline__ uint32_t i4_word(const float (&x)[8], I4Numbers n) {
  const float low = (float)n.low, step = (float)n.step;
  uint32_t w = 0;
  if (step > 0.f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float c = fminf(fmaxf(rintf((x[e] - low) / step), 0.f), 15.f);
      w |= (uint32_t)(int)c << 4 * (e / 2 + 4 * (e % 2));
    }
  }
  return w;
}

__device__ __forceinline__ void i4_load8(const half_t* p, float (&x)[8]) {
  const half8_t h = ld<half8_t>(p);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (float)h[e];
}

// The two octets of a row of K (or V), `at` lanes from the row's first one, as codes and numbers.
template <int D, bool VALUES>
__device__ __forceinline__ void i4_store_row(uint8_t* unit, int row, int at, const float (&x)[8],
                                             const float (&y)[8], bool bad) {
  typedef I4Unit<D> U;
  constexpr int HALF = D / 16;                             // octets of half a row, lanes of a row
  I4Span s = {INFINITY, -INFINITY}, t = {INFINITY, -INFINITY};
#pragma unroll
  for (int e = 0; e < 8; ++e) s.add(x[e]), (D >= 64 ? t : s).add(y[e]);
  constexpr int LANES = HALF < 4 ? HALF : 4;               // of a group
  if constexpr (LANES > 1) s.template meet<1>(), t.template meet<1>();
  if constexpr (LANES > 2) s.template meet<2>(), t.template meet<2>();
  I4Numbers n = i4_numbers(s), m = D >= 64 ? i4_numbers(t) : n;
  uint32_t a = i4_word(x, n), b = i4_word(y, m);
  if (bad) {
    a = b = 0;
    n = m = {(half_t)0.f, (half_t)__builtin_nanf("")};
  }
  *reinterpret_cast<uint32_t*>(unit + (VALUES ? U::v_word(row, at) : U::k_word(row, at))) = a;
  *reinterpret_cast<uint32_t*>(unit + (VALUES ? U::v_word(row, at + HALF) : U::k_word(row, at + HALF))) = b;
  if (at % LANES) return;
#pragma unroll
  for (int i = 0; i < (D >= 64 ? 2 : 1); ++i) {
    const int group = at / LANES + i * (U::GROUPS / 2);
    const I4Numbers z = i == 0 ? n : m;
    if constexpr (VALUES) {
      *reinterpret_cast<half_t*>(unit + U::v_numbers(row, group)) = z.step;
      *reinterpret_cast<half_t*>(unit + U::v_numbers(row, group) + 8) = z.low;
    } else {
      st<half2_t>(unit + U::k_numbers(row, group), half2_t{z.step, z.low});
    }
  }
}

__device__ __forceinline__ bool i4_not_fp16(const float (&x)[8]) {
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) bad = bad || !(fabsf(x[e]) <= 65504.f);
  return bad;
}

template <int D, bool ROPE>
__global__ void __launch_bounds__(kI4Threads) kv_write_int4_kernel(Int4WriteArgs a) {
  constexpr int HALF = D / 16;
  const int64_t id = (int64_t)blockIdx.x * kI4Threads + threadIdx.x;
  const int item = (int)(id / HALF), at = (int)(id % HALF);
  const int t = a.by_units(item), u = item - t * a.units;
  if (t >= a.num_tokens) return;                           // (whole rows: HALF divides the workgroup)
  float c[8], n[8];
  if constexpr (ROPE) {
    const int64_t pos = rope_row(a.positions[t], a.max_pos) * (D / 2) + 8 * at;
    const float4_t c0 = ld<float4_t>(a.cos_t + pos), c1 = ld<float4_t>(a.cos_t + pos + 4);
    const float4_t n0 = ld<float4_t>(a.sin_t + pos), n1 = ld<float4_t>(a.sin_t + pos + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) c[e] = c0[e], c[4 + e] = c1[e], n[e] = n0[e], n[4 + e] = n1[e];
  }
  if (ROPE && u < a.heads) {
    const half_t* src = a.q + t * a.q_st + (int64_t)u * D + 8 * at;
    half_t* dst = a.q_out + ((int64_t)t * a.heads + u) * D + 8 * at;
    float x[8], y[8];
    i4_load8(src, x), i4_load8(src + D / 2, y);
    half8_t p, r;
#pragma unroll
    for (int e = 0; e < 8; ++e) {                          // in fp32, rounded once
      p[e] = (half_t)fmaf(-y[e], n[e], x[e] * c[e]);
      r[e] = (half_t)fmaf(x[e], n[e], y[e] * c[e]);
    }
    st(dst, p);
    st(dst + D / 2, r);
    return;
  }
  const int h = ROPE ? u - a.heads : u;
  const int64_t slot = a.slots[t];
  const half_t* k = a.k + t * a.k_st + h * a.k_sh + 8 * at;
  const half_t* v = a.v + t * a.v_st + h * a.v_sh + 8 * at;
  float x[8], y[8], z[8], w[8];
  i4_load8(k, x), i4_load8(k + D / 2, y);
  i4_load8(v, z), i4_load8(v + D / 2, w);
  if (ROPE) {
    // in 64 bits, where the products are exact, rounded once to 32: a quotient's last bits decide a code
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const double f = x[e], g = y[e], cc = c[e], nn = n[e];
      x[e] = (float)fma(-g, nn, f * cc);
      y[e] = (float)fma(f, nn, g * cc);
    }
  }
  int bad = i4_not_fp16(x) || i4_not_fp16(y) || i4_not_fp16(z) || i4_not_fp16(w);
#pragma unroll
  for (int m = 1; m < HALF; m <<= 1) bad |= __shfl_xor(bad, m, kWave);
  const bool inside = slot >= 0 && slot < a.num_blocks * kBlockSize;
  if (!inside) return;                                     // (all lanes of a row)
  const int64_t unit = ((slot / kBlockSize) * a.kvh + h) * I4Unit<D>::BYTES;
  const int row = (int)(slot % kBlockSize);
  i4_store_row<D, false>(a.kc + unit, row, at, x, y, bad);
  i4_store_row<D, true>(a.vc + unit, row, at, z, w, bad);
}

struct Int4ReadArgs {
  const uint8_t* cache;
  const int32_t* blocks;
  half_t* out;
  int64_t num_blocks, layer_blocks;       // (layer, K or V) pairs times blocks asked for
  int n, kvh;
};

// One thread an octet: 16 bytes of fp16 from one word and its numbers.
template <int D>
__global__ void __launch_bounds__(kI4Threads) kv_read_int4_kernel(Int4ReadArgs a) {
  typedef I4Unit<D> U;
  constexpr int PER = kBlockSize * D / 8;                  // octets of a unit
  const int64_t id = (int64_t)blockIdx.x * kI4Threads + threadIdx.x;
  const int64_t unit = id / PER;                           // of the output: ((layer, side), block, head)
  const int in = (int)(id % PER), row = in / (D / 8), octet = in % (D / 8);
  const int64_t lb = unit / a.kvh;
  const int h = (int)(unit - lb * a.kvh);
  if (lb >= a.layer_blocks) return;
  const int64_t side = lb / a.n;
  const int blk = clamp_block(a.blocks[lb - side * a.n], a.num_blocks);
  const uint8_t* src = a.cache + ((side * a.num_blocks + blk) * a.kvh + h) * U::BYTES;
  const int group = octet * 8 / U::GROUP;
  uint32_t w, n;
  if (side % 2 == 0) {
    w = ld<uint32_t>(src + U::k_word(row, octet));
    n = ld<uint32_t>(src + U::k_numbers(row, group));
  } else {
    w = ld<uint32_t>(src + U::v_word(row, octet));
    n = ld<uint16_t>(src + U::v_numbers(row, group)) | (uint32_t)ld<uint16_t>(src + U::v_numbers(row, group) + 8) << 16;
  }
  st<half8_t>(a.out + id * 8, i4_octet(w, n));
}

static bool int4_head_dim(int D) { return D == 16 || D == 32 || D == 64 || D == 128 || D == 256; }

template <int D>
static void launch_write(const Int4WriteArgs& a, bool rope, unsigned grid, hipStream_t s) {
  if (rope)
    kv_write_int4_kernel<D, true><<<grid, kI4Threads, 0, s>>>(a);
  else
    kv_write_int4_kernel<D, false><<<grid, kI4Threads, 0, s>>>(a);
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
  a.num_tokens = (int)num_tokens, a.units = (int)units, a.by_units = I8Div::by((int)units);
  const int64_t grid = (num_tokens * units * (D / 16) + kI4Threads - 1) / kI4Threads;
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
  Int4ReadArgs a = {static_cast<const uint8_t*>(cache), blocks, static_cast<half_t*>(out), num_blocks,
                    2 * (int64_t)num_layers * n, n, num_kv_heads};
  const double octets = 4.0 * num_layers * n * num_kv_heads * head_dim;
  TS_REQUIRE(octets < (double)(1ll << 31) * kI4Threads, TS_ERR_UNSUPPORTED, "kv_read_int4: %d blocks of %d layers", n,
             num_layers);
  const unsigned grid = (unsigned)(((int64_t)octets + kI4Threads - 1) / kI4Threads);
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  switch (head_dim) {
    case 16: kv_read_int4_kernel<16><<<grid, kI4Threads, 0, s>>>(a); break;
    case 32: kv_read_int4_kernel<32><<<grid, kI4Threads, 0, s>>>(a); break;
    case 64: kv_read_int4_kernel<64><<<grid, kI4Threads, 0, s>>>(a); break;
    case 128: kv_read_int4_kernel<128><<<grid, kI4Threads, 0, s>>>(a); break;
    default: kv_read_int4_kernel<256><<<grid, kI4Threads, 0, s>>>(a); break;
  }
  return check_launch("kv_read_int4");
}
