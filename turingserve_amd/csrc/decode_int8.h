// Attention of one or a few query rows per sequence over the 8-bit paged cache (decode rows, the
// rows of a speculative step).
//
//   s_j = scale * ks[blk(j)] * (q . code_k[j]),  out = sum_j softmax(s)_j * vs[blk(j)] * code_v[j]
//
// A block's V scale goes into the exponent: with t_j = s_j + log2 vs[blk(j)] (s in base 2),
//   P'_j = 2^(t_j - m) is rounded to fp16 and multiplied by the codes of V, l = sum_j P'_j / vs[blk(j)],
//   out = sum_j P'_j code_v[j] / l,
// m being the row's own running maximum of t over the tokens that it sees. So the largest P' of a row is
// at least 1 whatever its other blocks hold, and tokens that it does not see have no say in its rounding
// (P against the largest V scale of a split's blocks rounded a row's weights away where hidden blocks
// had a V scale 2^20 above those that it saw). A V scale below 2^-40 counts as 2^-40, which moves a
// result by 127 * 2^-40 at most: 2^-8 of fp16's smallest half step.
//
// The rows of a sequence for one KV head, row = token * group + head, stand in tiles of 16 (the rows
// of an MFMA tile); row i's token sees the first seq_len - n + token + 1 tokens. One workgroup of
// four wavefronts takes one split of the sequence's blocks for one tile: every code is read once for
// a whole group of heads. The four wavefronts take pairs of blocks in turn with a running maximum and
// sum each, meet once at the end in LDS, and either write the row or leave a partial (m, l, O) for the
// merge launch.
//
// 64 sequences of 128 to 4096 tokens, 12/2 heads of 128: 12.7 us and 4.1 for the merge, 38 MB of codes
// and scales (7.7 us at a copy's 5.0 TB/s); one sequence of 6000: 7.1 to 8.2 and 3.8. What bounds it is the chain
// of a workgroup (lengths, table, scales and codes, LDS, partial) and then that of the merge: taking out
// a tenth of the loop's arithmetic (O scaled in every step) gained 1 %. Two tiles a workgroup (32 rows of
// a chunk, 253 registers, two workgroups a CU) took 29.0 us instead of 24.7 at 16 sequences of 5 rows,
// 28/4 heads on 300 to 3000 cached, and 16.5 instead of 13.9 at one of 8 rows on 1024, and were ahead
// only past some 1500 tiles (16 chunks of 128 rows on 512: 29.2 and 35.8).
#pragma once

#include "int8_kv.h"

namespace ts {

constexpr int kI8Waves = 4;
constexpr int kI8Threads = kI8Waves * kWave;
// Blocks of a split, as long as kI8MaxSplits suffice. 8, 16 and 32 blocks: 18.2, 17.8 and 18.3 us at the
// 64 sequences above, 18.9, 18.8 and 20.6 at four of 8000 to 32768 tokens, 11.0, 11.1 and 12.5 at one.
constexpr int kI8SplitBlocks = 16;
// A lane of the merge each. 32 and 64: 15.6 and 14.2 us at one sequence of 32768, 41.4 and 27.5 at one of
// 131072, 20.4 and 23.0 at four of 32768.
constexpr int kI8MaxSplits = 64;
constexpr float kI8Rescale = 8.f;      // a row's reference moves when a score passes it by 2^8

// Splits of a sequence of nb blocks, at most `most` (the partials that the workspace holds for a
// row, from the host's bound on the lengths): from its own length, so that a row's result does not
// depend on the rest of the batch.
__host__ __device__ inline int i8_splits(int nb, int most, int each = kI8SplitBlocks) {
  const int n = (nb + each - 1) / each;
  return n < 1 ? 1 : (n > most ? most : n);
}

// The first block of split `split` of nb blocks (of split `splits`: nb): the first nb % splits of them
// are one block longer. No product leaves 32 bits: split * (nb / splits) <= nb.
__host__ __device__ inline int i8_split_begin(int nb, int split, int splits) {
  const int each = (int)((unsigned)nb / (unsigned)splits), more = nb - each * splits;
  return split * each + (split < more ? split : more);
}

// Division of 0 <= x < 2^31 by a number that the host knows: x * mul >> 32 >> shift, with mul =
// ceil(2^(31 + l) / d) and shift = l - 1 for 2^(l - 1) < d <= 2^l, which is exact there.
struct I8Div {
  unsigned mul;
  int shift;                             // -1: by 1
  __host__ __device__ static I8Div by(int d) {
    if (d <= 1) return {0, -1};
    int l = 1;
    while ((1ll << l) < d) ++l;
    return {(unsigned)(((1ull << (31 + l)) + d - 1) / d), l - 1};
  }
  __device__ __forceinline__ int operator()(int x) const {
    return shift < 0 ? x : (int)(__umulhi((unsigned)x, mul) >> shift);
  }
};

struct Int8DecodeArgs {
  const half_t* q;
  int64_t q_st, q_sh;
  half_t* out;
  int64_t out_st;
  const int8_t *kc, *vc;
  const float *ks, *vs;
  int64_t num_blocks;
  const int32_t* block_tables;
  int64_t bt_stride;
  int max_blocks;
  const int32_t *seq_lens, *qsl;
  int64_t num_tokens;
  int num_seqs, num_decode;                      // sequences; the first num_decode have one row each
  int heads, kvh, group;                         // group = heads / kvh
  I8Div by_kvh, by_group, by_slots, by_units;    // (by num_seqs kvh)
  float sl2;                                     // scale * log2(e)
  // Partials, D floats each and (m, l): max_splits for each row of the first num_decode sequences, then
  // chunk_parts for each (sequence, KV head) of the others, whose rows have as many as they have
  // splits (merged where they are row_slots rows at most).
  int row_slots, max_splits, chunk_parts;
  float *part_o, *part_ml;
};

// The rows of a sequence.
struct I8Seq {
  int q0, n, kv, start;                          // first flat row, rows, tokens, position of row q0
};
__device__ __forceinline__ int i8_kv_len(int len, int max_blocks);

__device__ __forceinline__ I8Seq i8_seq(const Int8DecodeArgs& a, int b) {
  I8Seq s;
  const int len = a.seq_lens[b];
  s.q0 = b, s.n = 1;
  if (b >= a.num_decode) {
    const int q0 = a.qsl[b], q1 = a.qsl[b + 1];
    s.q0 = q0;
    s.n = q0 < 0 || q1 <= q0 || q1 > a.num_tokens ? 0 : q1 - q0;
  }
  s.kv = i8_kv_len(len, a.max_blocks);
  s.start = max(len, 0) - s.n;
  return s;
}

// Splits of a sequence's blocks, of EACH blocks: longer ones where several tiles of rows share them, so that
// its partials stay those of one tile. (chunk_parts holds them, and row_slots the rows, within the host's
// bounds; past those there is one split.)
template <int EACH = kI8SplitBlocks>
__device__ __forceinline__ int i8_splits(const Int8DecodeArgs& a, const I8Seq& s, bool decode) {
  const int rows = s.n * a.group, nb = (s.kv + kBlockSize - 1) / kBlockSize;
  if (decode) return i8_splits(nb, a.max_splits, EACH);
  if (rows > a.row_slots) return 1;
  const int tiles = s.n == 1 ? 1 : (rows + 15) / 16;
  const int n = i8_splits(nb, min(a.max_splits, kI8MaxSplits / tiles), EACH * tiles);
  return n * rows > a.chunk_parts ? 1 : n;
}

// The first partial of a row.
__device__ __forceinline__ int64_t i8_partial(const Int8DecodeArgs& a, int b, int h, int row, int splits) {
  return b < a.num_decode
             ? ((int64_t)(b * a.kvh + h) * a.group + row) * a.max_splits
             : (int64_t)a.num_decode * a.heads * a.max_splits +
                   (int64_t)((b - a.num_decode) * a.kvh + h) * a.chunk_parts + row * splits;
}

// Tokens of a sequence that its table holds.
__device__ __forceinline__ int i8_kv_len(int len, int max_blocks) {
  const int64_t most = (int64_t)max_blocks * kBlockSize;
  return len < 0 ? 0 : (len > most ? (int)most : len);
}

// A block's V scale in the exponent, and what a weight with it is multiplied by in the row's sum: its
// exact inverse but for rounding, so that the sum does not feel the logarithm's. (Scales above 2^100,
// whose inverse need not be a normal number, count as 2^100: any code of theirs is infinite in fp16.)
constexpr float kI8LeastScale = 0x1p-40f, kI8MostScale = 0x1p100f;
__device__ __forceinline__ void i8_value_factors(float vs, float& lv, float& back) {
  lv = __builtin_amdgcn_logf(__builtin_amdgcn_fmed3f(vs, kI8LeastScale, kI8MostScale));
  back = fast_exp2(-lv);
}

// A block with a scale that is not finite makes the scores of its visible tokens NaN, and its V
// scale 0: tokens which a row does not see stay out of it (0 * NaN would not).
__device__ __forceinline__ void i8_poison(float& ks, float& vs) {
  if (!(fabsf(ks) < INFINITY && fabsf(vs) < INFINITY)) ks = __builtin_nanf(""), vs = 0.f;
}

template <int D>
struct I8Pair {
  // K: lane (c, g) holds codes of token c; V: tokens 4 g + r, dims VW c .. VW c + VW - 1.
  static constexpr int KW = D >= 64 ? D / 16 : (D == 32 ? 2 : 1);   // words of K per block and lane
  static constexpr int VW = D / 16;
  static constexpr int VWORDS = (VW + 3) / 4;
  uint32_t k[2][KW], v[2][4][VWORDS];
};

template <int D>
__device__ __forceinline__ void i8_load_k(const int8_t* base, int c, int g, uint32_t (&k)[I8Pair<D>::KW]) {
  if constexpr (D >= 64) {
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const uint4_t x = ld<uint4_t>(base + c * D + 64 * i + 16 * g);
#pragma unroll
      for (int w = 0; w < 4; ++w) k[4 * i + w] = x[w];
    }
  } else if constexpr (D == 32) {
    const int2_t x = ld<int2_t>(base + c * D + 8 * g);
    k[0] = x[0], k[1] = x[1];
  } else {
    k[0] = ld<uint32_t>(base + c * D + 4 * g);
  }
}

template <int D>
__device__ __forceinline__ void i8_load_v(const int8_t* base, int c, int g,
                                          uint32_t (&v)[4][I8Pair<D>::VWORDS]) {
  constexpr int VW = I8Pair<D>::VW;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int8_t* p = base + (4 * g + r) * D + VW * c;
    if constexpr (VW == 16) {
      const uint4_t x = ld<uint4_t>(p);
#pragma unroll
      for (int w = 0; w < 4; ++w) v[r][w] = x[w];
    } else if constexpr (VW == 8) {
      const int2_t x = ld<int2_t>(p);
      v[r][0] = x[0], v[r][1] = x[1];
    } else if constexpr (VW == 4) {
      v[r][0] = ld<uint32_t>(p);
    } else if constexpr (VW == 2) {
      v[r][0] = ld<uint16_t>(p);
    } else {
      v[r][0] = ld<uint8_t>(p);
    }
  }
}

// q as the B operand of S^T = K . Q^T, in the order of dims in which i8_load_k lays K out.
template <int D>
struct I8Query {
  static constexpr int N = D >= 32 ? D / 32 : 1;
  half8_t x[N];
};

template <int D>
__device__ __forceinline__ void i8_load_q(const half_t* row, int g, bool real, I8Query<D>& q) {
  const half8_t zero = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < I8Query<D>::N; ++i) q.x[i] = zero;
  if (!real) return;
  if constexpr (D >= 64) {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) q.x[i] = ld<half8_t>(row + 64 * (i / 2) + 16 * g + 8 * (i % 2));
  } else if constexpr (D == 32) {
    q.x[0] = ld<half8_t>(row + 8 * g);
  } else {
    const half4_t t = ld<half4_t>(row + 4 * g);
    q.x[0] = {t[0], t[1], t[2], t[3], 0, 0, 0, 0};
  }
}

template <int D>
__device__ __forceinline__ float4_t i8_scores(const uint32_t (&k)[I8Pair<D>::KW], const I8Query<D>& q) {
  float4_t s = {0.f, 0.f, 0.f, 0.f};
  if constexpr (D >= 32) {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) s = mfma16x16x32(codes8(k[2 * i], k[2 * i + 1]), q.x[i], s);
  } else {
    const uint32_t u = k[0] ^ 0x80808080u;
    const half2_t a = codes01(u), b = codes23(u);
    s = mfma16x16x16(half4_t{a[0], a[1], b[0], b[1]}, lo4(q.x[0]), s);
  }
  return s;
}

// V^T operand of output tile t (dims VW i + t): tokens 4 g .. 4 g + 3 of block a, then of block b.
template <int D, int t>
__device__ __forceinline__ half8_t i8_vt(const uint32_t (&v)[2][4][I8Pair<D>::VWORDS]) {
  constexpr int w = t / 4, q = t % 4;
  const half2_t a = column2<q>(v[0][0][w], v[0][1][w]), b = column2<q>(v[0][2][w], v[0][3][w]);
  const half2_t c = column2<q>(v[1][0][w], v[1][1][w]), d = column2<q>(v[1][2][w], v[1][3][w]);
  return {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

template <int D, int t = 0>
__device__ __forceinline__ void i8_pv(float4_t (&o)[D / 16], const uint32_t (&v)[2][4][I8Pair<D>::VWORDS],
                                      half8_t p) {
  if constexpr (t < D / 16) {
    o[t] = mfma16x16x32(i8_vt<D, t>(v), p, o[t]);
    i8_pv<D, t + 1>(o, v, p);
  }
}

// The state of one wavefront's 16 rows: reference, sum, and O^T in units of kColumnUnit.
template <int D>
struct I8State {
  float m, l;
  float4_t o[D / 16];
};

// A row's result in fp16. FINITE: V's values are fp16 numbers, and so is their mean in exact arithmetic; but
// weights are rounded for the product and not in their sum, which moves a mean of 65504s by up to 2^-11 of
// it, past the largest number. (NaN stays.)
template <bool FINITE>
__device__ __forceinline__ half4_t i8_result(float4_t o) {
  if constexpr (FINITE) {
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = __builtin_elementwise_minimum(vmax(o[e], -65504.f), 65504.f);
  }
  return to_half4(o);
}

// What a block multiplies its scores by (scale * log2 e * ks), adds to them, and multiplies its weights
// by in a row's sum (i8_value_factors).
struct I8Factors {
  float fk, lv, back;
};

// One pair of blocks (tokens ta .. and tb .. of the sequence). A row sees the tokens below `vis`, all
// rows of the tile those below `least`.
template <int D>
__device__ __forceinline__ void i8_step(I8State<D>& st, const I8Pair<D>& x, const I8Query<D>& q,
                                        const I8Factors& fa, const I8Factors& fb, int ta, int tb, int vis,
                                        int least, int g) {
  float4_t sa = i8_scores<D>(x.k[0], q), sb = i8_scores<D>(x.k[1], q);
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    sa[r] = fmaf(sa[r], fa.fk, fa.lv);
    sb[r] = fmaf(sb[r], fb.fk, fb.lv);
  }
  if (tb + kBlockSize > least || ta + kBlockSize > least) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      sa[r] = ta + 4 * g + r < vis ? sa[r] : -INFINITY;
      sb[r] = tb + 4 * g + r < vis ? sb[r] : -INFINITY;
    }
  }
  const float top = rows_max(vmax(vmax(vmax(sa[0], sa[1]), vmax(sa[2], sa[3])),
                                  vmax(vmax(sb[0], sb[1]), vmax(sb[2], sb[3]))));
  // !(<=): a NaN score (a block whose scale is NaN) moves the reference to NaN, where it stays
  const bool move = !(top <= st.m + kI8Rescale);
  if (__ballot(move)) {
    const float to = vmax(st.m, top);
    const float alpha = move ? fast_exp2(st.m - to) : 1.f; // m = -inf: 0
    st.l *= alpha;
    st.m = move ? to : st.m;
#pragma unroll
    for (int t = 0; t < D / 16; ++t) st.o[t] *= alpha;
  }
  const float neg = st.m == -INFINITY ? 0.f : -st.m;
  float pa[4], pb[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) pa[r] = fast_exp2(sa[r] + neg), pb[r] = fast_exp2(sb[r] + neg);
  st.l = fmaf((pa[0] + pa[1]) + (pa[2] + pa[3]), fa.back, st.l);
  st.l = fmaf((pb[0] + pb[1]) + (pb[2] + pb[3]), fb.back, st.l);
  half8_t p;
#pragma unroll
  for (int r = 0; r < 4; ++r) p[r] = (half_t)pa[r], p[4 + r] = (half_t)pb[r];
  // Codes left past the end are finite, and p is 0 there.
  i8_pv<D>(st.o, x.v, p);
}

// One split [b0, b1) of a sequence's blocks by one wavefront (of kI8Waves). Blocks are taken 64
// at a time: lane i holds block i's id and factors.
template <int D>
__device__ __forceinline__ void i8_split(const Int8DecodeArgs& a, I8State<D>& st, const I8Query<D>& q, int b,
                                         int h, int b0, int b1, int len, int vis, int least, int wave) {
  const int lane = threadIdx.x % kWave, c = lane % 16, g = lane / 16;
  const int32_t* table = a.block_tables + b * a.bt_stride;
  const int64_t block_bytes = (int64_t)kBlockSize * D;
  for (int lo = b0; lo < b1; lo += kWave) {
    const int n = min(b1 - lo, kWave);
    int blk = 0;
    float ks = 0.f, vs = 0.f;
    if (lane < n) {
      blk = clamp_block(table[lo + lane], a.num_blocks);
      ks = a.ks[(int64_t)blk * a.kvh + h];
      vs = a.vs[(int64_t)blk * a.kvh + h];
      i8_poison(ks, vs);
    }
    // the first two pairs are requested behind the scales and before they are waited for
    auto lane_int = [&](int v, int i) { return __builtin_amdgcn_readlane(v, i); };
    auto lane_f = [&](float v, int i) {
      return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), i));
    };
    auto load = [&](I8Pair<D>& x, int i) {                 // blocks i, i + 1 of the 64
      const int j = min(i + 1, n - 1);
      const int64_t ua = ((int64_t)lane_int(blk, i) * a.kvh + h) * block_bytes;
      const int64_t ub = ((int64_t)lane_int(blk, j) * a.kvh + h) * block_bytes;
      i8_load_k<D>(a.kc + ua, c, g, x.k[0]);
      i8_load_k<D>(a.kc + ub, c, g, x.k[1]);
      i8_load_v<D>(a.vc + ua, c, g, x.v[0]);
      i8_load_v<D>(a.vc + ub, c, g, x.v[1]);
    };
    float lv, back;
    auto step = [&](I8Pair<D>& x, int i) {
      const int j = min(i + 1, n - 1);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int w = 0; w < I8Pair<D>::VWORDS; ++w) x.v[u][r][w] ^= 0x80808080u;
      // with an odd count the last pair's second block is its first, wholly past the end
      const int ta = (lo + i) * kBlockSize;
      const int tb = i + 1 < n ? ta + kBlockSize : len;
      i8_step<D>(st, x, q, {lane_f(ks, i), lane_f(lv, i), lane_f(back, i)},
                 {lane_f(ks, j), lane_f(lv, j), lane_f(back, j)}, ta, tb, vis, least, g);
    };
    constexpr int STEP = 2 * kI8Waves;
    I8Pair<D> x, y;
    int i = 2 * wave;
    if (i < n) load(x, i);
    if (i + STEP < n) load(y, i + STEP);
    i8_value_factors(vs, lv, back);
    ks *= a.sl2;

    if (i >= n) continue;
    while (true) {
      step(x, i);
      if (i + 2 * STEP < n) load(x, i + 2 * STEP);
      i += STEP;
      if (i >= n) break;
      step(y, i);
      if (i + 2 * STEP < n) load(y, i + 2 * STEP);
      i += STEP;
      if (i >= n) break;
    }
  }
}

template <int D>
struct I8DecodeLds {
  static constexpr int ROW = D + 4;      // floats of a row: rows start on different banks
  float o[kI8Waves * 16 * ROW];
  float ml[2 * kI8Waves * 16];
};

// The four wavefronts' states meet in LDS; the row (or its partial) is written.
template <int D>
__device__ __forceinline__ void i8_finish(const Int8DecodeArgs& a, I8State<D>& st, int b, int h,
                                          int q0, int row0, int rows, int split, int splits, int wave,
                                          float* s_o, float* s_ml) {
  constexpr int VW = D / 16;
  const int lane = threadIdx.x % kWave, c = lane % 16, g = lane / 16;
  const float l = rows_sum(st.l);
  __syncthreads();                                         // the last item's reads of LDS
  if (c < rows) {
    float* dst = s_o + (wave * 16 + c) * I8DecodeLds<D>::ROW;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int t = 0; t < VW; ++t) dst[VW * (4 * g + r) + t] = st.o[t][r];
    if (g == 0) {
      s_ml[2 * (wave * 16 + c)] = st.m;
      s_ml[2 * (wave * 16 + c) + 1] = l;
    }
  }
  __syncthreads();
  for (int u = threadIdx.x; u < rows * (D / 4); u += kI8Threads) {
    const int row = u / (D / 4), d = u % (D / 4) * 4;
    float m[kI8Waves], top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kI8Waves; ++w) m[w] = s_ml[2 * (w * 16 + row)], top = vmax(top, m[w]);
    float sum = 0.f;
    float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kI8Waves; ++w) {
      const float f = m[w] == -INFINITY ? 0.f : fast_exp2(m[w] - top);
      sum += f * s_ml[2 * (w * 16 + row) + 1];
      o += ld<float4_t>(s_o + (w * 16 + row) * I8DecodeLds<D>::ROW + d) * f;
    }
    o *= kColumnUnit;
    if (splits == 1) {
      const float f = sum == 0.f ? 0.f : 1.f / sum;        // no visible key: zeros
      const int token = a.by_group(row0 + row), head = h * a.group + row0 + row - token * a.group;
      ts::st<half4_t>(a.out + (int64_t)(q0 + token) * a.out_st + (int64_t)head * D + d, to_half4(o * f));
    } else {
      const int64_t at = i8_partial(a, b, h, row0 + row, splits) + split;
      ts::st<float4_t>(a.part_o + at * D + d, o);
      if (d == 0) {
        a.part_ml[2 * at] = top;
        a.part_ml[2 * at + 1] = sum;
      }
    }
  }
}

// Item `item` of the batch's (split, row tile) pairs, numbered densely over the sequences. Every
// wavefront looks it up for itself, 64 sequences at a time.
struct I8Item {
  int b, split, splits, tile;
  I8Seq seq;
};

template <int EACH = kI8SplitBlocks>
__device__ __forceinline__ bool i8_find(const Int8DecodeArgs& a, int item, I8Item& x) {
  const int lane = threadIdx.x % kWave;
  int base = 0;
  for (int s0 = 0; s0 < a.num_seqs; s0 += kWave) {
    int splits = 1, tiles = 0;
    I8Seq s = {};
    if (s0 + lane < a.num_seqs) {
      s = i8_seq(a, s0 + lane);
      splits = i8_splits<EACH>(a, s, s0 + lane < a.num_decode);
      tiles = (s.n * a.group + 15) / 16;
    }
    const int n = splits * tiles, sum = i8_scan(n);
    const uint64_t past = __ballot(base + sum > item);
    if (past) {
      const int i = __ffsll((unsigned long long)past) - 1;
      auto of = [&](int v) { return __builtin_amdgcn_readlane(v, i); };
      x.b = s0 + i;
      x.splits = of(splits);
      const unsigned in = item - (base + of(sum) - of(n)), t = of(tiles);
      x.split = (int)(t == 1 ? in : in / t), x.tile = (int)(in - x.split * t);
      x.seq = {of(s.q0), of(s.n), of(s.kv), of(s.start)};
      return x.split < x.splits;                           // (only offsets that do not ascend could have it)
    }
    base += __builtin_amdgcn_readlane(sum, kWave - 1);
  }
  return false;
}

// Workgroups that a CU holds at once, by registers.
constexpr int i8_decode_groups(int D) { return D > 128 ? 1 : (D == 128 ? 3 : 4); }

template <int D>
__global__ void __launch_bounds__(kI8Threads, i8_decode_groups(D)) decode_int8_kernel(Int8DecodeArgs a) {
  __shared__ __align__(16) I8DecodeLds<D> lds;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave, c = lane % 16, g = lane / 16;
  for (int64_t u = blockIdx.x;; u += gridDim.x) {
    if (u > INT32_MAX) return;                             // (the entry point refuses more)
    const int item = a.by_kvh((int)u), h = (int)u - item * a.kvh;
    I8Item x;
    if (!i8_find(a, item, x)) return;
    const int row0 = 16 * x.tile, rows = min(x.seq.n * a.group - row0, 16), kv = x.seq.kv;
    const int row = row0 + min(c, rows - 1), token = a.by_group(row);
    const int vis = min(kv, max(0, x.seq.start + token + 1));
    const int least = min(kv, max(0, x.seq.start + a.by_group(row0) + 1));
    I8Query<D> q;
    i8_load_q<D>(a.q + (int64_t)(x.seq.q0 + token) * a.q_st +
                     (int64_t)(h * a.group + row - token * a.group) * a.q_sh,
                 g, c < rows, q);
    I8State<D> st;
    st.m = -INFINITY, st.l = 0.f;
#pragma unroll
    for (int t = 0; t < D / 16; ++t) st.o[t] = {0.f, 0.f, 0.f, 0.f};
    const int nb = (kv + kBlockSize - 1) / kBlockSize;
    const int b0 = i8_split_begin(nb, x.split, x.splits), b1 = i8_split_begin(nb, x.split + 1, x.splits);
    i8_split<D>(a, st, q, x.b, h, b0, b1, kv, vis, least, wave);
    i8_finish<D>(a, st, x.b, h, x.seq.q0, row0, rows, x.split, x.splits, wave, lds.o, lds.ml);
  }
}

// Rows of sequences with more than one split: one wavefront a row, D / 4 lanes a partial. A decode
// row's first partials and every split's (m, l) are requested before the sequence's length is known
// (they lie in the workspace whatever it is), the others at once after it. (A workgroup a row, its
// eight groups meeting in LDS, took twice as long at 2240 rows of a few splits: 10.5 us. One partial ahead
// of the length and reductions by shuffles: 40.0 us a pass of four layers of one sequence of 6000 in 4 bits,
// 38.4 so; sixteen ahead no less.)
template <int D, int EACH = kI8SplitBlocks, bool FINITE = false>
__device__ __forceinline__ void i8_merge_row(const Int8DecodeArgs& a, int slot) {
  constexpr int PER_ROW = D / 4, GROUPS = kWave / PER_ROW;
  constexpr int N = 64 / GROUPS < 16 ? 64 / GROUPS : 16;   // partials of a lane at a time
  constexpr int FIRST = N < 8 ? N : 8;                     // of them requested before the length is known
  const int lane = threadIdx.x % kWave;
  const int behind = slot - a.num_decode * a.heads;        // of the sequences past num_decode
  const int unit = behind < 0 ? a.by_group(slot) : a.by_slots(behind);
  const int r = behind < 0 ? slot - unit * a.group : behind - unit * a.row_slots;
  const int seq0 = a.by_kvh(unit), h = unit - seq0 * a.kvh, b = behind < 0 ? seq0 : a.num_decode + seq0;
  if (b >= a.num_seqs) return;
  const int group = lane / PER_ROW, d = lane % PER_ROW * 4;
  float2_t ml;
  float4_t x[N];
  auto request = [&](int64_t row, int n) {                 // its first partials, all its (m, l)
    ml = ld<float2_t>(a.part_ml + 2 * (row + min(lane, n - 1)));
#pragma unroll
    for (int i = 0; i < FIRST; ++i) x[i] = ld<float4_t>(a.part_o + (row + min(group + i * GROUPS, n - 1)) * D + d);
  };
  if (behind < 0) request((int64_t)slot * a.max_splits, a.max_splits);
  const I8Seq seq = i8_seq(a, b);
  const int splits = i8_splits<EACH>(a, seq, behind < 0);
  if (splits == 1 || r >= seq.n * a.group) return;
  const int64_t row = i8_partial(a, b, h, r, splits);
  const float* part = a.part_o + row * D + d;
  if (behind >= 0) request(row, splits);
  // lane i: split i's weight
  const float m = lane < splits ? ml[0] : -INFINITY;
  float4_t o = {0.f, 0.f, 0.f, 0.f};
  float f = 0.f, sum = 0.f;
  for (int i0 = 0; i0 < splits; i0 += N * GROUPS) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int k = i0 + group + i * GROUPS;
      if ((i >= FIRST || i0 > 0) && k < splits) x[i] = ld<float4_t>(part + (int64_t)k * D);
    }
    if (i0 == 0) {
      const float top = i8_wave_max(m);                    // (by all lanes: not within the choice below)
      f = m == -INFINITY ? 0.f : fast_exp2(m - top);
      sum = i8_wave_sum(lane < splits ? f * ml[1] : 0.f);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int k = i0 + group + i * GROUPS;
      const float w = __shfl(f, min(k, kWave - 1), kWave);
      if (k < splits) o += x[i] * w;
    }
  }
#pragma unroll
  for (int k = PER_ROW; k < kWave; k <<= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += shfl_xor(o[e], k);
  if (group > 0) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;          // (nothing visible)
  const int token = a.by_group(r), head = h * a.group + r - token * a.group;
  st<half4_t>(a.out + (int64_t)(seq.q0 + token) * a.out_st + (int64_t)head * D + d, i8_result<FINITE>(o * inv));
}

// The wavefront's row, of workgroup `group`.
__device__ __forceinline__ int i8_merge_slot(int group) {
  return group * kI8Waves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
}

template <int D, int EACH = kI8SplitBlocks, bool FINITE = false>
__global__ void __launch_bounds__(kI8Threads) decode_int8_merge_kernel(Int8DecodeArgs a) {
  i8_merge_row<D, EACH, FINITE>(a, i8_merge_slot(blockIdx.x));
}

}  // namespace ts
