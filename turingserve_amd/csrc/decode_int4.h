// Attention of one or a few query rows per sequence over the 4-bit paged cache (decode rows, the
// rows of a speculative step).
//
//   s_j = scale * (q . k_j),  out = sum_j softmax(s)_j v_j,  k and v the fp16 numbers that the codes stand for
//
// Tiles of 16 rows, splits, partials and the merge are those of the 8-bit cache (decode_int8.h). A
// wavefront takes pairs of blocks: K's codes become the A operand of S^T = K . Q^T in registers, a lane
// holding its token's share of the row with that share's numbers; V's that of O^T += V^T . P^T, two
// tokens to a register, so that steps and lows are packed operands as they are loaded. P = 2^(s - m) is
// rounded to fp16, m being the row's running reference, which a new score moves only when it passes it
// by 2^8; sums and accumulators are fp32.
#pragma once

#include "decode_int8.h"
#include "int4_kv.h"

namespace ts {

// One block's words of a lane (c, g): K of token c, channels (D / 4) g .. of D >= 64 (8 g .. of 32, 4 g ..
// of 16); V of tokens 4 g + r, channels VW c .. VW c + VW - 1.
template <int D>
struct I4Block {
  static constexpr int KW = D >= 64 ? D / 32 : 1, KN = D == 256 ? 2 : 1;
  static constexpr int VW = D / 16, VO = D == 256 ? 2 : 1;
  uint32_t k[KW], kn[KN], v[VO][4], vn[4];                 // vn: steps of two tokens each, then lows
};

template <int D>
__device__ __forceinline__ void i4_load_k(const uint8_t* unit, int c, int g, I4Block<D>& x) {
  typedef I4Unit<D> U;
  if constexpr (D >= 128) {
#pragma unroll
    for (int i = 0; i < D / 128; ++i) {
      const uint4_t w = ld<uint4_t>(unit + U::k_word(c, 0) + (D / 8) * g + 16 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) x.k[4 * i + e] = w[e];
    }
  } else if constexpr (D == 64) {
    const int2_t w = ld<int2_t>(unit + U::k_word(c, 2 * g));
    x.k[0] = w[0], x.k[1] = w[1];
  } else {
    x.k[0] = ld<uint32_t>(unit + U::k_word(c, D == 32 ? g : g / 2));
  }
  if constexpr (D == 256) {
    const int2_t n = ld<int2_t>(unit + U::k_numbers(c, 2 * g));
    x.kn[0] = n[0], x.kn[1] = n[1];
  } else {
    x.kn[0] = ld<uint32_t>(unit + U::k_numbers(c, D == 128 ? g : (D == 64 ? g / 2 : 0)));
  }
}

template <int D>
__device__ __forceinline__ void i4_load_v(const uint8_t* unit, int c, int g, I4Block<D>& x) {
  typedef I4Unit<D> U;
  typedef I4Block<D> B;
  const int octet = D == 256 ? 2 * c : B::VW * c / 8;
#pragma unroll
  for (int i = 0; i < B::VO; ++i) {
    const uint4_t w = ld<uint4_t>(unit + U::v_word(4 * g, octet + i));
#pragma unroll
    for (int r = 0; r < 4; ++r) x.v[i][r] = w[r];
  }
  const uint4_t n = ld<uint4_t>(unit + U::v_numbers(4 * g, B::VW * c / U::GROUP));
#pragma unroll
  for (int r = 0; r < 4; ++r) x.vn[r] = n[r];
}

// q as the B operand of S^T = K . Q^T, in the order of channels in which i4_load_k lays K out.
template <int D>
__device__ __forceinline__ void i4_load_q(const half_t* row, int g, bool real, I8Query<D>& q) {
  const half8_t zero = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < I8Query<D>::N; ++i) q.x[i] = zero;
  if (!real) return;
  if constexpr (D >= 64) {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) q.x[i] = ld<half8_t>(row + (D / 4) * g + 8 * i);
  } else if constexpr (D == 32) {
    q.x[0] = ld<half8_t>(row + 8 * g);
  } else {
    const half4_t t = ld<half4_t>(row + 4 * g);
    q.x[0] = {t[0], t[1], t[2], t[3], 0, 0, 0, 0};
  }
}

template <int D>
__device__ __forceinline__ float4_t i4_scores(const I4Block<D>& x, const I8Query<D>& q, int g) {
  float4_t s = {0.f, 0.f, 0.f, 0.f};
  if constexpr (D >= 32) {
#pragma unroll
    for (int i = 0; i < I4Block<D>::KW; ++i) s = mfma16x16x32(i4_octet(x.k[i], x.kn[i / 4]), q.x[i], s);
  } else {
    const half8_t k = i4_octet(x.k[0] >> (8 * (g & 1)), x.kn[0]);    // (half an octet)
    s = mfma16x16x16(lo4(k), lo4(q.x[0]), s);
  }
  return s;
}

// V's words of a block ready for the columns: two tokens to a word, even and odd channels apart.
template <int D>
struct I4Columns {
  static constexpr int VO = I4Block<D>::VO;
  uint32_t w[VO][2][2], w8[VO][2][2];                      // [octet][tokens 0 1, 2 3][even, odd]
  half2_t step[2], low[2];
  __device__ __forceinline__ I4Columns(const I4Block<D>& x, int c) {
#pragma unroll
    for (int i = 0; i < VO; ++i) {
      uint32_t v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        v[r] = x.v[i][r];
        // the lane's channels first: 4 (c % 2) .., 2 (c % 4) .., c % 8 of the octet
        if constexpr (D == 64) v[r] >>= 8 * (c & 1);
        if constexpr (D == 32) v[r] >>= 4 * (c & 3);
        if constexpr (D == 16) v[r] >>= 4 * (c / 2 & 3) + 16 * (c & 1);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        w[i][j][0] = i4_even(v[2 * j], v[2 * j + 1]);
        w[i][j][1] = i4_odd(v[2 * j], v[2 * j + 1]);
#pragma unroll
        for (int o = 0; o < 2; ++o) w8[i][j][o] = w[i][j][o] >> 8;
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) step[j] = i4_half2(x.vn[j]), low[j] = i4_finite(x.vn[2 + j]);
  }
  // Tokens 2 j, 2 j + 1 of the lane's channel t.
  template <int t>
  __device__ __forceinline__ half2_t at(int j) const {
    return i4_values<t % 8 / 2>(w[t / 8][j][t % 2], w8[t / 8][j][t % 2], step[j], low[j]);
  }
};

// O^T += V^T . P^T over the pair, output tile t taking channels VW i + t.
template <int D, int t = 0>
__device__ __forceinline__ void i4_pv(float4_t (&o)[D / 16], const I4Columns<D>& va, const I4Columns<D>& vb,
                                      half8_t p) {
  if constexpr (t < D / 16) {
    const half2_t a = va.template at<t>(0), b = va.template at<t>(1);
    const half2_t c = vb.template at<t>(0), d = vb.template at<t>(1);
    o[t] = mfma16x16x32(half8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]}, p, o[t]);
    i4_pv<D, t + 1>(o, va, vb, p);
  }
}

// One pair of blocks (tokens ta .. and tb .. of the sequence). A row sees the tokens below `vis`, all
// rows of the tile those below `least`. sl2: scale * log2(e) > 0.
template <int D>
__device__ __forceinline__ void i4_step(I8State<D>& st, const I4Block<D> (&x)[2], const I8Query<D>& q, float sl2,
                                        int ta, int tb, int vis, int least, int c, int g) {
  float4_t sa = i4_scores<D>(x[0], q, g), sb = i4_scores<D>(x[1], q, g);
  if (tb + kBlockSize > least || ta + kBlockSize > least) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      sa[r] = ta + 4 * g + r < vis ? sa[r] : -INFINITY;
      sb[r] = tb + 4 * g + r < vis ? sb[r] : -INFINITY;
    }
  }
  const float top = rows_max(vmax(vmax(vmax(sa[0], sa[1]), vmax(sa[2], sa[3])),
                                  vmax(vmax(sb[0], sb[1]), vmax(sb[2], sb[3])))) * sl2;
  // !(<=): a NaN score (a token of NaN) moves the reference to NaN, where it stays
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
  for (int r = 0; r < 4; ++r) pa[r] = fast_exp2(fmaf(sa[r], sl2, neg)), pb[r] = fast_exp2(fmaf(sb[r], sl2, neg));
  st.l += ((pa[0] + pa[1]) + (pa[2] + pa[3])) + ((pb[0] + pb[1]) + (pb[2] + pb[3]));
  half8_t p;
#pragma unroll
  for (int r = 0; r < 4; ++r) p[r] = (half_t)pa[r], p[4 + r] = (half_t)pb[r];
  // What stands past the end is finite (i4_finite), and p is 0 there.
  const I4Columns<D> va(x[0], c), vb(x[1], c);
  i4_pv<D>(st.o, va, vb, p);
}

// One split [b0, b1) of a sequence's blocks by one wavefront (of kI8Waves). Blocks are taken 64 at a
// time: lane i holds block i's id; with `known` the first kI8SplitBlocks come from there.
template <int D, bool KNOWN>
__device__ __forceinline__ void i4_split(const Int8DecodeArgs& a, I8State<D>& st, const I8Query<D>& q, int b,
                                         int h, int b0, int b1, int len, int vis, int least, int wave,
                                         const int* known) {
  const int lane = threadIdx.x % kWave, c = lane % 16, g = lane / 16;
  const int32_t* table = a.block_tables + b * a.bt_stride;
  const uint8_t *kc = reinterpret_cast<const uint8_t*>(a.kc), *vc = reinterpret_cast<const uint8_t*>(a.vc);
  for (int lo = b0, n; lo < b1; lo += n) {
    const bool first = KNOWN && lo == b0;
    n = min(b1 - lo, first ? kI8SplitBlocks : kWave);
    int blk = 0;
    if (lane < n) blk = clamp_block(first ? known[lane] : table[lo + lane], a.num_blocks);
    auto load = [&](I4Block<D> (&x)[2], int i) {           // blocks i, i + 1 of the 64
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int id = __builtin_amdgcn_readlane(blk, min(i + u, n - 1));
        const int64_t unit = ((int64_t)id * a.kvh + h) * I4Unit<D>::BYTES;
        i4_load_k<D>(kc + unit, c, g, x[u]);
        i4_load_v<D>(vc + unit, c, g, x[u]);
      }
    };
    auto step = [&](I4Block<D> (&x)[2], int i) {
      // with an odd count the last pair's second block is its first, wholly past the end
      const int ta = (lo + i) * kBlockSize;
      const int tb = i + 1 < n ? ta + kBlockSize : len;
      i4_step<D>(st, x, q, a.sl2, ta, tb, vis, least, c, g);
    };
    constexpr int STEP = 2 * kI8Waves;
    I4Block<D> x[2], y[2];
    int i = 2 * wave;
    if (i < n) load(x, i);
    if (i + STEP < n) load(y, i + STEP);
#pragma unroll 1
    for (; i < n; i += STEP) {
      step(x, i);
      x[0] = y[0], x[1] = y[1];
      if (i + 2 * STEP < n) load(y, i + 2 * STEP);
    }
  }
}

template <int D>
__global__ void __launch_bounds__(kI8Threads, i8_decode_groups(D)) decode_int4_kernel(Int8DecodeArgs a) {
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
    i4_load_q<D>(a.q + (int64_t)(x.seq.q0 + token) * a.q_st +
                     (int64_t)(h * a.group + row - token * a.group) * a.q_sh,
                 g, c < rows, q);
    I8State<D> st;
    st.m = -INFINITY, st.l = 0.f;
#pragma unroll
    for (int t = 0; t < D / 16; ++t) st.o[t] = {0.f, 0.f, 0.f, 0.f};
    const int nb = (kv + kBlockSize - 1) / kBlockSize;
    const int b0 = i8_split_begin(nb, x.split, x.splits), b1 = i8_split_begin(nb, x.split + 1, x.splits);
    i4_split<D, false>(a, st, q, x.b, h, b0, b1, kv, vis, least, wave, nullptr);
    i8_finish<D, 1>(a, st, x.b, h, x.seq.q0, row0, rows, x.split, x.splits, wave, lds.o, lds.ml);
  }
}

// Four dims of a row from its n partials: load(k, m, l, o) gives partial k's. Unnormalised, with the row's
// sum in `sum`. Both forms of the merge come here, so that a row has the same bits from either. Little code
// in a loop: what a launch of a few microseconds runs once, it waits for from the instruction cache.
template <typename Load>
__device__ __forceinline__ float4_t i4_merge(int n, Load load, float& sum) {
  constexpr int N = 8;                                     // requested at a time
  float m = -INFINITY;
  float4_t o = {0.f, 0.f, 0.f, 0.f};
  sum = 0.f;
#pragma unroll 1
  for (int k0 = 0; k0 < n; k0 += N) {
    float mk[N], lk[N], to = m;
    float4_t x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) load(min(k0 + i, n - 1), mk[i], lk[i], x[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) to = vmax(to, mk[i]);
    const float neg = to == -INFINITY ? 0.f : -to, alpha = fast_exp2(m + neg);
    m = to;
    sum *= alpha;
    o *= alpha;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float w = k0 + i < n ? fast_exp2(mk[i] + neg) : 0.f;
      sum = fmaf(w, lk[i], sum);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(w, x[i][e], o[e]);
    }
  }
  return o;
}

// Rows of sequences with more than one split, as a launch of its own: four dims of a row a thread.
template <int D>
__global__ void __launch_bounds__(kI8Threads) decode_int4_merge_kernel(Int8DecodeArgs a) {
  constexpr int PER_ROW = D / 4;
  const int id = blockIdx.x * (kI8Threads / PER_ROW) + threadIdx.x / PER_ROW, d = threadIdx.x % PER_ROW * 4;
  const int behind = id - a.num_decode * a.heads;          // of the sequences past num_decode
  const int unit = behind < 0 ? a.by_group(id) : a.by_slots(behind);
  const int r = behind < 0 ? id - unit * a.group : behind - unit * a.row_slots;
  const int seq0 = a.by_kvh(unit), h = unit - seq0 * a.kvh, b = behind < 0 ? seq0 : a.num_decode + seq0;
  if (b >= a.num_seqs) return;
  const I8Seq seq = i8_seq(a, b);
  const int splits = i8_splits(a, seq, behind < 0);
  if (splits == 1 || r >= seq.n * a.group) return;
  const int64_t row = i8_partial(a, b, h, r, splits);
  float sum;
  const float4_t o = i4_merge(splits, [&](int k, float& m, float& l, float4_t& x) {
    const float2_t ml = ld<float2_t>(a.part_ml + 2 * (row + k));
    m = ml[0], l = ml[1], x = ld<float4_t>(a.part_o + (row + k) * D + d);
  }, sum);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;          // (nothing visible)
  const int token = a.by_group(r), head = h * a.group + r - token * a.group;
  st<half4_t>(a.out + (int64_t)(seq.q0 + token) * a.out_st + (int64_t)head * D + d, to_half4(o * inv));
}

// A pure-decode step's split map: what decode_int4_kernel looks up, worked out once for all layers of
// the step, and the counters that let a launch merge its own splits. int32: a header that names the
// plan, an entry for each split that the host's bounds allow (numbered densely, the real ones first) and a
// counter for each (sequence, KV head, tile of 16 heads), 0 between launches.
struct I4Map {
  static constexpr int kMagic = 0x344d5354, kHeader = 32, kEntry = 32, kIds = 8, kMaxSeqs = 4096;
  // of an entry: sequence (-1: behind the last split), split, splits, tokens, first and last block of
  // the split, id of the sequence's last block; from kIds on those of the split's first 16 blocks
  int* at;
  __host__ __device__ static int64_t entries(int num_seqs, int max_splits) { return (int64_t)num_seqs * max_splits; }
  __host__ __device__ static int64_t ints(int num_seqs, int max_splits, int kvh, int group) {
    return kHeader + entries(num_seqs, max_splits) * kEntry + (int64_t)num_seqs * kvh * ((group + 15) / 16);
  }
  __device__ __forceinline__ bool names(const Int8DecodeArgs& a) const {
    return table_entry(at) == kMagic && table_entry(at + 1) == a.num_seqs && table_entry(at + 2) == a.max_splits &&
           table_entry(at + 3) == a.kvh && table_entry(at + 4) == a.group && table_entry(at + 5) == a.max_blocks;
  }
  __device__ __forceinline__ const int* entry(int slot) const { return at + kHeader + (int64_t)slot * kEntry; }
  __device__ __forceinline__ int* counter(const Int8DecodeArgs& a, int b, int h, int tile) const {
    return at + kHeader + entries(a.num_seqs, a.max_splits) * kEntry +
           ((int64_t)b * a.kvh + h) * ((a.group + 15) / 16) + tile;
  }
};
static_assert(I4Map::kEntry >= I4Map::kIds + kI8SplitBlocks, "a split's blocks fit its entry");

// A wavefront an entry.
static __global__ void __launch_bounds__(kI8Threads) decode_int4_map_kernel(Int8DecodeArgs a, I4Map map) {
  const int lane = threadIdx.x % kWave;
  const int64_t id = (int64_t)blockIdx.x * kI8Threads + threadIdx.x;
  const int64_t counters = (int64_t)a.num_seqs * a.kvh * ((a.group + 15) / 16);
  for (int64_t i = id; i < counters; i += (int64_t)gridDim.x * kI8Threads) *(map.counter(a, 0, 0, 0) + i) = 0;
  if (id < I4Map::kHeader) {
    const int name[6] = {I4Map::kMagic, a.num_seqs, a.max_splits, a.kvh, a.group, a.max_blocks};
    int v = 0;
#pragma unroll
    for (int i = 0; i < 6; ++i) v = id == i ? name[i] : v;
    map.at[id] = v;
  }
  const int64_t slot = id / kWave;
  if (slot >= I4Map::entries(a.num_seqs, a.max_splits)) return;
  // one tile of heads: item = split (a.group = 1 for the lookup, every sequence one row)
  Int8DecodeArgs one = a;
  one.group = 1;
  I8Item x;
  int v = lane == 0 ? -1 : 0;
  if (i8_find(one, (int)slot, x)) {
    const int32_t* table = a.block_tables + x.b * a.bt_stride;
    const int nb = (x.seq.kv + kBlockSize - 1) / kBlockSize;
    const int b0 = i8_split_begin(nb, x.split, x.splits), b1 = i8_split_begin(nb, x.split + 1, x.splits);
    const int name[6] = {x.b, x.split, x.splits, x.seq.kv, b0, b1};
    if (lane >= I4Map::kIds && lane < I4Map::kIds + kI8SplitBlocks && b0 + lane - I4Map::kIds < b1)
      v = clamp_block(table[b0 + lane - I4Map::kIds], a.num_blocks);
    if (lane == 6 && nb > 0) v = clamp_block(table[nb - 1], a.num_blocks);
#pragma unroll
    for (int i = 0; i < 6; ++i) v = lane == i ? name[i] : v;
  }
  if (lane < I4Map::kEntry) const_cast<int*>(map.entry((int)slot))[lane] = v;
}

// decode_int4_kernel for a step with a map: decode rows only. A workgroup has its split and block ids one
// load after it starts, and the last split of a row tile to finish merges all of them, so that no
// launch follows.
template <int D>
__global__ void __launch_bounds__(kI8Threads, i8_decode_groups(D))
decode_int4_mapped_kernel(Int8DecodeArgs a, I4Map map, I8Div by_units) {
  __shared__ __align__(16) I8DecodeLds<D> lds;
  __shared__ int s_last;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave, c = lane % 16, g = lane / 16;
  const int tiles = (a.group + 15) / 16, units = a.kvh * tiles;
  if (!map.names(a)) {                                     // built for another plan: every row is NaN
    const half_t nan = (half_t)__builtin_nanf("");
    for (int64_t row = blockIdx.x; row < a.num_seqs; row += gridDim.x)
      for (int i = threadIdx.x; i < a.heads * D; i += kI8Threads) a.out[row * a.out_st + i] = nan;
    return;
  }
  const int64_t slots = I4Map::entries(a.num_seqs, a.max_splits);
  for (int64_t u = blockIdx.x; u < slots * units; u += gridDim.x) {
    const int slot = by_units((int)u), unit = (int)u - slot * units;
    const int h = tiles == 1 ? unit : unit / tiles, tile = tiles == 1 ? 0 : unit - h * tiles;
    const int* e = map.entry(slot);
    const int b = table_entry(e), split = table_entry(e + 1), splits = table_entry(e + 2);
    const int kv = table_entry(e + 3), b0 = table_entry(e + 4), b1 = table_entry(e + 5), last = table_entry(e + 6);
    if (b < 0) return;
    const int row0 = 16 * tile, rows = min(a.group - row0, 16);
    I8Query<D> q;
    i4_load_q<D>(a.q + (int64_t)b * a.q_st + (int64_t)(h * a.group + row0 + min(c, rows - 1)) * a.q_sh, g, c < rows, q);
    // a map of an earlier step: the sequence's length or its last block have moved
    const int len = i8_kv_len(a.seq_lens[b], a.max_blocks);
    const int end = kv > 0 ? clamp_block(a.block_tables[b * a.bt_stride + (kv - 1) / kBlockSize], a.num_blocks) : last;
    I8State<D> st;
    st.m = -INFINITY, st.l = 0.f;
#pragma unroll
    for (int t = 0; t < D / 16; ++t) st.o[t] = {0.f, 0.f, 0.f, 0.f};
    i4_split<D, true>(a, st, q, b, h, b0, b1, kv, kv, kv, wave, e + I4Map::kIds);
    if (len != kv || end != last) st.m = __builtin_nanf("");
    if (splits == 1) {
      i8_finish<D, 1>(a, st, b, h, b, row0, rows, 0, 1, wave, lds.o, lds.ml);
      continue;
    }
    // device-coherent partials: another workgroup, of any XCD, may merge them
    const int64_t base = ((int64_t)(b * a.kvh + h) * a.group + row0) * a.max_splits;
    const auto r_o = coherent_rsrc(a.part_o + base * D), r_ml = coherent_rsrc(a.part_ml + base * 2);
    i8_meet<D, 1>(st, rows, wave, lds.o, lds.ml, [&](int row, int d, float4_t o, float top, float sum) {
      const int at = row * a.max_splits + split;
      coherent_store4(r_o, (at * D + d) * 4, o);
      if (d == 0) coherent_store(r_ml, at * 8, top), coherent_store(r_ml, at * 8 + 4, sum);
    });
    __builtin_amdgcn_s_waitcnt(kWaitVmcntZero);            // they have arrived before the workgroup counts
    __syncthreads();
    int* counter = map.counter(a, b, h, tile);
    if (threadIdx.x == 0)
      s_last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == splits - 1;
    __syncthreads();
    if (!s_last) continue;
    int id = threadIdx.x;                                  // (so that nothing of this is worked out ahead, and held)
    asm volatile("" : "+v"(id));
#pragma unroll 1
    for (; id < rows * (D / 4); id += kI8Threads) {
      const int row = id / (D / 4), d = id % (D / 4) * 4;
      float sum;
      const float4_t o = i4_merge(splits, [&](int k, float& m, float& l, float4_t& x) {
        const int at = row * a.max_splits + k;
        m = coherent_load(r_ml, at * 8), l = coherent_load(r_ml, at * 8 + 4), x = coherent_load4(r_o, (at * D + d) * 4);
      }, sum);
      const float f = sum == 0.f ? 0.f : 1.f / sum;
      ts::st<half4_t>(a.out + (int64_t)b * a.out_st + (int64_t)(h * a.group + row0 + row) * D + d, to_half4(o * f));
    }
    if (threadIdx.x == 0) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

}  // namespace ts
