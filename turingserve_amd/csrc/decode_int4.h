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
//
// 64 sequences of 128 to 4096 tokens, 12/2 heads of 128: 11.0 us (9.5 at least) and 4.0 for the merge, 24 MB of
// cache (4.9 us at a copy's 4.85 TB/s); one sequence of 6000: 5.1 (4.2) and 2.8 (2.3). Neither memory nor an
// issue port bounds the large ones: those 64 are 632 items (a split of a KV head) on 256 CUs, two or three a CU
// where the mean is 2.5, and vector instructions, some 400 a pair of blocks at head_dim 128 and half of them
// the widening, are issued in 42 % of a SIMD's cycles. An item's chain is much of what is left, and all of the
// small ones: length and table 1.2 us, first codes 0.75, two pairs 1.8, the wavefronts' meeting and the partial
// 0.9, then the merge's launch. Blocks a split, us a pass by events over replays, 16 / 32: one of 6000 (48
// items, four layers) 34.2 / 40.6, those 64 58.7 / 68.0, four of 8000 to 32768 (440) 62.7 / 63.0, 24 of 200 to
// 8192 over 14/2 heads of 64 (424, eight layers) 81.6 / 92.0; but 256 of 100 to 600 (800) 72.3 / 64.4, 48 rows
// beside a chunk of 512 (952) 90.1 / 85.6, 128 of 500 to 4000 (1814) 111.6 / 97.2, 200 of 200 to 4000 over 14/2
// heads of 64 (2180) 96.3 / 83.7, 32 of 500 to 16000 over 28/4 heads of 128 (2296, two layers) 57.9 / 53.3, 64
// of 2000 to 8000 over 8/8 heads of 64 (8888, two layers) 121.9 / 106.7: 16 are ahead or level up to some 630
// items, 32 from 800 on, by 5 to 14 %. The length is one for all batches. Earlier forms of the kernel, one of
// 6000 / those 64 / four long ones: 8 blocks 50 / 68 / 78 where 16 took 40.1 / 61.1 / 64.1, eight wavefronts
// with 32 45.6 / 66 / 72. Two 16-row tiles a workgroup, the codes widened once for both: 16 chunks of five rows
// 52 against 44, ahead only at chunks of 128 (57 / 64). The merge inside the launch, behind a map of the step's
// splits with counters: 48 to 56, 64 to 91 and 79 to 96, its loads past the caches and its code cold.
#pragma once

#include "decode_int8.h"
#include "int4_kv.h"

namespace ts {

constexpr int kI4Waves = 4, kI4Threads = kI4Waves * kWave;
// Blocks of a split, as long as kI8MaxSplits suffice: the length that batches of few items want (above).
constexpr int kI4SplitBlocks = 16;

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
__device__ __forceinline__ float4_t i4_scores(const I4Bits& k, const I4Block<D>& x, const I8Query<D>& q, int g) {
  float4_t s = {0.f, 0.f, 0.f, 0.f};
  if constexpr (D >= 32) {
#pragma unroll
    for (int i = 0; i < I4Block<D>::KW; ++i) s = mfma16x16x32(i4_octet(k, x.k[i], x.kn[i / 4]), q.x[i], s);
  } else {
    s = mfma16x16x16(lo4(i4_octet(k, x.k[0] >> (8 * (g & 1)), x.kn[0])), lo4(q.x[0]), s);   // (half an octet)
  }
  return s;
}

// Output tiles 2 P + ODD of an octet, P from 0 on: w the four pairs of tokens (blocks a and b), one channel a
// nibble.
template <int D, int ODD, int P>
__device__ __forceinline__ void i4_tiles(const I4Bits& k, float4_t* o, const uint32_t (&w)[4], const half2_t (&step)[4],
                                         const half2_t (&low)[4], half8_t p) {
  if constexpr (2 * P + ODD < D / 16 && P < 4) {
    half2_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i4_values<P>(k, w[i], w[i] >> 8, step[i], low[i]);
    const half8_t x = {v[0][0], v[0][1], v[1][0], v[1][1], v[2][0], v[2][1], v[3][0], v[3][1]};
    o[2 * P + ODD] = mfma16x16x32(x, p, o[2 * P + ODD]);
    i4_tiles<D, ODD, P + 1>(k, o, w, step, low, p);
  }
}

// O^T += V^T . P^T over the pair, output tile t taking channels VW i + t: the even channels of an octet, then
// the odd ones, two tokens to a register.
template <int D>
__device__ __forceinline__ void i4_pv(const I4Bits& k, float4_t (&o)[D / 16], const I4Block<D> (&x)[2], int c,
                                      half8_t p) {
  half2_t step[4], low[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) step[i] = i4_half2(x[i / 2].vn[i % 2]), low[i] = i4_finite(x[i / 2].vn[2 + i % 2]);
#pragma unroll
  for (int j = 0; j < I4Block<D>::VO; ++j) {
    uint32_t w[4];
    auto word = [&](int i) {
      uint32_t v = x[i / 4].v[j][i % 4];
      // the lane's channels first: 4 (c % 2) .., 2 (c % 4) .., c % 8 of the octet
      if constexpr (D == 64) v >>= 8 * (c & 1);
      if constexpr (D == 32) v >>= 4 * (c & 3);
      if constexpr (D == 16) v >>= 4 * (c / 2 & 3) + 16 * (c & 1);
      return v;
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = i4_even(word(2 * i), word(2 * i + 1));
    i4_tiles<D, 0, 0>(k, o + 8 * j, w, step, low, p);
    if constexpr (D >= 32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = i4_odd(word(2 * i), word(2 * i + 1));
      i4_tiles<D, 1, 0>(k, o + 8 * j, w, step, low, p);
    }
  }
}

// The softmax of the scores over a pair of blocks: its reference and sum moved on, O with them; P.
template <int D>
__device__ __forceinline__ half8_t i4_softmax(I8State<D>& st, const float4_t& sa, const float4_t& sb, float sl2) {
  const float top = rows_max(vmax(vmax(vmax(sa[0], sa[1]), vmax(sa[2], sa[3])),
                                  vmax(vmax(sb[0], sb[1]), vmax(sb[2], sb[3])))) * sl2;
  // !(<=): a NaN score (a token of NaN) moves the reference to NaN, where it stays
  const float was = st.m;
  const bool move = !(top <= was + kI8Rescale);
  st.m = move ? vmax(was, top) : was;
  if (__ballot(move && was != -INFINITY)) {                // (before a row's first token all is 0)
    const float alpha = move ? fast_exp2(was - st.m) : 1.f;
    st.l *= alpha;
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
  return p;
}

// One pair of blocks (tokens ta .. and tb .. of the sequence). A row sees the tokens below `vis`, all
// rows of the tile those below `least`. sl2: scale * log2(e) > 0. next_k() requests the next pair's K as
// soon as this one's is used up, next_v() its V.
template <int D, typename NextK, typename NextV>
__device__ __forceinline__ void i4_step(const I4Bits& k, I8State<D>& st, const I4Block<D> (&x)[2],
                                        const I8Query<D>& q, float sl2, int ta, int tb, int vis, int least, int c,
                                        int g, NextK next_k, NextV next_v) {
  float4_t sa = i4_scores<D>(k, x[0], q, g), sb = i4_scores<D>(k, x[1], q, g);
  next_k();
  if (tb + kBlockSize > least || ta + kBlockSize > least) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      sa[r] = ta + 4 * g + r < vis ? sa[r] : -INFINITY;
      sb[r] = tb + 4 * g + r < vis ? sb[r] : -INFINITY;
    }
  }
  const half8_t p = i4_softmax<D>(st, sa, sb, sl2);
  // What stands past the end is finite (i4_finite), and p is 0 there.
  i4_pv<D>(k, st.o, x, c, p);
  next_v();
}

// Entries of a sequence's table from block `from` on, one a lane, asked for ahead of its split (or none).
struct I4Window {
  int from = INT32_MAX, entry = 0;
};

// One split [b0, b1) of a sequence's blocks by one wavefront (of kI4Waves). Blocks are taken 64 at a
// time: lane i holds block i's id (i + from's that of a window that holds the split). x is the kernel's: as a local
// here it took four registers more.
template <int D>
__device__ __forceinline__ void i4_split(const Int8DecodeArgs& a, I8State<D>& st, const I8Query<D>& q, int b, int h,
                                         int b0, int b1, int len, int vis, int least, int wave, I4Window ahead,
                                         I4Block<D> (&x)[2]) {
  const int lane = threadIdx.x % kWave, c = lane % 16, g = lane / 16;
  const int32_t* table = a.block_tables + b * a.bt_stride;
  const uint8_t *kc = reinterpret_cast<const uint8_t*>(a.kc), *vc = reinterpret_cast<const uint8_t*>(a.vc);
  for (int lo = b0; lo < b1; lo += kWave) {
    const int n = min(b1 - lo, kWave);
    int blk = 0, first = 0;
    if (b0 >= ahead.from && b1 - ahead.from <= kWave)
      blk = clamp_block(ahead.entry, a.num_blocks), first = b0 - ahead.from;
    else if (lane < n)
      blk = clamp_block(table[lo + lane], a.num_blocks);
    auto unit = [&](int i) {                               // of block i of the 64, or of the last one
      return ((int64_t)__builtin_amdgcn_readlane(blk, first + min(i, n - 1)) * a.kvh + h) * I4Unit<D>::BYTES;
    };
    constexpr int STEP = 2 * kI4Waves;
    const I4Bits k;
    int i = 2 * wave;
    if (i >= n) continue;
    int64_t at[2] = {unit(i), unit(i + 1)};
#pragma unroll
    for (int u = 0; u < 2; ++u) i4_load_k<D>(kc + at[u], c, g, x[u]);
#pragma unroll
    for (int u = 0; u < 2; ++u) i4_load_v<D>(vc + at[u], c, g, x[u]);
#pragma unroll 1
    for (; i < n; i += STEP) {
      // with an odd count the last pair's second block is its first, wholly past the end
      const int ta = (lo + i) * kBlockSize;
      const int tb = i + 1 < n ? ta + kBlockSize : len;
      const bool more = i + STEP < n;
      if (more) at[0] = unit(i + STEP), at[1] = unit(i + STEP + 1);
      i4_step<D>(k, st, x, q, a.sl2, ta, tb, vis, least, c, g, [&] {
        if (!more) return;
#pragma unroll
        for (int u = 0; u < 2; ++u) i4_load_k<D>(kc + at[u], c, g, x[u]);
      }, [&] {
        if (!more) return;
#pragma unroll
        for (int u = 0; u < 2; ++u) i4_load_v<D>(vc + at[u], c, g, x[u]);
      });
    }
  }
}

template <int D>
struct I4DecodeLds {
  static constexpr int ROW = D + 4;      // floats of a row: rows start on different banks
  float o[kI4Waves * 16 * ROW];
  __align__(16) float m[16][kI4Waves], l[16][kI4Waves];
};

__device__ __forceinline__ float i4_largest(const float (&m)[kI4Waves]) {
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kI4Waves; i += 4) {
    const float4_t x = ld<float4_t>(m + i);
    top = vmax(top, vmax(vmax(x[0], x[1]), vmax(x[2], x[3])));
  }
  return top;
}

// The wavefronts' states meet in LDS, each brought to the rows' common reference first: emit(row, d, o,
// reference, sum) for 4 dims of each row, unnormalised.
template <int D, typename Emit>
__device__ __forceinline__ void i4_meet(const I8State<D>& st, int rows, int wave, I4DecodeLds<D>& lds, Emit emit) {
  constexpr int VW = D / 16, ROW = I4DecodeLds<D>::ROW;
  int id = threadIdx.x;                                    // (so that no place is worked out ahead, and held)
  asm volatile("" : "+v"(id));
  const int lane = id % kWave, c = lane % 16, g = lane / 16;
  const float l = rows_sum(st.l);
  __syncthreads();                                         // the last item's reads of LDS
  if (g == 0) lds.m[c][wave] = st.m;
  __syncthreads();
  if (c < rows) {
    const float top = i4_largest(lds.m[c]), f = st.m == -INFINITY ? 0.f : fast_exp2(st.m - top);
    float* dst = lds.o + (wave * 16 + c) * ROW;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int t = 0; t < VW; ++t) dst[VW * (4 * g + r) + t] = st.o[t][r] * f;
    if (g == 0) lds.l[c][wave] = l * f;
  }
  __syncthreads();
  for (int u = id; u < rows * (D / 4); u += kI4Threads) {
    const int row = u / (D / 4), d = u % (D / 4) * 4;
    float4_t o = ld<float4_t>(lds.o + row * ROW + d), s = ld<float4_t>(&lds.l[row][0]);
#pragma unroll
    for (int w = 1; w < kI4Waves; ++w) o += ld<float4_t>(lds.o + (w * 16 + row) * ROW + d);
#pragma unroll
    for (int i = 4; i < kI4Waves; i += 4) s += ld<float4_t>(&lds.l[row][i]);
    emit(row, d, o, i4_largest(lds.m[row]), (s[0] + s[1]) + (s[2] + s[3]));
  }
}

// The row (or its partial) is written.
template <int D>
__device__ __forceinline__ void i4_finish(const Int8DecodeArgs& a, const I8State<D>& st, int b, int h, int q0,
                                          int row0, int rows, int split, int splits, int wave, I4DecodeLds<D>& lds) {
  i4_meet<D>(st, rows, wave, lds, [&](int row, int d, float4_t o, float top, float sum) {
    if (splits == 1) {
      const float f = sum == 0.f ? 0.f : 1.f / sum;        // no visible key: zeros
      const int token = a.by_group(row0 + row), head = h * a.group + row0 + row - token * a.group;
      ts::st<half4_t>(a.out + (int64_t)(q0 + token) * a.out_st + (int64_t)head * D + d, i8_result<true>(o * f));
    } else {
      const int64_t at = i8_partial(a, b, h, row0 + row, splits) + split;
      ts::st<float4_t>(a.part_o + at * D + d, o);
      if (d == 0) ts::st<float2_t>(a.part_ml + 2 * at, float2_t{top, sum});
    }
  });
}

// Workgroups that a CU holds at once, by registers.
constexpr int i4_decode_groups(int D) { return D > 128 ? 2 : 4; }

// i8_find of up to 64 sequences in two parts: what a lane holds of its sequence, which every wavefront leaves in
// LDS (all of them the same), and an item's place, so that a workgroup's later items need neither the lengths nor
// the sums again.
struct I4Found {
  int kv, start, q0, n, splits, tiles, sum;                // sum: items up to and with this sequence
};
__device__ __forceinline__ I4Found i4_found(const Int8DecodeArgs& a) {
  const int lane = threadIdx.x % kWave;
  I4Found f = {};
  if (lane < a.num_seqs) {
    const I8Seq s = i8_seq(a, lane);
    f.kv = s.kv, f.start = s.start, f.q0 = s.q0, f.n = s.n;
    f.splits = i8_splits<kI4SplitBlocks>(a, s, lane < a.num_decode);
    f.tiles = (s.n * a.group + 15) / 16;
  }
  f.sum = i8_scan(f.splits * f.tiles);
  return f;
}
__device__ __forceinline__ bool i4_pick(const I4Found& f, int item, I8Item& x) {
  const uint64_t past = __ballot(f.sum > item);
  if (!past) return false;
  x.b = __ffsll((unsigned long long)past) - 1;
  auto of = [&](int v) { return __builtin_amdgcn_readlane(v, x.b); };
  x.splits = of(f.splits);
  const unsigned t = of(f.tiles), in = item - (of(f.sum) - x.splits * (int)t);
  x.split = (int)(t == 1 ? in : in / t), x.tile = (int)(in - x.split * t);
  x.seq = {of(f.q0), of(f.n), of(f.kv), of(f.start)};
  return x.split < x.splits;                               // (as i8_find)
}

// The blocks of an item's split.
__device__ __forceinline__ void i4_blocks(const I8Item& x, int& b0, int& b1) {
  const int nb = (x.seq.kv + kBlockSize - 1) / kBlockSize;
  b0 = i8_split_begin(nb, x.split, x.splits), b1 = i8_split_begin(nb, x.split + 1, x.splits);
}

// The rows of q of an item of KV head h.
template <int D>
__device__ __forceinline__ void i4_query(const Int8DecodeArgs& a, const I8Item& x, int h, I8Query<D>& q) {
  const int c = threadIdx.x % 16, g = threadIdx.x % kWave / 16;
  const int row0 = 16 * x.tile, rows = min(x.seq.n * a.group - row0, 16);
  const int row = row0 + min(c, rows - 1), token = a.by_group(row);
  i4_load_q<D>(a.q + (int64_t)(x.seq.q0 + token) * a.q_st +
                   (int64_t)(h * a.group + row - token * a.group) * a.q_sh,
               g, c < rows, q);
}

template <int D>
__device__ __forceinline__ void i4_item(const Int8DecodeArgs& a, const I8Item& x, int h, const I8Query<D>& q,
                                        const I4Window& ahead, I8State<D>& st, int wave, I4Block<D> (&blocks)[2]) {
  const int row0 = 16 * x.tile, rows = min(x.seq.n * a.group - row0, 16), kv = x.seq.kv;
  const int token = a.by_group(row0 + min((int)threadIdx.x % 16, rows - 1));
  const int vis = min(kv, max(0, x.seq.start + token + 1));
  const int least = min(kv, max(0, x.seq.start + a.by_group(row0) + 1));
  st.m = -INFINITY, st.l = 0.f;
#pragma unroll
  for (int t = 0; t < D / 16; ++t) st.o[t] = {0.f, 0.f, 0.f, 0.f};
  int b0, b1;
  i4_blocks(x, b0, b1);
  i4_split<D>(a, st, q, x.b, h, b0, b1, kv, vis, least, wave, ahead, blocks);
}
template <int D>
__device__ __forceinline__ void i4_finish(const Int8DecodeArgs& a, const I8Item& x, int h, const I8State<D>& st,
                                          int wave, I4DecodeLds<D>& lds) {
  const int row0 = 16 * x.tile;
  i4_finish<D>(a, st, x.b, h, x.seq.q0, row0, min(x.seq.n * a.group - row0, 16), x.split, x.splits, wave, lds);
}

// Decode rows of one tile alone, a workgroup for each split that the host's bound allows. It knows its split at
// once, so that the row of q, the length and the part of the table where the split must lie (as long as
// splits are of kI4SplitBlocks) are requested together. First splits come first: those past a sequence's
// end, which a graph's bound leaves many of, are dispatched behind the real ones. A split's (sequence, KV
// head)s are shifted by its number, and by half of them every 256 workgroups, so that no XCD (a workgroup in
// eight) and no CU has the splits of one sequence alone.
template <int D>
__global__ void __launch_bounds__(kI4Threads, i4_decode_groups(D)) decode_int4_direct_kernel(Int8DecodeArgs a) {
  __shared__ __align__(16) I4DecodeLds<D> lds;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int units = a.num_seqs * a.kvh, u = blockIdx.x;
  I8Item x;
  x.split = a.by_units(u), x.tile = 0;
  const int first = x.split * units;
  int unit = u - first + x.split + first / 256 * (units / 2);
  unit -= a.by_units(unit) * units;
  x.b = a.by_kvh(unit);
  const int h = unit - x.b * a.kvh;
  I4Window ahead;
  ahead.from = max(x.split - 1, 0) * kI4SplitBlocks;
  ahead.entry = a.block_tables[x.b * a.bt_stride + min(ahead.from + lane, a.max_blocks - 1)];
  x.seq.q0 = x.b, x.seq.n = 1;
  I8Query<D> q;
  i4_query<D>(a, x, h, q);
  x.seq = i8_seq(a, x.b);
  x.splits = i8_splits<kI4SplitBlocks>(a, x.seq, true);
  if (x.split >= x.splits) return;
  I8State<D> st;
  I4Block<D> blocks[2];
  i4_item<D>(a, x, h, q, ahead, st, wave, blocks);
  i4_finish<D>(a, x, h, st, wave, lds);
}

// Every item of a batch, as many workgroups as the CUs hold, which go round. FEW: up to 64 sequences, of which
// the next item's place and the ids of its blocks are at hand when one ends, or that there is none (what it
// saves where a batch has fewer items than workgroups).
template <int D, bool FEW>
__global__ void __launch_bounds__(kI4Threads, i4_decode_groups(D)) decode_int4_kernel(Int8DecodeArgs a) {
  __shared__ __align__(16) I4DecodeLds<D> lds;
  __shared__ int saved[FEW ? 7 : 1][kWave];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  I8Item x;
  I4Window ahead;
  if constexpr (FEW) {
    const I4Found f = i4_found(a);
    if (!i4_pick(f, a.by_kvh((int)blockIdx.x), x)) return;
    saved[0][lane] = f.kv, saved[1][lane] = f.start, saved[2][lane] = f.q0, saved[3][lane] = f.n;
    saved[4][lane] = f.splits, saved[5][lane] = f.tiles, saved[6][lane] = f.sum;
  }
  for (int64_t u = blockIdx.x; u <= INT32_MAX; u += gridDim.x) {     // (the entry point refuses more)
    const int item = a.by_kvh((int)u), h = (int)u - item * a.kvh;
    if constexpr (!FEW) {
      if (!i8_find<kI4SplitBlocks>(a, item, x)) return;
    }
    I8Query<D> q;
    i4_query<D>(a, x, h, q);
    I8State<D> st;
    I4Block<D> blocks[2];
    i4_item<D>(a, x, h, q, ahead, st, wave, blocks);
    const I8Item now = x;
    bool more = true;
    if constexpr (FEW) {
      const int64_t next = u + gridDim.x;
      const I4Found f = {saved[0][lane], saved[1][lane], saved[2][lane], saved[3][lane],
                         saved[4][lane], saved[5][lane], saved[6][lane]};
      more = next <= INT32_MAX && i4_pick(f, a.by_kvh((int)next), x);
      ahead.from = INT32_MAX;
      if (more) {
        int b0, b1;
        i4_blocks(x, b0, b1);
        if (b1 > b0) ahead.from = b0, ahead.entry = a.block_tables[x.b * a.bt_stride + min(b0 + lane, b1 - 1)];
      }
    }
    i4_finish<D>(a, now, h, st, wave, lds);
    if (!more) return;
  }
}

}  // namespace ts
