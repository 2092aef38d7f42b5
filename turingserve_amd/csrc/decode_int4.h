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
// time: lane i holds block i's id.
template <int D>
__device__ __forceinline__ void i4_split(const Int8DecodeArgs& a, I8State<D>& st, const I8Query<D>& q, int b,
                                         int h, int b0, int b1, int len, int vis, int least, int wave) {
  const int lane = threadIdx.x % kWave, c = lane % 16, g = lane / 16;
  const int32_t* table = a.block_tables + b * a.bt_stride;
  const uint8_t *kc = reinterpret_cast<const uint8_t*>(a.kc), *vc = reinterpret_cast<const uint8_t*>(a.vc);
  for (int lo = b0; lo < b1; lo += kWave) {
    const int n = min(b1 - lo, kWave);
    int blk = 0;
    if (lane < n) blk = clamp_block(table[lo + lane], a.num_blocks);
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
    i4_split<D>(a, st, q, x.b, h, b0, b1, kv, vis, least, wave);
    i8_finish<D, 1>(a, st, x.b, h, x.seq.q0, row0, rows, x.split, x.splits, wave, lds.o, lds.ml);
  }
}

}  // namespace ts
