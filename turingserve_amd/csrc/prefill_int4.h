// Causal attention of several query rows per sequence over the 4-bit paged cache: the prompt kernel of the
// 8-bit cache (prefill_int8.h: rows in one list per KV head, 32 a wavefront, 64 tokens a step, the
// batch's steps shared evenly over the workgroups, tiles that are cut merged by a second launch) with
// another staging and a plainer softmax. A step's codes become fp16 numbers once, in registers on the
// way to LDS; there are no scales left over, so a score's exponent is one product-sum, P = 2^(s - m), and a
// row's sum is that of its P.
//
// 2048 rows on 4096 cached, 12/2 heads of 128: 84.3 to 88.5 us, 0.73 to 0.76 PFLOP/s (a product of 8192^3 in
// fp16 reaches 1.09), and 9.2 for the merge; the 8-bit kernel 84.9 and 9.5. Bound as that one: matrix units, vector units and LDS
// are each busy about two fifths of the time, in two wavefronts a SIMD. Five ragged prompts of 90 to 1100 rows,
// 14/2 heads of 64: 25.0 and 4.9 us, a tile's start before some eight steps. Without effect (a pass of two
// layers 182.0 to 182.2, or 191.4 to 192.0): a higher priority for half of the wavefronts or for one phase of a
// step; V's units to threads so that two lanes' stores meet in a bank, not four.
#pragma once

#include "decode_int4.h"
#include "prefill_int8.h"

namespace ts {

template <int D>
struct I4PrefillLds {
  __align__(16) half_t k[2][I8Tile<D>::HALVES], v[2][I8Tile<D>::HALVES];
  int walk[5][kWave];                                      // I8Walk
  int blk[kI8Window];
};

// The codes of a step that one thread widens: units of 16 channels of a K row, and of 4 tokens x 4
// channels of V (the even or the odd ones of an octet); 4 D of each in a step. Unit u belongs to block
// u / D of the step.
template <int D, int THREADS>
struct I4Stage {
  typedef I4Unit<D> U;
  static constexpr int UNITS = 4 * D;
  static constexpr int N = (UNITS + THREADS - 1) / THREADS;
  static constexpr bool ALL = UNITS % THREADS == 0;        // every thread has N units
  static constexpr bool UNIFORM = D >= kWave;              // a wavefront's unit lies in one block
  I4Bits bits;
  uint32_t k[N][2], kn[N];
  uint4_t v[N], vn[N];

  static __device__ __forceinline__ int unit(int i) { return threadIdx.x + i * THREADS; }
  // The ids of blocks w0 .. w0 + 3 of the window (the last real one again past the end).
  static __device__ __forceinline__ void ids(const I4PrefillLds<D>& lds, int w0, int last, int (&id)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) id[i] = lds.blk[min(w0 + min(unit(i), UNITS - 1) / D, last)];
  }
  // ... of a step's blocks from the table itself.
  static __device__ __forceinline__ void ids(const Int8DecodeArgs& a, const int32_t* table, int last,
                                             int (&id)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      int at = min(unit(i), UNITS - 1) / D;
      if (UNIFORM) at = __builtin_amdgcn_readfirstlane(at);
      id[i] = clamp_block(table_entry(table + min(at, last)), a.num_blocks);
    }
  }
  static __device__ __forceinline__ int64_t base(const Int8DecodeArgs& a, int id, int h) {
    const int blk = UNIFORM ? __builtin_amdgcn_readfirstlane(id) : id;
    return ((int64_t)blk * a.kvh + h) * U::BYTES;
  }
  __device__ __forceinline__ void request_k(const Int8DecodeArgs& a, const int (&id)[N], int h) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (ALL || unit(i) < UNITS) {
        const int in = unit(i) % D, row = in / (D / 16), group = 16 * (in % (D / 16)) / U::GROUP;
        const uint8_t* p = reinterpret_cast<const uint8_t*>(a.kc) + base(a, id[i], h);
        const int2_t w = ld<int2_t>(p + 8 * in);
        k[i][0] = w[0], k[i][1] = w[1];
        kn[i] = ld<uint32_t>(p + U::k_numbers(row, group));
      }
  }
  __device__ __forceinline__ void request_v(const Int8DecodeArgs& a, const int (&id)[N], int h, int part) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (ALL || unit(i) < UNITS) {
        const int in = unit(i) % D, quad = in / (D / 4), octet = in % (D / 4) / 2;
        const uint8_t* p = reinterpret_cast<const uint8_t*>(a.vc) + base(a, id[i], h);
        if (part == 0)
          v[i] = ld<uint4_t>(p + U::v_word(4 * quad, octet));
        else
          vn[i] = ld<uint4_t>(p + U::v_numbers(4 * quad, 8 * octet / U::GROUP));
      }
  }
  __device__ __forceinline__ void place_k(half_t* tile) const {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (ALL || unit(i) < UNITS) {
        const int key = unit(i) / (D / 16), chunk = 2 * (unit(i) % (D / 16));
        st<half8_t>(tile + I8Tile<D>::k_at(key, chunk), i4_octet(bits, k[i][0], kn[i]));
        st<half8_t>(tile + I8Tile<D>::k_at(key, chunk + 1), i4_octet(bits, k[i][1], kn[i]));
      }
  }
  template <int P>
  __device__ __forceinline__ void place_column(half_t* tile, uint32_t a, uint32_t a8, uint32_t b, uint32_t b8,
                                                      uint4_t n, half2_t low0, half2_t low1, int block, int quad,
                                               int d0) const {
    const half2_t x = i4_values<P>(bits, a, a8, i4_half2(n[0]), low0);
    const half2_t y = i4_values<P>(bits, b, b8, i4_half2(n[1]), low1);
    st<half4_t>(tile + I8Tile<D>::v_at(d0 + 2 * P, block, quad & 1) + 4 * (quad >> 1),
                half4_t{x[0], x[1], y[0], y[1]});
  }
  __device__ __forceinline__ void place_v(half_t* tile) const {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (ALL || unit(i) < UNITS) {
        const int in = unit(i) % D, block = unit(i) / D, quad = in / (D / 4);
        const int octet = in % (D / 4) / 2, odd = in % 2;
        const uint32_t half = odd ? 0x07060302u : 0x05040100u;     // (i4_odd, i4_even)
        const uint32_t a = __builtin_amdgcn_perm(v[i][1], v[i][0], half);
        const uint32_t b = __builtin_amdgcn_perm(v[i][3], v[i][2], half);
        const half2_t low0 = i4_finite(vn[i][2]), low1 = i4_finite(vn[i][3]);
        place_column<0>(tile, a, a >> 8, b, b >> 8, vn[i], low0, low1, block, quad, 8 * octet + odd);
        place_column<1>(tile, a, a >> 8, b, b >> 8, vn[i], low0, low1, block, quad, 8 * octet + odd);
        place_column<2>(tile, a, a >> 8, b, b >> 8, vn[i], low0, low1, block, quad, 8 * octet + odd);
        place_column<3>(tile, a, a >> 8, b, b >> 8, vn[i], low0, low1, block, quad, 8 * octet + odd);
      }
  }
};

// The exponentials of a step's 32 scores per lane, a few at a time (I8Exp without factors).
struct I4Exp {
  float t[32], x[32], sum[4][2];
  template <int N>
  __device__ __forceinline__ void share(int j, const float16_t (&s)[2], float sl2, float neg, float& l,
                                        half8_t (&p)[4]) {
    constexpr int PER = 32 / N;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = (j - 2) * PER + i, b = e / 8;          // summed
      if (e < 0 || e >= 32) continue;
      sum[b][e % 2] = e % 8 < 2 ? x[e] : sum[b][e % 2] + x[e];
      i8_pin(sum[b][e % 2]);
      p[b][e % 8] = (half_t)x[e];
      if (e % 8 == 7) {
        l += sum[b][0] + sum[b][1];
        i8_pin(l), i8_pin(p[b]);
      }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = (j - 1) * PER + i;
      if (e >= 0 && e < 32) x[e] = fast_exp2(t[e]), i8_pin(x[e]);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = j * PER + i;
      if (e < 32) t[e] = fmaf(s[e / 16][e % 16], sl2, neg), i8_pin(t[e]);
    }
  }
};

__device__ __forceinline__ float i4_top(const float (&top)[4]) {
  return vmax(vmax(top[0], top[1]), vmax(top[2], top[3]));
}

// Before the first step of a window: its scores, and the staging that a step does (i8_first).
template <int D, typename Mask, typename Work>
__device__ __forceinline__ float i4_first(I8Rows<D>& w, const half_t* kn, float16_t (&sc)[2], Mask mask,
                                          Work work) {
  typedef I8Rows<D> R;
  work(0);
#pragma unroll
  for (int v = 3; v < 5; ++v) work(v);
  float16_t zero;
#pragma unroll
  for (int i = 0; i < 16; ++i) zero[i] = 0.f;
#pragma unroll
  for (int j = 0; j < 2 * R::NQ; ++j)
    sc[j / R::NQ] = mfma_i8(w.operand(nullptr, kn, nullptr, R::NP + j), w.q[j % R::NQ],
                            j % R::NQ == 0 ? zero : sc[j / R::NQ]);
  mask(sc);
  float top[4];
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = sc[b / 2][8 * (b % 2) + e];
      top[b] = e == 0 ? x : vmax(top[b], x);
    }
  work(1);
  work(2);
  return i4_top(top);
}

// One step of a wavefront, in the phases of i8_step64. Returns each row's largest next score.
template <int D, typename Mask, typename Work>
__device__ __forceinline__ float i4_step64(I8Rows<D>& w, const half_t* vp, const half_t* kn, const half_t* vc,
                                           float16_t (&sc)[2], half8_t (&pr)[4], float sl2, Mask mask, Work work) {
  typedef I8Rows<D> R;
  constexpr int NQ = R::NQ, NP = R::NP, AHEAD = R::AHEAD;
  half8_t op[AHEAD];
#pragma unroll
  for (int j = 0; j < AHEAD && j < NP; ++j) op[j] = w.operand(vp, kn, vc, j);
  // Operand j, and the request of a later one below `end`. (The ring starts anew behind the barrier.)
  auto next = [&](int j, int end) {
    const half8_t x = op[j % AHEAD];
    if (j + AHEAD < end) op[j % AHEAD] = w.operand(vp, kn, vc, j + AHEAD);
    return x;
  };
  const float neg = w.m == -INFINITY ? 0.f : -w.m;
  // exponentials: NP + NQ shares beside the first two phases' MFMAs where both have as many
  constexpr int N = 2 * (NP < NQ ? NP : NQ);
  I4Exp ex;
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    w.o[j % R::DT] = mfma_i8(next(j, NP), pr[2 + j / R::DT], w.o[j % R::DT]);
    if (j < N / 2) ex.share<N>(j, sc, sl2, neg, w.l, pr);
    if (j == 0) work(0);                                   // requests of K to come
    __builtin_amdgcn_sched_barrier(0);
  }
  __syncthreads();
#pragma unroll
  for (int j = NP; j < NP + AHEAD; ++j) op[j % AHEAD] = w.operand(vp, kn, vc, j);
  if (w.moved) {
#pragma unroll
    for (int i = 0; i < R::DT; ++i) w.o[i] *= w.alpha;
  }
  float16_t zero;
#pragma unroll
  for (int i = 0; i < 16; ++i) zero[i] = 0.f;
#pragma unroll
  for (int j = 0; j < NQ; ++j) {
    sc[0] = mfma_i8(next(NP + j, R::ALL), w.q[j], j == 0 ? zero : sc[0]);
    if (j < N / 2) ex.share<N>(N / 2 + j, sc, sl2, neg, w.l, pr);
    for (int v = j * 2 / NQ; v < (j + 1) * 2 / NQ; ++v) work(3 + v);   // V's requests
    __builtin_amdgcn_sched_barrier(0);
  }
#pragma unroll
  for (int j = 0; j < NQ; ++j) {
    sc[1] = mfma_i8(next(NP + NQ + j, R::ALL), w.q[j], j == 0 ? zero : sc[1]);
    if (j < 2) ex.share<N>(N + j, sc, sl2, neg, w.l, pr);
    if (NQ < 2) ex.share<N>(N + 1, sc, sl2, neg, w.l, pr);
    if (j == NQ / 4) work(1);                              // K of a later step to LDS
    __builtin_amdgcn_sched_barrier(0);
  }
  mask(sc);
  float top[4];
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    w.o[j % R::DT] = mfma_i8(next(NP + 2 * NQ + j, R::ALL), pr[j / R::DT], w.o[j % R::DT]);
#pragma unroll
    for (int i = j * 32 / NP; i < (j + 1) * 32 / NP; ++i) {
      const int b = i / 2 % 4, e = i / 8 * 2 + i % 2;      // two scores of each block in turn
      const float x = sc[b / 2][8 * (b % 2) + e];
      top[b] = e == 0 ? x : vmax(top[b], x);
    }
    if (j == NP / 2) work(2);                              // V
    __builtin_amdgcn_sched_barrier(0);
  }
  return i4_top(top);
}

// One tile's steps [s0, s1) by the workgroup.
template <int D, int WAVES>
__device__ __forceinline__ void i4_piece(const Int8PrefillArgs& p, I4PrefillLds<D>& lds, const I8Chunk& k,
                                         int b, int tile, int h, int s0, int s1, bool whole, int slot) {
  typedef I8Rows<D> R;
  typedef I4Stage<D, WAVES * kWave> S;
  constexpr int DT = R::DT, THREADS = WAVES * kWave, ROWS = 32 * WAVES;
  const Int8DecodeArgs& a = p.a;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave, c = lane % 32, hh = lane / 32;
  const int rows = k.n * a.group, wrow = tile * ROWS + 32 * wave;
  const int row = min(wrow + c, rows - 1);                 // (rows past the last one stand in for it)
  const int token = a.by_group(row), head = h * a.group + row - token * a.group, vis = i8_sees(k, token);
  // rows ascend in tokens: the wavefront's first row sees least
  const int least = i8_sees(k, a.by_group(min(wrow, rows - 1)));
  const int sees = i8_sees(k, a.by_group(min(rows, (tile + 1) * ROWS) - 1));
  const int nb = (sees + kBlockSize - 1) / kBlockSize;     // blocks that the tile sees
  R w;
  w.kat = I8Tile<D>::k_at(c, hh);
#pragma unroll
  for (int i = 0; i < 4; ++i) w.vat[i] = I8Tile<D>::v_at(D < 32 ? c % D : c, i, hh);
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) w.o[t][i] = 0.f;
  w.m = -INFINITY, w.l = 0.f, w.alpha = 1.f, w.moved = false;

  s1 = min(s1, (nb + kI8StepBlocks - 1) / kI8StepBlocks);  // (nothing visible: no step)
  for (int w0 = s0; w0 < s1; w0 += kI8Window / kI8StepBlocks) {
    // a window of the sequence's blocks
    const int n = min(s1 - w0, kI8Window / kI8StepBlocks);
    const int blocks = min(nb - w0 * kI8StepBlocks, n * kI8StepBlocks), last = blocks - 1;
    __syncthreads();                                       // the last window's and piece's reads
    const int32_t* table = a.block_tables + b * a.bt_stride + w0 * kI8StepBlocks;
    S stage;
    int id0[S::N], id1[S::N], id2[S::N];                   // of the next step, the second, the third
    S::ids(a, table, last, id0);
    stage.request_k(a, id0, h);
    for (int at = threadIdx.x; at < blocks; at += THREADS) lds.blk[at] = clamp_block(table[at], a.num_blocks);
    if (w0 == s0) {                                        // q behind what the first scores wait for
      const half_t* qrow = a.q + (int64_t)(k.q0 + token) * a.q_st + (int64_t)head * a.q_sh;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) w.q[i] = ld<half8_t>(qrow + 16 * i + 8 * hh);
    }
    for (int i = threadIdx.x; i < I8Tile<D>::HALVES / 8; i += THREADS)
      st<half8_t>(lds.v[1] + 8 * i, half8_t{0, 0, 0, 0, 0, 0, 0, 0});
    stage.place_k(lds.k[0]);
    __syncthreads();
    S::ids(lds, 0, last, id0);
    S::ids(lds, kI8StepBlocks, last, id1);

    // The pipeline of the 8-bit kernel: step i reads K of step i + 1 in k[(i + 1) % 2], V of steps i - 1
    // and i in v[(i - 1) % 2] and v[i % 2], and stages K of step i + 2 and V of step i + 1. Past the
    // window's end the last blocks are staged again, and the scores of the step behind it are not used.
    float16_t sc[2];
    half8_t pr[4];
#pragma unroll
    for (int e = 0; e < 8; ++e) pr[2][e] = pr[3][e] = (half_t)0.f;
    auto step = [&](auto parity, auto first, int i) {
      constexpr int P = decltype(parity)::value;           // i % 2
      auto work = [&](int part) {
        if (part == 0) {
          stage.request_k(a, id1, h);
          S::ids(lds, (i + 3) * kI8StepBlocks, last, id2);
        }
        if (part >= 3) stage.request_v(a, id0, h, part - 3);
        if (part == 1) stage.place_k(lds.k[P]);
        if (part == 2) stage.place_v(lds.v[1 - P]);
      };
      auto mask = [&](float16_t (&x)[2]) {
        const int at = w0 + i + 1;
        if ((at + 1) * kI8Keys > least) {
          const int key0 = at * kI8Keys + 4 * hh;
#pragma unroll
          for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              x[kt][e] = key0 + 32 * kt + 8 * (e / 4) + e % 4 < vis ? x[kt][e] : -INFINITY;
        }
      };
      const float best = decltype(first)::value
                             ? i4_first<D>(w, lds.k[0], sc, mask, work)
                             : i4_step64<D>(w, lds.v[1 - P], lds.k[1 - P], lds.v[P], sc, pr, a.sl2, mask, work);
      i8_reference<D>(w, i + 1 < n ? best * a.sl2 : w.m);  // (its own reference moves none, also a NaN)
#pragma unroll
      for (int e = 0; e < S::N; ++e) id0[e] = id1[e], id1[e] = id2[e];
    };
    step(I8Const<1>(), I8Const<1>(), -1);
    for (int i = 0; i < n; i += 2) {
      step(I8Const<0>(), I8Const<0>(), i);
      if (i + 1 < n) step(I8Const<1>(), I8Const<0>(), i + 1);
    }
    const half_t* vl = lds.v[(n - 1) & 1];                 // the last step's second half
#pragma unroll
    for (int j = 0; j < R::NP; ++j)
      w.o[j % DT] = mfma_i8(ld<half8_t>(vl + w.vat[2 + j / DT] + j % DT * 32 * kI8Keys), pr[2 + j / DT],
                            w.o[j % DT]);
  }

  // lanes c and c + 32 hold the two halves of row c's sum
  const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(w.l), __float_as_uint(w.l), false, false);
  const float l = __uint_as_float(both[0]) + __uint_as_float(both[1]);
  if (wrow + c >= rows) return;
  const int64_t at = (int64_t)slot * ROWS + 32 * wave + c;
  if (!whole && hh == 0) st<float2_t>(a.part_ml + 2 * at, float2_t{w.m, l});
  const float f = !whole ? 1.f : l == 0.f ? 0.f : 1.f / l;     // nothing visible: zeros
  half_t* dst = a.out + (int64_t)(k.q0 + token) * a.out_st + (int64_t)head * D;
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int d = 32 * t + 8 * (i / 4) + 4 * hh;
      if (D < 32 && d >= D) break;
      const float4_t x = float4_t{w.o[t][i], w.o[t][i + 1], w.o[t][i + 2], w.o[t][i + 3]} * f;
      if (whole)
        st<half4_t>(dst + d, i8_result<true>(x));
      else
        st<float4_t>(a.part_o + at * D + d, x);
    }
}

template <int D>
__global__ void __launch_bounds__(i8_prefill_waves(D) * kWave, D > 128 ? 1 : 2)
prefill_int4_kernel(Int8PrefillArgs p) {
  constexpr int WAVES = i8_prefill_waves(D), ROWS = 32 * WAVES;
  __shared__ __align__(16) I4PrefillLds<D> lds;
  i8_share<ROWS>(p, lds.walk, [&](const I8Place& place, int h, int s0, int s1, bool whole, int slot) {
    i4_piece<D, WAVES>(p, lds, place.k, place.seq, place.tile, h, s0, s1, whole, slot);
  });
}

}  // namespace ts
