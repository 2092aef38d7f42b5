// Causal attention of several query rows per sequence over the 8-bit paged cache (prompt chunks,
// speculative verification): the bottom-right mask, row i of a sequence with n query rows sees the
// first seq_len - n + i + 1 tokens.
//
// The query rows of all heads that share a KV head stand in one list (row = token * group + head),
// so a workgroup's tile of 32 rows per wavefront reads each code once for all of them. Per step of
// 64 tokens the workgroup widens the codes of K and V to fp16 once, in registers on the way to
// LDS (exact; the scales stay out of the tiles), and each wavefront computes, on
// v_mfma_f32_32x32x16_f16,
//   S^T[64 tokens][32 rows] = K . Q^T,   online softmax in fp32,   O^T += V^T . P^T.
// A block's K scale multiplies its scores in fp32. Its V scale, measured against the largest one
// so far (vref), goes into the exponent: P' = 2^(s - m + log2(vs / vref)) is what is rounded to
// fp16 and multiplied by the codes of V, and a row's sum adds each block's P' times vref / vs. A
// ratio below 2^-30 counts as 2^-30: at most 127 * 2^-30 of vref.
//
// Lane l is split into c = l % 32 and h = l / 32: a result lane holds S^T[8 (i / 4) + 4 h + i % 4][c],
// i = 0..15, so a lane's scores all belong to row c, and its P values for a block's 16 tokens (i % 8
// of one half) are the B operand of the P.V step as they stand when V^T lies in LDS with the
// tokens of a block in the order {0-3, 8-11 | 4-7, 12-15}.
//
// The batch's steps (of every sequence, tile and KV head, in that order) are shared evenly over
// the launched workgroups. Where a share begins or ends inside a tile, its part of the tile is left
// as a partial (m, l, O in fp32) for the merge launch; a workgroup leaves two at most. Every
// workgroup works the shares out for itself from the sequences' lengths.
#pragma once

#include "decode_int8.h"

namespace ts {

typedef float float16_t __attribute__((ext_vector_type(16)));

constexpr int kI8Keys = 64;              // tokens of a step
constexpr int kI8StepBlocks = kI8Keys / kBlockSize;
constexpr int kI8Window = 256;           // blocks whose ids and scales are held in LDS at a time
constexpr int kI8MinShare = 4;           // steps that a workgroup is worth
constexpr float kI8LeastRatio = -30.f;   // log2 of the least V scale ratio
constexpr float kI8LeastFactor = 1e-30f;
constexpr int kI8Kept = 4;               // times 64 pairs (sequence, tile) whose steps are kept

template <int N>
struct I8Const {
  static constexpr int value = N;
};

struct Int8PrefillArgs {
  Int8DecodeArgs a;                      // (part_o, part_ml: two partials of a tile per workgroup)
  const int32_t* qsl;
  int64_t num_tokens;
  int num_seqs, first;                   // sequences first .. num_seqs - 1
  int tiles;                             // of the longest chunk by the host's bound
  int groups;                            // workgroups of the main launch
};

__device__ __forceinline__ float16_t mfma_i8(half8_t a, half8_t b, float16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

template <int D>
struct I8Tile {
  static constexpr int KCHUNKS = D / 8;                    // 16-byte chunks of a K row
  static constexpr int KSWZ = (KCHUNKS < 16 ? KCHUNKS : 16) - 1;
  static constexpr int HALVES = kI8Keys * D;               // of a K or V tile
  // chunk (8 dims) of a token's K row
  static __device__ __forceinline__ int k_at(int key, int chunk) {
    return key * D + 8 * (chunk ^ (key & KSWZ));
  }
  // 8 tokens (block u, half h) of dim d: rows of 8 chunks, placed so that both the operand reads
  // (consecutive dims) and the staging writes (every fourth dim) fall on distinct banks
  static __device__ __forceinline__ int v_at(int d, int u, int h) {
    return d * kI8Keys + 8 * ((2 * u + h) ^ ((d & 7) ^ ((d >> 3) & 3)));
  }
};

template <int D>
struct I8PrefillLds {
  static constexpr int NV = D > 128 ? 2 : 3;               // (what fits)
  __align__(16) half_t k[2][I8Tile<D>::HALVES], v[NV][I8Tile<D>::HALVES];
  int n[kI8Kept * kWave], scan[kI8Kept * kWave];           // the walk's kept pairs
  int blk[kI8Window];
  __align__(16) float fk[kI8Window + 4], vs[kI8Window];        // scale * log2 e * ks; log2(vs / vref)
  __align__(16) float back[kI8Window];                     // vref / vs
  bool bad[kI8Window + 4];                                 // a scale is not finite
};

// Rows of one sequence's chunk.
struct I8Chunk {
  int64_t q0, start;                     // its first flat row, that row's position
  int n, kv;                             // rows, tokens in the cache
};

__device__ __forceinline__ I8Chunk i8_chunk(const Int8PrefillArgs& p, int b) {
  const int64_t q0 = p.qsl[b], q1 = p.qsl[b + 1];
  const int len = p.a.seq_lens[b];
  I8Chunk k;
  k.q0 = q0;
  k.n = q0 < 0 || q1 <= q0 || q1 > p.num_tokens ? 0 : (int)(q1 - q0);
  k.kv = i8_kv_len(len, p.a.max_blocks);
  k.start = (int64_t)len - k.n;
  return k;
}

// Tokens that a row of a chunk sees.
__device__ __forceinline__ int i8_sees(const I8Chunk& k, int64_t token) {
  return (int)max((int64_t)0, min((int64_t)k.kv, k.start + token + 1));
}

// Steps of tile t of a chunk: one at least, so that somebody writes the rows.
template <int ROWS>
__device__ __forceinline__ int i8_steps(const I8Chunk& k, int group, int t) {
  const int64_t rows = (int64_t)k.n * group;
  if ((int64_t)t * ROWS >= rows) return 0;
  const int sees = i8_sees(k, (int)(min(rows, (int64_t)(t + 1) * ROWS) - 1) / group);
  return max(1, (sees + kI8Keys - 1) / kI8Keys);
}

// Where the batch's steps lie: pairs (sequence, tile) in order, each with all its KV heads.
struct I8Place {
  int pair, steps;
  int64_t before;                        // steps of the pairs before it, for one KV head
};

// The pairs' steps, a pair a lane: the first kI8Kept * 64 pairs are kept, further ones are worked out
// again where they are asked for. Every wavefront for itself.
template <int ROWS>
struct I8Walk {
  int n[kI8Kept], scan[kI8Kept];         // steps, and their sums from the first lane of the 64
  int64_t total;                         // of all pairs, for one KV head

  static __device__ __forceinline__ int steps(const Int8PrefillArgs& p, int pair) {
    if (pair >= (p.num_seqs - p.first) * p.tiles) return 0;
    return i8_steps<ROWS>(i8_chunk(p, p.first + pair / p.tiles), p.a.group, pair % p.tiles);
  }
  __device__ __forceinline__ I8Walk(const Int8PrefillArgs& p) {
    const int lane = threadIdx.x % kWave, pairs = (p.num_seqs - p.first) * p.tiles;
    total = 0;
#pragma unroll
    for (int i = 0; i < kI8Kept; ++i) {
      n[i] = scan[i] = 0;
      if (i * kWave < pairs) n[i] = steps(p, i * kWave + lane);
    }
#pragma unroll
    for (int i = 0; i < kI8Kept; ++i) {
      if (i * kWave < pairs) scan[i] = i8_scan(n[i]);
      total += __builtin_amdgcn_readlane(scan[i], kWave - 1);
    }
    for (int base = kI8Kept * kWave; base < pairs; base += kWave)
      total += __builtin_amdgcn_readlane(i8_scan(steps(p, base + lane)), kWave - 1);
  }
  // Kept in LDS while a tile needs the registers.
  __device__ __forceinline__ void save(int* ln, int* ls) const {
#pragma unroll
    for (int i = 0; i < kI8Kept; ++i) {
      ln[i * kWave + threadIdx.x % kWave] = n[i];
      ls[i * kWave + threadIdx.x % kWave] = scan[i];
    }
  }
  __device__ __forceinline__ I8Walk(const int* ln, const int* ls) {
#pragma unroll
    for (int i = 0; i < kI8Kept; ++i) {
      n[i] = ln[i * kWave + threadIdx.x % kWave];
      scan[i] = ls[i * kWave + threadIdx.x % kWave];
    }
  }
  static __device__ __forceinline__ bool in(int n, int scan, int base, int64_t sum, int64_t at, I8Place& place) {
    const uint64_t past = __ballot(sum + scan > at);
    if (!past) return false;
    const int i = __ffsll((unsigned long long)past) - 1;
    place.pair = base + i;
    place.steps = __builtin_amdgcn_readlane(n, i);
    place.before = sum + __builtin_amdgcn_readlane(scan, i) - place.steps;
    return true;
  }
  // The pair that step `at` (below total) falls in.
  __device__ __forceinline__ I8Place find(const Int8PrefillArgs& p, int64_t at) const {
    const int lane = threadIdx.x % kWave;
    I8Place place;
    int64_t sum = 0;
#pragma unroll
    for (int i = 0; i < kI8Kept; ++i) {
      if (in(n[i], scan[i], i * kWave, sum, at, place)) return place;
      sum += __builtin_amdgcn_readlane(scan[i], kWave - 1);
    }
    for (int base = kI8Kept * kWave;; base += kWave) {
      const int k = steps(p, base + lane), ks = i8_scan(k);
      if (in(k, ks, base, sum, at, place)) return place;
      sum += __builtin_amdgcn_readlane(ks, kWave - 1);
    }
  }
  // Steps of the pairs before `pair`.
  __device__ __forceinline__ int64_t before(const Int8PrefillArgs& p, int pair) const {
    const int lane = threadIdx.x % kWave;
    int64_t sum = 0;
#pragma unroll
    for (int i = 0; i < kI8Kept; ++i) {
      const int last = pair - 1 - i * kWave;               // lane of the last pair before it
      if (last >= 0) sum += __builtin_amdgcn_readlane(scan[i], min(last, kWave - 1));
    }
    for (int base = kI8Kept * kWave; base < pair; base += kWave) {
      const int scan = i8_scan(steps(p, base + lane));
      sum += __builtin_amdgcn_readlane(scan, min(pair - 1 - base, kWave - 1));
    }
    return sum;
  }
};

// Workgroups that share `total` steps.
__device__ __forceinline__ int64_t i8_shares(int64_t total, int groups) {
  return max((int64_t)1, min((int64_t)groups, total / kI8MinShare));
}

// The codes of a step that one thread widens: units of 16 codes of a K row, and of 4 tokens x 4
// dims of V; 4 D of each in a step. Unit u belongs to block u / D of the step.
template <int D, int THREADS>
struct I8Stage {
  static constexpr int UNITS = 4 * D;
  static constexpr int N = (UNITS + THREADS - 1) / THREADS;
  static constexpr bool ALL = UNITS % THREADS == 0;        // every thread has N units
  uint4_t k[N];
  uint32_t v[N][4];

  static __device__ __forceinline__ int unit(int i) { return threadIdx.x + i * THREADS; }
  static __device__ __forceinline__ int64_t base(const Int8DecodeArgs& a, const I8PrefillLds<D>& lds, int w0,
                                                 int last, int h, int u) {
    return ((int64_t)lds.blk[min(w0 + u / D, last)] * a.kvh + h) * (kBlockSize * D);
  }
  // Requests blocks w0 .. w0 + 3 of the window (the last real one again past the end).
  __device__ __forceinline__ void request_k(const Int8DecodeArgs& a, const I8PrefillLds<D>& lds, int w0,
                                            int last, int h) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (ALL || unit(i) < UNITS)
        k[i] = ld<uint4_t>(a.kc + base(a, lds, w0, last, h, unit(i)) + 16 * (unit(i) % D));
  }
  __device__ __forceinline__ void request_v(const Int8DecodeArgs& a, const I8PrefillLds<D>& lds, int w0,
                                            int last, int h) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (ALL || unit(i) < UNITS) {
        const int in = unit(i) % D;                        // 4 tokens at 4 (in / (D / 4)), 4 dims
        const int8_t* p = a.vc + base(a, lds, w0, last, h, unit(i)) + 4 * (in / (D / 4)) * D + 4 * (in % (D / 4));
#pragma unroll
        for (int r = 0; r < 4; ++r) v[i][r] = ld<uint32_t>(p + r * D);
      }
  }
  __device__ __forceinline__ void place_k(half_t* tile) const {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (ALL || unit(i) < UNITS) {
        const int key = unit(i) / (D / 16), chunk = 2 * (unit(i) % (D / 16));
        st<half8_t>(tile + I8Tile<D>::k_at(key, chunk), codes8(k[i][0], k[i][1]));
        st<half8_t>(tile + I8Tile<D>::k_at(key, chunk + 1), codes8(k[i][2], k[i][3]));
      }
  }
  template <int q>
  static __device__ __forceinline__ void place_column(half_t* tile, const uint32_t (&x)[4], int block,
                                                      int group, int d0) {
    const half2_t a = column2<q>(x[0], x[1]), b = column2<q>(x[2], x[3]);
    st<half4_t>(tile + I8Tile<D>::v_at(d0 + q, block, group & 1) + 4 * (group >> 1),
                half4_t{a[0], a[1], b[0], b[1]});
  }
  __device__ __forceinline__ void place_v(half_t* tile) const {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (ALL || unit(i) < UNITS) {
        uint32_t x[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = v[i][r] ^ 0x80808080u;
        const int in = unit(i) % D, block = unit(i) / D, group = in / (D / 4), d0 = 4 * (in % (D / 4));
        place_column<0>(tile, x, block, group, d0);
        place_column<1>(tile, x, block, group, d0);
        place_column<2>(tile, x, block, group, d0);
        place_column<3>(tile, x, block, group, d0);
      }
  }
};

// The rows of one wavefront: q as MFMA operand, O^T, each lane's reference and partial sum, and the
// operands' places in their tiles.
template <int D>
struct I8Rows {
  static constexpr int DT = (D + 31) / 32;                 // output tiles of 32 dims
  static constexpr int NQ = D / 16, NP = 2 * DT;           // MFMAs of 32 tokens: K . Q^T, V^T . P^T
  static constexpr int ALL = 2 * NQ + 2 * NP, AHEAD = 4;   // of a step; operands requested ahead
  half8_t q[D / 16];
  float16_t o[DT];
  float m, l, alpha;
  bool moved;                                              // alpha has not reached o yet
  int kat[NQ], vat[4];

  // Operand j of a step: V of the last step's last 32 tokens, K of the next step, V of this step's
  // first 32 tokens (block by block, so that consecutive MFMAs add to different tiles).
  __device__ __forceinline__ half8_t operand(const half_t* vp, const half_t* kn, const half_t* vc, int j) const {
    if (j < NP) return ld<half8_t>(vp + vat[2 + j / DT] + (j % DT) * 32 * kI8Keys);
    j -= NP;
    if (j < 2 * NQ) return ld<half8_t>(kn + kat[j % NQ] + (j / NQ) * 32 * D);
    j -= 2 * NQ;
    return ld<half8_t>(vc + vat[j / DT] + (j % DT) * 32 * kI8Keys);
  }
};

// Scores j * 16 / N .. of one 32-token tile to P' (blocks `blk`, `blk` + 1) and the row's sum.
template <int N>
__device__ __forceinline__ void i8_exp(float& l, const float16_t& s, int j, float fk0, float fk1, float off0,
                                       float off1, float back0, float back1, float& sum, half8_t& p0,
                                       half8_t& p1) {
#pragma unroll
  for (int e = j * 16 / N; e < (j + 1) * 16 / N; ++e) {
    const float x = fast_exp2(fmaf(s[e], e < 8 ? fk0 : fk1, e < 8 ? off0 : off1));
    sum = e % 8 == 0 ? x : sum + x;
    if (e < 8) p0[e] = (half_t)x; else p1[e - 8] = (half_t)x;
    if (e % 8 == 7) l = fmaf(sum, e < 8 ? back0 : back1, l);
  }
}

// Keeps a value's computation where it stands: without it the exponentials sink past the MFMAs they
// are meant to run beside, down to the block that uses them.
template <typename T>
__device__ __forceinline__ void i8_pin(T& v) { asm volatile("" : "+v"(v)); }

// One step of a wavefront. Its scores stand in sc (tokens 0-31, 32-63), P' of the last step's
// second half in pr[2], pr[3]; the next step's scores replace them. Four phases, each a run of MFMAs beside a share of the vector work:
//   P'(sc[0])  beside  O += V P' of the last step's second half
//   P'(sc[1])  beside  sc[0] = K . Q^T of the next step
//   staging    beside  sc[1] = K . Q^T of the next step
//   maxima of the next scores  beside  O += V P' of this step's first half
// so that no second set of scores is needed (the registers of two wavefronts a SIMD). The order is
// pinned, MFMA by MFMA: left to itself the compiler sets MFMAs and exponentials one after the other.
// Returns the row's largest next score.
template <int D, typename Mask, typename Work>
__device__ __forceinline__ float i8_step64(I8Rows<D>& w, const half_t* vp, const half_t* kn, const half_t* vc,
                                           float16_t (&sc)[2], half8_t (&pr)[4], const float* fkp,
                                           const float* fvp, const float* backp, Mask mask, Work work) {
  typedef I8Rows<D> R;
  constexpr int NQ = R::NQ, NP = R::NP, AHEAD = R::AHEAD;
  half8_t op[AHEAD];
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) op[j] = w.operand(vp, kn, vc, j);
  auto next = [&](int j) {                                 // operand j, and the request of a later one
    const half8_t x = op[j % AHEAD];
    if (j + AHEAD < R::ALL) op[j % AHEAD] = w.operand(vp, kn, vc, j + AHEAD);
    return x;
  };
  const float4_t fk = ld<float4_t>(fkp), fv = ld<float4_t>(fvp), back = ld<float4_t>(backp);
  const float neg = w.m == -INFINITY ? 0.f : -w.m;
  const float off0 = neg + fv[0], off1 = neg + fv[1], off2 = neg + fv[2], off3 = neg + fv[3];
  float sum;
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    w.o[j % R::DT] = mfma_i8(next(j), pr[2 + j / R::DT], w.o[j % R::DT]);
    i8_exp<NP>(w.l, sc[0], j, fk[0], fk[1], off0, off1, back[0], back[1], sum, pr[0], pr[1]);
    if (j == NP - 1) i8_pin(pr[0]), i8_pin(pr[1]), i8_pin(w.l);
    __builtin_amdgcn_sched_barrier(0);
  }
  if (w.moved) {
#pragma unroll
    for (int i = 0; i < R::DT; ++i) w.o[i] *= w.alpha;
  }
  if constexpr (I8PrefillLds<D>::NV == 2) __syncthreads();  // V of the last step is staged over
  float16_t zero;
#pragma unroll
  for (int i = 0; i < 16; ++i) zero[i] = 0.f;
#pragma unroll
  for (int j = 0; j < NQ; ++j) {
    sc[0] = mfma_i8(next(NP + j), w.q[j], j == 0 ? zero : sc[0]);
    i8_exp<NQ>(w.l, sc[1], j, fk[2], fk[3], off2, off3, back[2], back[3], sum, pr[2], pr[3]);
    if (j == NQ - 1) i8_pin(pr[2]), i8_pin(pr[3]), i8_pin(w.l);
    __builtin_amdgcn_sched_barrier(0);
  }
#pragma unroll
  for (int j = 0; j < NQ; ++j) {
    sc[1] = mfma_i8(next(NP + NQ + j), w.q[j], j == 0 ? zero : sc[1]);
    if (j == 0) work(0);
    if (j == NQ / 2) work(1);
    __builtin_amdgcn_sched_barrier(0);
  }
  mask(sc);
  float top[4];
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    w.o[j % R::DT] = mfma_i8(next(NP + 2 * NQ + j), pr[j / R::DT], w.o[j % R::DT]);
#pragma unroll
    for (int e = j * 32 / NP; e < (j + 1) * 32 / NP; ++e)
      top[e / 8] = e % 8 == 0 ? sc[e / 16][e % 16] : vmax(top[e / 8], sc[e / 16][e % 16]);
    __builtin_amdgcn_sched_barrier(0);
  }
  const float4_t fkn = ld<float4_t>(fkp + 4);
  return vmax(vmax(top[0] * fkn[0], top[1] * fkn[1]), vmax(top[2] * fkn[2], top[3] * fkn[3]));
}

// A row's largest score moves its reference; O follows in the next step, behind what was computed
// against the old one.
template <int D>
__device__ __forceinline__ void i8_reference(I8Rows<D>& w, float best) {
  const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(best), __float_as_uint(best), false, false);
  best = vmax(__uint_as_float(both[0]), __uint_as_float(both[1]));
  const bool move = !(best <= w.m + kI8Rescale);           // NaN moves it too
  w.moved = __ballot(move) != 0;
  if (w.moved) {
    w.alpha = move ? fast_exp2(w.m - best) : 1.f;
    w.l *= w.alpha;
    w.m = move ? best : w.m;
  }
}

// One tile's steps [s0, s1) by the workgroup.
template <int D, int WAVES>
__device__ __forceinline__ void i8_piece(const Int8PrefillArgs& p, I8PrefillLds<D>& lds, const I8Chunk& k,
                                         int b, int tile, int h, int s0, int s1, bool whole, int64_t slot) {
  constexpr int THREADS = WAVES * kWave, ROWS = 32 * WAVES;
  constexpr int DT = (D + 31) / 32;                        // output tiles of 32 dims
  const Int8DecodeArgs& a = p.a;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave, c = lane % 32, hh = lane / 32;
  const int64_t rows = (int64_t)k.n * a.group, wrow = (int64_t)tile * ROWS + 32 * wave, row = wrow + c;
  const bool real = row < rows;
  const int token = real ? (int)row / a.group : 0;
  const int head = h * a.group + (real ? (int)row % a.group : 0);
  const int vis = real ? i8_sees(k, token) : 0;
  // rows ascend in tokens: the wavefront's first row sees least
  const int least = wrow < rows ? i8_sees(k, (int)wrow / a.group) : 0;
  const int sees = i8_sees(k, (int)(min(rows, (int64_t)(tile + 1) * ROWS) - 1) / a.group);
  const int nb = (sees + kBlockSize - 1) / kBlockSize;     // blocks that the tile sees

  I8Rows<D> w;
  const half_t* qrow = a.q + (k.q0 + token) * a.q_st + (int64_t)head * a.q_sh;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    w.q[i] = ld<half8_t>(qrow + 16 * i + 8 * hh);
    w.kat[i] = I8Tile<D>::k_at(c, 2 * i + hh);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) w.vat[i] = I8Tile<D>::v_at(D < 32 ? c % D : c, i, hh);
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) w.o[t][i] = 0.f;
  w.m = -INFINITY, w.l = 0.f, w.alpha = 1.f, w.moved = false;
  float vref = 0.f;

  I8Stage<D, THREADS> stage;
  s1 = min(s1, (nb + kI8StepBlocks - 1) / kI8StepBlocks);  // (nothing visible: no step)
  for (int w0 = s0; w0 < s1; w0 += kI8Window / kI8StepBlocks) {
    // a window of the sequence's blocks: ids, scales
    const int n = min(s1 - w0, kI8Window / kI8StepBlocks);
    const int blocks = min(nb - w0 * kI8StepBlocks, n * kI8StepBlocks), last = blocks - 1;
    __syncthreads();                                       // the last window's and piece's reads
    constexpr int PER = (kI8Window + THREADS - 1) / THREADS;
    int blk[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = threadIdx.x + i * THREADS;
      blk[i] = at < blocks ? clamp_block(a.block_tables[b * a.bt_stride + w0 * kI8StepBlocks + at], a.num_blocks) : 0;
      if (at < kI8Window) lds.blk[at] = blk[i];
    }
    __syncthreads();
    float ks[PER], vs[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const bool there = threadIdx.x + i * THREADS < blocks;
      ks[i] = there ? a.ks[(int64_t)blk[i] * a.kvh + h] : 0.f;
      vs[i] = there ? a.vs[(int64_t)blk[i] * a.kvh + h] : 0.f;
    }
    I8Stage<D, THREADS> early;                             // K of the window's second step
    stage.request_k(a, lds, 0, last, h);
    early.request_k(a, lds, kI8StepBlocks, last, h);
    stage.request_v(a, lds, 0, last, h);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = threadIdx.x + i * THREADS;
      i8_poison(ks[i], vs[i]);
      // A K factor of 0 or NaN would leave hidden tokens (-inf) NaN: scores of a factor as small as
      // the least one are 0, and those of blocks without finite scales become NaN in the mask.
      const float f = ks[i] * a.sl2;
      if (at < kI8Window) {
        lds.fk[at] = f > kI8LeastFactor ? f : kI8LeastFactor;
        lds.vs[at] = vs[i];
        lds.bad[at] = f != f;
      }
    }
    __syncthreads();
    float top = 0.f;
    bool some = false;
#pragma unroll
    for (int i = 0; i < kI8Window; i += kWave) {
      top = fmaxf(top, lds.vs[i + lane]);
      some = some || lds.bad[i + lane];
    }
    top = i8_most(top);
    const bool bad = __ballot(some) != 0;
    if (top > vref) {
      const float f = vref / top;
      vref = top;
#pragma unroll
      for (int t = 0; t < DT; ++t) w.o[t] *= f;
    }
    __syncthreads();                                       // every wavefront has the maximum
    for (int i = threadIdx.x; i < kI8Window; i += THREADS) {
      const float f = vref > 0.f ? fmaxf(__builtin_amdgcn_logf(lds.vs[i] / vref), kI8LeastRatio) : 0.f;
      lds.vs[i] = f;
      lds.back[i] = fast_exp2(-f);
    }
    stage.place_k(lds.k[0]);
    early.place_k(lds.k[1]);
    stage.place_v(lds.v[0]);
    __syncthreads();

    // Step i reads K of step i + 1 in k[(i + 1) % 2] and V of steps i - 1 and i in two of three
    // tiles; meanwhile K of step i + 2 and V of step i + 1 go to tiles whose last readers were in
    // step i - 1.
    auto mask = [&](float16_t (&x)[2], int step) {
      if (bad || (step + 1) * kI8Keys > least) {
        const int key0 = step * kI8Keys + 4 * hh;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            x[kt][i] = key0 + 32 * kt + 8 * (i / 4) + i % 4 < vis ? x[kt][i] : -INFINITY;
        if (bad)
#pragma unroll
          for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (lds.bad[(step - w0) * kI8StepBlocks + 2 * kt + i / 8] && x[kt][i] != -INFINITY)
                x[kt][i] = __builtin_nanf("");
      }
    };
    float16_t sc[2];
    half8_t pr[4];
    {
      constexpr int NQ = I8Rows<D>::NQ;
      float16_t zero;
#pragma unroll
      for (int i = 0; i < 16; ++i) zero[i] = 0.f;
#pragma unroll
      for (int j = 0; j < 2 * NQ; ++j)
        sc[j / NQ] = mfma_i8(ld<half8_t>(lds.k[0] + w.kat[j % NQ] + j / NQ * 32 * D), w.q[j % NQ],
                             j % NQ == 0 ? zero : sc[j / NQ]);
      mask(sc, w0);
      const float4_t fk = ld<float4_t>(lds.fk);
      float t[4];
#pragma unroll
      for (int e = 0; e < 32; ++e) t[e / 8] = e % 8 == 0 ? sc[e / 16][e % 16] : vmax(t[e / 8], sc[e / 16][e % 16]);
      i8_reference<D>(w, vmax(vmax(t[0] * fk[0], t[1] * fk[1]), vmax(t[2] * fk[2], t[3] * fk[3])));
      // no step before the first: its P' is 0, beside finite codes
#pragma unroll
      for (int e = 0; e < 8; ++e) pr[2][e] = pr[3][e] = (half_t)0.f;
    }
    // The loop has no branch but the mask's and the reference's: past the window's end the last
    // blocks are staged again, and the scores of the step behind it are computed and not used.
    constexpr int NV = I8PrefillLds<D>::NV;
    int v0 = 0, v1 = 1, v2 = NV - 1;                       // V of this step, the next, the last one
    for (int i = 0; i < n; ++i) {
      stage.request_k(a, lds, (i + 2) * kI8StepBlocks, last, h);
      stage.request_v(a, lds, (i + 1) * kI8StepBlocks, last, h);
      auto work = [&](int part) {
        if (part == 0) stage.place_k(lds.k[i & 1]); else stage.place_v(lds.v[v1]);
      };
      auto masked = [&](float16_t (&x)[2]) { mask(x, w0 + i + 1); };
      const int wb = i * kI8StepBlocks;
      const float best = i8_step64<D>(w, lds.v[i == 0 ? v0 : v2], lds.k[(i + 1) & 1], lds.v[v0], sc, pr,
                                      lds.fk + wb, lds.vs + wb, lds.back + wb, masked, work);
      i8_reference<D>(w, i + 1 < n ? best : w.m);          // (its own reference moves none, also a NaN)
      __syncthreads();
      const int v = v2;
      v2 = v0, v0 = v1, v1 = NV == 2 ? v2 : v;
    }
#pragma unroll
    for (int j = 0; j < I8Rows<D>::NP; ++j)                // the last step's second half
      w.o[j % DT] = mfma_i8(ld<half8_t>(lds.v[v2] + w.vat[2 + j / DT] + j % DT * 32 * kI8Keys), pr[2 + j / DT],
                            w.o[j % DT]);
  }

  // lanes c and c + 32 hold the two halves of row c's sum
  const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(w.l), __float_as_uint(w.l), false, false);
  const float l = __uint_as_float(both[0]) + __uint_as_float(both[1]);
  if (!real) return;
  if (whole) {
    const float f = l == 0.f ? 0.f : vref / l;             // nothing visible: zeros
    half_t* dst = a.out + (k.q0 + token) * a.out_st + (int64_t)head * D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int d = 32 * dt + 8 * (i / 4) + 4 * hh;
        if (D < 32 && d >= D) break;
        st<half4_t>(dst + d, to_half4(float4_t{w.o[dt][i], w.o[dt][i + 1], w.o[dt][i + 2], w.o[dt][i + 3]} * f));
      }
  } else {
    const int64_t at = slot * ROWS + 32 * wave + c;
    if (hh == 0) st<float2_t>(a.part_ml + 2 * at, float2_t{w.m, l});
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int d = 32 * dt + 8 * (i / 4) + 4 * hh;
        if (D < 32 && d >= D) break;
        st<float4_t>(a.part_o + at * D + d,
                     float4_t{w.o[dt][i], w.o[dt][i + 1], w.o[dt][i + 2], w.o[dt][i + 3]} * vref);
      }
  }
}

template <int D, int WAVES>
__global__ void __launch_bounds__(WAVES* kWave, D >= 256 ? 1 : 2) prefill_int8_kernel(Int8PrefillArgs p) {
  constexpr int ROWS = 32 * WAVES;
  __shared__ __align__(16) I8PrefillLds<D> lds;
  const Int8DecodeArgs& a = p.a;
  int64_t at, hi;
  {
    const I8Walk<ROWS> walk(p);
    const int64_t total = walk.total * a.kvh, shares = i8_shares(total, p.groups);
    if (blockIdx.x >= shares || total == 0) return;
    at = total * blockIdx.x / shares, hi = total * (blockIdx.x + 1) / shares;
    if (threadIdx.x < kWave) walk.save(lds.n, lds.scan);
    __syncthreads();
  }
  int b = 0, h = 0, tile = 0;
  for (bool extra = false; extra || at < hi;) {
    int s0 = 0, s1, steps;
    if (!extra) {
      const I8Place place = I8Walk<ROWS>(lds.n, lds.scan).find(p, at / a.kvh);
      const int64_t in = at - place.before * a.kvh;
      steps = place.steps;
      h = (int)(in / steps), s0 = (int)(in % steps);
      s1 = (int)min((int64_t)steps, s0 + (hi - at));
      b = p.first + place.pair / p.tiles, tile = place.pair % p.tiles;
      at += s1 - s0;
    }
    const I8Chunk k = i8_chunk(p, b);
    if (extra) s1 = steps = i8_steps<ROWS>(k, a.group, tile);
    i8_piece<D, WAVES>(p, lds, k, b, tile, h, s0, s1, s0 == 0 && s1 == steps,
                       2 * (int64_t)blockIdx.x + (s0 == 0));
    // Tiles past the host's bound on the rows follow, whole, the first step of the last tile that it
    // allows for.
    extra = (extra || (tile == p.tiles - 1 && s0 == 0)) && i8_steps<ROWS>(k, a.group, tile + 1) > 0;
    if (extra) ++tile;
  }
}

// Tiles that several workgroups share: D / 4 threads a row, 32 rows a workgroup.
constexpr int kI8MergeRows = 32;
template <int D, int ROWS>
__global__ void __launch_bounds__(256) prefill_int8_merge_kernel(Int8PrefillArgs p) {
  constexpr int PER = 256 / (D / 4), N = 4;                // rows at a time, partials requested at once
  const Int8DecodeArgs& a = p.a;
  const int64_t unit = blockIdx.x / (ROWS / kI8MergeRows);
  const int row0 = (int)(blockIdx.x % (ROWS / kI8MergeRows)) * kI8MergeRows;
  const int h = (int)(unit % a.kvh), pair = (int)(unit / a.kvh);
  const int b = p.first + pair / p.tiles, tile = pair % p.tiles;
  const I8Chunk k = i8_chunk(p, b);
  const int64_t rows = (int64_t)k.n * a.group;
  if ((int64_t)tile * ROWS + row0 >= rows) return;
  const I8Walk<ROWS> walk(p);
  const int steps = i8_steps<ROWS>(k, a.group, tile);
  const int64_t total = walk.total * a.kvh, shares = i8_shares(total, p.groups);
  const int64_t g0 = walk.before(p, pair) * a.kvh + (int64_t)h * steps, g1 = g0 + steps;
  // share w begins at total * w / shares: the last one that begins at or before a step
  const int64_t first = ((g0 + 1) * shares - 1) / total, last = (g1 * shares - 1) / total;
  if (first == last) return;                               // one workgroup wrote it
  const int d = threadIdx.x % (D / 4) * 4;
  for (int in = row0 + threadIdx.x / (D / 4); in < row0 + kI8MergeRows; in += PER) {
    const int64_t row = (int64_t)tile * ROWS + in;
    if (row >= rows) return;
    float top = -INFINITY, sum = 0.f;
    float4_t o = {0.f, 0.f, 0.f, 0.f};
    for (int64_t i0 = first; i0 <= last; i0 += N) {
      float2_t ml[N];
      float4_t x[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int64_t at = (2 * min(i0 + i, last) + (i0 + i == first)) * ROWS + in;
        ml[i] = ld<float2_t>(a.part_ml + 2 * at);
        x[i] = ld<float4_t>(a.part_o + at * D + d);
      }
      float now = top;
#pragma unroll
      for (int i = 0; i < N; ++i) now = i0 + i <= last ? vmax(now, ml[i][0]) : now;
      const float f = top == -INFINITY ? 0.f : fast_exp2(top - now);
      sum *= f;
      o *= f;
      top = now;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (i0 + i > last || ml[i][0] == -INFINITY) continue;
        const float g = fast_exp2(ml[i][0] - top);
        sum = fmaf(g, ml[i][1], sum);
        o += x[i] * g;
      }
    }
    const float f = sum == 0.f ? 0.f : 1.f / sum;
    const int token = (int)row / a.group, head = h * a.group + (int)row % a.group;
    st<half4_t>(a.out + (k.q0 + token) * a.out_st + (int64_t)head * D + d, to_half4(o * f));
  }
}

}  // namespace ts
