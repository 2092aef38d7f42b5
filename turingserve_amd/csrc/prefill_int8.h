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
// A block's K scale multiplies its scores in fp32. Its V scale goes into the exponent, and the row's
// reference is the largest of both together among the tokens that it sees (decode_int8.h):
// P' = 2^(s + log2 vs - m) is what is rounded to fp16 and multiplied by the codes of V, and a row's sum
// adds each block's P' divided by vs.
//
// Lane l is split into c = l % 32 and h = l / 32: a result lane holds S^T[8 (i / 4) + 4 h + i % 4][c],
// i = 0..15, so a lane's scores all belong to row c, and its P values for a block's 16 tokens (i % 8
// of one half) are the B operand of the P.V step as they stand when V^T lies in LDS with the
// tokens of a block in the order {0-3, 8-11 | 4-7, 12-15}.
//
// The batch's steps (of every sequence, tile and KV head, in that order) are shared evenly over
// the launched workgroups. Where a share begins or ends inside a tile, its part of the tile is left
// as a partial (m, l, O in fp32) for the merge launch; a workgroup leaves two at most. Every
// workgroup works the shares out for itself from the sequences' lengths, a sequence a lane: the steps
// of a sequence's first t tiles have a closed form, so a batch of one long and many short prompts
// costs what its rows cost.
//
// 2048 rows on 4096 cached, 12/2 heads of 128: 84 to 87 us and 9.5 for the merge, 64.4 GFLOP: 690
// TFLOP/s where a large matrix product reaches 1210. A step of 64 tokens takes eight wavefronts some 3700
// cycles, of which the MFMAs are 2050; exponentials, operand reads, staging and requests are worth 10 to
// 14 % each when taken out, so it is the issue of all of them together that bounds it. 64 rows a
// wavefront (four of them) read half the operands and took 115 us: the registers moved through AGPRs.
// (Three registers are spilled at head_dim 128: stored once a workgroup, read once a tile's piece.)
#pragma once

#include "decode_int8.h"

namespace ts {

typedef float float16_t __attribute__((ext_vector_type(16)));

constexpr int kI8Keys = 64;              // tokens of a step
constexpr int kI8StepBlocks = kI8Keys / kBlockSize;
constexpr int kI8Window = 256;           // blocks whose ids and scales are held in LDS at a time
// Steps (and tiles' costs) that a workgroup is worth: 31.0, 30.6 and 31.1 us with 4, 6 and 8 at five
// chunks of 90 to 1100 rows, 14/2 heads of 64.
constexpr int kI8MinShare = 6;
constexpr float kI8LeastFactor = 1e-30f;

template <int N>
struct I8Const {
  static constexpr int value = N;
};

// What the merge launch does about the beginning of a share (left by the share's workgroup, so that
// the merge need not look the tile up): the tile's rows and the shares that its partials come from,
// where it is the first one inside the tile.
struct I8Joint {
  int first, last;                       // equal: nothing
  int q0, rows, row0, h;                 // the chunk's first flat row and rows per KV head, the tile's first
  int pad[2];
};

struct Int8PrefillArgs {
  Int8DecodeArgs a;                      // (part_o, part_ml: two partials of a tile per workgroup)
  I8Joint* joints;                       // one for each workgroup
  int num_seqs, first;                   // sequences first .. num_seqs - 1
  int groups;                            // workgroups of the main launch
  int rate;                              // i8_rate
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
  __align__(16) half_t k[2][I8Tile<D>::HALVES], v[2][I8Tile<D>::HALVES];
  int walk[5][kWave];                                      // I8Walk
  int blk[kI8Window];                                      // the sign bit: a scale is not finite
  __align__(16) float fk[kI8Window + 4], lv[kI8Window + 4];    // scale * log2 e * ks; log2 vs
  __align__(16) float back[kI8Window];                     // 1 / vs
};

// Rows of one sequence's chunk. (The entry point refuses batches whose rows times heads or steps
// pass 31 bits.)
struct I8Chunk {
  int q0, start;                         // its first flat row, that row's position
  int n, kv;                             // rows, tokens in the cache
};

__device__ __forceinline__ I8Chunk i8_chunk(const Int8PrefillArgs& p, int b) {
  const int q0 = p.a.qsl[b], q1 = p.a.qsl[b + 1], len = p.a.seq_lens[b];
  I8Chunk k;
  k.q0 = q0;
  k.n = q0 < 0 || q1 <= q0 || q1 > p.a.num_tokens ? 0 : q1 - q0;
  k.kv = i8_kv_len(len, p.a.max_blocks);
  k.start = max(len, 0) - k.n;
  return k;
}

// Tokens that a row of a chunk sees.
__device__ __forceinline__ int i8_sees(const I8Chunk& k, int token) {
  return max(0, min(k.kv, k.start + token + 1));
}

// The steps of a tile that sees `sees` tokens (one at least, so that somebody writes its rows).
template <int ROWS>
__device__ __forceinline__ int i8_steps(const Int8DecodeArgs& a, const I8Chunk& k, int t) {
  const int sees = i8_sees(k, a.by_group(min(k.n * a.group, (t + 1) * ROWS) - 1));
  return max(1, (sees + kI8Keys - 1) / kI8Keys);
}

// What a tile counts for: kI8TileCost for its start (the sequence's lookup, q, the first blocks' ids,
// scales and codes, one after the other: 11 to 15 thousand cycles beside 2.8 thousand a step at
// head_dim 64), then its steps, then what makes the sum over a sequence's first t tiles
//   C(t) = t (kI8TileCost + 2) + floor((t start + t (t + 1) / 2 ROWS / group) / 64):
// C(t + 1) - C(t) > kI8TileCost + 1 + (start + (t + 1) ROWS / group) / 64, and tile t sees at most
// start + ((t + 1) ROWS - 1) / group + 1 tokens, whose steps are fewer than the sum's last two terms.
// Steps of a share that fall on a tile's start or behind its last one are nobody's. (At
// 2048 rows on 4096 cached, 12/2 heads of 128, and five chunks of 90 to 1100, 14/2 heads of 64: 93.5 and
// 30.3 us with kI8TileCost 3, 93.0 and 30.6 with 5, 94.3 and 31.0 with 7; 100.4 and 36.1 with 1, when those
// with 5 were 97.8 and 36.3.)
constexpr int kI8TileCost = 5;
// ROWS / (2 group) of a step's 64 tokens in units of 2^-12, rounded up.
constexpr int i8_rate(int rows, int group) { return (32 * rows + group - 1) / group; }

__device__ __forceinline__ int i8_cost(const Int8PrefillArgs& p, int start, int t) {
  const int64_t sees = (int64_t)t * ((int64_t)start << 6) + (int64_t)t * (t + 1) * p.rate;
  return t * (kI8TileCost + 2) + (int)(sees >> 12);
}

// Where the batch's steps lie: tiles in order, each with all its KV heads.
struct I8Place {
  I8Chunk k;
  int seq, tile, cost;
  int before;                            // what the tiles before it count for, for one KV head
};

// The sequences' costs, a sequence a lane: the first 64 are kept, further ones are worked out again
// where they are asked for. Every wavefront for itself.
template <int ROWS>
struct I8Walk {
  I8Chunk k;
  int scan;                              // sums of the costs from the first lane of the 64
  int total;                             // of all sequences, for one KV head

  static __device__ __forceinline__ int tiles(const Int8PrefillArgs& p, int n) {
    return (n * p.a.group + ROWS - 1) / ROWS;
  }
  static __device__ __forceinline__ int start(const I8Chunk& k) { return max(0, min(k.start, k.kv)); }
  // This lane's sequence of those from `first` on.
  static __device__ __forceinline__ int cost(const Int8PrefillArgs& p, int first, I8Chunk& k) {
    const int b = first + threadIdx.x % kWave;
    k = {};
    if (b < p.num_seqs) k = i8_chunk(p, b);
    return i8_cost(p, start(k), tiles(p, k.n));
  }
  __device__ __forceinline__ I8Walk(const Int8PrefillArgs& p) {
    scan = i8_scan(cost(p, p.first, k));
    total = __builtin_amdgcn_readlane(scan, kWave - 1);
    I8Chunk x;
    for (int first = p.first + kWave; first < p.num_seqs; first += kWave)
      total += __builtin_amdgcn_readlane(i8_scan(cost(p, first, x)), kWave - 1);
  }
  // Kept in LDS while a tile needs the registers.
  __device__ __forceinline__ void save(int (*to)[kWave]) const {
    const int lane = threadIdx.x % kWave;
    to[0][lane] = k.q0, to[1][lane] = k.start, to[2][lane] = k.n, to[3][lane] = k.kv, to[4][lane] = scan;
  }
  __device__ __forceinline__ I8Walk(const int (*from)[kWave]) {
    const int lane = threadIdx.x % kWave;
    k.q0 = from[0][lane], k.start = from[1][lane], k.n = from[2][lane], k.kv = from[3][lane];
    scan = from[4][lane];
  }
  // The tile that step `at` (below total) falls in. False where there is none, as only lengths that
  // contradict themselves could have it; a tile that is found is one of its sequence's.
  __device__ __forceinline__ bool find(const Int8PrefillArgs& p, int at, I8Place& place) const {
    const int lane = threadIdx.x % kWave;
    I8Chunk x = k;
    int sums = scan, sum = 0, first = p.first;
    uint64_t past;
    while ((past = __ballot(sum + sums > at)) == 0) {
      sum += __builtin_amdgcn_readlane(sums, kWave - 1);
      first += kWave;
      if (first >= p.num_seqs) return false;
      sums = i8_scan(cost(p, first, x));
    }
    const int i = __ffsll((unsigned long long)past) - 1;
    place.k = {__builtin_amdgcn_readlane(x.q0, i), __builtin_amdgcn_readlane(x.start, i),
               __builtin_amdgcn_readlane(x.n, i), __builtin_amdgcn_readlane(x.kv, i)};
    place.seq = first + i;
    if (i > 0) sum += __builtin_amdgcn_readlane(sums, i - 1);
    // the last tile whose steps start at or before it: 64 candidates at a time
    const int from = start(place.k);
    int tile = 0;
    for (int span = tiles(p, place.k.n); span > 1;) {
      const int stride = (span + kWave - 1) / kWave, t = lane * stride;
      const uint64_t behind = __ballot(t < span && sum + i8_cost(p, from, tile + t) <= at);
      const int last = (63 - __clzll((long long)(behind | 1))) * stride;
      tile += last;
      span = min(stride, span - last);
    }
    place.tile = tile;
    const int cost = i8_cost(p, from, tile);
    place.before = sum + cost;
    place.cost = i8_cost(p, from, tile + 1) - cost;
    return place.k.n > 0;
  }
};

// `total` steps shared over workgroups: share w is [begin(w), begin(w + 1)), the first `more` of
// them one step longer.
struct I8Shares {
  int count, each, more;
  __device__ __forceinline__ I8Shares(int total, int groups) {
    count = max(1, min(groups, total / kI8MinShare));
    each = (int)((unsigned)total / (unsigned)count);
    more = total - each * count;
  }
  __device__ __forceinline__ int begin(int w) const { return w * each + min(w, more); }
  __device__ __forceinline__ int of(int step) const {      // the share that a step belongs to
    const int longer = more * (each + 1);
    return step < longer ? (int)((unsigned)step / (unsigned)(each + 1))
                         : more + (int)((unsigned)(step - longer) / (unsigned)each);
  }
};

// The codes of a step that one thread widens: units of 16 codes of a K row, and of 4 tokens x 4
// dims of V; 4 D of each in a step. Unit u belongs to block u / D of the step.
template <int D, int THREADS>
struct I8Stage {
  static constexpr int UNITS = 4 * D;
  static constexpr int N = (UNITS + THREADS - 1) / THREADS;
  static constexpr bool ALL = UNITS % THREADS == 0;        // every thread has N units
  static constexpr bool UNIFORM = D >= kWave;              // a wavefront's unit lies in one block
  uint4_t k[N];
  uint32_t v[N][4];
  half2_t off[N];                                          // what the codes of K are off by

  static __device__ __forceinline__ int unit(int i) { return threadIdx.x + i * THREADS; }
  // The ids of blocks w0 .. w0 + 3 of the window (the last real one again past the end).
  static __device__ __forceinline__ void ids(const I8PrefillLds<D>& lds, int w0, int last, int (&id)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) id[i] = lds.blk[min(w0 + min(unit(i), UNITS - 1) / D, last)];
  }
  static __device__ __forceinline__ int64_t base(const Int8DecodeArgs& a, int id, int h) {
    int blk = id & 0x7fffffff;
    if (UNIFORM) blk = __builtin_amdgcn_readfirstlane(blk);
    return ((int64_t)blk * a.kvh + h) * (kBlockSize * D);
  }
  __device__ __forceinline__ void request_k(const Int8DecodeArgs& a, const int (&id)[N], int h) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (ALL || unit(i) < UNITS) {
        k[i] = ld<uint4_t>(a.kc + base(a, id[i], h) + 16 * (unit(i) % D));
      }
    finite(id);
  }
  // Ids of a step's blocks from the table itself, and, once the scales are known, their finite ones.
  static __device__ __forceinline__ void ids(const Int8DecodeArgs& a, const int32_t* table, int last,
                                             int (&id)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      int at = min(unit(i), UNITS - 1) / D;
      if (UNIFORM) at = __builtin_amdgcn_readfirstlane(at);
      id[i] = clamp_block(table_entry(table + min(at, last)), a.num_blocks);
    }
  }
  __device__ __forceinline__ void finite(const int (&id)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const half_t o = id[i] < 0 ? (half_t)__builtin_nanf("") : (half_t)1152.f;
      off[i] = {o, o};
    }
  }
  // Row r of the 4 tokens (one at a time, so that they stand between other work).
  __device__ __forceinline__ void request_v(const Int8DecodeArgs& a, const int (&id)[N], int h, int r) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (ALL || unit(i) < UNITS) {
        const int in = unit(i) % D;                        // 4 tokens at 4 (in / (D / 4)), 4 dims
        const int8_t* p = a.vc + base(a, id[i], h) + (4 * (in / (D / 4)) * D + 4 * (in % (D / 4)));
        v[i][r] = ld<uint32_t>(p + r * D);
      }
  }
  __device__ __forceinline__ void place_k(half_t* tile) const {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (ALL || unit(i) < UNITS) {
        const int key = unit(i) / (D / 16), chunk = 2 * (unit(i) % (D / 16));
        st<half8_t>(tile + I8Tile<D>::k_at(key, chunk), codes8(k[i][0], k[i][1], off[i]));
        st<half8_t>(tile + I8Tile<D>::k_at(key, chunk + 1), codes8(k[i][2], k[i][3], off[i]));
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

// The 32 rows of one wavefront: q as MFMA operand, O^T, each lane's reference and partial sum, and
// the operands' places in LDS.
template <int D>
struct I8Rows {
  static constexpr int DT = (D + 31) / 32;                 // output tiles of 32 dims
  static constexpr int NQ = D / 16, NP = 2 * DT;           // operands of 32 tokens: K, V^T
  static constexpr int ALL = 2 * NQ + 2 * NP, AHEAD = 4;   // of a step; requested ahead
  half8_t q[NQ];
  float16_t o[DT];
  float m, l, alpha;
  bool moved;                                              // alpha has not reached o yet
  int kat, vat[4];                                         // (chunks of a K row: kat ^ 16 i)

  // Operand j of a step: V of the last step's last 32 tokens, K of the next step, V of this step's
  // first 32 tokens (block by block, so that consecutive MFMAs add to different tiles).
  __device__ __forceinline__ half8_t operand(const half_t* vp, const half_t* kn, const half_t* vc, int j) const {
    if (j < NP) return ld<half8_t>(vp + vat[2 + j / DT] + (j % DT) * 32 * kI8Keys);
    j -= NP;
    if (j < 2 * NQ) return ld<half8_t>(kn + (kat ^ 16 * (j % NQ)) + (j / NQ) * 32 * D);
    j -= 2 * NQ;
    return ld<half8_t>(vc + vat[j / DT] + (j % DT) * 32 * kI8Keys);
  }
};

// Keeps a value's computation where it stands: without it the exponentials sink past the MFMAs they
// are meant to run beside, down to the block that uses them.
template <typename T>
__device__ __forceinline__ void i8_pin(T& v) { asm volatile("" : "+v"(v)); }

// The exponentials of a step's 32 scores per lane, a few at a time: P' in fp16 and the row's sum. In
// call j of N, the products of the j-th share are formed, the exponentials of the share before it
// taken, and the share before that summed and rounded, so that nothing waits for the result in
// front of it. Calls N and N + 1 finish.
struct I8Exp {
  float t[32], x[32], sum[4][2];
  template <int N>
  __device__ __forceinline__ void share(int j, const float16_t (&s)[2], const float4_t& fk, const float (&off)[4],
                                        const float4_t& back, float& l, half8_t (&p)[4]) {
    constexpr int PER = 32 / N;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = (j - 2) * PER + i, b = e / 8;          // summed
      if (e < 0 || e >= 32) continue;
      sum[b][e % 2] = e % 8 < 2 ? x[e] : sum[b][e % 2] + x[e];
      i8_pin(sum[b][e % 2]);
      p[b][e % 8] = (half_t)x[e];
      if (e % 8 == 7) {
        l = fmaf(sum[b][0] + sum[b][1], back[b], l);
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
      if (e < 32) t[e] = fmaf(s[e / 16][e % 16], fk[e / 8], off[e / 8]), i8_pin(t[e]);
    }
  }
};

// A row's largest s + log2 vs from its largest score in each of four blocks.
__device__ __forceinline__ float i8_best(const float (&top)[4], const float4_t& fk, const float4_t& lv) {
  return vmax(vmax(fmaf(top[0], fk[0], lv[0]), fmaf(top[1], fk[1], lv[1])),
              vmax(fmaf(top[2], fk[2], lv[2]), fmaf(top[3], fk[3], lv[3])));
}

// Before the first step of a window: its scores, and the staging that a step does, without a barrier of
// its own: K of that step (and the V codes of 0 before it) stand behind the one that ends the window's
// set-up, and what is staged here, over neither, is read behind the first step's.
template <int D, typename Mask, typename Work>
__device__ __forceinline__ float i8_first(I8Rows<D>& w, const half_t* kn, float16_t (&sc)[2], const float* fknp,
                                          const float* lvnp, Mask mask, Work work) {
  typedef I8Rows<D> R;
  work(0);
#pragma unroll
  for (int v = 3; v < 7; ++v) work(v);
  float16_t zero;
#pragma unroll
  for (int i = 0; i < 16; ++i) zero[i] = 0.f;
#pragma unroll
  for (int j = 0; j < 2 * R::NQ; ++j)
    sc[j / R::NQ] = mfma_i8(w.operand(nullptr, kn, nullptr, R::NP + j), w.q[j % R::NQ],
                            j % R::NQ == 0 ? zero : sc[j / R::NQ]);
  const float4_t fkn = ld<float4_t>(fknp), lvn = ld<float4_t>(lvnp);
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
  return i8_best(top, fkn, lvn);
}

// One step of a wavefront. Its scores stand in sc (tokens 0-31, 32-63), P' of the last step's
// second half in pr[2], pr[3]; the next step's scores replace them. Four phases, each a run of MFMAs
// beside a share of the vector work:
//   P'(sc[0])  beside  O += V P' of the last step's second half
//   P'(sc[1])  beside  sc[0] = K . Q^T of the next step
//   staging    beside  sc[1] = K . Q^T of the next step
//   maxima of the next scores, more staging  beside  O += V P' of this step's first half
// so that no second set of scores is needed (two wavefronts share a SIMD's registers). The order is
// pinned, MFMA by MFMA: left to itself the compiler sets MFMAs and exponentials one after the other.
// The workgroup meets behind the first phase, with no LDS read under way: what the step before staged
// (K in its third phase, V in its fourth) is read behind that, and this step stages over what was
// read before it. Returns each row's largest next score.
template <int D, typename Mask, typename Work>
__device__ __forceinline__ float i8_step64(I8Rows<D>& w, const half_t* vp, const half_t* kn, const half_t* vc,
                                           float16_t (&sc)[2], half8_t (&pr)[4], const float* fkp,
                                           const float* lvp, const float* backp, const float* fknp,
                                           const float* lvnp, Mask mask, Work work) {
  typedef I8Rows<D> R;
  constexpr int NQ = R::NQ, NP = R::NP, AHEAD = R::AHEAD;
  half8_t op[AHEAD];
  const float4_t fk = ld<float4_t>(fkp), lv = ld<float4_t>(lvp);
#pragma unroll
  for (int j = 0; j < AHEAD && j < NP; ++j) op[j] = w.operand(vp, kn, vc, j);
  const float4_t back = ld<float4_t>(backp);
  // Operand j, and the request of a later one below `end`. (The ring starts anew behind the barrier.)
  auto next = [&](int j, int end) {
    const half8_t x = op[j % AHEAD];
    if (j + AHEAD < end) op[j % AHEAD] = w.operand(vp, kn, vc, j + AHEAD);
    return x;
  };
  const float neg = w.m == -INFINITY ? 0.f : -w.m;
  const float off[4] = {neg + lv[0], neg + lv[1], neg + lv[2], neg + lv[3]};
  // exponentials: NP + NQ shares beside the first two phases' MFMAs where both have as many
  constexpr int N = 2 * (NP < NQ ? NP : NQ);
  I8Exp ex;
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    w.o[j % R::DT] = mfma_i8(next(j, NP), pr[2 + j / R::DT], w.o[j % R::DT]);
    if (j < N / 2) ex.share<N>(j, sc, fk, off, back, w.l, pr);
    if (j == 0) work(0);                                   // requests of K, V to come
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
    if (j < N / 2) ex.share<N>(N / 2 + j, sc, fk, off, back, w.l, pr);
    for (int v = j * 4 / NQ; v < (j + 1) * 4 / NQ; ++v) work(3 + v);
    __builtin_amdgcn_sched_barrier(0);
  }
#pragma unroll
  for (int j = 0; j < NQ; ++j) {
    sc[1] = mfma_i8(next(NP + NQ + j, R::ALL), w.q[j], j == 0 ? zero : sc[1]);
    if (j < 2) ex.share<N>(N + j, sc, fk, off, back, w.l, pr);
    if (NQ < 2) ex.share<N>(N + 1, sc, fk, off, back, w.l, pr);
    if (j == NQ / 4) work(1);                              // K of a later step to LDS
    __builtin_amdgcn_sched_barrier(0);
  }
  const float4_t fkn = ld<float4_t>(fknp), lvn = ld<float4_t>(lvnp);
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
  return i8_best(top, fkn, lvn);
}

// A row's largest s + log2 vs moves its reference; O follows in the next step, behind what was computed
// against the old one.
template <int D>
__device__ __forceinline__ void i8_reference(I8Rows<D>& w, float best) {
  const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(best), __float_as_uint(best), false, false);
  best = vmax(__uint_as_float(both[0]), __uint_as_float(both[1]));
  const bool move = !(best <= w.m + kI8Rescale);           // NaN moves it too
  w.moved = __ballot(move) != 0;
  if (w.moved) {
    const float to = vmax(w.m, best);                      // (a NaN stays)
    w.alpha = move ? fast_exp2(w.m - to) : 1.f;
    w.l *= w.alpha;
    w.m = move ? to : w.m;
  }
}

// One tile's steps [s0, s1) by the workgroup.
template <int D, int WAVES>
__device__ __forceinline__ void i8_piece(const Int8PrefillArgs& p, I8PrefillLds<D>& lds, const I8Chunk& k,
                                         int b, int tile, int h, int s0, int s1, bool whole, int slot) {
  typedef I8Rows<D> R;
  typedef I8Stage<D, WAVES * kWave> S;
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
    // a window of the sequence's blocks: ids, scales
    const int n = min(s1 - w0, kI8Window / kI8StepBlocks);
    const int blocks = min(nb - w0 * kI8StepBlocks, n * kI8StepBlocks), last = blocks - 1;
    __syncthreads();                                       // the last window's and piece's reads
    constexpr int PER = (kI8Window + THREADS - 1) / THREADS;
    const int32_t* table = a.block_tables + b * a.bt_stride + w0 * kI8StepBlocks;
    S stage;
    int id0[S::N], id1[S::N], id2[S::N];                   // of the next step, the second, the third
    S::ids(a, table, last, id0);
    int blk[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = threadIdx.x + i * THREADS;
      blk[i] = at < blocks ? clamp_block(table[at], a.num_blocks) : 0;
    }
    float scales[PER][2];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const bool real = (int)threadIdx.x + i * THREADS < blocks;
      scales[i][0] = real ? a.ks[(int64_t)blk[i] * a.kvh + h] : 0.f;
      scales[i][1] = real ? a.vs[(int64_t)blk[i] * a.kvh + h] : 0.f;
    }
    stage.request_k(a, id0, h);
    if (w0 == s0) {                                        // q behind what the first scores wait for
      const half_t* qrow = a.q + (int64_t)(k.q0 + token) * a.q_st + (int64_t)head * a.q_sh;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) w.q[i] = ld<half8_t>(qrow + 16 * i + 8 * hh);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = threadIdx.x + i * THREADS;
      float ks = scales[i][0], vs = scales[i][1];
      i8_poison(ks, vs);
      // A K factor of 0 or NaN would leave hidden tokens (-inf) NaN: scores of a factor as small as
      // the least one are 0, and the codes of blocks without finite scales are staged as NaN.
      const float f = ks * a.sl2;
      if (at < kI8Window) {
        lds.blk[at] = f == f ? blk[i] : blk[i] | (int)0x80000000;
        lds.fk[at] = f > kI8LeastFactor ? f : kI8LeastFactor;
        i8_value_factors(vs, lds.lv[at], lds.back[at]);
      }
    }
    __syncthreads();
    S::ids(lds, 0, last, id0);
    S::ids(lds, kI8StepBlocks, last, id1);
    stage.finite(id0);
    stage.place_k(lds.k[0]);
    for (int i = threadIdx.x; i < I8Tile<D>::HALVES / 8; i += THREADS)
      st<half8_t>(lds.v[1] + 8 * i, half8_t{0, 0, 0, 0, 0, 0, 0, 0});
    __syncthreads();

    // Step i reads K of step i + 1 in k[(i + 1) % 2], V of steps i - 1 and i in v[(i - 1) % 2] and
    // v[i % 2], and stages K of step i + 2 and V of step i + 1. Before the first of them the scores of
    // step 0 are formed (i8_first; P' of a step before it is 0, on V codes of 0). The loop has no
    // branch but the mask's and the reference's: past the window's end the last blocks are staged
    // again, and the scores of the step behind it are not used.
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
      const int wb = i * kI8StepBlocks;
      const float best = decltype(first)::value
                             ? i8_first<D>(w, lds.k[0], sc, lds.fk, lds.lv, mask, work)
                             : i8_step64<D>(w, lds.v[1 - P], lds.k[1 - P], lds.v[P], sc, pr,
                                            lds.fk + wb, lds.lv + wb, lds.back + wb,
                                            lds.fk + wb + kI8StepBlocks, lds.lv + wb + kI8StepBlocks, mask, work);
      i8_reference<D>(w, i + 1 < n ? best : w.m);          // (its own reference moves none, also a NaN)
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
      const float4_t x = float4_t{w.o[t][i], w.o[t][i + 1], w.o[t][i + 2], w.o[t][i + 3]} * kColumnUnit * f;
      if (whole)
        st<half4_t>(dst + d, to_half4(x));
      else
        st<float4_t>(a.part_o + at * D + d, x);
    }
}

// Wavefronts of a workgroup, and the workgroups that a CU holds by registers. At head_dim 128 eight
// wavefronts stage a step together (85 us at 2048 rows on 4096 cached, 12/2 heads; two workgroups of
// four 102 us); at 64 and below a step's codes are one unit a thread for four (27 us against 40 at
// five chunks of 90 to 1100 rows, 14/2 heads).
constexpr int i8_prefill_waves(int D) { return D == 128 ? 8 : 4; }
constexpr int i8_prefill_groups(int D) { return D > 128 ? 1 : 8 / i8_prefill_waves(D); }

template <int D>
__global__ void __launch_bounds__(i8_prefill_waves(D) * kWave, D > 128 ? 1 : 2)
prefill_int8_kernel(Int8PrefillArgs p) {
  constexpr int WAVES = i8_prefill_waves(D), ROWS = 32 * WAVES;
  __shared__ __align__(16) I8PrefillLds<D> lds;
  const Int8DecodeArgs& a = p.a;
  int at, hi, h;
  I8Place place;
  {
    const I8Walk<ROWS> walk(p);
    const int total = walk.total * a.kvh;
    const I8Shares shares(total, p.groups);
    I8Joint joint = {};
    bool found = false;
    if (total > 0 && (int)blockIdx.x < shares.count) {
      at = shares.begin(blockIdx.x), hi = shares.begin(blockIdx.x + 1);
      found = walk.find(p, a.by_kvh(at), place);
      h = (int)((unsigned)(at - place.before * a.kvh) / (unsigned)place.cost);
      found = found && (unsigned)h < (unsigned)a.kvh;
    }
    if (found) {
      const int s0 = place.before * a.kvh + h * place.cost + kI8TileCost;
      const int g = blockIdx.x;
      if (g > 0 && shares.begin(g - 1) <= s0 && s0 < at) {
        const int last = shares.of(s0 + i8_steps<ROWS>(a, place.k, place.tile) - 1);
        if (last >= g && last < shares.count)
          joint = {g - 1, last, place.k.q0, place.k.n * a.group, place.tile * ROWS, h};
      }
    }
    if (threadIdx.x == 0) p.joints[blockIdx.x] = joint;
    if (!found) return;
    if (threadIdx.x < kWave) walk.save(lds.walk);
  }
  __syncthreads();                                         // (saved)
  while (true) {
    const int c0 = at - place.before * a.kvh - h * place.cost, c1 = min(place.cost, c0 + (hi - at));
    at += c1 - c0;
    const int steps = i8_steps<ROWS>(a, place.k, place.tile);
    const int s0 = max(0, c0 - kI8TileCost), s1 = min(c1 - kI8TileCost, steps);
    if (s1 > s0)
      i8_piece<D, WAVES>(p, lds, place.k, place.seq, place.tile, h, s0, s1, s0 == 0 && s1 == steps,
                         2 * blockIdx.x + (s0 == 0));
    if (at >= hi) return;
    if (!I8Walk<ROWS>(lds.walk).find(p, a.by_kvh(at), place)) return;
    h = (int)((unsigned)(at - place.before * a.kvh) / (unsigned)place.cost);
    if ((unsigned)h >= (unsigned)a.kvh) return;
  }
}

// Tiles that several workgroups share: kI8MergeRows rows a workgroup, D / 4 threads a row. The
// workgroups stand for the shares' beginnings: the first one inside a tile has it merged. (At
// 2048 rows on 4096 cached, 12/2 heads of 128: 9.5 us, 53 MB of partials; 10.5 when each workgroup
// looked the tile up; 32 rows a workgroup are 1 to 2 us slower.)
constexpr int kI8MergeRows = 16;
template <int D, int ROWS>
__global__ void __launch_bounds__(256) prefill_int8_merge_kernel(Int8PrefillArgs p) {
  constexpr int PER = 256 / (D / 4);                       // rows at a time
  constexpr int R = kI8MergeRows > PER ? kI8MergeRows / PER : 1, N = 4;   // rows of a thread, partials at a time
  const Int8DecodeArgs& a = p.a;
  const int g = 1 + (int)(blockIdx.x / (ROWS / kI8MergeRows));
  const int row0 = (int)(blockIdx.x % (ROWS / kI8MergeRows)) * kI8MergeRows;
  const I8Joint j = p.joints[g];
  if (j.first == j.last || j.row0 + row0 >= j.rows) return;
  const int in = row0 + threadIdx.x / (D / 4), d = threadIdx.x % (D / 4) * 4;
  if (PER > kI8MergeRows && in >= row0 + kI8MergeRows) return;
  float top[R], sum[R];
  float4_t o[R];
#pragma unroll
  for (int r = 0; r < R; ++r) top[r] = -INFINITY, sum[r] = 0.f, o[r] = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = j.first; i0 <= j.last; i0 += N) {
    float2_t ml[N][R];
    float4_t x[N][R];
#pragma unroll
    for (int i = 0; i < N; ++i) {                          // (rows past the last one hold anything)
      if (i0 + i > j.last) continue;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int64_t at = (int64_t)(2 * (i0 + i) + (i0 + i == j.first)) * ROWS + in + r * PER;
        ml[i][r] = ld<float2_t>(a.part_ml + 2 * at);
        x[i][r] = ld<float4_t>(a.part_o + at * D + d);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float now = top[r];
#pragma unroll
      for (int i = 0; i < N; ++i) now = i0 + i <= j.last ? vmax(now, ml[i][r][0]) : now;
      const float f = top[r] == -INFINITY ? 0.f : fast_exp2(top[r] - now);
      sum[r] *= f;
      o[r] *= f;
      top[r] = now;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (i0 + i > j.last || ml[i][r][0] == -INFINITY) continue;
        const float e = fast_exp2(ml[i][r][0] - now);
        sum[r] = fmaf(e, ml[i][r][1], sum[r]);
        o[r] += x[i][r] * e;
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = j.row0 + in + r * PER;
    if (row >= j.rows) return;
    const float f = sum[r] == 0.f ? 0.f : 1.f / sum[r];
    const int token = a.by_group(row), head = j.h * a.group + row - token * a.group;
    st<half4_t>(a.out + (int64_t)(j.q0 + token) * a.out_st + (int64_t)head * D + d, to_half4(o[r] * f));
  }
}

}  // namespace ts
