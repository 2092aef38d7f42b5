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
// A block's K scale multiplies its scores in fp32. Its V scale multiplies P, measured against the
// largest V scale so far, before P is rounded to fp16.
//
// Lane l is split into c = l % 32 and h = l / 32: a result lane holds S^T[8 (i / 4) + 4 h + i % 4][c],
// i = 0..15, so a lane's scores all belong to row c, and its P values for a block's 16 tokens (i % 8
// of one half) are the B operand of the P.V step as they stand when V^T lies in LDS with the
// tokens of a block in the order {0-3, 8-11 | 4-7, 12-15}.
#pragma once

#include "decode_int8.h"

namespace ts {

typedef float float16_t __attribute__((ext_vector_type(16)));

constexpr int kI8Keys = 64;              // tokens of a step
constexpr int kI8StepBlocks = kI8Keys / kBlockSize;
constexpr int kI8Window = 128;           // blocks whose ids and scales are held in LDS at a time

struct Int8PrefillArgs {
  Int8DecodeArgs a;                      // (part_o, part_ml: the prefill partials)
  const int32_t* qsl;
  int64_t num_tokens;
  int num_seqs, first;                   // sequences first .. num_seqs - 1
  int tiles, splits;                     // launched per (sequence, KV head)
};

__device__ __forceinline__ float16_t mfma_i8(half8_t a, half8_t b, float16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

template <int D>
struct I8Tile {
  static constexpr int KCHUNKS = D / 8;                    // 16-byte chunks of a K row
  static constexpr int KSWZ = (KCHUNKS < 16 ? KCHUNKS : 16) - 1;
  half_t k[kI8Keys * D];
  half_t v[D * kI8Keys];
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
  I8Tile<D> tile[2];
  int blk[kI8Window];
  float fk[kI8Window], vs[kI8Window];
};

// The codes of a step that one thread widens: units of 16 codes of a K row, and of 4 tokens x 4
// dims of V; 4 D of each in a step.
template <int D, int THREADS>
struct I8Stage {
  static constexpr int UNITS = 4 * D;
  static constexpr int N = (UNITS + THREADS - 1) / THREADS;
  uint4_t k[N];
  uint32_t v[N][4];
};

// Requests the codes of blocks w0 .. w0 + 3 of the window (the last real one again past the end).
template <int D, int THREADS>
__device__ __forceinline__ void i8_request(const Int8DecodeArgs& a, const I8PrefillLds<D>& lds, int w0,
                                           int last, int h, I8Stage<D, THREADS>& x) {
  typedef I8Stage<D, THREADS> S;
#pragma unroll
  for (int i = 0; i < S::N; ++i) {
    const int u = threadIdx.x + i * THREADS;
    if (S::UNITS % THREADS != 0 && u >= S::UNITS) break;
    // K: key = u / (D / 16), 16 codes at 16 (u % (D / 16)); V: token group and dims below. Both
    // belong to block u / D of the step.
    const int64_t base = ((int64_t)lds.blk[min(w0 + u / D, last)] * a.kvh + h) * (kBlockSize * D);
    const int in = u % D;
    x.k[i] = ld<uint4_t>(a.kc + base + 16 * in);
    const int8_t* v = a.vc + base + (int64_t)(4 * (in / (D / 4))) * D + 4 * (in % (D / 4));
#pragma unroll
    for (int r = 0; r < 4; ++r) x.v[i][r] = ld<uint32_t>(v + r * D);
  }
}

template <int D, int q>
__device__ __forceinline__ void i8_place_v(I8Tile<D>& t, const uint32_t (&v)[4], int block, int group, int d0) {
  const half2_t a = column2<q>(v[0], v[1]), b = column2<q>(v[2], v[3]);
  st<half4_t>(t.v + I8Tile<D>::v_at(d0 + q, block, group & 1) + 4 * (group >> 1),
              half4_t{a[0], a[1], b[0], b[1]});
}

template <int D, int THREADS>
__device__ __forceinline__ void i8_place(I8Tile<D>& t, const I8Stage<D, THREADS>& x) {
  typedef I8Stage<D, THREADS> S;
#pragma unroll
  for (int i = 0; i < S::N; ++i) {
    const int u = threadIdx.x + i * THREADS;
    if (S::UNITS % THREADS != 0 && u >= S::UNITS) break;
    const int key = u / (D / 16), chunk = 2 * (u % (D / 16));
    st<half8_t>(t.k + I8Tile<D>::k_at(key, chunk), codes8(x.k[i][0], x.k[i][1]));
    st<half8_t>(t.k + I8Tile<D>::k_at(key, chunk + 1), codes8(x.k[i][2], x.k[i][3]));
    uint32_t v[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = x.v[i][r] ^ 0x80808080u;
    const int in = u % D, block = u / D, group = in / (D / 4), d0 = 4 * (in % (D / 4));
    i8_place_v<D, 0>(t, v, block, group, d0);
    i8_place_v<D, 1>(t, v, block, group, d0);
    i8_place_v<D, 2>(t, v, block, group, d0);
    i8_place_v<D, 3>(t, v, block, group, d0);
  }
}

template <int D, int WAVES>
__global__ void __launch_bounds__(WAVES* kWave, D >= 256 ? 1 : 2) prefill_int8_kernel(Int8PrefillArgs p) {
  constexpr int THREADS = WAVES * kWave, ROWS = 32 * WAVES;
  constexpr int DT = (D + 31) / 32;                        // output tiles of 32 dims
  __shared__ __align__(16) I8PrefillLds<D> lds;
  const Int8DecodeArgs& a = p.a;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave, c = lane % 32, hh = lane / 32;

  // blockIdx.x: split, KV head, tile (the longest first), sequence
  int64_t u = blockIdx.x;
  const int split = (int)(u % p.splits);
  u /= p.splits;
  const int h = (int)(u % a.kvh);
  u /= a.kvh;
  const int tile0 = p.tiles - 1 - (int)(u % p.tiles);
  const int b = p.first + (int)(u / p.tiles);
  const int len = table_entry(a.seq_lens + b);
  const int64_t q0 = table_entry(p.qsl + b), q1 = table_entry(p.qsl + b + 1);
  if (q0 < 0 || q1 <= q0 || q1 > p.num_tokens) return;
  const int n = (int)(q1 - q0);
  const int64_t rows = (int64_t)n * a.group;
  const int kv = i8_kv_len(len, a.max_blocks);
  const int64_t start = (int64_t)len - n;                  // position of row q0

  // Tiles past the launched ones (a host bound below the batch's real rows) are taken unsplit by
  // the first split's workgroup.
  for (int tile = tile0; (int64_t)tile * ROWS < rows; tile += p.tiles) {
    const bool extra = tile >= p.tiles;
    if (extra && split > 0) return;
    const int splits = extra ? 1 : p.splits;
    const int64_t last_row = min(rows, (int64_t)(tile + 1) * ROWS) - 1;
    // tokens that the tile's last row sees, and its steps
    const int64_t sees = min((int64_t)kv, start + last_row / a.group + 1);
    const int steps = sees > 0 ? (int)((sees + kI8Keys - 1) / kI8Keys) : 0;
    const int s0 = (int)((int64_t)steps * split / splits), s1 = (int)((int64_t)steps * (split + 1) / splits);

    const int64_t row = (int64_t)tile * ROWS + 32 * wave + c;
    const bool real = row < rows;
    const int token = real ? (int)(row / a.group) : 0;
    const int head = h * a.group + (real ? (int)(row % a.group) : 0);
    const int vis = real ? (int)max((int64_t)0, min((int64_t)kv, start + token + 1)) : 0;
    // bounds over the wavefront's rows: rows ascend in tokens, so its first row sees least
    const int64_t wrow = (int64_t)tile * ROWS + 32 * wave;
    const int64_t wlast = min(rows - 1, wrow + 31);
    const int wave_least =
        wrow < rows ? (int)max((int64_t)0, min((int64_t)kv, start + wrow / a.group + 1)) : 0;
    const int wave_most = wrow < rows ? (int)max((int64_t)0, min((int64_t)kv, start + wlast / a.group + 1)) : 0;

    half8_t q[D / 16];
    const half_t* qrow = a.q + (q0 + token) * a.q_st + (int64_t)head * a.q_sh;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) q[i] = ld<half8_t>(qrow + 16 * i + 8 * hh);

    float16_t o[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[t][i] = 0.f;
    float m = -INFINITY, l = 0.f, vref = 0.f;

    const int nb = (int)((sees + kBlockSize - 1) / kBlockSize);   // real blocks of the tile
    I8Stage<D, THREADS> stage;
    for (int w0 = s0; w0 < s1; w0 += kI8Window / kI8StepBlocks) {
      // a window of the sequence's blocks: ids and scales
      const int w1 = min(s1, w0 + kI8Window / kI8StepBlocks);
      const int blocks = min(nb - w0 * kI8StepBlocks, (w1 - w0) * kI8StepBlocks);
      __syncthreads();                                     // the last window's and tile's reads
      for (int i = threadIdx.x; i < kI8Window; i += THREADS) {
        int blk = 0;
        float ks = 0.f, vs = 0.f;
        if (i < blocks) {
          blk = clamp_block(a.block_tables[b * a.bt_stride + w0 * kI8StepBlocks + i], a.num_blocks);
          ks = a.ks[(int64_t)blk * a.kvh + h];
          vs = a.vs[(int64_t)blk * a.kvh + h];
          i8_poison(ks, vs);
        }
        lds.blk[i] = blk, lds.fk[i] = ks * a.sl2, lds.vs[i] = vs;
      }
      __syncthreads();
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < kI8Window; i += kWave) top = fmaxf(top, lds.vs[i + lane]);
      top = i8_most(top);
      if (top > vref) {
        const float f = vref / top;
        vref = top;
#pragma unroll
        for (int t = 0; t < DT; ++t) o[t] *= f;
      }
      const float inv = vref > 0.f ? 1.f / vref : 0.f;

      i8_request<D, THREADS>(a, lds, 0, blocks - 1, h, stage);
      i8_place<D, THREADS>(lds.tile[0], stage);
      for (int s = w0; s < w1; ++s) {
        const int buf = (s - w0) & 1, wb = (s - w0) * kI8StepBlocks;
        const bool more = s + 1 < w1;
        if (more) i8_request<D, THREADS>(a, lds, wb + kI8StepBlocks, blocks - 1, h, stage);
        __syncthreads();                                   // tile `buf` is whole
        const I8Tile<D>& t = lds.tile[buf];
        if (s * kI8Keys < wave_most) {
          float16_t sc[2];
#pragma unroll
          for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[kt][i] = 0.f;
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
              sc[kt] = mfma_i8(ld<half8_t>(t.k + I8Tile<D>::k_at(32 * kt + c, 2 * i + hh)), q[i], sc[kt]);
          }
          float fk[kI8StepBlocks], fv[kI8StepBlocks];
#pragma unroll
          for (int i = 0; i < kI8StepBlocks; ++i) fk[i] = lds.fk[wb + i], fv[i] = lds.vs[wb + i] * inv;
          // scores in log2 units
#pragma unroll
          for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[kt][i] *= fk[2 * kt + i / 8];
          if ((s + 1) * kI8Keys > wave_least) {
            const int key0 = s * kI8Keys + 4 * hh;
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
              for (int i = 0; i < 16; ++i)
                sc[kt][i] = key0 + 32 * kt + 8 * (i / 4) + i % 4 < vis ? sc[kt][i] : -INFINITY;
          }
          float best = vmax(sc[0][0], sc[1][0]);
#pragma unroll
          for (int i = 1; i < 16; ++i) best = vmax(best, vmax(sc[0][i], sc[1][i]));
          const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(best), __float_as_uint(best), false, false);
          best = vmax(__uint_as_float(both[0]), __uint_as_float(both[1]));
          const bool move = !(best <= m + kI8Rescale);     // NaN moves it too
          if (__ballot(move)) {
            const float alpha = move ? fast_exp2(m - best) : 1.f;
            l *= alpha;
            m = move ? best : m;
#pragma unroll
            for (int i = 0; i < DT; ++i) o[i] *= alpha;
          }
          const float neg = m == -INFINITY ? 0.f : -m;
          half8_t pr[kI8StepBlocks];
#pragma unroll
          for (int blk = 0; blk < kI8StepBlocks; ++blk)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float x = fast_exp2(sc[blk / 2][8 * (blk % 2) + e] + neg);
              l += x;
              pr[blk][e] = (half_t)(x * fv[blk]);
            }
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int blk = 0; blk < kI8StepBlocks; ++blk)
              o[dt] = mfma_i8(ld<half8_t>(t.v + I8Tile<D>::v_at(D < 32 ? c % D : 32 * dt + c, blk, hh)),
                              pr[blk], o[dt]);
        }
        if (more) i8_place<D, THREADS>(lds.tile[buf ^ 1], stage);
      }
    }

    // lanes c and c + 32 hold the two halves of row c's sum
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    l = __uint_as_float(both[0]) + __uint_as_float(both[1]);
    if (!real) continue;
    if (splits == 1) {
      const float f = l == 0.f ? 0.f : vref / l;           // nothing visible: zeros
      half_t* dst = a.out + (q0 + token) * a.out_st + (int64_t)head * D;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const int d = 32 * dt + 8 * (i / 4) + 4 * hh;
          if (D < 32 && d >= D) break;
          st<half4_t>(dst + d, to_half4(float4_t{o[dt][i], o[dt][i + 1], o[dt][i + 2], o[dt][i + 3]} * f));
        }
    } else {
      const int64_t at =
          ((((int64_t)(b - p.first) * p.tiles + tile) * a.kvh + h) * p.splits + split) * ROWS + 32 * wave + c;
      if (hh == 0) {
        a.part_ml[2 * at] = m;
        a.part_ml[2 * at + 1] = l;
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const int d = 32 * dt + 8 * (i / 4) + 4 * hh;
          if (D < 32 && d >= D) break;
          st<float4_t>(a.part_o + at * D + d,
                       float4_t{o[dt][i], o[dt][i + 1], o[dt][i + 2], o[dt][i + 3]} * vref);
        }
    }
  }
}

// The splits' partials of the launched tiles: D / 4 threads a row, several rows a workgroup.
template <int D, int ROWS>
__global__ void __launch_bounds__(256) prefill_int8_merge_kernel(Int8PrefillArgs p) {
  const Int8DecodeArgs& a = p.a;
  constexpr int PER = 256 / (D / 4);                       // rows of a workgroup
  const int64_t unit = blockIdx.x / (ROWS / PER);
  const int in = (int)(blockIdx.x % (ROWS / PER)) * PER + threadIdx.x / (D / 4);
  const int d = threadIdx.x % (D / 4) * 4;
  const int h = (int)(unit % a.kvh);
  const int tile = (int)(unit / a.kvh % p.tiles);
  const int b = p.first + (int)(unit / a.kvh / p.tiles);
  const int64_t q0 = table_entry(p.qsl + b), q1 = table_entry(p.qsl + b + 1);
  if (q0 < 0 || q1 <= q0 || q1 > p.num_tokens) return;
  const int64_t row = (int64_t)tile * ROWS + in;
  if (row >= (q1 - q0) * a.group) return;
  const int64_t at = unit * p.splits * ROWS + in;
  float top = -INFINITY;
  for (int i = 0; i < p.splits; ++i) top = vmax(top, a.part_ml[2 * (at + (int64_t)i * ROWS)]);
  float sum = 0.f;
  float4_t o = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < p.splits; ++i) {
    const int64_t k = at + (int64_t)i * ROWS;
    const float m = a.part_ml[2 * k];
    if (m == -INFINITY) continue;
    const float f = fast_exp2(m - top);
    sum += f * a.part_ml[2 * k + 1];
    o += ld<float4_t>(a.part_o + k * D + d) * f;
  }
  const float f = sum == 0.f ? 0.f : 1.f / sum;
  const int64_t token = q0 + row / a.group;
  const int64_t head = h * a.group + row % a.group;
  st<half4_t>(a.out + token * a.out_st + head * D + d, to_half4(o * f));
}

}  // namespace ts
