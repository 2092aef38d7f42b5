// The 4-bit paged cache shared by its write, read and attention kernels. One block of one KV head is a
// unit of bytes: 16 rows of 4-bit codes, then, for each row and group of 32 channels (16 at head_dim
// 16), two fp16 numbers, step and low; a code stands for fp16(low + code * step), rounded once.
//
//   codes    8 channels (an octet) are a word; its nibbles hold the channels 0 2 4 6 | 1 3 5 7, low
//            ones first, so that a mask leaves two neighbours where two fp16 mantissas lie
//   K units  words [16 rows][D / 8], numbers [16 rows][groups][step, low]: a lane of the score
//            product's operand reads its token's share of the row, at head_dim 128 the 16 bytes of one
//            group, and the group's numbers in one word
//   V units  words [D / 8][16 rows], numbers [groups][4][step, low][4 rows]: a lane of the output
//            product's operand reads an octet of four tokens in 16 bytes, and their numbers in 16 bytes,
//            two tokens to a word, as that product's operand has them
//
// A row's numbers depend on that row alone, so rows are written without a look at their block. Groups
// of 32 with two numbers cost a fourth on top of the codes (5 bits a value); one group for a row of 128
// would cost 4.25 and have all channels of K, which differ in size, share a step.
#pragma once

#include "common.h"

namespace ts {

template <int D>
struct I4Unit {
  static constexpr int GROUP = D < 32 ? D : 32, GROUPS = D / GROUP;
  static constexpr int CODES = kBlockSize * D / 2;                   // bytes
  static constexpr int BYTES = CODES + kBlockSize * GROUPS * 4;
  static __host__ __device__ constexpr int k_word(int row, int octet) { return (row * (D / 8) + octet) * 4; }
  static __host__ __device__ constexpr int v_word(int row, int octet) { return (octet * kBlockSize + row) * 4; }
  // K: step and low side by side; V: the step, the low 8 bytes on
  static __host__ __device__ constexpr int k_numbers(int row, int group) { return CODES + (row * GROUPS + group) * 4; }
  static __host__ __device__ constexpr int v_numbers(int row, int group) {
    return CODES + (group * 4 + row / 4) * 16 + row % 4 * 2;
  }
};

__device__ __forceinline__ half2_t i4_half2(uint32_t w) { return __builtin_bit_cast(half2_t, w); }

// What the widening takes beside a word, held in registers: with the exponent of 1024 in one and the masks in
// scalar ones a nibble is masked and placed by one instruction (literals would make two of it).
struct I4Bits {
  uint32_t one, low, high;
  __device__ __forceinline__ I4Bits() {
    asm("v_mov_b32 %0, 0x64006400" : "=v"(one));
    asm("s_mov_b32 %0, 0x000f000f" : "=s"(low));
    asm("s_mov_b32 %0, 0x00f000f0" : "=s"(high));
  }
};

// Nibble P of each half of w (w8: w >> 8) as packed fp16, exactly: under the exponent of 1024 a nibble in
// bits 0 .. 3 is 1024 + code, one in bits 4 .. 7 is 1024 + 16 code.
template <int P>
__device__ __forceinline__ half2_t i4_codes(const I4Bits& k, uint32_t w, uint32_t w8) {
  const uint32_t x = P < 2 ? w : w8;
  if constexpr (P % 2 == 0) {
    const half2_t off = {(half_t)-1024.f, (half_t)-1024.f};
    return i4_half2((x & k.low) | k.one) + off;
  } else {
    const half2_t by = {(half_t)0.0625f, (half_t)0.0625f}, off = {(half_t)-64.f, (half_t)-64.f};
    return __builtin_elementwise_fma(i4_half2((x & k.high) | k.one), by, off);
  }
}
template <int P>
__device__ __forceinline__ half2_t i4_values(const I4Bits& k, uint32_t w, uint32_t w8, half2_t step, half2_t low) {
  return __builtin_elementwise_fma(i4_codes<P>(k, w, w8), step, low);
}

// The octet of a word whose numbers are `n` (step in the low half, low in the high one), in the order of
// its channels.
__device__ __forceinline__ half8_t i4_octet(const I4Bits& k, uint32_t w, uint32_t n) {
  const half2_t p = i4_half2(n), step = {p[0], p[0]}, low = {p[1], p[1]};
  const uint32_t w8 = w >> 8;
  const half2_t a = i4_values<0>(k, w, w8, step, low), b = i4_values<1>(k, w, w8, step, low);
  const half2_t c = i4_values<2>(k, w, w8, step, low), d = i4_values<3>(k, w, w8, step, low);
  return {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Even (odd) channels of an octet for two tokens: nibble j of a half is channel 2 j (2 j + 1).
__device__ __forceinline__ uint32_t i4_even(uint32_t row0, uint32_t row1) {
  return __builtin_amdgcn_perm(row1, row0, 0x05040100u);
}
__device__ __forceinline__ uint32_t i4_odd(uint32_t row0, uint32_t row1) {
  return __builtin_amdgcn_perm(row1, row0, 0x07060302u);
}

// A low of NaN stands for a token whose row was not finite. Its K makes the scores of the rows that see it
// NaN; its V has to stay out of the rows that do not, where its weight is 0: any number does.
// (The instruction returns the other operand for a NaN; maxnum would quiet its operand first.)
__device__ __forceinline__ half2_t i4_finite(uint32_t lows) {
  uint32_t x;
  asm("v_pk_max_f16 %0, %1, %2" : "=v"(x) : "v"(lows), "s"(0xfbfffbffu));    // -65504
  return i4_half2(x);
}

}  // namespace ts
