// The 8-bit paged cache shared by its write and attention kernels: int8 codes
// [num_blocks, KVH, 16, D] with one fp32 scale per (block, KV head), [num_blocks, KVH]; a code
// stands for code * scale.
//
// Codes become fp16 exactly in registers: u = code + 128 (the sign bit flipped) under the high
// byte 0x64 is the fp16 number 1024 + u, and subtracting 1152 leaves the code (every integer up to
// 2048 is an fp16 number, so nothing rounds).
#pragma once

#include "common.h"

namespace ts {

constexpr float kCodeMax = 127.f;

__device__ __forceinline__ half2_t as_half2(uint32_t w) { return __builtin_bit_cast(half2_t, w); }

// 1024 + u (two packed) -> the codes.
__device__ __forceinline__ half2_t unbias(uint32_t w, half2_t off = {(half_t)1152.f, (half_t)1152.f}) {
  return as_half2(w) - off;
}

// Codes 0, 1 and 2, 3 of a word (sign bits flipped already) as packed fp16.
__device__ __forceinline__ half2_t codes01(uint32_t u, half2_t off = {(half_t)1152.f, (half_t)1152.f}) {
  return unbias(__builtin_amdgcn_perm(0x64646464u, u, 0x04010400u), off);
}
__device__ __forceinline__ half2_t codes23(uint32_t u, half2_t off = {(half_t)1152.f, (half_t)1152.f}) {
  return unbias(__builtin_amdgcn_perm(0x64646464u, u, 0x04030402u), off);
}

// Eight consecutive codes (two words) as an MFMA operand; off: 1152, or NaN for codes that mean
// nothing.
__device__ __forceinline__ half8_t codes8(uint32_t w0, uint32_t w1,
                                          half2_t off = {(half_t)1152.f, (half_t)1152.f}) {
  w0 ^= 0x80808080u;
  w1 ^= 0x80808080u;
  const half2_t a = codes01(w0, off), b = codes23(w0, off), c = codes01(w1, off), d = codes23(w1, off);
  return {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Code `q` of each of two words (sign bits flipped already) as packed fp16, in units of
// 1 / kColumnUnit: a column of the rows that the words come from. u alone in a half is the fp16
// subnormal u 2^-24; times 2^15 minus 1/4 it is (u - 128) 2^-9, exactly, in one packed instruction.
constexpr float kColumnUnit = 512.f;
template <int q>
__device__ __forceinline__ half2_t column2(uint32_t row0, uint32_t row1) {
  const half2_t up = {(half_t)32768.f, (half_t)32768.f}, off = {(half_t)-0.25f, (half_t)-0.25f};
  return __builtin_elementwise_fma(as_half2(__builtin_amdgcn_perm(row1, row0, 0x0c040c00u + q * 0x00010001u)),
                                   up, off);
}

// Wavefront scans on the VALU (DPP row shifts, then the rows' last lanes broadcast on): a step costs
// a few cycles where a shuffle through the LDS unit costs over a hundred, and the scans stand in
// front of a launch's K/V requests or stores.
template <int CTRL, int ROWS>
__device__ __forceinline__ int i8_dpp(int v) {             // 0 where no lane moves in
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int i8_scan(int v) {            // inclusive sums
  v += i8_dpp<0x111, 0xf>(v);
  v += i8_dpp<0x112, 0xf>(v);
  v += i8_dpp<0x114, 0xf>(v);
  v += i8_dpp<0x118, 0xf>(v);
  v += i8_dpp<0x142, 0xa>(v);
  return v + i8_dpp<0x143, 0xc>(v);
}
__device__ __forceinline__ float i8_most(float x) {        // the largest of 64 values >= 0 (or NaN)
  int v = __float_as_int(x);
  v = max(v, i8_dpp<0x111, 0xf>(v));
  v = max(v, i8_dpp<0x112, 0xf>(v));
  v = max(v, i8_dpp<0x114, 0xf>(v));
  v = max(v, i8_dpp<0x118, 0xf>(v));
  v = max(v, i8_dpp<0x142, 0xa>(v));
  v = max(v, i8_dpp<0x143, 0xc>(v));
  return __int_as_float(__builtin_amdgcn_readlane(v, kWave - 1));
}

}  // namespace ts
