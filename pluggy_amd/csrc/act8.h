// Activations saved in 8 bits (activation checkpoints): the format.
//
// A row's columns are taken in groups of kAct8Group = 32 (the last group of a
// row may be shorter). With a the largest |x| of a group's finite values,
//   e = the least integer >= -126 with rint(a * 2^-e) <= 127,
//   code = rint(x * 2^-e) in [-127, 127] (ties to even), int8;
//   code = -128 for a value that is not finite;
//   the group's exponent byte is e + 127, in [1, 249].
// A code stands for code * 2^e, kept within the type's finite range (near the
// largest values the nearest multiple of 2^e can lie past it), and -128 for
// NaN. A power of two makes both the scaling and its inverse exact, so the one
// rounding is the code's: at most 2^(e-1), that is a / 127 at most (a / 255 at
// best). Every code * 2^e fits bf16's 8 significant bits, and fp16's except
// below its normal range. 32 columns: a row of a 32-column half of a gate_up
// wave tile, so that the GEMM epilogues have a whole group in four lanes.
#pragma once

#include "common.h"

namespace pmoe {

constexpr int kAct8Group = 32;

// Number of groups (exponent bytes) of a row of C columns.
__host__ __device__ inline int act8_groups(int C) { return (C + kAct8Group - 1) / kAct8Group; }

// Exponent byte of a group whose largest finite magnitude has the bits m. With a
// = f 2^k, 1 <= f < 2: e = k - 6 takes a to [64, 128), and to 127.5 or more (which
// would round to 128) where f >= 1.9921875, i.e. from mantissa bits 0x7f0000 on,
// where adding 0x10000 carries into the exponent.
__device__ __forceinline__ uint32_t act8_exponent(uint32_t m) { return (uint32_t)max(1, (int)((m + 0x10000u) >> 23) - 6); }

__device__ __forceinline__ float act8_scale(uint32_t eb) { return __uint_as_float(eb << 23); }              // 2^e
__device__ __forceinline__ float act8_inv_scale(uint32_t eb) { return __uint_as_float((254u - eb) << 23); }  // 2^-e

// The largest of four lanes' values (a group), in each of them (DPP quad permutations).
__device__ __forceinline__ uint32_t act8_quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));
}

constexpr uint32_t kAct8Inf = 0x7f800000u;

// Eight values' codes (code i in byte i) at 2^-e = inv, all of them finite: adding
// 1.5 * 2^23 to x 2^-e rounds it to a whole number, ties to even, and leaves that
// in the low byte.
__device__ __forceinline__ uint2 act8_codes(const float* v, float inv) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = __float_as_uint(__builtin_fmaf(v[4 * h + i], inv, 12582912.0f));
    const uint32_t lo = __builtin_amdgcn_perm(q[1], q[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(q[3], q[2], 0x0c0c0400u);
    w[h] = lo | (hi << 16);  // byte 0 of each
  }
  return make_uint2(w[0], w[1]);
}

// The same where some are not finite: a group's exponent from the finite ones, code -128 for the others.
__device__ __forceinline__ uint32_t act8_encode_some(const float* v, bool in, uint2& codes) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
    m = max(m, b < kAct8Inf ? b : 0u);
  }
  const uint32_t eb = act8_exponent(act8_quad_max(in ? m : 0u));
  const float inv = act8_inv_scale(eb);
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int q = (__float_as_uint(v[i]) & 0x7fffffffu) < kAct8Inf ? (int)rintf(v[i] * inv) : -128;
    w[i / 4] |= ((uint32_t)q & 0xffu) << (8 * (i & 3));
  }
  codes = make_uint2(w[0], w[1]);
  return eb;
}

// A lane's eight values of a group that four consecutive lanes hold (all of
// them call this; `in`: this lane's columns exist) -> their codes; returns the
// group's exponent byte.
__device__ __forceinline__ uint32_t act8_encode(const float* v, bool in, uint2& codes) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  m = act8_quad_max(in ? m : 0u);
  if (m >= kAct8Inf) return act8_encode_some(v, in, codes);
  const uint32_t eb = act8_exponent(m);
  codes = act8_codes(v, act8_inv_scale(eb));
  return eb;
}

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// The same from 16-bit values as they are stored: their magnitudes order like
// whole numbers, so the maximum is taken two at a time.
template <typename T>
__device__ __forceinline__ uint32_t act8_encode16(const u32x4& x, bool in, uint2& codes) {
  u16x2 m = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, x[i] & 0x7fff7fffu));
  const uint32_t top = act8_quad_max(in ? max((uint32_t)m[0], (uint32_t)m[1]) : 0u);  // the group's, 16 bits
  float v[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[2 * i] = Fmt16<T>::lo(x[i]); v[2 * i + 1] = Fmt16<T>::hi(x[i]); }
  const uint32_t a = __float_as_uint(Fmt16<T>::lo(top));
  if (a >= kAct8Inf) return act8_encode_some(v, in, codes);
  const uint32_t eb = act8_exponent(a);
  codes = act8_codes(v, act8_inv_scale(eb));
  return eb;
}

// The largest finite value of a type, and the exponent byte from which on 127 *
// 2^e can pass it.
template <typename T> struct Act8Range { static constexpr uint32_t large = 249; static constexpr float limit = 3.402823466e38f; };
template <> struct Act8Range<bf16_t> { static constexpr uint32_t large = 249; static constexpr float limit = 3.389531390e38f; };
template <> struct Act8Range<f16_t> { static constexpr uint32_t large = 137; static constexpr float limit = 65504.0f; };

// A word has a byte 0x80 (code -128).
__device__ __forceinline__ bool act8_has_nan(uint32_t w) {
  const uint32_t x = w ^ 0x80808080u;
  return ((x - 0x01010101u) & ~x & 0x80808080u) != 0u;
}

// The values of eight codes for type T.
template <typename T>
__device__ __forceinline__ void act8_decode(uint2 w, uint32_t eb, float* v) {
  const float scale = act8_scale(eb);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = (float)(int8_t)(w.x >> (8 * i)) * scale;
    v[4 + i] = (float)(int8_t)(w.y >> (8 * i)) * scale;
  }
  if (act8_has_nan(w.x) || act8_has_nan(w.y) || eb >= Act8Range<T>::large) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = (int)(int8_t)((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
      v[i] = c == -128 ? __uint_as_float(0x7fc00000u) : fminf(fmaxf(v[i], -Act8Range<T>::limit), Act8Range<T>::limit);
    }
  }
}

}  // namespace pmoe
