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

// Magnitude of x for the group's maximum: 0 where x is not finite.
__device__ __forceinline__ float act8_mag(float x) {
  const uint32_t m = __float_as_uint(x) & 0x7fffffffu;
  return m < 0x7f800000u ? __uint_as_float(m) : 0.0f;
}

// Exponent byte of a group whose largest finite magnitude is a. With a = m 2^k,
// 1 <= m < 2: e = k - 6 takes a to [64, 128), and to 127.5 or more (which would
// round to 128) where m >= 1.9921875, i.e. from mantissa bits 0x7f0000 on, where
// adding 0x10000 carries into the exponent.
__device__ __forceinline__ uint32_t act8_exponent(float a) {
  return (uint32_t)max(1, (int)((__float_as_uint(a) + 0x10000u) >> 23) - 6);
}

__device__ __forceinline__ float act8_scale(uint32_t eb) { return __uint_as_float(eb << 23); }              // 2^e
__device__ __forceinline__ float act8_inv_scale(uint32_t eb) { return __uint_as_float((254u - eb) << 23); }  // 2^-e

__device__ __forceinline__ int act8_code(float x, float inv) {
  return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u ? -128 : (int)rintf(x * inv);
}

// Largest finite value of the type a checkpoint is restored to.
template <typename T> __device__ __forceinline__ float act8_limit();
template <> __device__ __forceinline__ float act8_limit<float>() { return 3.402823466e38f; }
template <> __device__ __forceinline__ float act8_limit<bf16_t>() { return 3.389531390e38f; }  // 0x7f7f
template <> __device__ __forceinline__ float act8_limit<f16_t>() { return 65504.0f; }

template <typename T>
__device__ __forceinline__ float act8_value(int code, float scale) {
  const float lim = act8_limit<T>();
  const float v = fminf(fmaxf((float)code * scale, -lim), lim);
  return code == -128 ? __uint_as_float(0x7fc00000u) : v;
}

// Eight codes in two dwords (code i in byte i).
__device__ __forceinline__ uint2 act8_pack(const float* v, float inv) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    w[h] = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[h] |= ((uint32_t)act8_code(v[4 * h + i], inv) & 0xffu) << (8 * i);
  }
  return make_uint2(w[0], w[1]);
}

template <typename T>
__device__ __forceinline__ void act8_unpack(uint2 w, float scale, float* v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = act8_value<T>((int)(int8_t)(w.x >> (8 * i)), scale);
    v[4 + i] = act8_value<T>((int)(int8_t)(w.y >> (8 * i)), scale);
  }
}

}  // namespace pmoe
