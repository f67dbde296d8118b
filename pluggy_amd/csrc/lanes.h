// Reductions over a wave's lanes without LDS traffic: by DPP within 16 lanes, by
// lane swaps beyond (gfx950). At each step two halves that agree within themselves
// are joined, so every lane ends with the same bits, whatever the operation's
// rounding.
#pragma once

#include "common.h"

namespace pmoe {

// Lane l's value from another lane by a DPP control (quad permutation, row mirrors and rotations).
template <int CTRL>
__device__ __forceinline__ int dpp(int v) { return __builtin_amdgcn_mov_dpp(v, CTRL, 0xF, 0xF, true); }

// The two halves' values of an exchange between lanes 16 or 32 apart, in both.
__device__ __forceinline__ u32x2 swap16(int v) { return __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false); }
__device__ __forceinline__ u32x2 swap32(int v) { return __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false); }

// All-reduce over N consecutive lanes (a power of two) by `op`.
template <int N, class Op>
__device__ __forceinline__ int lanes_reduce(int v, Op op) {
  if constexpr (N >= 2) v = op(v, dpp<0xB1>(v));
  if constexpr (N >= 4) v = op(v, dpp<0x4E>(v));
  if constexpr (N >= 8) v = op(v, dpp<0x141>(v));   // lane i of 8 takes lane 7 - i
  if constexpr (N >= 16) v = op(v, dpp<0x140>(v));  // lane i of 16 takes lane 15 - i
  if constexpr (N >= 32) { const u32x2 r = swap16(v); v = op((int)r[0], (int)r[1]); }
  if constexpr (N >= 64) { const u32x2 r = swap32(v); v = op((int)r[0], (int)r[1]); }
  return v;
}

struct AddF {
  __device__ __forceinline__ int operator()(int a, int b) const {
    return __float_as_int(__int_as_float(a) + __int_as_float(b));
  }
};
struct AddI {
  __device__ __forceinline__ int operator()(int a, int b) const { return a + b; }
};

template <int N>
__device__ __forceinline__ float lanes_sum(float v) {
  return __int_as_float(lanes_reduce<N>(__float_as_int(v), AddF()));
}
template <int N>
__device__ __forceinline__ int lanes_sum(int v) { return lanes_reduce<N>(v, AddI()); }

// The sum over a wave's lanes l, l + N, l + 2 N, .. in lane l < N (N >= 4); order fixed.
template <int N, class Op>
__device__ __forceinline__ int lanes_across(int v, Op op) {
  static_assert(N >= 4, "groups of four lanes or more");
  if constexpr (N <= 8) v = op(v, dpp<0x128>(v));  // rotated by 8 of 16
  if constexpr (N <= 4) v = op(v, dpp<0x124>(v));
  if constexpr (N <= 16) { const u32x2 r = swap16(v); v = op((int)r[0], (int)r[1]); }
  if constexpr (N <= 32) { const u32x2 r = swap32(v); v = op((int)r[0], (int)r[1]); }
  return v;
}

}  // namespace pmoe
