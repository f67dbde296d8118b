// Activations saved in 8 bits and read back (format: act8.h).
//
// Both are one pass over the tensor, bound by HBM: saving reads C elements and
// writes C codes and C / 32 exponents a row; restoring the reverse. A lane
// holds 8 consecutive columns (a 16-byte load of 16-bit values, an 8-byte store of
// codes), so a group of 32 is four lanes and its maximum two DPP steps. 65536 x 1536
// bf16, 305 MB each way: saving 57 us, restoring 64, 5.4 and 4.8 TB/s, what a large
// copy reaches (5.1). Stores stay cached: non-temporal ones restore faster in a row
// (67 -> 47), but whatever reads the result next pays for it (96 MB, restoring and
// then reading: 38 + 31 us cached, 35 + 52 not). The MoE's own checkpoint needs
// neither launch: the GEMM epilogues write and read the codes (gemm_persist.h).
#include "act8.h"
#include "kernels.h"

namespace pmoe {
namespace {

// Columns c .. c+7 of a row of C, zero past its end. VEC: rows are whole 16-byte
// pieces (C a multiple of 8, 16-byte aligned); otherwise a row's pieces are read and
// written where they lie, and its last one element by element where it is cut.
// 65536 x 1536 bf16 53 us saving and 66 restoring, x 1535 85 and 94 (x 1001: 32 and 31).
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* row, int c, int C, float* v) {
  if constexpr (VEC) {
    Vec8<T>::load(row + c, v);
  } else if (c + 8 <= C) {
    load8_loose<T>(row + c, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < C ? load_scalar<T>(row + c + i) : 0.0f;
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* row, int c, int C, const float* v) {
  if constexpr (VEC) {
    Vec8<T>::store(row + c, v);
  } else if (c + 8 <= C) {
    store8_loose<T>(row + c, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < C) store_scalar<T>(row + c + i, v[i]);
  }
}

typedef u32x2 u32x2_by1 __attribute__((aligned(1)));

template <bool VEC>
__device__ __forceinline__ uint2 load_codes(const int8_t* row, int c, int C) {
  if constexpr (VEC) {
    return *reinterpret_cast<const uint2*>(row + c);
  } else if (c + 8 <= C) {
    const u32x2 w = *reinterpret_cast<const u32x2_by1*>(row + c);
    return make_uint2(w[0], w[1]);
  } else {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < C) w[i / 4] |= ((uint32_t)(uint8_t)row[c + i]) << (8 * (i % 4));
    return make_uint2(w[0], w[1]);
  }
}

template <bool VEC>
__device__ __forceinline__ void store_codes(int8_t* row, int c, int C, uint2 w) {
  if constexpr (VEC) {
    *reinterpret_cast<uint2*>(row + c) = w;
  } else if (c + 8 <= C) {
    *reinterpret_cast<u32x2_by1*>(row + c) = u32x2{w.x, w.y};
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (c + k < C) row[c + k] = (int8_t)((k < 4 ? w.x : w.y) >> (8 * (k % 4)));
  }
}

// One thread per 8 columns, groups padded to four threads: thread i of the
// grid holds columns 8 (i % W) .. of row i / W, W = 4 * groups.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void act8_save_kernel(const T* __restrict__ x, int64_t R, int C, int G,
                                                        int8_t* __restrict__ codes, uint8_t* __restrict__ exps) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t r = i / (4 * G);
  const int c = (int)(i - r * (4 * G)) * 8;
  const bool in = r < R && c < C;
  float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (in) load8<T, VEC>(x + r * C, c, C, v);
  uint2 w;
  const uint32_t eb = act8_encode(v, in, w);
  if (!in) return;
  store_codes<VEC>(codes + r * C, c, C, w);
  if (c % kAct8Group == 0) exps[r * G + c / kAct8Group] = (uint8_t)eb;
}

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void act8_restore_kernel(const int8_t* __restrict__ codes,
                                                           const uint8_t* __restrict__ exps, int64_t R, int C, int G,
                                                           T* __restrict__ x) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t r = i / (4 * G);
  const int c = (int)(i - r * (4 * G)) * 8;
  if (r >= R || c >= C) return;
  float v[8];
  act8_decode<T>(load_codes<VEC>(codes + r * C, c, C), exps[r * G + c / kAct8Group], v);
  store8<T, VEC>(x + r * C, c, C, v);
}

// gate_up rows (P, 2I) from their checkpoint, and mid = w * silu(gate) * up of
// the restored values: what the forward saved and what it computed from it.
// I is a multiple of 8, so rows are whole 16-byte pieces.
template <typename T>
__global__ __launch_bounds__(256) void act8_restore_swiglu_kernel(const int8_t* __restrict__ codes,
                                                                  const uint8_t* __restrict__ exps,
                                                                  const float* __restrict__ row_w, int64_t P, int I,
                                                                  int G, T* __restrict__ gu, T* __restrict__ mid) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t r = i / (I / 8);
  if (r >= P) return;
  const int c = (int)(i - r * (I / 8)) * 8;
  const int8_t* row = codes + r * 2 * I;
  const uint8_t* er = exps + r * 2 * G + c / kAct8Group;
  float g[8], u[8], m[8];
  act8_decode<T>(load_codes<true>(row, c, I), er[0], g);
  act8_decode<T>(load_codes<true>(row + I, c, I), er[G], u);
  const float w = row_w != nullptr ? row_w[r] : 1.0f;
#pragma unroll
  for (int k = 0; k < 8; ++k) m[k] = g[k] * (sizeof(T) == 2 ? fast_sigmoid(g[k]) : sigmoidf_(g[k])) * u[k] * w;
  Vec8<T>::store(gu + r * 2 * I + c, g);
  Vec8<T>::store(gu + r * 2 * I + I + c, u);
  Vec8<T>::store(mid + r * I + c, m);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Threads of the grid that act8_save / act8_restore walk; the caller has checked that the blocks fit a launch.
unsigned blocks_of(int64_t threads) { return (unsigned)((threads + 255) / 256); }

}  // namespace

template <typename T>
hipError_t act8_save(const T* x, int64_t R, int C, int8_t* codes, uint8_t* exps, hipStream_t s) {
  const int G = act8_groups(C);
  const unsigned nb = blocks_of(R * 4 * G);
  if (nb == 0) return hipSuccess;
  if (C % 8 == 0 && aligned16(x) && reinterpret_cast<uintptr_t>(codes) % 8 == 0)
    hipLaunchKernelGGL((act8_save_kernel<T, true>), dim3(nb), dim3(256), 0, s, x, R, C, G, codes, exps);
  else
    hipLaunchKernelGGL((act8_save_kernel<T, false>), dim3(nb), dim3(256), 0, s, x, R, C, G, codes, exps);
  return hipGetLastError();
}

template <typename T>
hipError_t act8_restore(const int8_t* codes, const uint8_t* exps, int64_t R, int C, T* x, hipStream_t s) {
  const int G = act8_groups(C);
  const unsigned nb = blocks_of(R * 4 * G);
  if (nb == 0) return hipSuccess;
  if (C % 8 == 0 && aligned16(x) && reinterpret_cast<uintptr_t>(codes) % 8 == 0)
    hipLaunchKernelGGL((act8_restore_kernel<T, true>), dim3(nb), dim3(256), 0, s, codes, exps, R, C, G, x);
  else
    hipLaunchKernelGGL((act8_restore_kernel<T, false>), dim3(nb), dim3(256), 0, s, codes, exps, R, C, G, x);
  return hipGetLastError();
}

template <typename T>
hipError_t act8_restore_swiglu(const int8_t* codes, const uint8_t* exps, const float* row_w, int64_t P, int I, T* gu,
                               T* mid, hipStream_t s) {
  const unsigned nb = blocks_of(P * (I / 8));
  if (nb == 0) return hipSuccess;
  hipLaunchKernelGGL((act8_restore_swiglu_kernel<T>), dim3(nb), dim3(256), 0, s, codes, exps, row_w, P, I,
                     act8_groups(I), gu, mid);
  return hipGetLastError();
}

#define PMOE_INST_ACT8(T)                                                                                          \
  template hipError_t act8_save<T>(const T*, int64_t, int, int8_t*, uint8_t*, hipStream_t);                         \
  template hipError_t act8_restore<T>(const int8_t*, const uint8_t*, int64_t, int, T*, hipStream_t);                \
  template hipError_t act8_restore_swiglu<T>(const int8_t*, const uint8_t*, const float*, int64_t, int, T*, T*,     \
                                             hipStream_t);
PMOE_INST_ACT8(float)
PMOE_INST_ACT8(bf16_t)
PMOE_INST_ACT8(f16_t)

}  // namespace pmoe
