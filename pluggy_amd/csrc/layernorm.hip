// Layer norm over the last dimension, forward and backward.
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) r
//   y = xh w + b
//   gx = r (g w - mean(g w) - xh mean(g w xh)),  gw = sum_t g xh,  gb = sum_t g
//
// Both directions are bound by HBM: the forward reads x and writes y, the
// backward reads x and g and writes gx. Rows are held in registers (the
// variance is the mean of squared differences from the mean, not a difference
// of two large sums), fp32 arithmetic; a row belongs to one wave up to 2048
// columns, to a block of four waves up to 16384, and wider rows are walked by a
// block in passes. Sums run in a fixed order, so results are deterministic.
#include "kernels.h"

namespace pmoe {
namespace {

constexpr int kLnBlock = 256;       // threads of a block
constexpr int kLnWaveH = 2048;      // widest row of one wave
constexpr int kLnRegH = 16384;      // widest row held in registers
constexpr int kLnMaxBlocks = 1024;  // blocks (partial rows) of the backward
constexpr int kLnColRows = 256;     // rows of a block of the wide rows' column sums

__host__ __device__ inline int64_t ln_pad(int64_t H) { return (H + 31) / 32 * 32; }

// The norm's weight or bias at a column, in any of the three types; null: `none`.
__device__ __forceinline__ float param(const void* p, int code, int c, float none) {
  if (p == nullptr) return none;
  if (code == 0) return static_cast<const float*>(p)[c];
  if (code == 1) return bf16_to_f32(static_cast<const bf16_t*>(p)[c]);
  return (float)static_cast<const f16_t*>(p)[c];
}

__device__ __forceinline__ void param8(const void* p, int code, int c, float none, float* v) {
  if (p == nullptr) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = none;
  } else if (code == 0) {
    Vec8<float>::load(static_cast<const float*>(p) + c, v);
  } else if (code == 1) {
    Vec8<bf16_t>::load(static_cast<const bf16_t*>(p) + c, v);
  } else {
    Vec8<f16_t>::load(static_cast<const f16_t*>(p) + c, v);
  }
}

// The columns of a thread: NCH chunks of 8. VEC: 8 consecutive columns, read
// and written as 16-byte pieces (rows start on 16 bytes, H a multiple of 8);
// otherwise one column every TPR threads, so that a wave's accesses are consecutive.
template <int TPR, int NCH, bool VEC>
struct Cols {
  __device__ static __forceinline__ int at(int t, int i, int e) {
    return VEC ? (i * TPR + t) * 8 + e : (i * 8 + e) * TPR + t;
  }
  __device__ static __forceinline__ bool in(int t, int i, int e, int H) { return at(t, i, VEC ? 0 : e) < H; }
  template <typename T>
  __device__ static __forceinline__ void load(const T* row, int t, int H, float (&v)[NCH][8]) {
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = 0.0f;
      if constexpr (VEC) {
        if (at(t, i, 0) < H) Vec8<T>::load(row + at(t, i, 0), v[i]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (at(t, i, e) < H) v[i][e] = load_scalar<T>(row + at(t, i, e));
      }
    }
  }
  template <typename T>
  __device__ static __forceinline__ void store(T* row, int t, int i, int H, const float* v) {
    if constexpr (VEC) {
      if (at(t, i, 0) < H) Vec8<T>::store(row + at(t, i, 0), v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (at(t, i, e) < H) store_scalar<T>(row + at(t, i, e), v[e]);
    }
  }
  __device__ static __forceinline__ void params(const void* p, int code, float none, int t, int i, int H, float* v) {
    if constexpr (VEC) {
      if (at(t, i, 0) < H) param8(p, code, at(t, i, 0), none, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = at(t, i, e) < H ? param(p, code, at(t, i, e), none) : 0.0f;
    }
  }
};

// The sum of one value over the WPR waves of a row, in every thread of it.
// One barrier a call; calls take turns with the two halves of `s`.
template <int WPR>
__device__ __forceinline__ float row_sum(float v, float (*s)[WPR], int turn) {
  v = wave_sum(v);
  if constexpr (WPR == 1) return v;
  if ((threadIdx.x & 63) == 0) s[turn & 1][threadIdx.x >> 6] = v;
  __syncthreads();
  float a = s[turn & 1][0];
#pragma unroll
  for (int k = 1; k < WPR; ++k) a += s[turn & 1][k];
  return a;
}

template <typename TX, typename TO, int WPR, int NCH, bool VEC>
__global__ __launch_bounds__(kLnBlock) void layernorm_fwd_kernel(const TX* __restrict__ x, const void* __restrict__ w,
                                                                 const void* __restrict__ b, int w_code, float eps,
                                                                 int64_t T_, int H, TO* __restrict__ out,
                                                                 float* __restrict__ mean, float* __restrict__ rstd) {
  constexpr int TPR = kWave * WPR, RPB = kLnBlock / TPR;
  typedef Cols<TPR, NCH, VEC> C;
  __shared__ float s_sum[2][WPR];
  const int t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
  if (row >= T_) return;  // WPR 4: the whole block; WPR 1: no barrier follows
  float v[NCH][8];
  C::load(x + row * H, t, H, v);
  float a = 0.0f;
#pragma unroll
  for (int i = 0; i < NCH; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) a += v[i][e];
  const float mu = row_sum<WPR>(a, s_sum, 0) / (float)H;
  a = 0.0f;
#pragma unroll
  for (int i = 0; i < NCH; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[i][e] -= mu;
      if (C::in(t, i, e, H)) a += v[i][e] * v[i][e];
    }
  const float r = 1.0f / sqrtf(row_sum<WPR>(a, s_sum, 1) / (float)H + eps);
  if (t == 0 && mean != nullptr) {
    mean[row] = mu;
    rstd[row] = r;
  }
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    float wv[8], bv[8];
    C::params(w, w_code, 1.0f, t, i, H, wv);
    C::params(b, w_code, 0.0f, t, i, H, bv);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[i][e] = (v[i][e] * r) * wv[e] + bv[e];
    C::store(out + row * H, t, i, H, v[i]);
  }
}

// gx, and this block's sums of g xh and g over its rows: partial rows
// part[2 blockIdx.x] and part[2 blockIdx.x + 1] of ld columns (part null: not wanted).
template <typename TX, typename TG, int WPR, int NCH, bool VEC>
__global__ __launch_bounds__(kLnBlock) void layernorm_bwd_kernel(const TG* __restrict__ g, const TX* __restrict__ x,
                                                                 const void* __restrict__ w, int w_code,
                                                                 const float* __restrict__ mean,
                                                                 const float* __restrict__ rstd, int64_t T_, int H,
                                                                 TX* __restrict__ gx, float* __restrict__ part,
                                                                 int64_t ld) {
  constexpr int TPR = kWave * WPR, RPB = kLnBlock / TPR;
  typedef Cols<TPR, NCH, VEC> C;
  __shared__ float s_a[2][WPR], s_b[2][WPR];
  __shared__ float s_part[WPR == 1 ? 3 : 1][WPR == 1 ? TPR * 8 * NCH : 1];
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  float gw[NCH][8], gb[NCH][8];
#pragma unroll
  for (int i = 0; i < NCH; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) gw[i][e] = gb[i][e] = 0.0f;
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * RPB + sub; row < T_; row += (int64_t)gridDim.x * RPB, ++turn) {
    float xv[NCH][8], gv[NCH][8];
    C::load(x + row * H, t, H, xv);
    C::load(g + row * H, t, H, gv);
    const float mu = mean[row], r = rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      float wv[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      C::params(w, w_code, 1.0f, t, i, H, wv);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float xh = (xv[i][e] - mu) * r, ge = gv[i][e];
        xv[i][e] = xh;
        gb[i][e] += ge;
        gw[i][e] += C::in(t, i, e, H) ? ge * xh : 0.0f;
        gv[i][e] = ge * wv[e];
        s1 += gv[i][e];
        s2 += C::in(t, i, e, H) ? gv[i][e] * xh : 0.0f;
      }
    }
    if (gx != nullptr) {  // uniform over the grid
      s1 = row_sum<WPR>(s1, s_a, turn);
      s2 = row_sum<WPR>(s2, s_b, turn);
      const float c1 = s1 / (float)H, c2 = s2 / (float)H;
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
#pragma unroll
        for (int e = 0; e < 8; ++e) gv[i][e] = r * (gv[i][e] - c1 - xv[i][e] * c2);
        C::store(gx + row * H, t, i, H, gv[i]);
      }
    }
  }
  if (part == nullptr) return;  // uniform over the grid
  // WPR 1: the block's four waves hold the same columns; summed in wave order
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float(&acc)[NCH][8] = which == 0 ? gw : gb;
    if constexpr (WPR == 1) {
      if (sub > 0)
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) s_part[sub - 1][(i * 8 + e) * TPR + t] = acc[i][e];
      __syncthreads();
      if (sub == 0)
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int k = (i * 8 + e) * TPR + t;
            acc[i][e] = ((acc[i][e] + s_part[0][k]) + s_part[1][k]) + s_part[2][k];
          }
      __syncthreads();
    }
    if (WPR > 1 || sub == 0) {
      float* row = part + (2 * (int64_t)blockIdx.x + which) * ld;
#pragma unroll
      for (int i = 0; i < NCH; ++i) C::store(row, t, i, H, acc[i]);
    }
  }
}

// Rows wider than kLnRegH: a block a row, in passes over it.
template <typename TX, typename TO>
__global__ __launch_bounds__(kLnBlock) void layernorm_fwd_wide_kernel(const TX* __restrict__ x,
                                                                      const void* __restrict__ w,
                                                                      const void* __restrict__ b, int w_code,
                                                                      float eps, int H, TO* __restrict__ out,
                                                                      float* __restrict__ mean,
                                                                      float* __restrict__ rstd) {
  __shared__ float s_sum[2][4];
  const int64_t row = blockIdx.x;
  const TX* xr = x + row * H;
  float a = 0.0f;
  for (int c = threadIdx.x; c < H; c += kLnBlock) a += load_scalar<TX>(xr + c);
  const float mu = row_sum<4>(a, s_sum, 0) / (float)H;
  a = 0.0f;
  for (int c = threadIdx.x; c < H; c += kLnBlock) {
    const float d = load_scalar<TX>(xr + c) - mu;
    a += d * d;
  }
  const float r = 1.0f / sqrtf(row_sum<4>(a, s_sum, 1) / (float)H + eps);
  if (threadIdx.x == 0 && mean != nullptr) {
    mean[row] = mu;
    rstd[row] = r;
  }
  for (int c = threadIdx.x; c < H; c += kLnBlock)
    store_scalar<TO>(out + row * H + c, ((load_scalar<TX>(xr + c) - mu) * r) * param(w, w_code, c, 1.0f) +
                                            param(b, w_code, c, 0.0f));
}

template <typename TX, typename TG>
__global__ __launch_bounds__(kLnBlock) void layernorm_bwd_wide_kernel(const TG* __restrict__ g,
                                                                      const TX* __restrict__ x,
                                                                      const void* __restrict__ w, int w_code,
                                                                      const float* __restrict__ mean,
                                                                      const float* __restrict__ rstd, int H,
                                                                      TX* __restrict__ gx) {
  __shared__ float s_a[2][4], s_b[2][4];
  const int64_t row = blockIdx.x;
  const float mu = mean[row], r = rstd[row];
  float s1 = 0.0f, s2 = 0.0f;
  for (int c = threadIdx.x; c < H; c += kLnBlock) {
    const float gv = load_scalar<TG>(g + row * H + c) * param(w, w_code, c, 1.0f);
    s1 += gv;
    s2 += gv * ((load_scalar<TX>(x + row * H + c) - mu) * r);
  }
  const float c1 = row_sum<4>(s1, s_a, 0) / (float)H, c2 = row_sum<4>(s2, s_b, 0) / (float)H;
  for (int c = threadIdx.x; c < H; c += kLnBlock) {
    const float gv = load_scalar<TG>(g + row * H + c) * param(w, w_code, c, 1.0f);
    const float xh = (load_scalar<TX>(x + row * H + c) - mu) * r;
    store_scalar<TX>(gx + row * H + c, r * (gv - c1 - xh * c2));
  }
}

// The wide rows' partial column sums: block (column strip, row chunk), one thread a column.
template <typename TX, typename TG>
__global__ __launch_bounds__(kLnBlock) void layernorm_cols_kernel(const TG* __restrict__ g, const TX* __restrict__ x,
                                                                  const float* __restrict__ mean,
                                                                  const float* __restrict__ rstd, int64_t T_, int H,
                                                                  int64_t rows, float* __restrict__ part, int64_t ld) {
  const int c = blockIdx.x * kLnBlock + threadIdx.x;
  if (c >= H) return;
  const int64_t r0 = blockIdx.y * rows, r1 = min(r0 + rows, T_);
  float gw = 0.0f, gb = 0.0f;
  for (int64_t t = r0; t < r1; ++t) {
    const float gv = load_scalar<TG>(g + t * H + c);
    gw += gv * ((load_scalar<TX>(x + t * H + c) - mean[t]) * rstd[t]);
    gb += gv;
  }
  part[(2 * (int64_t)blockIdx.y) * ld + c] = gw;
  part[(2 * (int64_t)blockIdx.y + 1) * ld + c] = gb;
}

// gw, gb = the sums of nb partial rows each, in a fixed order: 32 columns a
// block (a lane has four), 32 groups of rows summed through LDS. No rows: zeros.
__global__ __launch_bounds__(256) void layernorm_reduce_kernel(const float* __restrict__ part, int nb, int64_t ld,
                                                               int H, void* __restrict__ gw, void* __restrict__ gb,
                                                               int w_code) {
  __shared__ f32x4 s[32][8];
  const int which = blockIdx.y, q = threadIdx.x % 8, grp = threadIdx.x / 8;
  const int c = blockIdx.x * 32 + q * 4;
  void* out = which == 0 ? gw : gb;
  if (out == nullptr) return;  // uniform over the block
  f32x4 a = {0, 0, 0, 0};
  for (int b = grp; b < nb; b += 32) a += *reinterpret_cast<const f32x4*>(part + (2 * (int64_t)b + which) * ld + c);
  s[grp][q] = a;
  __syncthreads();
  if (threadIdx.x >= 32) return;
  const int col = blockIdx.x * 32 + threadIdx.x;
  if (col >= H) return;
  float v = 0.0f;
  for (int k = 0; k < 32; ++k) v += s[k][threadIdx.x / 4][threadIdx.x % 4];
  if (w_code == 0) static_cast<float*>(out)[col] = v;
  else if (w_code == 1) static_cast<bf16_t*>(out)[col] = f32_to_bf16(v);
  else static_cast<f16_t*>(out)[col] = (f16_t)v;
}

bool all16(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
  return true;
}

// Calls f(waves a row, chunks a thread) for a row of H <= kLnRegH columns.
template <class F>
hipError_t by_width(int H, F&& f) {
  using std::integral_constant;
  if (H <= 512) return f(integral_constant<int, 1>(), integral_constant<int, 1>());
  if (H <= 1024) return f(integral_constant<int, 1>(), integral_constant<int, 2>());
  if (H <= kLnWaveH) return f(integral_constant<int, 1>(), integral_constant<int, 4>());
  if (H <= 4096) return f(integral_constant<int, 4>(), integral_constant<int, 2>());
  if (H <= 8192) return f(integral_constant<int, 4>(), integral_constant<int, 4>());
  return f(integral_constant<int, 4>(), integral_constant<int, 8>());
}

int rows_a_block(int H) { return H <= kLnWaveH ? 4 : 1; }
int64_t wide_rows(int64_t T_) { return std::max<int64_t>(kLnColRows, (T_ + kLnMaxBlocks - 1) / kLnMaxBlocks); }

}  // namespace

int layernorm_bwd_blocks(int64_t T_, int H) {
  if (T_ <= 0) return 0;
  if (H > kLnRegH) return (int)((T_ + wide_rows(T_) - 1) / wide_rows(T_));
  const int rpb = rows_a_block(H);
  return (int)std::min<int64_t>((T_ + 2 * rpb - 1) / (2 * rpb), kLnMaxBlocks);
}

int64_t layernorm_part_ld(int H) { return ln_pad(H); }

template <typename TX, typename TO>
hipError_t layernorm_fwd(const TX* x, const void* w, const void* b, int w_code, float eps, int64_t T_, int H, TO* out,
                         float* mean, float* rstd, hipStream_t s) {
  if (T_ == 0) return hipSuccess;
  if (H > kLnRegH) {
    hipLaunchKernelGGL((layernorm_fwd_wide_kernel<TX, TO>), dim3((unsigned)T_), dim3(kLnBlock), 0, s, x, w, b, w_code,
                       eps, H, out, mean, rstd);
    return hipGetLastError();
  }
  const bool vec = H % 8 == 0 && all16({x, w, b, out});
  return by_width(H, [&](auto wpr, auto nch) {
    constexpr int WPR = decltype(wpr)::value, NCH = decltype(nch)::value, RPB = 4 / WPR;
    const dim3 grid((unsigned)((T_ + RPB - 1) / RPB));
    if (vec)
      hipLaunchKernelGGL((layernorm_fwd_kernel<TX, TO, WPR, NCH, true>), grid, dim3(kLnBlock), 0, s, x, w, b, w_code,
                         eps, T_, H, out, mean, rstd);
    else
      hipLaunchKernelGGL((layernorm_fwd_kernel<TX, TO, WPR, NCH, false>), grid, dim3(kLnBlock), 0, s, x, w, b, w_code,
                         eps, T_, H, out, mean, rstd);
    return hipGetLastError();
  });
}

template <typename TX, typename TG>
hipError_t layernorm_bwd(const TG* g, const TX* x, const void* w, int w_code, const float* mean, const float* rstd,
                         int64_t T_, int H, TX* gx, float* part, void* gw, void* gb, hipStream_t s) {
  const int nb = layernorm_bwd_blocks(T_, H);
  const int64_t ld = layernorm_part_ld(H);
  hipError_t st = hipSuccess;
  if (T_ > 0 && H > kLnRegH) {
    if (gx != nullptr)
      hipLaunchKernelGGL((layernorm_bwd_wide_kernel<TX, TG>), dim3((unsigned)T_), dim3(kLnBlock), 0, s, g, x, w,
                         w_code, mean, rstd, H, gx);
    if (part != nullptr)
      hipLaunchKernelGGL((layernorm_cols_kernel<TX, TG>), dim3((H + kLnBlock - 1) / kLnBlock, nb), dim3(kLnBlock), 0,
                         s, g, x, mean, rstd, T_, H, wide_rows(T_), part, ld);
    st = hipGetLastError();
  } else if (T_ > 0) {
    const bool vec = H % 8 == 0 && all16({g, x, w, gx, part});
    st = by_width(H, [&](auto wpr, auto nch) {
      constexpr int WPR = decltype(wpr)::value, NCH = decltype(nch)::value;
      if (vec)
        hipLaunchKernelGGL((layernorm_bwd_kernel<TX, TG, WPR, NCH, true>), dim3(nb), dim3(kLnBlock), 0, s, g, x, w,
                           w_code, mean, rstd, T_, H, gx, part, ld);
      else
        hipLaunchKernelGGL((layernorm_bwd_kernel<TX, TG, WPR, NCH, false>), dim3(nb), dim3(kLnBlock), 0, s, g, x, w,
                           w_code, mean, rstd, T_, H, gx, part, ld);
      return hipGetLastError();
    });
  }
  if (st != hipSuccess || (gw == nullptr && gb == nullptr)) return st;
  hipLaunchKernelGGL(layernorm_reduce_kernel, dim3((H + 31) / 32, 2), dim3(256), 0, s, part, nb, ld, H, gw, gb, w_code);
  return hipGetLastError();
}

// Element types: x and y (or its gradient) alike, or fp32 x with a 16-bit y (a
// norm that feeds 16-bit products from an fp32 stream).
#define PMOE_INST_LN(TX, TO)                                                                                        \
  template hipError_t layernorm_fwd<TX, TO>(const TX*, const void*, const void*, int, float, int64_t, int, TO*,     \
                                            float*, float*, hipStream_t);                                           \
  template hipError_t layernorm_bwd<TX, TO>(const TO*, const TX*, const void*, int, const float*, const float*,     \
                                            int64_t, int, TX*, float*, void*, void*, hipStream_t);
PMOE_INST_LN(float, float)
PMOE_INST_LN(float, bf16_t)
PMOE_INST_LN(float, f16_t)
PMOE_INST_LN(bf16_t, bf16_t)
PMOE_INST_LN(f16_t, f16_t)

}  // namespace pmoe
