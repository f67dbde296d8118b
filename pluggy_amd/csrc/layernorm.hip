// Layer norm over the last dimension, forward and backward.
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) r
//   y = xh w + b
//   gx = r (g w - mean(g w) - xh mean(g w xh)),  gw = sum_t g xh,  gb = sum_t g
//
// Both directions are bound by HBM: the forward reads x and writes y, the
// backward reads x and g and writes gx. Rows are held in registers (the
// variance is the mean of squared differences from the mean, not a difference
// of two large sums), fp32 arithmetic; a row belongs to one wave, or to two, four or
// eight up to 16384 columns, and wider rows are walked by a block in passes. Sums
// run in a fixed order, so results are deterministic.
#include "kernels.h"
#include "lanes.h"

namespace pmoe {
namespace {

constexpr int kLnBlock = 512;       // threads of a block
constexpr int kLnRegH = 16384;      // widest row held in registers
constexpr int kLnMaxBlocks = 256;   // blocks (partial rows) of the backward: one a compute unit, ...
constexpr int kLnTwoH = 2048;       // ... two for 16-bit rows up to this width
constexpr int kLnFwdBlocks = 768;   // most blocks of the forward: three a compute unit
constexpr int kLnColBlocks = 1024;  // most row chunks of the wide rows' column sums, ...
constexpr int kLnColRows = 256;     // each of at least so many rows

__host__ __device__ inline int64_t ln_pad(int64_t H) { return (H + 31) / 32 * 32; }

// The norm's weight or bias at a column, in any of the three types; null: `none`.
__device__ __forceinline__ float param(const void* p, int code, int c, float none) {
  if (p == nullptr) return none;
  if (code == 0) return static_cast<const float*>(p)[c];
  if (code == 1) return bf16_to_f32(static_cast<const bf16_t*>(p)[c]);
  return (float)static_cast<const f16_t*>(p)[c];
}

// Eight of them from column c on; LOOSE: at any element's alignment.
template <bool LOOSE>
__device__ __forceinline__ void param8(const void* p, int code, int c, float none, float* v) {
  if (p == nullptr) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = none;
  } else if (code == 0) {
    typedef std::conditional_t<LOOSE, u32x4_by4, u32x4> P;
    const P* q = reinterpret_cast<const P*>(static_cast<const float*>(p) + c);
    const u32x4 lo = q[0], hi = q[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[e] = __uint_as_float(lo[e]); v[4 + e] = __uint_as_float(hi[e]); }
  } else {
    typedef std::conditional_t<LOOSE, u32x4_by2, u32x4> P;
    const u32x4 w = *reinterpret_cast<const P*>(static_cast<const bf16_t*>(p) + c);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = code == 1 ? bf16lo(w[e]) : f16lo(w[e]);
      v[2 * e + 1] = code == 1 ? bf16hi(w[e]) : f16hi(w[e]);
    }
  }
}

// The columns of a thread: NCH chunks of 8 consecutive ones, TPR threads apart.
// VEC: rows are whole 16-byte pieces (they start on 16 bytes, H a multiple of 8).
// Otherwise chunks are read and written as 16-byte pieces where they lie, and the
// row's last one element by element where it is cut.
template <int TPR, int NCH, bool VEC>
struct Cols {
  __device__ static __forceinline__ int at(int t, int i) { return (i * TPR + t) * 8; }
  __device__ static __forceinline__ bool in(int t, int i, int e, int H) { return at(t, i) + (VEC ? 0 : e) < H; }
  template <typename T>
  __device__ static __forceinline__ void store(T* row, int t, int i, int H, const float* v) {
    const int c = at(t, i);
    if (c >= H) return;
    if constexpr (VEC) {
      Vec8<T>::store(row + c, v);
    } else if (c + 8 <= H) {
      store8_loose<T>(row + c, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < H) store_scalar<T>(row + c + e, v[e]);
    }
  }
  __device__ static __forceinline__ void params(const void* p, int code, float none, int t, int i, int H, float* v) {
    const int c = at(t, i);
    if (c + (VEC ? 0 : 7) < H) {
      param8<!VEC>(p, code, c, none, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = c + e < H ? param(p, code, c + e, none) : 0.0f;
    }
  }
  // A row's chunks as read, to be unpacked when they are used. The one that the row's
  // end cuts is read as the row's last 8 elements and moved down then, so that no
  // load is waited for before its use. Against reading it element by element, bf16,
  // forward and backward: 32768 x 511 20 + 39 -> 18 + 28 us, 8192 x 2001 13.5 + 25 ->
  // 16 + 24.5, 8192 x 6001 45 + 113 -> 45 + 72, 4096 x 16383 71 + 148 -> 60 + 109.
  template <typename T> struct Raw {
    static constexpr int PIECES = (int)sizeof(T) / 2, PER = 16 / (int)sizeof(T);  // 16-byte pieces a chunk, elements a piece
    u32x4 p[NCH][PIECES];
    __device__ __forceinline__ void load(const T* row, int t, int H) {
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const int c = at(t, i);
#pragma unroll
        for (int k = 0; k < PIECES; ++k) p[i][k] = u32x4{0, 0, 0, 0};
        if (c >= H) continue;
        if constexpr (VEC) {
#pragma unroll
          for (int k = 0; k < PIECES; ++k) p[i][k] = *reinterpret_cast<const u32x4*>(row + c + k * PER);
        } else if (c + 8 <= H) {
#pragma unroll
          for (int k = 0; k < PIECES; ++k)
            p[i][k] = *reinterpret_cast<const typename Loose<T>::type*>(row + c + k * PER);
        } else if (H >= 8) {
#pragma unroll
          for (int k = 0; k < PIECES; ++k)
            p[i][k] = *reinterpret_cast<const typename Loose<T>::type*>(row + H - 8 + k * PER);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (c + e >= H) continue;
            if constexpr (sizeof(T) == 4)
              p[i][e / 4][e % 4] = __float_as_uint((float)row[c + e]);
            else
              p[i][0][e / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, row[c + e]) << (16 * (e % 2));
          }
        }
      }
    }
    __device__ __forceinline__ void unpack(int t, int H, float (&v)[NCH][8]) const {
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if constexpr (sizeof(T) == 4) v[i][e] = __uint_as_float(p[i][e / 4][e % 4]);
          else v[i][e] = e % 2 ? Fmt16<T>::hi(p[i][0][e / 2]) : Fmt16<T>::lo(p[i][0][e / 2]);
        }
        const int c = at(t, i), down = c + 8 - H;
        if (!VEC && H >= 8 && c < H && down > 0) {
#pragma unroll
          for (int by = 4; by > 0; by /= 2)
            if (down & by)
#pragma unroll
              for (int e = 0; e < 8; ++e) v[i][e] = e + by < 8 ? v[i][e + by] : 0.0f;
        }
      }
    }
  };
};

// The sums of M values over the WPR waves of a row, in every thread of it. One
// barrier of the block a call where WPR > 1; calls take turns with the halves of `s`.
template <int WPR, int M>
__device__ __forceinline__ void row_sums(float (&v)[M], float (*s)[kLnBlock / kWave][M], int turn) {
#pragma unroll
  for (int m = 0; m < M; ++m) v[m] = lanes_sum<kWave>(v[m]);
  if constexpr (WPR > 1) {
    const int wave = threadIdx.x >> 6, first = wave / WPR * WPR;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int m = 0; m < M; ++m) s[turn & 1][wave][m] = v[m];
    __syncthreads();
#pragma unroll
    for (int m = 0; m < M; ++m) {
      v[m] = s[turn & 1][first][m];
#pragma unroll
      for (int k = 1; k < WPR; ++k) v[m] += s[turn & 1][first + k][m];
    }
  }
}

// Rows blockIdx.x * RPB + sub, + gridDim.x * RPB, ..: the weight and the bias stay
// in registers. (Read from L1 for every row they are four times a bf16 row's
// bytes.) Two chunks a thread leave room for four waves a SIMD, which cover each
// other's loads; four chunks (the widest rows) for two, and there the next row is
// on its way while a row is worked on. 8192 x 2048 bf16: 14.4 us, 67 MB at 4.7 TB/s;
// 16384 x 4096: 49 us, 268 MB at 5.4; 1531 x 1001 fp32: 6.3 us; 7 x 2048: 3.5.
template <typename TX, typename TO, int WPR, int NCH, bool VEC>
__global__ __launch_bounds__(kLnBlock) void layernorm_fwd_kernel(const TX* __restrict__ x, const void* __restrict__ w,
                                                                 const void* __restrict__ b, int w_code, float eps,
                                                                 int64_t T_, int H, TO* __restrict__ out,
                                                                 float* __restrict__ mean, float* __restrict__ rstd) {
  constexpr int TPR = kWave * WPR, RPB = kLnBlock / TPR;
  typedef Cols<TPR, NCH, VEC> C;
  __shared__ float s_sum[2][kLnBlock / kWave][1];
  const int t = threadIdx.x % TPR;
  const int64_t first = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR, step = (int64_t)gridDim.x * RPB;
  typename C::template Raw<TX> next;
  constexpr bool AHEAD = NCH > 2;
  if (AHEAD && first < T_) next.load(x + first * H, t, H);
  float wv[NCH][8], bv[NCH][8];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    C::params(w, w_code, 1.0f, t, i, H, wv[i]);
    C::params(b, w_code, 0.0f, t, i, H, bv[i]);
  }
  for (int64_t base = (int64_t)blockIdx.x * RPB, row = first; base < T_; base += step, row += step) {  // uniform over the block
    float v[NCH][8];
    if (!AHEAD && row < T_) next.load(x + row * H, t, H);
    next.unpack(t, H, v);
    if (AHEAD && row + step < T_) next.load(x + (row + step) * H, t, H);
    float a[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) a[0] += v[i][e];
    row_sums<WPR>(a, s_sum, 0);
    const float mu = a[0] / (float)H;
    a[0] = 0.0f;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[i][e] -= mu;
        if (C::in(t, i, e, H)) a[0] += v[i][e] * v[i][e];
      }
    row_sums<WPR>(a, s_sum, 1);
    const float r = 1.0f / sqrtf(a[0] / (float)H + eps);
    if (row < T_) {
      if (t == 0 && mean != nullptr) {
        mean[row] = mu;
        rstd[row] = r;
      }
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = (v[i][e] * r) * wv[i][e] + bv[i][e];
        C::store(out + row * H, t, i, H, v[i]);
      }
    }
  }
}

// gx, and this block's sums of g xh and g over its rows: partial rows
// part[2 blockIdx.x] and part[2 blockIdx.x + 1] of ld columns (part null: not
// wanted). The weight stays in registers and the next row is on its way while a row
// is worked on. The sums stay in registers too (a thread has the same columns in
// every row), so they cost 8 H bytes a block beside the rows' own: one or two
// blocks of eight waves a compute unit, no more. 8192 x 2048 bf16: 21.5 us, 101 MB
// at 4.7 TB/s; 16384 x 4096: 84 us, 403 MB at 4.8; 1531 x 1001 fp32: 9.6 us.
template <typename TX, typename TG, int WPR, int NCH, bool VEC>
__global__ __launch_bounds__(kLnBlock, sizeof(TX) == 2 && WPR <= 2 && NCH <= 2 ? 4 : 2) void layernorm_bwd_kernel(const TG* __restrict__ g, const TX* __restrict__ x,
                                                                 const void* __restrict__ w, int w_code,
                                                                 const float* __restrict__ mean,
                                                                 const float* __restrict__ rstd, int64_t T_, int H,
                                                                 TX* __restrict__ gx, float* __restrict__ part,
                                                                 int64_t ld) {
  constexpr int TPR = kWave * WPR, RPB = kLnBlock / TPR;
  typedef Cols<TPR, NCH, VEC> C;
  __shared__ float s_sum[2][kLnBlock / kWave][2];
  __shared__ float s_part[RPB > 1 ? RPB - 1 : 1][RPB > 1 ? TPR * 8 * NCH : 1];
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const int64_t first = (int64_t)blockIdx.x * RPB + sub, step = (int64_t)gridDim.x * RPB;
  typename C::template Raw<TX> nx;
  typename C::template Raw<TG> ng;
  float nmu = 0.0f, nr = 0.0f;
  auto fetch = [&](int64_t row) {
    nx.load(x + row * H, t, H);
    ng.load(g + row * H, t, H);
    nmu = mean[row];
    nr = rstd[row];
  };
  if (first < T_) fetch(first);
  float wv[NCH][8], gw[NCH][8], gb[NCH][8];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
#pragma unroll
    for (int e = 0; e < 8; ++e) gw[i][e] = gb[i][e] = wv[i][e] = 0.0f;
    C::params(w, w_code, 1.0f, t, i, H, wv[i]);
  }
  int turn = 0;
  for (int64_t base = (int64_t)blockIdx.x * RPB, row = first; base < T_; base += step, row += step, ++turn) {  // uniform
    const bool on = row < T_;
    float xv[NCH][8], gv[NCH][8];
    nx.unpack(t, H, xv);
    ng.unpack(t, H, gv);
    const float mu = nmu, r = nr;
    if (row + step < T_) fetch(row + step);
    float s[2] = {0.0f, 0.0f};
    if (on) {
#pragma unroll
      for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float ge = gv[i][e], xh = C::in(t, i, e, H) ? (xv[i][e] - mu) * r : 0.0f;
          xv[i][e] = xh;
          gb[i][e] += ge;
          gw[i][e] += ge * xh;
          gv[i][e] = ge * wv[i][e];
          s[0] += gv[i][e];
          s[1] += gv[i][e] * xh;
        }
    }
    if (gx == nullptr) continue;  // uniform over the grid
    row_sums<WPR>(s, s_sum, turn);
    const float c1 = s[0] / (float)H, c2 = s[1] / (float)H;
    if (on) {
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
#pragma unroll
        for (int e = 0; e < 8; ++e) gv[i][e] = r * (gv[i][e] - c1 - xv[i][e] * c2);
        C::store(gx + row * H, t, i, H, gv[i]);
      }
    }
  }
  if (part == nullptr) return;  // uniform over the grid
  // the block's RPB rows at a time hold the same columns: joined in their order
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float(&acc)[NCH][8] = which == 0 ? gw : gb;
    if constexpr (RPB > 1) {
      if (which > 0) __syncthreads();  // the first sums have been read
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
          for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int k = 0; k < RPB - 1; ++k) acc[i][e] += s_part[k][(i * 8 + e) * TPR + t];
    }
    if (sub == 0) {
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
  __shared__ float s_sum[2][kLnBlock / kWave][1];
  const int64_t row = blockIdx.x;
  const TX* xr = x + row * H;
  float a[1] = {0.0f};
  for (int c = threadIdx.x; c < H; c += kLnBlock) a[0] += load_scalar<TX>(xr + c);
  row_sums<8>(a, s_sum, 0);
  const float mu = a[0] / (float)H;
  a[0] = 0.0f;
  for (int c = threadIdx.x; c < H; c += kLnBlock) {
    const float d = load_scalar<TX>(xr + c) - mu;
    a[0] += d * d;
  }
  row_sums<8>(a, s_sum, 1);
  const float r = 1.0f / sqrtf(a[0] / (float)H + eps);
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
  __shared__ float s_sum[2][kLnBlock / kWave][2];
  const int64_t row = blockIdx.x;
  const float mu = mean[row], r = rstd[row];
  float s[2] = {0.0f, 0.0f};
  for (int c = threadIdx.x; c < H; c += kLnBlock) {
    const float gv = load_scalar<TG>(g + row * H + c) * param(w, w_code, c, 1.0f);
    s[0] += gv;
    s[1] += gv * ((load_scalar<TX>(x + row * H + c) - mu) * r);
  }
  row_sums<8>(s, s_sum, 0);
  const float c1 = s[0] / (float)H, c2 = s[1] / (float)H;
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
// A latency, 4 us: 256 partial rows of 2048 columns are 4 MB, in L2 or close by.
__global__ __launch_bounds__(256) void layernorm_reduce_kernel(const float* __restrict__ part, int nb, int64_t ld,
                                                               int H, void* __restrict__ gw, void* __restrict__ gb,
                                                               int w_code) {
  __shared__ f32x4 s[32][8];
  const int which = blockIdx.y, q = threadIdx.x % 8, grp = threadIdx.x / 8;
  const int c = blockIdx.x * 32 + q * 4;
  void* out = which == 0 ? gw : gb;
  if (out == nullptr) return;  // uniform over the block
  f32x4 a = {0, 0, 0, 0};
#pragma unroll 8
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

// Calls f(waves a row, chunks a thread, VEC) for a row of H <= kLnRegH columns.
// The forward: two chunks a thread, spread over more waves, against four (bf16): 7 x
// 2048 3.5 / 4.6 us, 8192 x 2048 14.0 / 16.0, 16384 x 4096 49 / 62.
template <class F>
hipError_t by_width_fwd(int H, bool vec, F&& f) {
  using std::integral_constant;
  auto go = [&](auto wpr, auto nch) { return vec ? f(wpr, nch, std::true_type()) : f(wpr, nch, std::false_type()); };
  if (H <= 512) return go(integral_constant<int, 1>(), integral_constant<int, 1>());
  if (H <= 1024) return go(integral_constant<int, 1>(), integral_constant<int, 2>());
  if (H <= 2048) return go(integral_constant<int, 2>(), integral_constant<int, 2>());
  if (H <= 4096) return go(integral_constant<int, 4>(), integral_constant<int, 2>());
  if (H <= 8192) return go(integral_constant<int, 8>(), integral_constant<int, 2>());
  return go(integral_constant<int, 8>(), integral_constant<int, 4>());
}
// The backward holds six values a column, in two chunks a thread up to 2048 columns,
// and beyond them where four would spill or gain nothing: fp32, 8192 x 2048, two /
// four chunks 38 / 42 us, with bf16 gradients 33 / 37; rows of 16 bits that do not
// start on 16 bytes up to 4096 columns, 8192 x 4001 39 / 43, but 8192 x 6001 80 / 72
// (aligned: 16384 x 4096 82 / 80, 4096 x 8192 46 / 45).
// 16-bit rows in two chunks leave room for two blocks a compute unit. Two / one (of
// four chunks from 1025 columns on), with the sums' launch, bf16: 32768 x 512 24.0 /
// 26.9 us, 32768 x 1024 40.4 / 42.1, 2048 x 2048 14.0 / 16.2, 8192 x 2048 25.4 / 27.5;
// but 16384 x 4096 82 / 80, 4096 x 8192 53 / 44, and fp32, whose registers do not
// fit, 8192 x 2048 42 / 39.
template <bool HALF, class F>
hipError_t by_width_bwd(int H, bool vec, F&& f) {
  using std::integral_constant;
  auto go = [&](auto wpr, auto nch) { return vec ? f(wpr, nch, std::true_type()) : f(wpr, nch, std::false_type()); };
  if (H <= 512) return go(integral_constant<int, 1>(), integral_constant<int, 1>());
  if (H <= 1024) return go(integral_constant<int, 1>(), integral_constant<int, 2>());
  if (H <= 2048) return go(integral_constant<int, 2>(), integral_constant<int, 2>());
  if constexpr (HALF) {
    if (H <= 4096)
      return vec ? f(integral_constant<int, 2>(), integral_constant<int, 4>(), std::true_type())
                 : f(integral_constant<int, 4>(), integral_constant<int, 2>(), std::false_type());
    if (H <= 8192) return go(integral_constant<int, 4>(), integral_constant<int, 4>());
  } else {
    if (H <= 4096) return go(integral_constant<int, 4>(), integral_constant<int, 2>());
    if (H <= 8192) return go(integral_constant<int, 8>(), integral_constant<int, 2>());
  }
  return go(integral_constant<int, 8>(), integral_constant<int, 4>());
}

// Rows that a block of the backward has at a time (in two chunks a thread: as many, or half).
int rows_a_block(int H) { return H <= 2048 ? 8 : H <= 4096 ? 4 : H <= 8192 ? 2 : 1; }
int64_t wide_rows(int64_t T_) { return std::max<int64_t>(kLnColRows, (T_ + kLnColBlocks - 1) / kLnColBlocks); }

}  // namespace

int layernorm_bwd_blocks(int64_t T_, int H, bool half) {
  if (T_ <= 0) return 0;
  if (H > kLnRegH) return (int)((T_ + wide_rows(T_) - 1) / wide_rows(T_));
  const int rpb = rows_a_block(H);
  return (int)std::min<int64_t>((T_ + rpb - 1) / rpb, half && H <= kLnTwoH ? 2 * kLnMaxBlocks : kLnMaxBlocks);
}

int64_t layernorm_part_ld(int H) { return ln_pad(H); }

// Rows walked in passes have a block each: fewer than 2^32 threads a launch.
int64_t layernorm_max_rows(int H) { return H > kLnRegH ? ((int64_t)1 << 32) / kLnBlock - 1 : 0x7fffffff; }

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
  return by_width_fwd(H, vec, [&](auto wpr, auto nch, auto v) {
    constexpr int WPR = decltype(wpr)::value, NCH = decltype(nch)::value, RPB = kLnBlock / kWave / WPR;
    const int64_t most = NCH > 2 ? kLnMaxBlocks : kLnFwdBlocks;
    hipLaunchKernelGGL((layernorm_fwd_kernel<TX, TO, WPR, NCH, decltype(v)::value>),
                       dim3((unsigned)std::min<int64_t>((T_ + RPB - 1) / RPB, most)), dim3(kLnBlock), 0, s, x, w,
                       b, w_code, eps, T_, H, out, mean, rstd);
    return hipGetLastError();
  });
}

template <typename TX, typename TG>
hipError_t layernorm_bwd(const TG* g, const TX* x, const void* w, int w_code, const float* mean, const float* rstd,
                         int64_t T_, int H, TX* gx, float* part, void* gw, void* gb, hipStream_t s) {
  const bool vec = H % 8 == 0 && all16({g, x, w, gx, part});
  const int nb = layernorm_bwd_blocks(T_, H, sizeof(TX) == 2);
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
    st = by_width_bwd<sizeof(TX) == 2>(H, vec, [&](auto wpr, auto nch, auto v) {
      constexpr int WPR = decltype(wpr)::value, NCH = decltype(nch)::value;
      hipLaunchKernelGGL((layernorm_bwd_kernel<TX, TG, WPR, NCH, decltype(v)::value>), dim3(nb), dim3(kLnBlock), 0, s, g,
                         x, w, w_code, mean, rstd, T_, H, gx, part, ld);
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
