// The router's auxiliary loss over all layers at once: per-expert counts,
// load-balance loss and z-loss from the logits, and every layer's gradient
// (load_balancing_loss, router_z_loss, _update_expert_counts:
// qwen3_moe.py:285-316, :417-426).
//
//   p = softmax(l_t), S_t = the K largest logits (equal ones: the lower id)
//   c_e = #{valid t : e in S_t}, n = the number of valid rows of all layers
//   LB = E sum_e (c_e / n) (sum_t p_te / n),  Z = sum_t lse_t^2 / n
//   dl_tj = dloss p_tj [a E / n (f_j - sum_e f_e p_te) + 2 z / n lse_t]
// with f_e = c_e / n - K / E: the softmax sums to one, so the mean K / E drops
// out of f_j - sum_e f_e p_te, and taking it off first (in whole numbers) keeps
// a nearly balanced router's gradient from being a difference of close values.
//
// The forward reads the logits once; the backward reads them again and writes
// the gradients. Both hold a row in LPR lanes of V values; sums over rows stay
// in registers, are joined per block in a fixed order and written as partial
// rows, which a second launch sums: no floating atomics, so the same inputs
// give the same bits.
#include "kernels.h"

namespace pmoe {
namespace {

constexpr int kBlock = 256;
constexpr int kWaves = kBlock / kWave;

// The largest / the sum over the LPR lanes (consecutive, a power of two) of a row.
template <int LPR>
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
#pragma unroll
  for (int o = 1; o < LPR; o <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, kWave));
  return v;
}
template <int LPR>
__device__ __forceinline__ int row_add(int v) {
#pragma unroll
  for (int o = 1; o < LPR; o <<= 1) v += __shfl_xor(v, o, kWave);
  return v;
}
template <int LPR>
__device__ __forceinline__ float row_add(float v) {
#pragma unroll
  for (int o = 1; o < LPR; o <<= 1) v += __shfl_xor(v, o, kWave);
  return v;
}

// Unsigned keys in the order of the values: -0 and +0 alike, NaN above all
// (torch's order). Every key is above 0, which stands for "no expert".
__device__ __forceinline__ uint32_t order_key(float x) {
  const float y = x + 0.0f;  // -0 -> +0
  const uint32_t u = y != y ? 0x7fc00000u : __float_as_uint(y);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// A row's columns in a lane: J pieces of W consecutive ones (W elements are one
// load), piece j of lane l from column (j * LPR + l) * W.
template <int LPR, int V, int W>
struct Row {
  static constexpr int J = V / W;
  __device__ static __forceinline__ int col(int l, int i) { return ((i / W) * LPR + l) * W + i % W; }
  template <typename T>
  __device__ static __forceinline__ void load(const T* row, int l, int E, float fill, float (&v)[V]) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int c = (j * LPR + l) * W;
      if (c < E) {
        if constexpr (W == 1) {
          v[j] = load_scalar<T>(row + c);
        } else if constexpr (sizeof(T) == 2 && W == 8) {
          Vec8<T>::load(row + c, &v[j * 8]);
        } else if constexpr (sizeof(T) == 2) {
          const uint2 w = *reinterpret_cast<const uint2*>(row + c);
          v[j * 4] = Fmt16<T>::lo(w.x); v[j * 4 + 1] = Fmt16<T>::hi(w.x);
          v[j * 4 + 2] = Fmt16<T>::lo(w.y); v[j * 4 + 3] = Fmt16<T>::hi(w.y);
        } else {
          const f32x4 w = *reinterpret_cast<const f32x4*>(row + c);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[j * 4 + e] = w[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < W; ++e) v[j * W + e] = fill;
      }
    }
  }
  template <typename T>
  __device__ static __forceinline__ void store(T* row, int l, int E, const float (&v)[V]) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int c = (j * LPR + l) * W;
      if (c >= E) continue;
      if constexpr (W == 1) {
        store_scalar<T>(row + c, v[j]);
      } else if constexpr (sizeof(T) == 2 && W == 8) {
        Vec8<T>::store(row + c, &v[j * 8]);
      } else if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint2*>(row + c) =
            make_uint2(Fmt16<T>::pack2(v[j * 4], v[j * 4 + 1]), Fmt16<T>::pack2(v[j * 4 + 2], v[j * 4 + 3]));
      } else {
        const f32x4 w = {v[j * 4], v[j * 4 + 1], v[j * 4 + 2], v[j * 4 + 3]};
        *reinterpret_cast<f32x4*>(row + c) = w;
      }
    }
  }
};

// Bit i of the result: the lane's value i is among the row's K largest. Each of
// up to K steps takes the largest key below the last one with all its equals;
// the step in which they no longer all fit takes the lowest ids of them. Keys 0
// (columns past E) are never taken, K <= E.
template <int LPR, int V, int W>
__device__ __forceinline__ uint32_t select_top(const uint32_t (&key)[V], uint32_t top, int K, int l) {
  uint32_t m = top;
  int left = K;
  bool done = false;
  for (int k = 0; k < K; ++k) {
    int eq = 0;
    uint32_t t = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      eq += key[i] == m;
      t = max(t, key[i] < m ? key[i] : 0u);
    }
    eq = row_add<LPR>(eq);
    t = row_max<LPR>(t);
    done = done || eq >= left;
    if (!done) { left -= eq; m = t; }
  }
  // of the keys equal to m the first `left` by id, piece by piece
  uint32_t sel = 0;
  int before = 0;  // equals in earlier pieces
#pragma unroll
  for (int j = 0; j < V / W; ++j) {
    int mine = 0;
#pragma unroll
    for (int e = 0; e < W; ++e) mine += key[j * W + e] == m;
    int below = 0, all = 0;  // equals of this piece in lower lanes, and in all lanes
#pragma unroll
    for (int o = 0; o < LPR; ++o) {
      const int c = __shfl(mine, o, LPR);
      below += o < l ? c : 0;
      all += c;
    }
    int rank = before + below;
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const bool same = key[j * W + e] == m;
      if (key[j * W + e] > m || (same && rank < left)) sel |= 1u << (j * W + e);
      rank += same;
    }
    before += all;
  }
  return sel;
}

// Partial sums over the rows of (layer blockIdx.y, block blockIdx.x of it):
// psum[b][e], counts[b][e], lse2[b], rows[b], b = blockIdx.y * gridDim.x + blockIdx.x.
template <typename T, int LPR, int V, int W>
__global__ __launch_bounds__(kBlock) void aux_stats_kernel(AuxLayers layers, const uint8_t* __restrict__ mask, int E,
                                                           int K, float* __restrict__ psum, int32_t* __restrict__ counts,
                                                           float* __restrict__ lse2, int32_t* __restrict__ rows) {
  typedef Row<LPR, V, W> R;
  constexpr int RPW = kWave / LPR;  // rows of a wave
  __shared__ float s_p[kWaves][LPR * V];
  __shared__ int s_c[kWaves][LPR * V];
  __shared__ float s_l[kWaves];
  __shared__ int s_n[kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane % LPR, sub = lane / LPR;
  const T* logits = static_cast<const T*>(layers.logits[blockIdx.y]);
  const int64_t N = layers.rows[blockIdx.y];
  float ps[V];
  int ct[V];
#pragma unroll
  for (int i = 0; i < V; ++i) { ps[i] = 0.0f; ct[i] = 0; }
  float l2 = 0.0f;
  int n = 0;
  const int64_t step = (int64_t)gridDim.x * kWaves * RPW;
  for (int64_t base = ((int64_t)blockIdx.x * kWaves + wave) * RPW; base < N; base += step) {  // uniform over the wave
    const int64_t t = base + sub;
    const bool valid = t < N && (mask == nullptr || mask[t] != 0);
    float v[V];
    R::load(logits + (valid ? t : base) * E, l, E, 0.0f, v);
    uint32_t key[V], top = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      key[i] = R::col(l, i) < E ? order_key(v[i]) : 0u;
      top = max(top, key[i]);
    }
    top = row_max<LPR>(top);
    const float mx = key_value(top);
    const uint32_t sel = select_top<LPR, V, W>(key, top, K, l);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      v[i] = key[i] != 0u ? expf(v[i] - mx) : 0.0f;
      s += v[i];
    }
    s = row_add<LPR>(s);
    const float inv = 1.0f / s, lse = mx + logf(s);
    if (valid) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        ps[i] += v[i] * inv;
        ct[i] += (sel >> i) & 1;
      }
      if (l == 0) { l2 += lse * lse; ++n; }
    }
  }
  // the wave's rows, then the block's waves, in a fixed order
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int o = LPR; o < kWave; o <<= 1) {
      ps[i] += __shfl_xor(ps[i], o, kWave);
      ct[i] += __shfl_xor(ct[i], o, kWave);
    }
  l2 = wave_sum(l2);
  n = row_add<kWave>(n);
  if (sub == 0) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      s_p[wave][R::col(l, i)] = ps[i];
      s_c[wave][R::col(l, i)] = ct[i];
    }
  }
  if (lane == 0) { s_l[wave] = l2; s_n[wave] = n; }
  __syncthreads();
  const int64_t b = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  for (int e = threadIdx.x; e < E; e += kBlock) {
    float p = s_p[0][e];
    int c = s_c[0][e];
#pragma unroll
    for (int k = 1; k < kWaves; ++k) { p += s_p[k][e]; c += s_c[k][e]; }
    psum[b * E + e] = p;
    counts[b * E + e] = c;
  }
  if (threadIdx.x == 0) {
    lse2[b] = ((s_l[0] + s_l[1]) + s_l[2]) + s_l[3];
    rows[b] = s_n[0] + s_n[1] + s_n[2] + s_n[3];
  }
}

// Sums of the partial rows for 16 experts a block: counts per layer, their
// total and the probabilities' sum (16 groups of rows, joined in order).
__global__ __launch_bounds__(kBlock) void aux_columns_kernel(const float* __restrict__ psum,
                                                             const int32_t* __restrict__ part_counts, int L, int bpl,
                                                             int E, int32_t* __restrict__ counts,
                                                             double* __restrict__ col_p, int64_t* __restrict__ col_c) {
  __shared__ double s_p[16][16];
  __shared__ int64_t s_c[16][16];
  const int q = threadIdx.x % 16, grp = threadIdx.x / 16, e = blockIdx.x * 16 + q;
  double p = 0.0;
  int64_t c = 0;
  if (e < E) {
    for (int b = grp; b < L * bpl; b += 16) p += psum[(int64_t)b * E + e];
    for (int layer = grp; layer < L; layer += 16) {
      int own = 0;
      for (int b = 0; b < bpl; ++b) own += part_counts[((int64_t)layer * bpl + b) * E + e];
      counts[(int64_t)layer * E + e] = own;
      c += own;
    }
  }
  s_p[grp][q] = p;
  s_c[grp][q] = c;
  __syncthreads();
  if (grp != 0 || e >= E) return;
  for (int k = 1; k < 16; ++k) { p += s_p[k][q]; c += s_c[k][q]; }
  col_p[e] = p;
  col_c[e] = c;
}

__device__ __forceinline__ double block_sum(double v, double* s) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  double a = s[0];
  for (int k = 1; k < kWaves; ++k) a += s[k];
  __syncthreads();
  return a;
}

// The three losses from the columns' sums, and what the backward takes: f_e and 1 / n.
__device__ __forceinline__ void finish(const double* col_p, const int64_t* col_c, int64_t n, double lse2, int E, int K,
                                       float a, float z, const AuxOut& out, double* s) {
  const double inv = n > 0 ? 1.0 / (double)n : 0.0;
  double lb = 0.0;
  for (int e = threadIdx.x; e < E; e += kBlock) {
    lb += (double)col_c[e] * inv * (col_p[e] * inv);
    out.f[e] = (float)((double)(col_c[e] * E - (int64_t)K * n) * inv / (double)E);
  }
  lb = block_sum(lb, s) * (double)E;
  if (threadIdx.x != 0) return;
  const double zl = lse2 * inv;
  out.loss[0] = (float)((double)a * lb + (double)z * zl);
  out.balance[0] = (float)lb;
  out.z[0] = (float)zl;
  out.f[E] = (float)inv;
}

__global__ __launch_bounds__(kBlock) void aux_finish_kernel(const double* __restrict__ col_p,
                                                            const int64_t* __restrict__ col_c,
                                                            const float* __restrict__ lse2,
                                                            const int32_t* __restrict__ rows, int nb, int E, int K,
                                                            float a, float z, AuxOut out) {
  __shared__ double s[kWaves];
  double n = 0.0, l2 = 0.0;
  for (int b = threadIdx.x; b < nb; b += kBlock) {
    n += rows[b];  // whole numbers below 2^53: exact
    l2 += lse2[b];
  }
  n = block_sum(n, s);
  l2 = block_sum(l2, s);
  finish(col_p, col_c, (int64_t)n, l2, E, K, a, z, out, s);
}

// The same from the statistics that the fused routers already have (one block).
__global__ __launch_bounds__(kBlock) void aux_from_stats_kernel(AuxStats st, int L, int64_t n, int E, int K, float a,
                                                                float z, int32_t* __restrict__ counts,
                                                                double* __restrict__ col_p,
                                                                int64_t* __restrict__ col_c, int first, int last,
                                                                double* __restrict__ lse2_sum, AuxOut out) {
  __shared__ double s[kWaves];
  for (int e = threadIdx.x; e < E; e += kBlock) {  // each thread's own columns: read back below by the same thread
    double p = first ? 0.0 : col_p[e];
    int64_t c = first ? 0 : col_c[e];
    for (int i = 0; i < L; ++i) {
      const int32_t k = st.counts[i][e];
      counts[(int64_t)i * E + e] = k;
      c += k;
      p += st.prob_sum[i][e];
    }
    col_p[e] = p;
    col_c[e] = c;
  }
  double l2 = 0.0;
  for (int i = threadIdx.x; i < L; i += kBlock) l2 += st.lse_sq_sum[i][0];
  l2 = block_sum(l2, s) + (first ? 0.0 : lse2_sum[0]);
  __syncthreads();
  if (threadIdx.x == 0) lse2_sum[0] = l2;
  if (last) finish(col_p, col_c, n, l2, E, K, a, z, out, s);
}

template <typename T, int LPR, int V, int W>
__global__ __launch_bounds__(kBlock) void aux_grad_kernel(AuxLayers layers, AuxGrads grads,
                                                          const uint8_t* __restrict__ mask, int E,
                                                          const float* __restrict__ f, const float* __restrict__ dloss,
                                                          float a, float z) {
  typedef Row<LPR, V, W> R;
  constexpr int RPW = kWave / LPR;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane % LPR, sub = lane / LPR;
  const T* logits = static_cast<const T*>(layers.logits[blockIdx.y]);
  T* out = static_cast<T*>(grads.grad[blockIdx.y]);
  const int64_t N = layers.rows[blockIdx.y];
  if (out == nullptr) return;  // this layer's gradient is not wanted
  const float g = dloss[0] * f[E];
  const float ca = g * a * (float)E, cz = 2.0f * g * z;
  float fe[V];
#pragma unroll
  for (int i = 0; i < V; ++i) fe[i] = R::col(l, i) < E ? f[R::col(l, i)] : 0.0f;
  const int64_t step = (int64_t)gridDim.x * kWaves * RPW;
  for (int64_t base = ((int64_t)blockIdx.x * kWaves + wave) * RPW; base < N; base += step) {
    const int64_t t = base + sub;
    if (t >= N) continue;  // whole rows: the row's lanes go together
    float v[V];
    if (mask != nullptr && mask[t] == 0) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = 0.0f;
      R::store(out + t * E, l, E, v);
      continue;
    }
    R::load(logits + t * E, l, E, -INFINITY, v);
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; ++i) mx = fmaxf(mx, v[i]);
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o, kWave));
    float s = 0.0f, d = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      v[i] = R::col(l, i) < E ? expf(v[i] - mx) : 0.0f;
      s += v[i];
      d += v[i] * fe[i];
    }
    s = row_add<LPR>(s);
    const float inv = 1.0f / s, lse = mx + logf(s);
    const float mean_f = row_add<LPR>(d) * inv, zl = cz * lse;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = v[i] * inv * (ca * (fe[i] - mean_f) + zl);
    R::store(out + t * E, l, E, v);
  }
}

// Calls f(lanes a row, values a lane, elements a load) for E experts; low: the
// tensors' addresses or-ed (what their alignment allows a load to be).
template <typename T, class F>
hipError_t by_experts(int E, uintptr_t low, F&& f) {
  using std::integral_constant;
  constexpr int WMAX = 16 / (int)sizeof(T);
  low |= (uintptr_t)E * sizeof(T);
  auto by_w = [&](auto lpr, auto v) {
    constexpr int V = decltype(v)::value;
    if constexpr (V >= WMAX)
      if (low % 16 == 0) return f(lpr, v, integral_constant<int, WMAX>());
    if constexpr (WMAX == 8)
      if (low % 8 == 0) return f(lpr, v, integral_constant<int, 4>());
    return f(lpr, v, integral_constant<int, 1>());
  };
  if (E <= 16) return by_w(integral_constant<int, 4>(), integral_constant<int, 4>());
  if (E <= 32) return by_w(integral_constant<int, 4>(), integral_constant<int, 8>());
  if (E <= 64) return by_w(integral_constant<int, 4>(), integral_constant<int, 16>());
  if (E <= 128) return by_w(integral_constant<int, 8>(), integral_constant<int, 16>());
  if (E <= 256) return by_w(integral_constant<int, 16>(), integral_constant<int, 16>());
  if (E <= 512) return by_w(integral_constant<int, 32>(), integral_constant<int, 16>());
  return by_w(integral_constant<int, 64>(), integral_constant<int, 16>());
}

uintptr_t low_bits(const AuxLayers& a, const AuxGrads* g, int L) {
  uintptr_t low = 0;
  for (int i = 0; i < L; ++i) low |= reinterpret_cast<uintptr_t>(a.logits[i]) | (g != nullptr ? reinterpret_cast<uintptr_t>(g->grad[i]) : 0);
  return low;
}

}  // namespace

// Blocks of one layer: about kAuxBlocks in all, each with at least 64 rows.
int aux_blocks_per_layer(int L, int64_t max_rows) {
  const int64_t want = std::max(1, kAuxBlocks / std::max(1, L));
  return (int)std::max<int64_t>(1, std::min<int64_t>(want, (max_rows + 63) / 64));
}

template <typename T>
hipError_t aux_stats(const AuxLayers& layers, int L, const uint8_t* mask, int E, int K, int bpl, float* psum,
                     int32_t* counts, float* lse2, int32_t* rows, hipStream_t s) {
  return by_experts<T>(E, low_bits(layers, nullptr, L), [&](auto lpr, auto v, auto w) {
    hipLaunchKernelGGL((aux_stats_kernel<T, decltype(lpr)::value, decltype(v)::value, decltype(w)::value>),
                       dim3(bpl, L), dim3(kBlock), 0, s, layers, mask, E, K, psum, counts, lse2, rows);
    return hipGetLastError();
  });
}

hipError_t aux_finish(const float* psum, const int32_t* part_counts, const float* lse2, const int32_t* rows, int L,
                      int bpl, int E, int K, float a, float z, int32_t* counts, double* col_p, int64_t* col_c,
                      const AuxOut& out, hipStream_t s) {
  hipLaunchKernelGGL(aux_columns_kernel, dim3((E + 15) / 16), dim3(kBlock), 0, s, psum, part_counts, L, bpl, E, counts,
                     col_p, col_c);
  hipLaunchKernelGGL(aux_finish_kernel, dim3(1), dim3(kBlock), 0, s, col_p, col_c, lse2, rows, L * bpl, E, K, a, z,
                     out);
  return hipGetLastError();
}

hipError_t aux_from_stats(const AuxStats& st, int L, int64_t n, int E, int K, float a, float z, int32_t* counts,
                          double* col_p, int64_t* col_c, bool first, bool last, double* lse2_sum, const AuxOut& out,
                          hipStream_t s) {
  hipLaunchKernelGGL(aux_from_stats_kernel, dim3(1), dim3(kBlock), 0, s, st, L, n, E, K, a, z, counts, col_p, col_c,
                     (int)first, (int)last, lse2_sum, out);
  return hipGetLastError();
}

template <typename T>
hipError_t aux_grad(const AuxLayers& layers, const AuxGrads& grads, int L, int64_t max_rows, const uint8_t* mask,
                    int E, const float* f, const float* dloss, float a, float z, hipStream_t s) {
  return by_experts<T>(E, low_bits(layers, &grads, L), [&](auto lpr, auto v, auto w) {
    constexpr int RPB = kWaves * (kWave / decltype(lpr)::value);
    const int64_t want = std::max(1, 4096 / std::max(1, L));
    const int bpl = (int)std::max<int64_t>(1, std::min<int64_t>(want, (max_rows + RPB - 1) / RPB));
    hipLaunchKernelGGL((aux_grad_kernel<T, decltype(lpr)::value, decltype(v)::value, decltype(w)::value>),
                       dim3(bpl, L), dim3(kBlock), 0, s, layers, grads, mask, E, f, dloss, a, z);
    return hipGetLastError();
  });
}

#define PMOE_INST_AUX(T)                                                                                             \
  template hipError_t aux_stats<T>(const AuxLayers&, int, const uint8_t*, int, int, int, float*, int32_t*, float*,   \
                                   int32_t*, hipStream_t);                                                           \
  template hipError_t aux_grad<T>(const AuxLayers&, const AuxGrads&, int, int64_t, const uint8_t*, int,              \
                                  const float*, const float*, float, float, hipStream_t);
PMOE_INST_AUX(float)
PMOE_INST_AUX(bf16_t)
PMOE_INST_AUX(f16_t)

}  // namespace pmoe
