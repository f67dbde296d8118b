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
#include "lanes.h"

namespace pmoe {
namespace {

constexpr int kBlock = 256;        // threads of a block: the gradient, the statistics' sums
constexpr int kFinishBlock = 1024;  // of the second launch
constexpr int64_t kAuxOneBlock = 1 << 15;  // partial sums up to which it has one block
constexpr int kCols = 32;           // its experts a block where it has several blocks
// Threads of a block of the forward's pass over the logits, by the columns a row is
// padded to: a compute unit's worth of waves, as far as their sums fit LDS together,
// since each block's partial rows cost the second launch their reading. With 256
// threads everywhere: 48 layers of 8192 x 128 64 + 12 -> 71 + 18 us, 6 of 1531 x 60
// (bf16) 8.8 + 6.7 -> 6.9 + 12.4, one of 613 x 32 5.2 + 5.8 -> 4.3 + 6.2.
constexpr int stats_block(int cols) { return cols <= 256 ? 1024 : 256; }

template <int LPR>
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  return (uint32_t)lanes_reduce<LPR>((int)v, [](int a, int b) { return (int)max((uint32_t)a, (uint32_t)b); });
}
template <int LPR>
__device__ __forceinline__ uint32_t row_min(uint32_t v) {
  return (uint32_t)lanes_reduce<LPR>((int)v, [](int a, int b) { return (int)min((uint32_t)a, (uint32_t)b); });
}
template <int LPR>
__device__ __forceinline__ float row_fmax(float v) {
  return __int_as_float(lanes_reduce<LPR>(__float_as_int(v), [](int a, int b) {
    return __float_as_int(fmaxf(__int_as_float(a), __int_as_float(b)));
  }));
}
// e^x for x <= 0 (or NaN) from the hardware exp2: x log2 e is rounded once, so the relative error is |x| 2^-24 and 1 ulp.
__device__ __forceinline__ float exp_neg(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }

// Unsigned keys in the order of the values: -0 and +0 alike, NaN above all
// (torch's order). Every key is above 0, which stands for "no expert".
__device__ __forceinline__ uint32_t order_bits(uint32_t u) { return (u & 0x80000000u) ? ~u : (u | 0x80000000u); }
__device__ __forceinline__ uint32_t value_bits(uint32_t k) { return (k & 0x80000000u) ? (k & 0x7fffffffu) : ~k; }

// fp32: the value's own 32 bits; equal values have equal keys. 16 bits: the
// value's 16 bits above, and below them the column counted down, so that all keys
// of a row differ and equal values are in the order of their ids (16-bit logits
// are often equal).
template <typename T> struct Key {
  static constexpr bool unique = false;
  __device__ static __forceinline__ uint32_t of(float x, int) {
    const float y = x + 0.0f;  // -0 -> +0
    return order_bits(y != y ? 0x7fc00000u : __float_as_uint(y));
  }
  __device__ static __forceinline__ float value(uint32_t k) { return __uint_as_float(value_bits(k)); }
};
template <> struct Key<bf16_t> {
  static constexpr bool unique = true;
  __device__ static __forceinline__ uint32_t of(float x, int col) {
    return (Key<float>::of(x, 0) & 0xffff0000u) | (0xffffu - (uint32_t)col);
  }
  __device__ static __forceinline__ float value(uint32_t k) {
    return __uint_as_float(value_bits(k) & 0xffff0000u);
  }
};
template <> struct Key<f16_t> {
  static constexpr bool unique = true;
  __device__ static __forceinline__ uint32_t of(float x, int col) {
    const float y = x + 0.0f;
    const uint32_t u = y != y ? 0x7e00u : (uint32_t)__builtin_bit_cast(uint16_t, (f16_t)y);
    return (order_bits(u << 16) & 0xffff0000u) | (0xffffu - (uint32_t)col);
  }
  __device__ static __forceinline__ float value(uint32_t k) {
    const uint32_t u = value_bits(k) >> 16;
    return (float)__builtin_bit_cast(f16_t, (uint16_t)u);
  }
};

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

// The K-th largest of a row's distinct keys: each step takes the largest key
// below the last one. key - m as an unsigned number is largest for the key just
// below m (keys at or above m wrap to less), so a step is one subtraction a key
// and the maximum.
template <int LPR, int V>
__device__ __forceinline__ uint32_t kth_largest(const uint32_t (&key)[V], uint32_t top, int K) {
  uint32_t m = top;
  for (int k = 1; k < K; ++k) {
    uint32_t t = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) t = max(t, key[i] - m);
    m += row_max<LPR>(t);
  }
  return m;
}

// One above the K-th smallest of a row's keys, the smallest being 0, where the K
// smallest are distinct: each step takes the smallest key from m on, key - m (keys
// below m wrap to more). Where fewer than K distinct keys exist the result is of
// no use, which the caller sees from how many keys lie below it.
template <int LPR, int V>
__device__ __forceinline__ uint32_t above_kth_smallest(const uint32_t (&key)[V], int K) {
  uint32_t m = 1;
  for (int k = 1; k < K; ++k) {
    uint32_t t = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < V; ++i) t = min(t, key[i] - m);
    m += row_min<LPR>(t) + 1u;
  }
  return m;
}

// The selection where equal keys decide it. Bit i of the result: the lane's
// value i is among the row's K largest. Each of up to K steps takes the largest
// key below the last one with all its equals; the step in which they no longer
// all fit takes the lowest ids of them. Keys 0 (columns past E) are never taken,
// K <= E.
template <int LPR, int V, int W>
__device__ __forceinline__ uint32_t select_ties(const uint32_t (&key)[V], uint32_t top, int K, int l) {
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
    eq = lanes_sum<LPR>(eq);
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
    int upto = mine;  // equals of this piece in lanes up to this one
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) {
      const int c = __shfl_up(upto, o, LPR);
      upto += l >= o ? c : 0;
    }
    int rank = before + upto - mine;
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const bool same = key[j * W + e] == m;
      if (key[j * W + e] > m || (same && rank < left)) sel |= 1u << (j * W + e);
      rank += same;
    }
    before += __shfl(upto, LPR - 1, LPR);
  }
  return sel;
}

// Partial sums over the rows of (layer blockIdx.y, block blockIdx.x of it):
// psum[b][e], counts[b][e], lse2[b], rows[b], b = blockIdx.y * gridDim.x +
// blockIdx.x; clears `arrived` for the second launch.
//
// Bound by arithmetic: a pass over E logits a row for each of the K picks. The
// fewest lanes that hold a row in registers (16 values each) make the row's
// reductions short: two to four steps in one DPP row, not six over a wave. 48
// layers of 8192 x 128 fp32, K 8: 64 us, 201 MB at 3.2 TB/s (their copy would take
// 39); 12 of 8192 x 32, K 4: 8.8 us.
template <typename T, int LPR, int V, int W>
__global__ __launch_bounds__(stats_block(LPR * V)) void aux_stats_kernel(AuxLayers layers, const uint8_t* __restrict__ mask,
                                                                int E, int K, float* __restrict__ psum,
                                                                int32_t* __restrict__ counts, float* __restrict__ lse2,
                                                                int32_t* __restrict__ rows, uint32_t* arrived) {
  typedef Row<LPR, V, W> R;
  constexpr int RPW = kWave / LPR;  // rows of a wave
  constexpr int NT = stats_block(LPR * V), NW = NT / kWave;
  constexpr int PAD = LPR * V;
  __shared__ float s_p[NW][PAD];
  __shared__ int s_c[NW][PAD];
  __shared__ float s_l[NW];
  __shared__ int s_n[NW];
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *arrived = 0;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane % LPR, sub = lane / LPR;
  const T* logits = static_cast<const T*>(layers.logits[blockIdx.y]);
  const int64_t N = layers.rows[blockIdx.y];
  float ps[V];
  int ct[V];
#pragma unroll
  for (int i = 0; i < V; ++i) { ps[i] = 0.0f; ct[i] = 0; }
  float l2 = 0.0f;
  int n = 0;
  const int64_t step = (int64_t)gridDim.x * NW * RPW;
  for (int64_t base = ((int64_t)blockIdx.x * NW + wave) * RPW; base < N; base += step) {  // uniform over the wave
    const int64_t t = base + sub;
    const bool valid = t < N && (mask == nullptr || mask[t] != 0);
    // A lane past the end reads the wave's first row, and what it makes of it is not
    // counted. (Reading the next rows ahead: 48 layers of 8192 x 128 62 -> 95 us, its
    // registers do not fit four waves a SIMD; at 32 experts, where they do, no gain.)
    const T* row = logits + (t < N ? t : base) * E;
    float v[V], mx, s = 0.0f;
    R::load(row, l, E, Key<T>::unique ? 0.0f : -INFINITY, v);
    uint32_t key[V];
    if constexpr (Key<T>::unique) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        key[i] = R::col(l, i) < E ? Key<T>::of(v[i], R::col(l, i)) : 0u;
        top = max(top, key[i]);
      }
      top = row_max<LPR>(top);
      mx = Key<T>::value(top);
      uint32_t kth = kth_largest<LPR, V>(key, top, K);
      if (!valid) kth = 0xffffffffu;  // above every key
#pragma unroll
      for (int i = 0; i < V; ++i) {
        ct[i] += key[i] >= kth;
        v[i] = key[i] != 0u ? exp_neg(v[i] - mx) : 0.0f;
        s += v[i];
      }
      s = lanes_sum<LPR>(s);
    } else {
      // Keys: the bits of max - x, which are in order where max - x >= 0 is finite or
      // infinite, and never put a smaller x first (the rounding of a difference is
      // monotonic): if exactly K keys lie below a border, they are the K largest x.
      mx = v[0];
#pragma unroll
      for (int i = 1; i < V; ++i) mx = fmaxf(mx, v[i]);
      mx = row_fmax<LPR>(mx) + 0.0f;  // never -0: +0 and -0 both have the key 0 then
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = mx - v[i];
        key[i] = R::col(l, i) < E ? __float_as_uint(d) : 0xffffffffu;
        v[i] = R::col(l, i) < E ? exp_neg(-d) : 0.0f;
        s += v[i];
      }
      s = lanes_sum<LPR>(s);
      const uint32_t border = above_kth_smallest<LPR, V>(key, K);
      int below = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) below += key[i] < border;
      below = lanes_sum<LPR>(below);
      // equal keys at a row's K-th place, or NaN or +inf in it (then s is NaN): the wave's rows again, by exact keys and ids
      if (__any(valid && (below != K || s != s))) {
        float x[V];
        R::load(row, l, E, 0.0f, x);
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          key[i] = R::col(l, i) < E ? Key<T>::of(x[i], 0) : 0u;
          top = max(top, key[i]);
        }
        const uint32_t sel = select_ties<LPR, V, W>(key, row_max<LPR>(top), K, l);
        if (valid) {
#pragma unroll
          for (int i = 0; i < V; ++i) ct[i] += (sel >> i) & 1;
        }
      } else if (valid) {
#pragma unroll
        for (int i = 0; i < V; ++i) ct[i] += key[i] < border;
      }
    }
    const float inv = 1.0f / s, lse = mx + logf(s);
    if (valid) {
#pragma unroll
      for (int i = 0; i < V; ++i) ps[i] += v[i] * inv;
      if (l == 0) { l2 += lse * lse; ++n; }
    }
  }
  // the wave's rows, then the block's waves, in a fixed order
#pragma unroll
  for (int i = 0; i < V; ++i) {
    ps[i] = __int_as_float(lanes_across<LPR>(__float_as_int(ps[i]), AddF()));
    ct[i] = lanes_across<LPR>(ct[i], AddI());
    if (sub == 0) {
      s_p[wave][R::col(l, i)] = ps[i];
      s_c[wave][R::col(l, i)] = ct[i];
    }
  }
  l2 = lanes_sum<kWave>(l2);
  n = lanes_sum<kWave>(n);
  if (lane == 0) { s_l[wave] = l2; s_n[wave] = n; }
  __syncthreads();
  const int64_t b = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  for (int e = threadIdx.x; e < E; e += NT) {
    float p = 0.0f;
    int c = 0;
#pragma unroll
    for (int k = 0; k < NW; ++k) { p += s_p[k][e]; c += s_c[k][e]; }
    psum[b * E + e] = p;
    counts[b * E + e] = c;
  }
  if (threadIdx.x == NT - 1) {
    float a = 0.0f;
    int c = 0;
#pragma unroll
    for (int k = 0; k < NW; ++k) { a += s_l[k]; c += s_n[k]; }
    lse2[b] = a;
    rows[b] = c;
  }
}

// The sum over a block of NT threads, in every thread (s: NT / 64 values).
template <int NT>
__device__ __forceinline__ double block_sum(double v, double* s) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  double a = s[0];
#pragma unroll
  for (int k = 1; k < NT / kWave; ++k) a += s[k];
  return a;
}

// The three losses from the columns' sums, and what the backward takes: f_e and
// 1 / n. FAR: the sums come from other blocks (read past this compute unit's cache).
template <int NT, bool FAR>
__device__ __forceinline__ void finish(const double* col_p, const int64_t* col_c, int64_t n, double lse2, int E, int K,
                                       float a, float z, const AuxOut& out, double* s) {
  const double inv = n > 0 ? 1.0 / (double)n : 0.0;
  double lb = 0.0;
  for (int e = threadIdx.x; e < E; e += NT) {
    const double p = FAR ? __hip_atomic_load(col_p + e, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : col_p[e];
    const int64_t c = FAR ? __hip_atomic_load(col_c + e, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : col_c[e];
    lb += (double)c * inv * (p * inv);
    out.f[e] = (float)((double)(c * E - (int64_t)K * n) * inv / (double)E);
  }
  lb = block_sum<NT>(lb, s) * (double)E;
  if (threadIdx.x != 0) return;
  const double zl = lse2 * inv;
  out.loss[0] = (float)((double)a * lb + (double)z * zl);
  out.balance[0] = (float)lb;
  out.z[0] = (float)zl;
  out.f[E] = (float)inv;
}

// The second launch: a block sums the partial rows of `cols` experts (a power of
// two of at least 32), 1024 / cols groups of rows joined in order. One block then
// makes the losses; of several, the last to finish does. A latency: two dozen loads
// in flight a thread, then the joins; 5.8 us for one layer, 11.6 for 48 of 128
// experts.
__global__ __launch_bounds__(kFinishBlock) void aux_finish_kernel(const float* __restrict__ psum,
                                                                  const int32_t* __restrict__ part_counts,
                                                                  const float* __restrict__ lse2,
                                                                  const int32_t* __restrict__ rows, int L, int bpl,
                                                                  int E, int K, int cols, float a, float z,
                                                                  int32_t* __restrict__ counts, double* col_p,
                                                                  int64_t* col_c, uint32_t* arrived, AuxOut out) {
  __shared__ int s_c[kFinishBlock];  // a layer's counts where several groups share it: then L * cols < 1024
  __shared__ double s_p[kFinishBlock];
  __shared__ int64_t s_t[kFinishBlock];
  __shared__ double s[kFinishBlock / kWave];
  __shared__ double s_l2[kFinishBlock / kWave];
  __shared__ int s_n[kFinishBlock / kWave];
  __shared__ bool s_last;
  const int groups = kFinishBlock / cols;
  const int q = threadIdx.x & (cols - 1), grp = threadIdx.x / cols, e = blockIdx.x * cols + q;
  // S groups share a layer, each S-th row of it (few layers), or a group has every groups-th layer (S = 1)
  const int S = max(1, groups / L), sub = grp % S, lstep = groups / S;
  double p = 0.0;
  int64_t c = 0;
  s_c[threadIdx.x] = 0;
  __syncthreads();
  if (e < E && sub < bpl) {
    constexpr int U = 12;  // rows in flight
    const int per = (bpl - sub + S - 1) / S;  // this thread's rows of a layer
    int ll = grp / S, lj = 0;                 // the next row to load
    int l = ll, j = 0, own = 0;               // the next row to add, its layer's count so far
    while (l < L) {
      float pv[U];
      int cv[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        pv[u] = 0.0f;
        cv[u] = 0;
        if (ll < L) {
          const int64_t at = ((int64_t)ll * bpl + sub + (int64_t)lj * S) * E + e;
          pv[u] = psum[at];
          cv[u] = part_counts[at];
        }
        if (++lj == per) { lj = 0; ll += lstep; }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (l < L) {
          p += pv[u];
          own += cv[u];
          if (++j == per) {
            if (S > 1) atomicAdd(&s_c[l * cols + q], own);  // whole numbers: any order
            else counts[(int64_t)l * E + e] = own;
            c += own;
            own = j = 0;
            l += lstep;
          }
        }
      }
    }
  }
  s_p[threadIdx.x] = p;
  s_t[threadIdx.x] = c;
  int n = 0;
  double l2 = 0.0;
  for (int b = threadIdx.x; b < L * bpl; b += kFinishBlock) {
    n += rows[b];
    l2 += lse2[b];
  }
  n = lanes_sum<kWave>(n);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) l2 += __shfl_xor(l2, o, kWave);
  if ((threadIdx.x & 63) == 0) { s_n[threadIdx.x >> 6] = n; s_l2[threadIdx.x >> 6] = l2; }
  __syncthreads();
  n = 0;
  l2 = 0.0;
#pragma unroll
  for (int k = 0; k < kFinishBlock / kWave; ++k) { n += s_n[k]; l2 += s_l2[k]; }
  if (S > 1 && e < E && grp < L) counts[(int64_t)grp * E + e] = s_c[grp * cols + q];
  const bool one = gridDim.x == 1;
  if (grp == 0 && e < E) {
    for (int k = 1; k < groups; ++k) { p += s_p[k * cols + q]; c += s_t[k * cols + q]; }
    if (one) {
      s_p[q] = p;
      s_t[q] = c;
    } else {
      __hip_atomic_store(col_p + e, p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(col_c + e, c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  if (one) {  // a column's sums are read by the thread that wrote them
    finish<kFinishBlock, false>(s_p, s_t, n, l2, E, K, a, z, out, s);
    return;
  }
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) s_last = atomicAdd(arrived, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  finish<kFinishBlock, true>(col_p, col_c, n, l2, E, K, a, z, out, s);
}

// The same from the statistics that the fused routers already have (one block).
__global__ __launch_bounds__(kBlock) void aux_from_stats_kernel(AuxStats st, int L, int64_t n, int E, int K, float a,
                                                                float z, int32_t* __restrict__ counts, double* col_p,
                                                                int64_t* col_c, int first, int last,
                                                                double* lse2_sum, AuxOut out) {
  __shared__ double s[kBlock / kWave];
  for (int e = threadIdx.x; e < E; e += kBlock) {  // each thread's own columns: read back in finish() by the same thread
    double p = first ? 0.0 : col_p[e];
    int64_t c = first ? 0 : col_c[e];
#pragma unroll 4
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
  l2 = block_sum<kBlock>(l2, s) + (first ? 0.0 : lse2_sum[0]);
  __syncthreads();
  if (threadIdx.x == 0) lse2_sum[0] = l2;
  if (last) finish<kBlock, false>(col_p, col_c, n, l2, E, K, a, z, out, s);
}

// Every layer's gradient in one launch, bound by HBM: the logits are read again (p
// and lse are cheaper to compute again than to keep: N E values) and the gradients
// written. 48 layers of 8192 x 128 fp32: 403 MB in 68 us, 5.9 TB/s.
template <typename T, int LPR, int V, int W>
__global__ __launch_bounds__(kBlock) void aux_grad_kernel(AuxLayers layers, AuxGrads grads,
                                                          const uint8_t* __restrict__ mask, int E,
                                                          const float* __restrict__ f, const float* __restrict__ dloss,
                                                          float a, float z) {
  typedef Row<LPR, V, W> R;
  constexpr int RPW = kWave / LPR, kWaves = kBlock / kWave;
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
    mx = row_fmax<LPR>(mx);
    float s = 0.0f, d = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      v[i] = R::col(l, i) < E ? exp_neg(v[i] - mx) : 0.0f;
      s += v[i];
      d += v[i] * fe[i];
    }
    s = lanes_sum<LPR>(s);
    const float inv = 1.0f / s, lse = mx + logf(s);
    const float mean_f = lanes_sum<LPR>(d) * inv, zl = cz * lse;
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
  for (int i = 0; i < L; ++i) {
    low |= reinterpret_cast<uintptr_t>(a.logits[i]);
    if (g != nullptr) low |= reinterpret_cast<uintptr_t>(g->grad[i]);
  }
  return low;
}

}  // namespace

// Blocks of one layer: a block a compute unit in all (two where there are more
// layers than let that come out even, or blocks are small), each with rows for
// all its waves.
int aux_blocks_per_layer(int L, int64_t max_rows, int E) {
  const bool small = stats_block(E) < 1024;
  const int blocks = small || L > kAuxMaxLayers ? 2 * kAuxBlocks : kAuxBlocks;
  const int64_t want = L <= kAuxMaxLayers ? blocks / std::max(1, L) : (blocks + L - 1) / L;
  return (int)std::max<int64_t>(1, std::min<int64_t>(want, (max_rows + (small ? 15 : 63)) / (small ? 16 : 64)));
}

template <typename T>
hipError_t aux_stats(const AuxLayers& layers, int L, const uint8_t* mask, int E, int K, int bpl, float* psum,
                     int32_t* counts, float* lse2, int32_t* rows, uint32_t* arrived, hipStream_t s) {
  return by_experts<T>(E, low_bits(layers, nullptr, L), [&](auto lpr, auto v, auto w) {
    hipLaunchKernelGGL((aux_stats_kernel<T, decltype(lpr)::value, decltype(v)::value, decltype(w)::value>),
                       dim3(bpl, L), dim3(stats_block(decltype(lpr)::value * decltype(v)::value)), 0, s, layers, mask,
                       E, K, psum, counts, lse2, rows, arrived);
    return hipGetLastError();
  });
}

hipError_t aux_finish(const float* psum, const int32_t* part_counts, const float* lse2, const int32_t* rows, int L,
                      int bpl, int E, int K, float a, float z, int32_t* counts, double* col_p, int64_t* col_c,
                      uint32_t* arrived, const AuxOut& out, hipStream_t s) {
  // One block while it reads the partial sums in a few microseconds; several need
  // device-wide fences between them. One / several, us: 6 layers of 60 experts 6.7 /
  // 12.6; 48 of 128 (just under 2^15 sums) 11.6 / 12.5; 128 of 128 (2^16) 19.6 / 15.1;
  // 48 of 256 (just under 2^16) 18.1 / 13.0.
  int cols = kCols;
  if (E <= 256 && (int64_t)L * bpl * E <= kAuxOneBlock)
    while (cols < E) cols *= 2;
  hipLaunchKernelGGL(aux_finish_kernel, dim3((E + cols - 1) / cols), dim3(kFinishBlock), 0, s, psum, part_counts,
                     lse2, rows, L, bpl, E, K, cols, a, z, counts, col_p, col_c, arrived, out);
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
    constexpr int RPB = kBlock / decltype(lpr)::value;
    const int64_t want = std::max(1, 4096 / std::max(1, L));
    const int bpl = (int)std::max<int64_t>(1, std::min<int64_t>(want, (max_rows + RPB - 1) / RPB));
    hipLaunchKernelGGL((aux_grad_kernel<T, decltype(lpr)::value, decltype(v)::value, decltype(w)::value>),
                       dim3(bpl, L), dim3(kBlock), 0, s, layers, grads, mask, E, f, dloss, a, z);
    return hipGetLastError();
  });
}

#define PMOE_INST_AUX(T)                                                                                             \
  template hipError_t aux_stats<T>(const AuxLayers&, int, const uint8_t*, int, int, int, float*, int32_t*, float*,   \
                                   int32_t*, uint32_t*, hipStream_t);                                                \
  template hipError_t aux_grad<T>(const AuxLayers&, const AuxGrads&, int, int64_t, const uint8_t*, int,              \
                                  const float*, const float*, float, float, hipStream_t);
PMOE_INST_AUX(float)
PMOE_INST_AUX(bf16_t)
PMOE_INST_AUX(f16_t)

}  // namespace pmoe
