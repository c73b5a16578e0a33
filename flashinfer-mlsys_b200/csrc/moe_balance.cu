// moe_balance.cu — the router's training term: DeepSeek-V3's sequence-wise
// balance loss (DeepSeek-V3 technical report, eqs. 17-20) with the per-expert
// counts it needs, and its gradient with respect to the routing logits.
//
// For sequence s (tokens off[s] .. off[s+1]-1, T_s of them), E experts, K
// slots a token and scores a = sigmoid or exp of the logits l:
//   f_i = E / (K T_s) * #{(t, k) : topk_ids[t][k] = i}
//   p_ti = a_ti / sum_j a_tj,   P_i = 1/T_s sum_t p_ti
//   loss_s = coeff * sum_i f_i P_i
//   d loss_s / d l_tj = coeff / T_s * p_tj (f_j - sum_i f_i p_ti) * (1 - sigmoid(l_tj) for sigmoid, 1 for exp)
// An empty sequence has loss 0; a token whose scores sum to zero (every logit
// -inf) has p = 0 and no gradient; ids outside [0, E) are not counted; tokens
// of no sequence get a zero gradient.
//
// HBM-bound: one pass over the logits forward, one (and the gradient) back.
// Forward: CTAs own equal runs of tokens, whatever the sequences' lengths. A
// run meets a sequence in one segment; (run index + sequence index) grows
// along the segments, so it numbers them without gaps to search for, and each
// segment's fp32 column sums and counts go to a slot of their own. A second
// kernel adds a sequence's slots in order. No atomics on floats: results do
// not depend on the order in which CTAs run.
#include "moe_kernels.h"

namespace moe {

namespace {

constexpr int kBalWarps = 8;
constexpr int kBalThreads = kBalWarps * 32;

template <int kDt>
__device__ __forceinline__ float bal_load(const void* row, int c) {
  if constexpr (kDt == 0) return __bfloat162float(static_cast<const __nv_bfloat16*>(row)[c]);
  if constexpr (kDt == 1) return __half2float(static_cast<const __half*>(row)[c]);
  return static_cast<const float*>(row)[c];
}
template <int kDt>
__device__ __forceinline__ void bal_store(void* row, int c, float v) {
  if constexpr (kDt == 0)
    static_cast<__nv_bfloat16*>(row)[c] = __float2bfloat16_rn(v);
  else if constexpr (kDt == 1)
    static_cast<__half*>(row)[c] = __float2half_rn(v);
  else
    static_cast<float*>(row)[c] = v;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

struct BalArgs {
  const void* logits;   // [T][ld]
  int64_t ld;
  const int32_t* ids;   // [T][K]
  const int32_t* off;   // [S + 1], or nullptr: one sequence of T
  int64_t T;
  int E, K, S;
  int run;              // tokens of a CTA
  int softmax;
  float coeff;
};

// Sequence bounds, kept inside [0, T] and in order whatever `off` holds.
__device__ __forceinline__ void bal_bounds(const BalArgs& a, int s, int64_t* lo, int64_t* hi) {
  if (!a.off) {
    *lo = 0;
    *hi = a.T;
    return;
  }
  const int64_t l = a.off[s], h = a.off[s + 1];
  *lo = l < 0 ? 0 : (l > a.T ? a.T : l);
  *hi = h < *lo ? *lo : (h > a.T ? a.T : h);
}

// First sequence that ends after token t (S if none).
__device__ __forceinline__ int bal_first(const BalArgs& a, int64_t t) {
  if (!a.off) return 0;
  int lo = 0, hi = a.S;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.off[mid + 1] > t)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

// The warp's row: scores x[j] -> a_j (columns lane + 32 j), returns 1 / sum (0
// for a row whose scores sum to zero).
template <int kJ>
__device__ __forceinline__ float bal_scores(float (&x)[kJ], int lane, int E, int softmax) {
  float z = 0.f;
  if (softmax) {
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < kJ; ++j)
      if (lane + 32 * j < E) m = fmaxf(m, x[j]);
    m = warp_max(m);
    // a row of -inf: exp(-inf - 0) = 0 everywhere (a NaN row keeps its NaN)
    if (m == -INFINITY) m = 0.f;
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
      x[j] = lane + 32 * j < E ? expf(x[j] - m) : 0.f;
      z += x[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
      x[j] = lane + 32 * j < E ? 1.0f / (1.0f + expf(-x[j])) : 0.f;
      z += x[j];
    }
  }
  z = warp_sum(z);
  return z == 0.f ? 0.f : 1.0f / z;
}

// Slot layout: psum float [slots][E], pcnt int32 [slots][E].
template <int kDt, int kJ>
__global__ void __launch_bounds__(kBalThreads)
    balance_partial_kernel(BalArgs a, float* __restrict__ psum, int32_t* __restrict__ pcnt) {
  extern __shared__ float sm[];  // [kBalWarps][E] column sums, then [E] counts
  int32_t* cnt = reinterpret_cast<int32_t*>(sm + kBalWarps * a.E);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  griddep_wait();
  griddep_launch_dependents();
  const int64_t t0 = blockIdx.x * static_cast<int64_t>(a.run);
  const int64_t t1 = t0 + a.run < a.T ? t0 + a.run : a.T;
  constexpr int kSize = kDt == 2 ? 4 : 2;
  for (int s = bal_first(a, t0); s < a.S; ++s) {
    int64_t lo, hi;
    bal_bounds(a, s, &lo, &hi);
    if (lo >= t1) break;
    lo = lo > t0 ? lo : t0;
    hi = hi < t1 ? hi : t1;
    if (lo >= hi) continue;
    for (int c = tid; c < a.E; c += kBalThreads) cnt[c] = 0;
    float acc[kJ];
#pragma unroll
    for (int j = 0; j < kJ; ++j) acc[j] = 0.f;
    for (int64_t t = lo + warp; t < hi; t += kBalWarps) {
      const uint8_t* row = static_cast<const uint8_t*>(a.logits) + t * a.ld * kSize;
      float x[kJ];
#pragma unroll
      for (int j = 0; j < kJ; ++j)
        if (lane + 32 * j < a.E) x[j] = bal_load<kDt>(row, lane + 32 * j);
      const float rz = bal_scores<kJ>(x, lane, a.E, a.softmax);
#pragma unroll
      for (int j = 0; j < kJ; ++j) acc[j] = fmaf(x[j], rz, acc[j]);
    }
#pragma unroll
    for (int j = 0; j < kJ; ++j)
      if (lane + 32 * j < a.E) sm[warp * a.E + lane + 32 * j] = acc[j];
    __syncthreads();
    const int64_t n = (hi - lo) * a.K;
    for (int64_t i = tid; i < n; i += kBalThreads) {
      const int32_t id = a.ids[lo * a.K + i];
      if (static_cast<uint32_t>(id) < static_cast<uint32_t>(a.E)) atomicAdd(&cnt[id], 1);
    }
    __syncthreads();
    const int64_t slot = blockIdx.x + static_cast<int64_t>(s);
    for (int c = tid; c < a.E; c += kBalThreads) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kBalWarps; ++w) v += sm[w * a.E + c];
      psum[slot * a.E + c] = v;
      pcnt[slot * a.E + c] = cnt[c];
    }
    __syncthreads();
  }
}

constexpr int kBalFinThreads = 512;

// One CTA a sequence: thread groups of 32 columns x 16 slot lanes.
__global__ void __launch_bounds__(kBalFinThreads)
    balance_final_kernel(BalArgs a, const float* __restrict__ psum, const int32_t* __restrict__ pcnt,
                         float* __restrict__ loss, int32_t* __restrict__ counts) {
  constexpr int kLanes = kBalFinThreads / 32;
  __shared__ double ssum[kLanes][32];
  __shared__ int32_t scnt[kLanes][32];
  const int tid = threadIdx.x, lane = tid & 31, part = tid >> 5;
  const int s = blockIdx.x;
  griddep_wait();
  griddep_launch_dependents();
  int64_t lo, hi;
  bal_bounds(a, s, &lo, &hi);
  const int64_t c0 = lo / a.run + s, c1 = lo < hi ? (hi - 1) / a.run + s + 1 : c0;
  double total = 0.0;
  for (int e0 = 0; e0 < a.E; e0 += 32) {
    const int e = e0 + lane;
    double p = 0.0;
    int32_t n = 0;
    if (e < a.E) {
#pragma unroll 4
      for (int64_t k = c0 + part; k < c1; k += kLanes) {
        p += psum[k * a.E + e];
        n += pcnt[k * a.E + e];
      }
    }
    ssum[part][lane] = p;
    scnt[part][lane] = n;
    __syncthreads();
    if (part == 0 && e < a.E) {
      p = 0.0;
      n = 0;
#pragma unroll
      for (int w = 0; w < kLanes; ++w) {
        p += ssum[w][lane];
        n += scnt[w][lane];
      }
      counts[static_cast<int64_t>(s) * a.E + e] = n;
      total += p * n;
    }
    __syncthreads();
  }
  if (part == 0) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (lane == 0) {
      const double len = static_cast<double>(hi - lo);
      loss[s] = hi > lo ? static_cast<float>(a.coeff * total * a.E / (a.K * len * len)) : 0.f;
    }
  }
}

// Gradient of sum_s grad_loss[s] * loss[s]: one warp a token, f of the
// token's sequence in registers.
template <int kDt, int kJ>
__global__ void __launch_bounds__(kBalThreads)
    balance_backward_kernel(BalArgs a, const int32_t* __restrict__ counts, const float* __restrict__ grad_loss,
                            void* __restrict__ grad) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  griddep_wait();
  griddep_launch_dependents();
  const int64_t t0 = blockIdx.x * static_cast<int64_t>(a.run);
  const int64_t t1 = t0 + a.run < a.T ? t0 + a.run : a.T;
  constexpr int kSize = kDt == 2 ? 4 : 2;
  int64_t done = t0;  // tokens before this one have their gradient
  auto zero = [&](int64_t lo, int64_t hi) {
    for (int64_t t = lo + warp; t < hi; t += kBalWarps) {
      uint8_t* row = static_cast<uint8_t*>(grad) + t * a.E * kSize;
      for (int c = lane; c < a.E; c += 32) bal_store<kDt>(row, c, 0.f);
    }
  };
  for (int s = bal_first(a, t0); s < a.S; ++s) {
    int64_t lo, hi;
    bal_bounds(a, s, &lo, &hi);
    if (lo >= t1) break;
    const float len = static_cast<float>(hi - lo);
    lo = lo > done ? lo : done;
    hi = hi < t1 ? hi : t1;
    if (lo >= hi) continue;
    zero(done, lo);
    const float unit = static_cast<float>(a.E) / (static_cast<float>(a.K) * len);
    const float g = grad_loss[s] * a.coeff / len;
    float f[kJ];
#pragma unroll
    for (int j = 0; j < kJ; ++j)
      f[j] = lane + 32 * j < a.E ? unit * static_cast<float>(counts[static_cast<int64_t>(s) * a.E + lane + 32 * j]) : 0.f;
    for (int64_t t = lo + warp; t < hi; t += kBalWarps) {
      const uint8_t* row = static_cast<const uint8_t*>(a.logits) + t * a.ld * kSize;
      uint8_t* out = static_cast<uint8_t*>(grad) + t * a.E * kSize;
      float x[kJ];
#pragma unroll
      for (int j = 0; j < kJ; ++j)
        if (lane + 32 * j < a.E) x[j] = bal_load<kDt>(row, lane + 32 * j);
      const float rz = bal_scores<kJ>(x, lane, a.E, a.softmax);
      float dot = 0.f;
#pragma unroll
      for (int j = 0; j < kJ; ++j) dot = fmaf(f[j], x[j], dot);
      dot = warp_sum(dot) * rz;
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        float d = g * (x[j] * rz) * (f[j] - dot);
        if (!a.softmax) d *= 1.0f - x[j];
        if (lane + 32 * j < a.E) bal_store<kDt>(out, lane + 32 * j, d);
      }
    }
    done = hi;
  }
  zero(done, t1);
}

// Tokens of a CTA: two CTAs' worth on every SM before runs grow past 16 tokens.
int bal_run(int64_t T) {
  const int64_t per = (T + 2 * kSMs - 1) / (2 * kSMs);
  return static_cast<int>(per < 16 ? 16 : per);
}

#define BAL_J(KERNEL, D)                                             \
  (E <= 32 ? KERNEL<D, 1> : E <= 64 ? KERNEL<D, 2> : E <= 128 ? KERNEL<D, 4> \
   : E <= 256 ? KERNEL<D, 8> : E <= 512 ? KERNEL<D, 16> : KERNEL<D, 32>)

BalArgs bal_args(const BalanceCall& c) {
  BalArgs a{};
  a.logits = c.logits;
  a.ld = c.ld;
  a.ids = c.ids;
  a.off = c.off;
  a.T = c.T;
  a.E = c.E;
  a.K = c.K;
  a.S = c.S;
  a.run = bal_run(c.T);
  a.softmax = c.softmax;
  a.coeff = c.coeff;
  return a;
}

uint32_t bal_grid(const BalArgs& a) { return static_cast<uint32_t>((a.T + a.run - 1) / a.run); }

}  // namespace

int64_t balance_slots(int64_t T, int64_t S) {
  const int run = bal_run(T);
  return (T + run - 1) / run + S;
}

cudaError_t launch_balance(const BalanceCall& c, void* work, float* loss, int32_t* counts, cudaStream_t s) {
  const BalArgs a = bal_args(c);
  const int E = c.E;
  float* psum = static_cast<float*>(work);
  int32_t* pcnt = reinterpret_cast<int32_t*>(psum + balance_slots(c.T, c.S) * E);
  if (a.T > 0) {
    auto k = c.dt == 0 ? BAL_J(balance_partial_kernel, 0) : c.dt == 1 ? BAL_J(balance_partial_kernel, 1)
                                                                       : BAL_J(balance_partial_kernel, 2);
    const size_t smem = static_cast<size_t>(kBalWarps + 1) * E * 4;  // 36 KB at E = 1024
    const cudaError_t e = launch_k(k, dim3(bal_grid(a)), dim3(kBalThreads), smem, s, true, a, psum, pcnt);
    if (e != cudaSuccess) return e;
  }
  return launch_k(balance_final_kernel, dim3(c.S), dim3(kBalFinThreads), 0, s, true, a,
                  static_cast<const float*>(psum), static_cast<const int32_t*>(pcnt), loss, counts);
}

cudaError_t launch_balance_backward(const BalanceCall& c, const int32_t* counts, const float* grad_loss, void* grad,
                                    cudaStream_t s) {
  if (c.T == 0) return cudaSuccess;
  const BalArgs a = bal_args(c);
  const int E = c.E;
  auto k = c.dt == 0 ? BAL_J(balance_backward_kernel, 0) : c.dt == 1 ? BAL_J(balance_backward_kernel, 1)
                                                                      : BAL_J(balance_backward_kernel, 2);
  return launch_k(k, dim3(bal_grid(a)), dim3(kBalThreads), 0, s, true, a, counts, grad_loss, grad);
}

}  // namespace moe
