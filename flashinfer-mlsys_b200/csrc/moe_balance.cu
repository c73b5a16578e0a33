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
// An empty sequence has loss 0; a token whose float32 scores sum to zero (every
// logit -inf, or under -87 for sigmoids) has p = 0 and no gradient; ids outside
// [0, E) are not counted; tokens of no sequence get a zero gradient.
//
// HBM-bound: one pass over the logits forward, one (and the gradient) back.
// Forward: CTAs own equal runs of tokens, whatever the sequences' lengths. A
// run meets a sequence in one segment; (run index + sequence index) grows
// along the segments, so it numbers them without gaps to search for, and each
// segment's fp32 column sums and counts go to a slot of their own. A second
// kernel adds a sequence's slots in order. No atomics on floats: results do
// not depend on the order in which CTAs run. 65536 x 256 fp32 in 13 sequences:
// forward 22.8 us (2.9 TB/s), backward 28.9 us (4.6 TB/s); 16384 x 256: 11.5 and
// 10.7 us, of which launches and dependent loads are the most.
#include "moe_kernels.h"

namespace moe {

namespace {

constexpr int kBalWarps = 16;
constexpr int kBalThreads = kBalWarps * 32;
// Rows a warp has in flight, for `n` columns a lane (more registers than there are beyond that).
__host__ __device__ constexpr int bal_batch(int n) { return n >= 32 ? 1 : 4; }

// Columns of a lane: kV neighbours, every 32 kV (kV = 4 where the rows allow
// vector loads, else 1).
template <int kDt, int kV>
__device__ __forceinline__ void bal_load(const void* row, int c, float* v) {
  if constexpr (kV == 1) {
    if constexpr (kDt == 0) v[0] = __bfloat162float(static_cast<const __nv_bfloat16*>(row)[c]);
    if constexpr (kDt == 1) v[0] = __half2float(static_cast<const __half*>(row)[c]);
    if constexpr (kDt == 2) v[0] = static_cast<const float*>(row)[c];
  } else if constexpr (kDt == 2) {
    const float4 t = *reinterpret_cast<const float4*>(static_cast<const float*>(row) + c);
    v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
  } else {
    const uint2 t = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(row) + c);
    const uint32_t w[2] = {t.x, t.y};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 f = kDt == 0 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]))
                                : __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}
template <int kDt, int kV>
__device__ __forceinline__ void bal_store(void* row, int c, const float* v) {
  if constexpr (kV == 1) {
    if constexpr (kDt == 0) static_cast<__nv_bfloat16*>(row)[c] = __float2bfloat16_rn(v[0]);
    if constexpr (kDt == 1) static_cast<__half*>(row)[c] = __float2half_rn(v[0]);
    if constexpr (kDt == 2) static_cast<float*>(row)[c] = v[0];
  } else if constexpr (kDt == 2) {
    *reinterpret_cast<float4*>(static_cast<float*>(row) + c) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (kDt == 0) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&t);
      } else {
        const __half2 t = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&t);
      }
    }
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(row) + c) = make_uint2(w[0], w[1]);
  }
}

// Sums (maxima) over the warp of several rows at once: their shuffles overlap.
template <int kB>
__device__ __forceinline__ void warp_sums(float (&v)[kB]) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1)
#pragma unroll
    for (int b = 0; b < kB; ++b) v[b] += __shfl_xor_sync(0xffffffffu, v[b], o);
}
template <int kB>
__device__ __forceinline__ void warp_maxima(float (&v)[kB]) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1)
#pragma unroll
    for (int b = 0; b < kB; ++b) v[b] = fmaxf(v[b], __shfl_xor_sync(0xffffffffu, v[b], o));
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

// Sequence bounds, kept inside [0, T], and the end not before the start. Offsets
// that decrease from one sequence to the next are not put in order: sequences
// then overlap, may share a slot and have no defined sums, inside their bounds.
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

// First sequence that ends after token t (S if none): the number of those that
// do not, counted by the whole CTA (one load deep, where a search is five or more).
__device__ __forceinline__ int bal_first(const BalArgs& a, int64_t t) {
  if (!a.off) return 0;
  int n = 0;
  for (int s0 = 0; s0 < a.S; s0 += kBalThreads) {
    const int s = s0 + threadIdx.x;
    const int got = __syncthreads_count(s < a.S && a.off[s + 1] <= t);
    n += got;
    if (got < kBalThreads) break;
  }
  return n;
}

// The logits of rows t, t + kBalWarps, ... (nb of them, at most kB) -> scores
// a_j (0 in columns that are not there); rz: 1 / their sum, 0 where the scores
// sum to zero. For the gradient (kBack) x becomes d a_j / d l_j instead, a
// sigmoid's y (1 - y) as y e y with e = exp(-l), as 1 - y has lost all digits of
// a y near 1; and dot becomes sum_j f_j a_j. The quotient's fast form is within
// 2 steps of float32 for the 1 + e it meets. The exponential's is not taken: its
// error grows by 1.2 |l| steps, for 4 us of 53 (65536 x 256 fp32 forward and
// backward).
template <int kDt, int kV, int kJ, int kB, bool kBack>
__device__ __forceinline__ void bal_scores(const BalArgs& a, int64_t t, int nb, int lane, const float* f,
                                           float (&x)[kB][kJ * kV], float (&rz)[kB], float (&dot)[kB]) {
  constexpr int kSize = kDt == 2 ? 4 : 2;
#pragma unroll
  for (int b = 0; b < kB; ++b) {
    if (b >= nb) break;
    const uint8_t* row = static_cast<const uint8_t*>(a.logits) + (t + b * kBalWarps) * a.ld * kSize;
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
      const int c = (j * 32 + lane) * kV;
      if (c < a.E) {
        bal_load<kDt, kV>(row, c, &x[b][j * kV]);
      } else {
#pragma unroll
        for (int v = 0; v < kV; ++v) x[b][j * kV + v] = -INFINITY;  // scores 0
      }
    }
  }
  float m[kB];
  if (a.softmax) {
#pragma unroll
    for (int b = 0; b < kB; ++b) {
      m[b] = -INFINITY;
      if (b >= nb) continue;
#pragma unroll
      for (int i = 0; i < kJ * kV; ++i) m[b] = fmaxf(m[b], x[b][i]);
    }
    warp_maxima(m);
  }
#pragma unroll
  for (int b = 0; b < kB; ++b) {
    rz[b] = 0.f;
    dot[b] = 0.f;
    if (b >= nb) continue;
    if (a.softmax) {
      // a row of -inf: exp(-inf - 0) = 0 everywhere (a NaN row keeps its NaN)
      const float top = m[b] == -INFINITY ? 0.f : m[b];
#pragma unroll
      for (int i = 0; i < kJ * kV; ++i) {
        const float y = expf(x[b][i] - top);
        rz[b] += y;
        if constexpr (kBack) dot[b] = fmaf(f[i], y, dot[b]);
        x[b][i] = y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kJ * kV; ++i) {
        const float e = expf(-x[b][i]), y = __fdividef(1.0f, 1.0f + e);  // 0 where e passes 2^126
        rz[b] += y;
        if constexpr (kBack) {
          dot[b] = fmaf(f[i], y, dot[b]);
          x[b][i] = fminf(e, 0x1p127f) * y * y;
        } else {
          x[b][i] = y;
        }
      }
    }
  }
  warp_sums(rz);
  if constexpr (kBack) warp_sums(dot);
#pragma unroll
  for (int b = 0; b < kB; ++b) rz[b] = rz[b] == 0.f ? 0.f : 1.0f / rz[b];
}

// Rows of a warp's next batch: t, t + kBalWarps, ... below hi.
template <int kB>
__device__ __forceinline__ int bal_rows(int64_t t, int64_t hi) {
  const int64_t n = (hi - t + kBalWarps - 1) / kBalWarps;
  return n < kB ? static_cast<int>(n) : kB;
}

// Slot layout: psum float [slots][E], pcnt int32 [slots][E].
template <int kDt, int kV, int kJ>
__global__ void __launch_bounds__(kBalThreads, kJ * kV <= 8 ? 2 : 1)
    balance_partial_kernel(BalArgs a, float* __restrict__ psum, int32_t* __restrict__ pcnt) {
  extern __shared__ float sm[];  // [kBalWarps][E] column sums, then [E] counts
  int32_t* cnt = reinterpret_cast<int32_t*>(sm + kBalWarps * a.E);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  griddep_wait();
  griddep_launch_dependents();
  const int64_t t0 = blockIdx.x * static_cast<int64_t>(a.run);
  const int64_t t1 = t0 + a.run < a.T ? t0 + a.run : a.T;
  for (int s = bal_first(a, t0); s < a.S; ++s) {
    int64_t lo, hi;
    bal_bounds(a, s, &lo, &hi);
    if (lo >= t1) break;
    lo = lo > t0 ? lo : t0;
    hi = hi < t1 ? hi : t1;
    if (lo >= hi) continue;
    for (int c = tid; c < a.E; c += kBalThreads) cnt[c] = 0;
    __syncthreads();
    const int64_t n = (hi - lo) * a.K;
    for (int64_t i = tid; i < n; i += kBalThreads) {
      const int32_t id = a.ids[lo * a.K + i];
      if (static_cast<uint32_t>(id) < static_cast<uint32_t>(a.E)) atomicAdd(&cnt[id], 1);
    }
    float acc[kJ * kV];
#pragma unroll
    for (int i = 0; i < kJ * kV; ++i) acc[i] = 0.f;
    constexpr int kB = bal_batch(kJ * kV);
    for (int64_t t = lo + warp; t < hi; t += kB * kBalWarps) {
      float x[kB][kJ * kV], rz[kB], unused[kB];
      const int nb = bal_rows<kB>(t, hi);
      bal_scores<kDt, kV, kJ, kB, false>(a, t, nb, lane, nullptr, x, rz, unused);
#pragma unroll
      for (int b = 0; b < kB; ++b) {
        if (b >= nb) break;
#pragma unroll
        for (int i = 0; i < kJ * kV; ++i) acc[i] = fmaf(x[b][i], rz[b], acc[i]);
      }
    }
#pragma unroll
    for (int j = 0; j < kJ; ++j)
#pragma unroll
      for (int v = 0; v < kV; ++v) {
        const int c = (j * 32 + lane) * kV + v;
        if (c < a.E) sm[warp * a.E + c] = acc[j * kV + v];
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

constexpr int kBalFinThreads = 1024;

// One CTA a sequence: 256 columns at a time x 4 threads, which take every
// fourth slot each, thirty-two loads in flight.
__global__ void __launch_bounds__(kBalFinThreads)
    balance_final_kernel(BalArgs a, const float* __restrict__ psum, const int32_t* __restrict__ pcnt,
                         float* __restrict__ loss, int32_t* __restrict__ counts) {
  constexpr int kCols = 256, kParts = kBalFinThreads / kCols;
  __shared__ double ssum[kParts][kCols];
  __shared__ int32_t scnt[kParts][kCols];
  __shared__ double wsum[kCols / 32];
  const int tid = threadIdx.x, col = tid % kCols, part = tid / kCols;
  const int s = blockIdx.x;
  griddep_wait();
  griddep_launch_dependents();
  int64_t lo, hi;
  bal_bounds(a, s, &lo, &hi);
  const int64_t c0 = lo / a.run + s, c1 = lo < hi ? (hi - 1) / a.run + s + 1 : c0;
  double total = 0.0;
  for (int e0 = 0; e0 < a.E; e0 += kCols) {
    const int e = e0 + col;
    double p = 0.0;
    int32_t n = 0;
    if (e < a.E) {
#pragma unroll 16
      for (int64_t k = c0 + part; k < c1; k += kParts) {
        p += psum[k * a.E + e];
        n += pcnt[k * a.E + e];
      }
    }
    ssum[part][col] = p;
    scnt[part][col] = n;
    __syncthreads();
    if (part == 0 && e < a.E) {
      p = 0.0;
      n = 0;
#pragma unroll
      for (int w = 0; w < kParts; ++w) {
        p += ssum[w][col];
        n += scnt[w][col];
      }
      counts[static_cast<int64_t>(s) * a.E + e] = n;
      total += p * n;
    }
    __syncthreads();
  }
  if (part == 0) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if ((col & 31) == 0) wsum[col / 32] = total;
  }
  __syncthreads();
  if (tid == 0) {
    total = 0.0;
#pragma unroll
    for (int w = 0; w < kCols / 32; ++w) total += wsum[w];
    const double len = static_cast<double>(hi - lo);
    loss[s] = hi > lo ? static_cast<float>(a.coeff * total * a.E / (a.K * len * len)) : 0.f;
  }
}

// Gradient of sum_s grad_loss[s] * loss[s]: a warp takes some tokens at a
// time, f of their sequence in registers.
template <int kDt, int kV, int kJ>
__global__ void __launch_bounds__(kBalThreads, kJ * kV <= 8 ? 2 : 1)
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
    const float z[1] = {0.f};
    for (int64_t t = lo + warp; t < hi; t += kBalWarps) {
      uint8_t* row = static_cast<uint8_t*>(grad) + t * a.E * kSize;
      for (int c = lane; c < a.E; c += 32) bal_store<kDt, 1>(row, c, z);
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
    const float per = static_cast<float>(a.E) / (static_cast<float>(a.K) * len);  // f of one slot
    const float g = grad_loss[s] * a.coeff / len;
    float f[kJ * kV];
#pragma unroll
    for (int j = 0; j < kJ; ++j)
#pragma unroll
      for (int v = 0; v < kV; ++v) {
        const int c = (j * 32 + lane) * kV + v;
        f[j * kV + v] = c < a.E ? per * static_cast<float>(counts[static_cast<int64_t>(s) * a.E + c]) : 0.f;
      }
    constexpr int kB = bal_batch(kJ * kV);
    for (int64_t t = lo + warp; t < hi; t += kB * kBalWarps) {
      float x[kB][kJ * kV], rz[kB], dot[kB];
      const int nb = bal_rows<kB>(t, hi);
      bal_scores<kDt, kV, kJ, kB, true>(a, t, nb, lane, f, x, rz, dot);
#pragma unroll
      for (int b = 0; b < kB; ++b) {
        if (b >= nb) break;
        const int64_t r = t + b * kBalWarps;
        const float mean = dot[b] * rz[b];
        uint8_t* row = static_cast<uint8_t*>(grad) + r * a.E * kSize;
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
          const int c = (j * 32 + lane) * kV;
          float d[kV];
#pragma unroll
          for (int v = 0; v < kV; ++v) d[v] = g * (x[b][j * kV + v] * rz[b]) * (f[j * kV + v] - mean);
          if (c < a.E) bal_store<kDt, kV>(row, c, d);
        }
      }
    }
    done = hi;
  }
  zero(done, t1);
}

// Tokens of a CTA: a CTA on every SM, two for many tokens, before runs grow past
// a row of every warp. (Two at 16384 x 256 leave the second kernel twice the
// slots to add: a single sequence took 17.0 instead of 14.5 us.)
int bal_run(int64_t T) {
  const int64_t ctas = T > 32768 ? 2 * kSMs : kSMs;
  const int64_t per = (T + ctas - 1) / ctas;
  return static_cast<int>(per < kBalWarps ? kBalWarps : per);
}

// Vector columns where every row of 4 is aligned.
bool bal_vector(const BalanceCall& c, const void* grad) {
  const int64_t size = c.dt == 2 ? 4 : 2;
  return c.E % 4 == 0 && c.ld % 4 == 0 && reinterpret_cast<uintptr_t>(c.logits) % (4 * size) == 0 &&
         reinterpret_cast<uintptr_t>(grad) % (4 * size) == 0;
}

#define BAL_DT(KERNEL, V, J) (dt == 0 ? KERNEL<0, V, J> : dt == 1 ? KERNEL<1, V, J> : KERNEL<2, V, J>)
#define BAL_PICK(KERNEL)                                                                                      \
  (vec ? (E <= 128 ? BAL_DT(KERNEL, 4, 1) : E <= 256 ? BAL_DT(KERNEL, 4, 2)                                   \
                   : E <= 512 ? BAL_DT(KERNEL, 4, 4) : BAL_DT(KERNEL, 4, 8))                                  \
       : (E <= 32 ? BAL_DT(KERNEL, 1, 1) : E <= 128 ? BAL_DT(KERNEL, 1, 4)                                    \
                  : E <= 512 ? BAL_DT(KERNEL, 1, 16) : BAL_DT(KERNEL, 1, 32)))

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

dim3 bal_grid(const BalArgs& a) { return dim3(static_cast<uint32_t>((a.T + a.run - 1) / a.run)); }

}  // namespace

int64_t balance_slots(int64_t T, int64_t S) {
  const int run = bal_run(T);
  return (T + run - 1) / run + S;
}

cudaError_t launch_balance(const BalanceCall& c, void* work, float* loss, int32_t* counts, cudaStream_t s) {
  const BalArgs a = bal_args(c);
  const int E = c.E, dt = c.dt;
  const bool vec = bal_vector(c, nullptr);
  float* psum = static_cast<float*>(work);
  int32_t* pcnt = reinterpret_cast<int32_t*>(psum + balance_slots(c.T, c.S) * E);
  if (a.T > 0) {
    auto k = BAL_PICK(balance_partial_kernel);
    const size_t smem = static_cast<size_t>(kBalWarps + 1) * E * 4;  // 68 KB at E = 1024
    if (smem > 48 * 1024) {
      const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
      if (e != cudaSuccess) return e;
    }
    const cudaError_t e = launch_k(k, bal_grid(a), dim3(kBalThreads), smem, s, true, a, psum, pcnt);
    if (e != cudaSuccess) return e;
  }
  return launch_k(balance_final_kernel, dim3(c.S), dim3(kBalFinThreads), 0, s, true, a,
                  static_cast<const float*>(psum), static_cast<const int32_t*>(pcnt), loss, counts);
}

cudaError_t launch_balance_backward(const BalanceCall& c, const int32_t* counts, const float* grad_loss, void* grad,
                                    cudaStream_t s) {
  if (c.T == 0) return cudaSuccess;
  const BalArgs a = bal_args(c);
  const int E = c.E, dt = c.dt;
  const bool vec = bal_vector(c, grad);
  auto k = BAL_PICK(balance_backward_kernel);
  return launch_k(k, bal_grid(a), dim3(kBalThreads), 0, s, true, a, counts, grad_loss, grad);
}

}  // namespace moe
