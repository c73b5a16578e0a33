// moe_mx_quant.cu — rows of bf16, fp16 or fp32 to a microscaled format
// (moe_mx.cuh) and back, and the residual add + RMSNorm that ends in one.
//
// All three are one pass over the data and HBM-bound. One thread owns one unit
// (32 columns): a block's scale needs no exchange between threads, the packed
// values leave as one or two 16-byte stores, and neighbouring threads' units
// are adjacent, so every 32-byte sector is used whole.
#include "moe_kernels.h"
#include "moe_mx.cuh"

namespace moe {

namespace {

constexpr int kMxThreads = 256;

__device__ __forceinline__ void store_scale(void* scale, uint64_t unit, int per_unit, uint32_t sc) {
  if (per_unit == 2)
    static_cast<uint16_t*>(scale)[unit] = static_cast<uint16_t>(sc);
  else
    static_cast<uint8_t*>(scale)[unit] = static_cast<uint8_t>(sc);
}

// x [rows][x_ld] -> q, scale (both contiguous); `per_row` units a row.
template <int kFmt, int kDt>
__global__ void __launch_bounds__(kMxThreads)
    mx_quant_kernel(const uint8_t* __restrict__ x, int64_t x_ld_bytes, uint64_t units, uint32_t per_row,
                    const float* __restrict__ global_scale, uint8_t* __restrict__ q, void* __restrict__ scale) {
  const uint64_t u = blockIdx.x * static_cast<uint64_t>(kMxThreads) + threadIdx.x;
  griddep_wait();
  griddep_launch_dependents();
  if (u >= units) return;
  const uint64_t row = u / per_row;
  const uint32_t c = static_cast<uint32_t>(u - row * per_row);
  constexpr int kW = MxWords<kDt>::n;
  uint32_t w[kW];
  mx_load<kW>(x + row * x_ld_bytes + static_cast<uint64_t>(c) * (4 * kW), w);
  const float g = (kFmt == kFmtNvfp4 && global_scale) ? __ldg(global_scale) : 1.0f;
  float f[32];
  mx_to_float<kDt>(w, f);
  uint32_t am[2];
  if constexpr (kDt == kDtFp32)
    mx_amax<kFmt>(f, am);
  else
    mx_amax_packed<kFmt, kDt>(w, am);
  uint32_t o[8];
  const uint32_t sc = mx_quant_unit<kFmt>(f, am, g, o);
  constexpr int kB = mx_unit_bytes(kFmt);
  mx_store<kB / 4>(q + u * kB, o);
  store_scale(scale, u, mx_unit_scales(kFmt), sc);
}

// q, scale (contiguous) -> x [rows][x_ld]: (value * scale) * global_scale in
// float32 (the first product is exact), rounded once to the output's type.
template <int kFmt, int kDt>
__global__ void __launch_bounds__(kMxThreads)
    mx_dequant_kernel(const uint8_t* __restrict__ q, const void* __restrict__ scale, uint64_t units, uint32_t per_row,
                      const float* __restrict__ global_scale, uint8_t* __restrict__ x, int64_t x_ld_bytes) {
  const uint64_t u = blockIdx.x * static_cast<uint64_t>(kMxThreads) + threadIdx.x;
  griddep_wait();
  griddep_launch_dependents();
  if (u >= units) return;
  const uint64_t row = u / per_row;
  const uint32_t c = static_cast<uint32_t>(u - row * per_row);
  constexpr int kB = mx_unit_bytes(kFmt);
  uint32_t o[kB / 4];
  mx_load<kB / 4>(q + u * kB, o);
  float s[2];
  if constexpr (kFmt == kFmtNvfp4) {
    const float2 v = e4m3x2_to_f2(static_cast<const uint16_t*>(scale)[u]);
    s[0] = v.x;
    s[1] = v.y;
  } else {
    s[0] = s[1] = e8m0_to_f(static_cast<const uint8_t*>(scale)[u]);
  }
  const float g = (kFmt == kFmtNvfp4 && global_scale) ? __ldg(global_scale) : 1.0f;
  float f[32];
#pragma unroll
  for (int i = 0; i < kB / 4; ++i) {
    if constexpr (kFmt == kFmtMxfp8) {
      const float2 lo = e4m3x2_to_f2(o[i] & 0xFFFFu), hi = e4m3x2_to_f2(o[i] >> 16);
      f[4 * i] = lo.x;
      f[4 * i + 1] = lo.y;
      f[4 * i + 2] = hi.x;
      f[4 * i + 3] = hi.y;
    } else {
      e2m1x8_to_f8(o[i], f + 8 * i);
    }
  }
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    f[i] *= s[i / 16];
    if (kFmt == kFmtNvfp4) f[i] *= g;
  }
  constexpr int kW = MxWords<kDt>::n;
  uint32_t w[kW];
  mx_from_float<kDt>(f, w);
  mx_store<kW>(x + row * x_ld_bytes + static_cast<uint64_t>(c) * (4 * kW), w);
}

// h = T(residual + x) (written back), y = h / sqrt(mean(h^2) + eps) * weight
// in float32, then the unit's quantisation. `tpr` threads hold a row (one unit
// each): a power of two up to 32, several rows a CTA, or one row a CTA. The
// sum of squares goes through 32 values a thread, an xor butterfly over the
// row's lanes and the warps in order, all in float32, so it does not depend on
// the launch. Without a weight: y = h.
template <int kFmt, int kDt, int kMaxT>
__global__ void __launch_bounds__(kMaxT)
    mx_norm_kernel(const uint8_t* __restrict__ x, int64_t x_ld_bytes, uint8_t* residual, int64_t res_ld_bytes,
                   const uint8_t* __restrict__ weight, float eps, int64_t rows, uint32_t per_row, uint32_t tpr,
                   const float* __restrict__ global_scale, uint8_t* __restrict__ q, void* __restrict__ scale) {
  __shared__ float warp_ss[32];
  griddep_wait();
  griddep_launch_dependents();
  const uint32_t tid = threadIdx.x;
  const bool whole = tpr > 32;  // one row for the CTA
  const int64_t row = whole ? blockIdx.x : blockIdx.x * static_cast<int64_t>(blockDim.x / tpr) + tid / tpr;
  const uint32_t c = whole ? tid : tid % tpr;
  const bool live = row < rows && c < per_row;
  constexpr int kW = MxWords<kDt>::n;
  float f[32];
  if (live) {
    uint32_t w[kW];
    mx_load<kW>(x + row * x_ld_bytes + static_cast<int64_t>(c) * (4 * kW), w);
    if (residual) {
      uint8_t* rp = residual + row * res_ld_bytes + static_cast<int64_t>(c) * (4 * kW);
      uint32_t rw[kW];
      mx_load<kW>(rp, rw);
      float r[32];
      mx_to_float<kDt>(w, f);
      mx_to_float<kDt>(rw, r);
#pragma unroll
      for (int i = 0; i < 32; ++i) f[i] += r[i];
      mx_from_float<kDt>(f, w);
      mx_store<kW>(rp, w);
    }
    mx_to_float<kDt>(w, f);
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) f[i] = 0.f;
  }
  if (weight) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) ss = fmaf(f[i], f[i], ss);
    for (uint32_t off = whole ? 16 : tpr / 2; off >= 1; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
    if (whole) {
      if ((tid & 31) == 0) warp_ss[tid >> 5] = ss;
      __syncthreads();
      ss = 0.f;
      for (uint32_t i = 0; i < blockDim.x / 32; ++i) ss += warp_ss[i];
    }
    const float mean = __fdiv_rn(ss, static_cast<float>(per_row * kMxUnit));
    const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(mean, eps)));
    if (live) {
      uint32_t w[kW];
      const uint4* wp = reinterpret_cast<const uint4*>(weight + static_cast<int64_t>(c) * (4 * kW));
#pragma unroll
      for (int i = 0; i < kW / 4; ++i) {
        const uint4 v = __ldg(wp + i);
        w[4 * i] = v.x;
        w[4 * i + 1] = v.y;
        w[4 * i + 2] = v.z;
        w[4 * i + 3] = v.w;
      }
      float wf[32];
      mx_to_float<kDt>(w, wf);
#pragma unroll
      for (int i = 0; i < 32; ++i) f[i] = __fmul_rn(__fmul_rn(f[i], inv), wf[i]);
    }
  }
  if (!live) return;
  uint32_t am[2];
  mx_amax<kFmt>(f, am);
  const float g = (kFmt == kFmtNvfp4 && global_scale) ? __ldg(global_scale) : 1.0f;
  uint32_t o[8];
  const uint32_t sc = mx_quant_unit<kFmt>(f, am, g, o);
  constexpr int kB = mx_unit_bytes(kFmt);
  const uint64_t u = static_cast<uint64_t>(row) * per_row + c;
  mx_store<kB / 4>(q + u * kB, o);
  store_scale(scale, u, mx_unit_scales(kFmt), sc);
}

constexpr int64_t dt_bytes(int dt) { return dt == kDtFp32 ? 4 : 2; }

// Calls fn<fmt, dt>() for the run-time pair.
#define MX_DISPATCH(fmt, dt, CALL)                     \
  switch ((fmt) * 3 + (dt)) {                          \
    case 0: return CALL(kFmtNvfp4, kDtBf16);           \
    case 1: return CALL(kFmtNvfp4, kDtFp16);           \
    case 2: return CALL(kFmtNvfp4, kDtFp32);           \
    case 3: return CALL(kFmtMxfp4, kDtBf16);           \
    case 4: return CALL(kFmtMxfp4, kDtFp16);           \
    case 5: return CALL(kFmtMxfp4, kDtFp32);           \
    case 6: return CALL(kFmtMxfp8, kDtBf16);           \
    case 7: return CALL(kFmtMxfp8, kDtFp16);           \
    default: return CALL(kFmtMxfp8, kDtFp32);          \
  }

template <int kFmt, int kDt>
cudaError_t norm_launch(const MxNormCall& c, cudaStream_t s) {
  const uint32_t per_row = static_cast<uint32_t>(c.cols / kMxUnit);
  uint32_t tpr = 1;
  while (tpr < per_row && tpr < 32) tpr *= 2;
  const bool whole = per_row > 32;
  const uint32_t threads = whole ? (per_row + 31) / 32 * 32 : 128;
  if (whole) tpr = threads;
  const int64_t grid = whole ? c.rows : (c.rows + 128 / tpr - 1) / (128 / tpr);
  auto go = [&](auto kernel) {
    return launch_k(kernel, dim3(static_cast<uint32_t>(grid)), dim3(threads), 0, s, true,
                    static_cast<const uint8_t*>(c.x), c.x_ld * dt_bytes(kDt), static_cast<uint8_t*>(c.residual),
                    c.res_ld * dt_bytes(kDt), static_cast<const uint8_t*>(c.weight), c.eps, c.rows, per_row, tpr,
                    c.global_scale, static_cast<uint8_t*>(c.q), c.scale);
  };
  // rows of up to 8192 columns keep a bound that leaves the compiler 255 registers
  if (threads <= 256) return go(mx_norm_kernel<kFmt, kDt, 256>);
  return go(mx_norm_kernel<kFmt, kDt, 1024>);
}

}  // namespace

cudaError_t launch_mx_quant(const void* x, int dt, int64_t x_ld, int64_t rows, int64_t cols, int fmt,
                            const float* global_scale, void* q, void* scale, cudaStream_t s) {
  const uint32_t per_row = static_cast<uint32_t>(cols / kMxUnit);
  const uint64_t units = static_cast<uint64_t>(rows) * per_row;
  if (units == 0) return cudaSuccess;
  const dim3 grid(static_cast<uint32_t>((units + kMxThreads - 1) / kMxThreads));
#define CALL(F, D)                                                                                              \
  launch_k(mx_quant_kernel<F, D>, grid, dim3(kMxThreads), 0, s, true, static_cast<const uint8_t*>(x),           \
           x_ld * dt_bytes(D), units, per_row, global_scale, static_cast<uint8_t*>(q), scale)
  MX_DISPATCH(fmt, dt, CALL)
#undef CALL
}

cudaError_t launch_mx_dequant(const void* q, const void* scale, int64_t rows, int64_t cols, int fmt,
                              const float* global_scale, int dt, void* x, int64_t x_ld, cudaStream_t s) {
  const uint32_t per_row = static_cast<uint32_t>(cols / kMxUnit);
  const uint64_t units = static_cast<uint64_t>(rows) * per_row;
  if (units == 0) return cudaSuccess;
  const dim3 grid(static_cast<uint32_t>((units + kMxThreads - 1) / kMxThreads));
#define CALL(F, D)                                                                                              \
  launch_k(mx_dequant_kernel<F, D>, grid, dim3(kMxThreads), 0, s, true, static_cast<const uint8_t*>(q), scale, units, \
           per_row, global_scale, static_cast<uint8_t*>(x), x_ld * dt_bytes(D))
  MX_DISPATCH(fmt, dt, CALL)
#undef CALL
}

cudaError_t launch_mx_norm(const MxNormCall& c, int fmt, int dt, cudaStream_t s) {
  if (c.rows == 0 || c.cols == 0) return cudaSuccess;
#define CALL(F, D) norm_launch<F, D>(c, s)
  MX_DISPATCH(fmt, dt, CALL)
#undef CALL
}

}  // namespace moe
