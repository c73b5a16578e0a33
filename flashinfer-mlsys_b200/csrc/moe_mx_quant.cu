// moe_mx_quant.cu — rows of bf16, fp16 or fp32 to a microscaled format
// (moe_mx.cuh) and back, and the residual add + RMSNorm that ends in one.
//
// All three are one pass over the data and HBM-bound. The register bounds are
// measured at 16384 x 7168: 16-bit rows gain 3 to 5% from more CTAs on an SM
// (the norm 149 -> 142 us with nvfp4, 140 -> 136 us with mxfp8), fp32 rows
// would spill (233 -> 354 us) and keep three CTAs (two: 140 us at 8192 rows, not 119). At 16384 x 7168 bf16: quantisation 54 us nvfp4
// (5.5 TB/s; some 12 instructions a value nearly bind), 46 us mxfp4, 52 us mxfp8
// (6.8 TB/s), dequantisation 45 us (6.6 TB/s), residual + norm + mxfp8 134 us
// (6.1 TB/s), nvfp4 144 us; fp32 rows 6.3 to 7.1 TB/s.
#include "moe_kernels.h"
#include "moe_mx.cuh"

namespace moe {

namespace {

constexpr int kMxThreads = 256;
constexpr int kQuantPer = 2;    // spans of a quantising thread, all loaded before the first is used
constexpr int kDequantPer = 4;  // octets of a dequantising one
constexpr int kMxOctet = 8;

// The span's packed words; the block's first lane stores its scale.
template <int kFmt>
__device__ __forceinline__ void mx_store_packed(uint8_t* q, uint8_t* scale, uint64_t span, const uint32_t* w,
                                                uint32_t sc) {
  if constexpr (kFmt == kFmtMxfp8)
    reinterpret_cast<uint4*>(q)[span] = make_uint4(w[0], w[1], w[2], w[3]);
  else
    reinterpret_cast<uint2*>(q)[span] = make_uint2(w[0], w[1]);
  constexpr int kLanes = mx_block(kFmt) / kMxSpan;
  if (span % kLanes == 0) scale[span / kLanes] = static_cast<uint8_t>(sc);
}

// Byte offset of piece `i` of kB bytes in rows `ld_bytes` apart (per_row pieces each).
template <int kB>
__device__ __forceinline__ int64_t mx_at(uint64_t i, uint32_t per_row, int64_t ld_bytes) {
  if (ld_bytes == static_cast<int64_t>(per_row) * kB) return static_cast<int64_t>(i) * kB;
  const uint64_t row = i / per_row;
  return static_cast<int64_t>(row) * ld_bytes + static_cast<int64_t>(i - row * per_row) * kB;
}

// x [rows][x_ld] -> q, scale (both contiguous); `per_row` spans a row. Spans
// past the end load nothing and take part in the shuffles only: a block never
// straddles the end.
template <int kFmt, int kDt>
__global__ void __launch_bounds__(kMxThreads, kDt == kDtFp32 ? 1 : 6)
    mx_quant_kernel(const uint8_t* __restrict__ x, int64_t x_ld_bytes, bool wide, uint64_t spans, uint32_t per_row,
                    const float* __restrict__ global_scale, uint8_t* __restrict__ q, uint8_t* __restrict__ scale) {
  const uint64_t u0 = blockIdx.x * static_cast<uint64_t>(kMxThreads * kQuantPer) + threadIdx.x;
  griddep_wait();
  griddep_launch_dependents();
  constexpr int kW = MxWords<kDt, kMxSpan>::n;
  uint32_t w[kQuantPer][kW];
#pragma unroll
  for (int j = 0; j < kQuantPer; ++j) {
    const uint64_t u = u0 + j * kMxThreads;
    if (u < spans) {
      mx_load<kW>(x + mx_at<4 * kW>(u, per_row, x_ld_bytes), wide, w[j]);
    } else {
#pragma unroll
      for (int i = 0; i < kW; ++i) w[j][i] = 0;
    }
  }
  const MxGlobal gl = mx_global(kFmt == kFmtNvfp4 ? global_scale : nullptr);
#pragma unroll
  for (int j = 0; j < kQuantPer; ++j) {
    const uint64_t u = u0 + j * kMxThreads;
    float f[kMxSpan];
    mx_to_float<kDt>(w[j], f);
    uint32_t am;
    if constexpr (kDt == kDtFp32)
      am = mx_span_max(f);
    else
      am = mx_span_max_packed<kDt>(w[j]);
    am = mx_block_max<kFmt>(am);
    uint32_t p[4];
    const uint32_t sc = mx_quant_span<kFmt>(f, am, gl, p);
    if (u < spans) mx_store_packed<kFmt>(q, scale, u, p, sc);
  }
}

// q, scale (contiguous) -> x [rows][x_ld]: (value * scale) * global_scale in
// float32 (the first product is exact), rounded once to the output's type.
template <int kFmt, int kDt>
__global__ void __launch_bounds__(kMxThreads)
    mx_dequant_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ scale, uint64_t octets,
                      uint32_t per_row, const float* __restrict__ global_scale, uint8_t* __restrict__ x,
                      int64_t x_ld_bytes, bool wide) {
  const uint64_t o0 = blockIdx.x * static_cast<uint64_t>(kMxThreads * kDequantPer) + threadIdx.x;
  griddep_wait();
  griddep_launch_dependents();
  constexpr int kLanes = mx_block(kFmt) / kMxOctet;
  uint2 v[kDequantPer];
  uint32_t sb[kDequantPer];
#pragma unroll
  for (int j = 0; j < kDequantPer; ++j) {
    const uint64_t o = o0 + j * kMxThreads;
    v[j] = make_uint2(0, 0);
    sb[j] = 0;
    if (o < octets) {
      if constexpr (kFmt == kFmtMxfp8)
        v[j] = __ldcs(reinterpret_cast<const uint2*>(q) + o);
      else
        v[j].x = __ldcs(reinterpret_cast<const uint32_t*>(q) + o);
      sb[j] = __ldg(scale + o / kLanes);
    }
  }
  const float g = (kFmt == kFmtNvfp4 && global_scale) ? __ldg(global_scale) : 1.0f;
#pragma unroll
  for (int j = 0; j < kDequantPer; ++j) {
    const uint64_t o = o0 + j * kMxThreads;
    if (o >= octets) continue;
    float f[kMxOctet];
    if constexpr (kFmt == kFmtMxfp8) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t b = i ? v[j].y : v[j].x;
        const float2 lo = e4m3x2_to_f2(b & 0xFFFFu), hi = e4m3x2_to_f2(b >> 16);
        f[4 * i] = lo.x;
        f[4 * i + 1] = lo.y;
        f[4 * i + 2] = hi.x;
        f[4 * i + 3] = hi.y;
      }
    } else {
      e2m1x8_to_f8(v[j].x, f);
    }
    const float s = kFmt == kFmtNvfp4 ? e4m3x2_to_f2(sb[j]).x : e8m0_to_f(sb[j]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f[i] *= s;
      if (kFmt == kFmtNvfp4) f[i] *= g;
    }
    constexpr int kW = MxWords<kDt, kMxOctet>::n;
    uint32_t w[kW];
    mx_from_float<kDt>(f, w);
    mx_store<kW>(x + mx_at<4 * kW>(o, per_row, x_ld_bytes), wide, w);
  }
}

// Two floats at a time: the same operations in half the instructions.
__device__ __forceinline__ uint64_t f2_pack(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_unpack(uint64_t v, float* a, float* b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(*a), "=f"(*b) : "l"(v));
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t f2_fma_rz(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rz.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// Two values h * w / sqrt(v), rounded to odd: cut off to float32, with the last
// bit set where something was cut. A second rounding, to a format of at most 22
// bits, then gives what rounding the exact value would, so the quantisation that
// follows sees no float32 tie that is none. 1 / sqrt(v) lies between hi + lo0
// and hi + lo1; h w is exact as p (16-bit types) or p + e. Where the bounds cut
// to two float32 numbers, the value is the outer one to within the bounds and
// is taken for it: a row of +-7 has y = +-1, not the number below. One value at a
// time the second bound costs 3% (16384 x 7168 bf16 mxfp8: 140 us, in pairs 136 us).
constexpr uint64_t kMinus = 0x8000000080000000ull;  // both signs
template <int kDt>
__device__ __forceinline__ void mx_norm_pair(float* h, const float* w, uint64_t hi, uint64_t lo0, uint64_t lo1) {
  const uint64_t h2 = f2_pack(h[0], h[1]), w2 = f2_pack(w[0], w[1]);
  const uint64_t p = f2_mul(h2, w2);
  uint64_t t0 = f2_mul(p, lo0), t1 = f2_mul(p, lo1);
  if (kDt == kDtFp32) {
    const uint64_t e = f2_fma(h2 ^ kMinus, w2, p);  // -e, +0 of zeros: what is subtracted leaves a -0 as it is
    t0 = f2_fma(e, hi ^ kMinus, t0);
    t1 = f2_fma(e, hi ^ kMinus, t1);
  }
  float in[2], out[2];
  f2_unpack(f2_fma_rz(p, hi, t0), in, in + 1);
  f2_unpack(f2_fma_rz(p, hi, t1), out, out + 1);
#pragma unroll
  for (int i = 0; i < 2; ++i) h[i] = __uint_as_float(__float_as_uint(out[i]) | (in[i] == out[i] ? 1u : 0u));
}

// hi, lo0 and lo1 of inv = 1 / sqrt(v): the sum in v is within 2^-47, inv within 2^-48; lo
// and its products add 2^-46. Neither lo is negative: the products of -0 stay -0.
__device__ __forceinline__ float3 mx_root_bounds(double inv) {
  const float hi = __double2float_rd(inv * (1.0 - 0x1p-41));
  const float lo = static_cast<float>(inv - static_cast<double>(hi));
  return make_float3(hi, lo - 0x1p-42f * hi, lo + 0x1p-42f * hi);
}

// The same where v is far from 1, whose reciprocal root may not be a float32:
// that of v 4^e, with its sign turned for a sign, and 2^e in the place of lo1
// (mx_norm_scaled multiplies h by it). Zero, infinite and NaN v: 1 / sqrt(v).
__device__ __noinline__ float3 mx_far_root(double v) {
  const double inv = 1.0 / sqrt(v);
  if (!(v > 0.0 && v < INFINITY)) return make_float3(static_cast<float>(inv), 0.f, 0.f);
  const int e = min((__double2hiint(inv) >> 20) - 1023, 127);  // -128 at least: v is below 2^256
  const float3 r = mx_root_bounds(inv * __hiloint2double((1023 - e) << 20, 0));
  return make_float3(-r.x, r.y, static_cast<float>(__hiloint2double((1023 + e) << 20, 0)));
}

constexpr uint32_t kMaxBits = 0x7F7FFFFFu;  // float32's largest number

// A span in which h w or y passes float32's range, or of a row whose v is far
// from 1 (mx_far_root): from h times the power of two that takes sqrt(v) to about 1.
// Its products pass the range only where y does; a y that reaches the largest
// number counts as infinite. Apart, so that it takes no registers of the others.
template <int kDt>
__device__ __noinline__ void mx_norm_scaled(const uint8_t* hp, const uint8_t* wp, float hi, float lo0, float lo1, float* y) {
  constexpr int kW = MxWords<kDt, 2>::n;
  float down = lo1;
  if (hi < 0.f) {  // from mx_far_root
    hi = -hi;
    lo1 = lo0 + 0x1p-41f * hi;
  } else {
    const uint32_t e = __float_as_uint(hi) >> 23;
    const float up = __uint_as_float((254u - e) << 23);  // hi up is in [1, 2)
    down = __uint_as_float(e << 23);
    hi *= up;
    lo0 *= up;
    lo1 *= up;
  }
#pragma unroll 1
  for (int i = 0; i < kMxSpan; i += 2) {
    uint32_t hw[kW], ww[kW];
#pragma unroll
    for (int k = 0; k < kW; ++k) {
      hw[k] = reinterpret_cast<const volatile uint32_t*>(hp)[i / 2 * kW + k];
      ww[k] = __ldg(reinterpret_cast<const uint32_t*>(wp) + i / 2 * kW + k);
    }
    float h[2], w[2];
    mx_to_float<kDt>(hw, h);
    mx_to_float<kDt>(ww, w);
    h[0] *= down;
    h[1] *= down;
    mx_norm_pair<kDt>(h, w, f2_pack(hi, hi), f2_pack(lo0, lo0), f2_pack(lo1, lo1));
#pragma unroll
    for (int k = 0; k < 2; ++k) y[i + k] = fabsf(h[k]) < __uint_as_float(kMaxBits) ? h[k] : h[k] + copysignf(INFINITY, h[k]);
  }
}

constexpr int kNormPer = 2;  // spans of a thread

// h = T(residual + x) (written back), y = h / sqrt(mean(h^2) + eps) * weight,
// then the block's quantisation. `tpr` threads hold a row: a power of two up
// to 32 (several rows a CTA), or the CTA. Squares are summed eight at a time in
// float32 and from there on in float64, in an order that depends on the width
// alone; their sum's error is then far below the float32 steps of y, which
// decides how often a value lands on the wrong side of a border of the format.
// Without a weight: y = h.
template <int kFmt, int kDt, int kMaxT>
__global__ void __launch_bounds__(kMaxT, kMaxT == 256 ? (kDt != kDtFp32 ? 5 : 3) : 1)
    mx_norm_kernel(const uint8_t* __restrict__ x, int64_t x_ld_bytes, uint8_t* residual, int64_t res_ld_bytes,
                   const uint8_t* __restrict__ weight, bool wide, float eps, int64_t rows, uint32_t per_row,
                   uint32_t tpr, const float* __restrict__ global_scale, uint8_t* __restrict__ q,
                   uint8_t* __restrict__ scale) {
  __shared__ double warp_ss[32];
  griddep_wait();
  griddep_launch_dependents();
  const uint32_t tid = threadIdx.x;
  const bool whole = tpr > 32;  // one row for the CTA
  const int64_t row = whole ? blockIdx.x : blockIdx.x * static_cast<int64_t>(blockDim.x / tpr) + tid / tpr;
  const uint32_t c0 = whole ? tid : tid % tpr;
  constexpr int kW = MxWords<kDt, kMxSpan>::n;
  constexpr int kB = 4 * kW;
  uint32_t w[kNormPer][kW];
  bool live[kNormPer];
#pragma unroll
  for (int j = 0; j < kNormPer; ++j) {
    const uint32_t c = c0 + j * tpr;
    live[j] = row < rows && c < per_row;
    if (live[j]) {
      mx_load<kW>(x + row * x_ld_bytes + static_cast<int64_t>(c) * kB, wide, w[j]);
    } else {
#pragma unroll
      for (int i = 0; i < kW; ++i) w[j][i] = 0;
    }
  }
  if (residual) {
    uint8_t* rp = residual + row * res_ld_bytes + static_cast<int64_t>(c0) * kB;
    uint32_t rw[kNormPer][kW];
#pragma unroll
    for (int j = 0; j < kNormPer; ++j)
      if (live[j]) mx_load<kW>(rp + static_cast<int64_t>(j) * tpr * kB, wide, rw[j]);
#pragma unroll
    for (int j = 0; j < kNormPer; ++j) {
      if (!live[j]) continue;
      float f[kMxSpan], r[kMxSpan];
      mx_to_float<kDt>(w[j], f);
      mx_to_float<kDt>(rw[j], r);
#pragma unroll
      for (int i = 0; i < kMxSpan; ++i) f[i] += r[i];
      mx_from_float<kDt>(f, w[j]);
      mx_store<kW>(rp + static_cast<int64_t>(j) * tpr * kB, wide, w[j]);
    }
  }
  float hi = 1.f, lo0 = 0.f, lo1 = 0.f;
  uint32_t again_at = kMaxBits;  // spans whose largest value has these bits or more go to mx_norm_scaled
  if (weight) {
    double part[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
    for (int j = 0; j < kNormPer; ++j) {
      float f[kMxSpan];
      mx_to_float<kDt>(w[j], f);
#pragma unroll
      for (int i = 0; i < kMxSpan; ++i) part[i % 4] = fma(static_cast<double>(f[i]), static_cast<double>(f[i]), part[i % 4]);
    }
    double ss = (part[0] + part[1]) + (part[2] + part[3]);
    for (uint32_t off = whole ? 16 : tpr / 2; off >= 1; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
    if (whole) {
      if ((tid & 31) == 0) warp_ss[tid >> 5] = ss;
      __syncthreads();
      ss = 0.0;
      for (uint32_t i = 0; i < blockDim.x / 32; ++i) ss += warp_ss[i];
    }
    const double v = ss / static_cast<double>(per_row * kMxSpan) + static_cast<double>(eps);
    if (v > 1e-30 && v < 1e30) {
      // two Newton steps from the float32 estimate: 2^-22, 2^-43, 2^-51
      double inv = static_cast<double>(rsqrtf(static_cast<float>(v)));
#pragma unroll
      for (int k = 0; k < 2; ++k) inv = fma(inv * fma(-v * inv, inv, 1.0), 0.5, inv);
      const float3 r = mx_root_bounds(inv);
      hi = r.x, lo0 = r.y, lo1 = r.z;
    } else {
      const float3 r = mx_far_root(v);
      hi = r.x, lo0 = r.y, lo1 = r.z;
      again_at = hi < 0.f ? 0u : 0xFFFFFFFFu;
    }
  }
  const MxGlobal gl = mx_global(kFmt == kFmtNvfp4 ? global_scale : nullptr);
#pragma unroll
  for (int j = 0; j < kNormPer; ++j) {
    const uint32_t c = c0 + j * tpr;
    float f[kMxSpan];
    mx_to_float<kDt>(w[j], f);
    uint32_t am;
    if (weight && live[j]) {
      uint32_t ww[kW];
      const uint4* wp = reinterpret_cast<const uint4*>(weight + static_cast<int64_t>(c) * kB);
#pragma unroll
      for (int i = 0; i < kW / 4; ++i) {
        const uint4 v = __ldg(wp + i);
        ww[4 * i] = v.x;
        ww[4 * i + 1] = v.y;
        ww[4 * i + 2] = v.z;
        ww[4 * i + 3] = v.w;
      }
      float wf[kMxSpan];
      mx_to_float<kDt>(ww, wf);
#pragma unroll
      for (int i = 0; i < kMxSpan; i += 2)
        mx_norm_pair<kDt>(f + i, wf + i, f2_pack(hi, hi), f2_pack(lo0, lo0), f2_pack(lo1, lo1));
      am = mx_span_max(f);
      if (am >= again_at) {
        const uint8_t* hp = residual ? residual + row * res_ld_bytes : x + row * x_ld_bytes;
        float again[kMxSpan];
        mx_norm_scaled<kDt>(hp + static_cast<int64_t>(c) * kB, weight + static_cast<int64_t>(c) * kB, hi, lo0, lo1, again);
#pragma unroll
        for (int i = 0; i < kMxSpan; ++i) f[i] = again[i];
        am = mx_span_max(f);
      }
    } else {
      am = mx_span_max(f);
    }
    am = mx_block_max<kFmt>(am);
    uint32_t p[4];
    const uint32_t sc = mx_quant_span<kFmt>(f, am, gl, p);
    if (live[j]) mx_store_packed<kFmt>(q, scale, static_cast<uint64_t>(row) * per_row + c, p, sc);
  }
}

constexpr int64_t dt_bytes(int dt) { return dt == kDtFp32 ? 4 : 2; }

// Calls CALL(fmt, dt) for the run-time pair.
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

bool wide_rows(const void* p, int64_t ld_bytes) {
  return ((reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(ld_bytes)) & 31u) == 0;
}

dim3 mx_grid(uint64_t pieces, int per) {
  return dim3(static_cast<uint32_t>((pieces + kMxThreads * per - 1) / (kMxThreads * per)));
}

template <int kFmt, int kDt>
cudaError_t norm_launch(const MxNormCall& c, cudaStream_t s) {
  const uint32_t per_row = static_cast<uint32_t>(c.cols / kMxSpan);
  // up to two spans a thread: narrow rows share a CTA of 128 threads
  uint32_t tpr = 2;
  while (tpr < per_row && tpr < 32) tpr *= 2;
  uint32_t threads = 128;
  const bool whole = per_row > 32 * kNormPer;
  if (whole) tpr = threads = (per_row + 32 * kNormPer - 1) / (32 * kNormPer) * 32;
  const int64_t grid = whole ? c.rows : (c.rows + threads / tpr - 1) / (threads / tpr);
  const int64_t x_ld = c.x_ld * dt_bytes(kDt), res_ld = c.res_ld * dt_bytes(kDt);
  const bool wide = wide_rows(c.x, x_ld) && wide_rows(c.residual, c.residual ? res_ld : 0);
  auto go = [&](auto kernel) {
    return launch_k(kernel, dim3(static_cast<uint32_t>(grid)), dim3(threads), 0, s, true,
                    static_cast<const uint8_t*>(c.x), x_ld, static_cast<uint8_t*>(c.residual), res_ld,
                    static_cast<const uint8_t*>(c.weight), wide, c.eps, c.rows, per_row, tpr, c.global_scale,
                    static_cast<uint8_t*>(c.q), static_cast<uint8_t*>(c.scale));
  };
  // rows of up to 8192 columns take the variants of 256 threads, with their bounds on registers
  if (threads <= 256) return go(mx_norm_kernel<kFmt, kDt, 256>);
  return go(mx_norm_kernel<kFmt, kDt, 1024>);
}

}  // namespace

cudaError_t launch_mx_quant(const void* x, int dt, int64_t x_ld, int64_t rows, int64_t cols, int fmt,
                            const float* global_scale, void* q, void* scale, cudaStream_t s) {
  const uint32_t per_row = static_cast<uint32_t>(cols / kMxSpan);
  const uint64_t spans = static_cast<uint64_t>(rows) * per_row;
  if (spans == 0) return cudaSuccess;
#define CALL(F, D)                                                                                                    \
  launch_k(mx_quant_kernel<F, D>, mx_grid(spans, kQuantPer), dim3(kMxThreads), 0, s, true, static_cast<const uint8_t*>(x), \
           x_ld * dt_bytes(D), wide_rows(x, x_ld * dt_bytes(D)), spans, per_row, global_scale,                       \
           static_cast<uint8_t*>(q), static_cast<uint8_t*>(scale))
  MX_DISPATCH(fmt, dt, CALL)
#undef CALL
}

cudaError_t launch_mx_dequant(const void* q, const void* scale, int64_t rows, int64_t cols, int fmt,
                              const float* global_scale, int dt, void* x, int64_t x_ld, cudaStream_t s) {
  const uint32_t per_row = static_cast<uint32_t>(cols / kMxOctet);
  const uint64_t octets = static_cast<uint64_t>(rows) * per_row;
  if (octets == 0) return cudaSuccess;
#define CALL(F, D)                                                                                                      \
  launch_k(mx_dequant_kernel<F, D>, mx_grid(octets, kDequantPer), dim3(kMxThreads), 0, s, true, static_cast<const uint8_t*>(q), \
           static_cast<const uint8_t*>(scale), octets, per_row, global_scale, static_cast<uint8_t*>(x),                 \
           x_ld * dt_bytes(D), wide_rows(x, x_ld * dt_bytes(D)))
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
