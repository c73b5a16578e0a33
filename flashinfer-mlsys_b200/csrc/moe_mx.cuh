// moe_mx.cuh — the microscaled formats: blocks of values along a row that
// share one scale, as the tensor cores read them.
//   nvfp4  e2m1 values, blocks of 16, e4m3 scale (and one fp32 scale per tensor)
//   mxfp4  e2m1 values, blocks of 32, power-of-two scale (e8m0, 2^(byte - 127))
//   mxfp8  e4m3 values, blocks of 32, power-of-two scale (e8m0)
// e2m1 values are packed two a byte, the even column in the low half.
#pragma once
#include "moe_common.cuh"

namespace moe {

constexpr int kFmtNvfp4 = 0, kFmtMxfp4 = 1, kFmtMxfp8 = 2;
constexpr int kDtBf16 = 0, kDtFp16 = 1, kDtFp32 = 2;

// A unit is 32 consecutive columns of a row: two nvfp4 blocks or one mx block.
constexpr int kMxUnit = 32;

__host__ __device__ constexpr int mx_block(int fmt) { return fmt == kFmtNvfp4 ? 16 : 32; }
__host__ __device__ constexpr int mx_unit_bytes(int fmt) { return fmt == kFmtMxfp8 ? 32 : 16; }
__host__ __device__ constexpr int mx_unit_scales(int fmt) { return kMxUnit / mx_block(fmt); }

// Eight floats -> eight e2m1 codes (to nearest even, saturating at 6), v[0] in the low half of byte 0.
__device__ __forceinline__ uint32_t f8_to_e2m1x8(const float* v) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// Eight e2m1 codes -> floats (exact).
__device__ __forceinline__ void e2m1x8_to_f8(uint32_t w, float* v) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// Two e4m3 bytes (the low 16 bits) -> floats (exact; 0x7F and 0xFF are NaN).
__device__ __forceinline__ float2 e4m3x2_to_f2(uint32_t w) {
  uint32_t h;
  asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(h) : "r"(w));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// 2^(b - 127) of an e8m0 byte: 0 is 2^-127 (a subnormal float), 255 is NaN.
__device__ __forceinline__ float e8m0_to_f(uint32_t b) {
  return __uint_as_float(b == 0 ? 0x00400000u : (b == 255 ? 0x7FC00000u : b << 23));
}

constexpr uint32_t kInfBits = 0x7F800000u;

// Quantises one unit. `f`: its 32 values; `am`: the bits of the largest
// absolute value of each block (am[1] is used by nvfp4 only); g: the tensor
// scale. Writes the packed words and returns the scale bytes.
//
// All roundings are to nearest even, so a float32 host computation of the same
// steps gives the same bytes. A block with an infinity or a NaN (am >= inf as
// an integer: both order above every finite value) gets a NaN scale and zeros.
//
// nvfp4: s = e4m3(min(448, amax / (6 g))), q = e2m1(x / (s g)). The quotient
// decides ties, so it has to be the correctly rounded one: with r = RN(1/d),
// q0 = RN(x r), e = x - q0 d (exact, one fma), RN(q0 + e r) is that quotient
// (P. Markstein, IA-64 division, 1990) when nothing leaves the normal range,
// which holds for d and amax within 2^+-60; other blocks divide. Three
// operations a value instead of a division's ten or so.
// mx: the scale is the power of two 2^(floor(log2 amax) - emax), emax = 2
// (e2m1) or 8 (e4m3), the shared exponent of the OCP microscaling formats;
// scaling by it is exact (down to subnormal numbers, which round to zero in
// either format).
template <int kFmt>
__device__ __forceinline__ uint32_t mx_quant_unit(const float (&f)[32], const uint32_t (&am)[2], float g, uint32_t* w) {
  if constexpr (kFmt == kFmtNvfp4) {
    uint32_t sc = 0;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const bool fine = am[b] < kInfBits;
      const float amax = __uint_as_float(am[b]);
      const float want = fminf(__fdiv_rn(amax, 6.0f * g), 448.0f);
      uint32_t s8 = f2_to_e4m3x2(want, 0.f) & 0xFFu;
      if (!fine) s8 = 0x7F;
      const float d = e4m3x2_to_f2(s8).x * g;
      sc |= s8 << (8 * b);
      float y[16];
      if (d > 0x1p-60f && d < 0x1p60f && amax < 0x1p60f) {
        const float r = __frcp_rn(d);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float x = f[16 * b + i];
          const float q0 = x * r;
          y[i] = fmaf(fmaf(-q0, d, x), r, q0);
        }
      } else {
        const bool zero = !fine || !(d > 0.f);
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] = zero ? 0.f : __fdiv_rn(f[16 * b + i], d);
      }
      w[2 * b] = f8_to_e2m1x8(y);
      w[2 * b + 1] = f8_to_e2m1x8(y + 8);
    }
    return sc;
  } else {
    constexpr int kEmax = kFmt == kFmtMxfp4 ? 2 : 8;
    const bool fine = am[0] < kInfBits;
    const int b = max(static_cast<int>(am[0] >> 23) - kEmax, 0);  // <= 254 - kEmax
    const uint32_t rb = 254u - b;
    const float r = fine ? __uint_as_float(rb << 23) : 0.f;  // 2^(127 - b), normal: b <= 252
    float y[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) y[i] = fine ? f[i] * r : 0.f;
    if constexpr (kFmt == kFmtMxfp4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = f8_to_e2m1x8(y + 8 * i);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        w[i] = f2_to_e4m3x2(y[4 * i], y[4 * i + 1]) | (static_cast<uint32_t>(f2_to_e4m3x2(y[4 * i + 2], y[4 * i + 3])) << 16);
    }
    return fine ? b : 255u;
  }
}

// ---- 32 columns of bf16, fp16 or fp32 -------------------------------------
template <int kDt>
struct MxWords {
  static constexpr int n = kDt == kDtFp32 ? 32 : 16;  // 32-bit words of a unit
};

template <int kDt>
__device__ __forceinline__ void mx_to_float(const uint32_t* w, float (&f)[32]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    if constexpr (kDt == kDtBf16) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    } else if constexpr (kDt == kDtFp16) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    } else {
      f[2 * i] = __uint_as_float(w[2 * i]);
      f[2 * i + 1] = __uint_as_float(w[2 * i + 1]);
    }
  }
}

template <int kDt>
__device__ __forceinline__ void mx_from_float(const float (&f)[32], uint32_t* w) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    if constexpr (kDt == kDtBf16) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&v);
    } else if constexpr (kDt == kDtFp16) {
      const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&v);
    } else {
      w[2 * i] = __float_as_uint(f[2 * i]);
      w[2 * i + 1] = __float_as_uint(f[2 * i + 1]);
    }
  }
}

// Bits of the largest absolute value of each block, from floats (integers order like the values).
template <int kFmt>
__device__ __forceinline__ void mx_amax(const float (&f)[32], uint32_t (&am)[2]) {
  am[0] = am[1] = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    uint32_t& m = am[kFmt == kFmtNvfp4 ? i / 16 : 0];
    m = max(m, __float_as_uint(f[i]) & 0x7FFFFFFFu);
  }
}

// The same from the packed 16-bit words, two values at a time.
template <int kFmt, int kDt>
__device__ __forceinline__ void mx_amax_packed(const uint32_t* w, uint32_t (&am)[2]) {
  uint32_t m[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    uint32_t& p = m[kFmt == kFmtNvfp4 ? i / 8 : 0];
    p = __vmaxu2(p, w[i] & 0x7FFF7FFFu);
  }
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const uint32_t v = max(m[b] & 0xFFFFu, m[b] >> 16);
    am[b] = kDt == kDtBf16 ? v << 16 : __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(v))));
  }
}

template <int kWords>
__device__ __forceinline__ void mx_load(const void* p, uint32_t* w) {
#pragma unroll
  for (int i = 0; i < kWords / 4; ++i) {
    const uint4 v = __ldcs(static_cast<const uint4*>(p) + i);
    w[4 * i] = v.x;
    w[4 * i + 1] = v.y;
    w[4 * i + 2] = v.z;
    w[4 * i + 3] = v.w;
  }
}

template <int kWords>
__device__ __forceinline__ void mx_store(void* p, const uint32_t* w) {
#pragma unroll
  for (int i = 0; i < kWords / 4; ++i)
    static_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
}

}  // namespace moe
