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

// A quantising thread holds a span of 16 consecutive columns: an nvfp4 block,
// or half of an mx block, whose largest value takes one shuffle. 16-bit spans
// are one 32-byte access, so a warp's loads are contiguous. Measured at 16384
// x 7168 bf16: threads of 8 columns spend their time on the scales (nvfp4 72
// us), of 32 columns load in strides (54 us, and fp32 rows at 4.9 TB/s).
// A dequantising thread holds half a span: its scale costs nothing.
constexpr int kMxSpan = 16;
constexpr int kMxCols = 32;  // the width is a multiple of this in every format

__host__ __device__ constexpr int mx_block(int fmt) { return fmt == kFmtNvfp4 ? 16 : 32; }

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

// The block's largest absolute value as bits, from this lane's span's.
template <int kFmt>
__device__ __forceinline__ uint32_t mx_block_max(uint32_t m) {
  return kFmt == kFmtNvfp4 ? m : max(m, __shfl_xor_sync(0xffffffffu, m, 1));
}

// RN(x / d) by Markstein's correction (P. Markstein, IA-64 division, 1990):
// with r = RN(1/d) and q0 = RN(x r), the remainder q0 d - x is exact in one
// fma and RN(q0 - remainder r) is the correctly rounded quotient while nothing
// leaves the normal range. (The remainder's sign matters for x = -0: of q0 = -0
// only a subtraction of +0 keeps the sign.)
__device__ __forceinline__ float mx_quotient(float x, float d, float r) {
  const float q0 = x * r;
  return fmaf(-fmaf(q0, d, -x), r, q0);
}
__device__ __forceinline__ bool mx_mid(float v) { return v > 0x1p-60f && v < 0x1p60f; }

// What an nvfp4 call's thread needs of the tensor scale.
struct MxGlobal {
  float g, d6, r6;  // g, 6 g, 1 / (6 g)
  bool mid;
};
__device__ __forceinline__ MxGlobal mx_global(const float* global_scale) {
  MxGlobal t;
  t.g = global_scale ? __ldg(global_scale) : 1.0f;
  t.d6 = 6.0f * t.g;
  t.mid = mx_mid(t.d6);
  t.r6 = __frcp_rn(t.d6);
  return t;
}

// Quantises one span. `am`: the bits of its block's largest absolute value.
// Writes two words of e2m1 or four of e4m3 and returns the block's scale byte.
//
// All roundings are to nearest even, so a float32 host computation of the same
// steps gives the same bytes. A block with an infinity or a NaN (am >= inf as
// an integer: both order above every finite value) gets a NaN scale and zeros.
//
// nvfp4: s = e4m3(min(448, amax / (6 g))), q = e2m1(x / (s g)). Quotients
// decide ties, so they have to be the correctly rounded ones: mx_quotient for
// divisors and amax within 2^+-60 (three operations a value instead of a
// division's ten or so), divisions for other blocks.
// mx: the scale is the power of two 2^(floor(log2 amax) - emax), emax = 2
// (e2m1) or 8 (e4m3), the shared exponent of the OCP microscaling formats;
// scaling by it is exact (down to subnormal numbers, which round to zero in
// either format).
template <int kFmt>
__device__ __forceinline__ uint32_t mx_quant_span(const float (&f)[kMxSpan], uint32_t am, const MxGlobal& gl, uint32_t* w) {
  const bool fine = am < kInfBits;
  const float amax = __uint_as_float(am);
  if constexpr (kFmt == kFmtNvfp4) {
    const bool small = amax < 0x1p60f && (amax > 0x1p-60f || amax == 0.f);
    const float want = gl.mid && small ? mx_quotient(amax, gl.d6, gl.r6) : __fdiv_rn(amax, gl.d6);
    uint32_t s8 = f2_to_e4m3x2(fminf(want, 448.0f), 0.f) & 0xFFu;
    if (!fine) s8 = 0x7F;
    const float d = e4m3x2_to_f2(s8).x * gl.g;
    float y[kMxSpan];
    if (mx_mid(d) && amax < 0x1p60f) {
      const float r = __frcp_rn(d);
#pragma unroll
      for (int i = 0; i < kMxSpan; ++i) y[i] = mx_quotient(f[i], d, r);
    } else {
      const bool zero = !fine || !(d > 0.f);
#pragma unroll
      for (int i = 0; i < kMxSpan; ++i) y[i] = zero ? 0.f : __fdiv_rn(f[i], d);
    }
    w[0] = f8_to_e2m1x8(y);
    w[1] = f8_to_e2m1x8(y + 8);
    return s8;
  } else {
    constexpr int kEmax = kFmt == kFmtMxfp4 ? 2 : 8;
    const int b = max(static_cast<int>(am >> 23) - kEmax, 0);                  // <= 254 - kEmax
    const float r = __uint_as_float((254u - static_cast<uint32_t>(b)) << 23);  // 2^(127 - b), a normal number
    float y[kMxSpan];
#pragma unroll
    for (int i = 0; i < kMxSpan; ++i) y[i] = fine ? f[i] * r : 0.f;
    if constexpr (kFmt == kFmtMxfp4) {
      w[0] = f8_to_e2m1x8(y);
      w[1] = f8_to_e2m1x8(y + 8);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = f2_to_e4m3x2(y[4 * i], y[4 * i + 1]) |
               (static_cast<uint32_t>(f2_to_e4m3x2(y[4 * i + 2], y[4 * i + 3])) << 16);
    }
    return fine ? b : 255u;
  }
}

// ---- n columns of bf16, fp16 or fp32 ----------------------------------------
template <int kDt, int kN>
struct MxWords {
  static constexpr int n = kDt == kDtFp32 ? kN : kN / 2;  // 32-bit words
};

template <int kDt, int kN>
__device__ __forceinline__ void mx_to_float(const uint32_t* w, float (&f)[kN]) {
#pragma unroll
  for (int i = 0; i < kN / 2; ++i) {
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

template <int kDt, int kN>
__device__ __forceinline__ void mx_from_float(const float (&f)[kN], uint32_t* w) {
#pragma unroll
  for (int i = 0; i < kN / 2; ++i) {
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

// Bits of the span's largest absolute value (integers order like the values).
__device__ __forceinline__ uint32_t mx_span_max(const float (&f)[kMxSpan]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < kMxSpan; ++i) m = max(m, __float_as_uint(f[i]) & 0x7FFFFFFFu);
  return m;
}

// The same from 16-bit words, two values at a time.
template <int kDt>
__device__ __forceinline__ uint32_t mx_span_max_packed(const uint32_t* w) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < kMxSpan / 2; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
  const uint32_t v = max(m & 0xFFFFu, m >> 16);
  return kDt == kDtBf16 ? v << 16 : __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(v))));
}

// Words of a row: 32 bytes an access where `wide` (32-byte aligned rows) allows it, else 16.
template <int kWords>
__device__ __forceinline__ void mx_load(const void* p, bool wide, uint32_t* w) {
  if (kWords >= 8 && wide) {
#pragma unroll
    for (int i = 0; i + 8 <= kWords; i += 8)
      asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]), "=r"(w[i + 4]), "=r"(w[i + 5]),
                     "=r"(w[i + 6]), "=r"(w[i + 7])
                   : "l"(static_cast<const uint32_t*>(p) + i)
                   : "memory");
    return;
  }
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
__device__ __forceinline__ void mx_store(void* p, bool wide, const uint32_t* w) {
  if (kWords >= 8 && wide) {
#pragma unroll
    for (int i = 0; i + 8 <= kWords; i += 8)
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(static_cast<uint32_t*>(p) + i),
                   "r"(w[i]), "r"(w[i + 1]), "r"(w[i + 2]), "r"(w[i + 3]), "r"(w[i + 4]), "r"(w[i + 5]), "r"(w[i + 6]),
                   "r"(w[i + 7])
                   : "memory");
    return;
  }
#pragma unroll
  for (int i = 0; i < kWords / 4; ++i)
    __stcs(static_cast<uint4*>(p) + i, make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]));
}

}  // namespace moe
