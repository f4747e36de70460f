// fp8.cuh -- block-scaled e4m3: the quantisation rule, packing, and the
// instruction descriptor of the 8-bit MMA, shared by rmsnorm.cu,
// quantize.cu and gemm_fp8.cu.
//
// A block of values y (1 x 128 along a row for activations, 128 x 128 for
// weights) is held as q = e4m3(y / s), round to nearest even, with the fp32
// scale s = max(amax|y| / 448, 2^-126); 448 is the largest e4m3 value.  The
// lower limit keeps y / s finite for a block of zeros or subnormals.  A NaN or
// an infinity makes s NaN or infinite, and so every value the block stands
// for NaN (finite / inf = 0, and 0 * inf is NaN).
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace tjb {

constexpr int kQBlock = 128;      // columns (and weight rows) per scale
constexpr int kLiveTileRows = 128;  // rows per entry of a live-tile list
// Longest row: counts of its pieces, rounded up, stay below 2^31.
constexpr int kMaxColumns = 2147483647 - 1024;

// |v| as an integer: ordered like the magnitude, with NaN above infinity, so
// an integer maximum propagates both.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// max(|a|, |b|) that propagates NaN.
__device__ __forceinline__ float max_abs(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)));
  return r;
}

// max(|a|, |b|, |c|) in one instruction (sm_100), NaN propagated.
__device__ __forceinline__ float max_abs(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ float max_abs4(float4 v) {
  return max_abs(max_abs(v.x, v.y, v.z), v.w, v.w);
}

// Largest magnitude over the warp (NaN included).
__device__ __forceinline__ float warp_max_abs(float v) {
  return __uint_as_float(__reduce_max_sync(0xffffffffu, abs_bits(v)));
}

// v / s given inv = 1 / s: the quotient from the reciprocal, corrected once by
// its remainder (Markstein, IBM J. Res. Dev. 34, 1990).  The plain product
// v * inv moves about one value in 10^6 across a rounding border of the 8-bit
// type, and full divisions bound the memory-bound kernels here by their
// instructions (a 65536 x 4096 norm in its first form: 540 us, 461 with this).
__device__ __forceinline__ float div_by(float v, float s, float inv) {
  const float q = v * inv;
  return fmaf(fmaf(-q, s, v), inv, q);
}

// 1 / s for s in [2^-126, 2^126]: the hardware's approximation and one step
// of Newton's iteration.  Larger s give zero.
__device__ __forceinline__ float reciprocal(float s) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  return fmaf(fmaf(-s, r, 1.f), r, r);
}

// Scale of a block whose largest magnitude is amax.
__device__ __forceinline__ float block_scale(float amax) {
  const float s = div_by(amax, 448.f, 1.f / 448.f);
  if (abs_bits(amax) >= 0x7f800000u) return amax;  // NaN or infinite
  return fmaxf(s, 1.17549435e-38f);
}

// A scale as quantize4 divides by it: s and 1 / s.  An infinite s becomes the
// largest number, whose reciprocal underflows to zero here: finite values give
// zero and infinite ones NaN, as finite / inf and inf / inf do.  A NaN stays.
struct Divisor {
  float s, inv;
};
__device__ __forceinline__ Divisor divisor(float s) {
  Divisor d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d.s) : "f"(s), "f"(3.40282347e38f));
  d.inv = reciprocal(d.s);
  return d;
}

// Four e4m3 bytes of v / d.s, the first in the lowest byte.
__device__ __forceinline__ uint32_t quantize4(const float* v, Divisor d) {
  float q[4], e[4];
#pragma unroll
  for (int i = 0; i < 4; i += 2) {  // div_by on packed pairs
    asm("{\n\t.reg .b64 ra, rb;\n\t"
        "mov.b64 ra, {%2, %3};\n\t"
        "mov.b64 rb, {%4, %4};\n\t"
        "mul.rn.f32x2 ra, ra, rb;\n\t"
        "mov.b64 {%0, %1}, ra;\n\t}"
        : "=f"(q[i]), "=f"(q[i + 1])
        : "f"(v[i]), "f"(v[i + 1]), "f"(d.inv));
    fma2v(e[i], e[i + 1], q[i], q[i + 1], -d.s, -d.s, v[i], v[i + 1]);
    fma2v(q[i], q[i + 1], e[i], e[i + 1], d.inv, d.inv, q[i], q[i + 1]);
  }
  const __nv_fp8x2_storage_t lo =
      __nv_cvt_float2_to_fp8x2(make_float2(q[0], q[1]), __NV_SATFINITE, __NV_E4M3);
  const __nv_fp8x2_storage_t hi =
      __nv_cvt_float2_to_fp8x2(make_float2(q[2], q[3]), __NV_SATFINITE, __NV_E4M3);
  return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}

__device__ __forceinline__ uint32_t quantize4(float4 v, Divisor d) {
  const float f[4] = {v.x, v.y, v.z, v.w};
  return quantize4(f, d);
}

// log2 Phi(b) of two values b <= 0, as -1 + c[0] b + c[1] b^2 + ...
template <int N>
__device__ __forceinline__ void log2_phi(float& q0, float& q1, float b0, float b1,
                                         const float (&c)[N]) {
  q0 = q1 = c[N - 1];
#pragma unroll
  for (int i = N - 2; i >= 0; --i) fma2v(q0, q1, q0, q1, b0, b1, c[i], c[i]);
  fma2v(q0, q1, q0, q1, b0, b1, -1.f, -1.f);
}

// max(x, 0), a NaN stays one.
__device__ __forceinline__ float relu_nan(float x) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(0.f));
  return r;
}

// Erf GELU of two values, packed (gelu_erf in common.cuh takes twice the issue
// slots and two MUFU operations a value; with one or two warps a sub-partition
// an activation of 128 values a thread is bound by them):
//   GELU(x) = max(x, 0) + b Phi(b), b = -|x|,
// with log2 Phi(b) by a polynomial on [-13.3, 0], where 2^q leaves fp32's
// normal range and becomes zero.  Both are fitted by Lawson's iteration
// (weighted least squares towards the minimax) with Phi(0) = 1/2 exactly.
// 32-bit results, degree 13: Phi(b) to 3e-8 of itself down to -2, 2e-5 to -5
// and 3e-4 to the end, before the roundings in fp32 (2e-7, 3e-6 and up to 2e-3)
// and of 2^q (2^-22): for |x| <= 1 the GELU is within 12 x 2^-24 of itself.
// 16 and 8 bits (a rounding of 2e-4 or more), degree 7: the GELU to 4e-7
// absolute, 4e-6 of itself for |x| <= 2, 8e-4 to -5.5, 0.012 to -9 and a tenth
// to the end.
// Infinities: the factor of a negative x is not cut, and minus infinity times
// zero is NaN, as in 0.5 x (1 + erf(x / sqrt 2)); plus infinity stays.  For 8
// bits b is not cut either (this polynomial falls for good), which spares two
// instructions a value (M16384 N4096 K1024, e4m3: 103 us against 108): both
// infinities give NaN, and either way every value of the block stands for NaN.
template <int kBits>
__device__ __forceinline__ void gelu_pair(float& x0, float& x1) {
  const float b0 = kBits == 8 ? -fabsf(x0) : fmaxf(-fabsf(x0), -13.3f);
  const float b1 = kBits == 8 ? -fabsf(x1) : fmaxf(-fabsf(x1), -13.3f);
  float q0, q1, e0, e1;
  if constexpr (kBits == 32)
    log2_phi(q0, q1, b0, b1,
             {1.15110481f, -0.459216624f, 0.0524468757f, 0.00693850731f, -2.76900973e-05f,
              -0.000308792718f, -9.25991262e-05f, -1.62199449e-05f, -1.88740239e-06f,
              -1.47035465e-07f, -7.36164862e-09f, -2.13845219e-10f, -2.73576496e-12f});
  else
    log2_phi(q0, q1, b0, b1,
             {1.15114117f, -0.458884239f, 0.0533754863f, 0.00814140774f, 0.000821109221f,
              4.67876635e-05f, 1.11061843e-06f});
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(q0));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(q1));
  const float n0 = kBits == 8 ? b0 : fminf(b0, x0), n1 = kBits == 8 ? b1 : fminf(b1, x1);
  fma2v(x0, x1, n0, n1, e0, e1, relu_nan(x0), relu_nan(x1));
}

// Four consecutive elements of a row: raw as loaded (16 or 8 bytes), widened
// to fp32 when they are used, so that a load in flight is not waited for.
template <bool k16>
struct Raw4;
template <>
struct Raw4<false> {
  float4 v;
};
template <>
struct Raw4<true> {
  uint2 v;
};

template <bool k16>
__device__ __forceinline__ Raw4<k16> load_raw4(const void* p, int64_t idx) {
  Raw4<k16> r;
  if constexpr (k16)
    r.v = __ldcs(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + idx));
  else
    r.v = __ldcs(reinterpret_cast<const float4*>(static_cast<const float*>(p) + idx));
  return r;
}

template <bool k16>
__device__ __forceinline__ float4 widen4(const Raw4<k16>& r, bool bf16) {
  if constexpr (!k16) {
    return r.v;
  } else {
    float2 a, b;
    if (bf16) {
      a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&r.v.x));
      b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&r.v.y));
    } else {
      a = __half22float2(*reinterpret_cast<const __half2*>(&r.v.x));
      b = __half22float2(*reinterpret_cast<const __half2*>(&r.v.y));
    }
    return make_float4(a.x, a.y, b.x, b.y);
  }
}

// Sixteen bytes of a row (four fp32 or eight 16-bit elements) as loaded, with
// their largest magnitude and their fp32 values.
template <typename T>
struct Piece16;
template <>
struct Piece16<float> {
  static constexpr int kElems = 4;
  float4 v;
  __device__ __forceinline__ float max_abs() const { return max_abs4(v); }
  __device__ __forceinline__ void widen(float (&f)[4]) const {
    f[0] = v.x;
    f[1] = v.y;
    f[2] = v.z;
    f[3] = v.w;
  }
};
template <typename T, typename T2>
struct Piece16Half {
  static constexpr int kElems = 8;
  T2 v[4];
  __device__ __forceinline__ float max_abs() const {
    const T2 m = __hmax2_nan(__hmax2_nan(__habs2(v[0]), __habs2(v[1])),
                             __hmax2_nan(__habs2(v[2]), __habs2(v[3])));
    return tjb::max_abs(static_cast<float>(m.x), static_cast<float>(m.y));
  }
  __device__ __forceinline__ void widen(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = static_cast<float>(v[i].x);
      f[2 * i + 1] = static_cast<float>(v[i].y);
    }
  }
};
template <>
struct Piece16<__half> : Piece16Half<__half, __half2> {};
template <>
struct Piece16<__nv_bfloat16> : Piece16Half<__nv_bfloat16, __nv_bfloat162> {};

template <typename T>
__device__ __forceinline__ Piece16<T> load_piece16(const T* p) {
  const uint4 raw = __ldcs(reinterpret_cast<const uint4*>(p));
  return *reinterpret_cast<const Piece16<T>*>(&raw);
}

// Four consecutive fp32 values rounded once to `dtype` (f32, f16, bf16).
__device__ __forceinline__ void store4(void* out, int dtype, int64_t idx, float4 y) {
  if (dtype == TJB_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(out) + idx) = y;
    return;
  }
  uint2 raw;
  if (dtype == TJB_BF16) {
    raw.x = Pack2<__nv_bfloat16>::pack(y.x, y.y);
    raw.y = Pack2<__nv_bfloat16>::pack(y.z, y.w);
  } else {
    raw.x = Pack2<__half>::pack(y.x, y.y);
    raw.y = Pack2<__half>::pack(y.z, y.w);
  }
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + idx) = raw;
}

// Eight consecutive fp32 values rounded once to `dtype` (16-byte stores).
__device__ __forceinline__ void store8(void* out, int dtype, int64_t idx, const float (&y)[8]) {
  if (dtype == TJB_F32) {
    float4* p = reinterpret_cast<float4*>(static_cast<float*>(out) + idx);
    p[0] = make_float4(y[0], y[1], y[2], y[3]);
    p[1] = make_float4(y[4], y[5], y[6], y[7]);
    return;
  }
  uint4 raw;
  if (dtype == TJB_BF16)
    raw = make_uint4(
        Pack2<__nv_bfloat16>::pack(y[0], y[1]), Pack2<__nv_bfloat16>::pack(y[2], y[3]),
        Pack2<__nv_bfloat16>::pack(y[4], y[5]), Pack2<__nv_bfloat16>::pack(y[6], y[7]));
  else
    raw = make_uint4(Pack2<__half>::pack(y[0], y[1]), Pack2<__half>::pack(y[2], y[3]),
                     Pack2<__half>::pack(y[4], y[5]), Pack2<__half>::pack(y[6], y[7]));
  *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + idx) = raw;
}

// Instruction descriptor of kind::f8f6f4 with e4m3 operands (format 0), fp32
// accumulation, both K-major; the fields sit as in idesc_f16.
__host__ __device__ constexpr uint32_t idesc_e4m3(int M, int N) {
  return (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

}  // namespace tjb
