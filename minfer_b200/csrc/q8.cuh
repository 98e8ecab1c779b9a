// 8-bit vectors of a cache: codes and one float32 scale a vector, x = code * scale.
//
//   a     = max(max |x_d|, 2^-100)
//   scale = a / L,  code_d = round(x_d * (L / a)),  L = 448 for e4m3 and 127 for int8
//
// The rounding is to nearest, ties to even: a code is off by half a step at most, 2^-4 of the
// value in e4m3 (2^-10 of scale where a code is subnormal) and scale / 2 in int8.  2^-100 keeps
// both quotients in range for vectors of zeros.  A vector that holds an infinity or a NaN is kept
// as codes of zero with a scale of NaN: it reads back as NaN wherever it is seen, and nowhere else,
// since attention masks scores and probabilities (which the scales go into) and a masked probability
// only ever meets codes, which are finite.  (Codes of places that no query sees may be anything.)
#pragma once
#include "common.cuh"
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#define MF_Q8_E4M3 0
#define MF_Q8_INT8 1
#define MF_Q8_TINY 7.888609052210118e-31f       // 2^-100

template <int FMT> __host__ __device__ constexpr float q8_limit() { return FMT == MF_Q8_E4M3 ? 448.0f : 127.0f; }

// two values that are in the format's range already, the first in the low byte
template <int FMT> __device__ __forceinline__ uint32_t q8_pack2(float lo, float hi) {
    if (FMT == MF_Q8_E4M3)
        return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
    const int a = max(-127, min(127, __float2int_rn(lo))), b = max(-127, min(127, __float2int_rn(hi)));
    return (uint32_t)(a & 0xff) | ((uint32_t)(b & 0xff) << 8);
}

// Codes as halves, exactly: a warp turns two e4m3 codes in one instruction (measured: as many a clock
// as any other integer or logic instruction; moving sign, exponent and mantissa into place by hand takes
// four).  int8: byte b as the half 1024 + (b + 128), of which 1152 is taken off; the caller flips the
// bytes' sign bits first (q8_prepare).
template <int FMT> __device__ __forceinline__ uint32_t q8_prepare(uint32_t w) {
    return FMT == MF_Q8_INT8 ? w ^ 0x80808080u : w;
}
// the low (HIGH: the high) two bytes of `w`, the first in the low half
template <int FMT, bool HIGH> __device__ __forceinline__ uint32_t q8_halves(uint32_t w) {
    uint32_t r;
    if (FMT == MF_Q8_E4M3) {
        if (HIGH)
            asm("{\n .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %1;\n cvt.rn.f16x2.e4m3x2 %0, hi;\n}" : "=r"(r) : "r"(w));
        else
            asm("{\n .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %1;\n cvt.rn.f16x2.e4m3x2 %0, lo;\n}" : "=r"(r) : "r"(w));
        return r;
    }
    const uint32_t h = __byte_perm(w, 0x64646464u, HIGH ? 0x4342 : 0x4140);
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&d);
}
// four codes of a word (not prepared) as float values of the codes
template <int FMT> __device__ __forceinline__ void q8_floats(uint32_t w, float* out) {
    if (FMT == MF_Q8_INT8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = (float)(int)(signed char)(w >> (8 * i));
        return;
    }
    const uint32_t lo = q8_halves<FMT, false>(w), hi = q8_halves<FMT, true>(w);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    out[0] = a.x; out[1] = a.y; out[2] = b.x; out[3] = b.y;
}
