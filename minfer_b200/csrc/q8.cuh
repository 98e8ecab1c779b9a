// 8-bit vectors of a cache: codes and one float32 scale a vector, x = code * scale.
//
//   a     = max(max |x_d|, 2^-100)
//   scale = a / L,  code_d = round(x_d * (L / a)),  L = 448 for e4m3 and 127 for int8
//
// The rounding is to nearest, ties to even: a code is off by half a step at most, 2^-4 of the
// value in e4m3 (2^-10 of scale where a code is subnormal) and scale / 2 in int8.  2^-100 keeps
// both quotients in range for vectors of zeros.  A vector that holds an infinity or a NaN is kept
// as codes of zero with a scale of NaN: it reads back as NaN wherever it is seen, and nowhere else,
// since attention masks scores and probabilities (which the scales go into) and never multiplies a
// masked probability with anything but finite codes.
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

// The half-precision value of a code times this is the code's value.  An e4m3 code's sign, exponent
// and mantissa bits shifted into a half's places stand for the value times 2^-8 (the exponents'
// biases are 7 and 15), subnormal codes included; there is no infinity among e4m3 codes, and the
// pattern of its NaN comes out finite (480), which is what unwritten memory should do.
template <int FMT> __host__ __device__ constexpr float q8_half_unit() { return FMT == MF_Q8_E4M3 ? 256.0f : 1.0f; }

// code patterns of two vectors' or two dimensions' codes -> two halves.  `w` holds the codes that
// bytes LO and HI of the pair {a, b} (0-3: a's bytes, 4-7: b's) select; int8 expects w ^ 0x80808080.
template <int FMT, int LO, int HI> __device__ __forceinline__ uint32_t q8_halves(uint32_t a, uint32_t b) {
    if (FMT == MF_Q8_E4M3) {
        // the code in the upper byte of each half; the lower byte is whatever and is masked off
        const uint32_t p = __byte_perm(a, b, LO << 4 | HI << 12);
        return (p & 0x80008000u) | ((p >> 1) & 0x3f803f80u);
    }
    // 0x64 in the upper byte: the half 1024 + (code + 128)
    const uint32_t p = __byte_perm(a, b, LO | HI << 8);
    const uint32_t h = (p & 0x00ff00ffu) | 0x64006400u;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&r);
}
template <int FMT> __device__ __forceinline__ uint32_t q8_prepare(uint32_t w) {
    return FMT == MF_Q8_INT8 ? w ^ 0x80808080u : w;
}
// the two halves of bytes LO, HI of the word `w` (prepared) alone
template <int FMT, int LO, int HI> __device__ __forceinline__ uint32_t q8_halves(uint32_t w) {
    if (FMT == MF_Q8_E4M3) return q8_halves<FMT, LO, HI>(w, 0u);
    const uint32_t h = __byte_perm(w, 0x64646464u, LO | 4 << 4 | HI << 8 | 4 << 12);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&r);
}
// four codes of a word (not prepared) as float values of the codes
template <int FMT> __device__ __forceinline__ void q8_floats(uint32_t w, float* out) {
    if (FMT == MF_Q8_INT8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = (float)(int)(signed char)(w >> (8 * i));
        return;
    }
    const uint32_t lo = q8_halves<FMT, 0, 1>(w), hi = q8_halves<FMT, 2, 3>(w);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    out[0] = a.x * 256.0f; out[1] = a.y * 256.0f; out[2] = b.x * 256.0f; out[3] = b.y * 256.0f;
}
