// K/V caches in 8 bits: a page's rows are codes, and each 16 neighbouring positions of a page and kv head have one scale 2^e, kept as the byte e + 127
// ([n_pages][n_head_kv][page / 16]). A value is its code times the scale. With powers of two every value is exact in f16 and bf16, and codes that are
// taken to a larger scale lose bits at their end only (e4m3 none but of what becomes subnormal); they cost at most one of an i8 code's 8 bits, and nothing of e4m3's.
#pragma once
#include "paged.cuh"

namespace llamd {

// The largest code, and the exponents of an append's scales: between them every value is exact in f16, subnormals included. f16x2: two codes as they are, or times a
// Times<C> of up to 2^kTimes (and from 2^kLow on), exactly.
template <int C> struct Cache8;
template <int C> struct Times;
template <> struct Cache8<kPagedI8> {
    static constexpr float kMost = 127.0f;
    static constexpr int kLow = -24, kHigh = 9;
    static constexpr int kTimes = 5;  // (1152 2^5 is in f16)
    // f16x2 of the codes in bytes 0, 1 (half 0) or 2, 3 (half 1) of x. 1024 + 128 + c is a half whose low byte is c with its sign bit flipped.
    template <int HALF> static __device__ __forceinline__ uint32_t f16x2(uint32_t x) {
        const uint32_t y = __byte_perm(x ^ 0x80808080u, 0x64646464u, HALF ? 0x4342 : 0x4140), bias = 0x64806480u;
        const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&y), *reinterpret_cast<const __half2 *>(&bias));
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    template <int HALF> static __device__ __forceinline__ uint32_t f16x2(uint32_t x, const Times<kPagedI8> &t);
};
template <> struct Cache8<kPagedE4m3> {
    static constexpr float kMost = 448.0f;
    static constexpr int kLow = -15, kHigh = 7;
    static constexpr int kTimes = 7;
    // (33 pairs a clock and SM measured, where a permutation, a shift and two logical operations, which give 2^-8 of a pair, go at 64 a clock each)
    template <int HALF> static __device__ __forceinline__ uint32_t f16x2(uint32_t x) {
        uint32_t y;
        if constexpr (HALF) asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, b;\n\t}" : "=r"(y) : "r"(x));
        else asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\t}" : "=r"(y) : "r"(x));
        return y;
    }
    template <int HALF> static __device__ __forceinline__ uint32_t f16x2(uint32_t x, const Times<kPagedE4m3> &t);
};

__device__ __forceinline__ float scale_of(int byte) { return __int_as_float(byte << 23); }             // 2^e of the byte e + 127, 1 to 254
__device__ __forceinline__ float scale_inverse(int byte) { return __int_as_float((254 - byte) << 23); }  // 2^-e, of 0 to 253

// A power of two that codes are taken times, as f16 takes it: that of a scale, but for what is above 2^kTimes or below 2^kLow of it, which `rest` has (as a scale's byte).
template <> struct Times<kPagedE4m3> {
    __half2 by;
    int rest;
    __device__ __forceinline__ explicit Times(int byte) {
        const int part = min(max(byte, Cache8<kPagedE4m3>::kLow + 127), Cache8<kPagedE4m3>::kTimes + 127);
        by = __float2half2_rn(scale_of(part)), rest = byte - part + 127;
    }
};
template <> struct Times<kPagedI8> {
    __half2 by, bias;
    int rest;
    __device__ __forceinline__ explicit Times(int byte) {
        const int part = min(max(byte, Cache8<kPagedI8>::kLow + 127), Cache8<kPagedI8>::kTimes + 127);
        by = __float2half2_rn(scale_of(part)), bias = __float2half2_rn(-1152.0f * scale_of(part)), rest = byte - part + 127;
    }
};
template <int HALF> __device__ __forceinline__ uint32_t Cache8<kPagedE4m3>::f16x2(uint32_t x, const Times<kPagedE4m3> &t) {
    const uint32_t y = f16x2<HALF>(x);
    const __half2 h = __hmul2(*reinterpret_cast<const __half2 *>(&y), t.by);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <int HALF> __device__ __forceinline__ uint32_t Cache8<kPagedI8>::f16x2(uint32_t x, const Times<kPagedI8> &t) {  // (1152 + c) 2^e - 1152 2^e: no more than f16x2 of the codes
    const uint32_t y = __byte_perm(x ^ 0x80808080u, 0x64646464u, HALF ? 0x4342 : 0x4140);
    const __half2 h = __hfma2(*reinterpret_cast<const __half2 *>(&y), t.by, t.bias);
    return *reinterpret_cast<const uint32_t *>(&h);
}

}  // namespace llamd
