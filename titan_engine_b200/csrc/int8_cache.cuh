// int8_cache.cuh — the tile of an INT8 pool and the rounding its rows are defined by.
//
// Tile (page, kv head), contiguous: 16 K rows of D codes, 16 V rows of D codes, 16 K scales, 16 V scales (f32): codes and
// scales of a page travel in ONE copy (4224 bytes at D = 128, 2176 at D = 64), and whatever moves pages (a fork's
// copy) moves the scales with them.  A code is stored as code + 128: an unsigned byte u is the 16-bit float 1024 + u
// when it is put under the byte 0x64, so that expanding two codes costs one byte permute and one subtraction.
#pragma once

#include "tk_kernels.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace tk {

constexpr int kI8Page = 16;                             // tokens per page of an INT8 pool
constexpr float kI8AmaxMin = 9.094947017729282e-13f;    // 2^-40: the scale of an all-zero row stays positive
constexpr float kI8AmaxMax = 18446744073709551616.0f;   // 2^64: larger values saturate, scales of one pool span < 2^105

__host__ __device__ constexpr int i8_tile_bytes(int D) { return 2 * kI8Page * D + 2 * kI8Page * (int)sizeof(float); }
// byte offset of a row of codes / of its scale inside a tile
__host__ __device__ constexpr int i8_row_off(int D, int kv, int r) { return (kv * kI8Page + r) * D; }
__host__ __device__ constexpr int i8_scale_off(int D, int kv, int r) { return 2 * kI8Page * D + (kv * kI8Page + r) * (int)sizeof(float); }

// What a row's largest magnitude makes of it: `to_code`, 127 / amax to four parts in 2^24, and the scale, amax / 127 rounded to
// nearest (amax has at most 11 significant bits: a product with the rounded 1/127 and one residual step, Markstein's
// correction, give the quotient's nearest float, checked for every significand).  A NaN among the values makes the scale NaN, so that the row reads
// as NaN; infinities saturate like any large value.
struct I8Row { float to_code, scale; };
__device__ __forceinline__ I8Row i8_row(float amax) {
    const float a = fminf(fmaxf(amax, kI8AmaxMin), kI8AmaxMax);           // (a NaN becomes the minimum here)
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(a));               // within one unit in the last place
    constexpr float k127 = 1.0f / 127.0f;
    const float q = a * k127;
    return I8Row{127.0f * inv, amax != amax ? amax : fmaf(fmaf(-q, 127.0f, a), k127, q)};
}

// code + 128 in the low byte of the result: the integer nearest to 127 x / amax, ties to even, EXACTLY.
// x and amax have at most 11 significant bits, A and B: the quotient Q = 127 x / amax is 127 A 2^-n / B for some n, so it is a
// half-integer or at least 1 / (2 B 2^n) = Q / (254 A) > Q 2^-19 away from every one: 16 units in the last place (ulp) of Q.
// y = x to_code has relative errors of 2^-23 (the reciprocal) and twice 2^-24 (two products): less than 4 ulps.  Snapped
// to a multiple of 16 ulps (20 significant bits, half-integers among them) y is the half-integer itself where Q is one, and
// otherwise within 12 ulps of a Q that is at least 16 ulps from it: on the right side.  The addition of a constant whose
// neighbours are 1 apart then rounds to the nearest integer, ties to even.  Checked against exact arithmetic for every pair of
// significands.  CLAMP: amax may have been cut to 2^64.
template <bool CLAMP>
__device__ __forceinline__ uint32_t i8_code(float x, float to_code) {
    float y = x * to_code;
    if (CLAMP) y = fminf(fmaxf(y, -127.0f), 127.0f);
    const float snapped = __uint_as_float((__float_as_uint(y) + 8u) & ~15u);
    return __float_as_uint(__fadd_rn(snapped, 12582912.0f + 128.0f));
}

// Two bytes of `w`, picked by SEL, -> two codes as fp16, exact: 1024 + u, minus 1152.
template <uint32_t SEL>
__device__ __forceinline__ uint32_t i8_expand(uint32_t w) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(w), "r"(0x64646464u), "n"(SEL));
    const uint32_t bias = 0x64806480u;
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&r), *reinterpret_cast<const __half2*>(&bias));
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Shared-memory accesses by 32-bit address (a pointer that went through a lambda or a conditional may be taken for a generic one)
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, const uint4& v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ float lds32(uint32_t addr) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void sts32(uint32_t addr, float v) {
    asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ unsigned long long lds64(uint32_t addr) {
    unsigned long long v;
    asm volatile("ld.shared.b64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
    return v;
}

// two 16-bit values held in one word -> floats
template <bool BF16>
__device__ __forceinline__ float2 i8_unpack2(uint32_t w) {
    if (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    const __half2 h = *reinterpret_cast<const __half2*>(&w);
    return __half22float2(h);
}

// Eight 16-bit values (16 bytes) -> eight codes (8 bytes).
template <bool BF16, bool CLAMP>
__device__ __forceinline__ uint2 i8_codes8(const uint4& x, float to_code) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = i8_unpack2<BF16>(w[i]);
        c[i] = __byte_perm(i8_code<CLAMP>(f.x, to_code), i8_code<CLAMP>(f.y, to_code), 0x0040);
    }
    return make_uint2(__byte_perm(c[0], c[1], 0x5410), __byte_perm(c[2], c[3], 0x5410));
}

// Largest magnitude of eight 16-bit values, as the 16-bit pattern without its sign: patterns order like the magnitudes, and
// a NaN's is above every number's.
__device__ __forceinline__ uint32_t i8_absmax8(const uint4& x) {
    uint32_t m = __vmaxu2(__vmaxu2(x.x & 0x7FFF7FFFu, x.y & 0x7FFF7FFFu), __vmaxu2(x.z & 0x7FFF7FFFu, x.w & 0x7FFF7FFFu));
    return max(m & 0xFFFFu, m >> 16);
}
template <bool BF16>
__device__ __forceinline__ float i8_amax_value(uint32_t pattern) {
    return BF16 ? __uint_as_float(pattern << 16) : __half2float(__ushort_as_half((unsigned short)pattern));
}

}  // namespace tk
