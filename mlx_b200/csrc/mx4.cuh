// Microscaled 4-bit floating point: what the kernels that write and read the format share.
//
// A code is E2M1 (sign, two exponent bits, one mantissa bit: 0 .5 1 1.5 2 3 4 6), eight of them per 32-bit word along K, lowest
// bits first.  A block of neighbouring codes of a row shares a scale byte:
//   E8M0: 32 codes, 2^(byte - 127), 255 = NaN         E4M3: 16 codes, an 8-bit float (no infinities, 0x7F = NaN)
// Scales lie in tiles of 128 rows x 4 blocks, 512 bytes, the order in which the tensor cores take them: mx4_scale_at.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "lux_cuda_quant.h"
#include "pair.cuh"

namespace luxcuda {

__host__ __device__ constexpr int mx4_block(int format) { return format == LUX_CUDA_MX4_E8M0 ? 32 : 16; }
// tiles of scales along K (4 blocks each)
__host__ __device__ constexpr int mx4_tiles_k(int K, int format) { return (K / mx4_block(format) + 3) / 4; }
// byte offset of the scale word of (row, tile along K): the scales of blocks 4*tk .. 4*tk + 3
__host__ __device__ constexpr size_t mx4_scale_at(size_t row, int tk, int tiles_k) {
    return ((row >> 7) * tiles_k + tk) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}

// the largest magnitude of three, of two; NaN if one is
__device__ __forceinline__ float max_abs(float a, float b, float c) {
    float d;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float max_abs(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(fabsf(a)), "f"(fabsf(b)));
    return d;
}
// eight values to eight codes, nearest, ties to the even code, at most +-6
__device__ __forceinline__ uint32_t e2m1x8(Pair a, Pair b, Pair c, Pair d) {
    uint32_t r;
    asm("{ .reg .b8 w, x, y, z; cvt.rn.satfinite.e2m1x2.f32 w, %2, %1; cvt.rn.satfinite.e2m1x2.f32 x, %4, %3;\n"
        "  cvt.rn.satfinite.e2m1x2.f32 y, %6, %5; cvt.rn.satfinite.e2m1x2.f32 z, %8, %7; mov.b32 %0, {w, x, y, z}; }"
        : "=r"(r) : "f"(lo_of(a)), "f"(hi_of(a)), "f"(lo_of(b)), "f"(hi_of(b)), "f"(lo_of(c)), "f"(hi_of(c)), "f"(lo_of(d)), "f"(hi_of(d)));
    return r;
}
// two codes (the low byte of v) to their values, which are exact
__device__ __forceinline__ float2 e2m1x2_value(uint32_t v) {
    uint32_t h;
    asm("{ .reg .b8 t; cvt.u8.u16 t, %1; cvt.rn.f16x2.e2m1x2 %0, t; }" : "=r"(h) : "h"((uint16_t)v));
    return __half22float2(*reinterpret_cast<__half2*>(&h));
}
__device__ __forceinline__ uint32_t e4m3_of(float v) {  // nearest, at most 448; NaN: 0x7F
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(v));
    return r & 0xFFu;
}
__device__ __forceinline__ float e4m3_value(uint32_t b) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)b));
    return __half2float(__ushort_as_half((unsigned short)(h & 0xFFFFu)));
}
template <int FMT>
__device__ __forceinline__ float mx4_scale_value(uint32_t b) {
    if (FMT == LUX_CUDA_MX4_E4M3) return e4m3_value(b);
    return b == 255u ? __uint_as_float(0x7FC00000u) : __uint_as_float(b ? b << 23 : 1u << 22);
}

// E neighbouring values of a row per lane (8 or 16), neighbouring lanes side by side: their codes, and their block's scale byte
// (in all lanes of the block).  Every lane of the warp comes here.
//   E8M0: the scale is the power of two two below the largest value's own: that value lands in [4, 8), above 6 it is cut off.
//         Values times its reciprocal are exact.
//   E4M3: the scale is the largest value / 6, rounded to fp32 and then to the nearest 8-bit float; codes are those of the exact
//         quotients.  A quotient rounded to fp32 lies on the same side of every border between two codes as the exact one (border *
//         scale has at most seven significant bits, so a value that is not on it is at least an ulp away, and so, nearly, is the
//         quotient): fp32 division would do.  It costs eight operations a value; one multiplication by the rounded
//         reciprocal and one correction by the exact remainder gives the same number (Markstein 1990, theorem 8.1) in three.
template <int FMT, int E>
__device__ __forceinline__ void mx4_encode(Pair (&u)[E / 2], uint32_t (&codes)[E / 8], uint32_t& byte) {
    float m = max_abs(lo_of(u[0]), hi_of(u[0]));
#pragma unroll
    for (int i = 1; i < E / 2; i++) m = max_abs(m, lo_of(u[i]), hi_of(u[i]));
#pragma unroll
    for (int o = 1; o < mx4_block(FMT) / E; o <<= 1) m = max_abs(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (FMT == LUX_CUDA_MX4_E8M0) {
        const uint32_t field = min(__float_as_uint(m) >> 23, 254u);  // (an infinity as the largest finite value)
        byte = field > 2u ? field - 2u : 0u;
        const uint32_t inv = (254u - byte) << 23;
        if (m != m) byte = 255u;
#pragma unroll
        for (int i = 0; i < E / 2; i++) u[i] = mul2(u[i], pair_of(inv, inv));
    } else {
        // (the same correction for m / 6, and one step for the reciprocal of a scale: 126 numbers, all of them tested)
        const float top = m == INFINITY ? 3e38f : m, q = __fmul_rn(top, 1.0f / 6.0f);
        byte = e4m3_of(__fmaf_rn(__fmaf_rn(-6.0f, q, top), 1.0f / 6.0f, q));
        const float s = e4m3_value(byte);
        float inv;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
        inv = s > 0.0f ? __fmaf_rn(__fmaf_rn(-s, inv, 1.0f), inv, inv) : 0.0f;
        if (m == INFINITY) {  // (infinity - infinity below)
#pragma unroll
            for (int i = 0; i < E / 2; i++) u[i] = pair_of(fminf(fmaxf(lo_of(u[i]), -3e38f), 3e38f), fminf(fmaxf(hi_of(u[i]), -3e38f), 3e38f));
        }
        const Pair inv2 = pair_of(inv, inv), neg2 = pair_of(-s, -s);
#pragma unroll
        for (int i = 0; i < E / 2; i++) {
            const Pair t = mul2(u[i], inv2);
            u[i] = fma2(fma2(t, neg2, u[i]), inv2, t);
        }
    }
#pragma unroll
    for (int w = 0; w < E / 8; w++) codes[w] = e2m1x8(u[4 * w], u[4 * w + 1], u[4 * w + 2], u[4 * w + 3]);
}
// The scale word (4 blocks) that the lane's block belongs to, from the blocks' bytes; lanes of a word side by side.
template <int FMT, int E>
__device__ __forceinline__ uint32_t mx4_scale_word(uint32_t byte, int lane) {
    constexpr int LPB = mx4_block(FMT) / E;  // lanes per block
    uint32_t w = byte << (8 * ((lane / LPB) & 3));
    w |= __shfl_xor_sync(0xffffffffu, w, LPB);
    w |= __shfl_xor_sync(0xffffffffu, w, 2 * LPB);
    return w;
}

}  // namespace luxcuda
