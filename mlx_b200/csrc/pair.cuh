// Two fp32 values in a register pair: the fp32 pipe takes both in one instruction.
#pragma once
#include <cstdint>

namespace luxcuda {

using Pair = unsigned long long;
__device__ __forceinline__ Pair pair_of(uint32_t lo, uint32_t hi) { return (Pair)hi << 32 | lo; }
__device__ __forceinline__ Pair pair_of(float lo, float hi) { return pair_of(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ float lo_of(Pair p) { return __uint_as_float((uint32_t)p); }
__device__ __forceinline__ float hi_of(Pair p) { return __uint_as_float((uint32_t)(p >> 32)); }
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
// bf16 pairs
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t w;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    return w;
}
__device__ __forceinline__ Pair unpack2(uint32_t w) { return pair_of(w << 16, w & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t pack2(Pair p) { return pack_bf16(lo_of(p), hi_of(p)); }

// 32 bytes, each read or written once: past L1
struct Words8 {
    uint32_t v[8];
};
__device__ __forceinline__ Words8 ld_once_32(const void* p) {
    Words8 r;
    asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r.v[0]), "=r"(r.v[1]), "=r"(r.v[2]), "=r"(r.v[3]), "=r"(r.v[4]), "=r"(r.v[5]), "=r"(r.v[6]), "=r"(r.v[7])
                 : "l"(p));
    return r;
}
__device__ __forceinline__ void st_once_32(void* p, const Words8& r) {
    asm volatile("st.global.L1::no_allocate.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r.v[0]), "r"(r.v[1]), "r"(r.v[2]), "r"(r.v[3]), "r"(r.v[4]),
                 "r"(r.v[5]), "r"(r.v[6]), "r"(r.v[7]) : "memory");
}

}  // namespace luxcuda
