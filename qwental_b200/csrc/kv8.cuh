// Codes and rows of the 8-bit key-value cache, device side.
#pragma once
#include "common.cuh"
#include "kv8.h"
#include <cuda_fp8.h>

namespace qw {

template <int FMT>
__device__ __forceinline__ constexpr float kv8_largest() {
    return FMT == QW_KV8_E4M3 ? 448.f : 127.f;
}
// An e4m3 code's bits, moved one place down behind the sign, are the fp16 number 2^-8 times its value: exact, subnormal codes too, and never a NaN
// (0x7f becomes 480 * 2^-8).  An int8 code becomes its value.  KV8_UNIT * the fp16 number is what the code stands for.
template <int FMT>
__device__ __forceinline__ constexpr float kv8_unit() {
    return FMT == QW_KV8_E4M3 ? 256.f : 1.f;
}
// Two codes, in the upper bytes of the two halves of v, as fp16 numbers (e4m3).
__device__ __forceinline__ uint32_t kv8_e4m3_half2(uint32_t v) { return ((v >> 1) & 0x3f803f80u) | (v & 0x80008000u); }
// Two codes plus 128, in the lower bytes of the two halves of v whose upper bytes are 0x64 (1024 + byte), as fp16 numbers (int8).
__device__ __forceinline__ uint32_t kv8_int8_half2(uint32_t v) {
    const __half2 h = __hsub2(*(const __half2 *)&v, __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));  // 1152
    return *(const uint32_t *)&h;
}
// Four codes -> fp16 pairs (0, 1) and (2, 3)
template <int FMT>
__device__ __forceinline__ void kv8_halves(uint32_t w, uint32_t &h01, uint32_t &h23) {
    if (FMT == QW_KV8_E4M3) {
        h01 = kv8_e4m3_half2(__byte_perm(w, 0, 0x1404));
        h23 = kv8_e4m3_half2(__byte_perm(w, 0, 0x3424));
    } else {
        w ^= 0x80808080u;
        h01 = kv8_int8_half2(__byte_perm(w, 0x64646464u, 0x4140));
        h23 = kv8_int8_half2(__byte_perm(w, 0x64646464u, 0x4342));
    }
}
// The same for products: their values as fp16 numbers; an e4m3 code that is no number becomes a NaN.  (Two conversions per four codes instead of eight
// operations; as many cycles of the pipe each.)
template <int FMT>
__device__ __forceinline__ void kv8_operands(uint32_t w, uint32_t &h01, uint32_t &h23) {
    if (FMT == QW_KV8_E4M3)
        asm("{\n\t.reg .b16 l, h;\n\t"
            "mov.b32 {l, h}, %2;\n\t"
            "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
            "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
            : "=r"(h01), "=r"(h23)
            : "r"(w));
    else kv8_halves<FMT>(w, h01, h23);
}
template <int FMT>
__device__ __forceinline__ void kv8_decode4(uint32_t w, float (&x)[4]) {
    uint32_t a, b;
    kv8_halves<FMT>(w, a, b);
    const float2 f = __half22float2(*(const __half2 *)&a), g = __half22float2(*(const __half2 *)&b);
    x[0] = f.x * kv8_unit<FMT>(), x[1] = f.y * kv8_unit<FMT>(), x[2] = g.x * kv8_unit<FMT>(), x[3] = g.y * kv8_unit<FMT>();
}
// Two numbers within the format's range -> two codes in the low bytes, to nearest, ties to even.
template <int FMT>
__device__ __forceinline__ uint32_t kv8_encode2(float a, float b) {
    if (FMT == QW_KV8_E4M3) return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    return ((uint32_t)__float2int_rn(a) & 0xff) | ((uint32_t)__float2int_rn(b) & 0xff) << 8;
}

__device__ __forceinline__ float kv8_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float kv8_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T kv8_round(float x);
template <>
__device__ __forceinline__ __half kv8_round<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 kv8_round<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// E (2, 4 or 8) consecutive 2-byte values: one load or store where the address allows it (strides are the caller's), else one each.
template <int E>
struct Kv8Pack;
template <> struct Kv8Pack<2> { typedef uint32_t t; };
template <> struct Kv8Pack<4> { typedef uint2 t; };
template <> struct Kv8Pack<8> { typedef uint4 t; };
template <int E, class T>
__device__ __forceinline__ void kv8_load(const T *p, float *x) {
    typedef typename Kv8Pack<E>::t P;
    union { P v; T e[E]; };
    if (((uintptr_t)p & (2 * E - 1)) == 0) v = __ldcg((const P *)p);
    else {
#pragma unroll
        for (int i = 0; i < E; i++) e[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < E; i++) x[i] = kv8_float(e[i]);
}
template <int E, class T>
__device__ __forceinline__ void kv8_store(T *p, const float *x) {
    typedef typename Kv8Pack<E>::t P;
    union { P v; T e[E]; };
#pragma unroll
    for (int i = 0; i < E; i++) e[i] = kv8_round<T>(x[i]);
    if (((uintptr_t)p & (2 * E - 1)) == 0) *(P *)p = v;
    else {
#pragma unroll
        for (int i = 0; i < E; i++) p[i] = e[i];
    }
}

// Eight consecutive 2-byte values as four words, whatever the address.
template <class T>
__device__ __forceinline__ void kv8_load_raw8(const T *p, uint32_t (&w)[4]) {
    const uint16_t *u = (const uint16_t *)p;
    if (((uintptr_t)p & 15) == 0) {
        const uint4 v = *(const uint4 *)p;  // (through L1: the warps of a block mostly want the same)
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = (uint32_t)u[2 * i] | (uint32_t)u[2 * i + 1] << 16;
    }
}
template <class T>
__device__ __forceinline__ float2 kv8_float2(uint32_t w);
template <>
__device__ __forceinline__ float2 kv8_float2<__half>(uint32_t w) { return __half22float2(*(const __half2 *)&w); }
template <>
__device__ __forceinline__ float2 kv8_float2<__nv_bfloat16>(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }

__device__ __forceinline__ void lds128(uint32_t (&v)[4], uint32_t addr) {
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void lds64(uint32_t &a, uint32_t &b, uint32_t addr) {
    asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(a), "=r"(b) : "r"(addr) : "memory");
}

}  // namespace qw
