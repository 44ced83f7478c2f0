// Element types of the row operators (MGGB_F32 / MGGB_BF16 / MGGB_F16): loads widen to fp32, stores round once to
// nearest even.  All sums, statistics and exponentials of those operators are fp32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <initializer_list>
#include <type_traits>
#include "common.h"

namespace mggb {

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// Two fp32 operations in one instruction (sm_100); each half rounds as the scalar operation does.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
        "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
        "add.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
        "mul.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// Loads that stay where they are written: the compiler may otherwise move them behind what comes in between, next to their use.
__device__ __forceinline__ void load_now(uint4& r, const void* p) {
    asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
}
__device__ __forceinline__ void load_now(uint2& r, const void* p) { asm volatile("ld.global.nc.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p)); }
__device__ __forceinline__ void load_now(unsigned& r, const void* p) { asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(r) : "l"(p)); }
__device__ __forceinline__ void load_now(unsigned short& r, const void* p) { asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(r) : "l"(p)); }

// A vector of VB bytes of T as it lies in memory; get() widens one element.
template <int VB> struct RawOf;
template <> struct RawOf<16> { using R = uint4; };
template <> struct RawOf<8> { using R = uint2; };
template <> struct RawOf<4> { using R = unsigned; };
template <> struct RawOf<2> { using R = unsigned short; };

template <typename T, int VB>
struct Pack {
    static constexpr int VE = VB / (int)sizeof(T);
    using R = typename RawOf<VB>::R;
    union { R raw; T e[VE]; };
    __device__ __forceinline__ Pack() : raw{} {}
    __device__ __forceinline__ float get(int i) const { return to_f32(e[i]); }
    __device__ __forceinline__ void widen(float (&f)[VE]) const {
#pragma unroll
        for (int i = 0; i < VE; i++) f[i] = get(i);
    }
    // rounds VE values; 16-bit ones in pairs, one conversion instruction for two
    __device__ __forceinline__ void narrow(const float (&f)[VE]) {
        if constexpr (sizeof(T) == 2 && VE > 1) {
#pragma unroll
            for (int i = 0; i < VE; i += 2) {
                if constexpr (std::is_same<T, __half>::value) *reinterpret_cast<__half2*>(&e[i]) = __floats2half2_rn(f[i], f[i + 1]);
                else *reinterpret_cast<__nv_bfloat162*>(&e[i]) = __floats2bfloat162_rn(f[i], f[i + 1]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < VE; i++) e[i] = from_f32<T>(f[i]);
        }
    }
    // streaming: read or written once (a row is not read again, so it need not stay in a cache)
    __device__ __forceinline__ void load(const T* p) { raw = __ldcs(reinterpret_cast<const R*>(p)); }
    __device__ __forceinline__ void store(T* p) const { __stcs(reinterpret_cast<R*>(p), raw); }
};

// Largest power of two up to 16 that divides the address and every stride (both in bytes).
inline int common_alignment(std::initializer_list<uint64_t> v) {
    uint64_t a = 16;
    for (uint64_t x : v) a |= x;
    return (int)(a & (~a + 1));
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int off = 16; off; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}

inline int elem_bytes(int dtype) { return dtype == MGGB_F32 ? 4 : 2; }

}  // namespace mggb

#define MGGB_REQUIRE_DTYPE(dtype, who) \
    MGGB_REQUIRE((dtype) == MGGB_F32 || (dtype) == MGGB_BF16 || (dtype) == MGGB_F16, who ": dtype must be MGGB_F32, MGGB_BF16 or MGGB_F16, got %d", (int)(dtype))

// Calls fn<T>(args...) for the dtype (already checked).
#define MGGB_BY_DTYPE(dtype, fn, ...)                                   \
    ((dtype) == MGGB_F32 ? fn<float>(__VA_ARGS__)                       \
     : (dtype) == MGGB_BF16 ? fn<__nv_bfloat16>(__VA_ARGS__) : fn<__half>(__VA_ARGS__))
