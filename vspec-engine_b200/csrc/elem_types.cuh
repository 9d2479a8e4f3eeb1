// elem_types.cuh -- element types of the verification operators (fp32, fp16,
// bf16): conversions to and from fp32 and vectors of up to 16 bytes.
#pragma once

#include "common.cuh"

#include <initializer_list>

namespace vb200 {

template <typename T> __device__ __forceinline__ float elem_to_f32(T v);
template <> __device__ __forceinline__ float elem_to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float elem_to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float elem_to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T> __device__ __forceinline__ T elem_from_f32(float v);
template <> __device__ __forceinline__ float elem_from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half elem_from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 elem_from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V elements moved by one load or store of V * sizeof(T) bytes.
template <typename T, int V>
struct alignas(V * sizeof(T)) Vec {
    T e[V];
};

// Widest vector (16 bytes of T) that every listed count (elements) and address
// allows, else 2 elements, else 1.
template <typename T>
inline int elem_vec(uintptr_t addresses, size_t counts) {
    constexpr int full = 16 / (int)sizeof(T);
    if (counts % full == 0 && addresses % 16 == 0) return full;
    if (counts % 2 == 0 && addresses % (2 * sizeof(T)) == 0) return 2;
    return 1;
}

inline bool elem_type_known(int t) { return t == VSPEC_B200_T_F32 || t == VSPEC_B200_T_F16 || t == VSPEC_B200_T_BF16; }
inline size_t elem_bytes(int t) { return t == VSPEC_B200_T_F32 ? 4 : 2; }

// Whether one of the addresses is no multiple of its values' size, which would fault on the device.
inline bool off_type(size_t size, std::initializer_list<const void*> addresses) {
    for (const void* a : addresses)
        if ((uintptr_t)a % size != 0) return true;
    return false;
}

// Two fp32 values an instruction, each rounded as by itself.
typedef unsigned long long pair32;
__device__ __forceinline__ pair32 pack2(float a, float b) {
    pair32 y;
    asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ void unpack2(pair32 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ float low2(pair32 v) { return __uint_as_float((unsigned)v); }
__device__ __forceinline__ float high2(pair32 v) { return __uint_as_float((unsigned)(v >> 32)); }
__device__ __forceinline__ pair32 add2(pair32 a, pair32 b) {
    pair32 y;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
    return y;
}
__device__ __forceinline__ pair32 mul2(pair32 a, pair32 b) {
    pair32 y;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
    return y;
}
__device__ __forceinline__ pair32 fma2(pair32 a, pair32 b, pair32 c) {
    pair32 y;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(a), "l"(b), "l"(c));
    return y;
}

}  // namespace vb200
