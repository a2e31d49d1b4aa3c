// Element types as the token operators' kernels see them: 16-byte pieces widened to f32 and rounded back, and single
// elements for rows that are not aligned to 16 bytes.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace oxz {

// Launches overlap (launch_after, programmatic dependent launch): a kernel may start while the one before it in the stream still runs.
// after_previous() waits until that one has ended and what it wrote is visible; every thread of every kernel calls it before it ends,
// so that the end of a kernel is also the end of all before it. let_next() allows the next kernel to start.
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// N consecutive elements as one access of N * sizeof(T) bytes (32 as two of 16).
template <typename T, int N>
struct Vec {
    static constexpr int BYTES = N * (int)sizeof(T);
    union {
        T e[N];
        uint4 q[(BYTES + 15) / 16];
    };
    __device__ __forceinline__ Vec() {}
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (BYTES >= 16) {
#pragma unroll
            for (int i = 0; i < BYTES / 16; i++) q[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
        } else if constexpr (BYTES == 8) {
            *reinterpret_cast<uint2*>(q) = __ldg(reinterpret_cast<const uint2*>(p));
        } else {
            static_assert(N == 1, "a piece is 8, 16 or 32 bytes, or one element");
            e[0] = *p;
        }
    }
    // for memory that the same kernel, or one that may overlap it, also writes
    __device__ __forceinline__ void load_coherent(const T* p) {
        if constexpr (BYTES >= 16) {
#pragma unroll
            for (int i = 0; i < BYTES / 16; i++) q[i] = reinterpret_cast<const uint4*>(p)[i];
        } else {
            static_assert(N == 1, "a piece is 16 or 32 bytes, or one element");
            e[0] = *p;
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (BYTES >= 16) {
#pragma unroll
            for (int i = 0; i < BYTES / 16; i++) reinterpret_cast<uint4*>(p)[i] = q[i];
        } else if constexpr (BYTES == 8) {
            *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(q);
        } else {
            static_assert(N == 1, "a piece is 8, 16 or 32 bytes, or one element");
            *p = e[0];
        }
    }
};

// 32 bytes as one access: a whole sector per thread.
__device__ __forceinline__ void load32(const void* p, uint32_t* w) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(p) : "memory");
}
__device__ __forceinline__ void store32(void* p, const uint32_t* w) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
// Two f32 in one instruction, each rounded as alone
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{ .reg .b64 a, b, d; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; add.rn.f32x2 d, a, b; mov.b64 {%0, %1}, d; }"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{ .reg .b64 a, b, d; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; mul.rn.f32x2 d, a, b; mov.b64 {%0, %1}, d; }"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

template <typename S>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {  // two 16-bit values, rounded
    const S a = from_f32<S>(lo), b = from_f32<S>(hi);
    return (uint32_t)*reinterpret_cast<const uint16_t*>(&a) | (uint32_t)*reinterpret_cast<const uint16_t*>(&b) << 16;
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename S> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

}  // namespace oxz
