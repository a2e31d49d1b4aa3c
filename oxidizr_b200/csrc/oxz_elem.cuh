// Element types as the token operators' kernels see them: 16-byte pieces widened to f32 and rounded back, and single
// elements for rows that are not aligned to 16 bytes.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace oxz {

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// N consecutive elements as one access of N * sizeof(T) bytes (16 at most; 32 as two).
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
        } else {
            static_assert(N == 1, "a piece is 16 bytes or one element");
            e[0] = *p;
        }
    }
    // for memory that the same kernel, or one that may overlap it, also writes
    __device__ __forceinline__ void load_coherent(const T* p) {
        if constexpr (BYTES >= 16) {
#pragma unroll
            for (int i = 0; i < BYTES / 16; i++) q[i] = reinterpret_cast<const uint4*>(p)[i];
        } else {
            e[0] = *p;
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (BYTES >= 16) {
#pragma unroll
            for (int i = 0; i < BYTES / 16; i++) reinterpret_cast<uint4*>(p)[i] = q[i];
        } else {
            *p = e[0];
        }
    }
};

}  // namespace oxz
