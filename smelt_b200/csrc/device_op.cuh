// Shared by the kernels of the operators on device memory (paged.cu, paged_attn.cu, logprobs.cu):
// storage types, vectors of eight elements, and the programmatic dependent launch.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>
#include <utility>

#include "tcgen05.cuh"

namespace gpt2q {

bool pdl_enabled();  // kernels.cu

using bf16 = __nv_bfloat16;

// Programmatic dependent launch, as in kernels.cu: every kernel launched through it waits (pdl_wait)
// before it reads or writes anything, so only its launch overlaps the previous kernel.
template <typename... KArgs, typename... Args>
inline cudaError_t launch_dependent(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                                    Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = pdl_enabled() ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(bf16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ bf16 from_f<bf16>(float x) { return __float2bfloat16_rn(x); }

__device__ __forceinline__ float ex2(float x) {  // 2^x to 2 ulp; results under 2^-126 are 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two fp32 operations in one instruction
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)),
          "l"(reinterpret_cast<unsigned long long&>(c)));
    return d;
}

// V consecutive elements; V = 8, and V = 4 of a store, move vectors (the address is a multiple of their bytes).
template <class T, int V>
__device__ __forceinline__ void load_vec(const T* p, float* f) {
    if constexpr (V == 8) {
        constexpr int N = sizeof(T) * 8 / 16;
        union {
            uint4 u[N];
            T t[8];
        } r;
#pragma unroll
        for (int i = 0; i < N; ++i) r.u[i] = reinterpret_cast<const uint4*>(p)[i];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = to_f(r.t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = to_f(p[i]);
    }
}
template <class T, int V>
__device__ __forceinline__ void store_vec(T* p, const float* f) {
    if constexpr (V == 8) {
        constexpr int N = sizeof(T) * 8 / 16;
        union {
            uint4 u[N];
            T t[8];
        } r;
#pragma unroll
        for (int i = 0; i < 8; ++i) r.t[i] = from_f<T>(f[i]);
#pragma unroll
        for (int i = 0; i < N; ++i) reinterpret_cast<uint4*>(p)[i] = r.u[i];
    } else if constexpr (V == 4) {
        using W = std::conditional_t<sizeof(T) == 4, uint4, uint2>;
        union {
            W u;
            T t[4];
        } r;
#pragma unroll
        for (int i = 0; i < 4; ++i) r.t[i] = from_f<T>(f[i]);
        *reinterpret_cast<W*>(p) = r.u;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) p[i] = from_f<T>(f[i]);
    }
}

}  // namespace gpt2q
