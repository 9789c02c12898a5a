// Element types of the operators that take more than FP32: FP32, FP16 and BF16 values, computed on in FP32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace infmoe {

inline bool known_dtype(int dtype) { return dtype == INFMOE_F32 || dtype == INFMOE_F16 || dtype == INFMOE_BF16; }
inline int dtype_bytes(int dtype) { return dtype == INFMOE_F32 ? 4 : 2; }

#ifdef __CUDACC__
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N consecutive elements, in one access where N of them are 16 bytes (the pointer is then 16-byte aligned).
template <typename T, int N>
__device__ __forceinline__ void load_elems(const T* p, float (&v)[N]) {
    if constexpr (N * sizeof(T) == 16) {
        union {
            uint4 raw;
            T e[N];
        } u;
        u.raw = *reinterpret_cast<const uint4*>(p);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = to_float(u.e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = to_float(p[i]);
    }
}
template <typename T, int N>
__device__ __forceinline__ void store_elems(T* p, const float (&v)[N]) {
    if constexpr (N * sizeof(T) == 16) {
        union {
            uint4 raw;
            T e[N];
        } u;
#pragma unroll
        for (int i = 0; i < N; ++i) u.e[i] = from_float<T>(v[i]);
        *reinterpret_cast<uint4*>(p) = u.raw;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = from_float<T>(v[i]);
    }
}

// launch_chained (common.cuh) for a two-dimensional grid.
template <typename... Params, typename... Args>
inline cudaError_t launch_chained_2d(void (*kern)(Params...), dim3 grid, unsigned threads, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, Params(args)...);
}
#endif  // __CUDACC__

}  // namespace infmoe
