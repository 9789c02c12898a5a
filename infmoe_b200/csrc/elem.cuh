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

// Two neighbours in one 32-bit word (the first in the lower half), by one conversion.
template <typename T> __device__ __forceinline__ float2 unpack_pair(uint32_t w);
template <> __device__ __forceinline__ float2 unpack_pair<__half>(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <> __device__ __forceinline__ float2 unpack_pair<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <typename T> __device__ __forceinline__ uint32_t pack_pair(float a, float b);
template <> __device__ __forceinline__ uint32_t pack_pair<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack_pair<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The 16 / sizeof(T) elements of 16 bytes.
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& raw, float (&v)[16 / sizeof(T)]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            v[i] = __uint_as_float(w[i]);
        } else {
            const float2 f = unpack_pair<T>(w[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}
template <typename T>
__device__ __forceinline__ uint4 pack16(const float (&v)[16 / sizeof(T)]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4)
            w[i] = __float_as_uint(v[i]);
        else
            w[i] = pack_pair<T>(v[2 * i], v[2 * i + 1]);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// N consecutive elements, in one access where N of them are 16 bytes (the pointer is then 16-byte aligned).
template <typename T, int N>
__device__ __forceinline__ void load_elems(const T* p, float (&v)[N]) {
    if constexpr (N * sizeof(T) == 16) {
        unpack16<T>(*reinterpret_cast<const uint4*>(p), v);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = to_float(p[i]);
    }
}
template <typename T, int N>
__device__ __forceinline__ void store_elems(T* p, const float (&v)[N]) {
    if constexpr (N * sizeof(T) == 16) {
        *reinterpret_cast<uint4*>(p) = pack16<T>(v);
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
