// serve.cuh -- element types and small helpers shared by the batched-serving
// operators (attn_shared.cu, lora.cu, verify.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kernels.cuh"
#include "pdl.cuh"
#include "smem_limit.h"

namespace loom {

cudaStream_t rt_stream(void *s);
int rt_need_init();
int rt_decline(const char *why);
int rt_fail(const char *what, cudaError_t e);

constexpr int T_BF16 = 30;  // ggml type id; T_F16 is in common.cuh

template <class T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

inline size_t elem_bytes(int type) { return type == T_F32 ? 4 : (type == T_F16 || type == T_BF16) ? 2 : 0; }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Let kernel K use `smem` bytes of dynamic shared memory.
template <auto K> cudaError_t allow_smem(size_t smem) {
    static SmemLimit limit;
    int dev = 0;
    if (const cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
    return limit.need(dev, smem, [](size_t bytes) {
        cudaError_t e = cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        // kernels that are to share an SM need the same split of its memory: all of it shared
        if (e == cudaSuccess && bytes > 48 * 1024)
            e = cudaFuncSetAttribute(K, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        return e;
    });
}

// f(T{}) with the element type behind a type id (checked by the caller)
template <class F> auto by_type(int type, F f) {
    return type == T_F32 ? f(float{}) : type == T_F16 ? f(__half{}) : f(__nv_bfloat16{});
}

}  // namespace loom
