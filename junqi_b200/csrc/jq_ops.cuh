// jq_ops.cuh -- element types, vector loads and reductions of the policy
// operators (jq_norm.cu, jq_policy.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "jq_host.cuh"

namespace jq {

constexpr unsigned ALL = 0xffffffffu;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Element `i` of an array whose type is known at run time (float, or T).
template <typename T>
__device__ __forceinline__ float load_as(const void *p, bool f32, int64_t i) {
    return f32 ? ((const float *)p)[i] : to_f(((const T *)p)[i]);
}

// VEC consecutive elements, moved as one word of VEC * sizeof(T) bytes.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
    T v[VEC];
};

inline int elem_size(int dtype) { return dtype == JQ_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) { return dtype == JQ_F32 || dtype == JQ_F16 || dtype == JQ_BF16; }

}  // namespace jq
