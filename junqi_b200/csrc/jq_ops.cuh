// jq_ops.cuh -- element types, vector loads and reductions of the policy
// operators (jq_norm.cu, jq_policy.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>
#include <string.h>

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

// Two floats in a register pair, and the packed arithmetic on them: each
// instruction does the work of two.
struct f2 {
    uint64_t v;
};
__device__ __forceinline__ f2 make_f2(float a, float b) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ f2 both(float a) { return make_f2(a, a); }
__device__ __forceinline__ float2 parts(f2 a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
    return r;
}
__device__ __forceinline__ f2 operator+(f2 a, f2 b) {
    f2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ f2 operator*(f2 a, f2 b) {
    f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ f2 to_f2(const float *v) { return make_f2(v[0], v[1]); }
__device__ __forceinline__ f2 to_f2(const __half *v) {
    __half2 h;
    memcpy(&h, v, 4);
    const float2 p = __half22float2(h);
    return make_f2(p.x, p.y);
}
__device__ __forceinline__ f2 to_f2(const __nv_bfloat16 *v) {
    uint32_t u;
    memcpy(&u, v, 4);  // a bfloat16 is the upper half of its float
    return make_f2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ void from_f2(float *v, f2 a) {
    const float2 p = parts(a);
    v[0] = p.x, v[1] = p.y;
}
__device__ __forceinline__ void from_f2(__half *v, f2 a) {
    const float2 p = parts(a);
    const __half2 h = __floats2half2_rn(p.x, p.y);
    memcpy(v, &h, 4);
}
__device__ __forceinline__ void from_f2(__nv_bfloat16 *v, f2 a) {
    const float2 p = parts(a);
    const __nv_bfloat162 h = __floats2bfloat162_rn(p.x, p.y);
    memcpy(v, &h, 4);
}

// Asynchronous copies into shared memory, in groups that complete in order.
__device__ __forceinline__ void copy16(uint32_t to, const void *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void *from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_end_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait_but() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Bytes [from, from + bytes) of an array that spans [lo, hi) into shared
// memory at `to` + (from & 15), by threads t of n: the 16-byte blocks around
// them, as one copy each where the array has the whole block, by elements
// where it ends inside.  ALIGNED: from and bytes are multiples of 16.
template <typename T, bool ALIGNED>
__device__ __forceinline__ void copy_span(char *to, const char *from, int bytes, const char *lo, const char *hi, int t, int n) {
    const int skip = ALIGNED ? 0 : (int)((uintptr_t)from & 15), blocks = (skip + bytes + 15) >> 4;
    const char *first = from - skip;
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
    if constexpr (ALIGNED) {
        (void)lo, (void)hi;
#pragma unroll 2
        for (int k = t; k < blocks; k += n) copy16(at + 16 * k, first + 16 * k);
    } else {
        const bool all = first >= lo && first + 16 * blocks <= hi;
        for (int k = t; k < blocks; k += n) {
            const char *p = first + 16 * k;
            if (all || (p >= lo && p + 16 <= hi)) {
                copy16(at + 16 * k, p);
            } else {
                const char *a = p < from ? from : p, *e = p + 16 < from + bytes ? p + 16 : from + bytes;
                for (; a < e; a += sizeof(T)) *(T *)(to + (a - first)) = *(const T *)a;
            }
        }
    }
}

// Thread-block clusters: this CTA's place, a store into another CTA's shared
// memory, and the barrier that makes it visible.
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_store(double *mine, uint32_t rank, double v) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(mine)), "r"(rank));
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(v) : "memory");
}
__device__ __forceinline__ void cluster_store4(float4 *mine, uint32_t rank, float4 v) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(mine)), "r"(rank));
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

inline int elem_size(int dtype) { return dtype == JQ_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) { return dtype == JQ_F32 || dtype == JQ_F16 || dtype == JQ_BF16; }

}  // namespace jq
