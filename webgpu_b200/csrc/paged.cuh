// What the operators of a paged KV cache share (paged_ops.cu, paged_chunk.cu, verify_drafts.cu).
#pragma once

#include "common.cuh"

#include "lux/gpu/paged_ext.h"

#include <initializer_list>

namespace luxcuda {

inline size_t dtype_bytes(uint32_t dtype) {
    return dtype == LUX_QDTYPE_F32 ? 4 : dtype == LUX_QDTYPE_F16 || dtype == LUX_QDTYPE_BF16 ? 2 : 0;
}
inline bool holds(const Buffer* b, size_t elems, size_t elem_bytes = 4) {
    return b && b->ptr && (reinterpret_cast<uintptr_t>(b->ptr) % elem_bytes) == 0 && b->size / elem_bytes >= elems;
}
// products as a size, saturating
inline size_t mul(std::initializer_list<uint64_t> v) {
    unsigned __int128 r = 1;
    for (uint64_t x : v) {
        r *= x;
        if (r > (unsigned __int128)0x3fffffffffffffffull) return (size_t)0x3fffffffffffffffull;
    }
    return (size_t)r;
}

#ifdef __CUDACC__
// Accesses of L2 that stay where they stand: behind pdl_wait(), and either side of a barrier of the cluster.
__device__ __forceinline__ int32_t load_i32(const int32_t* src) {
    int32_t v;
    asm volatile("ld.global.cg.b32 %0, [%1];" : "=r"(v) : "l"(src) : "memory");
    return v;
}
__device__ __forceinline__ float load_f32(const float* src) { return __int_as_float(load_i32(reinterpret_cast<const int32_t*>(src))); }
__device__ __forceinline__ float2 load_f32x2(const float2* src) {
    float2 v;
    asm volatile("ld.global.cg.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "l"(src) : "memory");
    return v;
}
__device__ __forceinline__ uint4 load_u32x4(const void* src) {
    uint4 v;
    asm volatile("ld.global.cg.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(src) : "memory");
    return v;
}
__device__ __forceinline__ void store_i32(int32_t* dst, int32_t v) { asm volatile("st.global.cg.b32 [%0], %1;" ::"l"(dst), "r"(v) : "memory"); }

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
#endif

}  // namespace luxcuda
