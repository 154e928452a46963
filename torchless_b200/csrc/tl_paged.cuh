// tl_paged.cuh -- pieces shared by the operators of the paged serving step
// (tl_paged.cu, tl_paged_attn.cu, tl_paged_attn_tc.cu, tl_sample_rows.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tl_common.cuh"

namespace tl {
namespace paged {

// 8 consecutive elements rounded from fp32 (fp32 ones are read too), one 16-byte access (two for fp32).
template <typename T>
struct Vec8;
template <>
struct Vec8<float> {
    static __device__ __forceinline__ void load(float (&v)[8], const float* p) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
    static __device__ __forceinline__ void store(float* p, const float (&v)[8]) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
};
template <>
struct Vec8<__half> {
    static __device__ __forceinline__ void store(__half* p, const float (&v)[8]) {
        __half2 h[4];
#pragma unroll
        for (int j = 0; j < 4; j++) h[j] = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
        *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
    }
};
template <>
struct Vec8<__nv_bfloat16> {
    static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&v)[8]) {
        __nv_bfloat162 h[4];
#pragma unroll
        for (int j = 0; j < 4; j++) h[j] = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
        *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
    }
};

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

inline size_t dtype_size(tl_dtype t) { return t == TL_F32 ? 4 : 2; }
inline bool dtype_ok(tl_dtype t) { return t == TL_F32 || t == TL_F16 || t == TL_BF16; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The checks of a cache that every entry point makes.
tl_status check_cache(const char* who, const tl_paged_cache* c);

}  // namespace paged
}  // namespace tl
