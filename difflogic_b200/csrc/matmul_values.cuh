// Values of the types that dense layers and orthogonalised updates take, read as and written from fp32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace dl {

enum MatmulType { kFloat32 = 0, kBFloat16 = 1, kFloat16 = 2 };

#ifdef __CUDACC__
__device__ __forceinline__ float load_as_float(const void *p, int64_t i, int type) {
    if (type == kFloat32) return reinterpret_cast<const float *>(p)[i];
    const uint16_t v = reinterpret_cast<const uint16_t *>(p)[i];
    return type == kBFloat16 ? __uint_as_float((uint32_t)v << 16) : __half2float(__ushort_as_half(v));
}
__device__ __forceinline__ uint16_t to_16bit(float v, int type) {
    return type == kBFloat16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}
// Up to four neighbouring values, in one access where all are there and the address allows it.
__device__ __forceinline__ void load4(const void *p, int64_t i, int type, int valid, float (&v)[4]) {
    const char *at = reinterpret_cast<const char *>(p) + i * (type == kFloat32 ? 4 : 2);
    if (valid == 4 && type == kFloat32 && (reinterpret_cast<uintptr_t>(at) & 15) == 0) {
        const float4 f = *reinterpret_cast<const float4 *>(at);
        v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else if (valid == 4 && type != kFloat32 && (reinterpret_cast<uintptr_t>(at) & 7) == 0) {
        const ushort4 u = *reinterpret_cast<const ushort4 *>(at);
        v[0] = load_as_float(&u.x, 0, type); v[1] = load_as_float(&u.y, 0, type);
        v[2] = load_as_float(&u.z, 0, type); v[3] = load_as_float(&u.w, 0, type);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = j < valid ? load_as_float(p, i + j, type) : 0.f;
    }
}
__device__ __forceinline__ void store4(void *p, int64_t i, int type, int valid, const float (&v)[4]) {
    char *at = reinterpret_cast<char *>(p) + i * (type == kFloat32 ? 4 : 2);
    if (valid == 4 && type == kFloat32 && (reinterpret_cast<uintptr_t>(at) & 15) == 0) {
        *reinterpret_cast<float4 *>(at) = make_float4(v[0], v[1], v[2], v[3]);
    } else if (valid == 4 && type != kFloat32 && (reinterpret_cast<uintptr_t>(at) & 7) == 0) {
        *reinterpret_cast<ushort4 *>(at) = make_ushort4(to_16bit(v[0], type), to_16bit(v[1], type), to_16bit(v[2], type), to_16bit(v[3], type));
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < valid) {
                if (type == kFloat32) reinterpret_cast<float *>(p)[i + j] = v[j];
                else reinterpret_cast<uint16_t *>(p)[i + j] = to_16bit(v[j], type);
            }
    }
}

// m + (1 - mu)(g - m), and the update g + nesterov (m - g).
__device__ __forceinline__ float new_momentum(float m, float g, float keep) { return __fmaf_rn(keep, g - m, m); }
__device__ __forceinline__ float update_of(float m, float g, float nesterov) { return nesterov == 1.f ? m : __fmaf_rn(nesterov, m - g, g); }
#endif  // __CUDACC__

}  // namespace dl
