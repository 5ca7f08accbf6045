// Elements of user tensors in float32, bfloat16 or float16, read and written as float32.
#pragma once
#include "clava_hip.h"
#include "common.h"

namespace elem {

typedef float f32x4 __attribute__((ext_vector_type(4)));
// vectors at any element's address: rows of user tensors start wherever their stride puts them
typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short u16x8_u __attribute__((ext_vector_type(8), aligned(2)));

__device__ __forceinline__ float from_bf16(unsigned short h) { return __uint_as_float((unsigned)h << 16); }
__device__ __forceinline__ float from_f16(unsigned short h) { return (float)__builtin_bit_cast(_Float16, h); }
__device__ __forceinline__ unsigned short to_bf16(float v) { return __builtin_bit_cast(unsigned short, (__bf16)v); }
__device__ __forceinline__ unsigned short to_f16(float v) { return __builtin_bit_cast(unsigned short, (_Float16)v); }

template <int DT> __device__ __forceinline__ float load1(const void* p, size_t i) {
    if (DT == CLAVA_DT_F32) return static_cast<const float*>(p)[i];
    const unsigned short h = static_cast<const unsigned short*>(p)[i];
    return DT == CLAVA_DT_BF16 ? from_bf16(h) : from_f16(h);
}
template <int DT> __device__ __forceinline__ void store1(void* p, size_t i, float v) {
    if (DT == CLAVA_DT_F32) static_cast<float*>(p)[i] = v;
    else static_cast<unsigned short*>(p)[i] = DT == CLAVA_DT_BF16 ? to_bf16(v) : to_f16(v);
}
// n <= 8 values from element i on; the rest are zero
template <int DT> __device__ __forceinline__ void load8(const void* p, size_t i, int n, float* v) {
    if (n >= 8) {
        if (DT == CLAVA_DT_F32) {
            const f32x4_u* q = reinterpret_cast<const f32x4_u*>(static_cast<const float*>(p) + i);
            const f32x4_u a = q[0], b = q[1];
#pragma unroll
            for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
        } else {
            const u16x8_u h = *reinterpret_cast<const u16x8_u*>(static_cast<const unsigned short*>(p) + i);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = DT == CLAVA_DT_BF16 ? from_bf16(h[j]) : from_f16(h[j]);
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? load1<DT>(p, i + j) : 0.f;
}
template <int DT> __device__ __forceinline__ void store8(void* p, size_t i, int n, const float* v) {
    if (n >= 8) {
        if (DT == CLAVA_DT_F32) {
            f32x4_u* q = reinterpret_cast<f32x4_u*>(static_cast<float*>(p) + i);
            q[0] = f32x4_u{v[0], v[1], v[2], v[3]};
            q[1] = f32x4_u{v[4], v[5], v[6], v[7]};
        } else {
            u16x8_u h;
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] = DT == CLAVA_DT_BF16 ? to_bf16(v[j]) : to_f16(v[j]);
            *reinterpret_cast<u16x8_u*>(static_cast<unsigned short*>(p) + i) = h;
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (j < n) store1<DT>(p, i + j, v[j]);
}

}  // namespace elem
