// Microscaled 4-bit matrices (OCP MX, E2M1 elements over blocks of 32 columns of a row; layout in include/clava_hip.h).
#pragma once
#include "elem.h"

namespace mx4 {
using namespace elem;

constexpr int BLOCK = 32;       // columns that share a scale
constexpr int KSTEP = 128;      // columns of one matrix instruction; rows are padded to whole steps

__host__ __device__ __forceinline__ int steps(int cols) { return (int)(((long long)cols + KSTEP - 1) / KSTEP); }

// Exponent of a block's scale from the bits of its largest magnitude: floor(log2(max)) - 2, so that the largest element lies
// in [4, 8) and saturates at 6 only beyond it; -127 (the smallest scale) for zero and where float32 ends.  Returned with the
// bias of the scale byte; 255 when the block holds an infinity or a NaN.
__device__ __forceinline__ int scale_byte(unsigned max_bits) {
    const unsigned e = max_bits >> 23;              // the sign is gone
    if (e == 255) return 255;
    // a subnormal maximum is below 2^-126: its exponent - 2 is clamped like every other one under -127
    return e > 2 ? (int)e - 2 : 0;
}

// Eight float32 values over 2^(byte - 127) to eight E2M1 codes, nearest with ties to even, saturating; the multiplication by
// the inverse power is exact (2^127 at most; what falls below float32's range rounds to zero either way).
__device__ __forceinline__ unsigned pack8(const float* v, int byte) {
    if (byte == 255) return 0u;
    const float inv = __uint_as_float((unsigned)(254 - byte) << 23);      // byte <= 252 for a finite maximum
    unsigned q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0] * inv, v[1] * inv, 1.0f, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2] * inv, v[3] * inv, 1.0f, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4] * inv, v[5] * inv, 1.0f, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6] * inv, v[7] * inv, 1.0f, 3);
    return q;
}

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4_u4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u32x4_u2 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// Largest magnitude (as bits) of the 8 values of this lane and of the three lanes that hold the rest of its block, which
// differ from it in the lane bits of `A` and `B`.
template <int A, int B> __device__ __forceinline__ unsigned block_max(const float* v) {
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);      // bits order magnitudes, NaN above all
    m = max(m, (unsigned)__shfl_xor((int)m, A, 64));
    return max(m, (unsigned)__shfl_xor((int)m, B, 64));
}

}  // namespace mx4
