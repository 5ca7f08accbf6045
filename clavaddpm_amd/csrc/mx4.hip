// Microscaled 4-bit matrices: quantisation and reading back.
//
// pack: block of 32 columns -> e = floor(log2(max|v|)) - 2, code = nearest E2M1 of v / 2^e.  Eight columns a lane, so that a
// block is four neighbouring lanes, its maximum two exchanges and a lane's codes one 4-byte store.
// unpack: value(code) * 2^e.  Both move each byte once and are bound by that: 20000 x 1999 bfloat16 (101 MB) 22.8 and 17.7 us
// (4.4 and 5.7 TB/s, part of the codes still in the caches), 4096 x 1024 float32 4.5 and 7.0 us.
#include "clava_hip.h"
#include "mx4.h"

namespace {
using namespace mx4;

template <int DT>
__global__ void __launch_bounds__(256) mx4_pack_kernel(const void* __restrict__ src, long long ld, unsigned rows, int cols, unsigned lanes,
                                                       unsigned* __restrict__ codes, unsigned char* __restrict__ scales) {
    // `lanes` = 8-column groups of a padded row; a workgroup's 256 lanes hold whole blocks since `lanes` is a multiple of 16
    const unsigned i = blockIdx.x * 256u + threadIdx.x;
    if (i >= rows * lanes) return;
    const unsigned r = i / lanes, g = i - r * lanes;
    const int c = (int)(g * 8);
    float v[8];
    load8<DT>(src, (size_t)r * ld + c, cols - c, v);
    const int byte = scale_byte(block_max<1, 2>(v));
    codes[i] = pack8(v, byte);
    if ((g & 3) == 0) scales[i >> 2] = (unsigned char)byte;
}

// E2M1 codes of one lane (8 of them) times 2^(byte - 127); 255 reads as NaN.  The conversion takes the scale as a float32, which
// 2^-127 is not as a normal number: half of twice it is.
__device__ __forceinline__ void unpack8(unsigned q, int byte, float* v) {
    const float s = byte == 255 ? __uint_as_float(0x7fc00000u) : byte ? __uint_as_float((unsigned)byte << 23) : 0x1p-126f, half = byte ? 1.f : 0.5f;
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 1),
               c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 3);
    const float u[8] = {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = u[j] * s * half;
}

template <int DT>
__global__ void __launch_bounds__(256) mx4_unpack_kernel(const unsigned* __restrict__ codes, const unsigned char* __restrict__ scales,
                                                         unsigned rows, int cols, unsigned lanes, void* __restrict__ dst, long long ld) {
    const unsigned i = blockIdx.x * 256u + threadIdx.x;
    if (i >= rows * lanes) return;
    const unsigned r = i / lanes, g = i - r * lanes;
    const int c = (int)(g * 8);
    if (c >= cols) return;
    float v[8];
    unpack8(codes[i], scales[i >> 2], v);
    store8<DT>(dst, (size_t)r * ld + c, cols - c, v);
}

}  // namespace

extern "C" {

int clava_mx4_pack(const void* src, int dtype, long long ld, long long rows, int cols, void* codes, void* scales, void* stream) {
    CLAVA_CHECK_ARG(rows >= 0 && cols > 0, "mx4_pack: %lld x %d", rows, cols);
    if (rows == 0) return CLAVA_OK;
    CLAVA_CHECK_ARG(src && codes && scales, "mx4_pack: null pointer");
    CLAVA_CHECK_ARG(dtype >= 0 && dtype <= CLAVA_DT_F16, "mx4_pack: dtype %d", dtype);
    CLAVA_CHECK_ARG(ld >= cols || rows == 1, "mx4_pack: leading dimension %lld below %d columns", ld, cols);
    CLAVA_CHECK_ARG(cols <= 0x7fffff80, "mx4_pack: %d columns", cols);
    const hipStream_t st = (hipStream_t)stream;
    const unsigned lanes = (unsigned)steps(cols) * (KSTEP / 8);
    const int size = dtype == CLAVA_DT_F32 ? 4 : 2;
    const long long per = 0x7fffff00LL / lanes;           // rows of one launch: 32-bit indexes inside it
    for (long long r0 = 0; r0 < rows; r0 += per) {
        const unsigned n = (unsigned)(rows - r0 < per ? rows - r0 : per);
        const void* s = (const char*)src + (size_t)r0 * ld * size;
        unsigned* c = (unsigned*)codes + (size_t)r0 * lanes;
        unsigned char* e = (unsigned char*)scales + (size_t)r0 * (lanes / 4);
        const dim3 grid((n * lanes + 255) / 256);
        ProfScope prof(PROF_MX4, 0, (double)n * cols * (size + 17.0 / 32), st);
        if (dtype == CLAVA_DT_F32) mx4_pack_kernel<CLAVA_DT_F32><<<grid, 256, 0, st>>>(s, ld, n, cols, lanes, c, e);
        else if (dtype == CLAVA_DT_BF16) mx4_pack_kernel<CLAVA_DT_BF16><<<grid, 256, 0, st>>>(s, ld, n, cols, lanes, c, e);
        else mx4_pack_kernel<CLAVA_DT_F16><<<grid, 256, 0, st>>>(s, ld, n, cols, lanes, c, e);
        CLAVA_CHECK_LAUNCH("mx4_pack");
    }
    return CLAVA_OK;
}

int clava_mx4_unpack(const void* codes, const void* scales, long long rows, int cols, void* dst, int dtype, long long ld, void* stream) {
    CLAVA_CHECK_ARG(rows >= 0 && cols > 0, "mx4_unpack: %lld x %d", rows, cols);
    if (rows == 0) return CLAVA_OK;
    CLAVA_CHECK_ARG(dst && codes && scales, "mx4_unpack: null pointer");
    CLAVA_CHECK_ARG(dtype >= 0 && dtype <= CLAVA_DT_F16, "mx4_unpack: dtype %d", dtype);
    CLAVA_CHECK_ARG(ld >= cols || rows == 1, "mx4_unpack: leading dimension %lld below %d columns", ld, cols);
    CLAVA_CHECK_ARG(cols <= 0x7fffff80, "mx4_unpack: %d columns", cols);
    const hipStream_t st = (hipStream_t)stream;
    const unsigned lanes = (unsigned)steps(cols) * (KSTEP / 8);
    const int size = dtype == CLAVA_DT_F32 ? 4 : 2;
    const long long per = 0x7fffff00LL / lanes;
    for (long long r0 = 0; r0 < rows; r0 += per) {
        const unsigned n = (unsigned)(rows - r0 < per ? rows - r0 : per);
        const unsigned* c = (const unsigned*)codes + (size_t)r0 * lanes;
        const unsigned char* e = (const unsigned char*)scales + (size_t)r0 * (lanes / 4);
        void* d = (char*)dst + (size_t)r0 * ld * size;
        const dim3 grid((n * lanes + 255) / 256);
        ProfScope prof(PROF_MX4, 0, (double)n * cols * (size + 17.0 / 32), st);
        if (dtype == CLAVA_DT_F32) mx4_unpack_kernel<CLAVA_DT_F32><<<grid, 256, 0, st>>>(c, e, n, cols, lanes, d, ld);
        else if (dtype == CLAVA_DT_BF16) mx4_unpack_kernel<CLAVA_DT_BF16><<<grid, 256, 0, st>>>(c, e, n, cols, lanes, d, ld);
        else mx4_unpack_kernel<CLAVA_DT_F16><<<grid, 256, 0, st>>>(c, e, n, cols, lanes, d, ld);
        CLAVA_CHECK_LAUNCH("mx4_unpack");
    }
    return CLAVA_OK;
}

}  // extern "C"
