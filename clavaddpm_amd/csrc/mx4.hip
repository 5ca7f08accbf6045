// Microscaled 4-bit matrices: quantisation and reading back.
//
// pack: block of 32 columns -> e = floor(log2(max|v|)) - 2, code = nearest E2M1 of v / 2^e.  Eight columns a lane, so that a
// block is four neighbouring lanes, its maximum two exchanges and a lane's codes one 4-byte store.
// unpack: value(code) * 2^e.  Both move each byte once and are bound by that: 20000 x 2000 bfloat16 (101 MB) from memory 25.2 and
// 21.5 us, 4.0 and 4.7 TB/s; 1999 columns, whose rows start at any 2 bytes, 31 and 25; 4096 x 1024 float32 3.8 and 6.9 us (why
// the second takes longer for the same bytes has not been looked into: its stores fill half a line at a time).
#include "clava_hip.h"
#include "mx4.h"

namespace {
using namespace mx4;

// load8 of a 16-bit type from rows that do not start at 16 bytes: with 16-byte loads at any address 20000 x 1999 bfloat16 took
// 33 us, this way 28 (from memory, in one run).  A lane loads the aligned 16 bytes that hold its first column, takes the following ones from the next lane
// (`next`: it is the same row's) and shifts them together.  Nothing outside lo .. hi is read: lanes that would, load at any
// address.  All lanes of a row in the wavefront come here together.
template <int DT> __device__ __forceinline__ void load8_shifted(const void* src, size_t at, const char* lo, const char* hi, int n, bool next, float* v) {
    constexpr int WAVE_SHL1 = 0x130;
    const char* const p = static_cast<const char*>(src) + at * 2;
    const unsigned off = (unsigned)((uintptr_t)p & 15);
    const char* const a = p - off;
    u32x4 A = {0, 0, 0, 0}, B;
    if (a >= lo && a + 16 <= hi) A = *reinterpret_cast<const u32x4*>(a);
#pragma unroll
    for (int k = 0; k < 4; ++k) B[k] = (unsigned)__builtin_amdgcn_update_dpp(0, (int)A[k], WAVE_SHL1, 0xf, 0xf, true);
    if (a < lo || a + 32 > hi) {
        load8<DT>(src, at, n, v);
        return;
    }
    if (!next) B = *reinterpret_cast<const u32x4*>(a + 16);
    unsigned d[8] = {A[0], A[1], A[2], A[3], B[0], B[1], B[2], B[3]};
    const unsigned by2 = off & 8 ? ~0u : 0u, by1 = off & 4 ? ~0u : 0u;
#pragma unroll
    for (int k = 0; k < 6; ++k) d[k] = (d[k + 2] & by2) | (d[k] & ~by2);
#pragma unroll
    for (int k = 0; k < 5; ++k) d[k] = (d[k + 1] & by1) | (d[k] & ~by1);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const unsigned two = __builtin_amdgcn_alignbit(d[k + 1], d[k], (off & 2) * 8);
        const unsigned short h[2] = {(unsigned short)two, (unsigned short)(two >> 16)};
#pragma unroll
        for (int j = 0; j < 2; ++j) v[2 * k + j] = 2 * k + j < n ? (DT == CLAVA_DT_BF16 ? from_bf16(h[j]) : from_f16(h[j])) : 0.f;
    }
}

template <int DT, bool SHIFTED>
__global__ void __launch_bounds__(256) mx4_pack_kernel(const void* __restrict__ src, long long ld, unsigned rows, int cols, unsigned lanes,
                                                       unsigned* __restrict__ codes, unsigned char* __restrict__ scales) {
    // `lanes` = 8-column groups of a padded row; a workgroup's 256 lanes hold whole blocks since `lanes` is a multiple of 16
    const unsigned i = blockIdx.x * 256u + threadIdx.x;
    if (i >= rows * lanes) return;
    const unsigned r = i / lanes, g = i - r * lanes;
    const int c = (int)(g * 8);
    float v[8];
    if (SHIFTED) {
        const char* const lo = static_cast<const char*>(src);
        load8_shifted<DT>(src, (size_t)r * ld + c, lo, lo + ((size_t)(rows - 1) * ld + cols) * 2, cols - c, (threadIdx.x & 63) != 63 && g + 1 < lanes, v);
    } else load8<DT>(src, (size_t)r * ld + c, cols - c, v);
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
    CLAVA_CHECK_ARG(((uintptr_t)codes & 3) == 0, "mx4_pack: codes start at 4 bytes");
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
        const bool shifted = dtype != CLAVA_DT_F32 && (((uintptr_t)s | (n > 1 ? (uintptr_t)ld * 2 : 0)) & 15) != 0;
        auto* const kernel = dtype == CLAVA_DT_F32 ? mx4_pack_kernel<CLAVA_DT_F32, false>
                             : dtype == CLAVA_DT_BF16 ? (shifted ? mx4_pack_kernel<CLAVA_DT_BF16, true> : mx4_pack_kernel<CLAVA_DT_BF16, false>)
                                                      : (shifted ? mx4_pack_kernel<CLAVA_DT_F16, true> : mx4_pack_kernel<CLAVA_DT_F16, false>);
        kernel<<<grid, 256, 0, st>>>(s, ld, n, cols, lanes, c, e);
        CLAVA_CHECK_LAUNCH("mx4_pack");
    }
    return CLAVA_OK;
}

int clava_mx4_unpack(const void* codes, const void* scales, long long rows, int cols, void* dst, int dtype, long long ld, void* stream) {
    CLAVA_CHECK_ARG(rows >= 0 && cols > 0, "mx4_unpack: %lld x %d", rows, cols);
    if (rows == 0) return CLAVA_OK;
    CLAVA_CHECK_ARG(dst && codes && scales, "mx4_unpack: null pointer");
    CLAVA_CHECK_ARG(dtype >= 0 && dtype <= CLAVA_DT_F16, "mx4_unpack: dtype %d", dtype);
    CLAVA_CHECK_ARG(((uintptr_t)codes & 3) == 0, "mx4_unpack: codes start at 4 bytes");
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
