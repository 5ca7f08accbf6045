// Microscaled 4-bit matrices: quantisation, reading back, and the dense layer over them.
//
// pack: block of 32 columns -> e = floor(log2(max|v|)) - 2, code = nearest E2M1 of v / 2^e.  Eight columns a lane, so that a
// block is four neighbouring lanes, its maximum two exchanges and a lane's codes one 4-byte store.
// unpack: value(code) * 2^e.  Both move each byte once.
//
// linear: y[m][n] = act( sum over blocks of 2^(ex + ew) * (sum of 32 products of codes) + bias[n] ).  v_mfma_scale_f32_16x16x128
// takes both scales with the codes and accumulates in float32.  W is the instruction's first operand, so that a lane ends up
// with neighbouring columns of one row of y.
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

// E2M1 codes of one lane (8 of them) times 2^(byte - 127); 255 reads as NaN
__device__ __forceinline__ void unpack8(unsigned q, int byte, float* v) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const unsigned c = (q >> (4 * j)) & 15u, m = c & 7u;
        // 0, 1/2, then 1.m with exponent bias 1
        const float a = m < 2 ? 0.5f * (float)m : __uint_as_float(((m >> 1) + 126u) << 23 | (m & 1u) << 22);
        const float s = byte == 255 ? __uint_as_float(0x7fc00000u) : ldexpf(a, byte - 127);
        v[j] = c & 8u ? -s : s;
    }
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

// ---------------------------------------------------------------------------------------------------------------- linear
struct Mx4Args {
    const char* xq; const unsigned char* xs;      // [M, 64 * ks] codes, [M, 4 * ks] scales
    const char* wq; const unsigned char* ws;      // [N, ...]
    const float* bias;
    int act;
    void* y; long long ldy;                       // float outputs
    unsigned* yq; unsigned char* ys; int yks;     // or 4-bit ones, yks = steps(N)
    int M, N, ks;
};

__device__ __forceinline__ float activate(float v, int act) {
    if (act == CLAVA_ACT_RELU) return v > 0.f ? v : (v != v ? v : 0.f);
    if (act == CLAVA_ACT_LEAKY) return v > 0.f ? v : 0.01f * v;
    if (act == CLAVA_ACT_SILU) return v / (1.f + expf(-v));
    return v;
}

// Row of W behind row `r` of the first (odd = 0) or second tile of a pair: a lane's accumulators of the two tiles are then
// eight neighbouring columns of y.
__device__ __forceinline__ int pair_row(int r, int odd) { return 8 * (r >> 2) + 4 * odd + (r & 3); }

constexpr int OUT_MX4 = 3;
// A lane's eight columns n0 .. n0+7 of row m (n0 a multiple of 8; lanes l, l^16, l^32, l^48 hold one block of 32 columns):
// every lane of the wave calls this, also those outside of y.
template <int OUT> __device__ __forceinline__ void finish(const Mx4Args& g, int m, int n0, float* v) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float b = (g.bias && n0 + j < g.N) ? g.bias[n0 + j] : 0.f;
        v[j] = activate(v[j] + b, g.act);
    }
    if (OUT != OUT_MX4) {
        if (m < g.M && n0 < g.N) store8<OUT == OUT_MX4 ? 0 : OUT>(g.y, (size_t)m * g.ldy + n0, g.N - n0, v);
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (n0 + j >= g.N) v[j] = 0.f;
    const int byte = scale_byte(block_max<16, 32>(v));
    if (m < g.M && n0 < g.yks * KSTEP) {
        g.yq[((size_t)m * g.yks * KSTEP + n0) >> 3] = pack8(v, byte);
        if ((n0 & 31) == 0) g.ys[((size_t)m * g.yks * KSTEP + n0) >> 5] = (unsigned char)byte;
    }
}

// 16 rows x 32 columns a workgroup, its waves take every fourth step of K and add up through LDS.
template <int OUT> __global__ void __launch_bounds__(256) mx4_linear_kernel(Mx4Args g, int tiles_n) {
    __shared__ f32x4 part[3][2][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
    const int m0 = (int)(blockIdx.x / (unsigned)tiles_n) * 16, n0 = (int)(blockIdx.x % (unsigned)tiles_n) * 32;
    const size_t m = min(m0 + r, g.M - 1);
    const size_t na = min(n0 + pair_row(r, 0), g.N - 1), nb = min(n0 + pair_row(r, 1), g.N - 1);
    const char* x = g.xq + m * g.ks * 64 + q * 16;
    const char* wa = g.wq + na * g.ks * 64 + q * 16;
    const char* wb = g.wq + nb * g.ks * 64 + q * 16;
    const unsigned char *xs = g.xs + m * g.ks * 4 + q, *was = g.ws + na * g.ks * 4 + q, *wbs = g.ws + nb * g.ks * 4 + q;
    f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
    for (int k = wave; k < g.ks; k += 4) {
        const i32x4 xv = *reinterpret_cast<const i32x4*>(x + (size_t)k * 64);
        const i32x4 av = *reinterpret_cast<const i32x4*>(wa + (size_t)k * 64), bv = *reinterpret_cast<const i32x4*>(wb + (size_t)k * 64);
        const int sx = xs[k * 4], sa = was[k * 4], sb = wbs[k * 4];
        const i32x8 X = {xv[0], xv[1], xv[2], xv[3], 0, 0, 0, 0}, A = {av[0], av[1], av[2], av[3], 0, 0, 0, 0},
                    B = {bv[0], bv[1], bv[2], bv[3], 0, 0, 0, 0};
        a = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, X, a, 4, 4, 0, sa, 0, sx);
        b = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(B, X, b, 4, 4, 0, sb, 0, sx);
    }
    if (wave) { part[wave - 1][0][lane] = a; part[wave - 1][1][lane] = b; }
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int p = 0; p < 3; ++p) { a += part[p][0][lane]; b += part[p][1][lane]; }
    float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    finish<OUT>(g, m0 + r, n0 + 8 * q, v);
}

template <int OUT> int launch_linear(const Mx4Args& g, hipStream_t st) {
    // a 4-bit result also has the zero codes behind its last column written: its columns go to the whole step
    const int n_cols = OUT == OUT_MX4 ? g.yks * KSTEP : g.N;
    const int tiles_n = (n_cols + 31) / 32;
    const long long wgs = (long long)((g.M + 15) / 16) * tiles_n;
    if (wgs > 0x7fffffffLL) {
        clava_set_error("linear_mx4: %d x %d outputs are more than one launch takes", g.M, g.N);
        return CLAVA_ERR_LIMIT;
    }
    mx4_linear_kernel<OUT><<<dim3((unsigned)wgs), 256, 0, st>>>(g, tiles_n);
    return CLAVA_OK;
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

int clava_linear_mx4(const void* x_codes, const void* x_scales, const void* w_codes, const void* w_scales, const float* bias, int act,
                     void* y, int y_dtype, long long ldy, void* y_codes, void* y_scales, int M, int N, int K, void* stream) {
    CLAVA_CHECK_ARG(M >= 0 && N > 0 && K > 0, "linear_mx4: M %d, N %d, K %d", M, N, K);
    CLAVA_CHECK_ARG(act >= CLAVA_ACT_NONE && act <= CLAVA_ACT_SILU, "linear_mx4: activation %d", act);
    CLAVA_CHECK_ARG((y != nullptr) != (y_codes != nullptr) || M == 0, "linear_mx4: one of y and y_codes");
    if (M == 0) return CLAVA_OK;
    CLAVA_CHECK_ARG(x_codes && x_scales && w_codes && w_scales && (y || y_scales), "linear_mx4: null pointer");
    CLAVA_CHECK_ARG(!y || (y_dtype >= 0 && y_dtype <= CLAVA_DT_F16), "linear_mx4: dtype %d", y_dtype);
    CLAVA_CHECK_ARG(!y || ldy >= N || M == 1, "linear_mx4: leading dimension %lld below %d columns", ldy, N);
    CLAVA_CHECK_ARG(((uintptr_t)x_codes & 15) == 0 && ((uintptr_t)w_codes & 15) == 0, "linear_mx4: codes must start at 16 bytes");
    CLAVA_CHECK_ARG(N <= 0x7fffff00 && K <= 0x7fffff00 && M <= 0x7fffff00, "linear_mx4: M %d, N %d, K %d", M, N, K);
    const hipStream_t st = (hipStream_t)stream;
    Mx4Args g;
    g.xq = (const char*)x_codes; g.xs = (const unsigned char*)x_scales;
    g.wq = (const char*)w_codes; g.ws = (const unsigned char*)w_scales;
    g.bias = bias; g.act = act;
    g.y = y; g.ldy = ldy;
    g.yq = (unsigned*)y_codes; g.ys = (unsigned char*)y_scales; g.yks = steps(N);
    g.M = M; g.N = N; g.ks = steps(K);
    ProfScope prof(PROF_MX4, 2.0 * M * N * K, ((double)M * K + (double)N * K) * 17.0 / 32 + (double)M * N * (!y ? 17.0 / 32 : y_dtype == 0 ? 4 : 2), st);
    const int rc = !y ? launch_linear<OUT_MX4>(g, st)
                      : y_dtype == CLAVA_DT_F32 ? launch_linear<CLAVA_DT_F32>(g, st)
                      : y_dtype == CLAVA_DT_BF16 ? launch_linear<CLAVA_DT_BF16>(g, st) : launch_linear<CLAVA_DT_F16>(g, st);
    if (rc) return rc;
    CLAVA_CHECK_LAUNCH("linear_mx4");
    return CLAVA_OK;
}

}  // extern "C"
