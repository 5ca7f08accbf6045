// Dense layer over microscaled 4-bit matrices: y[m][n] = act( sum over blocks of 2^(ex + ew) * (sum of 32 products of codes)
// + bias[n] ).  v_mfma_scale_f32_16x16x128 takes both scales with the codes and accumulates in float32.  W is the instruction's
// first operand, so that a lane ends up with neighbouring columns of one row of y.
#include <cstdlib>

#include "clava_hip.h"
#include "mx4.h"

namespace {
using namespace mx4;

struct Mx4Args {
    const char* xq; const unsigned char* xs;      // [M, 64 * ks] codes, [M, 4 * ks] scales
    const char* wq; const unsigned char* ws;      // [N, ...]
    const float* bias;
    int act;
    void* y; long long ldy;                       // float outputs
    unsigned* yq; unsigned char* ys; int yks;     // or 4-bit ones, yks = steps(N)
    int M, N, ks;
};

// Eight values; NaN stays NaN
__device__ __forceinline__ void activate8(float* v, int act) {
    if (act == CLAVA_ACT_NONE) return;
    if (act == CLAVA_ACT_SILU) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = v[j] / (1.f + expf(-v[j]));
        return;
    }
    const bool relu = act == CLAVA_ACT_RELU;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float low = relu ? 0.f : 0.01f * v[j];
        v[j] = v[j] <= 0.f ? low : v[j];
    }
}

// Row of W behind row `r` of the first (odd = 0) or second tile of a pair: a lane's accumulators of the two tiles are then
// eight neighbouring columns of y.
__device__ __forceinline__ int pair_row(int r, int odd) { return 8 * (r >> 2) + 4 * odd + (r & 3); }

constexpr int OUT_MX4 = CLAVA_DT_MX4;
__device__ __forceinline__ void bias8(const Mx4Args& g, int n0, float* b) {
    if (g.bias) load8<CLAVA_DT_F32>(g.bias, (size_t)n0, g.N - n0, b);
    else
#pragma unroll
        for (int j = 0; j < 8; ++j) b[j] = 0.f;
}
// A lane's eight columns n0 .. n0+7 of row m (n0 a multiple of 8; lanes l, l^16, l^32, l^48 hold one block of 32 columns):
// every lane of the wave calls this, also those outside of y.
template <int OUT> __device__ __forceinline__ void finish(const Mx4Args& g, int m, int n0, const float* b, float* v) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += b[j];
    activate8(v, g.act);
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
    float bias[8];
    bias8(g, n0 + 8 * q, bias);
    finish<OUT>(g, m0 + r, n0 + 8 * q, bias, v);
}


// ------------------------------------------------------------------------------------------------------- many rows: tiles
__device__ __forceinline__ void dma16(const void* src, char* dst) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src, (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}
__device__ __forceinline__ void dma4(const void* src, char* dst) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src, (__attribute__((address_space(3))) void*)dst, 4, 0, 0);
}

// BN columns x BM rows of y a workgroup of WN x WM wavefronts.  A stage is 256 columns of K: 128 bytes of codes a row (its
// 16-byte chunks exchanged by row bits 1..3, so that the 16 rows of a fragment read hit different banks), then 8 bytes of
// scales a row.  Two stages: the next one is copied straight to LDS while this one is multiplied.
template <int BN, int BM, int WN, int WM, int OUT> __global__ void __launch_bounds__(WN * WM * 64) mx4_tile_kernel(Mx4Args g, int tiles_n, int tiles) {
    constexpr int R = BN + BM, NW = WN * WM, Q = R / 8 / NW, QS = R / 32 / NW > 0 ? R / 32 / NW : 1, STAGE = R * 136;
    constexpr int TN = BN / WN / 16, TM = BM / WM / 16;
    static_assert(R % (8 * NW) == 0 && TN % 2 == 0 && (R / 32) % NW == 0, "tile");
    extern __shared__ __align__(16) char smem[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wn = wave / WM, wm = wave % WM, r = lane & 15, q = lane >> 4;

    // workgroups go round robin over the 8 XCDs: each takes a run of tiles, for its L2
    const int xcd = (int)blockIdx.x & 7, per = tiles >> 3, rem = tiles & 7;
    const int tile = (xcd < rem ? xcd * (per + 1) : rem * (per + 1) + (xcd - rem) * per) + ((int)blockIdx.x >> 3);
    const int m0 = tile / tiles_n * BM, n0 = tile % tiles_n * BN;

    // LDS row `row` of W holds the column of y that puts a lane's accumulators of two neighbouring tiles side by side
    auto source_row = [&](int row) {
        if (row >= BN) return (size_t)min(m0 + row - BN, g.M - 1);
        return (size_t)min(n0 + (row & ~31) + pair_row(row & 15, row >> 4 & 1), g.N - 1);
    };
    const char* src[Q];
    int half[Q];
#pragma unroll
    for (int j = 0; j < Q; ++j) {
        const int row = (wave + j * NW) * 8 + (lane >> 3), chunk = (lane & 7) ^ (row >> 1 & 7);
        src[j] = (row < BN ? g.wq : g.xq) + source_row(row) * g.ks * 64 + (chunk & 3) * 16;
        half[j] = chunk >> 2;
    }
    const unsigned char* ssrc[QS];
#pragma unroll
    for (int j = 0; j < QS; ++j) {
        const int row = (wave + j * NW) * 32 + (lane >> 1);
        ssrc[j] = (row < BN ? g.ws : g.xs) + source_row(row) * g.ks * 4;
    }
    const int stages = (g.ks + 1) >> 1;
    auto copy = [&](int s, char* to) {
        // an odd number of steps: the second half of the last stage is a copy of the first, and not multiplied
        const bool whole = 2 * s + 1 < g.ks;
#pragma unroll
        for (int j = 0; j < Q; ++j) dma16(src[j] + (2 * s + (whole ? half[j] : 0)) * 64, to + (wave + j * NW) * 1024);
#pragma unroll
        for (int j = 0; j < QS; ++j)
            dma4(ssrc[j] + (2 * s + (whole ? lane & 1 : 0)) * 4, to + R * 128 + (wave + j * NW) * 256);
    };

    const int frag = r * 128, swz = r >> 1 & 7;
    const int wrow = wn * TN * 16, xrow = BN + wm * TM * 16;
    f32x4 acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    auto step = [&](const char* at, int ks) {
        const int off = frag + (((ks * 4 + q) ^ swz) << 4);
        const char* sc = at + R * 128 + r * 8 + ks * 4;
        i32x8 X[TM];
        int sx[TM];
#pragma unroll
        for (int j = 0; j < TM; ++j) {
            const i32x4 v = *reinterpret_cast<const i32x4*>(at + (xrow + j * 16) * 128 + off);
            X[j] = i32x8{v[0], v[1], v[2], v[3], 0, 0, 0, 0};
            sx[j] = (int)(*reinterpret_cast<const unsigned*>(sc + (xrow + j * 16) * 8) >> (8 * q));
        }
#pragma unroll
        for (int i = 0; i < TN; ++i) {
            const i32x4 v = *reinterpret_cast<const i32x4*>(at + (wrow + i * 16) * 128 + off);
            const i32x8 W = {v[0], v[1], v[2], v[3], 0, 0, 0, 0};
            const int sw = (int)(*reinterpret_cast<const unsigned*>(sc + (wrow + i * 16) * 8) >> (8 * q));
#pragma unroll
            for (int j = 0; j < TM; ++j) acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(W, X[j], acc[i][j], 4, 4, 0, sw, 0, sx[j]);
        }
    };
    copy(0, smem);
    int cur = 0;
    for (int s = 0; s < stages; ++s) {
        __syncthreads();          // stage s has landed, and nobody reads the other one any more
        if (s + 1 < stages) copy(s + 1, smem + (STAGE - cur));
        step(smem + cur, 0);
        if (2 * s + 1 < g.ks) step(smem + cur, 1);
        cur = STAGE - cur;
    }
#pragma unroll
    for (int i = 0; i < TN; i += 2) {
        const int n = n0 + (wn * TN + i) * 16 + 8 * q;
        float bias[8];
        bias8(g, n, bias);
#pragma unroll
        for (int j = 0; j < TM; ++j) {
            float v[8] = {acc[i][j][0],     acc[i][j][1],     acc[i][j][2],     acc[i][j][3],
                          acc[i + 1][j][0], acc[i + 1][j][1], acc[i + 1][j][2], acc[i + 1][j][3]};
            finish<OUT>(g, m0 + (wm * TM + j) * 16 + r, n, bias, v);
        }
    }
}

template <int BN, int BM, int WN, int WM, int OUT> int launch_tile(const Mx4Args& g, int n_cols, hipStream_t st) {
    constexpr int LDS = (BN + BM) * 136 * 2;
    static bool set[64] = {};     // by device (threads that race set the same value twice)
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) dev = 0;
    if (!set[dev]) {
        if (hipFuncSetAttribute((const void*)mx4_tile_kernel<BN, BM, WN, WM, OUT>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess) {
            clava_set_error("linear_mx4: %d bytes of LDS refused", LDS);
            return CLAVA_ERR_LAUNCH;
        }
        set[dev] = true;
    }
    const int tiles_n = (n_cols + BN - 1) / BN;
    const long long tiles = (long long)((g.M + BM - 1) / BM) * tiles_n;
    if (tiles > 0x7fffffffLL) {
        clava_set_error("linear_mx4: %d x %d outputs are more than one launch takes", g.M, g.N);
        return CLAVA_ERR_LIMIT;
    }
    mx4_tile_kernel<BN, BM, WN, WM, OUT><<<dim3((unsigned)tiles), WN * WM * 64, LDS, st>>>(g, tiles_n, (int)tiles);
    return CLAVA_OK;
}

template <int OUT> int launch_linear(const Mx4Args& g, hipStream_t st) {
    // a 4-bit result also has the zero codes behind its last column written: its columns go to the whole step
    const int n_cols = OUT == OUT_MX4 ? g.yks * KSTEP : g.N;
    const int tiles_n = (n_cols + 31) / 32;
    static const char* force = getenv("CLAVA_MX4_TILE");
    const int f = force ? atoi(force) : 0;
    if (f == 1 || (f == 0 && g.M > 64)) {
        if (f == 0 && (long long)((g.M + 255) / 256) * ((n_cols + 255) / 256) >= 256) return launch_tile<256, 256, 2, 4, OUT>(g, n_cols, st);
        return launch_tile<128, 128, 2, 2, OUT>(g, n_cols, st);
    }
    if (f == 2) return launch_tile<256, 256, 2, 4, OUT>(g, n_cols, st);
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

long long clava_linear_mx4_workspace_bytes(int M, int K, int x_dtype) {
    return M > 0 && K > 0 && x_dtype != CLAVA_DT_MX4 ? (long long)M * steps(K) * 68 : 0;
}

int clava_linear_mx4(const void* x, int x_dtype, long long ldx, const void* x_scales, const void* w_codes, const void* w_scales,
                     const float* bias, int act, void* y, int y_dtype, long long ldy, void* y_scales, int M, int N, int K,
                     void* workspace, void* stream) {
    CLAVA_CHECK_ARG(M >= 0 && N > 0 && K > 0, "linear_mx4: M %d, N %d, K %d", M, N, K);
    CLAVA_CHECK_ARG(act >= CLAVA_ACT_NONE && act <= CLAVA_ACT_SILU, "linear_mx4: activation %d", act);
    CLAVA_CHECK_ARG(x_dtype >= 0 && x_dtype <= CLAVA_DT_MX4 && y_dtype >= 0 && y_dtype <= CLAVA_DT_MX4, "linear_mx4: dtypes %d, %d", x_dtype, y_dtype);
    if (M == 0) return CLAVA_OK;
    const bool x4 = x_dtype == CLAVA_DT_MX4, y4 = y_dtype == CLAVA_DT_MX4;
    CLAVA_CHECK_ARG(x && w_codes && w_scales && y && (!y4 || y_scales) && (x4 ? x_scales : workspace), "linear_mx4: null pointer");
    CLAVA_CHECK_ARG(y4 || ldy >= N || M == 1, "linear_mx4: leading dimension %lld below %d columns", ldy, N);
    CLAVA_CHECK_ARG((((uintptr_t)(x4 ? x : workspace) | (uintptr_t)w_codes) & 15) == 0, "linear_mx4: codes and workspace start at 16 bytes");
    CLAVA_CHECK_ARG(N <= 0x7fffff00 && K <= 0x7fffff00 && M <= 0x7fffff00, "linear_mx4: M %d, N %d, K %d", M, N, K);
    const hipStream_t st = (hipStream_t)stream;
    Mx4Args g;
    g.ks = steps(K);
    g.xq = (const char*)x; g.xs = (const unsigned char*)x_scales;
    if (!x4) {
        g.xq = (const char*)workspace;
        g.xs = (const unsigned char*)workspace + (size_t)M * g.ks * 64;
        const int rc = clava_mx4_pack(x, x_dtype, ldx, M, K, (void*)g.xq, (void*)g.xs, stream);
        if (rc) return rc;
    }
    g.wq = (const char*)w_codes; g.ws = (const unsigned char*)w_scales;
    g.bias = bias; g.act = act;
    g.y = y; g.ldy = ldy;
    g.yq = (unsigned*)y; g.ys = (unsigned char*)y_scales; g.yks = steps(N);
    g.M = M; g.N = N;
    ProfScope prof(PROF_MX4, 2.0 * M * N * K, ((double)M * K + (double)N * K) * 17.0 / 32 + (double)M * N * (y4 ? 17.0 / 32 : y_dtype == 0 ? 4 : 2), st);
    const int rc = y4 ? launch_linear<OUT_MX4>(g, st)
                      : y_dtype == CLAVA_DT_F32 ? launch_linear<CLAVA_DT_F32>(g, st)
                      : y_dtype == CLAVA_DT_BF16 ? launch_linear<CLAVA_DT_BF16>(g, st) : launch_linear<CLAVA_DT_F16>(g, st);
    if (rc) return rc;
    CLAVA_CHECK_LAUNCH("linear_mx4");
    return CLAVA_OK;
}

}  // extern "C"
