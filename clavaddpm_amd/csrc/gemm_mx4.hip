// Dense layer over microscaled 4-bit matrices: y[m][n] = act( sum over blocks of 2^(ex + ew) * (sum of 32 products of codes)
// + bias[n] ).  v_mfma_scale_f32 (16x16x128, 32x32x64) takes both scales with the codes and accumulates in float32.  W is the instruction's
// first operand, so that a lane ends up with neighbouring columns of one row of y.
#include <type_traits>

#include "clava_hip.h"
#include "mx4.h"

namespace {
using namespace mx4;

struct Mx4Args {
    const char* xq; const unsigned char* xs;      // [M, 64 * ks] codes, [M, 4 * ks] scales; or, of few rows, floats
    int xt, K; long long ldx;                     // xt: CLAVA_DT_*
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
    if (act == CLAVA_ACT_RELU) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = v[j] <= 0.f ? 0.f : v[j];
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = v[j] <= 0.f ? 0.01f * v[j] : v[j];
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
// A lane's C = 8 or 16 columns n0 .. of row m (n0 a multiple of C).  The lanes that hold the rest of a block of 32 columns are
// l^16, l^32, l^48 (C = 8) or l^32 (C = 16); every lane of the wave calls this, also those outside of y.
template <int OUT, int C> __device__ __forceinline__ void finish(const Mx4Args& g, int m, int n0, const float* b, float* v) {
#pragma unroll
    for (int c = 0; c < C; c += 8) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[c + j] += b[c + j];
        activate8(v + c, g.act);
        if (OUT != OUT_MX4 && m < g.M && n0 + c < g.N) store8<OUT == OUT_MX4 ? 0 : OUT>(g.y, (size_t)m * g.ldy + n0 + c, g.N - n0 - c, v + c);
    }
    if (OUT != OUT_MX4) return;
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < C; ++j) {
        if (n0 + j >= g.N) v[j] = 0.f;
        top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
    }
    if (C == 8) top = max(top, (unsigned)__shfl_xor((int)top, 16, 64));
    top = max(top, (unsigned)__shfl_xor((int)top, 32, 64));
    const int byte = scale_byte(top);
    if (m < g.M && n0 < g.yks * KSTEP) {
        const size_t at = (size_t)m * g.yks * KSTEP + n0;
#pragma unroll
        for (int c = 0; c < C; c += 8) g.yq[(at + c) >> 3] = pack8(v + c, byte);
        if ((n0 & 31) == 0) g.ys[at >> 5] = (unsigned char)byte;
    }
}

// ---------------------------------------------------------------------------------------------------------------- few rows
// A lane's 32 columns of a row of floats are one block: its scale and codes without another lane.
template <int DT> __device__ __forceinline__ i32x4 pack32(const void* x, size_t at, int n, int& byte) {
    float v[32];
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < 32; j += 8) {
        load8<DT>(x, at + j, n - j, v + j);
#pragma unroll
        for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(v[j + k]) & 0x7fffffffu);
    }
    byte = scale_byte(top);
    return i32x4{(int)pack8(v, byte), (int)pack8(v + 8, byte), (int)pack8(v + 16, byte), (int)pack8(v + 24, byte)};
}

// 16 rows x 32 columns a workgroup; its NW wavefronts take every NW-th step of K and add up through LDS.  W streams from
// memory once, four steps of it on their way to a wavefront, and x (XT: floats or codes) comes from L2; floats are packed on
// the way, which saves the launch that packs them and its round trip (1 x 1024 x 1024: 5.3 us in two launches).  Bound by the
// latency of that stream: 7 x 4099 x 8001 (17.5 MB) 6.0 us, 2.9 TB/s; 1 x 1024 x 1024 4.5 us.
template <int XT, int NW, int OUT> __global__ void __launch_bounds__(NW * 64) mx4_few_kernel(Mx4Args g, int tiles_n) {
    __shared__ f32x4 part[NW - 1][2][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
    const int m0 = (int)(blockIdx.x / (unsigned)tiles_n) * 16, n0 = (int)(blockIdx.x % (unsigned)tiles_n) * 32;
    const size_t m = min(m0 + r, g.M - 1);
    const size_t na = min(n0 + pair_row(r, 0), g.N - 1), nb = min(n0 + pair_row(r, 1), g.N - 1);
    const char* wa = g.wq + na * g.ks * 64 + q * 16;
    const char* wb = g.wq + nb * g.ks * 64 + q * 16;
    const unsigned char *was = g.ws + na * g.ks * 4 + q, *wbs = g.ws + nb * g.ks * 4 + q;
    f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
    auto steps_from = [&](int k, auto count_t) {
        constexpr int COUNT = decltype(count_t)::value;
        i32x4 A[COUNT], B[COUNT], X[COUNT];
        int sa[COUNT], sb[COUNT], sx[COUNT];
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            const size_t at = (size_t)(k + i * NW);
            A[i] = *reinterpret_cast<const i32x4*>(wa + at * 64);
            B[i] = *reinterpret_cast<const i32x4*>(wb + at * 64);
            sa[i] = was[at * 4];
            sb[i] = wbs[at * 4];
        }
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            const size_t at = (size_t)(k + i * NW);
            if (XT == CLAVA_DT_MX4) {
                X[i] = *reinterpret_cast<const i32x4*>(g.xq + (m * g.ks + at) * 64 + q * 16);
                sx[i] = g.xs[(m * g.ks + at) * 4 + q];
            } else {
                const int c = (k + i * NW) * KSTEP + q * 32;
                X[i] = pack32<XT == CLAVA_DT_MX4 ? 0 : XT>(g.xq, m * (size_t)g.ldx + c, g.K - c, sx[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            const i32x8 x = {X[i][0], X[i][1], X[i][2], X[i][3], 0, 0, 0, 0}, va = {A[i][0], A[i][1], A[i][2], A[i][3], 0, 0, 0, 0},
                        vb = {B[i][0], B[i][1], B[i][2], B[i][3], 0, 0, 0, 0};
            a = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(va, x, a, 4, 4, 0, sa[i], 0, sx[i]);
            b = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(vb, x, b, 4, 4, 0, sb[i], 0, sx[i]);
        }
    };
    int k = wave;
    for (; k + 3 * NW < g.ks; k += 4 * NW) steps_from(k, std::integral_constant<int, 4>{});
    for (; k < g.ks; k += NW) steps_from(k, std::integral_constant<int, 1>{});
    if (wave) { part[wave - 1][0][lane] = a; part[wave - 1][1][lane] = b; }
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int p = 0; p < NW - 1; ++p) { a += part[p][0][lane]; b += part[p][1][lane]; }
    float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    float bias[8];
    bias8(g, n0 + 8 * q, bias);
    finish<OUT, 8>(g, m0 + r, n0 + 8 * q, bias, v);
}

// ------------------------------------------------------------------------------------------------------- many rows: tiles
__device__ __forceinline__ void dma16(const void* src, char* dst) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src, (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}
__device__ __forceinline__ void dma4(const void* src, char* dst) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src, (__attribute__((address_space(3))) void*)dst, 4, 0, 0);
}

// BN columns x BM rows of y a workgroup of WN x WM wavefronts, on v_mfma_scale_f32_32x32x64: one wavefront a SIMD reaches
// 9.0 PFLOP/s with it, and 3.3 with 16x16x128, whose scale load costs as much as its product (registers only, 256 workgroups).
// A stage is 256 columns of K: 128 bytes of codes a row (its 16-byte chunks exchanged by row bits 1..3, so that the rows of a
// fragment read hit different banks), NS of them in a ring.  Scales have a ring of their own.  S16: 16 bytes of them a row, 512
// columns, in one copy (rows of whole 16 bytes: K a multiple of 512); else 4 bytes in each.  A copy of scales touches a cache
// line per row, whatever it takes from it: with 4 bytes the scales took the copies of a 256 x 256 tile from 1.3 to 1.8 us a stage.
// 16384 x 8192 x 8192 to bfloat16: 1.10 million cycles, 48 % of them with the matrix cores busy: 500 us (4.4 PFLOP/s) to 571 by the
// clock that a card holds; bound by the requests that a CU can have in flight (85 % of them hit L2, which is at a third of its
// rate), and 11 us a tile of start and result.  4-bit results of a hidden layer, 20000 x 1024 x 1024: 25 to 28 us (8.1 by its
// operations, 4.7 by its bytes): a tile has four stages, so that start and result count, and packing the result is vector
// instructions, 26 000 cycles of a SIMD in all.
template <int BN, int BM, int WN, int WM, int NS, bool S16, int OUT>
__global__ void __launch_bounds__(WN * WM * 64) mx4_tile_kernel(Mx4Args g, int tiles_n, int tiles) {
    constexpr int R = BN + BM, NW = WN * WM, Q = R / 8 / NW, STAGE = R * 128;
    // copies of scales: of a group (S16: of two stages), of a wave; bytes of a row and of a group, groups in the ring
    constexpr int SU = S16 ? R / 64 : R / 32, QS = (SU + NW - 1) / NW, SROW = S16 ? 16 : 8, SGROUP = R * SROW, SRING = S16 ? NS / 2 + 1 : NS;
    constexpr int WAIT = (NS - 2) * Q + (S16 ? (NS - 2) / 2 : NS - 2) * QS;      // copies behind those of the stage that is next
    constexpr int TN = BN / WN / 32, TM = BM / WM / 32;
    static_assert(R % (8 * NW) == 0 && NW % 2 == 0 && NS % 2 == 0 && TN > 0 && TM > 0, "tile");
    extern __shared__ __align__(16) char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wn = wave / WM, wm = wave % WM, r = lane & 31, h = lane >> 5;

    // workgroups go round robin over the 8 XCDs: each takes a run of tiles, for its L2
    const int xcd = (int)blockIdx.x & 7, per = tiles >> 3, rem = tiles & 7;
    const int tile = (xcd < rem ? xcd * (per + 1) : rem * (per + 1) + (xcd - rem) * per) + ((int)blockIdx.x >> 3);
    // in it, DOWN tiles down before the next column: the 32 tiles that an XCD works on at a time then share 6 panels of X and 5
    // or 6 of W (a row of tiles: 1 and 32; 16384 x 8192 x 8192 to bfloat16, six down 546 us, four 544, eight 573, sixteen 576)
    constexpr int DOWN = 6;
    const int tiles_m = tiles / tiles_n, group = tile / (DOWN * tiles_n), gm = min(DOWN, tiles_m - DOWN * group), in = tile - group * DOWN * tiles_n;
    const int m0 = (DOWN * group + in % gm) * BM, n0 = in / gm * BN;

    // LDS row `row` of W holds the column of y that puts the 16 accumulators of a lane side by side: its half h of a 32 x 32
    // product has rows 8 G + 4 h + t, G, t < 4, and they are to be columns 16 h + 4 G + t.  Sources are a base of the tile (in scalar registers) and 32 bits of a lane's own.
    const int nb = min(n0, g.N - 1);
    const char *wq = g.wq + (size_t)nb * g.ks * 64, *xq = g.xq + (size_t)m0 * g.ks * 64;
    const unsigned char *ws = g.ws + (size_t)nb * g.ks * 4, *xs = g.xs + (size_t)m0 * g.ks * 4;
    auto source_row = [&](int row) {
        if (row >= BN) return (unsigned)(min(m0 + row - BN, g.M - 1) - m0);
        return (unsigned)(min(n0 + (row & ~31) + 16 * (row >> 2 & 1) + 4 * (row >> 3 & 3) + (row & 3), g.N - 1) - nb);
    };
    unsigned src[Q], ssrc[QS];
#pragma unroll
    for (int j = 0; j < Q; ++j) {
        const int row = (wave + j * NW) * 8 + (lane >> 3), chunk = (lane & 7) ^ (row >> 1 & 7);
        src[j] = source_row(row) * (unsigned)g.ks * 64u + (unsigned)chunk * 16u;
    }
#pragma unroll
    for (int j = 0; j < QS; ++j) {
        const int u = min(wave + j * NW, SU - 1);
        ssrc[j] = S16 ? source_row(u * 64 + lane) * (unsigned)g.ks * 4u : source_row(u * 32 + (lane >> 1)) * (unsigned)g.ks * 4u + (unsigned)(lane & 1) * 4u;
    }
    char* const scales = smem + NS * STAGE;
    const int stages = (g.ks + 1) >> 1;
    // (an odd number of steps: the second half of the last stage is a copy of the first, and not multiplied.  Which half a lane
    // copies does not depend on j: NW * 8 rows are a multiple of 16.)
    const unsigned second = (unsigned)((lane & 7) ^ ((wave * 8 + (lane >> 3)) >> 1 & 7)) >> 2;
    // Stage s, or behind the end the last one again (to where nobody reads), so that every wave always has the same number of
    // copies under way
    auto copy = [&](int s, char* to) {
        const int d = min(s, stages - 1);
        const bool whole = 2 * d + 1 < g.ks;
        const char *w = wq + (size_t)d * 128, *x = xq + (size_t)d * 128;
#pragma unroll
        for (int j = 0; j < Q; ++j) dma16(((wave + j * NW) * 8 < BN ? w : x) + (S16 || whole ? src[j] : src[j] - second * 64u), to + (wave + j * NW) * 1024);
        if (S16 && (s & 1)) return;
        const unsigned char *sw = ws + (size_t)(S16 ? d >> 1 : d) * SROW, *sx = xs + (size_t)(S16 ? d >> 1 : d) * SROW;
        char* const ring = scales + (S16 ? s >> 1 : s) % SRING * SGROUP;
#pragma unroll
        for (int j = 0; j < QS; ++j) {
            const int u = min(wave + j * NW, SU - 1);
            if (S16) dma16((u * 64 < BN ? sw : sx) + ssrc[j], ring + u * 1024);
            else dma4((u * 32 < BN ? sw : sx) + (whole ? ssrc[j] : ssrc[j] - (unsigned)(lane & 1) * 4u), ring + u * 256);
        }
    };

    const int wrow = wn * TN * 32, xrow = BN + wm * TM * 32, swz = r >> 1 & 7;
    f32x16 acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j)
#pragma unroll
            for (int k = 0; k < 16; ++k) acc[i][j][k] = 0.f;

    // One stage: STEPS (4, or 2 of a half one) steps of 64 columns, each TN groups of TM products.  W is read two groups ahead,
    // the next step's X one step ahead, so that a product does not wait for the read before it.
    auto multiply = [&](const char* at, int s, auto steps_t) {
        constexpr int STEPS = decltype(steps_t)::value, GROUPS = STEPS * TN;
        const char *w = at + (wrow + r) * 128, *x = at + (xrow + r) * 128;
        const char* const es_at = scales + (S16 ? s >> 1 : s) % SRING * SGROUP + (S16 ? (s & 1) * 8 : 0) + r * SROW;
        i32x4 X[2][TM], W[3];
        auto read_w = [&](int grp) { return *reinterpret_cast<const i32x4*>(w + (((grp / TN * 2 + h) ^ swz) << 4) + (grp % TN) * 4096); };
        auto read_x = [&](int ks, int j) { return *reinterpret_cast<const i32x4*>(x + (((ks * 2 + h) ^ swz) << 4) + j * 4096); };
        u32x2 es[TN], ex[TM];
#pragma unroll
        for (int j = 0; j < TM; ++j) ex[j] = *reinterpret_cast<const u32x2*>(es_at + (xrow + j * 32) * SROW);
#pragma unroll
        for (int i = 0; i < TN; ++i) es[i] = *reinterpret_cast<const u32x2*>(es_at + (wrow + i * 32) * SROW);
        W[0] = read_w(0);
#pragma unroll
        for (int j = 0; j < TM; ++j) X[0][j] = read_x(0, j);
        W[1] = read_w(1);
        // a lane's bytes of a dword are those of its half of two steps: bits 0 and 16 after the shift
#pragma unroll
        for (int j = 0; j < TM; ++j) ex[j] = ex[j] >> (unsigned)(8 * h);
#pragma unroll
        for (int i = 0; i < TN; ++i) es[i] = es[i] >> (unsigned)(8 * h);
#pragma unroll
        for (int grp = 0; grp < GROUPS; ++grp) {
            const int ks = grp / TN, i = grp % TN;
            if (grp + 2 < GROUPS) W[(grp + 2) % 3] = read_w(grp + 2);
            if (i == 0 && ks + 1 < STEPS)
#pragma unroll
                for (int j = 0; j < TM; ++j) X[(ks + 1) & 1][j] = read_x(ks + 1, j);
            const i32x4 v = W[grp % 3];
            const i32x8 A = {v[0], v[1], v[2], v[3], 0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < TM; ++j) {
                const i32x4 u = X[ks & 1][j];
                const i32x8 B = {u[0], u[1], u[2], u[3], 0, 0, 0, 0};
                if (ks & 1) acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(A, B, acc[i][j], 4, 4, 2, (int)es[i][ks >> 1], 2, (int)ex[j][ks >> 1]);
                else acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(A, B, acc[i][j], 4, 4, 0, (int)es[i][ks >> 1], 0, (int)ex[j][ks >> 1]);
            }
        }
    };
    // Stages s + 1 .. s + NS - 1 are on their way while stage s is multiplied; the counted wait says that stage s is there.  Behind
    // the barrier other waves' copies (or strips) go to where this one has read: its reads have returned by then, wherever the
    // compiler has put the products that use them.
#pragma unroll
    for (int s = 0; s < NS - 1; ++s) copy(s, smem + s * STAGE);
    int cur = 0, nxt = (NS - 1) * STAGE;
    for (int s = 0; s < g.ks >> 1; ++s) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(WAIT) : "memory");
        copy(s + NS - 1, smem + nxt);
        multiply(smem + cur, s, std::integral_constant<int, 4>{});
        nxt = cur;
        cur = cur + STAGE == NS * STAGE ? 0 : cur + STAGE;
    }
    if (!S16 && (g.ks & 1)) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(WAIT) : "memory");
        multiply(smem + cur, stages - 1, std::integral_constant<int, 2>{});
    }
    // the last copies land, and nobody reads the stages any more: their LDS is free
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (OUT == OUT_MX4) {
#pragma unroll
        for (int i = 0; i < TN; ++i) {
            const int n = n0 + (wn * TN + i) * 32 + 16 * h;
            float bias[16];
            bias8(g, n, bias);
            bias8(g, n + 8, bias + 8);
#pragma unroll
            for (int j = 0; j < TM; ++j) {
                float v[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) v[k] = acc[i][j][k];
                finish<OUT_MX4, 16>(g, m0 + (wm * TM + j) * 32 + r, n, bias, v);
            }
        }
        return;
    }
    // A lane holds 16 columns of one row, so that stores from the accumulators touch 32 rows at a time, 16 bytes each.  Strips
    // of 32 rows x 128 bytes (64 where a wavefront has one tile of 16-bit columns) turn in the wavefront's own LDS to whole
    // lines (4096 x 1024 x 1024 to float32: 13.5 -> 10.6 us).
    constexpr int SZ = OUT == CLAVA_DT_F32 ? 4 : 2, TILES = SZ == 2 && TN % 2 == 0 ? 2 : 1, ROW = 32 * TILES * SZ, PITCH = ROW + 16, PER = ROW / 16;
    static_assert(NW * 32 * PITCH <= NS * STAGE, "the strips fit into the stages");
    // Results of many tiles go past the caches, which they would take from the panels: 16384 x 8192 x 8192 540 -> 518 us, with the
    // pack that reads it 606 -> 580; 20000 x 1024 x 512 to bfloat16 15.1 -> 14.4, with it 23.3 -> 24.2; 4096 x 1024 x 1024 to float32
    // 9.5 -> 8.0, with it 18.1 -> 17.4.  Those of 64 x 64 tiles are small and stay for their reader.
    constexpr bool PAST = BN >= 128;
    auto put = [](auto u, auto* to) {
        if (PAST) __builtin_nontemporal_store(u, to);
        else *to = u;
    };
    char* const strip = smem + wave * 32 * PITCH;
#pragma unroll
    for (int i = 0; i < TN; i += TILES) {
        float bias[TILES][16];
#pragma unroll
        for (int p = 0; p < TILES; ++p) {
            const int n = n0 + (wn * TN + i + p) * 32 + 16 * h;
            bias8(g, n, bias[p]);
            bias8(g, n + 8, bias[p] + 8);
        }
#pragma unroll
        for (int j = 0; j < TM; ++j) {
#pragma unroll
            for (int p = 0; p < TILES; ++p) {
                float v[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) v[k] = acc[i + p][j][k] + bias[p][k];
                activate8(v, g.act);
                activate8(v + 8, g.act);
                char* const to = strip + r * PITCH + (p * 32 + 16 * h) * SZ;
                if (SZ == 4) {
#pragma unroll
                    for (int k = 0; k < 16; k += 4) *reinterpret_cast<f32x4*>(to + 4 * k) = f32x4{v[k], v[k + 1], v[k + 2], v[k + 3]};
                } else {
#pragma unroll
                    for (int k = 0; k < 16; k += 8) {
                        u16x8 u;
#pragma unroll
                        for (int e = 0; e < 8; ++e) u[e] = OUT == CLAVA_DT_BF16 ? to_bf16(v[k + e]) : to_f16(v[k + e]);
                        *reinterpret_cast<u16x8*>(to + 2 * k) = u;
                    }
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int k = 0; k < 32 * PER / 64; ++k) {
                const int row = k * (64 / PER) + lane / PER, c = lane % PER;
                const int m = m0 + (wm * TM + j) * 32 + row, n = n0 + (wn * TN + i) * 32 + c * (16 / SZ);
                const u32x4 u = *reinterpret_cast<const u32x4*>(strip + row * PITCH + c * 16);
                if (m >= g.M || n >= g.N) continue;
                char* const to = static_cast<char*>(g.y) + ((size_t)m * g.ldy + n) * SZ;
                if (n + 16 / SZ <= g.N) {
                    if (SZ == 4) put(u, reinterpret_cast<u32x4_u4*>(to));
                    else put(u, reinterpret_cast<u32x4_u2*>(to));
                } else {
#pragma unroll
                    for (int e = 0; e < 16 / SZ; ++e)
                        if (n + e < g.N) {
                            if (SZ == 4) reinterpret_cast<unsigned*>(to)[e] = u[e];
                            else reinterpret_cast<unsigned short*>(to)[e] = (unsigned short)(u[e / 2] >> (16 * (e & 1)));
                        }
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    }
}

template <int BN, int BM, int WN, int WM, int NS, bool S16, int OUT> int launch_tile_s(const Mx4Args& g, int n_cols, hipStream_t st) {
    constexpr int LDS = (BN + BM) * (128 * NS + (S16 ? 16 * (NS / 2 + 1) : 8 * NS));
    static bool set[64] = {};     // by device (threads that race set the same value twice)
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) dev = 0;
    if (!set[dev]) {
        if (hipFuncSetAttribute((const void*)mx4_tile_kernel<BN, BM, WN, WM, NS, S16, OUT>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess) {
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
    mx4_tile_kernel<BN, BM, WN, WM, NS, S16, OUT><<<dim3((unsigned)tiles), WN * WM * 64, LDS, st>>>(g, tiles_n, (int)tiles);
    return CLAVA_OK;
}

template <int BN, int BM, int WN, int WM, int NS, int OUT> int launch_tile(const Mx4Args& g, int n_cols, hipStream_t st) {
    if (g.ks % 4 == 0 && (((uintptr_t)g.xs | (uintptr_t)g.ws) & 15) == 0) return launch_tile_s<BN, BM, WN, WM, NS, true, OUT>(g, n_cols, st);
    return launch_tile_s<BN, BM, WN, WM, NS, false, OUT>(g, n_cols, st);
}

template <int OUT> int launch_linear(const Mx4Args& g, hipStream_t st) {
    // a 4-bit result also has the zero codes behind its last column written: its columns go to the whole step
    const int n_cols = OUT == OUT_MX4 ? g.yks * KSTEP : g.N;
    const int tiles_n = (n_cols + 31) / 32;
    // Few rows (M <= 64) go 16 at a time, which costs most where they are many and the layer is large (us, 16 rows at a time / tiles:
    // K = N = 1024, M = 17 / 64 / 256: 3.9 / 4.5, 3.9 / 4.6, 5.4 / 4.7; 2048: 5.1 / 5.6, 5.2 / 5.8, 13.2 / 6.0; 4096: 7.7 / 8.0,
    // 13.1 / 8.2, 44.5 / 9.4; 8192: 20.9 / 13.3, 44.8 / 13.9, 170 / 23.4: from 4096 on the border could be lower).
    // Many rows: the largest tile that still gives every CU two rounds of work (a large tile copies least per product; us for
    // 256 x 256 / 128 x 128 / 64 x 64 tiles, codes to bfloat16: 16384 x 8192 x 8192 540 / 690 / 1083, 20000 x 1024 x 1024
    // 27.7 / 23.3 / 38.8, 4096 x 1024 x 1024 13.9 / 7.7 / 10.3, 1024 x 1024 x 1024 13.0 / 6.4 / 4.7, 256 x 4096 x 4096
    // 30.2 / 13.0 / 8.4).
    auto tiles = [&](int t) { return (long long)((g.M + t - 1) / t) * ((n_cols + t - 1) / t); };
    // The tiles copy scales by dwords.  Those that start between two (a view into a loaded file) are read by bytes, as those of few
    // rows are: right for any number of rows, but 16 at a time (300 x 1024 x 1024 6.9 us instead of 4.9, 20000 rows 248 instead of 25).
    const bool dwords = (((uintptr_t)g.xs | (uintptr_t)g.ws) & 3) == 0;
    if (g.M > 64 && dwords) {
        if (tiles(256) >= 512) return launch_tile<256, 256, 2, 4, 2, OUT>(g, n_cols, st);
        if (tiles(128) >= 256) return launch_tile<128, 128, 2, 4, 2, OUT>(g, n_cols, st);
        return launch_tile<64, 64, 2, 2, 4, OUT>(g, n_cols, st);
    }
    const long long wgs = (long long)((g.M + 15) / 16) * tiles_n;
    if (wgs > 0x7fffffffLL) {
        clava_set_error("linear_mx4: %d x %d outputs are more than one launch takes", g.M, g.N);
        return CLAVA_ERR_LIMIT;
    }
    const dim3 grid((unsigned)wgs);
    auto few = [&](auto xt) {
        constexpr int XT = decltype(xt)::value;
        mx4_few_kernel<XT, 8, OUT><<<grid, 512, 0, st>>>(g, tiles_n);
    };
    if (g.xt == CLAVA_DT_MX4) few(std::integral_constant<int, CLAVA_DT_MX4>{});
    else if (g.xt == CLAVA_DT_F32) few(std::integral_constant<int, CLAVA_DT_F32>{});
    else if (g.xt == CLAVA_DT_BF16) few(std::integral_constant<int, CLAVA_DT_BF16>{});
    else few(std::integral_constant<int, CLAVA_DT_F16>{});
    return CLAVA_OK;
}

constexpr int MOST_COLUMNS = 1 << 25;         // 255 rows of codes are inside the 32 bits of a lane's source then
// Whether floats are packed by a launch of their own: for one tile of rows and few steps of K every workgroup packs them again
// on the way.  N hardly counts, since the workgroups pack side by side (us, on the way / first, 16 rows: K = 512, N = 256 and 8192
// 3.8 / 5.4 and 4.0 / 5.5; 1024: 4.6 / 6.1 and 4.9 / 6.2; 2048: 6.6 / 7.4 and 6.9 / 7.5; 4096: 10.2 / 10.1 and 11.8 / 10.5; one row:
// 2048: 5.6 / 6.2 and 6.0 / 6.3; 4096: 9.2 / 8.4 and 10.3 / 8.9)
bool packed_first(int M, int K) { return M > 16 || K > 2048; }

}  // namespace

extern "C" {

long long clava_linear_mx4_workspace_bytes(int M, int K, int x_dtype) {
    return M > 0 && K > 0 && packed_first(M, K) && x_dtype != CLAVA_DT_MX4 ? (long long)M * steps(K) * 68 : 0;
}

int clava_linear_mx4_sized(const void* x, int x_dtype, long long ldx, const void* x_scales, const void* w_codes, const void* w_scales,
                           const float* bias, int act, void* y, int y_dtype, long long ldy, void* y_scales, int M, int N, int K,
                           void* workspace, long long workspace_bytes, void* stream) {
    CLAVA_CHECK_ARG(M >= 0 && N > 0 && K > 0, "linear_mx4: M %d, N %d, K %d", M, N, K);
    CLAVA_CHECK_ARG(act >= CLAVA_ACT_NONE && act <= CLAVA_ACT_SILU, "linear_mx4: activation %d", act);
    CLAVA_CHECK_ARG(x_dtype >= 0 && x_dtype <= CLAVA_DT_MX4 && y_dtype >= 0 && y_dtype <= CLAVA_DT_MX4, "linear_mx4: dtypes %d, %d", x_dtype, y_dtype);
    if (M == 0) return CLAVA_OK;
    const bool x4 = x_dtype == CLAVA_DT_MX4, y4 = y_dtype == CLAVA_DT_MX4;
    CLAVA_CHECK_ARG(x && w_codes && w_scales && y && (!y4 || y_scales) && (x4 ? x_scales != nullptr : !packed_first(M, K) || workspace), "linear_mx4: null pointer");
    CLAVA_CHECK_ARG(y4 || ldy >= N || M == 1, "linear_mx4: leading dimension %lld below %d columns", ldy, N);
    CLAVA_CHECK_ARG((((uintptr_t)(x4 ? x : packed_first(M, K) ? workspace : nullptr) | (uintptr_t)w_codes | (uintptr_t)(y4 ? y : nullptr)) & 15) == 0,
                    "linear_mx4: codes and workspace start at 16 bytes");
    CLAVA_CHECK_ARG(N <= 0x7fffff00 && K <= 0x7fffff00 && M <= 0x7fffff00, "linear_mx4: M %d, N %d, K %d", M, N, K);
    if (K > MOST_COLUMNS) {
        clava_set_error("linear_mx4: %d columns are more than one call takes (%d)", K, MOST_COLUMNS);
        return CLAVA_ERR_LIMIT;
    }
    const hipStream_t st = (hipStream_t)stream;
    Mx4Args g;
    g.ks = steps(K);
    g.xq = (const char*)x; g.xs = (const unsigned char*)x_scales;
    g.xt = x_dtype; g.K = K; g.ldx = ldx;
    CLAVA_CHECK_ARG(x4 || ldx >= K || M == 1, "linear_mx4: leading dimension %lld below %d columns", ldx, K);
    const long long need = clava_linear_mx4_workspace_bytes(M, K, x_dtype);
    CLAVA_CHECK_ARG(workspace_bytes >= need, "linear_mx4: needs a workspace of %lld bytes, got %lld", need, workspace_bytes);
    if (need) {
        g.xt = CLAVA_DT_MX4;
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

int clava_linear_mx4(const void* x, int x_dtype, long long ldx, const void* x_scales, const void* w_codes, const void* w_scales,
                     const float* bias, int act, void* y, int y_dtype, long long ldy, void* y_scales, int M, int N, int K,
                     void* workspace, void* stream) {
    // (a workspace of a size that nobody gave is taken to have none)
    return clava_linear_mx4_sized(x, x_dtype, ldx, x_scales, w_codes, w_scales, bias, act, y, y_dtype, ldy, y_scales, M, N, K, workspace, 0, stream);
}

}  // extern "C"
