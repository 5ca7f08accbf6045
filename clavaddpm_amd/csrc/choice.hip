// One class per (row, feature) block from its logits: temperature, top-k, top-p, min-p and the draw from a given uniform.
//
// The kept classes of top-k and top-p are a prefix of the order (z falling, index rising), so each is a threshold: all classes
// with a key above t, and the first n of those with the key t.  Keys are float bits made monotone, so t is found bit by bit.
// Masses a = exp((z - max) / T) are float64: a float32 running sum would put draws next to a border on its wrong side.
#include "elem.h"
#include "rng.h"

namespace {
using namespace elem;

struct Choice {
    const void* z; long long ld;
    int B, m, sumK;
    const int* offsets;
    clava_choice p;
    const float* u; long long ld_u;
    unsigned long long seed, row_offset;
    unsigned step;
    int* idx; float* log_prob;
};

constexpr double LOG2E = 1.44269504088896340736;

// 2^y for y <= 0: n = rint(y), 2^(y - n) by its power series (12 terms: ln2/2 ^ 13 / 13! < 2e-16), scaled by 2^n.
__device__ __forceinline__ double exp2_nonpos(double y) {
    y = fmax(y, -1100.0);                     // below float64's smallest subnormal
    const double n = rint(y), r = (y - n) * 0.69314718055994530942;
    double p = 1.0 / 479001600;
    p = fma(p, r, 1.0 / 39916800);
    p = fma(p, r, 1.0 / 3628800);
    p = fma(p, r, 1.0 / 362880);
    p = fma(p, r, 1.0 / 40320);
    p = fma(p, r, 1.0 / 5040);
    p = fma(p, r, 1.0 / 720);
    p = fma(p, r, 1.0 / 120);
    p = fma(p, r, 1.0 / 24);
    p = fma(p, r, 1.0 / 6);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return ldexp(p, (int)n);
}

__device__ __forceinline__ unsigned key_of(float z) {
    const unsigned b = __float_as_uint(z + 0.f);              // -0 and +0 are one key
    return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}

// Logits of a block relative to its maximum, as masses: +inf logits, where there are any, share the mass.
struct Mass {
    double top, c;                            // maximum, log2(e) / T
    bool inf;
    __device__ __forceinline__ double operator()(float z) const {
        if (inf) return z == INFINITY ? 1.0 : 0.0;
        return z == -INFINITY ? 0.0 : exp2_nonpos(((double)z - top) * c);
    }
};

__device__ __forceinline__ double uniform_of(const Choice& g, int b, int f) {
    if (g.u) return (double)g.u[(size_t)b * g.ld_u + f];
    const unsigned long long e = (g.row_offset + (unsigned long long)b) * (unsigned long long)g.m + (unsigned long long)f;
    return (double)clava_rng::to_uniform(clava_rng::philox4x32_10(g.seed, e, g.step, clava_rng::STREAM_CHOICE).x);
}

constexpr int W = 256;

template <class T> struct Sum { __device__ T operator()(T a, T b) const { return a + b; } };
struct Max { __device__ float operator()(float a, float b) const { return fmaxf(a, b); } };

// Inclusive scan over the workgroup in thread order; s is W elements of LDS
template <class T, class Op> __device__ __forceinline__ T scan(T v, T* s, Op op) {
    const int t = threadIdx.x;
    __syncthreads();
    s[t] = v;
    for (int d = 1; d < W; d *= 2) {
        __syncthreads();
        const T o = t >= d ? s[t - d] : v;
        __syncthreads();
        if (t >= d) { v = op(o, v); s[t] = v; }
    }
    __syncthreads();
    return v;
}
template <class T, class Op> __device__ __forceinline__ T reduce(T v, T* s, Op op) {
    scan(v, s, op);
    return s[W - 1];
}

template <int DT> __global__ void __launch_bounds__(W) choose_kernel(Choice g) {
    __shared__ double sd[W];
    __shared__ float sf[W];
    __shared__ int si[W];
    const int t = threadIdx.x;
    for (long long blk = blockIdx.x; blk < (long long)g.B * g.m; blk += gridDim.x) {
        const int b = (int)(blk / g.m), f = (int)(blk - (long long)b * g.m);
        const int k0 = g.offsets ? max(0, min(g.offsets[f], g.sumK)) : 0;
        const int K = (g.offsets ? max(k0, min(g.offsets[f + 1], g.sumK)) : g.sumK) - k0;
        const size_t at = (size_t)b * g.ld + k0;
        const double u = uniform_of(g, b, f);
        const clava_choice& p = g.p;
        double T = p.temperature_t ? (double)p.temperature_t[b * p.temperature_rs + f * p.temperature_fs] : p.temperature;
        double top_p = p.top_p_t ? (double)p.top_p_t[b * p.top_p_rs + f * p.top_p_fs] : p.top_p;
        double min_p = p.min_p_t ? (double)p.min_p_t[b * p.min_p_rs + f * p.min_p_fs] : p.min_p;
        int top_k = p.top_k_t ? p.top_k_t[b * p.top_k_rs + f * p.top_k_fs] : p.top_k;
        float mx = -INFINITY;
        int nan = 0;
        for (int i = t; i < K; i += W) {
            const float z = load1<DT>(g.z, at + i);
            nan |= z != z;
            mx = fmaxf(mx, z);
        }
        mx = reduce(mx, sf, Max());
        nan = reduce(nan, si, Sum<int>());
        if (nan || mx == -INFINITY || u != u || !(T >= 0.0)) {
            if (t == 0) {
                g.idx[blk] = -1;
                if (g.log_prob) g.log_prob[blk] = __uint_as_float(0x7fc00000u);
            }
            continue;
        }
        if (T < 1e-290) { T = 1.0; top_k = 1; }           // 0, and what 1 / T has no float64 for
        min_p = fmin(fmax(min_p, 0.0), 1.0);              // (fmax of a NaN: 0)
        top_p = fmax(top_p, 1e-290);                      // the first of the order always stays
        const Mass mass{(double)mx, LOG2E / T, mx == INFINITY};
        // keep: key above `edge`, or the first `ties` with that key
        unsigned edge = 0;
        int ties = K;
        const bool cut_k = top_k > 0 && top_k < K, cut_p = top_p < 1.0;
        if (cut_k) {
            for (int bit = 31; bit >= 0; --bit) {
                const unsigned at_least = edge | 1u << bit;
                int n = 0;
                for (int i = t; i < K; i += W) n += key_of(load1<DT>(g.z, at + i)) >= at_least;
                if (reduce(n, si, Sum<int>()) >= top_k) edge = at_least;
            }
            int above = 0;
            for (int i = t; i < K; i += W) above += key_of(load1<DT>(g.z, at + i)) > edge;
            ties = top_k - reduce(above, si, Sum<int>());
        }
        if (cut_p) {
            // mass of the keys >= `least` that top-k left
            auto mass_from = [&](unsigned least) {
                double s = 0.0;
                for (int i = t; i < K; i += W) {
                    const float z = load1<DT>(g.z, at + i);
                    const unsigned k = key_of(z);
                    if (k >= least && (!cut_k || k > edge)) s += mass(z);
                }
                return reduce(s, sd, Sum<double>());
            };
            const float edge_z = __uint_as_float(edge & 0x80000000u ? edge ^ 0x80000000u : ~edge);
            const double at_edge = cut_k ? ties * mass(edge_z) : 0.0;
            const double goal = top_p * (mass_from(0) + at_edge);
            unsigned e = 0;
            for (int bit = 31; bit >= 0; --bit) {
                const unsigned least = e | 1u << bit;
                if (mass_from(least) + (cut_k && least <= edge ? at_edge : 0.0) >= goal) e = least;
            }
            // e: the key at which the prefix reaches the goal; how many of that key
            if (!cut_k || e > edge) {
                int n = 0;
                for (int i = t; i < K; i += W) n += key_of(load1<DT>(g.z, at + i)) == e;
                ties = reduce(n, si, Sum<int>());
            }
            const double before = e == 0xffffffffu ? 0.0 : mass_from(e + 1);
            edge = e;
            const double one = mass(__uint_as_float(e & 0x80000000u ? e ^ 0x80000000u : ~e));
            const double n = one > 0.0 ? ceil((goal - before) / one) : (double)ties;
            ties = max(1, (int)fmin(fmax(n, 1.0), (double)ties));
        }
        // the draw: a run of neighbouring classes a thread, so that sums follow the index
        const int per = (K + W - 1) / W, i0 = min(K, t * per), i1 = min(K, i0 + per);
        int eq = 0;
        for (int i = i0; i < i1; ++i) eq += key_of(load1<DT>(g.z, at + i)) == edge;
        int seen = scan(eq, si, Sum<int>()) - eq;
        const int seen0 = seen;
        auto kept = [&](float z) {
            const unsigned k = key_of(z);
            const bool in = k > edge || (k == edge && seen < ties);
            seen += k == edge;
            const double a = in ? mass(z) : 0.0;
            return a >= min_p ? a : 0.0;
        };
        double own = 0.0;
        for (int i = i0; i < i1; ++i) own += kept(load1<DT>(g.z, at + i));
        scan(own, sd, Sum<double>());
        const double total = sd[W - 1], goal = fmin(fmax(u, 0.0) * total, total * (1.0 - 0x1p-50));
        double run = t ? sd[t - 1] : 0.0;
        if (run <= goal && sd[t] > goal) {
            seen = seen0;
            int hit = -1;
            double a_hit = 0.0;
            for (int i = i0; i < i1; ++i) {
                const double a = kept(load1<DT>(g.z, at + i));
                run += a;
                if (a > 0.0) {
                    hit = i;
                    a_hit = a;
                    if (run > goal) break;
                }
            }
            g.idx[blk] = hit;
            if (g.log_prob) g.log_prob[blk] = (float)log(a_hit / total);
        }
    }
}

}  // namespace

extern "C" {

long long clava_choice_workspace_bytes(int, int, int) { return 0; }

int clava_sample_categories(const void* logits, int dtype, long long ld, int B, int m, int sumK, const int* offsets, int max_k,
                            const clava_choice* choice, const float* uniforms, long long ld_u, unsigned long long seed,
                            unsigned long long row_offset, unsigned step_index, int* idx, float* log_prob, void* workspace,
                            long long workspace_bytes, void* stream) {
    CLAVA_CHECK_ARG(B >= 0 && m > 0 && sumK >= 0, "sample_categories: B %d, m %d, sumK %d", B, m, sumK);
    CLAVA_CHECK_ARG(choice && (offsets || m == 1), "sample_categories: null choice, or null offsets with %d features", m);
    if (B == 0) return CLAVA_OK;
    CLAVA_CHECK_ARG((logits || sumK == 0) && idx, "sample_categories: null pointer");
    CLAVA_CHECK_ARG(dtype >= 0 && dtype <= CLAVA_DT_F16, "sample_categories: dtype %d", dtype);
    CLAVA_CHECK_ARG(ld >= sumK || B == 1, "sample_categories: leading dimension %lld below %d classes", ld, sumK);
    CLAVA_CHECK_ARG(!uniforms || ld_u >= m || B == 1, "sample_categories: leading dimension %lld below %d uniforms", ld_u, m);
    CLAVA_CHECK_ARG(sumK <= (1 << 30), "sample_categories: %d classes", sumK);
    const hipStream_t st = (hipStream_t)stream;
    Choice g;
    g.z = logits; g.ld = ld; g.B = B; g.m = m; g.sumK = sumK; g.offsets = offsets; g.p = *choice;
    g.u = uniforms; g.ld_u = ld_u; g.seed = seed; g.row_offset = row_offset; g.step = step_index;
    g.idx = idx; g.log_prob = log_prob;
    const long long blocks = (long long)B * m;
    const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536));
    ProfScope prof(PROF_CHOICE, 0, (double)B * sumK * (dtype == CLAVA_DT_F32 ? 4 : 2) + 12.0 * blocks, st);
    if (dtype == CLAVA_DT_F32) choose_kernel<CLAVA_DT_F32><<<grid, W, 0, st>>>(g);
    else if (dtype == CLAVA_DT_BF16) choose_kernel<CLAVA_DT_BF16><<<grid, W, 0, st>>>(g);
    else choose_kernel<CLAVA_DT_F16><<<grid, W, 0, st>>>(g);
    CLAVA_CHECK_LAUNCH("sample_categories");
    return CLAVA_OK;
}

}  // extern "C"
