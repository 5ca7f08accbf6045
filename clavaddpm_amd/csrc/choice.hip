// One class per (row, feature) block from its logits: temperature, top-k, top-p, min-p and the draw from a given uniform.
//
// Masses a = exp((z - max) / T) are float64, or 64-bit integers counting 2^-s of the largest mass: a float32 running sum puts
// draws next to a border on its wrong side, and integers add up to the same in every order.
//
// Top-k and top-p both keep a prefix of the order (z falling, index rising): the last kept class is the first one at which the
// running weight (1 a class, or its mass) reaches a goal (k, or top_p of the mass).  So both are one search, "the edge":
// classes fall into bins of falling z, the running weight over the bins names the bin of the edge, and only that bin's
// classes are put in order.  Bins are linear in max - z (a logit's neighbours in z are its neighbours in mass too; bins of the
// float's bits would put nearly all of them around z = 0), and where too many classes share one, its range of keys (float bits
// made monotone) is cut again: six bits a time, down to equal keys, of which the first by index stay.
//
// Which kernel: up to 64 classes, a class a lane, in groups of 8 / 16 / 32 / 64 lanes; up to 64 * NV, a wavefront with the
// block in LDS; wider ones are cut into chunks over many workgroups and joined (wide_*).
//
// Each logit is read once up to 2048 classes (wider: three or four times, from the caches mostly), so that memory would need
// 35 us for 4096 rows of 50 features with 10 047 classes (float32).  They take 111 us, all filters at 20000 rows 760 (174): bound
// by vector instructions, 258 and 379 a block, three quarters and four fifths of the issue cycles.  A mass takes 20 (64 classes at
// once): of the 258 about a third; with the filters it is the passes over the bins, the sort and the sums.  Parameters from
// tensors: 173 and 1010 us, since every block makes its own out of them.
#include "elem.h"
#include "rng.h"
#include "wave.h"

namespace {
using namespace elem;
typedef unsigned long long u64;

constexpr double LOG2E = 1.44269504088896340736, LN2 = 0.69314718055994530942;

// The parameters of a draw, ready to use
struct Params {
    double c, top_p, min_p;                   // log2(e) / T; in (0, 1], 1: off; in [0, 1]
    float T;                                  // for bin widths only
    int top_k;                                // 0: off
    bool bad;                                 // the temperature is negative, or one of them is no number
};
__host__ __device__ __forceinline__ Params params_of(double T, double top_p, double min_p, int top_k) {
    Params p;
    p.bad = !(T >= 0.0) || top_p != top_p || min_p != min_p;
    if (!(T >= 1e-290)) { T = 1.0; top_k = 1; }              // 0, and what 1 / T has no float64 for
    p.c = LOG2E / T;
    if (p.c < 1e-290) p.c = 1e-290;                          // (an infinite T: -inf * c stays -inf)
    p.T = T < 1e30 ? (float)T : 1e30f;
    p.top_k = top_k > 0 ? top_k : 0;
    p.min_p = min_p > 0.0 ? (min_p < 1.0 ? min_p : 1.0) : 0.0;
    p.top_p = top_p < 1.0 ? (top_p > 1e-290 ? top_p : 1e-290) : 1.0;       // the first of the order always stays
    return p;
}

struct Choice {
    const void* z; long long ld;
    int B, m, sumK;
    const int* offsets;
    clava_choice p;
    Params same;                              // for all blocks, unless one of them is a tensor
    const float* u; long long ld_u;
    unsigned long long seed, row_offset;
    unsigned step;
    int* idx; float* log_prob;
    bool wide;                                // blocks of more than wide_from, at most wide_to classes belong to the wide_* kernels
    int wide_from, wide_to;
};

// 2^y for y <= 0 (NaN and what is below float64: 0): n = rint(y), 2^(y - n) by its power series in base 2, ln2^k / k!, up to
// k = 11 (the next term is 6e-15 at |y - n| = 1/2), scaled by 2^n.
struct Exp2Terms {
    double t[12];
    constexpr Exp2Terms() : t{} {
        t[0] = 1.0;
        for (int k = 1; k < 12; ++k) t[k] = t[k - 1] * LN2 / k;
    }
};
__device__ __forceinline__ double exp2_nonpos(double y) {
    constexpr Exp2Terms c;
    y = fmax(y, -1100.0);
    const double n = rint(y), r = y - n;
    // Written out, since the terms belong in scalar registers: the compiler kept 22 vector registers of them and copied one for
    // every step (20000 x 50 filtered 884 -> 795 us together with lane moves that need no zero first).  The wait is for scalar
    // registers that a vector instruction wrote just before (a v_readlane of spilled ones): two states, which the compiler does
    // not count for written-out code.
    double p;
    asm("s_nop 1\n\t"
        "v_fma_f64 %0, %1, %2, %3\n\t"
        "v_fma_f64 %0, %0, %2, %4\n\t"
        "v_fma_f64 %0, %0, %2, %5\n\t"
        "v_fma_f64 %0, %0, %2, %6\n\t"
        "v_fma_f64 %0, %0, %2, %7\n\t"
        "v_fma_f64 %0, %0, %2, %8\n\t"
        "v_fma_f64 %0, %0, %2, %9\n\t"
        "v_fma_f64 %0, %0, %2, %10\n\t"
        "v_fma_f64 %0, %0, %2, %11\n\t"
        "v_fma_f64 %0, %0, %2, %12"
        : "=&v"(p)
        : "v"(c.t[11]), "v"(r), "s"(c.t[10]), "s"(c.t[9]), "s"(c.t[8]), "s"(c.t[7]), "s"(c.t[6]), "s"(c.t[5]), "s"(c.t[4]),
          "s"(c.t[3]), "s"(c.t[2]), "s"(c.t[1]));
    return ldexp(fma(p, r, 1.0), (int)n);
}
// log(x) for x >= 1: the float32 logarithm and one Newton step on e^y = x (its square, 1e-14, is what stays)
__device__ __forceinline__ double log_from1(double x) {
    const double y = (double)logf((float)x);
    return y + (x * exp2_nonpos(-y * LOG2E) - 1.0);
}

__device__ __forceinline__ unsigned key_of(float z) {
    const unsigned b = __float_as_uint(z + 0.f);              // -0 and +0 are one key
    return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
// Position in the order: larger comes first; equal keys by index
__device__ __forceinline__ u64 place_of(unsigned key, unsigned index) { return (u64)key << 32 | (unsigned)~index; }

__device__ __forceinline__ int first_of(const Choice& g, int f) { return g.offsets ? max(0, min(g.offsets[f], g.sumK)) : 0; }
__device__ __forceinline__ int classes_of(const Choice& g, int f) {
    return g.offsets ? max(0, min(g.offsets[f + 1], g.sumK) - first_of(g, f)) : g.sumK;
}
__device__ __forceinline__ double uniform_of(const Choice& g, int b, int f) {
    if (g.u) return (double)g.u[(size_t)b * g.ld_u + f];
    const unsigned long long e = (g.row_offset + (unsigned long long)b) * (unsigned long long)g.m + (unsigned long long)f;
    return (double)clava_rng::to_uniform(clava_rng::philox4x32_10(g.seed, e, g.step, clava_rng::STREAM_CHOICE).x);
}
// A block, its parameters and random number
struct Block : Params {
    int b, f, K;
    size_t at;
    double u;
};
// What a kernel is compiled for: numbers without top-k and top-p, numbers, tensors.  (Each leaves out the code and the
// arguments that it does not need; with all of them in one, 140 scalar registers were moved to lanes and back.)
enum { PLAIN = 0, FILTERED = 1, TENSORS = 2 };
template <int MODE> __device__ __forceinline__ Block block_of(const Choice& g, int b, int f, int k0, int K) {
    Block x;
    static_cast<Params&>(x) = g.same;
    if (MODE == TENSORS) {
        const clava_choice& p = g.p;
        const double T = p.temperature_t ? (double)p.temperature_t[b * p.temperature_rs + f * p.temperature_fs] : p.temperature;
        const double top_p = p.top_p_t ? (double)p.top_p_t[b * p.top_p_rs + f * p.top_p_fs] : p.top_p;
        const double min_p = p.min_p_t ? (double)p.min_p_t[b * p.min_p_rs + f * p.min_p_fs] : p.min_p;
        static_cast<Params&>(x) = params_of(T, top_p, min_p, p.top_k_t ? p.top_k_t[b * p.top_k_rs + f * p.top_k_fs] : p.top_k);
    }
    x.b = b; x.f = f; x.K = K;
    x.at = (size_t)b * g.ld + k0;
    x.u = uniform_of(g, b, f);
    x.bad |= x.u != x.u;
    x.u = fmax(x.u, 0.0);
    return x;
}
// +inf logits, where there are any, share the mass: as zeros among -inf
__device__ __forceinline__ float settle(float z, bool inf) { return inf ? (z == INFINITY ? 0.f : -INFINITY) : z; }
// log2 of a class's mass, and the mass, from its logit and the largest one, which is finite (-inf: no mass)
__device__ __forceinline__ double log2_mass(float z, float top, double c) { return ((double)z - (double)top) * c; }
__device__ __forceinline__ double mass_of(float z, float top, double c) { return exp2_nonpos(log2_mass(z, top, c)); }
// a in units of 2^-s, s <= 51, to the nearest: the fraction bits of a * 2^s + 2^52
__device__ __forceinline__ u64 units(double a, double scale) {
    return (u64)__double_as_longlong(fma(a, scale, 0x1p52)) & 0xfffffffffffffull;
}
// The scale for K classes: their sum stays under 2^63, one mass under 2^52
__device__ __forceinline__ double unit_scale(int K) {
    const int s = min(51, 62 - (K > 1 ? 32 - (int)__builtin_clz((unsigned)(K - 1)) : 0));
    return (double)(1ull << s);
}
// The goal of a draw among integer weights: the class up to which more than this is the one
__device__ __forceinline__ u64 draw_goal(double u, u64 total) {
    const double goal = u * (double)total;
    return goal < (double)total ? min((u64)goal, total - 1) : total - 1;
}

__device__ __forceinline__ void give(const Choice& g, int b, int f, int idx, float lp) {
    const size_t o = (size_t)b * g.m + f;
    g.idx[o] = idx;
    if (g.log_prob) g.log_prob[o] = lp;
}
__device__ __forceinline__ float no_number() { return __uint_as_float(0x7fc00000u); }

// ------------------------------------------------------------------------------------------------------ lanes of a group
// The value of the lane that CTRL names, 0 where there is none or the row is not in ROWS
template <int CTRL, int ROWS = 0xf> __device__ __forceinline__ unsigned dpp_d(unsigned b) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)b, CTRL, ROWS, 0xf, ROWS == 0xf);
}
template <int CTRL, int ROWS = 0xf> __device__ __forceinline__ u64 dpp_d(u64 b) {
    return (u64)dpp_d<CTRL, ROWS>((unsigned)(b >> 32)) << 32 | dpp_d<CTRL, ROWS>((unsigned)b);
}
template <int CTRL, int ROWS = 0xf> __device__ __forceinline__ double dpp_d(double v) {
    return __longlong_as_double((long long)dpp_d<CTRL, ROWS>((u64)__double_as_longlong(v)));
}
// The lane, computed anew: what follows from it (a lane mask for every step of a sort) is not kept over a loop of blocks,
// where it took 240 scalar registers
__device__ __forceinline__ int lane_here() {
    int l = threadIdx.x & 63;
    asm volatile("" : "+v"(l));
    return l;
}
// Inclusive sums in lane order within groups of G lanes
template <int G, class T> __device__ __forceinline__ T scan(T v) {
    if (G == 8) {
        const int l = lane_here();
        T o = dpp_d<0x111>(v);
        v += (l & 7) >= 1 ? o : T(0);
        o = dpp_d<0x112>(v);
        v += (l & 7) >= 2 ? o : T(0);
        o = dpp_d<0x114>(v);
        v += (l & 7) >= 4 ? o : T(0);
        return v;
    }
    v += dpp_d<0x111>(v);                     // row_shr within rows of 16
    v += dpp_d<0x112>(v);
    v += dpp_d<0x114>(v);
    v += dpp_d<0x118>(v);
    if (G >= 32) v += dpp_d<0x142, 0xa>(v);   // the last lane of row 0 to row 1, of row 2 to row 3
    if (G >= 64) v += dpp_d<0x143, 0xc>(v);   // lane 31 to rows 2 and 3
    return v;
}
__device__ __forceinline__ u64 from_lane(u64 v, int lane) {
    return (u64)(unsigned)__shfl((int)(v >> 32), lane, 64) << 32 | (unsigned)__shfl((int)v, lane, 64);
}
__device__ __forceinline__ double from_lane(double v, int lane) {
    return __longlong_as_double((long long)from_lane((u64)__double_as_longlong(v), lane));
}
// The same for a lane that is the same in the whole wavefront, without a way through LDS
__device__ __forceinline__ int at_lane(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ u64 at_lane(u64 v, int lane) { return (u64)(unsigned)at_lane((int)(v >> 32), lane) << 32 | (unsigned)at_lane((int)v, lane); }
__device__ __forceinline__ double at_lane(double v, int lane) {
    return __longlong_as_double((long long)at_lane((u64)__double_as_longlong(v), lane));
}
// Lane l's value of lane l ^ d: moves within rows of 16 lanes, exchanges of rows and halves
__device__ __forceinline__ int from_xor(int v, int d) {
    constexpr int QUAD_MIRROR = 0x1B;
    if (d == 1) return dpp_i<DPP_XOR1>(v);
    if (d == 2) return dpp_i<DPP_XOR2>(v);
    if (d == 4) return dpp_i<QUAD_MIRROR>(dpp_i<DPP_HALF_MIRROR>(v));            // l ^ 7 ^ 3
    if (d == 8) return dpp_i<DPP_HALF_MIRROR>(dpp_i<DPP_ROW_MIRROR>(v));         // l ^ 15 ^ 7
    const auto o = d == 16 ? __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, false, false)
                           : __builtin_amdgcn_permlane32_swap((unsigned)v, (unsigned)v, false, false);
    return (int)(__builtin_amdgcn_inverse_ballot_w64(d == 16 ? 0xffff0000ffff0000ull : 0xffffffff00000000ull) ? o[0] : o[1]);
}
__device__ __forceinline__ u64 from_xor(u64 v, int d) { return (u64)(unsigned)from_xor((int)(v >> 32), d) << 32 | (unsigned)from_xor((int)v, d); }
// Bitonic sort within groups of G lanes, largest first.  Which lanes keep the larger one in a step is a constant, as a mask.
constexpr u64 sort_mask(int G, int k, int d) {
    u64 m = 0;
    for (int l = 0; l < 64; ++l)
        if (((l & d) == 0) == ((l & k & (G - 1)) == 0 || k == G)) m |= 1ull << l;
    return m;
}
template <int G> __device__ __forceinline__ u64 sort_falling(u64 v) {
#pragma unroll
    for (int k = 2; k <= G; k *= 2)
#pragma unroll
        for (int d = k / 2; d > 0; d /= 2) {
            const u64 o = from_xor(v, d);
            v = __builtin_amdgcn_inverse_ballot_w64(~(__ballot(v > o) ^ sort_mask(G, k, d))) ? v : o;
        }
    return v;
}

// The same in one register: both lanes of a pair see the pair, the mask says which keeps the larger
template <int G> __device__ __forceinline__ unsigned sort_falling(unsigned v) {
#pragma unroll
    for (int k = 2; k <= G; k *= 2)
#pragma unroll
        for (int d = k / 2; d > 0; d /= 2) {
            unsigned o;
            if (d >= 16) {
                const auto pair = d == 16 ? __builtin_amdgcn_permlane16_swap(v, v, false, false) : __builtin_amdgcn_permlane32_swap(v, v, false, false);
                v = pair[0];
                o = pair[1];
            } else o = (unsigned)from_xor((int)v, d);
            v = __builtin_amdgcn_inverse_ballot_w64(sort_mask(G, k, d)) ? max(v, o) : min(v, o);
        }
    return v;
}
// The places (key, 63 - lane) of a group's lanes, largest first.  They are sorted by the leading 26 or 27 bits of max - z with
// the lane below them, in one register; where that has left two in the wrong order (bits that agree: under one block in a
// hundred at 50 classes) or max - z is no number, by all their bits.
template <int G> __device__ __forceinline__ u64 sort_places(unsigned key, float z, float top) {
    const int lane = threadIdx.x & 63, l = lane & (G - 1);
    const u64 place = (u64)key << 32 | (unsigned)(63 - lane);
    if (G < 32) return sort_falling<G>(place);
    const unsigned first = sort_falling<G>((~(__float_as_uint(top - z) << 1) & ~(unsigned)(G - 1)) | (unsigned)(G - 1 - l));
    const int from = (lane | (G - 1)) - (int)(first & (G - 1));
    const u64 sorted = (u64)(unsigned)__shfl((int)key, from, 64) << 32 | (unsigned)(63 - from);
    constexpr int WAVE_SHR1 = 0x138;
    const u64 above = dpp_d<WAVE_SHR1>(sorted);
    return __any(l > 0 && above < sorted) ? sort_falling<G>(place) : sorted;
}

// What a wavefront has chosen, a block a lane: the logarithms and the stores of 64 blocks are done together
struct Chosen {
    unsigned n, out;
    int index;
    double y, total;
    __device__ __forceinline__ void flush(const Choice& g) {
        if ((threadIdx.x & 63) < n) {
            g.idx[out] = index;
            if (g.log_prob) g.log_prob[out] = (float)(y * LN2 - log_from1(total));
        }
        n = 0;
    }
    __device__ __forceinline__ void add(const Choice& g, const Block& x, int i, double log2_a, double mass) {
        if ((threadIdx.x & 63) == n) {
            out = (unsigned)x.b * (unsigned)g.m + (unsigned)x.f;
            index = i;
            y = log2_a;
            total = mass;
        }
        if (++n == 64) flush(g);
    }
};

// The whole choice among the classes that a group's lanes hold, one each, in index order: `z` (-inf and key 0 where a lane holds
// none), their index, the block's maximum.  `nan`: the block holds a NaN.  All lanes of the wave come here together.
template <int G, int MODE> __device__ __forceinline__ void choose_lanes(const Choice& g, const Block& x, float z, unsigned key, int index, float top,
                                                              bool nan, bool live, Chosen* chosen) {
    const int lane = threadIdx.x & 63, base = lane & ~(G - 1), l = lane & (G - 1);
    const u64 group = (G == 64 ? ~0ull : ((1ull << (G & 63)) - 1)) << base;
    auto last_of = [&](auto v) { return G == 64 ? at_lane(v, 63) : from_lane(v, base + G - 1); };
    const bool inf = top == INFINITY;
    const double y = log2_mass(settle(z, inf), inf ? 0.f : top, x.c), a = exp2_nonpos(y);
    bool keep = a >= x.min_p;
    if (MODE != PLAIN && __any(x.top_k > 0 || x.top_p < 1.0)) {
        const u64 place = (u64)key << 32 | (unsigned)(63 - lane), sorted = sort_places<G>(key, z, top);
        const bool in = x.top_k == 0 || l < x.top_k;
        const double as = from_lane(a, 63 - (int)(unsigned)sorted);
        const double w = in ? as : 0.0, run = scan<G>(w);
        const double goal = x.top_p * last_of(run);
        const bool stay = in && (l == 0 || x.top_p >= 1.0 || run - w < goal);
        const u64 out = ~(__ballot(stay) >> base) | (G == 64 ? 0 : 1ull << (G & 63));
        const int n = out ? (int)__builtin_ctzll(out) : 64;      // those before the first that goes
        const u64 last = G == 64 ? at_lane(sorted, n - 1) : from_lane(sorted, base + n - 1);      // (of every lane: not behind `keep`)
        keep = keep && place >= last;
    }
    const double w = keep ? a : 0.0, run = scan<G>(w), total = last_of(run);
    const double goal = x.u * total;
    const u64 can = __ballot(w > 0.0) & group, past = __ballot(w > 0.0 && run > goal) & group;
    const bool none = nan || x.bad || top == -INFINITY;
    const int hit = past ? (int)__builtin_ctzll(past) : can ? 63 - (int)__builtin_clzll(can) : 0;
    if (G == 64) {
        if (none) {
            if (lane == 0) give(g, x.b, x.f, -1, no_number());
        } else chosen->add(g, x, at_lane(index, hit), at_lane(y, hit), total);
    } else {
        const float lp = g.log_prob ? (float)(y * LN2 - log_from1(total)) : 0.f;
        if (live && (none ? l == 0 : lane == hit)) give(g, x.b, x.f, none ? -1 : index, none ? no_number() : lp);
    }
}

// ---------------------------------------------------------------------------------------------------- a wavefront's block
// What a wavefront keeps in LDS beside its block's logits: bins, then the classes of one bin
struct WaveLds {
    u64 bin[64];
    u64 place[64];
    u64 weight[64];
};
// Bins per unit of max - z: over the range of the logits, or 40 T where that is less (no mass is left beyond it, and what
// shares the last bin is cut again if an edge falls into it).  0: all classes share the first bin, for ranges that are not
// numbers or have no inverse.
__device__ __forceinline__ float bins_per_unit(float top, float bottom, float T, float bins) {
    const float range = fminf(top - bottom, 40.f * T), inv = bins / range;
    return top < INFINITY && range > 0.f && range < 1e37f && inv < 1e37f ? inv : 0.f;
}
__device__ __forceinline__ int linear_bin(float z, float top, float inv, int bins) {
    return inv > 0.f ? (int)fminf((top - z) * inv, (float)(bins - 1)) : 0;
}
// LDS of one wavefront is read and written in program order; this keeps the compiler to it
__device__ __forceinline__ void lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ unsigned wave_min(unsigned v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = min(v, (unsigned)__shfl_xor((int)v, o, 64));
    return v;
}
__device__ __forceinline__ unsigned wave_max(unsigned v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, o, 64));
    return v;
}

// The block's classes by slots of 64: logit `z[j * 64 + lane]` in LDS, -inf behind the last one
struct WaveBlock {
    const float* z;
    int n;                                                   // slots
    float top, inv;
};
// Weights in 64 linear bins of falling z (lane l: bin l)
template <class In, class Weight> __device__ __forceinline__ u64 bins_of(const WaveBlock& w, WaveLds& s, In in, Weight weight) {
    const int lane = threadIdx.x & 63;
    s.bin[lane] = 0;
    lds_order();
    for (int j = 0; j < w.n; ++j) {
        const float z = w.z[j * 64 + lane];
        if (in(z, j)) atomicAdd(&s.bin[linear_bin(z, w.top, w.inv, 64)], weight(z));
    }
    lds_order();
    return s.bin[lane];
}
// The place of the first class, in falling order, at which the running weight reaches `goal`; 0 if none does.  The classes are
// those with in(z, slot), `bins` their weights by bins_of.
template <class In, class Weight>
__device__ __forceinline__ u64 find_edge(const WaveBlock& w, u64 bins, double goal, WaveLds& s, In in, Weight weight) {
    const int lane = threadIdx.x & 63;
    unsigned lo = 0, hi = 0xffffffffu;                       // keys of the classes that are left
    u64 before = 0;
    int shift = -1;                                          // < 0: linear bins
    for (;;) {
        const u64 run = scan<64>(bins), past = __ballot((double)(before + run) >= goal);
        if (past == 0) return 0;
        const int at = (int)__builtin_ctzll(past);
        before += at_lane(run - bins, at);
        // the classes of that bin
        int count = 0;
        unsigned klo = 0xffffffffu, khi = 0;
        for (int j = 0; j < w.n; ++j) {
            const float z = w.z[j * 64 + lane];
            const unsigned key = key_of(z);
            const bool is = in(z, j) && key >= lo && key <= hi &&
                            (shift < 0 ? linear_bin(z, w.top, w.inv, 64) : (int)((hi - key) >> shift)) == at;
            const u64 who = __ballot(is);
            if (who == 0) continue;
            const int pos = count + (int)__popcll(who & ((1ull << lane) - 1));
            if (is) {
                if (pos < 64) { s.place[pos] = place_of(key, (unsigned)(j * 64 + lane)); s.weight[pos] = weight(z); }
                klo = min(klo, key);
                khi = max(khi, key);
            }
            count += (int)__popcll(who);
        }
        lds_order();
        if (count <= 64) {
            const u64 mine = lane < count ? s.place[lane] : 0;
            // sorted with the position in the list, which is in index order, instead of the index
            const u64 sorted = sort_falling<64>(lane < count ? (mine >> 32 << 32 | (unsigned)(63 - lane)) : 0);
            const int pos = 63 - (int)(sorted & 63);
            const u64 sum = scan<64>(lane < count ? s.weight[pos] : (u64)0);
            const u64 there = __ballot(lane < count && (double)(before + sum) >= goal);
            return at_lane(mine, at_lane(pos, there ? (int)__builtin_ctzll(there) : count - 1));
        }
        lo = wave_min(klo);
        hi = wave_max(khi);
        if (lo == hi) {                                      // equal keys, equal weights: the first so many by index
            const double one = (double)s.weight[0], need = one > 0.0 ? ceil((goal - (double)before) / one) : (double)count;
            int left = max(1, (int)fmin(fmax(need, 1.0), (double)count));
            for (int j = 0; j < w.n; ++j) {
                const float z = w.z[j * 64 + lane];
                u64 who = __ballot(in(z, j) && key_of(z) == lo);
                const int c = (int)__popcll(who);
                if (left <= c) {
                    for (int k = 1; k < left; ++k) who &= who - 1;
                    return place_of(lo, (unsigned)(j * 64 + (int)__builtin_ctzll(who)));
                }
                left -= c;
            }
        }
        shift = max(0, 26 - (int)__builtin_clz(hi - lo));    // (hi - lo) >> shift < 64
        lds_order();
        s.bin[lane] = 0;
        lds_order();
        for (int j = 0; j < w.n; ++j) {
            const float z = w.z[j * 64 + lane];
            const unsigned key = key_of(z);
            if (in(z, j) && key >= lo && key <= hi) atomicAdd(&s.bin[(hi - key) >> shift], weight(z));
        }
        lds_order();
        bins = s.bin[lane];
    }
}

// Sums over the wave of four values at once: halves, then rows of 16 change places, so that the lanes of row r get value r's
__device__ __forceinline__ void swap_halves(double& a, double& b) {
    const u64 p = (u64)__double_as_longlong(a), q = (u64)__double_as_longlong(b);
    const auto lo = __builtin_amdgcn_permlane32_swap((unsigned)p, (unsigned)q, false, false);
    const auto hi = __builtin_amdgcn_permlane32_swap((unsigned)(p >> 32), (unsigned)(q >> 32), false, false);
    a = __longlong_as_double((long long)((u64)hi[0] << 32 | lo[0]));
    b = __longlong_as_double((long long)((u64)hi[1] << 32 | lo[1]));
}
__device__ __forceinline__ void swap_rows(double& a, double& b) {
    const u64 p = (u64)__double_as_longlong(a), q = (u64)__double_as_longlong(b);
    const auto lo = __builtin_amdgcn_permlane16_swap((unsigned)p, (unsigned)q, false, false);
    const auto hi = __builtin_amdgcn_permlane16_swap((unsigned)(p >> 32), (unsigned)(q >> 32), false, false);
    a = __longlong_as_double((long long)((u64)hi[0] << 32 | lo[0]));
    b = __longlong_as_double((long long)((u64)hi[1] << 32 | lo[1]));
}
__device__ __forceinline__ double row_sums(double v0, double v1, double v2, double v3) {
    swap_halves(v0, v2);
    swap_halves(v1, v3);
    double a = v0 + v2, b = v1 + v3;
    swap_rows(a, b);
    a += b;
    a += dpp_d<DPP_XOR1>(a);
    a += dpp_d<DPP_XOR2>(a);
    a += dpp_d<DPP_HALF_MIRROR>(a);
    return a + dpp_d<DPP_ROW_MIRROR>(a);
}

// A block of up to 64 * (floats of zs / 64) classes.  Its logits stay in LDS: the passes over them are loops of a run-time
// length then, and the compiler keeps no register per slot (with the block in registers the unrolled passes took 232 of them
// and two wavefronts a SIMD).
// `ahead` is called once the logits are there.
template <int DT, int MODE, class Ahead>
__device__ __forceinline__ void choose_wave(const Choice& g, const Block& x, float* zs, WaveLds& s, Chosen& chosen, Ahead ahead) {
    const int lane = threadIdx.x & 63;
    const bool cut_k = MODE != PLAIN && x.top_k > 0 && x.top_k < x.K, cut_p = MODE != PLAIN && x.top_p < 1.0;
    WaveBlock w;
    w.z = zs;
    w.n = (x.K + 63) >> 6;
    float top = -INFINITY;
    unsigned largest = 0;                                    // magnitude, as bits: above infinity's for a NaN
    lds_order();
    float bottom = INFINITY;                                 // above -inf
    auto take = [&](int j, float z) {
        largest = max(largest, __float_as_uint(z) & 0x7fffffffu);
        top = fmaxf(top, z);
        if (MODE != PLAIN) bottom = z == -INFINITY ? bottom : fminf(bottom, z);
        zs[j * 64 + lane] = z;
    };
#pragma unroll 4
    for (int j = 0; j < x.K >> 6; ++j) take(j, load1<DT>(g.z, x.at + j * 64 + lane));
    if (x.K & 63) {
        float z = 0.f;
        const bool is = (x.K & ~63) + lane < x.K;
        if (is) z = load1<DT>(g.z, x.at + (x.K & ~63) + lane);
        largest = max(largest, __float_as_uint(z) & 0x7fffffffu);
        z = is ? z : -INFINITY;
        top = fmaxf(top, z);
        if (MODE != PLAIN) bottom = z == -INFINITY ? bottom : fminf(bottom, z);
        zs[(x.K & ~63) + lane] = z;
    }
    lds_order();
    top = group_max<64>(top);
    ahead();
    if (__any(largest > 0x7f800000u) || x.bad || top == -INFINITY) {
        if (lane == 0) give(g, x.b, x.f, -1, no_number());
        return;
    }
    if (top == INFINITY) {
        for (int j = 0; j < w.n; ++j) zs[j * 64 + lane] = settle(zs[j * 64 + lane], true);
        lds_order();
        top = bottom = 0.f;
    }
    w.top = top;
    w.inv = cut_k || cut_p ? bins_per_unit(top, -group_max<64>(-bottom), x.T, 64.f) : 0.f;
    u64 edge = 0;
    if (cut_k) {
        auto in = [](float z, int) { return z > -INFINITY; };                    // (-inf: no mass, behind every other class)
        auto one = [](float) { return (u64)1; };
        unsigned* const count = reinterpret_cast<unsigned*>(s.bin);
        count[lane] = 0;
        lds_order();
#pragma unroll 2
        for (int j = 0; j < w.n; ++j) {
            const float z = zs[j * 64 + lane];
            if (z > -INFINITY) atomicAdd(&count[linear_bin(z, top, w.inv, 64)], 1u);
        }
        lds_order();
        const unsigned bin = count[lane], run = scan<64>(bin);
        const u64 past = __ballot((int)run >= x.top_k);
        const int at = past ? (int)__builtin_ctzll(past) : 63, n = at_lane((int)run, at);
        if (n <= 64) {
            // few enough for a class a lane: everything else is done there
            int count = 0;
            float zl = -INFINITY;
            // Exactly the classes that were counted into bins up to `at`: where that is the last bin (which has those, too, whose
            // product passes float32: the type's lowest value under an ordinary maximum) or the only one, all above -inf
            const bool all = at == 63 || w.inv == 0.f;
            const float limit = (float)(at + 1);
            lds_order();
#pragma unroll 2
            for (int j = 0; j < w.n; ++j) {
                const float z = zs[j * 64 + lane];
                const bool is = all ? z > -INFINITY : (top - z) * w.inv < limit;
                const u64 who = __ballot(is);
                const int pos = count + (int)__popcll(who & ((1ull << lane) - 1));
                if (is) s.place[pos] = (u64)__float_as_uint(z) << 32 | (unsigned)(j * 64 + lane);
                count += (int)__popcll(who);
            }
            lds_order();
            const u64 mine = s.place[lane];
            if (lane < count) zl = __uint_as_float((unsigned)(mine >> 32));
            choose_lanes<64, MODE>(g, x, zl, lane < count ? key_of(zl) : 0u, (int)(unsigned)mine, top, false, true, &chosen);
            return;
        }
        edge = find_edge(w, (u64)bin, (double)x.top_k, s, in, one);
    }
    auto stays = [&](float z, int j) { return MODE == PLAIN || edge == 0 || place_of(key_of(z), (unsigned)(j * 64 + lane)) >= edge; };
    if (cut_p) {
        const double scale = unit_scale(2048);
        auto in = [&](float z, int j) { return z > -INFINITY && stays(z, j); };
        auto weight = [&](float z) { return units(mass_of(z, top, x.c), scale); };
        const u64 bins = bins_of(w, s, in, weight);
        const u64 to = find_edge(w, bins, x.top_p * (double)at_lane(scan<64>(bins), 63), s, in, weight);
        edge = max(edge, to);
    }
    auto mass = [&](int j) {
        const float z = zs[j * 64 + lane];
        const double a = mass_of(z, top, x.c);
        return (MODE != PLAIN || x.min_p > 0.0) && !(stays(z, j) && a >= x.min_p) ? 0.0 : a;
    };
    // The kept mass of every slot: slot r * q + i goes to lane 16 r + i, so that lanes are in slot order
    const int q = (w.n + 3) >> 2;
    double slot = 0.0;
    for (int i = 0; i < q; ++i) {
        const double v0 = mass(i), v1 = q + i < w.n ? mass(q + i) : 0.0, v2 = 2 * q + i < w.n ? mass(2 * q + i) : 0.0,
                     v3 = 3 * q + i < w.n ? mass(3 * q + i) : 0.0;
        const double sums = row_sums(v0, v1, v2, v3);
        if ((lane & 15) == i) slot = sums;
    }
    const double slots = scan<64>(slot), total = at_lane(slots, 63), goal = x.u * total;
    const u64 with = __ballot(slot > 0.0), over = __ballot(slot > 0.0 && slots > goal);
    const int at = over ? (int)__builtin_ctzll(over) : 63 - (int)__builtin_clzll(with);
    const int j = (at >> 4) * q + (at & 15);
    const double mine = mass(j), run = at_lane(slots - slot, at) + scan<64>(mine);
    const u64 can = __ballot(mine > 0.0), past = __ballot(mine > 0.0 && run > goal);
    const int hit = past ? (int)__builtin_ctzll(past) : 63 - (int)__builtin_clzll(can);
    chosen.add(g, x, j * 64 + hit, at_lane(log2_mass(zs[j * 64 + lane], top, x.c), hit), total);
}

// --------------------------------------------------------------------------------------- any block, any number of classes
// A team of TH threads (a wavefront, or a workgroup) over data that it reads again in every pass: the edge byte by byte of
// the place.  Behind wide blocks whose bins hold too many classes, and for blocks wider than `max_k` said.
struct TeamLds {
    u64 weight[256];
    unsigned count[256];
    u64 part[8];
    u64 out[3];
};
template <int TH> __device__ __forceinline__ void team_sync() {
    if (TH == 64) lds_order();
    else __syncthreads();
}
// Inclusive sums in thread order; `total` gets the last
template <int TH> __device__ __forceinline__ u64 team_scan(u64 v, TeamLds& s, u64& total) {
    u64 run = scan<64>(v);
    if (TH == 64) {
        total = from_lane(run, 63);
        return run;
    }
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 63) s.part[wave] = run;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < TH / 64; ++w) {
        if (w < wave) run += s.part[w];
        total += s.part[w];
    }
    return run;
}
// The place of the first class in order at which `before` + the running weight reaches `goal`; 0 if none does.
// each(f): f(place, weight) for all classes, split over the team.
template <int TH, class Each> __device__ __forceinline__ u64 team_edge(double goal, u64 before, TeamLds& s, Each each) {
    const int t = TH == 64 ? (int)(threadIdx.x & 63) : (int)threadIdx.x;
    u64 prefix = 0, mask = 0;
    for (int shift = 56; shift >= 0; shift -= 8) {
        team_sync<TH>();
        for (int i = t; i < 256; i += TH) { s.weight[i] = 0; s.count[i] = 0; }
        team_sync<TH>();
        each([&](u64 place, u64 w) {
            if ((place & mask) == prefix) {
                const int bin = 255 - (int)(place >> shift & 255);
                atomicAdd(&s.weight[bin], w);
                atomicAdd(&s.count[bin], 1u);
            }
        });
        team_sync<TH>();
        if (t < 64) {
            u64 own[4], sum = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) { own[k] = s.weight[4 * t + k]; sum += own[k]; }
            const u64 run = scan<64>(sum);
            const u64 past = __ballot((double)(before + run) >= goal);
            if (past == 0) {
                if (t == 0) s.out[0] = 256;
            } else if (t == (int)__builtin_ctzll(past)) {
                u64 b = before + run - sum;
                int k = 0;
                while (k < 3 && (double)(b + own[k]) < goal) b += own[k++];
                s.out[0] = (u64)(4 * t + k);
                s.out[1] = b;
            }
        }
        team_sync<TH>();
        if (s.out[0] == 256) return 0;
        before = s.out[1];
        prefix |= (u64)(255 - s.out[0]) << shift;
        mask |= 255ull << shift;
        if (s.count[s.out[0]] == 1 && shift) {
            each([&](u64 place, u64) {
                if ((place & mask) == prefix) s.out[2] = place;
            });
            team_sync<TH>();
            return s.out[2];
        }
    }
    return prefix;
}
// The draw among classes i0 .. i1 of a block, as weights in index order: the first at which `before` + the running weight
// passes `goal` (u == 0: the first with any mass, also one that is under half a unit).  `total`: the kept mass in units.
template <int TH, int DT>
__device__ __forceinline__ void team_draw(const Choice& g, const Block& x, float top, bool inf, u64 edge, double scale, int i0, int i1, u64 before,
                                          u64 goal, u64 total, TeamLds& s) {
    const int t = TH == 64 ? (int)(threadIdx.x & 63) : (int)threadIdx.x;
    const int per = (i1 - i0 + TH - 1) / TH, from = min(i1, i0 + t * per), to = min(i1, from + per);
    auto weight = [&](int i, float z, bool& any) {
        const double a = place_of(key_of(z), (unsigned)i) >= edge ? mass_of(z, top, x.c) : 0.0;
        any = a > 0.0 && a >= x.min_p;
        return any ? x.u == 0.0 ? (u64)1 : units(a, scale) : (u64)0;
    };
    u64 own = 0, all;
    bool any;
    // f(class, weight, logit) for the thread's run, eight loads at a time
    auto run_over = [&](auto f) {
        for (int i = from; i < to; i += 8) {
            float z[8];
            const int n = to - i;
            load8<DT>(g.z, x.at + i, n, z);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < n) {
                    const float v = settle(z[j], inf);
                    f(i + j, weight(i + j, v, any), v);
                }
        }
    };
    run_over([&](int, u64 w, float) { own += w; });
    if (x.u == 0.0) { before = 0; goal = 0; }
    u64 run = before + team_scan<TH>(own, s, all) - own;
    if (own && run <= goal && run + own > goal) {
        int hit = from;
        float z = top;
        run_over([&](int i, u64 w, float v) {
            if (w && run <= goal) { hit = i; z = v; }
            run += w;
        });
        give(g, x.b, x.f, hit, (float)(log2_mass(z, top, x.c) * LN2 - log_from1((double)total / scale)));
    }
}
template <int TH, int DT> __device__ void choose_team(const Choice& g, const Block& x, TeamLds& s) {
    const int t = TH == 64 ? (int)(threadIdx.x & 63) : (int)threadIdx.x;
    float top = -INFINITY;
    u64 bad = 0;
    for (int i = t; i < x.K; i += TH) {
        const float z = load1<DT>(g.z, x.at + i);
        bad += z != z;
        top = fmaxf(top, z);
    }
    u64 nan;
    team_scan<TH>(bad, s, nan);
    team_sync<TH>();
    top = group_max<64>(top);
    if (TH > 64) {
        if ((t & 63) == 0) s.part[t >> 6] = __float_as_uint(top);
        __syncthreads();
#pragma unroll
        for (int w = 0; w < TH / 64; ++w) top = fmaxf(top, __uint_as_float((unsigned)s.part[w]));
        __syncthreads();
    }
    if (nan || x.bad || top == -INFINITY) {
        if (t == 0) give(g, x.b, x.f, -1, no_number());
        return;
    }
    const bool inf = top == INFINITY;
    if (inf) top = 0.f;
    auto z_at = [&](int i) { return settle(load1<DT>(g.z, x.at + i), inf); };
    const double scale = unit_scale(x.K);
    u64 edge = 0;
    if (x.top_k > 0 && x.top_k < x.K)
        edge = team_edge<TH>((double)x.top_k, 0, s, [&](auto f) {
            for (int i = t; i < x.K; i += TH) {
                const float z = z_at(i);
                if (z > -INFINITY) f(place_of(key_of(z), (unsigned)i), 1);
            }
        });
    u64 sum = 0, total;
    for (int i = t; i < x.K; i += TH) {
        const float z = z_at(i);
        if (place_of(key_of(z), (unsigned)i) >= edge) sum += units(mass_of(z, top, x.c), scale);
    }
    team_scan<TH>(sum, s, total);
    if (x.top_p < 1.0) {
        const u64 to = team_edge<TH>(x.top_p * (double)total, 0, s, [&](auto f) {
            for (int i = t; i < x.K; i += TH) {
                const float z = z_at(i);
                const u64 place = place_of(key_of(z), (unsigned)i);
                if (place >= edge) f(place, units(mass_of(z, top, x.c), scale));
            }
        });
        edge = max(edge, to);
    }
    if (x.top_p < 1.0 || x.min_p > 0.0) {
        sum = 0;
        for (int i = t; i < x.K; i += TH) {
            const float z = z_at(i);
            const double a = place_of(key_of(z), (unsigned)i) >= edge ? mass_of(z, top, x.c) : 0.0;
            if (a >= x.min_p) sum += units(a, scale);
        }
        team_scan<TH>(sum, s, total);
    }
    team_draw<TH, DT>(g, x, top, inf, edge, scale, 0, x.K, 0, draw_goal(x.u, total), total, s);
}

// ----------------------------------------------------------------------------------- rows of features, block by block
constexpr int WAVES = 4;
template <int NV> union WaveMemory {
    struct {
        WaveLds lds;
        float z[NV * 64];
    } wave;
    TeamLds team;
};

// The items of a wavefront: a run of neighbouring ones, or, where there are fewer items than wavefronts, at most one, behind
// the `before` ones that other kinds of items have given to the first wavefronts (1 row of 50 columns: no wavefront has two)
__device__ __forceinline__ void items_of(unsigned items, unsigned before, unsigned wave, unsigned waves, unsigned& from, unsigned& to) {
    if (items >= waves) {
        from = (unsigned)((u64)items * wave / waves);
        to = (unsigned)((u64)items * (wave + 1) / waves);
    } else {
        from = (wave + waves - before % waves) % waves;
        to = min(from + 1, items);
    }
}
// Blocks of at most G classes, 64 / G of one row at a time; returns the number of items
template <int DT, int G, int MODE>
__device__ __forceinline__ unsigned choose_narrow(const Choice& g, const int* perm, const int* off, int n, unsigned before, unsigned wave, unsigned waves) {
    if (n == 0) return 0;
    constexpr unsigned PER = 64 / G;
    const int lane = threadIdx.x & 63, l = lane & (G - 1);
    const unsigned per_row = ((unsigned)n + PER - 1) / PER, items = per_row * (unsigned)g.B;
    unsigned i0, i1;
    items_of(items, before, wave, waves, i0, i1);
    unsigned b = i0 / per_row, w = i0 - b * per_row;
    for (unsigned it = i0; it < i1; ++it) {
        const int slot = (int)(w * PER) + lane / G;
        const bool live = slot < n;
        const int f = perm[live ? slot : n - 1], k0 = off[f], K = max(0, off[f + 1] - k0);
        const Block x = block_of<MODE>(g, (int)b, f, k0, K);
        const float z = l < K ? load1<DT>(g.z, x.at + l) : -INFINITY;
        const u64 group = ((G == 64 ? 0ull : 1ull << (G & 63)) - 1) << (lane & ~(G - 1));
        const bool nan = (__ballot(z != z) & group) != 0;
        choose_lanes<G, MODE>(g, x, z, l < K ? key_of(z) : 0u, l, group_max<G>(z), nan, live, nullptr);
        if (++w == per_row) { w = 0; ++b; }
    }
    return items;
}

// A wavefront takes blocks of one width class after another: narrow ones share it, others have it to themselves.  Five of them a
// SIMD (NV = 16): the waits of one are the others' work (20000 x 50 filtered, five / six / seven: 795 / 842 / 894 us, six and seven
// spill; of an earlier state, four / five: 1111 / 960).
template <int DT, int NV, int MODE> __global__ void __launch_bounds__(WAVES * 64, NV == 16 ? 5 : 4) choose_kernel(Choice g) {
    extern __shared__ int s_tables[];                         // of up to MAX_LDS_FEATURES features: offsets, order
    __shared__ int s_start[5];
    __shared__ WaveMemory<NV> s_mem[WAVES];
    const bool order = g.m <= MAX_LDS_FEATURES;
    int *s_off = s_tables, *s_perm = s_tables + g.m + 1;
    if (order) {
        for (int i = threadIdx.x; i <= g.m; i += WAVES * 64)
            s_off[i] = g.offsets ? max(0, min(g.offsets[i], g.sumK)) : i ? g.sumK : 0;
        __syncthreads();
        order_features_by_width(g.m, s_off, s_perm, s_start);
    }
    const unsigned wave = blockIdx.x * WAVES + (threadIdx.x >> 6), waves = gridDim.x * WAVES;
    WaveMemory<NV>& mem = s_mem[threadIdx.x >> 6];
    unsigned before = 0;
    if (order) {
        before += choose_narrow<DT, 8, MODE>(g, s_perm, s_off, s_start[1], before, wave, waves);
        before += choose_narrow<DT, 16, MODE>(g, s_perm + s_start[1], s_off, s_start[2] - s_start[1], before, wave, waves);
        before += choose_narrow<DT, 32, MODE>(g, s_perm + s_start[2], s_off, s_start[3] - s_start[2], before, wave, waves);
    }
    const unsigned first = order ? (unsigned)s_start[3] : 0u, n = (unsigned)g.m - first;
    if (n == 0) return;
    unsigned i0, i1;
    items_of(n * (unsigned)g.B, before, wave, waves, i0, i1);
    unsigned b = i0 / n, w = i0 - b * n;
    const int lane = threadIdx.x & 63;
    Chosen chosen = {};
    for (unsigned it = i0; it < i1; ++it) {
        const int row = __builtin_amdgcn_readfirstlane((int)b);
        const int f = __builtin_amdgcn_readfirstlane(order ? s_perm[first + w] : (int)w);
        const int k0 = __builtin_amdgcn_readfirstlane(order ? s_off[f] : first_of(g, f));
        const int K = __builtin_amdgcn_readfirstlane(order ? max(0, s_off[f + 1] - k0) : classes_of(g, f));
        if (++w == n) { w = 0; ++b; }
        // A lane a 64-byte piece of the row from the next block on: its lines are on their way while this one is worked on
        // (20000 x 50 filtered, then 960, 890 us; to the end of a block as wide as this one 920; the next logits and uniforms kept
        // in registers 1240, from 48 of them spilled)
        float touched = 0.f;
        auto ahead = [&] {
            if (!order || it + 1 == i1) return;
            const int at = __builtin_amdgcn_readfirstlane(s_off[s_perm[first + w]]) + lane * (DT == CLAVA_DT_F32 ? 16 : 32);
            if (at < g.sumK) touched = load1<DT>(g.z, (size_t)b * g.ld + at);
        };
        if (!g.wide || K <= g.wide_from || K > g.wide_to) {
            const Block x = block_of<MODE>(g, row, f, k0, K);
            if (K <= 64) {
                const float z = lane < K ? load1<DT>(g.z, x.at + lane) : -INFINITY;
                choose_lanes<64, MODE>(g, x, z, lane < K ? key_of(z) : 0u, lane, group_max<64>(z), __any(z != z), true, &chosen);
            } else if (K <= NV * 64) {
                choose_wave<DT, MODE>(g, x, mem.wave.z, mem.wave.lds, chosen, ahead);
            } else {
                choose_team<64, DT>(g, x, mem.team);
            }
        }
        asm volatile("" : : "v"(touched));
    }
    chosen.flush(g);
}

// ------------------------------------------------------------------------------------------- very many classes, in chunks
// Four launches over chunks of a block (top -> bins -> collect) and over blocks (finish).  Weights are integers, so that the
// sums over chunks have no order.  64 x 131071 bfloat16 with top-p: 7.0 + 16.4 + 13.1 + 16.5 us; reading it once takes 3.6.  Vector
// instructions issue for 3, 9 and 7 us of the first three (half of the second's are its 8.4 million masses); the rest is the
// latency of the head, of a few dependent loads and of workgroup sums, and so is nearly all of the last (64 workgroups) and of
// all four of 1 x 262144 with top-k (3.2 + 7.4 + 6.5 + 9.3).  Where more than WIDE_LIST classes share the edges' bins - logits that
// are equal, or nearly - one workgroup goes over the whole block: 64 x 131071 equal ones take 2150 us instead of 52, 256 x 50257
// 1030 instead of 67.  Between the launches, for every wide block and in `ws`:
constexpr int WT = 256, WIDE_BINS = 256, WIDE_LIST = 4096, WIDE_CHUNKS = 1024;
struct Wide {
    char* ws;
    int chunk, chunks;                        // classes of a chunk, chunks of the widest block
    int per_row;                              // wide blocks a row can have
    long long stride;                         // bytes of a block
    bool k, p;                                // some block may have top-k / top-p
};
struct WideWs {
    unsigned* listed;                         // places in the list
    u64* mass;                                // [WIDE_BINS]
    u64* chunk_mass;                          // [chunks][WIDE_BINS]
    unsigned* count;                          // [WIDE_BINS] classes
    u64* list;                                // [WIDE_LIST] places in the edges' bins
    u64* sum;                                 // [chunks] mass that is kept whatever the edge's bin yields
    float* range;                             // [chunks][2] largest and smallest logit above -inf (NaN: the chunk holds one)
    unsigned* any;                            // [chunks] classes with such mass
};
long long wide_bytes(int chunks) { return 16 + 12LL * WIDE_BINS + 8LL * WIDE_LIST + 24LL * chunks + 8LL * WIDE_BINS * chunks; }
__device__ __forceinline__ WideWs wide_ws(const Wide& w, long long block) {
    char* p = w.ws + block * w.stride;
    WideWs s;
    s.listed = (unsigned*)p; p += 16;
    s.mass = (u64*)p; p += 8LL * WIDE_BINS;
    s.count = (unsigned*)p; p += 4LL * WIDE_BINS;
    s.list = (u64*)p; p += 8LL * WIDE_LIST;
    s.sum = (u64*)p; p += 8LL * w.chunks;
    s.chunk_mass = (u64*)p; p += 8LL * WIDE_BINS * w.chunks;
    s.range = (float*)p; p += 8LL * w.chunks;
    s.any = (unsigned*)p;
    return s;
}
// The n-th wide feature, or -1 (`s_n[0]`; ALL: and how many there are, `s_n[1]`).  Every thread of the workgroup calls it.
template <bool ALL = false> __device__ __forceinline__ int wide_feature(const Choice& g, int n, int* s_n) {
    if (g.m == 1) return n == 0 && classes_of(g, 0) > g.wide_from ? 0 : -1;
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x;
        int found = -1, before = 0;
        for (int f0 = 0; f0 < g.m && (ALL || found < 0); f0 += 64) {
            const int K = classes_of(g, min(f0 + lane, g.m - 1));
            u64 who = __ballot(f0 + lane < g.m && K > g.wide_from && K <= g.wide_to);
            const int c = (int)__popcll(who);
            if (found < 0 && n - before < c) {
                for (int k = before; k < n; ++k) who &= who - 1;
                found = f0 + (int)__builtin_ctzll(who);
            }
            before += c;
        }
        if (lane == 0) {
            s_n[0] = found;
            if (ALL) s_n[1] = before;
        }
    }
    __syncthreads();
    return s_n[0];
}
struct WideBlock {
    Block x;
    WideWs s;
    int chunks;                               // of this block
    float top;
    bool none, inf;
    double scale;
    float inv;
};
template <bool ALL = false> __device__ __forceinline__ bool wide_block(const Choice& g, const Wide& w, long long block, WideBlock& o, int* s_n) {
    const int b = (int)(block / w.per_row);
    const int f = wide_feature<ALL>(g, (int)(block - (long long)b * w.per_row), s_n);
    if (f < 0) return false;
    o.x = block_of<TENSORS>(g, b, f, first_of(g, f), classes_of(g, f));
    o.s = wide_ws(w, block);
    o.chunks = (o.x.K + w.chunk - 1) / w.chunk;
    o.scale = unit_scale(o.x.K);
    return true;
}
__device__ __forceinline__ int wide_bin(const WideBlock& o, float z) {
    return linear_bin(z, o.top, o.inv, WIDE_BINS);
}

// f(first class, logits) for the classes from .. to, eight neighbouring ones a thread; -inf where there are fewer
template <int DT, class F> __device__ __forceinline__ void wide_each(const Choice& g, const Block& x, int from, int to, F f) {
    for (int i = from + (int)threadIdx.x * 8; i < to; i += WT * 8) {
        float z[8];
        const int n = to - i;
        load8<DT>(g.z, x.at + i, n, z);
        if (n < 8)
#pragma unroll
            for (int j = 0; j < 8; ++j) z[j] = j < n ? z[j] : -INFINITY;
        f(i, z);
    }
}

// Blocks whose top-k fits well into the list: every class up to its bin is listed, and the rest is done there, so that no other
// class needs its mass (256 x 50257 with top-k and top-p: 75.5 -> 60.4 us)
__device__ __forceinline__ bool cuts_k(const Block& x) { return x.top_k > 0 && x.top_k < x.K; }
__device__ __forceinline__ bool few_k(const Block& x) { return cuts_k(x) && x.top_k <= WIDE_LIST / 4; }

// Which bins the edges fall into.  Top-k's is exact; the mass that top-k leaves is known up to its bin, so top-p's goal is one
// of a range, and its bin too.
struct Cut {
    int k_from, k_bin;                        // the bins that are listed for top-k, and the last one, its edge's; WIDE_BINS: none
    u64 k_before;                             // classes in the bins before these
    u64 m_before;                             // mass in the bins before top-k's; without one all of it
    int p_from, p_to;                         // bins that top-p's edge can fall into; p_from > p_to: none
    int sure;                                 // the bins before this one are kept
};
// What every workgroup of a block has to know of it before it starts.  One wavefront finds it, four bins a lane, and the
// others wait at one barrier (with scans over the workgroup instead, and a barrier or two for each, `collect` took 18.4 us for 17.0).
struct WideHead {
    float top, bottom;
    int nan;
    Cut cut;
};
template <bool CUT> __device__ __forceinline__ void wide_head(const WideBlock& o, WideHead& h, u64* s_mass) {
    if (threadIdx.x >= 64) return;
    const int lane = threadIdx.x;
    const bool k = CUT && cuts_k(o.x), few = CUT && few_k(o.x), p = CUT && o.x.top_p < 1.0 && !few;
    u64 count[4], mass[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        count[i] = k ? o.s.count[4 * lane + i] : 0;
        mass[i] = p ? o.s.mass[4 * lane + i] : 0;
    }
    float top = -INFINITY, bottom = INFINITY;
    bool nan = false;
    for (int i = lane; i < o.chunks; i += 64) {
        const float hi = o.s.range[2 * i], lo = o.s.range[2 * i + 1];
        nan |= hi != hi;
        top = fmaxf(top, hi);
        bottom = fminf(bottom, lo);
    }
    top = group_max<64>(top);
    bottom = -group_max<64>(-bottom);
    nan = __any(nan);
    Cut c = {WIDE_BINS, WIDE_BINS, 0, 0, 0, -1, WIDE_BINS};
    if (CUT) {
        // running sums, up to and with each bin of the lane
#pragma unroll
        for (int i = 1; i < 4; ++i) { count[i] += count[i - 1]; mass[i] += mass[i - 1]; }
        const u64 c0 = scan<64>(count[3]) - count[3], m0 = scan<64>(mass[3]) - mass[3];
#pragma unroll
        for (int i = 0; i < 4; ++i) { count[i] += c0; mass[i] += m0; }
        const u64 total = at_lane(mass[3], 63);
        if (s_mass)
#pragma unroll
            for (int i = 0; i < 4; ++i) s_mass[4 * lane + i] = mass[i];
        // the first bin whose running sum reaches a goal, and the sum before it and with it
        auto value = [](const u64* v, int i) { return i == 0 ? v[0] : i == 1 ? v[1] : i == 2 ? v[2] : v[3]; };
        auto first = [&](const u64* v, double goal) {
            const u64 past = __ballot((double)v[3] >= goal);
            const int i = ((double)v[0] < goal) + ((double)v[1] < goal) + ((double)v[2] < goal), at = past ? (int)__builtin_ctzll(past) : 0;
            return past ? 4 * at + at_lane(i, at) : -1;
        };
        auto upto = [&](const u64* v, int bin) { return bin < 0 ? (u64)0 : at_lane(value(v, bin & 3), bin >> 2); };
        u64 m_with = total;
        c.m_before = total;
        const int bin = k ? first(count, (double)o.x.top_k) : -1;
        if (few) c = Cut{0, bin < 0 ? WIDE_BINS - 1 : bin, 0, 0, 0, -1, 0};      // (fewer classes than top-k: all of them)
        else if (bin >= 0) {
            m_with = upto(mass, bin);
            c = Cut{bin, bin, upto(count, bin - 1), upto(mass, bin - 1), 0, -1, bin};
        }
        if (p) {
            c.p_from = first(mass, o.x.top_p * (double)c.m_before);
            c.p_to = first(mass, o.x.top_p * (double)m_with);
            c.sure = min(c.sure, c.p_from);
        }
    }
    if (lane == 0) h = WideHead{top, bottom, nan, c};
}
__device__ __forceinline__ void wide_look(WideBlock& o, const WideHead& h) {
    o.inf = h.top == INFINITY;
    o.top = o.inf ? 0.f : h.top;
    o.none = h.nan || o.x.bad || h.top == -INFINITY;
    o.inv = bins_per_unit(h.top, h.bottom, o.x.T, (float)WIDE_BINS);
}

template <int DT> __global__ void __launch_bounds__(WT) wide_top_kernel(Choice g, Wide w) {
    __shared__ int s_n[2];
    __shared__ TeamLds s_t;
    WideBlock o;
    if (!wide_block<true>(g, w, blockIdx.y, o, s_n)) return;
    const int c = blockIdx.x, t = threadIdx.x;
    // Features that overlap (offsets that fall in between) can be more wide ones than a row has room for side by side: nobody
    // draws those that are left, and the last one's first workgroup says so
    if (c == 0 && g.m > w.per_row && (int)(blockIdx.y % (unsigned)w.per_row) == w.per_row - 1) {
        const int wide = s_n[1];
        for (int n = w.per_row; n < wide; ++n) {
            __syncthreads();
            const int f = wide_feature(g, n, s_n);
            if (t == 0) give(g, o.x.b, f, -1, no_number());
        }
    }
    if (c == 0 && (w.k || w.p)) {
        if (t == 0) *o.s.listed = 0;
        o.s.mass[t] = 0;
        o.s.count[t] = 0;
    }
    if (c >= o.chunks) return;
    float top = -INFINITY, bottom = INFINITY;
    bool nan = false;
    const int to = min(o.x.K, (c + 1) * w.chunk);
    wide_each<DT>(g, o.x, c * w.chunk, to, [&](int, const float* z) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            nan |= z[j] != z[j];
            top = fmaxf(top, z[j]);
            bottom = z[j] == -INFINITY ? bottom : fminf(bottom, z[j]);
        }
    });
    top = group_max<64>(top);
    bottom = -group_max<64>(-bottom);
    if (__any(nan)) top = no_number();
    if ((t & 63) == 0) s_t.part[t >> 6] = (u64)__float_as_uint(top) << 32 | __float_as_uint(bottom);
    __syncthreads();
    if (t == 0) {
        for (int i = 1; i < WT / 64; ++i) {
            const float v = __uint_as_float((unsigned)(s_t.part[i] >> 32));
            top = top != top || v != v ? no_number() : fmaxf(top, v);
            bottom = fminf(bottom, __uint_as_float((unsigned)s_t.part[i]));
        }
        o.s.range[2 * c] = top;
        o.s.range[2 * c + 1] = bottom;
    }
}

template <int DT> __global__ void __launch_bounds__(WT) wide_bins_kernel(Choice g, Wide w) {
    __shared__ int s_n;
    __shared__ TeamLds s_t;
    __shared__ WideHead s_head;
    WideBlock o;
    if (!wide_block(g, w, blockIdx.y, o, &s_n)) return;
    const int c = blockIdx.x, t = threadIdx.x;
    if (c >= o.chunks) return;
    s_t.weight[t] = 0;
    s_t.count[t] = 0;
    wide_head<false>(o, s_head, nullptr);
    __syncthreads();
    wide_look(o, s_head);
    if (o.none) return;
    const int to = min(o.x.K, (c + 1) * w.chunk);
    const bool count = cuts_k(o.x), mass = o.x.top_p < 1.0 && !few_k(o.x);
    wide_each<DT>(g, o.x, c * w.chunk, to, [&](int, const float* v) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float z = settle(v[j], o.inf);
            if (z > -INFINITY) {
                const int bin = wide_bin(o, z);
                if (mass) atomicAdd(&s_t.weight[bin], units(mass_of(z, o.top, o.x.c), o.scale));
                if (count) atomicAdd(&s_t.count[bin], 1u);
            }
        }
    });
    __syncthreads();
    if (s_t.weight[t]) atomicAdd(&o.s.mass[t], s_t.weight[t]);
    if (mass) o.s.chunk_mass[c * WIDE_BINS + t] = s_t.weight[t];
    if (s_t.count[t]) atomicAdd(&o.s.count[t], s_t.count[t]);
}

// Whether a chunk's kept mass follows from its bins: then `collect` takes no exponentials (64 x 131071: 23 us with
// them, 18 without).  Not where min-p cuts inside a bin, nor for u = 0, which counts classes.
__device__ __forceinline__ bool mass_is_binned(const Block& x) { return x.top_p < 1.0 && x.min_p == 0.0 && x.u > 0.0 && !few_k(x); }

template <int DT> __global__ void __launch_bounds__(WT) wide_collect_kernel(Choice g, Wide w) {
    __shared__ int s_n;
    __shared__ WideHead s_head;
    __shared__ u64 s_list[1024], s_sum, s_any;
    __shared__ unsigned s_listed, s_base;
    WideBlock o;
    if (!wide_block(g, w, blockIdx.y, o, &s_n)) return;
    const int c = blockIdx.x, t = threadIdx.x;
    if (c >= o.chunks) return;
    if (t == 0) { s_listed = 0; s_sum = 0; s_any = 0; }
    const bool binned = mass_is_binned(o.x);
    const u64 chunk_mass = binned ? o.s.chunk_mass[c * WIDE_BINS + t] : 0;
    wide_head<true>(o, s_head, nullptr);
    __syncthreads();
    wide_look(o, s_head);
    if (o.none) return;
    const Cut cut = s_head.cut;
    const int to = min(o.x.K, (c + 1) * w.chunk);
    u64 sum = 0, any = 0;
    // (a class's bin is not cut to an integer here: it is compared with the ends of the listed ones)
    const float k_from = (float)cut.k_from, k_end = (float)(cut.k_bin + 1), p_from = (float)cut.p_from, p_end = (float)(cut.p_to + 1),
                sure = (float)cut.sure;
    wide_each<DT>(g, o.x, c * w.chunk, to, [&](int i, const float* v) {
        unsigned which = 0;
        float z[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            z[j] = settle(v[j], o.inf);
            const float bin = z[j] == -INFINITY ? INFINITY : o.inv > 0.f ? fminf((o.top - z[j]) * o.inv, (float)(WIDE_BINS - 1)) : 0.f;
            const bool is = (bin >= k_from && bin < k_end) || (bin >= p_from && bin < p_end);
            which |= is ? 1u << j : 0u;
            if (!binned && !is && bin < sure) {
                const double a = mass_of(z[j], o.top, o.x.c);
                if (a >= o.x.min_p) { sum += units(a, o.scale); any += a > 0.0; }
            }
        }
        if (which == 0) return;
        unsigned at = atomicAdd(&s_listed, (unsigned)__popc(which));
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (which >> j & 1) {
                const u64 place = place_of(key_of(z[j]), (unsigned)(i + j));
                if (at < 1024) s_list[at] = place;
                else {                                        // more than a chunk usually has
                    const unsigned far = atomicAdd(o.s.listed, 1u);
                    if (far < WIDE_LIST) o.s.list[far] = place;
                }
                ++at;
            }
    });
    if (binned) sum = t < cut.sure ? chunk_mass : 0;
    sum = scan<64>(sum);
    if ((t & 63) == 63 && sum) atomicAdd(&s_sum, sum);
    if (o.x.u == 0.0) {
        any = scan<64>(any);
        if ((t & 63) == 63 && any) atomicAdd(&s_any, any);
    }
    __syncthreads();
    const unsigned n = min(s_listed, 1024u);
    if (t == 0) {
        o.s.sum[c] = s_sum;
        o.s.any[c] = (unsigned)s_any;
        if (n) s_base = atomicAdd(o.s.listed, n);
    }
    if (n == 0) return;
    __syncthreads();
    for (unsigned i = t; i < n; i += WT)
        if (s_base + i < WIDE_LIST) o.s.list[s_base + i] = s_list[i];
}

// The place of the first of the listed classes with in(place), in order, at which `before` + the running weight reaches `goal`;
// 0 if none does.  The list's range of places is cut into 256 until at most 64 are left in one.
template <class In, class Weight>
__device__ __forceinline__ u64 list_edge(const u64* list, int n, double goal, u64 before, TeamLds& s, In in, Weight weight) {
    const int t = threadIdx.x, lane = t & 63;
    u64 lo = 0, hi = ~0ull;
    for (;;) {
        u64 first = ~0ull, last = 0, own = 0, count;
        for (int i = t; i < n; i += WT) {
            const u64 p = list[i];
            if (p < lo || p > hi || !in(p)) continue;
            first = min(first, p);
            last = max(last, p);
            ++own;
        }
        const u64 at = team_scan<WT>(own, s, count) - own;
        if (count == 0) return 0;
        if (count <= 64) {
            // one wavefront puts them in order
            int pos = (int)at;
            for (int i = t; i < n; i += WT) {
                const u64 p = list[i];
                if (p >= lo && p <= hi && in(p)) s.weight[pos++] = p;
            }
            __syncthreads();
            if (t < 64) {
                const u64 p = sort_falling<64>(lane < (int)count ? s.weight[lane] : 0), sum = scan<64>(lane < (int)count ? weight(p) : (u64)0);
                const u64 there = __ballot(lane < (int)count && (double)(before + sum) >= goal);
                const u64 edge = at_lane(p, there ? (int)__builtin_ctzll(there) : (int)count - 1);
                if (lane == 0) s.out[2] = edge;
            }
            __syncthreads();
            return s.out[2];
        }
#pragma unroll
        for (int o = 32; o; o >>= 1) {
            first = min(first, from_xor(first, o));
            last = max(last, from_xor(last, o));
        }
        __syncthreads();
        if (lane == 0) { s.part[t >> 6] = first; s.part[WT / 64 + (t >> 6)] = last; }
        s.weight[t] = 0;
        __syncthreads();
        lo = s.part[0];
        hi = s.part[WT / 64];
#pragma unroll
        for (int w = 1; w < WT / 64; ++w) { lo = min(lo, s.part[w]); hi = max(hi, s.part[WT / 64 + w]); }
        const int shift = max(0, 56 - (int)__builtin_clzll(hi - lo));           // (places differ: hi > lo)
        for (int i = t; i < n; i += WT) {
            const u64 p = list[i];
            if (p >= lo && p <= hi && in(p)) atomicAdd(&s.weight[(hi - p) >> shift], weight(p));
        }
        __syncthreads();
        const u64 bin = s.weight[t];
        u64 all;
        const u64 run = before + team_scan<WT>(bin, s, all);
        if (t == 0) s.out[0] = 256;
        __syncthreads();
        if ((double)run >= goal && (t == 0 || (double)(run - bin) < goal)) { s.out[0] = (u64)t; s.out[1] = run - bin; }
        __syncthreads();
        if (s.out[0] == 256) return 0;
        before = s.out[1];
        const u64 top = hi - (s.out[0] << shift);
        lo = max(lo, top - ((1ull << shift) - 1));
        hi = top;
        __syncthreads();
    }
}

template <int DT> __global__ void __launch_bounds__(WT) wide_finish_kernel(Choice g, Wide w) {
    __shared__ int s_n;
    __shared__ TeamLds s_t;
    __shared__ u64 s_mass[WIDE_BINS];
    __shared__ WideHead s_head;
    __shared__ u64 s_sum[WIDE_CHUNKS];
    __shared__ u64 s_list[WIDE_LIST];
    __shared__ int s_chunk;
    __shared__ u64 s_before;
    WideBlock o;
    if (!wide_block(g, w, blockIdx.x, o, &s_n)) return;
    const int t = threadIdx.x;
    wide_head<true>(o, s_head, s_mass);
    __syncthreads();
    wide_look(o, s_head);
    if (o.none) {
        if (t == 0) give(g, o.x.b, o.x.f, -1, no_number());
        return;
    }
    const Cut cut = s_head.cut;
    const unsigned listed = w.k || w.p ? *o.s.listed : 0;
    if (listed > WIDE_LIST) {                                 // too many classes in the edges' bins
        choose_team<WT, DT>(g, o.x, s_t);
        return;
    }
    const int n = (int)listed;
    for (int i = t; i < n; i += WT) s_list[i] = o.s.list[i];
    __syncthreads();
    auto z_of = [&](u64 place) {
        const unsigned key = (unsigned)(place >> 32);
        return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
    };
    auto weight = [&](u64 place) { return units(mass_of(z_of(place), o.top, o.x.c), o.scale); };
    u64 edge = 0;
    u64 k_mass = cut.m_before;
    const bool few = few_k(o.x);
    if (cut.k_bin < WIDE_BINS) {
        edge = list_edge(s_list, n, (double)o.x.top_k, cut.k_before, s_t, [&](u64 p) {
            const int bin = wide_bin(o, z_of(p));
            return bin >= cut.k_from && bin <= cut.k_bin;
        }, [](u64) { return (u64)1; });
        if (cut.p_from <= cut.p_to || few) {
            u64 own = 0, sum;
            for (int i = t; i < n; i += WT) {
                const int bin = wide_bin(o, z_of(s_list[i]));
                if (bin >= cut.k_from && bin <= cut.k_bin && s_list[i] >= edge) own += weight(s_list[i]);
            }
            team_scan<WT>(own, s_t, sum);
            k_mass = few ? sum : k_mass + sum;
        }
    }
    if (few && o.x.top_p < 1.0) {
        const u64 least = edge;
        edge = max(edge, list_edge(s_list, n, o.x.top_p * (double)k_mass, 0, s_t, [&](u64 p) { return p >= least; }, weight));
    } else if (cut.p_from <= cut.p_to) {
        const u64 least = edge;
        const u64 to = list_edge(s_list, n, o.x.top_p * (double)k_mass, cut.p_from ? s_mass[cut.p_from - 1] : 0, s_t, [&](u64 p) {
            const int bin = wide_bin(o, z_of(p));
            return bin >= cut.p_from && bin <= cut.p_to && p >= least;
        }, weight);
        edge = max(edge, to);
    }
    // the kept mass of every chunk
    u64 mass = 0;
    for (int c = t; c < o.chunks; c += WT) {
        const u64 m = o.s.sum[c];
        s_sum[c] = o.x.u == 0.0 ? (u64)o.s.any[c] : m;
        mass += m;
    }
    __syncthreads();
    for (int i = t; i < n; i += WT) {
        const u64 place = s_list[i];
        if (place < edge) continue;
        const double a = mass_of(z_of(place), o.top, o.x.c);
        if (a >= o.x.min_p && a > 0.0) {
            const u64 m = units(a, o.scale);
            mass += m;
            atomicAdd(&s_sum[(unsigned)~(unsigned)place / (unsigned)w.chunk], o.x.u == 0.0 ? (u64)1 : m);
        }
    }
    u64 total, all;
    team_scan<WT>(mass, s_t, total);
    __syncthreads();
    // the chunk in which the running mass passes the goal
    const int per = (o.chunks + WT - 1) / WT, c0 = min(o.chunks, t * per), c1 = min(o.chunks, c0 + per);
    u64 own = 0;
    for (int c = c0; c < c1; ++c) own += s_sum[c];
    u64 run = team_scan<WT>(own, s_t, all) - own;
    const u64 goal = draw_goal(o.x.u, all);
    if (own && run <= goal && run + own > goal) {
        int c = c0;
        while (c < c1 - 1 && run + s_sum[c] <= goal) run += s_sum[c++];
        s_chunk = c;
        s_before = run;
    }
    __syncthreads();
    team_draw<WT, DT>(g, o.x, o.top, o.inf, edge, o.scale, s_chunk * w.chunk, min(o.x.K, (s_chunk + 1) * w.chunk), s_before, goal, total, s_t);
}

// Classes of a chunk: 4096, or 2048 where that leaves the chip without work; more where there would be too many chunks (64 x
// 131071, 2048 / 4096 / 8192 / 16384 classes: 75 / 64 / 65 / 81 us)
int wide_chunk(int B, int K) {
    const int c = (K + WIDE_CHUNKS - 1) / WIDE_CHUNKS, usual = (long long)B * ((K + 4095) / 4096) < 512 ? 2048 : 4096;
    return c > usual ? c : usual;
}
constexpr int NARROW_MAX = 2048;              // classes that a wavefront keeps in LDS
int wide_per_row(int m, int sumK) {
    const int most = sumK / (NARROW_MAX + 1);
    return most < m ? most : m;
}
// The widest block that the wide kernels take, and have workspace for: wider ones than the caller said are a wavefront's
int wide_most(int m, int sumK, int max_k) { return m == 1 || max_k > sumK ? sumK : max_k; }
// Rows of one launch: 1024 wide blocks fill the chip, and the workspace need not hold more
int wide_rows(int per_row) { return per_row < 1024 ? 1024 / per_row : 1; }
bool filters_k(const clava_choice* c) { return c->top_k_t || c->top_k > 0 || c->temperature_t || c->temperature < 1e-290; }
bool filters_p(const clava_choice* c) { return c->top_p_t || c->top_p < 1.0; }

template <int DT> int launch_choice(Choice& g, Wide& w, int max_k, int mode, hipStream_t st) {
    const unsigned blocks = (unsigned)g.B * (unsigned)g.m;
    if (g.wide_from >= 0) {
        const unsigned grid = (blocks + WAVES - 1) / WAVES < 256 * 5 ? (blocks + WAVES - 1) / WAVES : 256 * 5;
        const int lds = g.m <= MAX_LDS_FEATURES ? (2 * g.m + 1) * 4 : 0;
        auto* const kernel = mode == PLAIN ? (max_k <= 1024 ? choose_kernel<DT, 16, PLAIN> : choose_kernel<DT, 32, PLAIN>)
                             : mode == FILTERED ? (max_k <= 1024 ? choose_kernel<DT, 16, FILTERED> : choose_kernel<DT, 32, FILTERED>)
                                                : (max_k <= 1024 ? choose_kernel<DT, 16, TENSORS> : choose_kernel<DT, 32, TENSORS>);
        kernel<<<grid, WAVES * 64, lds, st>>>(g);
        CLAVA_CHECK_LAUNCH("sample_categories");
    }
    if (g.wide) {
        const int rows = wide_rows(w.per_row);
        for (long long row = 0; row < g.B; row += rows) {
            Choice h = g;                                     // the rows of this launch
            h.z = (const char*)g.z + (size_t)row * g.ld * (DT == CLAVA_DT_F32 ? 4 : 2);
            h.B = (int)(g.B - row < rows ? g.B - row : rows);
            h.u = g.u ? g.u + row * g.ld_u : nullptr;
            h.row_offset = g.row_offset + (u64)row;
            h.idx = g.idx + row * g.m;
            h.log_prob = g.log_prob ? g.log_prob + row * g.m : nullptr;
            if (h.p.temperature_t) h.p.temperature_t += row * h.p.temperature_rs;
            if (h.p.top_p_t) h.p.top_p_t += row * h.p.top_p_rs;
            if (h.p.min_p_t) h.p.min_p_t += row * h.p.min_p_rs;
            if (h.p.top_k_t) h.p.top_k_t += row * h.p.top_k_rs;
            const unsigned pairs = (unsigned)h.B * (unsigned)w.per_row;
            const dim3 grid((unsigned)w.chunks, pairs);
            wide_top_kernel<DT><<<grid, WT, 0, st>>>(h, w);
            if (w.k || w.p) wide_bins_kernel<DT><<<grid, WT, 0, st>>>(h, w);
            wide_collect_kernel<DT><<<grid, WT, 0, st>>>(h, w);
            wide_finish_kernel<DT><<<pairs, WT, 0, st>>>(h, w);
            CLAVA_CHECK_LAUNCH("sample_categories (wide)");
        }
    }
    return CLAVA_OK;
}

}  // namespace

extern "C" {

long long clava_choice_workspace_bytes(int B, int m, int sumK, int max_k) {
    if (B <= 0 || m <= 0 || sumK <= NARROW_MAX || max_k <= NARROW_MAX) return 0;
    const int most = wide_most(m, sumK, max_k), chunk = wide_chunk(B, most), chunks = (most + chunk - 1) / chunk;
    const int per_row = wide_per_row(m, sumK), rows = wide_rows(per_row);
    return (long long)(B < rows ? B : rows) * per_row * ((wide_bytes(chunks) + 15) / 16 * 16);
}

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
    if (sumK > (1 << 30) || (long long)B * m > 0x7fffffffLL || wide_per_row(m, sumK) > 65535) {
        clava_set_error("sample_categories: %d rows of %d features and %d classes are more than one call takes", B, m, sumK);
        return CLAVA_ERR_LIMIT;
    }
    const long long need = clava_choice_workspace_bytes(B, m, sumK, max_k);
    CLAVA_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
                    "sample_categories: needs a 16-byte aligned workspace of %lld bytes, got %lld", need, workspace_bytes);
    const hipStream_t st = (hipStream_t)stream;
    Choice g;
    g.z = logits; g.ld = ld; g.B = B; g.m = m; g.sumK = sumK; g.offsets = offsets; g.p = *choice;
    g.same = params_of(choice->temperature, choice->top_p, choice->min_p, choice->top_k);
    const bool tensors = choice->temperature_t || choice->top_p_t || choice->min_p_t || choice->top_k_t;
    const int mode = tensors ? TENSORS : g.same.top_k > 0 || g.same.top_p < 1.0 ? FILTERED : PLAIN;
    g.u = uniforms; g.ld_u = ld_u; g.seed = seed; g.row_offset = row_offset; g.step = step_index;
    g.idx = idx; g.log_prob = log_prob;
    g.wide = need != 0;
    g.wide_from = m == 1 && g.wide ? -1 : NARROW_MAX;         // (one feature: wide kernels for it, whatever its classes)
    g.wide_to = wide_most(m, sumK, max_k);
    Wide w{};
    if (need) {
        w.ws = (char*)workspace;
        w.chunk = wide_chunk(B, g.wide_to);
        w.chunks = (g.wide_to + w.chunk - 1) / w.chunk;
        w.per_row = wide_per_row(m, sumK);
        w.stride = (wide_bytes(w.chunks) + 15) / 16 * 16;
        w.k = filters_k(choice);
        w.p = filters_p(choice);
    }
    ProfScope prof(PROF_CHOICE, 0, (double)B * sumK * (dtype == CLAVA_DT_F32 ? 4 : 2) + 12.0 * B * m, st);
    return dtype == CLAVA_DT_F32 ? launch_choice<CLAVA_DT_F32>(g, w, max_k, mode, st)
           : dtype == CLAVA_DT_BF16 ? launch_choice<CLAVA_DT_BF16>(g, w, max_k, mode, st) : launch_choice<CLAVA_DT_F16>(g, w, max_k, mode, st);
}

}  // extern "C"
