// route.cu -- routing to experts: scores, the k best experts of each token,
// their weights, the lists by expert, and the gradient of the logits.
//
// Choice.  A token's experts are ordered by c = s + bias (s = softmax or sigmoid
// of the logits) or, without a bias, by the logit itself, which orders alike and
// is exact.  With a bias the order is that of c in 64 bits: the kernel forms c in
// fp32, whose error is below tau, and takes the selection when every gap between
// neighbours in it (and at the cut between kept and dropped groups) exceeds
// tau; a closer cut, and the few candidates of a closer selection, are settled by scores
// in 64 bits.
//
// Lists.  The tokens are cut into tiles, one block each.  A block ranks its choices
// among those of the same expert in its tile (in order: warps own adjacent choices
// and count in histograms of their own) and leaves its count per expert; a second
// kernel sums the counts of the tiles before and scatters.  Nothing depends on
// the order in which blocks run.  Up to kClusterTokens tokens the tiles' blocks are one
// cluster, which exchanges the counts in shared memory and scatters by itself.
//
// Bound by instructions: 16,384 tokens x 256 experts in 8 groups with a bias (18.4 MB with
// the outputs, 2.9 us at the copy rate) take 33.7 us in the mean of 24 inputs (32 to 36: a
// cut that is settled in 64 bits holds one block up by 2 us), 26 of them in route_kernel at 0.7
// instructions a clock and scheduler; of a token's 925 instructions 265 load it and weigh
// its choice, 95 find the floor, 135 list what reaches it, 135 rank that, 110 form the
// scores and 180 choose groups.  64 tokens take 9.3 us.
//
// From k of about 29 on, more keys than a warp ranks (kCandMax) reach the floor of most
// tokens, and those are chosen from 64-bit scores one expert at a time: 4096 x 256 take
// 34.1 us at k = 28, 40.5 at 30 and 42.6 at 32.  512 experts with k = 32 take 75 us; 1024,
// whose 32 experts a lane leave one block of 8 warps an SM, 34 us at k = 8 and 174 at 32.
#include <cuda_runtime.h>

#include <climits>
#include <cstdio>

#include "mflat_cuda.h"
#include "select_ops.cuh"

namespace mflat_cu {

int operator_device(int device, int* out) {
    device = mflat_cu_default_device(device);
    const int n = mflat_cu_device_count();
    if (n <= 0) return fail(ST_DEVICE, "no CUDA device");
    if (device < 0 || device >= n) return fail(ST_BAD_ARG, "device index out of range");
    *out = device;
    return ST_OK;
}

namespace {

constexpr int kMaxExperts = 1024, kMaxRouteK = 32, kMaxGroups = 32;
constexpr int kGradThreads = 256;
constexpr int kCandMax = 64;        // candidates of a token that one warp ranks
constexpr int kTiles = 148;         // one tile an SM
constexpr int kClusterTiles = 8, kClusterTokens = 512;

struct RouteParams {
    const void* logits;
    int64_t stride;
    int tokens, experts, k;
    int softmax, renormalise, groups, groups_kept, group_top;
    float scale;
    int vec;                    // rows can be read in whole aligned packs
    const float* bias;
    const uint8_t* mask;
    int32_t* ids;
    float* weights;
    int k_lanes;                // k rounded up to a power of two
    int lane_groups;            // lanes that share a group where that is a power of two, else 0
    // lists
    int tiles, tile;            // tokens per tile
    int cluster;                // the tiles' blocks are one cluster
    uint16_t* ranks;            // workspace [tokens * k]: rank among the tile's choices of the expert
    uint16_t* counts;           // workspace [tiles][experts rounded up to 2]
    int32_t* start;
    int32_t* slots;
};

// Bounds of the errors of the two fp32 scores on the sides of a gap.  sigmoid = 1 / (1 + e):
// e is off by 2^-22 + |x| 2^-23 of itself, which reaches s times 1 - s (below 8e-8),
// 1 + e rounds (6e-8), the reciprocal is off by 2^-23.  softmax = e / sum, in parts of
// the row's largest score: e 2.9e-7; the sum 2.4e-7 and, |x - m| weighted by the terms
// averaging at most ln 1024 + 1, 1.1e-6, its additions 2^-24 each for a lane's experts
// and 5 levels; reciprocal and product 1.8e-7.  Adding the bias rounds once more, 6e-8
// of the result, and so does a group's sum of two.
__device__ __forceinline__ float tau_base(bool softmax, float largest, int per_lane) {
    return softmax ? 2.0f * (2.3e-6f + 6e-8f * per_lane) * largest : 5.4e-7f;
}
__device__ __forceinline__ float tau_of(float base, float c) { return base + 1.3e-7f * fabsf(c); }
__device__ __forceinline__ float tau_of_two(float base, float a, float b) {
    return tau_of(base, a) + tau_of(base, b) + 1.3e-7f * fabsf(a + b);
}

template <class S>
__device__ __forceinline__ S exp_of(S v);
constexpr float kLog2e = 1.4426950408889634f;
template <>
__device__ __forceinline__ float exp_of<float>(float v) { return exp2_fast(v * kLog2e); }
template <>
__device__ __forceinline__ double exp_of<double>(double v) { return exp(v); }

template <int LPT>
__device__ __forceinline__ uint64_t lane_max(uint64_t v) {
#pragma unroll
    for (int o = LPT / 2; o > 0; o >>= 1) {
        const uint64_t w = __shfl_xor_sync(kFullMask, v, o);
        v = w > v ? w : v;
    }
    return v;
}

template <int LPT, class S>
__device__ __forceinline__ S lane_sum(S v) {
#pragma unroll
    for (int o = LPT / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
    return v;
}

// e[j] = exp(x[j] - m), m the row's largest: 0 for -inf, and where m itself is infinite 1
// for the logits that are m.  Returns the lane's sum.
template <class S, int VPL>
__device__ __forceinline__ S exps_of(const float (&x)[VPL], float m, S (&e)[VPL]) {
    S sum = 0;
    if (fabsf(m) < -neg_inf()) {
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            e[j] = exp_of<S>(S(x[j]) - S(m));
            sum += e[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            e[j] = x[j] == m && m > 0.0f ? S(1) : S(0);
            sum += e[j];
        }
    }
    return sum;
}

template <class S>
__device__ __forceinline__ S inverse(S v) {
    if constexpr (sizeof(S) == 4) return inverse_fast(v);
    else return S(1) / v;
}
// Scores of the lane's experts, lane l of a token holding experts [l * VPL, (l + 1) * VPL),
// and a bound of the row's largest.  x: fp32 logits, -inf for "none".
template <class S, int LPT, int VPL>
__device__ __forceinline__ void scores_of(const float (&x)[VPL], bool softmax, S (&s)[VPL], S& largest) {
    largest = S(1);
    if (softmax) {
        float m = neg_inf();
#pragma unroll
        for (int j = 0; j < VPL; ++j) m = fmaxf(m, x[j]);
#pragma unroll
        for (int o = LPT / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFullMask, m, o));
        const S sum = lane_sum<LPT>(exps_of<S, VPL>(x, m, s));
        const S inv = sum > S(0) ? inverse(sum) : S(0);
        largest = inv;
#pragma unroll
        for (int j = 0; j < VPL; ++j) s[j] *= inv;
    } else {
#pragma unroll
        for (int j = 0; j < VPL; ++j) s[j] = inverse(S(1) + exp_of<S>(-S(x[j])));
    }
}

// Each group's score, group by group over all lanes, for any group size: lane g
// gets the score of group g; tau the bound of the sums' errors.
template <class S, int LPT, int VPL>
__device__ __forceinline__ S group_scores(const RouteParams& p, int lane, const S (&c)[VPL],
                                          const bool (&in)[VPL], float base, float& tau) {
    const S none = S(neg_inf());
    const int size = p.experts / p.groups;
    S mine = none;
    tau = 0.0f;
    for (int g = 0; g < p.groups; ++g) {
        S a = none, b = none;   // the group's two largest
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            const int e = lane * VPL + j;
            if (e >= g * size && e < (g + 1) * size && in[j]) {
                const S v = c[j];
                if (v > a) { b = a; a = v; } else if (v > b) { b = v; }
            }
        }
#pragma unroll
        for (int o = LPT / 2; o > 0; o >>= 1) {
            const S a2 = __shfl_xor_sync(kFullMask, a, o), b2 = __shfl_xor_sync(kFullMask, b, o);
            const S lo = a2 > a ? a : a2, hi = b2 > b ? b2 : b;
            a = a2 > a ? a2 : a;
            b = lo > hi ? lo : hi;
        }
        const bool two = p.group_top == 2 && b != none;
        if (lane == g) mine = two ? a + b : a;
        if (a != none) tau = fmaxf(tau, two ? tau_of_two(base, float(a), float(b)) : tau_of(base, float(a)));
    }
    return mine;
}

// The groups that stay, as bits: lane g holds the score of group g.  Ties to the
// lower group.
template <class S, int LPT>
__device__ __forceinline__ unsigned kept_groups(const RouteParams& p, int lane, S mine) {
    int rank = 0;
    const int base = (threadIdx.x & 31) - lane;
    for (int g = 0; g < p.groups; ++g) {
        const S v = __shfl_sync(kFullMask, mine, base + g);
        rank += (v > mine || (v == mine && g < lane)) ? 1 : 0;
    }
    const unsigned all = __ballot_sync(kFullMask, lane < p.groups && rank < p.groups_kept);
    return (all >> base) & (LPT == 32 ? kFullMask : (1u << (LPT & 31)) - 1u);
}

// The k largest keys, ties to the lowest expert: lane r of the token gets the
// r-th expert (or -1) and its logit.
template <int LPT, int VPL>
__device__ __forceinline__ void take_best(uint64_t (&key)[VPL], const float (&x)[VPL], int k, int lane,
                                          int& id, float& xid) {
    const int base = (threadIdx.x & 31) - lane;
    id = -1;
    xid = neg_inf();
    for (int r = 0; r < k; ++r) {
        uint64_t best = 0;
        int at = 0;
        float xb = 0.0f;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            if (key[j] > best) { best = key[j]; at = j; xb = x[j]; }
        }
        const uint64_t top = lane_max<LPT>(best);
        const unsigned who = __ballot_sync(kFullMask, best == top) >> base;
        const int src = __ffs(who) - 1;
        const int e = __shfl_sync(kFullMask, lane * VPL + at, base + src);
        xb = __shfl_sync(kFullMask, xb, base + src);
        if (lane == r && top != 0) { id = e; xid = xb; }
        if (lane == src) {
#pragma unroll
            for (int j = 0; j < VPL; ++j)
                if (j == at) key[j] = 0;
        }
    }
}

// Weights of the chosen experts: lane r holds the r-th one's logit.  Plain:
// the score.  Renormalised: scores over their sum, formed from exponents relative
// to the largest chosen logit (sigmoid: to min(that, 0)), so that scores too
// small for fp32 still have their quotient.  In fp32 with the special function unit's
// reciprocals: 7e-8 off in the mean where a single rounding would leave 3e-8.  Only the
// choice needs more, and has it.
__device__ __forceinline__ float weight_of(const RouteParams& p, bool chosen, float x, float m,
                                           float sum) {
    float w = 0.0f;
    if (p.renormalise) {
        // the choices are in the first lanes: exchanges over a power of two of them
        float top = chosen ? x : neg_inf();
        for (int o = p.k_lanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, o));
        if (chosen) {
            if (p.softmax) {
                w = x == top ? 1.0f : expf(x - top);
            } else if (top >= 0.0f) {
                const float e = expf(-fabsf(x));
                w = (x >= 0.0f ? 1.0f : e) * inverse_fast(1.0f + e);
            } else {
                w = expf(x - top) * inverse_fast(1.0f + expf(x));
            }
        }
        float total = w;
        for (int o = p.k_lanes / 2; o > 0; o >>= 1) total += __shfl_xor_sync(kFullMask, total, o);
        w = total > 0.0f ? w * inverse_fast(total) : 0.0f;
    } else if (chosen) {
        w = p.softmax ? (x == m ? 1.0f : expf(x - m)) * inverse_fast(sum) : inverse_fast(1.0f + expf(-x));
    }
    return w * p.scale;
}

template <class T, int LPT, int VPL>
__device__ __forceinline__ void load_row(const RouteParams& p, int64_t t, int lane, bool live,
                                         float (&x)[VPL]) {
    const T* row = static_cast<const T*>(p.logits) + t * p.stride;
    constexpr int N = VPL * sizeof(T) >= 16 ? 16 / sizeof(T) : VPL;
    if (p.vec) {
#pragma unroll
        for (int j = 0; j < VPL; j += N) {
            const int e = lane * VPL + j;
            float f[N];
#pragma unroll
            for (int i = 0; i < N; ++i) f[i] = neg_inf();
            if (live && e < p.experts) {
                Pack<T, N> v;
                v.load(row + e);
                v.unpack(f);
            }
#pragma unroll
            for (int i = 0; i < N; ++i) x[j + i] = f[i];
        }
    } else {
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            const int e = lane * VPL + j;
            x[j] = live && e < p.experts ? to_float(row[e]) : neg_inf();
        }
    }
#pragma unroll
    for (int j = 0; j < VPL; ++j)
        if (!(x[j] > neg_inf())) x[j] = neg_inf();
}

// A token's choice keys in 64 bits (0: no choice), from the row read again.
template <class T, int LPT, int VPL>
__device__ __forceinline__ void exact_keys(const RouteParams& p, const float (&x)[VPL], int lane,
                                           double (&c)[VPL], uint64_t (&key)[VPL]) {
    if (p.bias || (p.groups > 1 && p.group_top == 2)) {
        double largest;
        scores_of<double, LPT, VPL>(x, p.softmax, c, largest);
    } else {
#pragma unroll
        for (int j = 0; j < VPL; ++j) c[j] = x[j];
    }
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        const int e = lane * VPL + j;
        if (p.bias && e < p.experts) c[j] += static_cast<double>(p.bias[e]);
        key[j] = x[j] == neg_inf() ? 0ull : choice_key(p.bias ? c[j] : static_cast<double>(x[j]));
    }
}

// A token's kept groups in 64 bits, as bits; where a group is 2^n lanes, all bits of its
// lanes alike.  The row is read again, so that the common path need not keep it (at 256
// experts that path spills 68 bytes of its 64 registers a thread as it is).  Every lane of
// the warp calls it.
template <class T, int LPT, int VPL>
__device__ __noinline__ unsigned exact_groups(const RouteParams& p, int64_t t, int lane, bool live) {
    float x[VPL];
    load_row<T, LPT, VPL>(p, t, lane, live, x);
    uint64_t key[VPL];
    double c[VPL];
    exact_keys<T, LPT, VPL>(p, x, lane, c, key);
    if (p.lane_groups == 0) {
        bool in[VPL];
        float unused;
#pragma unroll
        for (int j = 0; j < VPL; ++j) in[j] = key[j] != 0;
        return kept_groups<double, LPT>(p, lane, group_scores<double, LPT, VPL>(p, lane, c, in, 0.0f, unused));
    }
    const double none = static_cast<double>(neg_inf());
    double a = none, b = none;
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        const double v = key[j] != 0 ? c[j] : none;
        b = fmax(b, fmin(a, v));
        a = fmax(a, v);
    }
    for (int o = 1; o < p.lane_groups; o <<= 1) {
        const double a2 = __shfl_xor_sync(kFullMask, a, o), b2 = __shfl_xor_sync(kFullMask, b, o);
        b = fmax(fmin(a, a2), fmax(b, b2));
        a = fmax(a, a2);
    }
    const double mine = p.group_top == 2 && b > none ? a + b : a;
    const int base = (threadIdx.x & 31) - lane, group = lane / p.lane_groups;
    int above = 0;
    for (int g = 0; g < p.groups; ++g) {
        const double v = __shfl_sync(kFullMask, mine, base + g * p.lane_groups);
        above += v > mine || (v == mine && g < group) ? 1 : 0;
    }
    return group < p.groups && above < p.groups_kept ? ~0u : 0u;
}

// Whether an expert's group is among those that exact_groups() keeps.
__device__ __forceinline__ bool group_kept(const RouteParams& p, unsigned kept, int expert) {
    return p.lane_groups ? kept != 0u : ((kept >> min(expert / (p.experts / p.groups), 31)) & 1u) != 0u;
}

// A token from scores in 64 bits, for any values.  Every lane of the warp calls it.
template <class T, int LPT, int VPL>
__device__ __noinline__ void exact_token(const RouteParams& p, int64_t t, int lane, bool live,
                                         int& id, float& xid) {
    const unsigned kept = p.groups > 1 ? exact_groups<T, LPT, VPL>(p, t, lane, live) : 0u;
    float x[VPL];
    load_row<T, LPT, VPL>(p, t, lane, live, x);
    uint64_t key[VPL];
    double c[VPL];
    exact_keys<T, LPT, VPL>(p, x, lane, c, key);
    if (p.groups > 1) {
#pragma unroll
        for (int j = 0; j < VPL; ++j)
            if (!group_kept(p, kept, lane * VPL + j)) key[j] = 0;
    }
    take_best<LPT, VPL>(key, x, p.k, lane, id, xid);
}

// The groups' part of the choice in fp32: `bits` as exact_groups() gives them.
// Returns whether the cut is too close for fp32 (exact: c are logits, no doubt but
// ties, which go to the lower group).  Where a group is 2^n lanes of a warp, their
// top two meet in n exchanges, and each group is compared with all others: kept for
// sure, dropped for sure, or in doubt.
template <int LPT, int VPL, bool exact>
__device__ __forceinline__ bool choose_groups(const RouteParams& p, int lane, const float (&c)[VPL],
                                              float base_tau, const float (&key)[VPL], unsigned& bits) {
    const float none = neg_inf();
    if (p.lane_groups == 0) {
        bool in[VPL];
        float tau;
#pragma unroll
        for (int j = 0; j < VPL; ++j) in[j] = key[j] > none;
        const float mine = group_scores<float, LPT, VPL>(p, lane, c, in, base_tau, tau);
        bits = kept_groups<float, LPT>(p, lane, mine);
        const bool here = lane < p.groups && ((bits >> lane) & 1u);
        float low = here ? mine : -none, cut = lane < p.groups && !here ? mine : none;
#pragma unroll
        for (int o = LPT / 2; o > 0; o >>= 1) {
            low = fminf(low, __shfl_xor_sync(kFullMask, low, o));
            cut = fmaxf(cut, __shfl_xor_sync(kFullMask, cut, o));
        }
        return !exact && cut > none && !(low - cut > tau);
    }
    float a = none, b = none;
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        const float v = c[j];       // -inf where there is no choice
        b = fmaxf(b, fminf(a, v));
        a = fmaxf(a, v);
    }
    for (int o = 1; o < p.lane_groups; o <<= 1) {
        const float a2 = __shfl_xor_sync(kFullMask, a, o), b2 = __shfl_xor_sync(kFullMask, b, o);
        b = fmaxf(fminf(a, a2), fmaxf(b, b2));
        a = fmaxf(a, a2);
    }
    const bool two = p.group_top == 2 && b > none;
    const float mine = two ? a + b : a;
    // all groups' largest; both terms are at least 0, so their bits order alike
    float tau = two ? tau_of_two(base_tau, a, b) : a > none ? tau_of(base_tau, a) : 0.0f;
    tau = __uint_as_float(__reduce_max_sync(kFullMask, __float_as_uint(tau)));
    if (exact) tau = 0.0f;
    const int base = (threadIdx.x & 31) - lane;
    const int group = lane / p.lane_groups;
    // groups above for sure, and those not below for sure (itself among them): the lanes
    // of a group share the comparisons; counts in half words
    int counts = 0;
    const float high = mine + tau, low = mine - tau;
    for (int g0 = 0; g0 < p.groups; g0 += p.lane_groups) {
        const int g = g0 + (lane & (p.lane_groups - 1));
        const float v = __shfl_sync(kFullMask, mine, base + min(g, p.groups - 1) * p.lane_groups);
        if (g >= p.groups) continue;
        if constexpr (exact) {
            counts += v > mine || (v == mine && g < group) ? 1 : 0;
        } else {
            counts += (v > high ? 1 : 0) + (v < low ? 0 : 1 << 16);
        }
    }
    for (int o = 1; o < p.lane_groups; o <<= 1) counts += __shfl_xor_sync(kFullMask, counts, o);
    const int above = counts & 0xffff, near = counts >> 16;
    const bool kept = exact ? above < p.groups_kept : near <= p.groups_kept;
    const bool dropped = above >= p.groups_kept || mine == none;
    bits = kept ? ~0u : 0u;
    return group < p.groups && !kept && !dropped;
}

// A warp's scratch for one token's candidates.
template <int VPL>
struct RouteScratch {
    float keys[VPL * 32];               // [j][lane]
    float2 cand[kCandMax];              // key, expert
    float2 best[kMaxRouteK + 1];
};

// The choice scores of a token's n candidates in 64 bits, lane l those of candidates
// l and l + 32.  The row is read again, so that the common path need not keep it.
template <class T>
__device__ __noinline__ void refine(const RouteParams& p, const T* row, const float2* cand, int n,
                                    double (&c)[2]) {
    const int lane = threadIdx.x & 31;
    double m = 0.0, sum = 1.0;
    if (p.softmax) {
        float mf = neg_inf();
        for (int e = lane; e < p.experts; e += 32) mf = fmaxf(mf, to_float(row[e]));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mf = fmaxf(mf, __shfl_xor_sync(kFullMask, mf, o));
        m = mf;
        sum = 0.0;
        for (int e = lane; e < p.experts; e += 32) {
            const float v = to_float(row[e]);
            if (v > neg_inf()) sum += v == mf ? 1.0 : exp(static_cast<double>(v) - m);
        }
        sum = lane_sum<32>(sum);
    }
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
        const int i = lane + 32 * h;
        c[h] = static_cast<double>(neg_inf());
        if (i < n) {
            const int e = __float_as_int(cand[i].y);
            const double v = to_float(row[e]);
            const double s = p.softmax ? (v == m ? 1.0 : exp(v - m)) / sum : 1.0 / (1.0 + exp(-v));
            c[h] = s + static_cast<double>(p.bias[e]);
        }
    }
}

// The k largest fp32 keys of a token that a whole warp holds (VPL > 1).  The k-th
// largest lane maximum is a floor that few keys reach; those are ranked by counting.
// Lane r gets the r-th expert, or -1.  With a bias, the floor is lower by tau, and
// where neighbours in the selection are too close for fp32, its candidates are ranked
// again by scores in 64 bits.  Returns whether there were more candidates than fit.
template <class T, int VPL>
__device__ __forceinline__ bool take_best_warp(const RouteParams& p, const T* row, const float (&key)[VPL],
                                               float base_tau,
                                               RouteScratch<VPL>& sh, int& id) {
    const int lane = threadIdx.x & 31, k = p.k;
    const bool check = p.bias != nullptr;
    float top = key[0];
#pragma unroll
    for (int j = 1; j < VPL; ++j) top = fmaxf(top, key[j]);
    float floor_v;
    if (k <= 8) {
        // k maxima, each with all its equals taken out: 3 instructions each
        uint32_t v = choice_key(top), m = 0;
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if (r < k) {
                m = __reduce_max_sync(kFullMask, v);
                v = v == m ? 0u : v;
            }
        floor_v = key_value(m);
    } else {
        float v = top;
#pragma unroll
        for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
            for (int o = size >> 1; o > 0; o >>= 1) {
                const float w = __shfl_xor_sync(kFullMask, v, o);
                const bool larger = ((lane & size) == 0) == ((lane & o) == 0);
                v = larger ? fmaxf(v, w) : fminf(v, w);
            }
        floor_v = __shfl_sync(kFullMask, v, k - 1);
    }
    if (check) floor_v -= tau_of(base_tau, floor_v);
    // few lanes have any: those list theirs one after the other, behind the lanes below
    uint32_t mine_bits = 0;
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        sh.keys[j * 32 + lane] = key[j];
        // (a floor of NaN, from infinite biases, lets all pass)
        if (!(key[j] < floor_v) && key[j] > neg_inf()) mine_bits |= 1u << j;
    }
    const int count = __popc(mine_bits);
    int at = 0, n = 0;
#pragma unroll
    for (int s = 0; (1 << s) <= VPL; ++s) {
        const unsigned who = __ballot_sync(kFullMask, (count >> s) & 1);
        at += __popc(who & ((1u << lane) - 1u)) << s;
        n += __popc(who) << s;
    }
    if (n > kCandMax) return true;
    while (mine_bits) {
        const int j = __ffs(mine_bits) - 1;
        mine_bits &= mine_bits - 1u;
        sh.cand[at++] = make_float2(sh.keys[j * 32 + lane], __int_as_float(lane * VPL + j));
    }
    __syncwarp();
    for (int i = lane; i < n; i += 32) {
        const float2 c = sh.cand[i];
        const int e = __float_as_int(c.y);
        int rank = 0;
#pragma unroll 4
        for (int m = 0; m < n; ++m) {
            const float2 d = sh.cand[m];
            rank += d.x > c.x || (d.x == c.x && __float_as_int(d.y) < e) ? 1 : 0;
        }
        if (rank <= k) sh.best[rank] = c;
    }
    __syncwarp();
    const float2 mine = lane < n && lane <= k ? sh.best[lane] : make_float2(neg_inf(), 0.0f);
    id = lane < k && lane < n ? __float_as_int(mine.y) : -1;
    if (check) {
        // lane k holds the first that stays out (k = 32: look it up)
        float next = __shfl_down_sync(kFullMask, mine.x, 1);
        if (lane == 31) next = k == 32 && n > 32 ? sh.best[32].x : neg_inf();
        const bool close = lane < k && next > neg_inf() && !(mine.x - next > tau_of(base_tau, mine.x));
        if (__any_sync(kFullMask, close)) {
            double c[2];
            refine<T>(p, row, sh.cand, n, c);
            __syncwarp();
            id = -1;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (32 * h >= n) break;
                const int e = lane + 32 * h < n ? __float_as_int(sh.cand[lane + 32 * h].y) : 0;
                int rank = 0;
                for (int m = 0; m < n; ++m) {
                    const double d = __shfl_sync(kFullMask, m < 32 ? c[0] : c[1], m & 31);
                    rank += d > c[h] || (d == c[h] && __float_as_int(sh.cand[m].y) < e) ? 1 : 0;
                }
                if (lane + 32 * h < n && rank < k) sh.best[rank].y = __int_as_float(e);
            }
            __syncwarp();
            if (lane < k && lane < n) id = __float_as_int(sh.best[lane].y);
        }
    }
    __syncwarp();
    return false;
}

// Exclusive sums of v[0, n) in shared memory, in place: a thread sums a run, the runs'
// sums are scanned over the block.
template <int NT>
__device__ __forceinline__ void block_exclusive(int* v, int n, int* warp_sum) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per = (n + NT - 1) / NT, i0 = threadIdx.x * per;
    int sum = 0;
    for (int i = 0; i < per; ++i) sum += i0 + i < n ? v[i0 + i] : 0;
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(kFullMask, incl, o);
        if (lane >= o) incl += u;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        int s = lane < NT / 32 ? warp_sum[lane] : 0;
        const int own = s;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(kFullMask, s, o);
            if (lane >= o) s += u;
        }
        if (lane < NT / 32) warp_sum[lane] = s - own;
    }
    __syncthreads();
    int run = warp_sum[warp] + incl - sum;
    for (int i = 0; i < per; ++i)
        if (i0 + i < n) {
            const int c = v[i0 + i];
            v[i0 + i] = run;
            run += c;
        }
    __syncthreads();
}

// One tile of tokens a block, LPT lanes per token, VPL experts per lane.  With lists,
// then the ranks of the tile's choices and its counts; a cluster goes all the way.
template <class T, int LPT, int VPL, int NT>
__global__ void __launch_bounds__(NT) route_kernel(const __grid_constant__ RouteParams p) {
    constexpr int kWarps = NT / 32, kAtOnce = NT / LPT, kMost = LPT * VPL;
    extern __shared__ __align__(16) char dyn[];
    RouteScratch<VPL>* scratch = reinterpret_cast<RouteScratch<VPL>*>(dyn);
    const int lane = threadIdx.x % LPT, warp = threadIdx.x >> 5;
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.tile;
    const int64_t t1 = max(t0, min(t0 + p.tile, static_cast<int64_t>(p.tokens)));
    const bool by_sums = p.bias || (p.groups > 1 && p.group_top == 2);
    float b[VPL];
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        const int e = lane * VPL + j;
        b[j] = p.bias && e < p.experts ? p.bias[e] : 0.0f;
    }
    for (int64_t tb = t0 + warp * (32 / LPT); tb < t1; tb += kAtOnce) {
        const int64_t t = tb + (threadIdx.x & 31) / LPT;
        const bool live = t < t1 && (!p.mask || p.mask[t] != 0);
        float x[VPL], key[VPL];
        load_row<T, LPT, VPL>(p, t, lane, live, x);
        // the row's maximum and sum, for softmax weights
        float m = 0.0f, sum = 1.0f;
        if (p.softmax && !p.renormalise) {
            m = neg_inf();
#pragma unroll
            for (int j = 0; j < VPL; ++j) m = fmaxf(m, x[j]);
#pragma unroll
            for (int o = LPT / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFullMask, m, o));
            sum = lane_sum<LPT>(exps_of<float, VPL>(x, m, key));
        }
        bool doubt = false;
        float base_tau = 0.0f;
        unsigned kept = 0;
        if (by_sums) {
            float c[VPL], largest;
            scores_of<float, LPT, VPL>(x, p.softmax, c, largest);
            base_tau = tau_base(p.softmax, largest, VPL);
#pragma unroll
            for (int j = 0; j < VPL; ++j) {
                c[j] += b[j];
                if (!(x[j] > neg_inf() && c[j] > neg_inf())) c[j] = neg_inf();     // a bias of NaN too
                key[j] = p.bias ? c[j] : x[j];
            }
            if (p.groups > 1 && __any_sync(kFullMask, choose_groups<LPT, VPL, false>(p, lane, c, base_tau, key, kept)))
                kept = exact_groups<T, LPT, VPL>(p, t, lane, live);
        } else {
#pragma unroll
            for (int j = 0; j < VPL; ++j) key[j] = x[j];
            if (p.groups > 1) choose_groups<LPT, VPL, true>(p, lane, x, 0.0f, key, kept);
        }
        if (p.groups > 1) {
#pragma unroll
            for (int j = 0; j < VPL; ++j)
                if (!group_kept(p, kept, lane * VPL + j)) key[j] = neg_inf();
        }
        int id = -1;
        float xid = neg_inf();
        if constexpr (VPL > 1) {
            doubt |= take_best_warp<T, VPL>(p, static_cast<const T*>(p.logits) + t * p.stride, key,
                                            base_tau, scratch[warp], id);
        } else {
            // one expert a lane: its rank by counting
            const int base = (threadIdx.x & 31) - lane;
            int rank = 0;
            float next = neg_inf();     // the largest below
#pragma unroll
            for (int e = 0; e < LPT; ++e) {
                const float v = __shfl_sync(kFullMask, key[0], base + e);
                const bool before = v > key[0] || (v == key[0] && e < lane);
                rank += before ? 1 : 0;
                next = !before && e != lane ? fmaxf(next, v) : next;
            }
            if (!(key[0] > neg_inf())) rank = LPT;
            if (p.bias && rank < p.k && next > neg_inf()) doubt |= !(key[0] - next > tau_of(base_tau, key[0]));
            for (int r = 0; r < p.k; ++r) {
                const unsigned who = __ballot_sync(kFullMask, rank == r) >> base;
                const unsigned own = LPT == 32 ? who : who & ((1u << (LPT & 31)) - 1u);
                if (lane == r && own) id = __ffs(own) - 1;
            }
        }
        if (__any_sync(kFullMask, doubt)) {
            exact_token<T, LPT, VPL>(p, t, lane, live, id, xid);
        } else if (id >= 0) {
            xid = to_float(static_cast<const T*>(p.logits)[t * p.stride + id]);
        }
        const float w = weight_of(p, id >= 0, xid, m, sum);
        if (t < t1 && lane < p.k) {
            p.ids[t * p.k + lane] = id;
            p.weights[t * p.k + lane] = w;
        }
    }
    if (!p.start) return;

    // ranks: warps own adjacent runs of the tile's choices
    __shared__ __align__(16) uint16_t hist[kWarps][kMost];      // cleared by words
    __shared__ int total[kMost + 1], before[kMost];
    __shared__ int warp_sum[32];
    const int full_lane = threadIdx.x & 31;
    for (int i = threadIdx.x; i < kWarps * kMost / 2; i += NT) reinterpret_cast<uint32_t*>(&hist[0][0])[i] = 0;
    __syncthreads();
    grid_release();
    const int64_t e0 = t0 * p.k, n = (t1 - t0) * p.k;
    const int64_t run = (n + kWarps * 32 - 1) / (kWarps * 32) * 32;
    const int64_t r0 = e0 + warp * run, r1 = min(r0 + run, e0 + n);
    // a run of one step (a tile of up to 32 choices a warp) stays in registers
    const bool one = run == 32;
    int own_id = -1, own_rank = 0;
    for (int64_t i0 = r0; i0 < r1; i0 += 32) {
        const int64_t i = i0 + full_lane;
        const int id = i < r1 ? p.ids[i] : -1;
        const unsigned peers = __match_any_sync(kFullMask, id);
        const int rank = __popc(peers & ((1u << full_lane) - 1u));
        int seen = 0;
        if (id >= 0 && rank == 0) {
            seen = hist[warp][id];
            hist[warp][id] = static_cast<uint16_t>(seen + __popc(peers));
        }
        seen = __shfl_sync(kFullMask, seen, __ffs(peers) - 1);
        own_id = id;
        own_rank = seen + rank;
        if (!one && id >= 0) p.ranks[i] = static_cast<uint16_t>(own_rank);
        __syncwarp();
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.experts; e += NT) {
        int s = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const int c = hist[w][e];
            hist[w][e] = static_cast<uint16_t>(s);
            s += c;
        }
        total[e] = s;
        if (!p.cluster) p.counts[static_cast<int64_t>(blockIdx.x) * ((p.experts + 1) & ~1) + e] = static_cast<uint16_t>(s);
    }
    // fn(choice, expert, rank in the tile) for the thread's choices
    auto each = [&](auto&& fn) {
        if (one) {
            if (own_id >= 0) fn(r0 + full_lane, own_id, own_rank + hist[warp][own_id]);
            return;
        }
        for (int64_t i = r0 + full_lane; i < r1; i += 32) {
            const int id = p.ids[i];
            if (id >= 0) fn(i, id, p.ranks[i] + hist[warp][id]);
        }
    };
    if (!p.cluster) {
        __syncthreads();
        each([&](int64_t i, int, int rank) { p.ranks[i] = static_cast<uint16_t>(rank); });
        return;
    }
    cluster_sync();             // every block's counts are in its total[]
    const uint32_t me = cluster_rank();
    int sums[(kMost + NT - 1) / NT];
#pragma unroll
    for (int j = 0; j < (kMost + NT - 1) / NT; ++j) {
        const int e = j * NT + threadIdx.x;
        int all = 0, ahead = 0;
        if (e < p.experts) {
#pragma unroll
            for (uint32_t r = 0; r < kClusterTiles; ++r) {
                int c;
                asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(c) : "r"(cluster_addr(&total[e], r)) : "memory");
                all += c;
                ahead += r < me ? c : 0;
            }
            before[e] = ahead;
        }
        sums[j] = all;
    }
    cluster_sync();             // and read by all: total[] is free again
#pragma unroll
    for (int j = 0; j < (kMost + NT - 1) / NT; ++j) {
        const int e = j * NT + threadIdx.x;
        if (e < p.experts) total[e] = sums[j];
    }
    if (threadIdx.x == 0) total[p.experts] = 0;
    __syncthreads();
    block_exclusive<NT>(total, p.experts + 1, warp_sum);
    if (me == 0)
        for (int e = threadIdx.x; e <= p.experts; e += NT) p.start[e] = total[e];
    each([&](int64_t i, int id, int rank) { p.slots[total[id] + before[id] + rank] = static_cast<int32_t>(i); });
}

// The lists of many tiles: where this tile's choices of each expert begin, then the
// scatter.  A thread sums two adjacent experts over its share of the tiles' counts.
constexpr int kListThreads = 1024;
__global__ void __launch_bounds__(kListThreads) lists_kernel(const __grid_constant__ RouteParams p) {
    __shared__ int before[kMaxExperts], total[kMaxExperts + 1];
    __shared__ int warp_sum[32];
    const int pairs = (p.experts + 1) / 2, groups = max(1, kListThreads / pairs);
    for (int e = threadIdx.x; e <= p.experts; e += kListThreads) {
        total[e] = 0;
        if (e < p.experts) before[e] = 0;
    }
    __syncthreads();
    grid_wait();
    // the thread's first choice is on its way while the counts are summed
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.tile;
    const int64_t t1 = min(t0 + p.tile, static_cast<int64_t>(p.tokens));
    const int64_t first = t0 * p.k + threadIdx.x;
    int id0 = -1, rank0 = 0;
    if (first < t1 * p.k) {
        id0 = p.ids[first];
        rank0 = p.ranks[first];
    }
    const int pair = threadIdx.x % pairs, group = threadIdx.x / pairs;
    if (group < groups) {
        int b0 = 0, b1 = 0, s0 = 0, s1 = 0;
        const uint32_t* rows = reinterpret_cast<const uint32_t*>(p.counts) + pair;
#pragma unroll 8
        for (int r = group; r < p.tiles; r += groups) {
            const uint32_t c = rows[static_cast<int64_t>(r) * pairs];
            const int lo = c & 0xffffu, hi = c >> 16;
            s0 += lo;
            s1 += hi;
            b0 += r < static_cast<int>(blockIdx.x) ? lo : 0;
            b1 += r < static_cast<int>(blockIdx.x) ? hi : 0;
        }
        // sums of whole numbers: the order of these additions changes nothing
        atomicAdd(&before[2 * pair], b0);
        atomicAdd(&total[2 * pair], s0);
        if (2 * pair + 1 < p.experts) {
            atomicAdd(&before[2 * pair + 1], b1);
            atomicAdd(&total[2 * pair + 1], s1);
        }
    }
    __syncthreads();
    block_exclusive<kListThreads>(total, p.experts + 1, warp_sum);
    if (blockIdx.x == 0)
        for (int e = threadIdx.x; e <= p.experts; e += kListThreads) p.start[e] = total[e];
    if (id0 >= 0) p.slots[total[id0] + before[id0] + rank0] = static_cast<int32_t>(first);
    for (int64_t i = first + kListThreads; i < t1 * p.k; i += kListThreads) {
        const int id = p.ids[i];
        if (id >= 0) p.slots[total[id] + before[id] + p.ranks[i]] = static_cast<int32_t>(i);
    }
}

// Gradient of the logits, LPT lanes per token as in the forward pass.  With w =
// scale * s (s a softmax p): dx_e = scale * p_e (g_e - sum_j g_j p_j); sigmoid:
// dx_e = scale * g_e s_e (1 - s_e).  Renormalised over the chosen (w = scale * s /
// S): dx_j = w_j (g_j - sum_i g_i w_i / scale), for a sigmoid times 1 - s_j.  32,768 x 128
// bf16 take 8.8 us (16.8 MB: 1.9 TB/s), bound by instructions; with 4 experts a lane and
// one token a warp they took 17.6.
template <class T, int LPT, int VPL>
__global__ void __launch_bounds__(kGradThreads)
    route_backward_kernel(const RouteParams p, const float* __restrict__ grad, T* out,
                          int64_t out_stride) {
    const int lane = threadIdx.x % LPT, base = (threadIdx.x & 31) - lane;
    const int64_t t = (static_cast<int64_t>(blockIdx.x) * kGradThreads + threadIdx.x) / LPT;
    const bool live = t < p.tokens;
    float x[VPL];
    load_row<T, LPT, VPL>(p, t, lane, live, x);
    int id = -1;
    float g = 0.0f;
    if (live && lane < p.k) {
        id = p.ids[t * p.k + lane];
        if (id < 0 || id >= p.experts) id = -1;
        else g = grad[t * p.k + lane];
    }
    float xid = neg_inf();
    if (id >= 0) xid = to_float(static_cast<const T*>(p.logits)[t * p.stride + id]);
    if (!(xid > neg_inf())) xid = neg_inf();
    const bool chosen = id >= 0 && xid > neg_inf();
    if (!chosen) g = 0.0f;
    float d[VPL], m = 0.0f, sum = 1.0f;
    const bool whole = p.softmax && !p.renormalise;
    if (whole) {
        m = neg_inf();
#pragma unroll
        for (int j = 0; j < VPL; ++j) m = fmaxf(m, x[j]);
#pragma unroll
        for (int o = LPT / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFullMask, m, o));
        sum = lane_sum<LPT>(exps_of<float, VPL>(x, m, d));
    } else {
#pragma unroll
        for (int j = 0; j < VPL; ++j) d[j] = 0.0f;
    }
    RouteParams q = p;
    q.scale = 1.0f;
    const float w = weight_of(q, chosen, xid, m, sum);
    const float dot = (p.softmax || p.renormalise) ? lane_sum<LPT>(g * w) : 0.0f;
    if (whole) {
        const float inv = sum > 0.0f ? p.scale * inverse_fast(sum) : 0.0f;
#pragma unroll
        for (int j = 0; j < VPL; ++j) d[j] *= inv;
        float mult[VPL];
#pragma unroll
        for (int j = 0; j < VPL; ++j) mult[j] = -dot;
        for (int r = 0; r < p.k; ++r) {
            const int e = __shfl_sync(kFullMask, id, base + r);
            const float ge = __shfl_sync(kFullMask, g, base + r);
#pragma unroll
            for (int j = 0; j < VPL; ++j)
                if (e == lane * VPL + j) mult[j] += ge;
        }
#pragma unroll
        for (int j = 0; j < VPL; ++j) d[j] *= mult[j];
    } else {
        float v = p.scale * w * (p.renormalise ? g - dot : g);
        if (!p.softmax) v *= inverse_fast(1.0f + expf(xid));    // 1 - s
        if (!chosen) v = 0.0f;
        for (int r = 0; r < p.k; ++r) {
            const int e = __shfl_sync(kFullMask, id, base + r);
            const float ve = __shfl_sync(kFullMask, v, base + r);
#pragma unroll
            for (int j = 0; j < VPL; ++j)
                if (e == lane * VPL + j) d[j] += ve;
        }
    }
    if (!live) return;
    T* row = out + t * out_stride;
    constexpr int N = VPL * sizeof(T) >= 16 ? 16 / sizeof(T) : VPL;
#pragma unroll
    for (int j = 0; j < VPL; j += N) {
        const int e = lane * VPL + j;
        if (p.vec) {
            float f[N];
#pragma unroll
            for (int i = 0; i < N; ++i) f[i] = d[j + i];
            Pack<T, N> v;
            v.pack(f);
            if (e < p.experts) v.store(row + e);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (e + i < p.experts) row[e + i] = from_float<T>(d[j + i]);
        }
    }
}

// One block a tile, all in one cluster or on their own.
template <class K>
cudaError_t launch_route(K kernel, unsigned threads, size_t smem, cudaStream_t st, const RouteParams& p) {
    if (smem > 0) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   static_cast<int>(smem));
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(p.tiles));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = static_cast<unsigned>(p.tiles);
    at.val.clusterDim.y = 1;
    at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = p.cluster ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

// Calls fn(LPT, VPL, NT) as integral constants for a router: as few lanes per
// token as hold its experts one each and its k choices; blocks of one to an SM as
// long as a thread's experts leave the registers for it.
template <class Fn>
cudaError_t with_layout(int experts, Fn&& fn) {
    using std::integral_constant;
    if (experts <= 8) return fn(integral_constant<int, 8>{}, integral_constant<int, 1>{}, integral_constant<int, 1024>{});
    if (experts <= 16) return fn(integral_constant<int, 16>{}, integral_constant<int, 1>{}, integral_constant<int, 1024>{});
    if (experts <= 32) return fn(integral_constant<int, 32>{}, integral_constant<int, 1>{}, integral_constant<int, 1024>{});
    if (experts <= 64) return fn(integral_constant<int, 32>{}, integral_constant<int, 2>{}, integral_constant<int, 1024>{});
    if (experts <= 128) return fn(integral_constant<int, 32>{}, integral_constant<int, 4>{}, integral_constant<int, 1024>{});
    if (experts <= 256) return fn(integral_constant<int, 32>{}, integral_constant<int, 8>{}, integral_constant<int, 1024>{});
    if (experts <= 512) return fn(integral_constant<int, 32>{}, integral_constant<int, 16>{}, integral_constant<int, 512>{});
    return fn(integral_constant<int, 32>{}, integral_constant<int, 32>{}, integral_constant<int, 256>{});
}

// The gradient's layout: 8 experts a lane (16 bytes of 16-bit logits), so that up to
// four tokens share a warp and its exchanges; else as above.
template <class Fn>
cudaError_t with_grad_layout(int experts, int k, Fn&& fn) {
    using std::integral_constant;
    const integral_constant<int, 8> eight{};
    if (experts > 32 && experts <= 64 && k <= 8) return fn(eight, eight);
    if (experts > 32 && experts <= 128 && k <= 16) return fn(integral_constant<int, 16>{}, eight);
    return with_layout(experts, [&](auto lpt, auto vpl, auto) { return fn(lpt, vpl); });
}

// Whether rows can be moved in whole packs of 16 bytes, or of a lane's vpl experts
// where those are less.
bool packed_rows(const void* p, int64_t stride, int experts, int vpl, size_t es) {
    const size_t n = vpl * es >= 16 ? 16 / es : static_cast<size_t>(vpl);
    return experts % n == 0 && stride % static_cast<int64_t>(n) == 0 && aligned_to(p, n * es);
}

int check_router(const mflat_cu_router_t* r, int tokens) {
    char msg[200];
    if (r->experts < 1 || r->experts > kMaxExperts) {
        std::snprintf(msg, sizeof msg, "experts=%d outside [1, %d]", r->experts, kMaxExperts);
        return fail(ST_BAD_ARG, msg);
    }
    if (r->k < 1 || r->k > kMaxRouteK || r->k > r->experts) {
        std::snprintf(msg, sizeof msg, "k=%d outside [1, min(%d, experts=%d)]", r->k, kMaxRouteK,
                      r->experts);
        return fail(ST_BAD_ARG, msg);
    }
    if (r->score < 0 || r->score > 1) return fail(ST_BAD_ARG, "unknown score");
    if (r->type < 0 || r->type > 2) return fail(ST_BAD_ARG, "unknown logits type");
    if (r->groups < 1 || r->groups > kMaxGroups || r->experts % r->groups != 0) {
        std::snprintf(msg, sizeof msg, "groups=%d must divide experts=%d and be in [1, %d]", r->groups,
                      r->experts, kMaxGroups);
        return fail(ST_BAD_ARG, msg);
    }
    if (r->groups_kept < 1 || r->groups_kept > r->groups)
        return fail(ST_BAD_ARG, "groups_kept outside [1, groups]");
    if (r->group_top < 1 || r->group_top > 2) return fail(ST_BAD_ARG, "group_top must be 1 or 2");
    if (tokens < 0 || static_cast<int64_t>(tokens) * r->k > INT_MAX) {
        std::snprintf(msg, sizeof msg, "tokens=%d: tokens * k must be in [0, 2^31)", tokens);
        return fail(ST_BAD_ARG, msg);
    }
    return ST_OK;
}

// Tiles: one to an SM, no more tokens in one than 16-bit counts hold; up to
// kClusterTokens tokens (with lists), one to a block of a cluster.
struct RoutePlan {
    bool cluster;
    int tiles, tile;
    size_t ranks, counts, end;
};
RoutePlan route_plan(const mflat_cu_router_t* r, int tokens) {
    RoutePlan l{};
    // a cluster's block keeps its choices in registers, one a thread
    const int threads = r->experts <= 256 ? 1024 : r->experts <= 512 ? 512 : 256;
    auto per = [tokens](int n) { return tokens / n + (tokens % n != 0); };      // up to 2^31 - 1 tokens
    l.tile = per(kClusterTiles);
    if (tokens <= kClusterTokens && l.tile * r->k <= threads) {
        l.cluster = true;
        l.tiles = kClusterTiles;
        return l;
    }
    l.tiles = kTiles;
    l.tile = per(kTiles);
    if (l.tile > 65535) l.tile = 65535;
    l.tiles = per(l.tile);
    auto round256 = [](size_t n) { return (n + 255) & ~size_t(255); };
    l.ranks = 0;
    l.counts = round256(static_cast<size_t>(tokens) * r->k * 2);
    l.end = l.counts + round256(static_cast<size_t>(l.tiles) * ((r->experts + 1) & ~1) * 2);
    return l;
}

int fill_params(const mflat_cu_router_t* r, const void* logits, int64_t& stride, int tokens,
                RouteParams& p) {
    if (stride == 0) stride = r->experts;
    if (stride < r->experts) return fail(ST_BAD_ARG, "logits stride below experts");
    if (!aligned_to(logits, type_bytes(r->type))) return fail(ST_BAD_ARG, "misaligned logits");
    p = {};
    p.logits = logits;
    p.stride = stride;
    p.tokens = tokens;
    p.experts = r->experts;
    p.k = r->k;
    p.softmax = r->score == 0;
    p.renormalise = r->renormalise != 0;
    p.groups = r->groups;
    p.groups_kept = r->groups_kept;
    p.group_top = r->group_top;
    p.scale = r->scale;
    p.k_lanes = 1;
    while (p.k_lanes < r->k) p.k_lanes *= 2;
    int vpl = 1;
    while (vpl * 32 < r->experts) vpl *= 2;
    p.vec = packed_rows(logits, stride, r->experts, vpl, type_bytes(r->type));
    const int size = r->experts / r->groups;
    const int lanes = size % vpl == 0 ? size / vpl : 0;
    p.lane_groups = lanes > 0 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
    return ST_OK;
}

}  // namespace
}  // namespace mflat_cu

using namespace mflat_cu;

extern "C" size_t mflat_cu_route_workspace(const mflat_cu_router_t* r, int tokens) {
    if (check_router(r, tokens) != ST_OK || tokens == 0) return 0;
    return route_plan(r, tokens).end;
}

extern "C" int mflat_cu_route(const mflat_cu_router_t* r, const void* logits, int64_t stride,
                              int tokens, const float* bias, const uint8_t* mask, int32_t* ids,
                              float* weights, int32_t* start, int32_t* slots, void* ws,
                              size_t ws_bytes, int device, void* stream) {
    int rc = check_router(r, tokens);
    if (rc != ST_OK) return rc;
    RouteParams p;
    rc = fill_params(r, logits, stride, tokens, p);
    if (rc != ST_OK) return rc;
    if (!aligned_to(bias, 4) || !aligned_to(ids, 4) || !aligned_to(weights, 4) ||
        !aligned_to(start, 4) || !aligned_to(slots, 4))
        return fail(ST_BAD_ARG, "misaligned pointer");
    if (tokens == 0 && !start) return ST_OK;
    const size_t need = start && tokens > 0 ? route_plan(r, tokens).end : 0;
    if (need > 0 && (!ws || ws_bytes < need || !aligned_to(ws, 256)))
        return fail(ST_BAD_ARG, "workspace missing, too small or not 256-byte aligned");
    rc = operator_device(device, &device);
    if (rc != ST_OK) return rc;
    DeviceGuard g(device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (tokens == 0) {
        CU_TRY(cudaMemsetAsync(start, 0, (static_cast<size_t>(r->experts) + 1) * 4, st), "empty lists");
        return ST_OK;
    }
    p.bias = bias;
    p.mask = mask;
    p.ids = ids;
    p.weights = weights;
    const RoutePlan l = route_plan(r, tokens);
    p.tiles = l.tiles;
    p.tile = l.tile;
    if (!start && l.cluster) {      // no lists: over all SMs
        p.tile = (tokens + kTiles - 1) / kTiles;
        p.tiles = (tokens + p.tile - 1) / p.tile;
    }
    p.cluster = start && l.cluster;
    p.start = start;
    p.slots = slots;
    p.ranks = reinterpret_cast<uint16_t*>(static_cast<char*>(ws) + l.ranks);
    p.counts = reinterpret_cast<uint16_t*>(static_cast<char*>(ws) + l.counts);
    CU_TRY(with_type(r->type, [&](auto zero) {
        using T = decltype(zero);
        return with_layout(r->experts, [&](auto lpt, auto vpl, auto nt) {
            constexpr int L = decltype(lpt)::value, V = decltype(vpl)::value, N = decltype(nt)::value;
            constexpr size_t smem = V > 1 ? sizeof(RouteScratch<V>) * (N / 32) : 0;
            return launch_route(route_kernel<T, L, V, N>, N, smem, st, p);
        });
    }), "route launch");
    if (start && !l.cluster)
        CU_TRY(launch_after(lists_kernel, dim3(l.tiles), kListThreads, 0, st, p), "lists launch");
    return ST_OK;
}

extern "C" int mflat_cu_route_backward(const mflat_cu_router_t* r, const void* logits,
                                       int64_t stride, int tokens, const int32_t* ids,
                                       const float* grad_weights, void* grad, int64_t grad_stride,
                                       int device, void* stream) {
    int rc = check_router(r, tokens);
    if (rc != ST_OK) return rc;
    RouteParams p;
    rc = fill_params(r, logits, stride, tokens, p);
    if (rc != ST_OK) return rc;
    if (grad_stride == 0) grad_stride = r->experts;
    if (grad_stride < r->experts) return fail(ST_BAD_ARG, "gradient stride below experts");
    if (!aligned_to(grad, type_bytes(r->type)) || !aligned_to(ids, 4) || !aligned_to(grad_weights, 4))
        return fail(ST_BAD_ARG, "misaligned pointer");
    if (grad == logits && grad_stride != stride)
        return fail(ST_BAD_ARG, "a gradient over the logits needs their stride");
    if (tokens == 0) return ST_OK;
    rc = operator_device(device, &device);
    if (rc != ST_OK) return rc;
    DeviceGuard g(device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const size_t es = type_bytes(r->type);
    auto vec_for = [&](int vpl) {
        return packed_rows(logits, stride, r->experts, vpl, es) && packed_rows(grad, grad_stride, r->experts, vpl, es);
    };
    p.ids = const_cast<int32_t*>(ids);
    CU_TRY(with_type(r->type, [&](auto zero) {
        using T = decltype(zero);
        return with_grad_layout(r->experts, r->k, [&](auto lpt, auto vpl) {
            constexpr int L = decltype(lpt)::value, V = decltype(vpl)::value;
            p.vec = vec_for(V);
            route_backward_kernel<T, L, V>
                <<<blocks_for(static_cast<int64_t>(tokens) * L, kGradThreads), kGradThreads, 0, st>>>(
                    p, grad_weights, static_cast<T*>(grad), grad_stride);
            return cudaGetLastError();
        });
    }), "route backward launch");
    return ST_OK;
}
