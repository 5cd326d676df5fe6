// route.cu -- routing to experts: scores, the k best experts of each token,
// their weights, the lists by expert, and the gradient of the logits.
//
// Choice.  A token's experts are ordered by c = s + bias (s = softmax or sigmoid
// of the logits) or, without a bias, by the logit itself, which orders alike and
// is exact.  With a bias the order is that of c in 64 bits: the kernel forms c in
// fp32, whose error is below tau, and takes the selection when every gap between
// neighbours in it (and at the cut between kept and dropped groups) exceeds
// tau; the other tokens are selected again from scores in 64 bits.
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
constexpr int kRouteThreads = 256;

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
};

// Error bounds of an fp32 choice score and of a sum of two.  The scores are in
// [0, 1] and formed with errors below 1e-6 (expf by exp2 of a rounded product:
// relative 2^-22 + |x| 2^-24, which sigmoid and softmax damp by their own
// value, a division of 2 ulp, and a sum of at most 1024 terms in a tree); adding
// the bias rounds once more.  Twice that, for the two sides of a gap.
__device__ __forceinline__ float tau_of(float c) { return 4e-6f + 3e-7f * fabsf(c); }

template <class S>
__device__ __forceinline__ S exp_of(S v);
template <>
__device__ __forceinline__ float exp_of<float>(float v) { return __expf(v); }
template <>
__device__ __forceinline__ double exp_of<double>(double v) { return exp(v); }

template <int LPT, class V>
__device__ __forceinline__ V lane_max(V v) {
    if constexpr (LPT == 32 && sizeof(V) == 4) {
        return __reduce_max_sync(kFullMask, v);
    } else {
#pragma unroll
        for (int o = LPT / 2; o > 0; o >>= 1) {
            const V w = __shfl_xor_sync(kFullMask, v, o);
            v = w > v ? w : v;
        }
        return v;
    }
}

template <int LPT, class S>
__device__ __forceinline__ S lane_sum(S v) {
#pragma unroll
    for (int o = LPT / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
    return v;
}

// Scores of the lane's experts, lane l of a token holding experts
// [l * VPL, (l + 1) * VPL).  x: fp32 logits, -inf for "none".
template <class S, int LPT, int VPL>
__device__ __forceinline__ void scores_of(const float (&x)[VPL], bool softmax, S (&s)[VPL]) {
    if (softmax) {
        float m = neg_inf();
#pragma unroll
        for (int j = 0; j < VPL; ++j) m = fmaxf(m, x[j]);
#pragma unroll
        for (int o = LPT / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFullMask, m, o));
        S sum = 0;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            s[j] = x[j] == neg_inf() ? S(0) : x[j] == m ? S(1) : exp_of<S>(S(x[j]) - S(m));
            sum += s[j];
        }
        sum = lane_sum<LPT>(sum);
        const S inv = sum > S(0) ? S(1) / sum : S(0);
#pragma unroll
        for (int j = 0; j < VPL; ++j) s[j] *= inv;
    } else {
#pragma unroll
        for (int j = 0; j < VPL; ++j) s[j] = S(1) / (S(1) + exp_of<S>(-S(x[j])));
    }
}

// Group selection: clears the keys of experts outside the groups_kept best
// groups.  Returns whether a gap at the cut is too small for fp32.
template <class S, int LPT, int VPL, class K>
__device__ __forceinline__ bool keep_groups(const RouteParams& p, int lane, const S (&c)[VPL],
                                            K (&key)[VPL]) {
    const S none = S(neg_inf());
    const int size = p.experts / p.groups;
    S mine = none;              // lane g: score of group g
    float tau = 0.0f;
    for (int g = 0; g < p.groups; ++g) {
        S a = none, b = none;   // the group's two largest
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            const int e = lane * VPL + j;
            if (e >= g * size && e < (g + 1) * size && key[j] != 0) {
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
        if (a != none) tau = fmaxf(tau, tau_of(float(a)) + (two ? tau_of(float(b)) : 0.0f));
    }
    // a group's rank among all (ties to the lower group)
    int rank = 0;
    const int base = (threadIdx.x & 31) - lane;
    for (int g = 0; g < p.groups; ++g) {
        const S v = __shfl_sync(kFullMask, mine, base + g);
        rank += (v > mine || (v == mine && g < lane)) ? 1 : 0;
    }
    const bool kept = lane < p.groups && rank < p.groups_kept;
    const unsigned all = __ballot_sync(kFullMask, kept);
    const unsigned bits = (all >> base) & (LPT == 32 ? kFullMask : (1u << (LPT & 31)) - 1u);
    bool doubt = false;
    if constexpr (sizeof(S) == 4) {
        const uint32_t cut = lane_max<LPT>(lane < p.groups && !kept ? choice_key(mine) : 0u);
        const uint32_t low = ~lane_max<LPT>(kept ? ~choice_key(mine) : 0u);
        if (cut != 0u && low != 0u) doubt = !(key_value(low) - key_value(cut) > tau);
    }
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        const int g = min((lane * VPL + j) / size, 31);
        if (!((bits >> g) & 1u)) key[j] = 0;
    }
    return doubt;
}

// The k largest keys, ties to the lowest expert: lane r of the token gets the
// r-th expert (or -1) and its logit.  With `check`, returns whether a gap in the
// selection is too small for fp32 scores.
template <int LPT, int VPL, class K>
__device__ __forceinline__ bool take_best(K (&key)[VPL], const float (&x)[VPL], int k, int lane,
                                          bool check, int& id, float& xid) {
    const int base = (threadIdx.x & 31) - lane;
    id = -1;
    xid = neg_inf();
    bool doubt = false;
    K before = 0;
    const int rounds = check ? k + 1 : k;
    for (int r = 0; r < rounds; ++r) {
        K best = 0;
        int at = 0;
        float xb = 0.0f;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            if (key[j] > best) { best = key[j]; at = j; xb = x[j]; }
        }
        const K top = lane_max<LPT>(best);
        const unsigned who = __ballot_sync(kFullMask, best == top) >> base;
        const int src = __ffs(who) - 1;
        const int e = __shfl_sync(kFullMask, lane * VPL + at, base + src);
        xb = __shfl_sync(kFullMask, xb, base + src);
        if (lane == r && r < k && top != 0) { id = e; xid = xb; }
        if (lane == src) {
#pragma unroll
            for (int j = 0; j < VPL; ++j)
                if (j == at) key[j] = 0;
        }
        if constexpr (sizeof(K) == 4) {
            if (check && r > 0 && top != 0) {
                const float hi = key_value(before), lo = key_value(top);
                if (!(hi - lo > tau_of(hi))) doubt = true;
            }
        }
        before = top;
    }
    return doubt;
}

// Weights of the chosen experts: lane r holds the r-th one's logit.  Plain:
// the score.  Renormalised: scores over their sum, formed from exponents relative
// to the largest chosen logit (sigmoid: to min(that, 0)), so that scores too
// small for fp32 still have their quotient.
template <int LPT>
__device__ __forceinline__ float weight_of(const RouteParams& p, bool chosen, float x, float m,
                                           float sum) {
    float w = 0.0f;
    if (p.renormalise) {
        float top = chosen ? x : neg_inf();
#pragma unroll
        for (int o = LPT / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, o));
        if (chosen) {
            if (p.softmax) w = x == top ? 1.0f : expf(x - top);
            else w = x >= 0.0f ? 1.0f / (1.0f + expf(-x)) : expf(x - fminf(top, 0.0f)) / (1.0f + expf(x));
        }
        const float total = lane_sum<LPT>(w);
        w = total > 0.0f ? w / total : 0.0f;
    } else if (chosen) {
        w = p.softmax ? (x == m ? 1.0f : expf(x - m)) / sum : 1.0f / (1.0f + expf(-x));
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
            Pack<T, N> v;
            const bool in = live && e < p.experts;
            if (in) v = *reinterpret_cast<const Pack<T, N>*>(row + e);
#pragma unroll
            for (int i = 0; i < N; ++i) x[j + i] = in ? to_float(v.v[i]) : neg_inf();
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

// LPT lanes per token, VPL experts per lane.
template <class T, int LPT, int VPL>
__global__ void __launch_bounds__(kRouteThreads) route_kernel(const RouteParams p) {
    const int lane = threadIdx.x % LPT;
    const int64_t t = (static_cast<int64_t>(blockIdx.x) * kRouteThreads + threadIdx.x) / LPT;
    const bool live = t < p.tokens && (!p.mask || p.mask[t] != 0);
    float x[VPL];
    load_row<T, LPT, VPL>(p, t, lane, live, x);

    // the row's maximum and sum, for softmax weights
    float m = 0.0f, sum = 1.0f;
    if (p.softmax && !p.renormalise) {
        m = neg_inf();
#pragma unroll
        for (int j = 0; j < VPL; ++j) m = fmaxf(m, x[j]);
#pragma unroll
        for (int o = LPT / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFullMask, m, o));
        sum = 0.0f;
#pragma unroll
        for (int j = 0; j < VPL; ++j)
            sum += x[j] == neg_inf() ? 0.0f : x[j] == m ? 1.0f : __expf(x[j] - m);
        sum = lane_sum<LPT>(sum);
    }

    float b[VPL];
    if (p.bias) {
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            const int e = lane * VPL + j;
            b[j] = e < p.experts ? p.bias[e] : 0.0f;
        }
    }
    const bool by_sums = p.groups > 1 && (p.bias || p.group_top == 2);
    int id;
    float xid;
    bool doubt = false;
    {
        uint32_t key[VPL];
        if (p.bias || by_sums) {
            float c[VPL];
            scores_of<float, LPT, VPL>(x, p.softmax, c);
#pragma unroll
            for (int j = 0; j < VPL; ++j) {
                if (p.bias) c[j] += b[j];
                key[j] = x[j] == neg_inf() ? 0u : choice_key(p.bias ? c[j] : x[j]);
            }
            if (p.groups > 1) doubt = keep_groups<float, LPT, VPL>(p, lane, c, key);
        } else {
#pragma unroll
            for (int j = 0; j < VPL; ++j) key[j] = choice_key(x[j]);
            if (p.groups > 1) keep_groups<float, LPT, VPL>(p, lane, x, key);   // exact: no doubt
        }
        doubt |= take_best<LPT, VPL>(key, x, p.k, lane, p.bias != nullptr, id, xid);
    }
    if (__any_sync(kFullMask, doubt)) {
        uint64_t key[VPL];
        double c[VPL];
        scores_of<double, LPT, VPL>(x, p.softmax, c);
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            if (p.bias) c[j] += static_cast<double>(b[j]);
            key[j] = x[j] == neg_inf() ? 0ull : choice_key(p.bias ? c[j] : static_cast<double>(x[j]));
        }
        if (p.groups > 1) keep_groups<double, LPT, VPL>(p, lane, c, key);
        take_best<LPT, VPL>(key, x, p.k, lane, false, id, xid);
    }
    const float w = weight_of<LPT>(p, id >= 0, xid, m, sum);
    if (t < p.tokens && lane < p.k) {
        p.ids[t * p.k + lane] = id;
        p.weights[t * p.k + lane] = w;
    }
}

// Lists by expert, one block per expert: how many choices are below it, then
// its own in order.
__global__ void __launch_bounds__(256) lists_kernel(const int32_t* __restrict__ ids, int n,
                                                    int experts, int32_t* start, int32_t* slots) {
    __shared__ int sh[8], sh_base;
    const int e = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int below = 0;
    for (int i = threadIdx.x; i < n; i += 256) {
        const int v = ids[i];
        below += v >= 0 && v < e;
    }
    below = __reduce_add_sync(kFullMask, below);
    if (lane == 0) sh[warp] = below;
    __syncthreads();
    if (threadIdx.x == 0) {
        int s = 0;
        for (int w = 0; w < 8; ++w) s += sh[w];
        sh_base = s;
        start[e] = s;
    }
    __syncthreads();
    int at = sh_base;
    if (e == experts) return;
    for (int i0 = 0; i0 < n; i0 += 256) {
        const int i = i0 + threadIdx.x;
        const bool mine = i < n && ids[i] == e;
        const unsigned b = __ballot_sync(kFullMask, mine);
        if (lane == 0) sh[warp] = __popc(b);
        __syncthreads();
        int before = 0, all = 0;
        for (int w = 0; w < 8; ++w) {
            before += w < warp ? sh[w] : 0;
            all += sh[w];
        }
        if (mine) slots[at + before + __popc(b & ((1u << lane) - 1u))] = i;
        at += all;
        __syncthreads();
    }
}

// Gradient of the logits, LPT lanes per token as in the forward pass.  With w =
// scale * s (s a softmax p): dx_e = scale * p_e (g_e - sum_j g_j p_j); sigmoid:
// dx_e = scale * g_e s_e (1 - s_e).  Renormalised over the chosen (w = scale * s /
// S): dx_j = w_j (g_j - sum_i g_i w_i / scale), for a sigmoid times 1 - s_j.
template <class T, int LPT, int VPL>
__global__ void __launch_bounds__(kRouteThreads)
    route_backward_kernel(const RouteParams p, const float* __restrict__ grad, T* out,
                          int64_t out_stride) {
    const int lane = threadIdx.x % LPT, base = (threadIdx.x & 31) - lane;
    const int64_t t = (static_cast<int64_t>(blockIdx.x) * kRouteThreads + threadIdx.x) / LPT;
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
    // the logit of each chosen expert, from the lane that holds it
    float xid = neg_inf();
    for (int r = 0; r < p.k; ++r) {
        const int e = __shfl_sync(kFullMask, id, base + r);
        float v = neg_inf();
#pragma unroll
        for (int j = 0; j < VPL; ++j)
            if (e == lane * VPL + j) v = x[j];
        v = __shfl_sync(kFullMask, v, base + (e < 0 ? 0 : e / VPL));
        if (lane == r) xid = v;
    }
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
        sum = 0.0f;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            d[j] = x[j] == neg_inf() ? 0.0f : x[j] == m ? 1.0f : __expf(x[j] - m);
            sum += d[j];
        }
        sum = lane_sum<LPT>(sum);
    } else {
#pragma unroll
        for (int j = 0; j < VPL; ++j) d[j] = 0.0f;
    }
    RouteParams q = p;
    q.scale = 1.0f;
    const float w = weight_of<LPT>(q, chosen, xid, m, sum);
    const float dot = (p.softmax || p.renormalise) ? lane_sum<LPT>(g * w) : 0.0f;
    if (whole) {
        const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
        for (int j = 0; j < VPL; ++j) d[j] *= inv * p.scale;
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
        if (!p.softmax) v *= 1.0f / (1.0f + expf(xid));   // 1 - s
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
            Pack<T, N> v;
#pragma unroll
            for (int i = 0; i < N; ++i) v.v[i] = from_float<T>(d[j + i]);
            if (e < p.experts) *reinterpret_cast<Pack<T, N>*>(row + e) = v;
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (e + i < p.experts) row[e + i] = from_float<T>(d[j + i]);
        }
    }
}

// Calls fn(LPT, VPL) as integral constants for a router: as few lanes per
// token as hold its experts one each and its k choices.
template <class Fn>
cudaError_t with_layout(int experts, Fn&& fn) {
    using std::integral_constant;
    if (experts <= 8) return fn(integral_constant<int, 8>{}, integral_constant<int, 1>{});
    if (experts <= 16) return fn(integral_constant<int, 16>{}, integral_constant<int, 1>{});
    if (experts <= 32) return fn(integral_constant<int, 32>{}, integral_constant<int, 1>{});
    if (experts <= 64) return fn(integral_constant<int, 32>{}, integral_constant<int, 2>{});
    if (experts <= 128) return fn(integral_constant<int, 32>{}, integral_constant<int, 4>{});
    if (experts <= 256) return fn(integral_constant<int, 32>{}, integral_constant<int, 8>{});
    if (experts <= 512) return fn(integral_constant<int, 32>{}, integral_constant<int, 16>{});
    return fn(integral_constant<int, 32>{}, integral_constant<int, 32>{});
}

int pack_elems(int experts, size_t es) {   // elements of one load of load_row()
    int vpl = 1;
    while (vpl * 32 < experts) vpl *= 2;
    return vpl * es >= 16 ? static_cast<int>(16 / es) : vpl;
}

bool packed_rows(const void* p, int64_t stride, int experts, size_t es) {
    const size_t n = pack_elems(experts, es);
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
    p.vec = packed_rows(logits, stride, r->experts, type_bytes(r->type));
    return ST_OK;
}

}  // namespace
}  // namespace mflat_cu

using namespace mflat_cu;

extern "C" size_t mflat_cu_route_workspace(const mflat_cu_router_t* r, int tokens) {
    (void)r;
    (void)tokens;
    return 0;
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
    CU_TRY(with_type(r->type, [&](auto zero) {
        using T = decltype(zero);
        return with_layout(r->experts, [&](auto lpt, auto vpl) {
            constexpr int L = decltype(lpt)::value, V = decltype(vpl)::value;
            route_kernel<T, L, V><<<blocks_for(static_cast<int64_t>(tokens) * L, kRouteThreads),
                                    kRouteThreads, 0, st>>>(p);
            return cudaGetLastError();
        });
    }), "route launch");
    if (start) {
        lists_kernel<<<r->experts + 1, 256, 0, st>>>(ids, tokens * r->k, r->experts, start, slots);
        CU_TRY(cudaGetLastError(), "lists launch");
    }
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
    p.vec = p.vec && packed_rows(grad, grad_stride, r->experts, type_bytes(r->type));
    p.ids = const_cast<int32_t*>(ids);
    CU_TRY(with_type(r->type, [&](auto zero) {
        using T = decltype(zero);
        return with_layout(r->experts, [&](auto lpt, auto vpl) {
            constexpr int L = decltype(lpt)::value, V = decltype(vpl)::value;
            route_backward_kernel<T, L, V>
                <<<blocks_for(static_cast<int64_t>(tokens) * L, kRouteThreads), kRouteThreads, 0, st>>>(
                    p, grad_weights, static_cast<T*>(grad), grad_stride);
            return cudaGetLastError();
        });
    }), "route backward launch");
    return ST_OK;
}
