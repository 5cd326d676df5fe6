// beam.cu -- beam search: the k best continuations over beams x vocabulary, and
// the reordering of states by parent beam.
//
// Selection.  key[w, v] = cum[w] + ((x[w, v] - m_w) - log sum_v exp(x[w, v] - m_w)).  Within
// a beam the order is the logits' own, exact in any precision; between beams it
// hangs on the sums.  So each row first yields its k best logits (ties to the lower
// token) and its sum from fp32 exponentials of a known error; the rows of a sequence
// are merged by their keys (ties to the lower beam), and where two beams' keys come
// closer than their errors those beams' sums are formed again from 64-bit terms, in an
// order and about a reference (the row's largest logit) that the row's values alone
// decide: equal rows get equal keys wherever they start.  Next to a cum of 1e12, or
// among logits of 1e-18, keys of different logits are equal too, and lists by logits
// need not hold the lowest tokens of the last key: those come from whole rows.
//
// 64 x 8 rows of 128,000 bf16 logits (131 MB, 20.5 us for a plain read) take 33.4 us in the
// row pass: 22.3 for loads and maxima, 4.4 for the exponentials (15 us of the special
// function units, mostly beside the loads), 6.6 for floors, packs set aside and lists.
// The merge adds 5 to 6 us of dependent exchanges, at any size without close beams.
//
// These paths are slower, and right for any values:
// - Close beams: a sequence's one merge block reads their rows again, one by one, with a
//   64-bit exponential a logit.  With one pair of equal beams among the 64 x 8 the call takes
//   400 us, with all beams equal 2.3 ms (1 x 4 x 32,000: 86 and 159 us).  Random logits
//   meet it rarely: none of 40 inputs of that size did (39.1 us, 39.4 at most).
// - Equal keys of different logits at the last place: the same second sum, then the rows
//   from their start.  64 x 1 x 128,000 with a cum of -3.4e38 take 168 us for 15.
// - k above 32: the floor is the least of the warps' (k / 8)-th maxima, which many packs of
//   a long segment reach.  Where they are more than kPackMax, it is read six times more
//   (segment_exact): 64 x 8 x 128,000 take 50 us at k = 40, 300 at 48, 350 at 64 and 940 at
//   128, 4 x 64 rows of that length 47, 755, 790 and 1400, 16 x 16 x 262,144 1.5 ms at 33.
// - More candidates over the merge's floor than kListMax: every place is a pass over all
//   of them.  1 x 64 x 50,257 take 26 us at k = 16, 180 at 96 and 2.5 ms at 128.
#include <cuda_runtime.h>

#include <climits>
#include <cstdio>

#include "mflat_cuda.h"
#include "select_ops.cuh"

namespace mflat_cu {
namespace {

constexpr int kMaxBeams = 64, kMaxBeamK = 128, kMaxVocab = 1 << 30;
constexpr int kRowThreads = 256, kRowWarps = kRowThreads / 32;
constexpr size_t round256(size_t n) { return (n + 255) & ~size_t(255); }
constexpr int kListMax = 1024;      // candidates that a block filters into shared memory
constexpr int kHeld = 4;            // candidates a thread of the merge holds
constexpr int kPackMax = 512;       // 16-byte packs set aside on the way

struct BeamParams {
    const void* logits;
    int64_t stride;
    const float* cum;
    const uint8_t* finished;
    int batch, beams, vocab, k, eos;
    int splits, per_split;      // segments of a row, and 16-byte packs in each
    int rounds;                 // ceil(k / warps of a block)
    uint64_t* cand;             // workspace, [rows][splits][k]: (logit key, ~token), best first, 0: none
    double* part_sum;           // [rows][splits]: sum of exp(x - part_ref)
    double* part_ref;
    int32_t* parents;
    int32_t* tokens;
    float* scores;
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.6931471805599453094;
// Logits beyond this leave the fast path: above it, or a segment with none above
// kLow (the gap between the two is far below any sum's last digit).
constexpr float kWild = 5e5f, kLow = -4e5f;
// Powers of 2 that a thread's largest logit may lie above its sum's reference.
constexpr float kAbove = 8.0f;

// 16 bytes of logits: as pairs of floats, and their maximum (which passes over NaN).
template <class T>
struct Logits {
    static constexpr int N = 16 / sizeof(T);
    uint4 raw;
    __device__ __forceinline__ float2 pair(int i) const {
        const uint32_t* u = reinterpret_cast<const uint32_t*>(&raw);
        if constexpr (sizeof(T) == 4) {
            return make_float2(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1]));
        } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
            return make_float2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
        } else {
            return __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        }
    }
    __device__ __forceinline__ float at(int i) const {
        const float2 f = pair(i >> 1);
        return (i & 1) ? f.y : f.x;
    }
    __device__ __forceinline__ float largest() const {
        if constexpr (sizeof(T) == 4) {
            const float2 a = pair(0), b = pair(1);
            return fmaxf(fmaxf(a.x, a.y), fmaxf(b.x, b.y));
        } else {
            using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
            const T2* h = reinterpret_cast<const T2*>(&raw);
            const T2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
            return fmaxf(to_float(m.x), to_float(m.y));
        }
    }
    __device__ __forceinline__ void fill(float v) {
        T t[N];
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = from_float<T>(v);
        raw = *reinterpret_cast<const uint4*>(t);
    }
};

// One add per thread, as written (few threads come here at a time, so gathering a
// warp's adds first costs more than it saves).
__device__ __forceinline__ int shared_add(int* p, int v) {
    int old;
    asm volatile("atom.shared.add.s32 %0, [%1], %2;"
                 : "=r"(old)
                 : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(v)
                 : "memory");
    return old;
}

// Bound of the relative error of a row's sum of exponentials, which is the
// absolute error of its logarithm.  ex2 is off by 2^-22; t = x log2(e) - ref rounds by half
// a step of itself: 2^-24 |x - m| as a relative error of the term where t < 0, which
// weighted by the term's share of the sum averages at most ln(vocab), and 2^-24 (kAbove + 1)
// ln 2 where t > 0; log2(e) in fp32 adds 2^-26 |x|.  A thread adds at most 64 terms in fp32,
// up to 4 in a row by twos and then 8 such parts (13 steps of 2^-24), all else is in
// 64 bits.
__device__ __forceinline__ float sum_error(float m, int vocab) {
    const float ln_v = __logf(static_cast<float>(vocab)) + 1.0f;
    return 2.4e-7f + 7.8e-7f + 3.8e-7f + 8e-8f * ln_v + 2e-8f * fabsf(m);
}

// a * 2^n for n <= 0.
__device__ __forceinline__ double scale_down(double a, int n) {
    return n < -1000 ? 0.0 : a * __longlong_as_double(static_cast<long long>(1023 + n) << 52);
}

// Ranks n entries by counting, for each, the better ones, eight threads an entry:
// put(rank, i) is called for every entry whose rank is below most.
template <class Better, class Put>
__device__ __forceinline__ void rank_into(int n, int most, Better better, Put put) {
    const int part = threadIdx.x & 7;
    for (int i0 = 0; i0 < n; i0 += kRowThreads / 8) {
        const int i = i0 + (threadIdx.x >> 3);
        const bool want = i < n;
        if (!__any_sync(kFullMask, want)) continue;
        int rank = 0;
        if (want)
            for (int j = part; j < n; j += 8) rank += better(j, i) ? 1 : 0;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) rank += __shfl_xor_sync(kFullMask, rank, o);
        if (want && part == 0 && rank < most) put(rank, i);
    }
}

// The rounds-th largest of a warp's keys (one a lane); lane r < 4 also gets the
// (r + 1)-th largest in `four` where there are as many rounds.
__device__ __forceinline__ uint32_t warp_floor(uint32_t mine, int rounds, uint32_t& four) {
    uint32_t t = 0;
    const int lane = threadIdx.x & 31;
    for (int r = 0; r < rounds; ++r) {
        t = __reduce_max_sync(kFullMask, mine);
        if (lane == r) four = t;
        const unsigned who = __ballot_sync(kFullMask, mine == t);
        if (lane == __ffs(who) - 1) mine = 0;
    }
    return t;
}

// Floor under the k best of what a block holds, from its threads' largest keys: at
// least k of those reach it.  k <= 32: the k-th largest of the 8 warps' four largest
// (a 32-lane bitonic sort in every warp; on random data about k entries reach it).
// Above: the least of the warps' rounds-th largest.  One block barrier; calls in a
// row pass sh of alternating halves.
struct FloorShared {
    uint32_t top[kRowWarps][4];
};
__device__ __forceinline__ uint32_t block_floor(uint32_t mine, int k, int rounds, FloorShared& sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (k <= 32) {
        uint32_t four = 0;
        warp_floor(mine, 4, four);
        // the fours come sorted: every other one backwards is the sort's third step
        if (lane < 4) sh.top[warp][(warp & 1) ? 3 - lane : lane] = four;
        __syncthreads();
        uint32_t v = sh.top[lane >> 2][lane & 3];
#pragma unroll
        for (int size = 8; size <= 32; size <<= 1)
#pragma unroll
            for (int o = size >> 1; o > 0; o >>= 1) {
                const uint32_t c = __shfl_xor_sync(kFullMask, v, o);
                const bool larger = ((lane & size) == 0) == ((lane & o) == 0);
                v = larger == (c > v) ? c : v;
            }
        return __shfl_sync(kFullMask, v, k - 1);
    }
    uint32_t unused = 0;
    const uint32_t t = warp_floor(mine, rounds, unused);
    if (lane == 0) sh.top[warp][0] = t;
    __syncthreads();
    uint32_t f = sh.top[0][0];
#pragma unroll
    for (int w = 1; w < kRowWarps; ++w) f = sh.top[w][0] < f ? sh.top[w][0] : f;
    return f;
}

template <class V, class Op>
__device__ V block_reduce(V v, Op op, V* sh) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(kFullMask, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh[0];
    for (int w = 1; w < kRowWarps; ++w) v = op(v, sh[w]);
    return v;
}

// The segment [t0, t1) of a row for any values: the k best by a radix select of the
// k-th key and an ordered pass for the lowest tokens among its equals, and with
// `sums` the sum from 64-bit terms.  For NaN or infinities among the logits and sizes
// beyond kWild (with sums), and for more equals than the lists hold.  `list` is scratch
// of at least k entries.
template <class T>
__device__ __noinline__ void segment_exact(const BeamParams& p, const T* row, int t0, int t1,
                                           int64_t part, bool sums, uint64_t* list) {
    __shared__ int hist[256];
    __shared__ double sh_d[kRowWarps];
    __shared__ int sh_count[kRowWarps];
    __shared__ uint32_t sh_prefix;
    __shared__ int sh_left, sh_n;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float m = neg_inf();
    int valid = 0;
    for (int v = t0 + threadIdx.x; v < t1; v += kRowThreads) {
        const float x = to_float(row[v]);
        m = fmaxf(m, x);
        valid += x > neg_inf() ? 1 : 0;
    }
    m = block_reduce(m, [](float a, float b) { return fmaxf(a, b); }, reinterpret_cast<float*>(sh_d));
    valid = block_reduce(valid, [](int a, int b) { return a + b; }, sh_count);
    if (sums) {
        double sum = 0.0;
        for (int v = t0 + threadIdx.x; v < t1; v += kRowThreads) {
            const float x = to_float(row[v]);
            if (x > neg_inf()) sum += x == m ? 1.0 : exp(static_cast<double>(x) - m);
        }
        sum = block_reduce(sum, [](double a, double b) { return a + b; }, sh_d);
        if (threadIdx.x == 0) {
            p.part_ref[part] = m;
            p.part_sum[part] = sum;
        }
    }
    const int want = min(p.k, valid);
    uint64_t* out = p.cand + part * p.k;
    for (int j = want + threadIdx.x; j < p.k; j += kRowThreads) out[j] = 0;
    if (threadIdx.x == 0) {
        sh_prefix = 0;
        sh_left = want;
        sh_n = 0;
    }
    if (want == 0) return;
    uint32_t mask = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += kRowThreads) hist[i] = 0;
        __syncthreads();
        const uint32_t prefix = sh_prefix;
        for (int v0 = t0; v0 < t1; v0 += kRowThreads) {
            const int v = v0 + threadIdx.x;
            const uint32_t key = v < t1 ? choice_key(to_float(row[v])) : 0u;
            const bool in = key != 0u && (key & mask) == prefix;
            const unsigned who = __ballot_sync(kFullMask, in);
            if (!in) continue;
            const unsigned d = (key >> shift) & 255u;
            // a warp of one digit (ties) adds once
            int same;
            __match_all_sync(who, d, &same);
            if (!same) atomicAdd(&hist[d], 1);
            else if (lane == __ffs(who) - 1) atomicAdd(&hist[d], __popc(who));
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            int left = sh_left, d = 255;
            while (d > 0 && hist[d] < left) left -= hist[d--];
            sh_prefix = prefix | (static_cast<uint32_t>(d) << shift);
            sh_left = left;
        }
        mask |= 255u << shift;
        __syncthreads();
    }
    const uint32_t cut = sh_prefix;
    const int ties = sh_left;
    int seen = 0;
    for (int v0 = t0; v0 < t1; v0 += kRowThreads) {
        const int v = v0 + threadIdx.x;
        const uint32_t key = v < t1 ? choice_key(to_float(row[v])) : 0u;
        const unsigned eq = __ballot_sync(kFullMask, key == cut);
        __syncthreads();
        if (lane == 0) sh_count[warp] = __popc(eq);
        __syncthreads();
        int rank = seen + __popc(eq & ((1u << lane) - 1u));
        for (int w = 0; w < kRowWarps; ++w) {
            rank += w < warp ? sh_count[w] : 0;
            seen += sh_count[w];
        }
        if (key > cut || (key == cut && rank < ties))
            list[shared_add(&sh_n, 1)] = (static_cast<uint64_t>(key) << 32) | (0xffffffffu - static_cast<uint32_t>(v));
    }
    __syncthreads();
    rank_into(want, want, [&](int j, int i) { return list[j] > list[i]; },
              [&](int rank, int i) { out[rank] = list[i]; });
}

// One segment of one row: its k best logits and its share of the sum.  The segment
// is read once, PACKS packs of 16 bytes a thread at a time.  The threads' largest
// logits so far give a floor under the k best (block_floor), raised after chunks 1, 4
// and the last: only packs that reach it are set aside, few in later chunks, and looked
// through at the end.
template <class T, int PACKS>
__global__ void __launch_bounds__(kRowThreads, 4) beam_segment_kernel(const __grid_constant__ BeamParams p) {
    constexpr int N = Logits<T>::N, kChunk = PACKS * kRowThreads;
    __shared__ uint64_t list[kListMax];
    __shared__ uint4 packs[kPackMax];
    __shared__ int pack_token[kPackMax];
    __shared__ FloorShared sh_floor[2];
    __shared__ double sh_sum[kRowWarps];
    __shared__ int sh_ref[kRowWarps];
    __shared__ uint32_t sh_top[kRowWarps];
    __shared__ int sh_packs, sh_n, sh_odd;
    const int64_t r = blockIdx.x / p.splits;
    const int s = blockIdx.x % p.splits;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if ((p.finished && p.finished[r]) || !isfinite(p.cum[r])) return;
    if (threadIdx.x == 0) { sh_packs = 0; sh_n = 0; sh_odd = 0; }
    const T* row = static_cast<const T*>(p.logits) + r * p.stride;
    // packs are counted from the 16-byte boundary at or below the row's start
    const int skew = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    const int start = s * p.per_split * N - skew;
    const int t0 = start + static_cast<int>(threadIdx.x) * N;
    auto token_of = [&](int c, int q) { return t0 + (c * PACKS + q) * (kRowThreads * N); };
    auto load = [&](int c, Logits<T> (&v)[PACKS]) {
        if ((c + 1) * kChunk <= p.per_split && start + c * kChunk * N >= 0 &&
            start + (c + 1) * kChunk * N <= p.vocab) {
#pragma unroll
            for (int q = 0; q < PACKS; ++q)
                v[q].raw = __ldcs(reinterpret_cast<const uint4*>(row + token_of(c, q)));
            return;
        }
#pragma unroll
        for (int q = 0; q < PACKS; ++q) {
            const int e = token_of(c, q);
            const bool mine = (c * PACKS + q) * kRowThreads + static_cast<int>(threadIdx.x) < p.per_split;
            v[q].fill(neg_inf());
            if (mine && e >= 0 && e + N <= p.vocab) {
                v[q].raw = __ldcs(reinterpret_cast<const uint4*>(row + e));
            } else if (mine && e < p.vocab) {           // an end of the row
                T t[N];
#pragma unroll
                for (int i = 0; i < N; ++i)
                    t[i] = e + i >= 0 && e + i < p.vocab ? row[e + i] : from_float<T>(neg_inf());
                v[q].raw = *reinterpret_cast<const uint4*>(t);
            }
        }
    };
    const int chunks = (p.per_split + kChunk - 1) / kChunk;
    float best = neg_inf(), floor_x = 0.0f;
    uint32_t floor_b = 0;
    double sum = 0.0;
    float ref = 0.0f;           // a whole number: sums of other references scale by powers of 2
    bool any = false, odd = false;
    int turn = 0;
    for (int c = 0; c < chunks; ++c) {
        Logits<T> v[PACKS];
        load(c, v);
        if (c + 1 == chunks) grid_release();
        float most[PACKS], m = neg_inf();
#pragma unroll
        for (int q = 0; q < PACKS; ++q) {
            most[q] = v[q].largest();
            m = fmaxf(m, most[q]);
        }
        best = fmaxf(best, m);
        odd |= m > kWild;
        if (m >= -kWild && m <= kWild) {
            const float mine = m * kLog2e;
            if (!any || mine > ref + kAbove) {
                const float now = rintf(mine);
                sum = any ? scale_down(sum, static_cast<int>(ref - now)) : 0.0;
                ref = now;
                any = true;
            }
            const float2 l2 = make_float2(kLog2e, kLog2e), shift = make_float2(-ref, -ref);
            float chunk = 0.0f;
#pragma unroll
            for (int q = 0; q < PACKS; ++q) {
                float2 part = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int i = 0; i < N / 2; ++i) {
                    const float2 t = fma2(v[q].pair(i), l2, shift);
                    part = add2(part, make_float2(exp2_fast(t.x), exp2_fast(t.y)));
                }
                chunk += part.x + part.y;
            }
            sum += static_cast<double>(chunk);
            odd |= chunk != chunk;      // NaN among the logits
        }
        if (c == 0 || c == 3 || c + 1 == chunks) {
            floor_b = block_floor(choice_key(best), p.k, p.rounds, sh_floor[turn & 1]);
            ++turn;
            // everything above -inf where fewer than k were seen
            floor_x = floor_b == 0u ? -3.402823466e38f : key_value(floor_b);
        }
#pragma unroll
        for (int q = 0; q < PACKS; ++q) {
            if (most[q] >= floor_x) {
                const int at = shared_add(&sh_packs, 1);
                if (at < kPackMax) {
                    packs[at] = v[q].raw;
                    pack_token[at] = token_of(c, q);
                }
            }
        }
    }
    // the block's largest logit and sum
    const uint32_t top_w = __reduce_max_sync(kFullMask, choice_key(best));
    const int ref_w = __reduce_max_sync(kFullMask, any ? static_cast<int>(ref) : INT_MIN / 2);
    if (any) sum = scale_down(sum, static_cast<int>(ref) - ref_w);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFullMask, sum, o);
    if (lane == 0) {
        sh_top[warp] = top_w;
        sh_sum[warp] = sum;
        sh_ref[warp] = ref_w;
    }
    if (odd) sh_odd = 1;
    __syncthreads();
    uint32_t top = sh_top[0];
    int ref_b = sh_ref[0];
#pragma unroll
    for (int w = 1; w < kRowWarps; ++w) {
        top = max(top, sh_top[w]);
        ref_b = max(ref_b, sh_ref[w]);
    }
    const bool wild = sh_odd || (top != 0u && key_value(top) < kLow);
    if (!wild && threadIdx.x == 0) {
        double total = 0.0;
        for (int w = 0; w < kRowWarps; ++w) total += scale_down(sh_sum[w], sh_ref[w] - ref_b);
        p.part_ref[blockIdx.x] = top == 0u ? static_cast<double>(neg_inf()) : ref_b * kLn2;
        p.part_sum[blockIdx.x] = total;
    }
    const int n_packs = sh_packs;
    if (!wild && n_packs <= kPackMax) {
        for (int i = threadIdx.x; i < n_packs; i += kRowThreads) {
            Logits<T> v;
            v.raw = packs[i];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float x = v.at(j);
                if (x >= floor_x) {
                    const int at = shared_add(&sh_n, 1);
                    if (at < kListMax)
                        list[at] = (static_cast<uint64_t>(choice_key(x)) << 32) |
                                   (0xffffffffu - static_cast<uint32_t>(pack_token[i] + j));
                }
            }
        }
    }
    __syncthreads();
    const int n = sh_n;
    if (wild || n_packs > kPackMax || n > kListMax) {
        const int from = max(start, 0);
        const int to = static_cast<int>(min(static_cast<int64_t>(start) + static_cast<int64_t>(p.per_split) * N,
                                            static_cast<int64_t>(p.vocab)));
        segment_exact(p, row, from, to, blockIdx.x, wild, list);
        return;
    }
    uint64_t* out = p.cand + static_cast<int64_t>(blockIdx.x) * p.k;
    rank_into(n, p.k, [&](int j, int i) { return list[j] > list[i]; },
              [&](int rank, int i) { out[rank] = list[i]; });
    for (int j = n + threadIdx.x; j < p.k; j += kRowThreads) out[j] = 0;
}

struct Choice {
    uint64_t key;       // choice_key of cum + log p in 64 bits
    uint64_t at;        // beam, token
};
__device__ __forceinline__ bool better(const Choice& a, const Choice& b) {
    return a.key > b.key || (a.key == b.key && a.at < b.at);
}

// A sequence's beams in the merge.
struct Beams {
    double cum[kMaxBeams];      // NaN: no candidates
    double log[kMaxBeams];      // log sum exp(x - ref)
    double ref[kMaxBeams];      // -inf: finished
    float off[kMaxBeams];       // error of the keys; 0: settled by the row's values alone
    int redo[kMaxBeams];
    int again, fill;

    // where there are logits of +inf only they count, key = cum - log(how many)
    __device__ __forceinline__ double key_of(int w, float x) const {
        const double r = ref[w];
        double d = static_cast<double>(x) - r;
        if (r == static_cast<double>(-neg_inf())) d = x == -neg_inf() ? 0.0 : static_cast<double>(neg_inf());
        return cum[w] + (d - log[w]);
    }
    __device__ __forceinline__ double error_of(const Choice& c) const {
        return off[c.at >> 32] + 0x1p-51 * fabs(key_value(c.key));
    }
    // how far two keys of a beam can be off from one another by their roundings
    __device__ __forceinline__ double rounding(int w, double key) const {
        return 0x1p-48 * fabs(cum[w]) + 0x1p-49 * fabs(key);
    }
};

// Neighbours in the order, x before y, that may be equal or the other way round.
template <class T>
__device__ __forceinline__ void beams_near(const BeamParams& p, Beams& sh, int64_t b, const Choice& x, const Choice& y) {
    const int u = static_cast<int>(x.at >> 32), w = static_cast<int>(y.at >> 32);
    if (sh.off[u] == 0.0f && sh.off[w] == 0.0f) return;
    if (u == w) {
        const T* row = static_cast<const T*>(p.logits) + (b * p.beams + u) * p.stride;
        if (to_float(row[x.at & 0xffffffffu]) == to_float(row[y.at & 0xffffffffu])) return;
    }
    sh.redo[u] = sh.redo[w] = 1;
    sh.again = 1;
}

// The thread's candidates that are their segments' k-th and reach the last key: if the
// logits next to one give the same key, the segment may hold others of that key.
template <class T>
__device__ __forceinline__ void segments_full(const BeamParams& p, Beams& sh, const uint64_t* cand, int first, int total,
                                              uint64_t last) {
    constexpr uint32_t kStep = std::is_same_v<T, float> ? 1u : std::is_same_v<T, __half> ? 1u << 13 : 1u << 16;
    for (int i = first; i < total; i += kRowThreads) {
        const int w = i / (p.splits * p.k);
        if (i % p.k != p.k - 1 || sh.cum[w] != sh.cum[w] || isinf(sh.ref[w])) continue;
        const uint32_t at = static_cast<uint32_t>(cand[i] >> 32);
        if (at == 0u) continue;
        const double key = sh.key_of(w, key_value(at)), most = sh.off[w] == 0.0f ? 0.0 : sh.rounding(w, key);
        if (choice_key(key) < last) continue;
        if (!(key - sh.key_of(w, key_value(at - kStep)) <= most || sh.key_of(w, key_value(at + kStep)) - key <= most))
            continue;
        if (sh.off[w] == 0.0f) {
            sh.fill = 1;
        } else {
            sh.redo[w] = 1;
            sh.again = 1;
        }
    }
}

// The places of the last key, from the whole rows of the beams that have it (redo): beam
// by beam, token by token.
template <class T>
__device__ __forceinline__ void fill_last_key(const BeamParams& p, const Beams& sh, int64_t b, Choice* best) {
    __shared__ int hits[kRowWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint64_t key = best[p.k - 1].key;
    int filled = __syncthreads_count(threadIdx.x < p.k && best[threadIdx.x].key > key);
    for (int w = 0; w < p.beams && filled < p.k; ++w) {
        if (!sh.redo[w]) continue;
        const uint64_t beam = static_cast<uint64_t>(w) << 32;
        if (sh.ref[w] == static_cast<double>(neg_inf())) {
            if (threadIdx.x == 0) best[filled] = Choice{key, beam | static_cast<uint32_t>(p.eos)};
            ++filled;
            continue;
        }
        const T* row = static_cast<const T*>(p.logits) + (b * p.beams + w) * p.stride;
        for (int v0 = 0; v0 < p.vocab && filled < p.k; v0 += kRowThreads) {
            const int v = v0 + threadIdx.x;
            const float x = v < p.vocab ? to_float(row[v]) : neg_inf();
            const bool hit = x > neg_inf() && choice_key(sh.key_of(w, x)) == key;
            const unsigned who = __ballot_sync(kFullMask, hit);
            __syncthreads();
            if (lane == 0) hits[warp] = __popc(who);
            __syncthreads();
            int place = filled + __popc(who & ((1u << lane) - 1u));
            for (int i = 0; i < kRowWarps; ++i) {
                place += i < warp ? hits[i] : 0;
                filled += hits[i];
            }
            if (hit && place < p.k) best[place] = Choice{key, beam | static_cast<uint32_t>(v)};
        }
    }
    __syncthreads();
}

// One sequence: its beams' sums, then the k best of the segments' candidates.  Few
// blocks run, so the time is the chain of loads and exchanges: all loads start
// together, and the first kHeld candidates of a thread stay in registers.
template <class T>
__global__ void __launch_bounds__(kRowThreads) beam_merge_kernel(const __grid_constant__ BeamParams p) {
    __shared__ Beams sh;
    __shared__ Choice list[kListMax];
    __shared__ Choice best[kMaxBeamK];
    __shared__ FloorShared sh_floor;
    __shared__ double sh_sum[kRowWarps];
    __shared__ int sh_n;
    const int64_t b = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per_beam = p.splits * p.k, total = p.beams * per_beam;
    const uint64_t* cand = p.cand + b * total;
    int lanes = 1;              // lanes that hold a segment's sum
    while (lanes < 32 && lanes < p.splits) lanes *= 2;
    // a warp takes every 8th candidate, of all beams: the floor is the better, the more
    // evenly the best ones lie over the warps
    const int first = lane * kRowWarps + warp;
    uint32_t ends = 0;          // held ones that are their segments' k-th
#pragma unroll
    for (int j = 0; j < kHeld; ++j) ends |= (j * kRowThreads + first) % p.k == p.k - 1 ? 1u << j : 0u;
    grid_wait();
    uint64_t held[kHeld];
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
        const int i = j * kRowThreads + first;
        held[j] = i < total ? cand[i] : 0;
    }
    for (int w = warp; w < p.beams; w += kRowWarps) {
        const int64_t r = b * p.beams + w;
        const double none = static_cast<double>(neg_inf());
        double f = none, part = 0.0;
        if (lane < p.splits) {
            f = p.part_ref[r * p.splits + lane];
            part = p.part_sum[r * p.splits + lane];
        }
        const float cum = p.cum[r];
        const bool done = p.finished && p.finished[r];
        double base = __longlong_as_double(0x7ff8000000000000ll), log_sum = 0.0, sum = 0.0;
        double ref = none;
        if (isfinite(cum) && !done) {       // else its segments wrote nothing
            ref = f;
            for (int s = lane + 32; s < p.splits; s += 32) ref = fmax(ref, p.part_ref[r * p.splits + s]);
            for (int o = lanes / 2; o > 0; o >>= 1) ref = fmax(ref, __shfl_xor_sync(kFullMask, ref, o));
            ref = __shfl_sync(kFullMask, ref, 0);
            for (int s = lane; s < p.splits; s += 32) {
                if (s != lane) {
                    f = p.part_ref[r * p.splits + s];
                    part = p.part_sum[r * p.splits + s];
                }
                if (f > none) sum += f == ref ? part : part * exp(f - ref);
            }
            for (int o = lanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(kFullMask, sum, o);
            if (ref > none) {
                base = cum;
                log_sum = log(sum);
            }
        } else if (isfinite(cum)) {
            base = cum;
        }
        if (lane == 0) {
            sh.cum[w] = base;
            sh.log[w] = log_sum;
            sh.ref[w] = ref;
            // beyond kWild segment_exact's sums: up to 2^22 64-bit additions in a row, in an
            // order that hangs on where the row starts.  A key's two differences and its sum
            // round by 2^-53 of themselves, below 2^-51 (|cum| + |key|) together (error_of has
            // the key's part).  A finished beam's key is its cum, and infinite logits only count.
            const bool fast = ref > -2.0 * kWild && ref < 2.0 * kWild;
            const bool summed = ref > none && ref < -none;
            sh.off[w] = !summed ? 0.0f
                                : (fast ? sum_error(static_cast<float>(ref), p.vocab) : 1e-9f) +
                                      0x1p-50f * fabsf(cum);
            sh.redo[w] = 0;
        }
    }
    auto choice_of = [&](int i, uint64_t v) {
        Choice c{0, 0};
        const int w = i / per_beam;
        const double cum = sh.cum[w];
        if (cum != cum) return c;
        c.at = static_cast<uint64_t>(w) << 32;
        if (p.finished && p.finished[b * p.beams + w]) {
            if (i == w * per_beam) {
                c.key = choice_key(cum);
                c.at |= static_cast<uint32_t>(p.eos);
            }
            return c;
        }
        const uint32_t key = static_cast<uint32_t>(v >> 32);
        if (key == 0u) return c;
        const float x = key_value(key);
        c.at |= 0xffffffffu - static_cast<uint32_t>(v);
        c.key = choice_key(sh.key_of(w, x));
        return c;
    };
    Choice own[kHeld];          // the held ones' keys, formed once an attempt
    auto form = [&] {
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
            const int i = j * kRowThreads + first;
            own[j] = i < total ? choice_of(i, held[j]) : Choice{0, 0};
        }
    };
    // fn(choice) for every candidate of the thread
    auto each = [&](auto&& fn) {
#pragma unroll
        for (int j = 0; j < kHeld; ++j)
            if (own[j].key != 0) fn(own[j]);
        for (int i = kHeld * kRowThreads + first; i < total; i += kRowThreads) fn(choice_of(i, cand[i]));
    };
    for (int attempt = 0; ; ++attempt) {
        __syncthreads();
        if (threadIdx.x == 0) {
            sh_n = 0;
            sh.again = 0;
            sh.fill = 0;
        }
        form();
        // a floor under the k largest of the keys less their errors; a key that with its
        // error stays below it cannot be among the k best
        double mine = static_cast<double>(neg_inf());
        each([&](const Choice& c) {
            if (c.key != 0) mine = fmax(mine, key_value(c.key) - sh.error_of(c));
        });
        const uint32_t floor_f = block_floor(choice_key(__double2float_rd(mine)), p.k, p.rounds, sh_floor);
        const double floor_v = static_cast<double>(key_value(floor_f));
        each([&](const Choice& c) {
            if (c.key == 0 || key_value(c.key) + sh.error_of(c) < floor_v) return;
            const int at = shared_add(&sh_n, 1);
            if (at < kListMax) list[at] = c;
        });
        for (int j = threadIdx.x; j < p.k; j += kRowThreads) best[j] = Choice{0, 0};
        __syncthreads();
        const int n = min(sh_n, kListMax);
        if (sh_n <= kListMax) {
            rank_into(n, p.k, [&](int j, int i) { return better(list[j], list[i]); },
                      [&](int rank, int i) { best[rank] = list[i]; });
            __syncthreads();
        } else {
            // more equal keys than the list holds: one block-wide best per place
            Choice last{~0ull, 0};
            for (int j = 0; j < p.k; ++j) {
                Choice c{0, 0};
                each([&](const Choice& x) {
                    if (x.key != 0 && better(last, x) && better(x, c)) c = x;
                });
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    Choice x;
                    x.key = __shfl_xor_sync(kFullMask, c.key, o);
                    x.at = __shfl_xor_sync(kFullMask, c.at, o);
                    if (better(x, c)) c = x;
                }
                __syncthreads();
                if (lane == 0) list[warp] = c;
                __syncthreads();
                c = list[0];
                for (int w = 1; w < kRowWarps; ++w)
                    if (better(list[w], c)) c = list[w];
                last = c;
                if (threadIdx.x == 0) best[j] = c;
                if (c.key == 0) break;
            }
            __syncthreads();
        }
        // Two beams' candidates closer than their sums' errors, in the selection or
        // across its end: those beams' sums are formed again from 64-bit terms.  So is one
        // beam's, where keys of different logits are equal or nearly so, because next to
        // a cum of 1e12 they end at 1e-4: which of them are equal hangs on the sum too.
        const Choice last = best[p.k - 1];
        auto close = [&](const Choice& x, const Choice& y) {
            const int u = static_cast<int>(x.at >> 32), w = static_cast<int>(y.at >> 32);
            const double kx = key_value(x.key), bound = u == w ? sh.rounding(u, kx) : sh.error_of(x) + sh.error_of(y);
            // (a beam's keys this close come of equal logits, but for logits below 2^26 times
            // the bound: larger ones lie further apart, those of fewer bits all the more)
            return y.key != 0 && !(kx - key_value(y.key) > bound) &&
                   !(u == w && fabs(kx - sh.cum[u] + sh.log[u] + sh.ref[u]) > 0x1p26 * bound);
        };
        // fn(x, y) for the pairs that decide
        auto pairs = [&](auto&& fn) {
            for (int j = threadIdx.x; j + 1 < p.k; j += kRowThreads) fn(best[j], best[j + 1]);
            if (sh_n <= kListMax) {
                for (int i = threadIdx.x; i < n; i += kRowThreads)
                    if (better(last, list[i])) fn(last, list[i]);
            } else {
                each([&](const Choice& c) {
                    if (better(last, c)) fn(last, c);
                });
            }
        };
        bool doubt = false;
        pairs([&](const Choice& x, const Choice& y) { doubt |= close(x, y); });
        // A segment whose k candidates all reach the last key may hold others of that key,
        // on lower tokens.
#pragma unroll
        for (int j = 0; j < kHeld; ++j) doubt |= ((ends >> j) & 1u) != 0u && last.key != 0 && own[j].key >= last.key;
        for (int i = kHeld * kRowThreads + first; last.key != 0 && i < total; i += kRowThreads)
            doubt |= i % p.k == p.k - 1 && choice_of(i, cand[i]).key >= last.key;
        if (!__syncthreads_or(doubt)) break;
        pairs([&](const Choice& x, const Choice& y) {
            if (close(x, y)) beams_near<T>(p, sh, b, x, y);
        });
        if (last.key != 0) segments_full<T>(p, sh, cand, first, total, last.key);
        __syncthreads();
        if (!sh.again) break;           // (by the third attempt every sum has been formed again)
        for (int w = 0; w < p.beams; ++w) {
            if (attempt == 0 && !sh.redo[w]) continue;
            if (sh.off[w] == 0.0f) continue;
            const int64_t r = b * p.beams + w;
            const T* row = static_cast<const T*>(p.logits) + r * p.stride;
            // the row's largest logit: the first of its segments' candidates
            uint32_t top = 0;
            for (int i = lane; i < p.splits; i += 32)
                top = max(top, static_cast<uint32_t>(cand[(w * p.splits + i) * p.k] >> 32));
            const double m = key_value(__reduce_max_sync(kFullMask, top));
            double sum = 0.0;
            for (int v = threadIdx.x; v < p.vocab; v += kRowThreads) {
                const float x = to_float(row[v]);
                if (x > neg_inf()) sum += exp(static_cast<double>(x) - m);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFullMask, sum, o);
            __syncthreads();
            if (lane == 0) sh_sum[warp] = sum;
            __syncthreads();
            if (threadIdx.x == 0) {
                double all = 0.0;
                for (int i = 0; i < kRowWarps; ++i) all += sh_sum[i];
                sh.log[w] = log(all);
                sh.ref[w] = m;
                sh.off[w] = 0.0f;
            }
        }
    }
    if (sh.fill) {
        for (int w = threadIdx.x; w < p.beams; w += kRowThreads) sh.redo[w] = 0;
        __syncthreads();
        each([&](const Choice& c) {
            if (c.key == best[p.k - 1].key) sh.redo[c.at >> 32] = 1;
        });
        __syncthreads();
        fill_last_key<T>(p, sh, b, best);
    }
    for (int j = threadIdx.x; j < p.k; j += kRowThreads) {
        const Choice c = best[j];
        p.parents[b * p.k + j] = c.key ? static_cast<int32_t>(c.at >> 32) : -1;
        p.tokens[b * p.k + j] = c.key ? static_cast<int32_t>(c.at & 0xffffffffu) : -1;
        p.scores[b * p.k + j] = static_cast<float>(key_value(c.key));
    }
}

// Reordering in place.  A thread owns the same bytes of all the rows of a
// sequence: it reads every row that moves, then writes, so no other thread's
// writes can come before its reads.  Bound by memory: 48 x 8 x 4 rows of 8 x 51 KB, about
// 860 MB that move, in 157 us (5.5 TB/s; the counters see 930 MB, and a copy of all rows
// would move 1.3 GB).  Rows of 33 to 64 beams spill 52 bytes of a thread's 255 registers.
struct ReorderParams {
    char* states;
    const int32_t* parents;
    int64_t parent_stride;
    int outer, batch, beams, segments;
    int64_t seg_vecs;           // vectors per segment
    int64_t seg_stride, row_stride, outer_stride;   // bytes
    int64_t columns;            // segments * seg_vecs
};

constexpr int kReorderThreads = 128;

template <class V, int W>
__global__ void __launch_bounds__(kReorderThreads) reorder_kernel(const ReorderParams p) {
    __shared__ int par[W];
    const int b = blockIdx.y % p.batch;
    if (threadIdx.x < W) {
        int q = -1;
        if (threadIdx.x < p.beams) {
            q = p.parents[b * p.parent_stride + threadIdx.x];
            if (q < 0 || q >= p.beams || q == static_cast<int>(threadIdx.x)) q = -1;
        }
        par[threadIdx.x] = q;
    }
    __syncthreads();
    const int64_t col = static_cast<int64_t>(blockIdx.x) * kReorderThreads + threadIdx.x;
    if (col >= p.columns) return;
    const int64_t seg = col / p.seg_vecs, at = col % p.seg_vecs;
    for (int64_t o = blockIdx.y / p.batch; o < p.outer; o += gridDim.y / p.batch) {
        char* base = p.states + o * p.outer_stride + static_cast<int64_t>(b) * p.beams * p.row_stride +
                     seg * p.seg_stride + at * static_cast<int64_t>(sizeof(V));
        V v[W];
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (par[i] >= 0) v[i] = *reinterpret_cast<const V*>(base + par[i] * p.row_stride);
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (par[i] >= 0) *reinterpret_cast<V*>(base + i * p.row_stride) = v[i];
    }
}

template <class V>
cudaError_t launch_reorder(const ReorderParams& p, cudaStream_t st) {
    const int64_t gx = (p.columns + kReorderThreads - 1) / kReorderThreads;
    int64_t outer = p.outer;            // up to 2^31 - 1
    while (outer * p.batch > 65535) outer = (outer + 1) / 2;
    const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(outer * p.batch));
    if (p.beams <= 4) reorder_kernel<V, 4><<<grid, kReorderThreads, 0, st>>>(p);
    else if (p.beams <= 8) reorder_kernel<V, 8><<<grid, kReorderThreads, 0, st>>>(p);
    else if (p.beams <= 16) reorder_kernel<V, 16><<<grid, kReorderThreads, 0, st>>>(p);
    else if constexpr (sizeof(V) <= 8) {
        if (p.beams <= 32) reorder_kernel<V, 32><<<grid, kReorderThreads, 0, st>>>(p);
        else reorder_kernel<V, 64><<<grid, kReorderThreads, 0, st>>>(p);
    }
    return cudaGetLastError();
}

// How rows are cut.  A block holds 8 packs of 16 bytes a thread at a time (32 KB) and
// runs through its segment.  Where all segments of one chunk would not fill the
// machine twice, chunks shrink to 4, 2 or 1 packs a thread, for more blocks.  Else
// the segments are as long as leaves the busiest SM the fewest chunks, each segment
// counting one more for its floors, lists and results.
struct BeamPlan {
    int packs, splits, per_split;
    size_t cand, sum, ref, end;
};
BeamPlan beam_plan(const mflat_cu_beam_t* b, int batch) {
    const int n = static_cast<int>(16 / type_bytes(b->type));
    const int64_t rows = static_cast<int64_t>(batch) * b->beams;
    // a row may start anywhere in its first pack
    const int64_t row_packs = (static_cast<int64_t>(b->vocab) + 2 * (n - 1)) / n;
    auto chunks_of = [&](int packs) { return (row_packs + packs * kRowThreads - 1) / (packs * kRowThreads); };
    BeamPlan p{};
    p.packs = 8;
    while (p.packs > 1 && rows * chunks_of(p.packs) < 2 * 148) p.packs /= 2;
    const int64_t chunks = chunks_of(p.packs);
    double least = 1e300;
    for (int64_t s = 1; s <= chunks; ++s) {
        const double cost = static_cast<double>((rows * s + 147) / 148) *
                            (static_cast<double>(chunks) / static_cast<double>(s) + 1.0);
        if (cost < least) {
            least = cost;
            p.splits = static_cast<int>(s);
        }
        if (s >= 256) break;
    }
    p.per_split = static_cast<int>((row_packs + p.splits - 1) / p.splits);
    const size_t parts = static_cast<size_t>(rows) * p.splits;
    p.cand = 0;
    p.sum = p.cand + round256(parts * b->k * 8);
    p.ref = p.sum + round256(parts * 8);
    p.end = p.ref + round256(parts * 8);
    return p;
}

int check_beam(const mflat_cu_beam_t* b, int batch) {
    char msg[200];
    if (b->beams < 1 || b->beams > kMaxBeams) {
        std::snprintf(msg, sizeof msg, "beams=%d outside [1, %d]", b->beams, kMaxBeams);
        return fail(ST_BAD_ARG, msg);
    }
    if (b->k < 1 || b->k > kMaxBeamK) {
        std::snprintf(msg, sizeof msg, "k=%d outside [1, %d]", b->k, kMaxBeamK);
        return fail(ST_BAD_ARG, msg);
    }
    if (b->vocab < 1 || b->vocab > kMaxVocab) {
        std::snprintf(msg, sizeof msg, "vocab=%d outside [1, %d]", b->vocab, kMaxVocab);
        return fail(ST_BAD_ARG, msg);
    }
    if (b->type < 0 || b->type > 2) return fail(ST_BAD_ARG, "unknown logits type");
    if (b->eos < -1 || b->eos >= b->vocab) return fail(ST_BAD_ARG, "eos outside [-1, vocab)");
    if (batch < 0 || static_cast<int64_t>(batch) * b->beams * b->k > INT_MAX) {
        std::snprintf(msg, sizeof msg, "batch=%d: batch * beams * k must be in [0, 2^31)", batch);
        return fail(ST_BAD_ARG, msg);
    }
    return ST_OK;
}

}  // namespace
}  // namespace mflat_cu

using namespace mflat_cu;

extern "C" size_t mflat_cu_beam_workspace(const mflat_cu_beam_t* b, int batch) {
    if (check_beam(b, batch) != ST_OK) return 0;
    return beam_plan(b, batch).end;
}

extern "C" int mflat_cu_beam_select(const mflat_cu_beam_t* b, const void* logits, int64_t stride,
                                    const float* cum, const uint8_t* finished, int batch,
                                    int32_t* parents, int32_t* tokens, float* scores, void* ws,
                                    size_t ws_bytes, int device, void* stream) {
    int rc = check_beam(b, batch);
    if (rc != ST_OK) return rc;
    if (stride == 0) stride = b->vocab;
    if (stride < b->vocab) return fail(ST_BAD_ARG, "logits stride below vocab");
    if (batch > 0 && static_cast<const void*>(scores) == cum && b->k != b->beams)
        return fail(ST_BAD_ARG, "scores over the cums need k = beams");
    if (finished && b->eos < 0) return fail(ST_BAD_ARG, "finished beams need an eos token");
    if (!aligned_to(logits, type_bytes(b->type)) || !aligned_to(cum, 4) || !aligned_to(parents, 4) ||
        !aligned_to(tokens, 4) || !aligned_to(scores, 4))
        return fail(ST_BAD_ARG, "misaligned pointer");
    if (batch == 0) return ST_OK;
    const BeamPlan l = beam_plan(b, batch);
    if (static_cast<int64_t>(batch) * b->beams * l.splits > INT_MAX)
        return fail(ST_BAD_ARG, "batch * beams * vocab too large for one call");
    if (!ws || ws_bytes < l.end || !aligned_to(ws, 256))
        return fail(ST_BAD_ARG, "workspace missing, too small or not 256-byte aligned");
    rc = operator_device(device, &device);
    if (rc != ST_OK) return rc;
    DeviceGuard g(device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    char* w = static_cast<char*>(ws);
    BeamParams p{};
    p.logits = logits;
    p.stride = stride;
    p.cum = cum;
    p.finished = finished;
    p.batch = batch;
    p.beams = b->beams;
    p.vocab = b->vocab;
    p.k = b->k;
    p.eos = b->eos;
    p.splits = l.splits;
    p.per_split = l.per_split;
    p.rounds = (b->k + kRowWarps - 1) / kRowWarps;
    p.cand = reinterpret_cast<uint64_t*>(w + l.cand);
    p.part_sum = reinterpret_cast<double*>(w + l.sum);
    p.part_ref = reinterpret_cast<double*>(w + l.ref);
    p.parents = parents;
    p.tokens = tokens;
    p.scores = scores;
    CU_TRY(with_type(b->type, [&](auto zero) {
        using T = decltype(zero);
        const unsigned grid = static_cast<unsigned>(static_cast<int64_t>(batch) * b->beams * l.splits);
        switch (l.packs) {
            case 1: beam_segment_kernel<T, 1><<<grid, kRowThreads, 0, st>>>(p); break;
            case 2: beam_segment_kernel<T, 2><<<grid, kRowThreads, 0, st>>>(p); break;
            case 4: beam_segment_kernel<T, 4><<<grid, kRowThreads, 0, st>>>(p); break;
            default: beam_segment_kernel<T, 8><<<grid, kRowThreads, 0, st>>>(p); break;
        }
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
        return launch_after(beam_merge_kernel<T>, dim3(batch), kRowThreads, 0, st, p);
    }), "beam select launch");
    return ST_OK;
}

extern "C" int mflat_cu_beam_reorder(void* states, const int32_t* parents, int64_t parent_stride,
                                     int outer, int batch, int beams, int segments,
                                     int64_t segment_bytes, int64_t segment_stride,
                                     int64_t row_stride, int64_t outer_stride, int device,
                                     void* stream) {
    char msg[200];
    if (beams < 1 || beams > kMaxBeams) {
        std::snprintf(msg, sizeof msg, "beams=%d outside [1, %d]", beams, kMaxBeams);
        return fail(ST_BAD_ARG, msg);
    }
    if (outer < 0 || batch < 0 || batch > 65535 || segments < 0 || segment_bytes < 0)
        return fail(ST_BAD_ARG, "outer, batch (at most 65535), segments or segment_bytes out of range");
    if (parent_stride == 0) parent_stride = beams;
    if (parent_stride < beams) return fail(ST_BAD_ARG, "parent stride below beams");
    if (segment_stride == 0) segment_stride = segment_bytes;
    // extents in 128 bits: nothing the caller passes can wrap around
    const __int128 row = static_cast<__int128>(segments - 1) * segment_stride + segment_bytes;
    __int128 step = row_stride, far = outer_stride;
    if (step == 0) step = static_cast<__int128>(segments) * segment_stride;
    if (far == 0) far = step * beams * batch;
    if (outer == 0 || batch == 0 || segments == 0 || segment_bytes == 0) return ST_OK;
    const __int128 plane = step * (static_cast<__int128>(batch) * beams - 1) + row;
    // pieces that overlap would be read by one thread and written by another
    if (segment_stride < segment_bytes || step < row || (outer > 1 && far < plane))
        return fail(ST_BAD_ARG, "strides let the rows overlap");
    if (far * (outer - 1) + plane > (static_cast<__int128>(1) << 56))
        return fail(ST_BAD_ARG, "states span more than 2^56 bytes");
    row_stride = static_cast<int64_t>(step);
    outer_stride = outer > 1 ? static_cast<int64_t>(far) : 0;
    if (!aligned_to(parents, 4)) return fail(ST_BAD_ARG, "misaligned pointer");
    int64_t bits = segment_bytes | row_stride | static_cast<int64_t>(reinterpret_cast<uintptr_t>(states) & 15);
    if (segments > 1) bits |= segment_stride;
    bits |= outer_stride;
    // a thread holds a vector of every row: 16 bytes of up to 16 rows, else 8 (256 MB of
    // 20 or 32 rows: 5.0 and 6.1 TB/s, against 2.2 and 3.3 with 16)
    const int most = beams <= 16 ? 16 : 8;
    int vec = bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : bits % 2 == 0 ? 2 : 1;
    if (vec > most) vec = most;
    ReorderParams p{};
    p.states = static_cast<char*>(states);
    p.parents = parents;
    p.parent_stride = parent_stride;
    p.outer = outer;
    p.batch = batch;
    p.beams = beams;
    p.segments = segments;
    p.seg_vecs = segment_bytes / vec;
    p.seg_stride = segment_stride;
    p.row_stride = row_stride;
    p.outer_stride = outer_stride;
    p.columns = p.seg_vecs * segments;
    if (p.columns > (int64_t{1} << 31) * 64) return fail(ST_BAD_ARG, "row too long");
    int rc = operator_device(device, &device);
    if (rc != ST_OK) return rc;
    if (beams == 1) return ST_OK;       // a single beam is its own parent
    DeviceGuard g(device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    switch (vec) {
        case 16: e = launch_reorder<uint4>(p, st); break;
        case 8: e = launch_reorder<uint2>(p, st); break;
        case 4: e = launch_reorder<uint32_t>(p, st); break;
        case 2: e = launch_reorder<uint16_t>(p, st); break;
        default: e = launch_reorder<uint8_t>(p, st); break;
    }
    CU_TRY(e, "reorder launch");
    return ST_OK;
}
