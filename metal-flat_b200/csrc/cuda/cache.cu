// cache.cu -- eviction from a key/value cache by accumulated attention weight.
//
// acc' = acc + the sum of the group's weights, formed in twice 24 bits and then rounded
// to fp32: all but very rarely what the exact sum rounds to, so that the kept set all but
// never hangs on an order of addition.  (The order is one of the call's sizes, strides and
// alignment alone: equal calls give equal bits.)  Of a cache over its
// budget m, the kept slots are the m largest of (protected, acc'), ties to the lower
// slot: a radix select of the m-th key, then one ordered pass.  Slots of dropped
// entries below m ("holes") take the kept entries at and behind m ("tails") in
// order: sources lie behind m and targets below it, so rows move in place in any
// order.
//
// One kernel does it all: a cluster of 1 to 8 blocks owns a (sequence, head), keeps
// its sums and keys in shared memory and exchanges histograms and counts there.  Above
// 196,608 slots a head the sums wait in the workspace (250,001 slots, 2 heads, 48,000 moves
// each: 212 us, against 1.4 ms by the three kernels behind it); those three are for
// caches of more than 393,216 slots, whose keys eight blocks cannot hold.
//
// 32 x 8 caches of 4097 slots and 4 weights each, one entry leaving (25 MB, 3.9 us at the
// copy rate): 14.4 us, of which 7 sum up and the rest are the exchanges of the select.
// 4 x 8 prompts of up to 16,384 slots and 64 rows cut to 1024 (84 MB, 13 us): 38 us,
// 17 for the sums (two-sums of packed floats), 9 for the select, 5 for lists and 5 for
// the rows.  Three kernels over global memory took 69 and 155.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdio>

#include "mflat_cuda.h"
#include "select_ops.cuh"

namespace mflat_cu {
namespace {

constexpr int kEvictThreads = 512, kEvictWarps = kEvictThreads / 32;
constexpr int kEvictSlots = 49152;      // keys a block holds, 4 bytes each; with half as many, sums too
constexpr int kEvictCluster = 8;
constexpr int kMaxCapacity = 1 << 30, kMaxRows = 1 << 30;
constexpr int kGather = 2048;           // keys of one digit that a block takes in
constexpr int kAccThreads = 256;
constexpr int kKeepThreads = 512, kKeepWarps = kKeepThreads / 32;

struct CacheParams {
    int heads, group, capacity, budget, recent, sink, queries;
    int64_t wb, wh, wq;
    int64_t kb, kh, ks, vb, vh, vs;     // bytes
    int64_t key_vecs, value_vecs;
    int rows_vec;                       // bytes of a vector of the rows: 16, 4 or 1 (0: no rows)
    const void* weights;
    const int32_t* rows;
    const int32_t* lens;
    const int32_t* seen;
    const float* acc;
    const int32_t* pos;
    float* out_acc;
    int32_t* out_pos;
    int32_t* out_lens;
    char* keys;
    char* values;
    int vec_w, vec_a;                   // weights, and acc and pos, can be moved by fours
    int range;                          // slots that a block of evict_kernel has room for
    int half;                           // most moves of a head: capacity / 2
    int64_t sums_row;                   // capacity rounded up to 4
    float* sums;                        // long caches [b][h][sums_row]: acc' (null: in shared memory)
    int32_t* holes;                     // workspace [b][h][half]
    int32_t* tails;                     // workspace [b][h][half]: slot,
    float* tail_acc;                    // acc' and
    int32_t* tail_pos;                  // position
    int32_t* moves;                     // long caches [b][h]
};

__device__ __forceinline__ int entries_of(const CacheParams& p, int b) {
    return min(max(p.lens[b], 0), p.capacity);
}

// The rows of a (sequence, head): keys then values, as one list of vectors.
struct RowsOf {
    char *keys, *values;
    int64_t key_stride, value_stride, key_vecs, value_vecs;
};

// Moves first, first + stride, ... of n, a warp each, four at a time: their rows'
// vectors are all read before the first is written.
template <class V>
__device__ __forceinline__ void move_rows(const RowsOf& p, const int32_t* holes, const int32_t* tails,
                                          int first, int stride, int n) {
    const int lane = threadIdx.x & 31;
    for (int i0 = first; i0 < n; i0 += 4 * stride) {
        int from[4], to[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = min(i0 + u * stride, n - 1);
            from[u] = tails[i];
            to[u] = holes[i];
        }
        for (int64_t c = lane; c < p.key_vecs + p.value_vecs; c += 32) {
            const bool key = c < p.key_vecs;
            char* base = (key ? p.keys : p.values) + (key ? c : c - p.key_vecs) * static_cast<int64_t>(sizeof(V));
            const int64_t slot = key ? p.key_stride : p.value_stride;
            V v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = *reinterpret_cast<const V*>(base + from[u] * slot);
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (i0 + u * stride < n) *reinterpret_cast<V*>(base + to[u] * slot) = v[u];
        }
    }
}

__device__ __forceinline__ uint32_t slot_key(const CacheParams& p, float acc, int pos, int64_t since) {
    if (pos < p.sink || pos >= since) return 0xffffffffu;
    return acc == neg_inf() ? 1u : choice_key(acc);     // NaN: 0
}

// Exclusive sum over the block's threads in order, and the block's total.
__device__ __forceinline__ int scan_block(int v, int* warp_sum, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(kFullMask, incl, o);
        if (lane >= o) incl += u;
    }
    __syncthreads();                // warp_sum is free
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kEvictWarps; ++w) {
        const int c = warp_sum[w];
        before += w < warp ? c : 0;
        total += c;
    }
    return before + incl - v;
}

__device__ __forceinline__ int cluster_load(const int* p, uint32_t rank) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(cluster_addr(p, rank)) : "memory");
    return v;
}

__device__ __forceinline__ int4 cluster_load4(const int* p, uint32_t rank) {
    int4 v;
    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(cluster_addr(p, rank))
                 : "memory");
    return v;
}

// Barrier over the blocks of a (sequence, head), for shared and global memory.
__device__ __forceinline__ void sync_blocks(uint32_t blocks) {
    if (blocks == 1) __syncthreads();
    else cluster_sync();
}

// A sum as hi + lo: every addition to hi leaves its exact rounding error (Knuth's
// two-sum), lo adds those up, itself rounded at 2^-24 of its own, much smaller, value.
struct TwoFloats {
    float hi, lo;
    __device__ __forceinline__ void add(float x) {
        const float s = hi + x, bb = s - hi;
        lo += (hi - (s - bb)) + (x - bb);
        hi = s;
    }
    // infinities and NaN are hi's alone
    __device__ __forceinline__ float rounded() const { return isfinite(hi) ? hi + lo : hi; }
};

// Two of them side by side.
struct TwoFloats2 {
    float2 hi, lo;
    __device__ __forceinline__ void add(float2 x) {
        const float2 s = add2(hi, x), bb = sub2(s, hi);
        lo = add2(lo, add2(sub2(hi, sub2(s, bb)), sub2(x, bb)));
        hi = s;
    }
};

// a[i] plus the weights of four slots over all rows (`rows` query rows of each of the
// group's heads), kAtOnce rows in flight.  kVec: four adjacent slots, w aligned for them;
// else the first `most` of w[0], w[kEvictThreads], ...
template <int kAtOnce, bool kVec, class T>
__device__ __forceinline__ void add_rows(const T* w, int64_t wh, int64_t wq, int group, int rows, int most,
                                         float (&a)[4]) {
    TwoFloats2 s0{make_float2(a[0], a[1]), make_float2(0.0f, 0.0f)}, s1{make_float2(a[2], a[3]), make_float2(0.0f, 0.0f)};
    const int64_t back = wh - static_cast<int64_t>(rows - 1) * wq;      // to the next head's first row
    const int all = group * rows;
    for (int i = 0, r = 0; i < all; i += kAtOnce) {
        Pack<T, 4> v[kAtOnce];
        T one[kAtOnce][4];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            if constexpr (kVec) {
                v[u].raw = {};
                if (i + u < all) v[u].load(w);
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    one[u][c] = i + u < all && c < most ? w[c * kEvictThreads] : from_float<T>(0.0f);
            }
            const bool last = ++r == rows;
            w += last ? back : wq;
            r = last ? 0 : r;
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            float x[4];
            if constexpr (kVec) {
                v[u].unpack(x);
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c) x[c] = to_float(one[u][c]);
            }
            s0.add(make_float2(x[0], x[1]));
            s1.add(make_float2(x[2], x[3]));
        }
    }
    a[0] = TwoFloats{s0.hi.x, s0.lo.x}.rounded();
    a[1] = TwoFloats{s0.hi.y, s0.lo.y}.rounded();
    a[2] = TwoFloats{s1.hi.x, s1.lo.x}.rounded();
    a[3] = TwoFloats{s1.hi.y, s1.lo.y}.rounded();
}

// One slot, a warp over its rows.
template <class T>
__device__ __forceinline__ float add_rows_warp(const T* w, int64_t wh, int64_t wq, int group, int rows, float a) {
    const int lane = threadIdx.x & 31;
    TwoFloats s{lane == 0 ? a : 0.0f, 0.0f};
#pragma unroll 4
    for (int i = lane; i < group * rows; i += 32) s.add(to_float(w[i / rows * wh + i % rows * wq]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float hi = __shfl_xor_sync(kFullMask, s.hi, o), lo = __shfl_xor_sync(kFullMask, s.lo, o);
        s.add(hi);
        s.lo += lo;
    }
    return s.rounded();
}

// A (sequence, head): blockIdx.y; its blocks' ranges of slots: blockIdx.x, one cluster.
// A thread adds up four adjacent slots at a time,
// then the m-th key is found by three digits of 11, 11 and 10 bits: histograms in
// shared memory, summed over the cluster by every block.  Behind that a thread owns
// a run of adjacent slots, so that one scan over the threads orders all of them.
template <class T>
__global__ void __launch_bounds__(kEvictThreads, 2) evict_kernel(const CacheParams p) {
    extern __shared__ __align__(16) uint32_t dyn[];
    __shared__ __align__(16) int hist[2][2048];
    __shared__ int warp_sum[kEvictWarps];
    __shared__ uint32_t sh_prefix;
    __shared__ __align__(16) int small[128];
    __shared__ int sh_left, sh_share, sh_own, sh_ties, sh_moves;
    uint32_t* keys = dyn;
    const int64_t bh = blockIdx.y;
    const int b = static_cast<int>(bh / p.heads), h = static_cast<int>(bh % p.heads);
    const uint32_t me = blockIdx.x, blocks = gridDim.x;
    const int n = entries_of(p, b), m = min(n, p.budget);
    // the live slots, spread over the blocks by fours
    const int range = ((n + static_cast<int>(blocks) - 1) / static_cast<int>(blocks) + 3) & ~3;
    const int lo = static_cast<int>(me) * range;
    const int mine = max(0, min(range, n - lo));
    float* sums = p.sums ? p.sums + bh * p.sums_row + lo : reinterpret_cast<float*>(dyn + p.range);
    const float* acc = p.acc + bh * p.capacity + lo;
    const int32_t* pos = p.pos + bh * p.capacity + lo;
    float* out_acc = p.out_acc + bh * p.capacity;
    int32_t* out_pos = p.out_pos + bh * p.capacity;
    if (threadIdx.x == 0 && me == 0 && h == 0) p.out_lens[b] = m;
    const bool over = n > p.budget;
    const int64_t since = static_cast<int64_t>(p.seen[b]) - p.recent;

    const int rows = !p.weights ? 0 : p.rows ? min(max(p.rows[b], 0), p.queries) : p.queries;
    const T* weights = rows > 0 ? static_cast<const T*>(p.weights) + b * p.wb + static_cast<int64_t>(h) * p.group * p.wh + lo : nullptr;
    // slots below m keep their place unless they turn out to be holes: written at once
    auto put = [&](int j, float a, int q) {
        if (lo + j < m) {
            out_acc[lo + j] = a;
            out_pos[lo + j] = q;
        }
        if (over) {
            sums[j] = a;
            keys[j] = slot_key(p, a, q, since);
        }
    };
    // aligned weights: whole fours, a thread each
    const int fours = p.vec_w ? mine & ~3 : 0;
    for (int j = threadIdx.x * 4; j < fours; j += kEvictThreads * 4) {
        float a[4];
        int q[4];
        if (p.vec_a) {
            const float4 va = *reinterpret_cast<const float4*>(acc + j);
            const int4 vq = *reinterpret_cast<const int4*>(pos + j);
            a[0] = va.x, a[1] = va.y, a[2] = va.z, a[3] = va.w;
            q[0] = vq.x, q[1] = vq.y, q[2] = vq.z, q[3] = vq.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = acc[j + i];
                q[i] = pos[j + i];
            }
        }
        // (a token's few rows, or a prompt's many: 16 in flight took 37.4 us where 8 took 39.3)
        if (p.group * rows > 4) add_rows<16, true>(weights + j, p.wh, p.wq, p.group, rows, 4, a);
        else if (rows > 0) add_rows<4, true>(weights + j, p.wh, p.wq, p.group, rows, 4, a);
        if (p.vec_a && (lo + j + 4 <= m || lo + j >= m)) {
            if (lo + j < m) {
                *reinterpret_cast<float4*>(out_acc + lo + j) = make_float4(a[0], a[1], a[2], a[3]);
                *reinterpret_cast<int4*>(out_pos + lo + j) = make_int4(q[0], q[1], q[2], q[3]);
            }
            if (over) {
                *reinterpret_cast<float4*>(sums + j) = make_float4(a[0], a[1], a[2], a[3]);
                *reinterpret_cast<uint4*>(keys + j) =
                    make_uint4(slot_key(p, a[0], q[0], since), slot_key(p, a[1], q[1], since),
                               slot_key(p, a[2], q[2], since), slot_key(p, a[3], q[3], since));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) put(j + i, a[i], q[i]);
        }
    }
    if (p.vec_w) {                      // at most three slots are left: a warp each
        const int j = fours + static_cast<int>(threadIdx.x >> 5);
        if (j < mine) {
            const float a = add_rows_warp(weights + j, p.wh, p.wq, p.group, rows, acc[j]);
            if ((threadIdx.x & 31) == 0) put(j, a, pos[j]);
        }
    } else {                            // rows at odd places: neighbouring threads, neighbouring slots
        for (int j = threadIdx.x; j < mine; j += kEvictThreads * 4) {
            const int most = (mine - j + kEvictThreads - 1) / kEvictThreads;
            float a[4];
            int q[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                a[c] = c < most ? acc[j + c * kEvictThreads] : 0.0f;
                q[c] = c < most ? pos[j + c * kEvictThreads] : 0;
            }
            if (rows > 0) add_rows<4, false>(weights + j, p.wh, p.wq, p.group, rows, most, a);
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (c < most) put(j + c * kEvictThreads, a[c], q[c]);
        }
    }
    if (!over) return;

    if (threadIdx.x == 0) { sh_prefix = 0; sh_left = m; sh_own = 0; }
    for (int i = threadIdx.x; i < 2048; i += kEvictThreads) hist[0][i] = 0;
    __syncthreads();
    // The m-th key: its first 11 bits by a histogram over the cluster.  The keys that
    // share them, few as a rule, are gathered by every block, which finds the other
    // 21 bits alone; more of them than a block takes in go on over the cluster.
    uint32_t mask = 0;
    bool alone = false;
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
        const uint32_t prefix = sh_prefix, digits = (1u << bits) - 1u;
        for (int j = threadIdx.x; j < mine; j += kEvictThreads) {
            const uint32_t key = keys[j];
            if ((key & mask) == prefix) atomicAdd(&hist[pass & 1][(key >> shift) & digits], 1);
        }
        sync_blocks(blocks);
        // four digits a thread, from the top down
        const int d0 = 2044 - static_cast<int>(threadIdx.x) * 4;
        int4 c = *reinterpret_cast<const int4*>(&hist[pass & 1][d0]);
        if (blocks > 1) {
            c = make_int4(0, 0, 0, 0);
#pragma unroll
            for (uint32_t r = 0; r < kEvictCluster; ++r)
                if (r < blocks) {
                    const int4 o = cluster_load4(&hist[pass & 1][d0], r);
                    c.x += o.x;
                    c.y += o.y;
                    c.z += o.z;
                    c.w += o.w;
                }
        }
        const int count[4] = {c.w, c.z, c.y, c.x}, sum = c.x + c.y + c.z + c.w;
        const int left = sh_left;
        int total;
        int above = scan_block(sum, warp_sum, total);       // its barriers: left is read
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (above < left && left <= above + count[i]) {
                sh_prefix = prefix | (static_cast<uint32_t>(2047 - (threadIdx.x * 4 + i)) << shift);
                sh_left = left - above;
                sh_share = count[i];
            }
            above += count[i];
        }
        mask |= digits << shift;
        __syncthreads();
        if (pass == 0 && sh_share <= kGather) {
            alone = true;
            break;
        }
        // (read by the other blocks before this pass's cluster barrier)
        if (pass < 2) {
            for (int i = threadIdx.x; i < 2048; i += kEvictThreads) hist[(pass + 1) & 1][i] = 0;
            __syncthreads();
        }
    }
    if (alone) {
        // hist[1] takes this block's keys, then hist[0] all blocks'
        uint32_t* own = reinterpret_cast<uint32_t*>(hist[1]);
        const uint32_t prefix = sh_prefix;
        for (int j = threadIdx.x; j < mine; j += kEvictThreads)
            if ((keys[j] & mask) == prefix) own[atomicAdd(&sh_own, 1)] = keys[j];
        sync_blocks(blocks);
        const uint32_t* all = own;
        const int n_all = sh_share;
        if (blocks > 1) {
            uint32_t* got = reinterpret_cast<uint32_t*>(hist[0]);
            int base = 0;
#pragma unroll
            for (uint32_t r = 0; r < kEvictCluster; ++r)
                if (r < blocks) {
                    const int c = cluster_load(&sh_own, r);
                    for (int i = threadIdx.x; i < c; i += kEvictThreads)
                        got[base + i] = static_cast<uint32_t>(cluster_load(reinterpret_cast<int*>(own + i), r));
                    base += c;
                }
            all = got;
        }
        for (int shift = 14; shift >= 0; shift -= 7) {
            if (threadIdx.x < 128) small[threadIdx.x] = 0;
            __syncthreads();
            const uint32_t prefix = sh_prefix;
            for (int i = threadIdx.x; i < n_all; i += kEvictThreads)
                if ((all[i] & mask) == prefix) atomicAdd(&small[(all[i] >> shift) & 127u], 1);
            __syncthreads();
            if (threadIdx.x < 32) {
                // four digits a lane, from the top down
                const int lane = threadIdx.x;
                const int4 c = *reinterpret_cast<const int4*>(&small[124 - 4 * lane]);
                const int count[4] = {c.w, c.z, c.y, c.x}, sum = c.x + c.y + c.z + c.w, left = sh_left;
                int above = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int u = __shfl_up_sync(kFullMask, above, o);
                    if (lane >= o) above += u;
                }
                above -= sum;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (above < left && left <= above + count[i]) {
                        sh_prefix = prefix | (static_cast<uint32_t>(127 - (4 * lane + i)) << shift);
                        sh_left = left - above;
                        sh_share = count[i];
                    }
                    above += count[i];
                }
            }
            mask |= 127u << shift;
            __syncthreads();
        }
    }
    const uint32_t cut = sh_prefix;
    const int ties = sh_left;           // entries at the cut that stay, the lowest slots

    // runs of an odd length: threads read different banks
    const int run = ((mine + kEvictThreads - 1) / kEvictThreads) | 1;
    const int j0 = min(mine, static_cast<int>(threadIdx.x) * run), j1 = min(mine, j0 + run);
    int tie = 0, total;                 // of the entries at the cut before the run's
    if (sh_share > ties) {              // (all of them stay: their order is no matter)
        int equal = 0;
        for (int j = j0; j < j1; ++j) equal += keys[j] == cut ? 1 : 0;
        tie = scan_block(equal, warp_sum, total);
        if (threadIdx.x == 0) sh_ties = total;
        sync_blocks(blocks);
        for (uint32_t r = 0; r < me; ++r) tie += cluster_load(&sh_ties, r);
    } else {
        tie = INT_MIN / 2;
    }
    const int tie0 = tie;
    // holes in the upper half word, tails in the lower: a block has fewer than 2^16 of each,
    // so sums stay apart (as unsigned: 2^15 holes reach the sign)
    static_assert(kEvictSlots < 65536, "counts in half words");
    int moved = 0;
    for (int j = j0; j < j1; ++j) {
        const uint32_t key = keys[j];
        const bool keep = key > cut || (key == cut && tie++ < ties);
        if (lo + j < m ? !keep : keep) moved += lo + j < m ? 1 << 16 : 1;
    }
    const int rank = scan_block(moved, warp_sum, total);
    if (threadIdx.x == 0) sh_moves = total;
    sync_blocks(blocks);
    int hole = static_cast<int>(static_cast<uint32_t>(rank) >> 16), tail = rank & 0xffff, moves = 0;
    for (uint32_t r = 0; r < blocks; ++r) {
        const int c = cluster_load(&sh_moves, r);
        const int there = static_cast<int>(static_cast<uint32_t>(c) >> 16);
        hole += r < me ? there : 0;
        tail += r < me ? c & 0xffff : 0;
        moves += there;
    }
    int32_t* holes = p.holes + bh * p.half;
    int32_t* tails = p.tails + bh * p.half;
    float* tail_acc = p.tail_acc + bh * p.half;
    int32_t* tail_pos = p.tail_pos + bh * p.half;
    tie = tie0;
    for (int j = moved ? j0 : j1; j < j1; ++j) {        // most runs have nothing to list
        const uint32_t key = keys[j];
        const bool keep = key > cut || (key == cut && tie++ < ties);
        if (lo + j < m) {
            if (!keep) holes[hole++] = lo + j;
        } else if (keep) {
            tails[tail] = lo + j;
            tail_acc[tail] = sums[j];
            tail_pos[tail++] = pos[j];
        }
    }
    sync_blocks(blocks);                // the lists are complete and in every block's sight
    const int at = static_cast<int>(me) * kEvictThreads + threadIdx.x, step = static_cast<int>(blocks) * kEvictThreads;
    for (int i = at; i < moves; i += step) {
        const int to = holes[i];
        out_acc[to] = tail_acc[i];
        out_pos[to] = tail_pos[i];
    }
    // rows: a warp per move, keys and values
    if (!p.rows_vec) return;
    char* k = p.keys ? p.keys + b * p.kb + h * p.kh : nullptr;
    char* v = p.values ? p.values + b * p.vb + h * p.vh : nullptr;
    const RowsOf rows_of{k, v, p.ks, p.vs, p.key_vecs, p.value_vecs};
    const int first = at >> 5, stride = step >> 5;
    if (p.rows_vec == 16) move_rows<uint4>(rows_of, holes, tails, first, stride, moves);
    else if (p.rows_vec == 4) move_rows<uint32_t>(rows_of, holes, tails, first, stride, moves);
    else move_rows<uint8_t>(rows_of, holes, tails, first, stride, moves);
}

template <class T>
__global__ void __launch_bounds__(kAccThreads) accumulate_kernel(const CacheParams p) {
    const int j = blockIdx.x * kAccThreads + threadIdx.x;
    const int64_t bh = blockIdx.y;
    const int b = static_cast<int>(bh / p.heads), h = static_cast<int>(bh % p.heads);
    if (j >= entries_of(p, b)) return;
    TwoFloats sum{p.acc[bh * p.capacity + j], 0.0f};
    if (p.weights) {
        const int q1 = p.rows ? min(max(p.rows[b], 0), p.queries) : p.queries;
        for (int g = 0; g < p.group; ++g) {
            const T* w = static_cast<const T*>(p.weights) + b * p.wb +
                         (static_cast<int64_t>(h) * p.group + g) * p.wh + j;
            for (int q = 0; q < q1; ++q) sum.add(to_float(w[q * p.wq]));
        }
    }
    p.sums[bh * p.sums_row + j] = sum.rounded();
}

__global__ void __launch_bounds__(kKeepThreads) keep_kernel(const CacheParams p) {
    __shared__ int hist[256];
    __shared__ int warp_sum[3][kKeepWarps];
    __shared__ uint32_t sh_prefix;
    __shared__ int sh_left;
    const int64_t bh = blockIdx.x;
    const int b = static_cast<int>(bh / p.heads);
    const int n = entries_of(p, b), m = min(n, p.budget);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float* sums = p.sums + bh * p.sums_row;
    const int32_t* pos = p.pos + bh * p.capacity;
    float* out_acc = p.out_acc + bh * p.capacity;
    int32_t* out_pos = p.out_pos + bh * p.capacity;
    if (threadIdx.x == 0 && bh % p.heads == 0) p.out_lens[b] = m;
    if (n <= p.budget) {
        for (int j = threadIdx.x; j < n; j += kKeepThreads) {
            out_acc[j] = sums[j];
            out_pos[j] = pos[j];
        }
        if (threadIdx.x == 0) p.moves[bh] = 0;
        return;
    }
    const int64_t since = static_cast<int64_t>(p.seen[b]) - p.recent;
    auto key_at = [&](int j) { return slot_key(p, sums[j], pos[j], since); };
    // the m-th largest key, 8 bits at a time
    if (threadIdx.x == 0) { sh_prefix = 0; sh_left = m; }
    uint32_t mask = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += kKeepThreads) hist[i] = 0;
        __syncthreads();
        const uint32_t prefix = sh_prefix;
        for (int j = threadIdx.x; j < n; j += kKeepThreads) {
            const uint32_t key = key_at(j);
            if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1);
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
    const int ties = sh_left;           // entries at the cut that stay
    int32_t* holes = p.holes + bh * p.half;
    int32_t* tails = p.tails + bh * p.half;
    int n_tie = 0, n_hole = 0, n_tail = 0;
    for (int j0 = 0; j0 < n; j0 += kKeepThreads) {
        const int j = j0 + threadIdx.x;
        const uint32_t key = j < n ? key_at(j) : 0u;
        const bool tie = j < n && key == cut;
        const unsigned tb = __ballot_sync(kFullMask, tie);
        if (lane == 0) warp_sum[0][warp] = __popc(tb);
        __syncthreads();
        int tie_rank = n_tie + __popc(tb & ((1u << lane) - 1u)), all = 0;
        for (int w = 0; w < kKeepWarps; ++w) {
            const int c = warp_sum[0][w];
            tie_rank += w < warp ? c : 0;
            all += c;
        }
        n_tie += all;
        const bool keep = j < n && (key > cut || (tie && tie_rank < ties));
        const bool hole = j < m && !keep, tail = keep && j >= m;
        const unsigned hb = __ballot_sync(kFullMask, hole), lb = __ballot_sync(kFullMask, tail);
        if (lane == 0) {
            warp_sum[1][warp] = __popc(hb);
            warp_sum[2][warp] = __popc(lb);
        }
        __syncthreads();
        int hole_rank = n_hole + __popc(hb & ((1u << lane) - 1u));
        int tail_rank = n_tail + __popc(lb & ((1u << lane) - 1u));
        for (int w = 0; w < kKeepWarps; ++w) {
            hole_rank += w < warp ? warp_sum[1][w] : 0;
            tail_rank += w < warp ? warp_sum[2][w] : 0;
            n_hole += warp_sum[1][w];
            n_tail += warp_sum[2][w];
        }
        if (hole) holes[hole_rank] = j;
        if (tail) tails[tail_rank] = j;
    }
    __syncthreads();
    // every position has been read: the outputs may be written over the inputs
    for (int j = threadIdx.x; j < m; j += kKeepThreads) {
        out_acc[j] = sums[j];
        if (out_pos != pos) out_pos[j] = pos[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n_hole; i += kKeepThreads) {
        out_acc[holes[i]] = sums[tails[i]];
        out_pos[holes[i]] = pos[tails[i]];
    }
    if (threadIdx.x == 0) p.moves[bh] = n_hole;
}

__global__ void __launch_bounds__(256) move_kernel(const CacheParams p) {
    const int64_t bh = blockIdx.y;
    const int b = static_cast<int>(bh / p.heads), h = static_cast<int>(bh % p.heads);
    const RowsOf rows_of{p.keys ? p.keys + b * p.kb + h * p.kh : nullptr,
                         p.values ? p.values + b * p.vb + h * p.vh : nullptr, p.ks, p.vs, p.key_vecs, p.value_vecs};
    const int32_t *holes = p.holes + bh * p.half, *tails = p.tails + bh * p.half;
    const int n = p.moves[bh], first = blockIdx.x * 8 + (threadIdx.x >> 5), stride = gridDim.x * 8;
    if (p.rows_vec == 16) move_rows<uint4>(rows_of, holes, tails, first, stride, n);
    else if (p.rows_vec == 4) move_rows<uint32_t>(rows_of, holes, tails, first, stride, n);
    else move_rows<uint8_t>(rows_of, holes, tails, first, stride, n);
}

constexpr size_t round256(size_t n) { return (n + 255) & ~size_t(255); }

// Slots that each of n blocks holds, a multiple of four.
int range_of(const mflat_cu_cache_t* c, int n) {
    return (c->capacity / n + (c->capacity % n ? 1 : 0) + 3) & ~3;
}

// Blocks of a cluster: as few as hold the slots, sums and keys, but enough to fill the
// machine with ranges of at least 1024 slots; eight hold twice as many keys alone.
// 0: too long for that.
int cluster_of(const mflat_cu_cache_t* c, int batch) {
    const int64_t bh = static_cast<int64_t>(batch) * c->heads;
    int n = 1;
    while (n < kEvictCluster && (range_of(c, n) > kEvictSlots / 2 || (bh * n < 148 && range_of(c, n) >= 2048))) n *= 2;
    return range_of(c, n) <= kEvictSlots ? n : 0;
}

struct CacheLayout {
    bool out;                   // sums are in the workspace
    size_t holes, tails, tail_acc, tail_pos, sums, moves, end;
};
CacheLayout cache_layout(const mflat_cu_cache_t* c, int batch) {
    const size_t bh = static_cast<size_t>(batch) * c->heads, half = bh * (c->capacity / 2);
    CacheLayout l;
    l.holes = 0;
    l.tails = l.holes + round256(half * 4);
    l.tail_acc = l.tails + round256(half * 4);
    l.tail_pos = l.tail_acc + round256(half * 4);
    l.sums = l.tail_pos + round256(half * 4);
    const int blocks = cluster_of(c, batch);
    l.out = blocks == 0 || range_of(c, blocks) > kEvictSlots / 2;
    l.moves = l.sums + (l.out ? round256(bh * ((static_cast<size_t>(c->capacity) + 3) & ~size_t(3)) * 4) : 0);
    l.end = l.moves + (blocks == 0 ? round256(bh * 4) : 0);
    return l;
}

int check_cache(const mflat_cu_cache_t* c, int batch) {
    char msg[200];
    if (c->heads < 1 || c->group < 1 || c->capacity < 1 || c->capacity > kMaxCapacity)
        return fail(ST_BAD_ARG, "heads and group must be at least 1, capacity in [1, 2^30]");
    if (c->budget < 1 || c->budget > c->capacity || c->recent < 0 || c->sink < 0 ||
        static_cast<int64_t>(c->recent) + c->sink > c->budget) {
        std::snprintf(msg, sizeof msg, "budget=%d recent=%d sink=%d: need 0 <= sink + recent <= budget <= "
                      "capacity=%d", c->budget, c->recent, c->sink, c->capacity);
        return fail(ST_BAD_ARG, msg);
    }
    if (c->type < 0 || c->type > 2) return fail(ST_BAD_ARG, "unknown weights type");
    if (c->key_bytes < 0 || c->value_bytes < 0) return fail(ST_BAD_ARG, "row bytes below 0");
    if (batch < 0 || static_cast<int64_t>(batch) * c->heads > 65535) {
        std::snprintf(msg, sizeof msg, "batch=%d: batch * heads must be in [0, 65535]", batch);
        return fail(ST_BAD_ARG, msg);
    }
    return ST_OK;
}

// blockIdx.x runs over the cluster, blockIdx.y over the heads.
template <class K>
cudaError_t launch_evict(K kernel, int blocks, unsigned bh, size_t smem, cudaStream_t st, const CacheParams& p) {
    // always the same bound: calls from several threads may set it at once
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kEvictSlots * 4);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks), bh);
    cfg.blockDim = dim3(kEvictThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = static_cast<unsigned>(blocks);
    at.val.clusterDim.y = 1;
    at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

// Dense strides where all are 0; false where two rows could overlap: the smallest
// stride has to span a row, each larger one all of what the one below it steps over.
bool fill_strides(const int64_t* s, int64_t bytes, int64_t batch, int heads, int capacity, int64_t& sb,
                  int64_t& sh, int64_t& ss) {
    sb = s[0];
    sh = s[1];
    ss = s[2];
    if (sb == 0 && sh == 0 && ss == 0) {
        ss = bytes;
        sh = ss * capacity;
        sb = sh * heads;
    }
    if (sb < 0 || sh < 0 || ss < 0) return false;
    if (bytes == 0) return true;
    struct Dim {
        __int128 stride;
        int64_t count;
    } dims[3] = {{sb, batch}, {sh, heads}, {ss, capacity}};
    std::sort(dims, dims + 3, [](const Dim& a, const Dim& b) { return a.stride < b.stride; });
    __int128 span = bytes;
    for (const Dim& d : dims) {
        if (d.count <= 1) continue;
        if (d.stride < span) return false;
        span = d.stride * d.count;
    }
    return span <= (static_cast<__int128>(1) << 56);
}

}  // namespace
}  // namespace mflat_cu

using namespace mflat_cu;

extern "C" size_t mflat_cu_cache_workspace(const mflat_cu_cache_t* c, int batch) {
    if (check_cache(c, batch) != ST_OK) return 0;
    return cache_layout(c, batch).end;
}

extern "C" int mflat_cu_cache_evict(const mflat_cu_cache_t* c, int batch, const int32_t* lens,
                                    const int32_t* seen, const void* weights, int queries,
                                    const int64_t* weight_stride, const int32_t* rows,
                                    const float* acc, const int32_t* pos, float* out_acc,
                                    int32_t* out_pos, int32_t* out_lens, void* keys, void* values,
                                    void* ws, size_t ws_bytes, int device, void* stream) {
    int rc = check_cache(c, batch);
    if (rc != ST_OK) return rc;
    // (the kernels count rows in steps of up to 32 past the last)
    if (weights && (queries < 0 || static_cast<int64_t>(c->group) * queries > kMaxRows))
        return fail(ST_BAD_ARG, "queries below 0, or group * queries above 2^30");
    CacheParams p{};
    p.heads = c->heads;
    p.group = c->group;
    p.capacity = c->capacity;
    p.budget = c->budget;
    p.recent = c->recent;
    p.sink = c->sink;
    p.queries = queries;
    if (weight_stride) {
        p.wb = weight_stride[0];
        p.wh = weight_stride[1];
        p.wq = weight_stride[2];
        if (p.wb < 0 || p.wh < 0 || p.wq < 0) return fail(ST_BAD_ARG, "negative weight stride");
    } else {
        const __int128 span = static_cast<__int128>(c->capacity) * queries * c->heads * c->group;
        if (weights && span > (static_cast<__int128>(1) << 56)) return fail(ST_BAD_ARG, "weights span more than 2^56");
        p.wq = c->capacity;
        p.wh = weights ? p.wq * queries : 0;
        p.wb = weights ? p.wh * c->heads * c->group : 0;
    }
    if (!fill_strides(c->key_stride, c->key_bytes, batch, c->heads, c->capacity, p.kb, p.kh, p.ks) ||
        !fill_strides(c->value_stride, c->value_bytes, batch, c->heads, c->capacity, p.vb, p.vh, p.vs))
        return fail(ST_BAD_ARG, "cache strides let rows overlap, or span more than 2^56 bytes");
    if (!aligned_to(weights, type_bytes(c->type)) || !aligned_to(lens, 4) || !aligned_to(seen, 4) ||
        !aligned_to(rows, 4) || !aligned_to(acc, 4) || !aligned_to(pos, 4) || !aligned_to(out_acc, 4) ||
        !aligned_to(out_pos, 4) || !aligned_to(out_lens, 4))
        return fail(ST_BAD_ARG, "misaligned pointer");
    if (batch == 0) return ST_OK;
    // one block writes a sequence's new length while its other heads' blocks still read these
    for (const int32_t* in : {lens, seen, rows})
        if (in && out_lens < in + batch && in < out_lens + batch)
            return fail(ST_BAD_ARG, "out_lens must not share memory with lens, seen or rows");
    const CacheLayout l = cache_layout(c, batch);
    if (l.end > 0 && (!ws || ws_bytes < l.end || !aligned_to(ws, 256)))
        return fail(ST_BAD_ARG, "workspace missing, too small or not 256-byte aligned");
    rc = operator_device(device, &device);
    if (rc != ST_OK) return rc;
    DeviceGuard g(device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    char* w = static_cast<char*>(ws);
    p.weights = weights;
    p.rows = rows;
    p.lens = lens;
    p.seen = seen;
    p.acc = acc;
    p.pos = pos;
    p.out_acc = out_acc;
    p.out_pos = out_pos;
    p.out_lens = out_lens;
    p.keys = c->key_bytes ? static_cast<char*>(keys) : nullptr;
    p.values = c->value_bytes ? static_cast<char*>(values) : nullptr;
    p.sums = l.out ? reinterpret_cast<float*>(w + l.sums) : nullptr;
    p.sums_row = (static_cast<int64_t>(c->capacity) + 3) & ~int64_t(3);
    p.holes = reinterpret_cast<int32_t*>(w + l.holes);
    p.tails = reinterpret_cast<int32_t*>(w + l.tails);
    p.moves = reinterpret_cast<int32_t*>(w + l.moves);
    p.tail_acc = reinterpret_cast<float*>(w + l.tail_acc);
    p.tail_pos = reinterpret_cast<int32_t*>(w + l.tail_pos);
    p.half = c->capacity / 2;
    p.vec_w = ((p.wb | p.wh | p.wq) & 3) == 0 && aligned_to(weights, 4 * type_bytes(c->type));
    p.vec_a = (c->capacity & 3) == 0 && aligned_to(acc, 16) && aligned_to(pos, 16) &&
              aligned_to(out_acc, 16) && aligned_to(out_pos, 16);
    int64_t bits = 0;
    if (p.keys) bits |= c->key_bytes | p.kb | p.kh | p.ks | static_cast<int64_t>(reinterpret_cast<uintptr_t>(keys) & 15);
    if (p.values) bits |= c->value_bytes | p.vb | p.vh | p.vs | static_cast<int64_t>(reinterpret_cast<uintptr_t>(values) & 15);
    const int vec = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
    p.rows_vec = p.keys || p.values ? vec : 0;
    p.key_vecs = p.keys ? c->key_bytes / vec : 0;
    p.value_vecs = p.values ? c->value_bytes / vec : 0;
    const unsigned bh = static_cast<unsigned>(batch * c->heads);
    const int blocks = cluster_of(c, batch);
    if (blocks > 0) {
        p.range = range_of(c, blocks);
        CU_TRY(with_type(c->type, [&](auto zero) {
            return launch_evict(evict_kernel<decltype(zero)>, blocks, bh, static_cast<size_t>(p.range) * (l.out ? 4 : 8), st, p);
        }), "evict launch");
        return ST_OK;
    }
    CU_TRY(with_type(c->type, [&](auto zero) {
        accumulate_kernel<decltype(zero)>
            <<<dim3(blocks_for(c->capacity, kAccThreads), bh), kAccThreads, 0, st>>>(p);
        return cudaGetLastError();
    }), "accumulate launch");
    keep_kernel<<<bh, kKeepThreads, 0, st>>>(p);
    CU_TRY(cudaGetLastError(), "keep launch");
    if (!p.rows_vec) return ST_OK;
    move_kernel<<<dim3(64, bh), 256, 0, st>>>(p);
    CU_TRY(cudaGetLastError(), "move launch");
    return ST_OK;
}
