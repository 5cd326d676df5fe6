// cache.cu -- eviction from a key/value cache by accumulated attention weight.
//
// acc' = acc + the sum of the group's weights, formed in 64 bits and rounded once,
// so that the kept set does not hang on an order of addition.  Of a cache over its
// budget m, the kept slots are the m largest of (protected, acc'), ties to the lower
// slot: a radix select of the m-th key, then one ordered pass.  Slots of dropped
// entries below m ("holes") take the kept entries at and behind m ("tails") in
// order: sources lie behind m and targets below it, so rows move in place in any
// order.
#include <cuda_runtime.h>

#include <climits>
#include <cstdio>

#include "mflat_cuda.h"
#include "select_ops.cuh"

namespace mflat_cu {
namespace {

constexpr int kAccThreads = 256;
constexpr int kKeepThreads = 512, kKeepWarps = kKeepThreads / 32;

struct CacheParams {
    int heads, group, capacity, budget, recent, sink, queries;
    int64_t wb, wh, wq;
    int64_t kb, kh, ks, vb, vh, vs;     // bytes
    int64_t key_vecs, value_vecs;
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
    float* sums;                        // workspace [b][h][capacity]: acc'
    int32_t* holes;                     // workspace [b][h][capacity]
    int32_t* tails;
    int32_t* moves;                     // workspace [b][h]
};

__device__ __forceinline__ int entries_of(const CacheParams& p, int b) {
    return min(max(p.lens[b], 0), p.capacity);
}

template <class T>
__global__ void __launch_bounds__(kAccThreads) accumulate_kernel(const CacheParams p) {
    const int j = blockIdx.x * kAccThreads + threadIdx.x;
    const int64_t bh = blockIdx.y;
    const int b = static_cast<int>(bh / p.heads), h = static_cast<int>(bh % p.heads);
    if (j >= entries_of(p, b)) return;
    double sum = p.acc[bh * p.capacity + j];
    if (p.weights) {
        const int q1 = p.rows ? min(max(p.rows[b], 0), p.queries) : p.queries;
        for (int g = 0; g < p.group; ++g) {
            const T* w = static_cast<const T*>(p.weights) + b * p.wb +
                         (static_cast<int64_t>(h) * p.group + g) * p.wh + j;
            for (int q = 0; q < q1; ++q) sum += static_cast<double>(to_float(w[q * p.wq]));
        }
    }
    p.sums[bh * p.capacity + j] = static_cast<float>(sum);
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
    const float* sums = p.sums + bh * p.capacity;
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
    auto key_at = [&](int j) {
        const int q = pos[j];
        if (q < p.sink || q >= since) return 0xffffffffu;
        const float a = sums[j];
        return a == neg_inf() ? 1u : choice_key(a);
    };
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
    int32_t* holes = p.holes + bh * p.capacity;
    int32_t* tails = p.tails + bh * p.capacity;
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

// Rows of keys (blockIdx.z 0) and values (1), a warp per move.
template <class V>
__global__ void __launch_bounds__(256) move_kernel(const CacheParams p) {
    const int64_t bh = blockIdx.y;
    const int b = static_cast<int>(bh / p.heads), h = static_cast<int>(bh % p.heads);
    char* base = blockIdx.z == 0 ? p.keys : p.values;
    if (!base) return;
    base += blockIdx.z == 0 ? b * p.kb + h * p.kh : b * p.vb + h * p.vh;
    const int64_t slot = blockIdx.z == 0 ? p.ks : p.vs;
    const int64_t vecs = blockIdx.z == 0 ? p.key_vecs : p.value_vecs;
    const int n = p.moves[bh];
    const int32_t* holes = p.holes + bh * p.capacity;
    const int32_t* tails = p.tails + bh * p.capacity;
    for (int i = blockIdx.x * 8 + (threadIdx.x >> 5); i < n; i += gridDim.x * 8) {
        const V* from = reinterpret_cast<const V*>(base + tails[i] * slot);
        V* to = reinterpret_cast<V*>(base + holes[i] * slot);
        for (int64_t v = threadIdx.x & 31; v < vecs; v += 32) to[v] = from[v];
    }
}

constexpr size_t round256(size_t n) { return (n + 255) & ~size_t(255); }

struct CacheLayout {
    size_t sums, holes, tails, moves, end;
};
CacheLayout cache_layout(const mflat_cu_cache_t* c, int batch) {
    const size_t bh = static_cast<size_t>(batch) * c->heads, n = bh * c->capacity;
    CacheLayout l;
    l.sums = 0;
    l.holes = l.sums + round256(n * 4);
    l.tails = l.holes + round256(n * 4);
    l.moves = l.tails + round256(n * 4);
    l.end = l.moves + round256(bh * 4);
    return l;
}

int check_cache(const mflat_cu_cache_t* c, int batch) {
    char msg[200];
    if (c->heads < 1 || c->group < 1 || c->capacity < 1)
        return fail(ST_BAD_ARG, "heads, group and capacity must be at least 1");
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

// Dense strides where all are 0; false where two rows could overlap.
bool fill_strides(const int64_t* s, int64_t bytes, int heads, int capacity, int64_t& sb, int64_t& sh,
                  int64_t& ss) {
    sb = s[0];
    sh = s[1];
    ss = s[2];
    if (sb == 0 && sh == 0 && ss == 0) {
        ss = bytes;
        sh = ss * capacity;
        sb = sh * heads;
    }
    return ss >= bytes && sh >= bytes && sb >= bytes;
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
    if (weights && queries < 0) return fail(ST_BAD_ARG, "queries below 0");
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
        p.wq = c->capacity;
        p.wh = p.wq * queries;
        p.wb = p.wh * c->heads * c->group;
    }
    if (!fill_strides(c->key_stride, c->key_bytes, c->heads, c->capacity, p.kb, p.kh, p.ks) ||
        !fill_strides(c->value_stride, c->value_bytes, c->heads, c->capacity, p.vb, p.vh, p.vs))
        return fail(ST_BAD_ARG, "cache strides below the row's bytes");
    if (!aligned_to(weights, type_bytes(c->type)) || !aligned_to(lens, 4) || !aligned_to(seen, 4) ||
        !aligned_to(rows, 4) || !aligned_to(acc, 4) || !aligned_to(pos, 4) || !aligned_to(out_acc, 4) ||
        !aligned_to(out_pos, 4) || !aligned_to(out_lens, 4))
        return fail(ST_BAD_ARG, "misaligned pointer");
    if (batch == 0) return ST_OK;
    if (out_lens == lens) return fail(ST_BAD_ARG, "out_lens must not be lens");
    const CacheLayout l = cache_layout(c, batch);
    if (!ws || ws_bytes < l.end || !aligned_to(ws, 256))
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
    p.sums = reinterpret_cast<float*>(w + l.sums);
    p.holes = reinterpret_cast<int32_t*>(w + l.holes);
    p.tails = reinterpret_cast<int32_t*>(w + l.tails);
    p.moves = reinterpret_cast<int32_t*>(w + l.moves);
    const unsigned bh = static_cast<unsigned>(batch * c->heads);
    CU_TRY(with_type(c->type, [&](auto zero) {
        accumulate_kernel<decltype(zero)>
            <<<dim3(blocks_for(c->capacity, kAccThreads), bh), kAccThreads, 0, st>>>(p);
        return cudaGetLastError();
    }), "accumulate launch");
    keep_kernel<<<bh, kKeepThreads, 0, st>>>(p);
    CU_TRY(cudaGetLastError(), "keep launch");
    if (!p.keys && !p.values) return ST_OK;
    int64_t bits = 0;
    if (p.keys) bits |= c->key_bytes | p.kb | p.kh | p.ks | static_cast<int64_t>(reinterpret_cast<uintptr_t>(keys) & 15);
    if (p.values) bits |= c->value_bytes | p.vb | p.vh | p.vs | static_cast<int64_t>(reinterpret_cast<uintptr_t>(values) & 15);
    const int vec = bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : bits % 2 == 0 ? 2 : 1;
    p.key_vecs = c->key_bytes / vec;
    p.value_vecs = c->value_bytes / vec;
    const int most = c->capacity - c->budget < c->budget ? c->capacity - c->budget : c->budget;
    if (most == 0) return ST_OK;
    const dim3 grid(blocks_for(most, 8) < 64 ? blocks_for(most, 8) : 64, bh, 2);
    switch (vec) {
        case 16: move_kernel<uint4><<<grid, 256, 0, st>>>(p); break;
        case 8: move_kernel<uint2><<<grid, 256, 0, st>>>(p); break;
        case 4: move_kernel<uint32_t><<<grid, 256, 0, st>>>(p); break;
        case 2: move_kernel<uint16_t><<<grid, 256, 0, st>>>(p); break;
        default: move_kernel<uint8_t><<<grid, 256, 0, st>>>(p); break;
    }
    CU_TRY(cudaGetLastError(), "move launch");
    return ST_OK;
}
