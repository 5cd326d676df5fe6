// beam.cu -- beam search: the k best continuations over beams x vocabulary, and
// the reordering of states by parent beam.
//
// Selection.  key[w, v] = cum[w] + ((x[w, v] - m_w) - log sum_v exp(x[w, v] - m_w)).  Within
// a beam the order is the logits' own, exact in any precision; between beams it
// hangs on the sums, which are formed in 64 bits.  So each row first yields its k
// best logits (ties to the lower token) with its maximum and sum, and the rows of
// a sequence are then merged by their keys in 64 bits (ties to the lower beam).
#include <cuda_runtime.h>

#include <climits>
#include <cstdio>

#include "mflat_cuda.h"
#include "select_ops.cuh"

namespace mflat_cu {
namespace {

constexpr int kMaxBeams = 64, kMaxBeamK = 128;
constexpr int kRowThreads = 256, kRowWarps = kRowThreads / 32;

struct BeamParams {
    const void* logits;
    int64_t stride;
    const float* cum;
    const uint8_t* finished;
    int batch, beams, vocab, k, eos;
    double* lse_sum;            // workspace, [rows]: sum of exp(x - max)
    float* row_max;             // [rows]
    float* cand_x;              // [rows][k]: best logits, best first (-inf: none)
    int32_t* cand_v;            // [rows][k]: their tokens
    int32_t* parents;
    int32_t* tokens;
    float* scores;
};

template <class V, class Op>
__device__ V block_reduce(V v, Op op, V* sh) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(kFullMask, v, o));
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh[0];
    for (int w = 1; w < kRowWarps; ++w) v = op(v, sh[w]);
    __syncthreads();
    return v;
}

template <class T>
__global__ void __launch_bounds__(kRowThreads) beam_row_kernel(const BeamParams p) {
    __shared__ uint64_t sh[kRowWarps];
    const int64_t r = blockIdx.x;
    const T* row = static_cast<const T*>(p.logits) + r * p.stride;
    if (p.finished && p.finished[r]) return;
    auto larger = [](auto a, auto b) { return a > b ? a : b; };
    float m = neg_inf();
    for (int v = threadIdx.x; v < p.vocab; v += kRowThreads) m = fmaxf(m, to_float(row[v]));
    m = block_reduce(m, larger, reinterpret_cast<float*>(sh));
    double sum = 0.0;
    for (int v = threadIdx.x; v < p.vocab; v += kRowThreads) {
        const float x = to_float(row[v]);
        if (x > neg_inf()) sum += x == m ? 1.0 : exp(static_cast<double>(x) - m);
    }
    sum = block_reduce(sum, [](double a, double b) { return a + b; }, reinterpret_cast<double*>(sh));
    if (threadIdx.x == 0) {
        p.row_max[r] = m;
        p.lse_sum[r] = sum;
    }
    // best first: (logit's key, then the lower token) as one number, each round
    // the largest below the last
    uint64_t last = ~0ull;
    for (int j = 0; j < p.k; ++j) {
        uint64_t best = 0;
        for (int v = threadIdx.x; v < p.vocab; v += kRowThreads) {
            const uint32_t key = choice_key(to_float(row[v]));
            const uint64_t c = (static_cast<uint64_t>(key) << 32) | (0xffffffffu - static_cast<uint32_t>(v));
            if (key != 0u && c < last && c > best) best = c;
        }
        best = block_reduce(best, larger, sh);
        last = best;
        if (threadIdx.x == 0) {
            p.cand_x[r * p.k + j] = key_value(static_cast<uint32_t>(best >> 32));
            p.cand_v[r * p.k + j] = best ? static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(best)) : -1;
        }
    }
}

__global__ void __launch_bounds__(32) beam_merge_kernel(const BeamParams p) {
    const int64_t b = blockIdx.x;
    const int lane = threadIdx.x;
    // lane l walks beams l and l + 32: its next candidate of each
    int next[2] = {0, 0};
    for (int j = 0; j < p.k; ++j) {
        uint64_t best = 0;
        int beam = INT_MAX, token = -1;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int w = lane + 32 * h;
            if (w >= p.beams || next[h] >= p.k) continue;
            const int64_t r = b * p.beams + w;
            const float cum = p.cum[r];
            if (!isfinite(cum)) continue;
            const bool done = p.finished && p.finished[r];
            double key;
            int v;
            if (done) {
                if (next[h] > 0) continue;
                key = cum;
                v = p.eos;
            } else {
                const float x = p.cand_x[r * p.k + next[h]];
                if (!(x > neg_inf())) continue;
                const float m = p.row_max[r];
                key = cum + ((x == m ? 0.0 : static_cast<double>(x) - m) - log(p.lse_sum[r]));
                v = p.cand_v[r * p.k + next[h]];
            }
            const uint64_t c = choice_key(key);
            if (c > best) { best = c; beam = w; token = v; }
        }
        uint64_t top = best;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const uint64_t c = __shfl_xor_sync(kFullMask, top, o);
            top = c > top ? c : top;
        }
        const int who = __reduce_min_sync(kFullMask, best == top ? beam : INT_MAX);
        token = __shfl_sync(kFullMask, token, who & 31);
        if (top != 0 && (who & 31) == lane) ++next[who >> 5];
        if (lane == 0) {
            p.parents[b * p.k + j] = top ? who : -1;
            p.tokens[b * p.k + j] = top ? token : -1;
            p.scores[b * p.k + j] = static_cast<float>(key_value(top));
        }
    }
}

// Reordering in place.  A thread owns the same bytes of all the rows of a
// sequence: it reads every row that moves, then writes, so no other thread's
// writes can come before its reads.
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
    int outer = p.outer;
    while (static_cast<int64_t>(outer) * p.batch > 65535) outer = (outer + 1) / 2;
    const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(outer * p.batch));
    if (p.beams <= 4) reorder_kernel<V, 4><<<grid, kReorderThreads, 0, st>>>(p);
    else if (p.beams <= 8) reorder_kernel<V, 8><<<grid, kReorderThreads, 0, st>>>(p);
    else if (p.beams <= 16) reorder_kernel<V, 16><<<grid, kReorderThreads, 0, st>>>(p);
    else reorder_kernel<V, 64><<<grid, kReorderThreads, 0, st>>>(p);
    return cudaGetLastError();
}

constexpr size_t round256(size_t n) { return (n + 255) & ~size_t(255); }

struct BeamLayout {
    size_t sum, max, x, v, end;
};
BeamLayout beam_layout(const mflat_cu_beam_t* b, int batch) {
    const size_t rows = static_cast<size_t>(batch) * b->beams;
    BeamLayout l;
    l.sum = 0;
    l.max = l.sum + round256(rows * 8);
    l.x = l.max + round256(rows * 4);
    l.v = l.x + round256(rows * b->k * 4);
    l.end = l.v + round256(rows * b->k * 4);
    return l;
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
    if (b->vocab < 1) return fail(ST_BAD_ARG, "vocab below 1");
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
    return beam_layout(b, batch).end;
}

extern "C" int mflat_cu_beam_select(const mflat_cu_beam_t* b, const void* logits, int64_t stride,
                                    const float* cum, const uint8_t* finished, int batch,
                                    int32_t* parents, int32_t* tokens, float* scores, void* ws,
                                    size_t ws_bytes, int device, void* stream) {
    int rc = check_beam(b, batch);
    if (rc != ST_OK) return rc;
    if (stride == 0) stride = b->vocab;
    if (stride < b->vocab) return fail(ST_BAD_ARG, "logits stride below vocab");
    if (finished && b->eos < 0) return fail(ST_BAD_ARG, "finished beams need an eos token");
    if (!aligned_to(logits, type_bytes(b->type)) || !aligned_to(cum, 4) || !aligned_to(parents, 4) ||
        !aligned_to(tokens, 4) || !aligned_to(scores, 4))
        return fail(ST_BAD_ARG, "misaligned pointer");
    if (batch == 0) return ST_OK;
    const BeamLayout l = beam_layout(b, batch);
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
    p.lse_sum = reinterpret_cast<double*>(w + l.sum);
    p.row_max = reinterpret_cast<float*>(w + l.max);
    p.cand_x = reinterpret_cast<float*>(w + l.x);
    p.cand_v = reinterpret_cast<int32_t*>(w + l.v);
    p.parents = parents;
    p.tokens = tokens;
    p.scores = scores;
    CU_TRY(with_type(b->type, [&](auto zero) {
        beam_row_kernel<decltype(zero)><<<batch * b->beams, kRowThreads, 0, st>>>(p);
        return cudaGetLastError();
    }), "beam rows launch");
    beam_merge_kernel<<<batch, 32, 0, st>>>(p);
    CU_TRY(cudaGetLastError(), "beam merge launch");
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
    const int vec = bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : bits % 2 == 0 ? 2 : 1;
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
