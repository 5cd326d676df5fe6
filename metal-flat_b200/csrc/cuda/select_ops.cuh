// select_ops.cuh -- what the selection operators (route.cu, beam.cu, cache.cu)
// share: element types, order-preserving keys, argument checks and launches.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "index_impl.cuh"
#include "ptx.cuh"

namespace mflat_cu {

constexpr unsigned kFullMask = 0xffffffffu;

__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <class T>
__device__ __forceinline__ T from_float(float v) {
    if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
    else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __float2bfloat16_rn(v);
    else return v;
}

// N elements as one aligned load or store of N * sizeof(T) bytes.  (By their raw bits:
// a struct of 16-bit floats is copied element by element.)
template <int BYTES>
using Raw = std::conditional_t<BYTES == 16, uint4,
            std::conditional_t<BYTES == 8, uint2, std::conditional_t<BYTES == 4, uint32_t, uint16_t>>>;

template <class T, int N>
struct Pack {
    using R = Raw<N * sizeof(T)>;
    R raw;
    __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const R*>(p); }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<R*>(p) = raw; }
    __device__ __forceinline__ void unpack(float (&x)[N]) const {
        if constexpr (N * sizeof(T) == 2) {
            x[0] = to_float(*reinterpret_cast<const T*>(&raw));
        } else {
            const uint32_t* u = reinterpret_cast<const uint32_t*>(&raw);
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int i = 0; i < N; ++i) x[i] = __uint_as_float(u[i]);
            } else {
#pragma unroll
                for (int i = 0; i < N / 2; ++i) {
                    if constexpr (std::is_same_v<T, __nv_bfloat16>) {
                        x[2 * i] = __uint_as_float(u[i] << 16);
                        x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
                    } else {
                        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
                        x[2 * i] = f.x;
                        x[2 * i + 1] = f.y;
                    }
                }
            }
        }
    }
    __device__ __forceinline__ void pack(const float (&x)[N]) {
        if constexpr (N * sizeof(T) == 2) {
            const T t = from_float<T>(x[0]);
            raw = *reinterpret_cast<const uint16_t*>(&t);
        } else {
            uint32_t* u = reinterpret_cast<uint32_t*>(&raw);
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int i = 0; i < N; ++i) u[i] = __float_as_uint(x[i]);
            } else {
#pragma unroll
                for (int i = 0; i < N / 2; ++i) {
                    if constexpr (std::is_same_v<T, __nv_bfloat16>) {
                        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
                        u[i] = *reinterpret_cast<const uint32_t*>(&h);
                    } else {
                        const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
                        u[i] = *reinterpret_cast<const uint32_t*>(&h);
                    }
                }
            }
        }
    }
};

// 2^t and 1/v by the special function unit, 2^-22 and 2 ulp off, subnormals flushed.
__device__ __forceinline__ float exp2_fast(float t) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    return e;
}
__device__ __forceinline__ float inverse_fast(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

__device__ __forceinline__ float2 sub2(float2 a, float2 b) { return fma2(b, make_float2(-1.0f, -1.0f), a); }

// Keys whose order is the value's, for selection by integer comparison.
// Equal values (-0 and +0 among them) get equal keys; 0 is left for "no
// candidate", which NaN and -inf map to: a selection never takes them.
__device__ __forceinline__ uint32_t choice_key(float v) {
    if (!(v > neg_inf())) return 0u;
    const uint32_t u = __float_as_uint(v + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ uint64_t choice_key(double v) {
    if (!(v > static_cast<double>(neg_inf()))) return 0ull;
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
    return (u >> 63) ? ~u : (u | (1ull << 63));
}
__device__ __forceinline__ float key_value(uint32_t k) {
    if (k == 0u) return neg_inf();
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ double key_value(uint64_t k) {
    if (k == 0ull) return static_cast<double>(neg_inf());
    return __longlong_as_double(static_cast<long long>((k >> 63) ? (k & ~(1ull << 63)) : ~k));
}

// Programmatic dependent launch: a kernel launched with launch_after() may start
// while the kernel before it in the stream drains, and reads that kernel's
// results only behind grid_wait().  The kernel before lets it start with
// grid_release(); its writes are visible behind the wait in any case.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_release() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

template <class... P, class... A>
cudaError_t launch_after(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem,
                         cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

inline size_t type_bytes(int type) { return type == 0 ? 4 : 2; }
inline bool aligned_to(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) % n) == 0; }

// Device of a call: resolved and present, or a status with its message.
int operator_device(int device, int* out);

// Calls fn with a value of the element type that `type` (mflat_storage_t) names.
template <class Fn>
cudaError_t with_type(int type, Fn&& fn) {
    switch (type) {
        case 0: return fn(float{});
        case 1: return fn(__half{});
        default: return fn(__nv_bfloat16{});
    }
}

}  // namespace mflat_cu
