// Shared by the typed operators (gated feed-forward, adapters): element types, their loads and
// stores, launches and the workspace cursor.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <stddef.h>

#include "common.cuh"

namespace atom {

inline int dtype_size(int dtype) { return dtype == ATOM_F32 ? 4 : 2; }

__device__ __forceinline__ float load_f(const void* p, long long i, int dtype) {
    if (dtype == ATOM_F32) return static_cast<const float*>(p)[i];
    if (dtype == ATOM_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_f(void* p, long long i, float v, int dtype) {
    if (dtype == ATOM_F32) static_cast<float*>(p)[i] = v;
    else if (dtype == ATOM_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// fp32 as three bf16 planes, x = hi + mid + lo exactly (8 significant bits each; hi is truncated, so
// that it is finite where x is). They have fp32's range, so nothing is scaled and a value keeps its
// bits whatever lies beside it, down to 2^-110 (where lo leaves the normal numbers). An infinity has a
// NaN in mid, so what is not finite comes out as NaN.
constexpr int kPlanes = 3;
// Plane `k` of two values, the first in the lower half; takes it off them, planes in order.
__device__ __forceinline__ uint32_t take_plane(float& x0, float& x1, int k) {
    uint32_t w;
    if (k == 0) {
        w = __byte_perm(__float_as_uint(x0), __float_as_uint(x1), 0x7632);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x0, x1);
        w = *reinterpret_cast<const uint32_t*>(&h);
    }
    x0 -= __uint_as_float(w << 16);
    x1 -= __uint_as_float(w & 0xFFFF0000u);
    return w;
}

// The last r in 0 .. n - 1 with value(r) <= key, or -1; value ascending, one warp.
template <typename V>
__device__ __forceinline__ int last_le(int n, int key, V value) {
    const int lane = threadIdx.x & 31;
    int lo = 0;
    while (n > 0) {
        const int step = (n + 31) / 32, i = lo + lane * step;
        const unsigned yes = __ballot_sync(0xffffffffu, lane * step < n && value(i) <= key);
        const int count = __popc(yes);
        if (count == 0) return lo - 1;
        if (step == 1) return lo + count - 1;
        lo += (count - 1) * step;
        n = min(step, n - (count - 1) * step);
        // value(lo) <= key holds: look behind it
        if (n == 1) return lo;
    }
    return lo - 1;
}

// Adds N values (64 or 32) over a warp by halves: lane l ends with sum l N / 32 and, of 64, the one
// behind it in v[0], v[1].
template <int N>
__device__ __forceinline__ void sum_halves(float* v, int lane) {
#pragma unroll
    for (int o = 16, n = N / 2; o > 0; o >>= 1, n >>= 1) {
        const bool up = lane & o;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const float mine = up ? v[n + i] : v[i], other = up ? v[i] : v[n + i];
            v[i] = mine + __shfl_xor_sync(0xffffffffu, other, o);
        }
    }
}
// Two 16-bit values of a word.
__device__ __forceinline__ float2 pair_f(uint32_t w, int dtype) {
    return dtype == ATOM_BF16 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w))
                              : __half22float2(*reinterpret_cast<const __half2*>(&w));
}

__device__ __forceinline__ uint32_t pair_w(float a, float b, int dtype) {
    if (dtype == ATOM_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// m16n8k16 of 16-bit operands, added to c.
template <bool BF16>
__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
            "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
            "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A call's kernels on its stream. Each after the first starts while the one before it still runs
// (it sets up, then waits in wait_before() for what that one writes), which hides the launches.
struct Chain {
    cudaStream_t st;
    bool after = false;
    Chain(cudaStream_t s) : st(s) {}
    template <typename... P, typename... A>
    int launch(const char* what, void (*kernel)(P...), dim3 grid, int block, size_t smem,
               const A&... args) {
        cudaLaunchConfig_t c{};
        cudaLaunchAttribute at;
        at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at.val.programmaticStreamSerializationAllowed = 1;
        c.gridDim = grid;
        c.blockDim = dim3(block);
        c.dynamicSmemBytes = smem;
        c.stream = st;
        c.attrs = &at;
        c.numAttrs = after ? 1 : 0;
        cudaLaunchKernelEx(&c, kernel, args...);
        after = true;
        return check_launch(what);
    }
};
// Waits for the kernel before this one (a launch without overlap: at once).
__device__ __forceinline__ void wait_before() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void let_next_start() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

inline bool aligned256(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 255u) == 0; }

// Pieces of a caller's workspace, 256-byte aligned; with base NULL it only adds up the sizes.
struct Cursor {
    char* base;
    size_t used = 0;
    explicit Cursor(void* p) : base(static_cast<char*>(p)) {}
    template <typename T>
    T* take(size_t n) {
        T* p = base ? reinterpret_cast<T*>(base + used) : nullptr;
        used += (n * sizeof(T) + 255) / 256 * 256;
        return p;
    }
};

}  // namespace atom
