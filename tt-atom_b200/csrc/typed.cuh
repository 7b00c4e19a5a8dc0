// Shared by the typed operators (gated feed-forward, adapters): element types, their loads and
// stores, the workspace cursor and a plain product.
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

// The gate's activation and its derivative (ACT 0 SiLU, 1 sigmoid, 2 GELU in its erf form).
__device__ __forceinline__ void act_grad(float g, int act, float& a, float& da) {
    if (act == 2) {
        const float phi = 0.5f * erfcf(-0.70710678f * g);
        a = g * phi;
        da = phi + g * 0.39894228f * expf(-0.5f * g * g);
    } else {
        const float p = sigmoid_f(g);
        a = act == 1 ? p : g * p;
        da = act == 1 ? p * (1.f - p) : p * (1.f + g * (1.f - p));
    }
}

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

// C[m, n] = sum_k A[m * am + k * ak] * B[n * bn + k * bk] (+ the same of A2, B2 where A2 is not
// NULL), types by code, sums in fp32.
struct PlainProduct {
    const void* A;
    long long am, ak;
    int ta;
    const void* B;
    long long bn, bk;
    int tb;
    void* C;
    long long ldc;
    int tc;
    long long M, N, K;
    const void* A2;
    const void* B2;
};

__global__ void plain_product_kernel(PlainProduct p);
int plain_product(const PlainProduct& p, cudaStream_t st);

}  // namespace atom
