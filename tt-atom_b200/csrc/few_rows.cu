// Products of a few rows: y = x W^T (or act(x Wg^T) (x Wu^T)) with at most 16 rows, where a
// tensor-core tile of 256 rows would be all but empty and the time goes into reading W and into
// launches. A block has 8 rows of W (of both matrices of a gate) and its 8 warps split K; each lane
// reads 16 bytes of W at a time straight into the fragments of m16n8k16 (rows of x are the 16,
// rows of W the 8; K runs in the order that the loads give, which both operands share), so a block
// has all its bytes of W in flight after a few instructions. Bound by HBM or L2: the launch that
// follows in an operator starts early and has its first weights before it waits for the rows.
#include "few_rows.cuh"

namespace atom {
namespace few {

template <bool BF16>
__device__ __forceinline__ void mma(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                    uint32_t b0, uint32_t b1) {
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
// The block's sums of 16 rows by 8 columns (red: [warp][matrix][16][8]) into out.
template <bool GATED>
__device__ __forceinline__ void finish(const Args& p, const float* red, int n0) {
    __syncthreads();
    const int i = threadIdx.x, m = i >> 3, n = n0 + (i & 7);
    if (i >= 128 || m >= p.M || n >= p.N) return;
    constexpr int kMats = GATED ? 2 : 1;
    float v = 0.f, u = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        v += red[k * kMats * 128 + i];
        if (GATED) u += red[k * kMats * 128 + 128 + i];
    }
    if (GATED) {
        if (p.act == 2) v *= 0.5f * erfcf(-0.70710678f * v);
        else v = (p.act == 1 ? 1.f : v) * sigmoid_f(v);
        v *= u;
    } else if (p.S) {
        const int a = p.slot[m];
        if (a >= 0) {
            const float* s = p.S + m * p.R;
            const long long b = ((long long)a * p.N + n) * p.R;
            for (int r = 0; r < p.R; ++r) v = fmaf(s[r], load_f(p.b, b + r, p.dtype), v);
        }
    }
    store_f(p.out, m * p.ldo + n, v, p.dtype);
}

// HALF: at most 8 rows, whose fragments' other half stays zero.
template <bool BF16, bool GATED, bool HALF>
__global__ void __launch_bounds__(256) few16_kernel(const __grid_constant__ Args p) {
    constexpr int kMats = GATED ? 2 : 1, U = GATED ? 4 : 8;
    __shared__ float red[8 * kMats * 128];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t8 = (lane & 3) * 8, n0 = blockIdx.x * 8;
    let_next_start();
    const bool in_w = n0 + g < p.N;
    const unsigned short* w[kMats];
#pragma unroll
    for (int j = 0; j < kMats; ++j)
        w[j] = static_cast<const unsigned short*>(p.w[j]) + (long long)(n0 + g) * p.K;
    const unsigned short* x0 = static_cast<const unsigned short*>(p.x) + g * p.ldx;
    const unsigned short* x1 = x0 + 8 * p.ldx;
    const bool in0 = g < p.M, in1 = !HALF && g + 8 < p.M;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    const int chunks = (p.K + 31) / 32, end = chunks * (warp + 1) / 8;
    float acc[kMats][4] = {};
    bool waited = false;
    for (int c = chunks * warp / 8; c < end || !waited; c += U) {
        uint4 v[U][kMats], a[U], b[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = (c + u) * 32 + t8;
            const bool in = c + u < end && k < p.K;
#pragma unroll
            for (int j = 0; j < kMats; ++j)
                v[u][j] = in && in_w ? __ldg(reinterpret_cast<const uint4*>(w[j] + k)) : zero;
        }
        if (!waited) {
            wait_before();
            waited = true;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = (c + u) * 32 + t8;
            const bool in = c + u < end && k < p.K;
            a[u] = in && in0 ? *reinterpret_cast<const uint4*>(x0 + k) : zero;
            b[u] = in && in1 ? *reinterpret_cast<const uint4*>(x1 + k) : zero;
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < kMats; ++j) {
                mma<BF16>(acc[j], a[u].x, b[u].x, a[u].y, b[u].y, v[u][j].x, v[u][j].y);
                mma<BF16>(acc[j], a[u].z, b[u].z, a[u].w, b[u].w, v[u][j].z, v[u][j].w);
            }
    }
#pragma unroll
    for (int j = 0; j < kMats; ++j) {
        float* r = red + (warp * kMats + j) * 128 + g * 8 + (lane & 3) * 2;
        *reinterpret_cast<float2*>(r) = make_float2(acc[j][0], acc[j][1]);
        *reinterpret_cast<float2*>(r + 64) = make_float2(acc[j][2], acc[j][3]);
    }
    finish<GATED>(p, red, n0);
}

// fp32: 8 rows of W by 8 of x a warp (16 rows in two passes over the block's W, the second from
// L1), float4 along K, the 64 sums added over the lanes by halves.
template <bool GATED>
__global__ void __launch_bounds__(256) few32_kernel(const __grid_constant__ Args p) {
    constexpr int kMats = GATED ? 2 : 1;
    __shared__ float red[8 * kMats * 128];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n0 = blockIdx.x * 8;
    let_next_start();
    const int chunks = (p.K + 127) / 128, first = chunks * warp / 8, end = chunks * (warp + 1) / 8;
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    bool waited = false;
    for (int m0 = 0; m0 < 16; m0 += 8) {
#pragma unroll
        for (int j = 0; j < kMats; ++j) {
            float acc[64];
#pragma unroll
            for (int i = 0; i < 64; ++i) acc[i] = 0.f;
            const float* w = static_cast<const float*>(p.w[j]) + (long long)n0 * p.K;
            const float* x = static_cast<const float*>(p.x) + m0 * p.ldx;
            for (int c = first; m0 < p.M && (c < end || !waited); ++c) {
                const int k = c * 128 + lane * 4;
                const bool in = c < end && k < p.K;
                float4 b[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    b[i] = in && n0 + i < p.N
                               ? __ldg(reinterpret_cast<const float4*>(w + (long long)i * p.K + k))
                               : zero;
                if (!waited) {
                    wait_before();
                    waited = true;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (m0 + i >= p.M) break;
                    const float4 a = in ? *reinterpret_cast<const float4*>(x + i * p.ldx + k) : zero;
#pragma unroll
                    for (int n = 0; n < 8; ++n)
                        acc[8 * i + n] = fmaf(a.x, b[n].x, fmaf(a.y, b[n].y,
                                         fmaf(a.z, b[n].z, fmaf(a.w, b[n].w, acc[8 * i + n]))));
                }
            }
            sum_halves<64>(acc, lane);
            *reinterpret_cast<float2*>(red + (warp * kMats + j) * 128 + m0 * 8 + 2 * lane) =
                make_float2(acc[0], acc[1]);
        }
    }
    finish<GATED>(p, red, n0);
}

// One warp a value of S, eight to a block; K along the lanes.
__global__ void __launch_bounds__(256) low_kernel(const __grid_constant__ LowArgs p) {
    const int lane = threadIdx.x & 31, m = blockIdx.y, r = blockIdx.x * 8 + (threadIdx.x >> 5);
    let_next_start();
    wait_before();
    const int q = last_le(p.nreq, m, [&](int i) { return min(max(p.ptr[i], 0), p.M); });
    int a = -1;
    if (q >= 0 && m < p.ptr[q + 1]) a = p.adapter[q];
    if (a >= p.nad) a = -1;
    if (threadIdx.x == 0 && blockIdx.x == 0) p.slot[m] = a;
    if (a < 0 || r >= p.R) return;
    float v = 0.f;
    const long long at = ((long long)a * p.R + r) * p.K;
    if (p.dtype == ATOM_F32) {
        const float* x = static_cast<const float*>(p.x) + m * p.ldx;
        const float* w = static_cast<const float*>(p.a) + at;
#pragma unroll 4
        for (int k = lane * 4; k < p.K; k += 128) {
            const float4 c = *reinterpret_cast<const float4*>(x + k);
            const float4 d = *reinterpret_cast<const float4*>(w + k);
            v = fmaf(c.x, d.x, fmaf(c.y, d.y, fmaf(c.z, d.z, fmaf(c.w, d.w, v))));
        }
    } else {
        const unsigned short* x = static_cast<const unsigned short*>(p.x) + m * p.ldx;
        const unsigned short* w = static_cast<const unsigned short*>(p.a) + at;
#pragma unroll 4
        for (int k = lane * 8; k < p.K; k += 256) {
            const uint4 c = *reinterpret_cast<const uint4*>(x + k);
            const uint4 d = *reinterpret_cast<const uint4*>(w + k);
            const uint32_t cc[4] = {c.x, c.y, c.z, c.w}, dd[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = pair_f(cc[j], p.dtype), h = pair_f(dd[j], p.dtype);
                v = fmaf(f.x, h.x, fmaf(f.y, h.y, v));
            }
        }
    }
    v = warp_sum(v);
    if (lane == 0) p.S[m * p.R + r] = v * p.scale[a];
}

bool suits(int dtype, long long M, int K, const void* x, long long ldx, const void* w0,
           const void* w1) {
    const int e = dtype == ATOM_F32 ? 4 : 8;
    return M <= kFewRows && K % e == 0 && ldx % e == 0 && aligned16(x) && aligned16(w0) &&
           aligned16(w1);
}

int product(const Args& p, Chain& st) {
    const dim3 grid((p.N + 7) / 8);
    const bool gated = p.w[1] != nullptr, half = p.M <= 8;
    void (*k)(Args) = nullptr;
#define ATOM_FEW(B, G, H) \
    if ((p.dtype == ATOM_BF16) == B && gated == G && half == H) k = few16_kernel<B, G, H>;
    if (p.dtype == ATOM_F32) {
        k = gated ? few32_kernel<true> : few32_kernel<false>;
    } else {
        ATOM_FEW(true, true, true)
        ATOM_FEW(true, true, false)
        ATOM_FEW(true, false, true)
        ATOM_FEW(true, false, false)
        ATOM_FEW(false, true, true)
        ATOM_FEW(false, true, false)
        ATOM_FEW(false, false, true)
        ATOM_FEW(false, false, false)
    }
#undef ATOM_FEW
    return st.launch("product of a few rows", k, grid, 256, 0, p);
}

int low_rank(const LowArgs& p, Chain& st) {
    return st.launch("low-rank part of a few rows", low_kernel, dim3((p.R + 7) / 8, p.M), 256, 0, p);
}

}  // namespace few
}  // namespace atom
