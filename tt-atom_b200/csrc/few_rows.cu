// Products of a few rows: y = x W^T (or act(x Wg^T) (x Wu^T)) with at most 16 rows, where a
// tensor-core tile of 256 rows would be all but empty and the time goes into reading W and into
// launches. A block has 8 rows of W (of both matrices of a gate) and its 8 warps split K; each lane
// reads 16 bytes of W at a time straight into the fragments of m16n8k16 (rows of x are the 16,
// rows of W the 8; K runs in the order that the loads give, which both operands share), so a block
// has all its bytes of W in flight after a few instructions. Bound by HBM or L2: the launch that
// follows in an operator starts early and has its first weights before it waits for the rows.
// 1 x 1,024 x 4,096 in bf16 (25 MB of weights): 8.7 us for both launches, 2.9 TB/s; the floor is 3.9.
// The backward pass sums down the columns of W (down_kernel: fp32 sums in registers, K shared out
// over warps and blocks) and writes outer products of the rows (outer_kernel), in fp32 throughout.
#include <algorithm>

#include "few_rows.cuh"

namespace atom {
namespace few {

// 8 (fp32: 4) elements of a row from k on, zeros past its end.
__device__ __forceinline__ uint4 load16(const unsigned short* row, int k, int K, bool vec) {
    if (vec) return *reinterpret_cast<const uint4*>(row + k);
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        w[j] = (k + 2 * j < K ? row[k + 2 * j] : 0u) |
               (k + 2 * j + 1 < K ? (uint32_t)row[k + 2 * j + 1] << 16 : 0u);
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ float4 load16(const float* row, int k, int K, bool vec) {
    if (vec) return *reinterpret_cast<const float4*>(row + k);
    return make_float4(row[k], k + 1 < K ? row[k + 1] : 0.f, k + 2 < K ? row[k + 2] : 0.f,
                       k + 3 < K ? row[k + 3] : 0.f);
}
// Whether rows of K elements, ld apart, start on 16 bytes and end there.
__device__ __forceinline__ bool rows16(const void* p, int K, long long ld, int dtype) {
    const int e = dtype == ATOM_F32 ? 4 : 8;
    return aligned16(p) && K % e == 0 && ld % e == 0;
}

// The block's sums of ROWS rows by 8 columns (red: [warp][matrix][ROWS][8]) into out.
template <bool GATED, int ROWS>
__device__ __forceinline__ void finish(const Args& p, const float* red, int n0) {
    __syncthreads();
    const int i = threadIdx.x, m = i >> 3, n = n0 + (i & 7);
    if (i >= ROWS * 8 || m >= p.M || n >= p.N) return;
    constexpr int kMats = GATED ? 2 : 1;
    float v = 0.f, u = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        v += red[k * kMats * ROWS * 8 + i];
        if (GATED) u += red[(k * kMats + 1) * ROWS * 8 + i];
    }
    if (GATED && p.dh) {
        float d = 0.f, a, da;
        const long long at = (long long)m * p.N + n, all = (long long)p.M * p.N;
#pragma unroll 8
        for (int k = 0; k < p.dh_parts; ++k) d += p.dh[k * all + at];
        if (p.act == 2) {
            const float phi = 0.5f * erfcf(-0.70710678f * v);
            a = v * phi;
            da = phi + v * 0.39894228f * expf(-0.5f * v * v);
        } else {
            const float s = sigmoid_f(v);
            a = p.act == 1 ? s : v * s;
            da = s * (p.act == 1 ? sigmoid_f(-v) : 1.f + v * (1.f - s));
        }
        p.grads[at] = d * u * da;
        p.grads[all + at] = d * a;
        p.grads[2 * all + at] = a * u;
        return;
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
    const bool xv = rows16(p.x, p.K, p.ldx, p.dtype), wv = rows16(p.w[0], p.K, p.K, p.dtype) &&
                                                           (!GATED || aligned16(p.w[kMats - 1]));
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
                v[u][j] = in && in_w ? load16(w[j], k, p.K, wv) : zero;
        }
        if (!waited) {
            wait_before();
            waited = true;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = (c + u) * 32 + t8;
            const bool in = c + u < end && k < p.K;
            a[u] = in && in0 ? load16(x0, k, p.K, xv) : zero;
            b[u] = in && in1 ? load16(x1, k, p.K, xv) : zero;
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < kMats; ++j) {
                mma16816<BF16>(acc[j], a[u].x, b[u].x, a[u].y, b[u].y, v[u][j].x, v[u][j].y);
                mma16816<BF16>(acc[j], a[u].z, b[u].z, a[u].w, b[u].w, v[u][j].z, v[u][j].w);
            }
    }
#pragma unroll
    for (int j = 0; j < kMats; ++j) {
        float* r = red + (warp * kMats + j) * 128 + g * 8 + (lane & 3) * 2;
        *reinterpret_cast<float2*>(r) = make_float2(acc[j][0], acc[j][1]);
        *reinterpret_cast<float2*>(r + 64) = make_float2(acc[j][2], acc[j][3]);
    }
    finish<GATED, 16>(p, red, n0);
}

// fp32: 8 rows of W by 8 of x a warp (more rows in passes over the block's W, all but the
// first from L1), float4 along K, the 64 sums added over the lanes by halves.
template <bool GATED>
__global__ void __launch_bounds__(256, 2) few32_kernel(const __grid_constant__ Args p) {
    constexpr int kMats = GATED ? 2 : 1;
    __shared__ float red[8 * kMats * kFewRows * 8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n0 = blockIdx.x * 8;
    let_next_start();
    const int chunks = (p.K + 127) / 128, first = chunks * warp / 8, end = chunks * (warp + 1) / 8;
    const bool xv = rows16(p.x, p.K, p.ldx, ATOM_F32), wv = rows16(p.w[0], p.K, p.K, ATOM_F32) &&
                                                            (!GATED || aligned16(p.w[kMats - 1]));
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    bool waited = false;
    for (int m0 = 0; m0 < p.M; m0 += 8) {
#pragma unroll 1
        for (int j = 0; j < kMats; ++j) {
            float acc[64];
#pragma unroll
            for (int i = 0; i < 64; ++i) acc[i] = 0.f;
            const float* w = static_cast<const float*>(p.w[j]) + (long long)n0 * p.K;
            const float* x = static_cast<const float*>(p.x) + m0 * p.ldx;
            for (int c = first; c < end || !waited; ++c) {
                const int k = c * 128 + lane * 4;
                const bool in = c < end && k < p.K;
                float4 b[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    b[i] = in && n0 + i < p.N ? load16(w + (long long)i * p.K, k, p.K, wv) : zero;
                if (!waited) {
                    wait_before();
                    waited = true;
                }
#pragma unroll
                for (int i0 = 0; i0 < 8; i0 += 4) {          // four rows' loads at once
                    if (m0 + i0 >= p.M) break;
                    float4 a[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        a[i] = in && m0 + i0 + i < p.M
                            ? load16(x + (i0 + i) * p.ldx, k, p.K, xv) : zero;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int n = 0; n < 8; ++n) {
                            float& v = acc[8 * (i0 + i) + n];
                            v = fmaf(a[i].x, b[n].x, fmaf(a[i].y, b[n].y,
                                fmaf(a[i].z, b[n].z, fmaf(a[i].w, b[n].w, v))));
                        }
                }
            }
            sum_halves<64>(acc, lane);
            *reinterpret_cast<float2*>(red + (warp * kMats + j) * kFewRows * 8 + m0 * 8 + 2 * lane) =
                make_float2(acc[0], acc[1]);
        }
    }
    finish<GATED, kFewRows>(p, red, n0);
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
    const bool xv = rows16(p.x, p.K, p.ldx, p.dtype), wv = rows16(p.a, p.K, p.K, p.dtype);
    if (p.dtype == ATOM_F32) {
        const float* x = static_cast<const float*>(p.x) + m * p.ldx;
        const float* w = static_cast<const float*>(p.a) + at;
#pragma unroll 4
        for (int k = lane * 4; k < p.K; k += 128) {
            const float4 c = load16(x, k, p.K, xv), d = load16(w, k, p.K, wv);
            v = fmaf(c.x, d.x, fmaf(c.y, d.y, fmaf(c.z, d.z, fmaf(c.w, d.w, v))));
        }
    } else {
        const unsigned short* x = static_cast<const unsigned short*>(p.x) + m * p.ldx;
        const unsigned short* w = static_cast<const unsigned short*>(p.a) + at;
#pragma unroll 4
        for (int k = lane * 8; k < p.K; k += 256) {
            const uint4 c = load16(x, k, p.K, xv), d = load16(w, k, p.K, wv);
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

// A block a row: threads have eight ranks and a share of O.
__global__ void __launch_bounds__(256) low_back_kernel(const __grid_constant__ LowBackArgs p) {
    __shared__ float red[256][9];
    let_next_start();
    wait_before();
    const int m = blockIdx.x, a = p.slot[m];
    if (a < 0) return;
    const int chunks = (p.R + 7) / 8, groups = 256 / chunks;
    const int g = threadIdx.x / chunks, r0 = (threadIdx.x - g * chunks) * 8;
    float acc[8] = {};
    const bool vec = p.R % 8 == 0 && aligned16(p.b);
    if (g < groups) {
        const int n = min(8, p.R - r0);
        const long long at = (long long)a * p.O * p.R + r0;
#pragma unroll 8
        for (int o = g; o < p.O; o += groups) {
            const float y = load_f(p.dy, m * p.ld + o, p.dtype);
            const long long e = at + (long long)o * p.R;
            float v[8];
            if (vec && p.dtype != ATOM_F32) {
                const uint4 w = *reinterpret_cast<const uint4*>(
                    static_cast<const unsigned short*>(p.b) + e);
                const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 f = pair_f(ww[j], p.dtype);
                    v[2 * j] = f.x, v[2 * j + 1] = f.y;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = j < n ? load_f(p.b, e + j, p.dtype) : 0.f;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] = fmaf(y, v[j], acc[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) red[threadIdx.x][j] = acc[j];
    __syncthreads();
    for (int r = threadIdx.x >> 5; r < p.R; r += 8) {        // a warp a rank
        float v = 0.f;
        for (int k = threadIdx.x & 31; k < groups; k += 32) v += red[k * chunks + (r >> 3)][r & 7];
        v = warp_sum(v);
        if ((threadIdx.x & 31) == 0) p.T[m * p.R + r] = v * p.scale[a];
    }
}

// A block has 64 columns, two a lane, and a share of K, of which its 8 warps take every eighth
// row; the warps' sums meet in shared memory, in order. Bound by loading W: few columns a thread
// leave registers for 32 warps an SM (8 columns: 178 registers, one block an SM, twice the time).
template <int DT, int MR>
__global__ void __launch_bounds__(256) down_kernel(const __grid_constant__ DownArgs p) {
    constexpr int kW = 64, kK = 128;
    __shared__ __align__(16) float as[kK][MR + 4];
    __shared__ __align__(8) float red[8][MR][kW / 2];
    let_next_start();
    wait_before();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockIdx.x * kW + lane * 2;
    const int lo = (int)((long long)p.K * blockIdx.y / p.shares);
    const int hi = (int)((long long)p.K * (blockIdx.y + 1) / p.shares);
    const bool vec = p.N % 2 == 0 && ((uintptr_t)p.w[0] & 7) == 0 && ((uintptr_t)p.w[1] & 7) == 0;
    float acc[2][MR] = {};
    for (int j = 0; j < (p.a[1] ? 2 : 1); ++j)
        for (int k0 = lo; k0 < hi; k0 += kK) {
            __syncthreads();
            for (int i = threadIdx.x; i < kK * MR; i += 256) {
                const int k = k0 + i % kK, m = i / kK;
                as[i % kK][m] = k < hi && m < p.M
                    ? load_f(p.a[j], m * p.lda + k, p.a32 ? ATOM_F32 : DT) : 0.f;
            }
            __syncthreads();
            if (n >= p.N) continue;
#pragma unroll 8
            for (int i = warp; i < min(kK, hi - k0); i += 8) {
                const long long at = (long long)(k0 + i) * p.N + n;
                float2 w;
                if (vec)
                    w = DT == ATOM_F32
                        ? *reinterpret_cast<const float2*>(static_cast<const float*>(p.w[j]) + at)
                        : pair_f(*reinterpret_cast<const uint32_t*>(
                                     static_cast<const unsigned short*>(p.w[j]) + at), DT);
                else
                    w = make_float2(load_f(p.w[j], at, DT),
                                    n + 1 < p.N ? load_f(p.w[j], at + 1, DT) : 0.f);
#pragma unroll
                for (int m = 0; m < MR; m += 4) {
                    const float4 x = *reinterpret_cast<const float4*>(&as[i][m]);
                    const float xx[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        acc[0][m + e] = fmaf(xx[e], w.x, acc[0][m + e]);
                        acc[1][m + e] = fmaf(xx[e], w.y, acc[1][m + e]);
                    }
                }
            }
        }
    for (int c = 0; c < 2; ++c) {                    // even columns, odd ones
        __syncthreads();
#pragma unroll
        for (int m = 0; m < MR; ++m) red[warp][m][lane] = c ? acc[1][m] : acc[0][m];
        __syncthreads();
        for (int i = threadIdx.x; i < p.M * 32; i += 256) {
            const int m = i >> 5, col = blockIdx.x * kW + 2 * lane + c;
            float v = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) v += red[k][m][lane];
            if (col < p.N) p.part[((long long)blockIdx.y * p.M + m) * p.N + col] = v;
        }
    }
}
// 32 columns of a row a block; its 8 warps share out the shares and the ranks.
__global__ void __launch_bounds__(256) sum_kernel(const __grid_constant__ SumArgs p) {
    __shared__ float red[8][32];
    let_next_start();
    wait_before();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockIdx.x * 32 + lane;
    const int m = blockIdx.y, a = p.T ? p.slot[m] : -1;
    float v = 0.f;
    if (n < p.N) {
#pragma unroll 8
        for (int k = warp; k < p.shares; k += 8) v += p.part[((long long)k * p.M + m) * p.N + n];
        if (a >= 0) {
            const long long at = (long long)a * p.R * p.N + n;
#pragma unroll 4
            for (int r = warp; r < p.R; r += 8)
                v = fmaf(p.T[m * p.R + r], load_f(p.a, at + (long long)r * p.N, p.dtype), v);
        }
    }
    red[warp][lane] = v;
    __syncthreads();
    if (warp || n >= p.N) return;
#pragma unroll
    for (int k = 1; k < 8; ++k) v += red[k][lane];
    store_f(p.out, m * p.ldo + n, v, p.dtype);
}

// 64 rows by 256 columns a block, twice 4 by 8 a thread. Bound by writing: three matrices of 2,000 x
// 5,784 in fp16 from 4 rows take 29 us, 2.4 TB/s.
__global__ void __launch_bounds__(256) outer_kernel(const __grid_constant__ OuterArgs p) {
    constexpr int kRows = 64;
    __shared__ float ps[kFewRows][kRows];
    __shared__ float qs[kFewRows][256];
    let_next_start();
    wait_before();
    int k = 0;
    while (k + 1 < p.n && blockIdx.x >= p.first[k + 1]) ++k;
    const OuterItem& it = p.it[k];
    const int tiles = (it.J + 255) / 256, b = blockIdx.x - p.first[k];
    const int i0 = b / tiles * kRows, j0 = b % tiles * 256;
    for (int i = threadIdx.x; i < p.M * kRows; i += 256) {
        const int m = i / kRows, c = i0 + i % kRows;
        ps[m][i % kRows] = c < it.I ? load_f(it.p, m * it.ldp + c, it.p32 ? ATOM_F32 : p.dtype) : 0.f;
    }
    for (int i = threadIdx.x; i < p.M * 256; i += 256) {
        const int m = i >> 8, c = j0 + (i & 255);
        qs[m][i & 255] = c < it.J ? load_f(it.q, m * it.ldq + c, it.q32 ? ATOM_F32 : p.dtype) : 0.f;
    }
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool vec = rows16(it.out, it.J, it.J, p.dtype);
    for (int r0 = 0; r0 < kRows && i0 + r0 < it.I; r0 += 32) {
        float acc[4][8] = {};
        for (int m = 0; m < p.M; ++m) {
            float x[4], y[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = ps[m][r0 + warp * 4 + i];
#pragma unroll
            for (int j = 0; j < 8; j += 4) {
                const float4 v = *reinterpret_cast<const float4*>(&qs[m][lane * 4 + 32 * j]);
                y[j] = v.x, y[j + 1] = v.y, y[j + 2] = v.z, y[j + 3] = v.w;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) acc[i][j] = fmaf(x[i], y[j], acc[i][j]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = i0 + r0 + warp * 4 + i;
            if (r >= it.I) continue;
#pragma unroll
            for (int h = 0; h < 8; h += 4) {
                const int c = j0 + lane * 4 + 32 * h;
                const long long at = (long long)r * it.J + c;
                const float* v = acc[i] + h;
                if (c >= it.J) continue;
                if (!vec) {
                    for (int j = 0; j < 4; ++j)
                        if (c + j < it.J) store_f(it.out, at + j, v[j], p.dtype);
                } else if (p.dtype == ATOM_F32) {
                    *reinterpret_cast<float4*>(static_cast<float*>(it.out) + at) =
                        make_float4(v[0], v[1], v[2], v[3]);
                } else {
                    *reinterpret_cast<uint2*>(static_cast<unsigned short*>(it.out) + at) =
                        make_uint2(pair_w(v[0], v[1], p.dtype), pair_w(v[2], v[3], p.dtype));
                }
            }
        }
    }
}

// Blocks of 256 columns of x, which write all ranks of dA, then blocks of 2,048 elements of dB.
__global__ void __launch_bounds__(256) adapter_grads_kernel(const __grid_constant__ GradArgs p) {
    let_next_start();
    wait_before();
    const int a = blockIdx.y, xb = p.da ? (p.D + 255) / 256 : 0;
    unsigned mine = 0;
#pragma unroll
    for (int m = 0; m < kFewRows; ++m)
        if (m < p.M && p.slot[m] == a) mine |= 1u << m;
    if ((int)blockIdx.x < xb) {
        const int k = blockIdx.x * 256 + threadIdx.x;
        if (k >= p.D) return;
        float v[kFewRows];
#pragma unroll
        for (int m = 0; m < kFewRows; ++m)
            v[m] = mine >> m & 1 ? load_f(p.x, m * p.ldx + k, p.dtype) : 0.f;
        for (int r = 0; r < p.R; ++r) {
            float s = 0.f;
#pragma unroll
            for (int m = 0; m < kFewRows; ++m)
                if (mine >> m & 1) s = fmaf(p.T[m * p.R + r], v[m], s);
            store_f(p.da, ((long long)a * p.R + r) * p.D + k, s, p.dtype);
        }
        return;
    }
    const long long all = (long long)p.O * p.R, at = (long long)(blockIdx.x - xb) * 2048 + threadIdx.x;
#pragma unroll 2
    for (int j = 0; j < 8; ++j) {
        const long long i = at + 256 * j;
        if (i >= all) return;
        const int o = (int)((unsigned)i / (unsigned)p.R), r = (int)(i - (long long)o * p.R);
        float s = 0.f;
        for (int m = 0; m < p.M; ++m)
            if (mine >> m & 1)
                s = fmaf(p.S[m * p.R + r], load_f(p.dy, m * p.lddy + o, p.dtype), s);
        store_f(p.db, a * all + i, s, p.dtype);
    }
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
int low_rank_back(const LowBackArgs& p, Chain& st) {
    return st.launch("low-rank part of a few rows", low_back_kernel, dim3(p.M), 256, 0, p);
}

// Shares of K that give the GPU some four blocks an SM, 32 rows each at least (11 rows, 2 x 7,688 x
// 224 in bf16: 27 us with 148, 52 with 32).
int down_shares(int K, int N, int most) {
    return std::max(1, std::min({592 / ((N + 63) / 64), K / 32, most}));
}
int down(const DownArgs& p, Chain& st) {
    const bool half = p.M <= 8;
    void (*k)(DownArgs) =
        p.dtype == ATOM_F32    ? (half ? down_kernel<ATOM_F32, 8> : down_kernel<ATOM_F32, 16>)
        : p.dtype == ATOM_BF16 ? (half ? down_kernel<ATOM_BF16, 8> : down_kernel<ATOM_BF16, 16>)
                               : (half ? down_kernel<ATOM_F16, 8> : down_kernel<ATOM_F16, 16>);
    return st.launch("product of a few rows", k, dim3((p.N + 63) / 64, p.shares), 256, 0, p);
}
int sum(const SumArgs& p, Chain& st) {
    return st.launch("sums of a few rows", sum_kernel, dim3((p.N + 31) / 32, p.M), 256, 0, p);
}
int outer(OuterArgs p, Chain& st) {
    int n = 0;
    for (int i = 0; i < p.n; ++i) {
        p.first[i] = n;
        n += (p.it[i].I + 63) / 64 * ((p.it[i].J + 255) / 256);
    }
    return n ? st.launch("outer products of a few rows", outer_kernel, dim3(n), 256, 0, p) : ATOM_OK;
}
int adapter_grads(const GradArgs& p, Chain& st) {
    const long long n = (p.da ? (p.D + 255) / 256 : 0) +
                        (p.db ? ((long long)p.O * p.R + 2047) / 2048 : 0);
    return st.launch("adapters' gradients of a few rows", adapter_grads_kernel, dim3(n, p.nad), 256,
                     0, p);
}

}  // namespace few
}  // namespace atom
