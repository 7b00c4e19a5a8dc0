// Low-rank adapters of many requests beside a shared projection, and their backward pass.
//
//   y = x W^T + S B^T,  S = s (x A^T) row by row with the row's own A, B and s
//
// The requests' rows are cut at every 256th row into pieces: piece t + r holds the rows of request
// r in row tile t (t + r grows along the requests, so it names a piece without a table). The
// shrink pass writes S of each piece as a block of 256 rows, zeros where the rows are not the
// request's, and the shared projection's product (pair_product.cu) then takes each piece of its
// row tile as one more K stage, S's block times the request's B: the adapters cost their own
// multiplications and no pass over y. The backward pass is the same with T = s (dy B), W and A in
// the place of S, W^T and B, and dA = T^T x, dB = dy^T S summed by pieces in their order.
//
// Zeros in a block keep other requests' rows as they are only where B is finite; an adapter that
// is not is found in the shrink pass, left out, and its own rows are set to NaN.
#include <algorithm>

#include "pair_product.cuh"

namespace atom {
namespace {

using namespace pair;

struct Requests {
    const int* ptr;
    const int* adapter;
    int n, nad;
    int M;
};
// Rows of request r, kept within 0 .. M whatever the table holds.
__device__ __forceinline__ int row_of(const Requests& q, int r) {
    return min(max(q.ptr[r], 0), q.M);
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

struct Shrink {
    Requests q;
    int pieces;              // row tiles + requests
    const void* rows;        // [M, K]
    long long ld;
    int K;
    const void* w;           // adapters: element (r, k) at a * wa + r * wr + k * wk
    long long wa, wr, wk;
    int R, Rs;               // rank, and the pitch of what is written
    const float* scale;
    const void* other;       // the adapters' other matrix: O * R (or R * D) values to look over
    long long other_n;
    int4* piece;             // adapter or -1, first row, behind the last row
    int2* tile_req;
    int tiles;
    int4* bad;               // per adapter: a quarter of `other` is not finite
    void* block;             // [pieces][256][Rs] (fp32: fp16 planes)
    long long plane;
    void* compact;           // [M][Rs], or NULL
    float* rinv;             // fp32: [M]
    int dtype;
};

// The parts of the shrink pass that are not products: the row tiles' requests, and whether the
// adapters' other matrix is finite. True when this block was one of them.
__device__ __forceinline__ bool side_work(const Shrink& p) {
    const int b = blockIdx.x - p.pieces;
    if (b < 0) return false;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (b == p.q.nad) {
        for (int t = blockIdx.y * 8 + warp; t < p.tiles; t += 32) {
            const int first = last_le(p.q.n, t * 256, [&](int r) { return row_of(p.q, r); });
            const int last = last_le(p.q.n, t * 256 + 255, [&](int r) { return row_of(p.q, r); });
            // a request that begins before the tile reaches into it at most as the last such one
            if (lane == 0) p.tile_req[t] = make_int2(max(first, 0), last + 1);
        }
        return true;
    }
    int found = 0;
    const long long lo = p.other_n * blockIdx.y / 4, hi = p.other_n * (blockIdx.y + 1) / 4;
    const long long at = (long long)b * p.other_n;
    if (p.dtype == ATOM_F32) {
        const unsigned* v = static_cast<const unsigned*>(p.other) + at;
        for (long long i = lo + threadIdx.x; i < hi; i += 256)
            found |= (v[i] & 0x7F800000u) == 0x7F800000u;
    } else {
        const unsigned short top = p.dtype == ATOM_BF16 ? 0x7F80 : 0x7C00;
        const unsigned short* v = static_cast<const unsigned short*>(p.other) + at;
        long long i = lo + threadIdx.x;
        if ((reinterpret_cast<uintptr_t>(v + lo) & 15) == 0) {
            const unsigned two = top * 0x10001u;
            const long long n8 = (hi - lo) / 8;
            for (long long j = threadIdx.x; j < n8; j += 256) {
                const uint4 x = *reinterpret_cast<const uint4*>(v + lo + 8 * j);
                const unsigned w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    found |= (w[k] & top) == top || ((w[k] & two) >> 16) == top;
            }
            i = lo + 8 * n8 + threadIdx.x;
        }
        for (; i < hi; i += 256) found |= (v[i] & top) == top;
    }
    found = __syncthreads_or(found);
    if (threadIdx.x == 0) reinterpret_cast<int*>(p.bad + b)[blockIdx.y] = found;
    return true;
}

struct Piece {
    int slot, lo, hi, m0;    // adapter; the request's rows in this tile; the tile's first row
};
// Finds piece blockIdx.x (every thread of every warp has it on return) and writes it down.
__device__ __forceinline__ Piece find_piece(const Shrink& p) {
    const int b = blockIdx.x;
    const int r = last_le(p.q.n, b, [&](int i) { return row_of(p.q, i) / 256 + i; });
    Piece c{-1, 0, 0, 0};
    if (r >= 0) {
        const int t = b - r;
        if (t < p.tiles) {
            c.m0 = t * 256;
            c.lo = max(row_of(p.q, r), c.m0);
            c.hi = min(row_of(p.q, r + 1), c.m0 + 256);
            const int a = p.q.adapter[r];
            if (c.lo < c.hi && a >= 0 && a < p.q.nad) c.slot = a;
        }
    }
    if (blockIdx.y == 0 && threadIdx.x == 0) p.piece[b] = make_int4(c.slot, c.lo, c.hi, 0);
    return c;
}

// 8 elements of a row from k on, zeros past its end.
__device__ __forceinline__ uint4 load8(const unsigned short* row, int k, int K) {
    if (k + 8 <= K) return *reinterpret_cast<const uint4*>(row + k);
    unsigned short v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k + j < K ? row[k + j] : 0;
    return *reinterpret_cast<const uint4*>(v);
}
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

// 16-bit: a block of 8 warps has 64 rows of a piece, 16 a warp, and the warps left over split K
// (all eight do for a piece of 16 rows or fewer). Rows and adapters go from memory into the
// fragments of m16n8k16 directly: the product does not mind in which order K runs, so each lane
// reads 8 consecutive elements of its row, half for one instruction and half for the next.
// Bound by reading x; an adapter's rows come from L1.
template <bool BF16, int NT>
__global__ void __launch_bounds__(256) shrink16_kernel(const __grid_constant__ Shrink p) {
    extern __shared__ float red[];       // [8 warps][16][8 NT]
    if (side_work(p)) return;
    const Piece c = find_piece(p);
    if (c.slot < 0) return;
    const int m0 = c.m0 + blockIdx.y * 64, lo = max(c.lo, m0), hi = min(c.hi, m0 + 64);
    unsigned short* block = static_cast<unsigned short*>(p.block) +
                            ((long long)blockIdx.x * 256 + blockIdx.y * 64) * p.Rs;
    if (lo >= hi) {
        for (int i = threadIdx.x; i < 64 * p.Rs; i += 256) block[i] = 0;
        return;
    }
    const int g0 = (lo - m0) / 16, groups = (hi - 1 - m0) / 16 - g0 + 1;
    const int gp = groups == 1 ? 1 : groups == 2 ? 2 : 4, parts = 8 / gp;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t8 = (lane & 3) * 8;
    const int grp = warp % gp, part = warp / gp;
    const int nt = (p.R + 7) / 8;
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
    if (grp < groups) {
        const int chunks = (p.K + 31) / 32;
        const int ra = m0 + (g0 + grp) * 16 + g, rb = ra + 8;
        const bool oka = ra >= lo && ra < hi, okb = rb >= lo && rb < hi;
        const unsigned short* xa = static_cast<const unsigned short*>(p.rows) + ra * p.ld;
        const unsigned short* xb = xa + 8 * p.ld;
        const unsigned short* w = static_cast<const unsigned short*>(p.w) + c.slot * p.wa + g * p.wr;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        constexpr int U = NT <= 4 ? 4 : 1;
        for (int ch = chunks * part / parts; ch < chunks * (part + 1) / parts; ch += U) {
            uint4 a[U], b[U], v[U][NT];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = (ch + u) * 32 + t8;
                const bool in = k < p.K && ch + u < chunks * (part + 1) / parts;
                a[u] = oka && in ? load8(xa, k, p.K) : zero;
                b[u] = okb && in ? load8(xb, k, p.K) : zero;
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    v[u][n] = in && n * 8 + g < p.R
                                  ? *reinterpret_cast<const uint4*>(w + n * 8 * p.wr + k) : zero;
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    if (n < nt) {
                        mma16816<BF16>(acc[n], a[u].x, b[u].x, a[u].y, b[u].y, v[u][n].x, v[u][n].y);
                        mma16816<BF16>(acc[n], a[u].z, b[u].z, a[u].w, b[u].w, v[u][n].z, v[u][n].w);
                    }
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        float* r = red + (warp * 16 + g) * 8 * NT + n * 8 + (lane & 3) * 2;
        *reinterpret_cast<float2*>(r) = make_float2(acc[n][0], acc[n][1]);
        *reinterpret_cast<float2*>(r + 64 * NT) = make_float2(acc[n][2], acc[n][3]);
    }
    __syncthreads();
    const float s = p.scale[c.slot];
    for (int i = threadIdx.x; i < 64 * p.Rs; i += 256) {
        const int row = i / p.Rs, r = i - row * p.Rs, m = m0 + row;
        float v = 0.f;
        const bool in = m >= lo && m < hi && r < p.R;
        if (in) {
            const float* q = red + ((row / 16 - g0) * 16 + row % 16) * 8 * NT + r;
            for (int k = 0; k < parts; ++k) v += q[(long long)k * gp * 128 * NT];
            v *= s;
        }
        store_f(block, i, v, p.dtype);
        if (p.compact && m >= lo && m < hi) store_f(p.compact, (long long)m * p.Rs + r, v, p.dtype);
    }
}

// fp32: FMA products of 64 rows by 32 ranks, 32 deep; then each row's planes.
__global__ void __launch_bounds__(256) shrink32_kernel(const __grid_constant__ Shrink p) {
    extern __shared__ float out[];       // [64][R + 1]
    __shared__ float xs[64][33], ws[32][33];
    if (side_work(p)) return;
    const Piece c = find_piece(p);
    if (c.slot < 0) return;
    const int m0 = c.m0 + blockIdx.y * 64, lo = max(c.lo, m0), hi = min(c.hi, m0 + 64);
    __half* block = static_cast<__half*>(p.block) +
                    ((long long)blockIdx.x * 256 + blockIdx.y * 64) * p.Rs;
    if (lo >= hi) {
        for (int i = threadIdx.x; i < 64 * p.Rs; i += 256) {
            block[i] = __float2half_rn(0.f);
            block[i + p.plane] = __float2half_rn(0.f);
        }
        return;
    }
    const float* x = static_cast<const float*>(p.rows);
    const float* w = static_cast<const float*>(p.w) + c.slot * p.wa;
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    const int pitch = p.R + 1;
    const float s = p.scale[c.slot];
    for (int r0 = 0; r0 < p.R; r0 += 32) {
        float acc[4][2] = {};
        for (int k0 = 0; k0 < p.K; k0 += 32) {
            for (int i = threadIdx.x; i < 64 * 32; i += 256) {
                const int m = m0 + (i >> 5), k = k0 + (i & 31);
                xs[i >> 5][i & 31] = m >= lo && m < hi && k < p.K ? x[m * p.ld + k] : 0.f;
            }
            for (int i = threadIdx.x; i < 32 * 32; i += 256) {
                const int r = p.wk == 1 ? i >> 5 : i & 31, k = p.wk == 1 ? i & 31 : i >> 5;
                ws[r][k] = r0 + r < p.R && k0 + k < p.K
                               ? w[(r0 + r) * p.wr + (k0 + k) * p.wk] : 0.f;
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < 32; ++k) {
                const float b0 = ws[tx][k], b1 = ws[tx + 16][k];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float a = xs[ty + 16 * i][k];
                    acc[i][0] = fmaf(a, b0, acc[i][0]);
                    acc[i][1] = fmaf(a, b1, acc[i][1]);
                }
            }
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (r0 + tx + 16 * j < p.R) out[(ty + 16 * i) * pitch + r0 + tx + 16 * j] = s * acc[i][j];
    }
    __syncthreads();
    const int lane = threadIdx.x & 31;
    for (int row = threadIdx.x >> 5; row < 64; row += 8) {
        const int m = m0 + row;
        const bool in = m >= lo && m < hi;
        unsigned mx = 0;
        if (in)
            for (int r = lane; r < p.R; r += 32) mx = max(mx, finite_bits(out[row * pitch + r]));
        mx = __reduce_max_sync(0xffffffffu, mx);
        const float sc = pow2_scale(mx);
        if (in && lane == 0) p.rinv[m] = pow2_inv(sc);
        for (int r = lane; r < p.Rs; r += 32) {
            const float v = in && r < p.R ? out[row * pitch + r] : 0.f;
            __half2 h, l;
            split_half2(v * sc, 0.f, h, l);
            block[row * p.Rs + r] = __low2half(h);
            block[row * p.Rs + r + p.plane] = __low2half(l);
            if (in && p.compact) static_cast<float*>(p.compact)[(long long)m * p.Rs + r] = v;
        }
    }
}

// dst[a][r][o] = src[a][o][r], 16-bit, dst's rows `pitch` apart and zero-filled.
__global__ void __launch_bounds__(256) transpose_kernel(const unsigned short* src, int O, int R,
                                                        int pitch, unsigned short* dst) {
    __shared__ unsigned short tile[32][33];
    const long long a = blockIdx.z;
    const int o0 = blockIdx.x * 32, r0 = blockIdx.y * 32;
    for (int i = threadIdx.x; i < 1024; i += 256) {
        const int o = o0 + (i >> 5), r = r0 + (i & 31);
        tile[i >> 5][i & 31] = o < O && r < R ? src[(a * O + o) * R + r] : 0;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 1024; i += 256) {
        const int r = r0 + (i >> 5), o = o0 + (i & 31);
        if (r < R && o < pitch) dst[(a * R + r) * pitch + o] = tile[i & 31][i >> 5];
    }
}

// dA[a] = T^T x and dB[a] = (S^T dy)^T over the pieces of adapter a, in their order.
struct Grads {
    const int4* piece;
    int pieces, nad, R, Rs;
    const void* low[2];      // T, S [M][Rs]
    const void* rows[2];     // x, dy
    long long ld[2];
    int width[2];            // D, O
    int tiles0;              // 128-column tiles of the first
    void* out[2];
    float* part;             // split > 1: [split][adapter](R D | R O)
    int split;
    int dtype;
};
__global__ void __launch_bounds__(256) grads_kernel(const __grid_constant__ Grads p) {
    __shared__ float ts[32][36], xs[32][132];
    const int which = blockIdx.x >= p.tiles0;
    const int c0 = (blockIdx.x - (which ? p.tiles0 : 0)) * 128, W = p.width[which];
    const int chunks = (p.R + 31) / 32;
    const int a = blockIdx.y / chunks, r0 = (blockIdx.y - a * chunks) * 32;
    const int lane = threadIdx.x & 31;
    const int ty = threadIdx.x >> 5, tx = lane;      // 4 ranks, 4 columns a thread
    float acc[4][4] = {};
    const int first = (int)((long long)p.pieces * blockIdx.z / p.split);
    const int behind = (int)((long long)p.pieces * (blockIdx.z + 1) / p.split);
    for (int b = first; b < behind; b += 32) {
        unsigned mine = __ballot_sync(0xffffffffu, b + lane < behind && p.piece[b + lane].x == a);
        while (mine) {
            const int4 c = p.piece[b + __ffs(mine) - 1];
            mine &= mine - 1;
            for (int m0 = c.y; m0 < c.z; m0 += 32) {
                for (int i = threadIdx.x; i < 1024; i += 256) {
                    const int m = m0 + (i >> 5), r = r0 + (i & 31);
                    ts[i >> 5][i & 31] = m < c.z && r < p.R
                        ? load_f(p.low[which], (long long)m * p.Rs + r, p.dtype) : 0.f;
                }
                for (int i = threadIdx.x; i < 4096; i += 256) {
                    const int m = m0 + (i >> 7), k = c0 + (i & 127);
                    xs[i >> 7][i & 127] = m < c.z && k < W
                        ? load_f(p.rows[which], m * p.ld[which] + k, p.dtype) : 0.f;
                }
                __syncthreads();
#pragma unroll 8
                for (int k = 0; k < 32; ++k) {
                    const float4 t = *reinterpret_cast<const float4*>(&ts[k][ty * 4]);
                    const float4 x = *reinterpret_cast<const float4*>(&xs[k][tx * 4]);
                    const float tt[4] = {t.x, t.y, t.z, t.w}, xx[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(tt[i], xx[j], acc[i][j]);
                }
                __syncthreads();
            }
        }
    }
    const long long per = (long long)p.R * (p.width[0] + p.width[1]);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = r0 + ty * 4 + i, k = c0 + tx * 4 + j;
            if (r >= p.R || k >= W) continue;
            const long long e = which ? (long long)k * p.R + r : (long long)r * W + k;
            if (p.split > 1)
                p.part[((long long)blockIdx.z * p.nad + a) * per +
                       (which ? (long long)p.R * p.width[0] : 0) + e] = acc[i][j];
            else
                store_f(p.out[which], (long long)a * p.R * W + e, acc[i][j], p.dtype);
        }
}
__global__ void __launch_bounds__(256) grads_sum_kernel(const __grid_constant__ Grads p) {
    const long long n0 = (long long)p.R * p.width[0], per = n0 + (long long)p.R * p.width[1];
    const long long all = per * p.nad;
    for (long long i = blockIdx.x * 256LL + threadIdx.x; i < all; i += gridDim.x * 256LL) {
        float v = 0.f;
        for (int s = 0; s < p.split; ++s) v += p.part[s * all + i];
        const long long a = i / per, e = i - a * per;
        const int which = e >= n0;
        if (p.out[which])
            store_f(p.out[which], which ? a * (per - n0) + e - n0 : a * n0 + e, v, p.dtype);
    }
}

struct AdSizes {
    int dtype;
    long long M;
    int D, O, nad, R, nreq;
    int tiles, pieces, Rs;
    long long Dp, Op;
    bool split, on;
    AdSizes(int t, long long m, int d, int o, int n, int r, int q)
        : dtype(t), M(m), D(d), O(o), nad(n), R(r), nreq(q), tiles((int)((m + 255) / 256)),
          pieces(tiles + q), Rs((int)up(r, 8)), Dp(up(d, 8)), Op(up(o, 8)), split(t == ATOM_F32),
          on(n > 0 && q > 0) {}
    Choice product(bool bwd) const {
        return choose(M, bwd ? D : O, ((bwd ? O : D) + 63) / 64, 1, false, split, true);
    }
    int grad_split() const {
        const long long blocks = (long long)nad * ((R + 31) / 32) * ((D + 127) / 128 + (O + 127) / 128);
        const long long s = blocks ? 592 / blocks : 1;
        return (int)std::max(1LL, std::min({s, 16LL, (long long)pieces}));
    }
};

struct AdSpace {
    __half *rows, *x, *w, *ad, *ext, *block, *bt;
    float *rinv, *ext_rinv, *part, *gpart;
    void *S, *T;
    int4 *piece, *bad;
    int2* tile_req;
    unsigned* max;           // rows, w, adapters
    size_t bytes;
    AdSpace(void* ws, const AdSizes& z, bool bwd) {
        memset(this, 0, sizeof(*this));
        Cursor c(ws);
        const long long k = z.split ? 2 : 1, e = dtype_size(z.dtype);
        rows = c.take<__half>(k * z.M * (bwd ? z.Op : z.Dp));
        w = c.take<__half>(k * z.O * z.Dp);
        part = c.take<float>(z.product(bwd).part);
        if (z.split) {
            max = c.take<unsigned>(4);
            rinv = c.take<float>(z.M);
        }
        if (z.on) {
            piece = c.take<int4>(z.pieces);
            bad = c.take<int4>(z.nad);
            tile_req = c.take<int2>(z.tiles);
            // the low-rank product's adapters, and those of the product beside the projection
            if (!z.split) ad = c.take<__half>((long long)z.nad * z.R * (bwd ? z.Op : z.Dp));
            ext = c.take<__half>(k * z.nad * (bwd ? z.R * z.Dp : (long long)z.O * z.Rs));
            block = c.take<__half>(k * z.pieces * 256 * z.Rs);
            if (z.split) ext_rinv = c.take<float>(z.M);
            if (bwd) {
                if (!z.split) {
                    x = c.take<__half>(z.M * z.Dp);
                    bt = c.take<__half>((long long)z.nad * z.R * z.Dp);
                }
                T = c.take<char>(z.M * z.Rs * e);
                S = c.take<char>(z.M * z.Rs * e);
                const long long s = z.grad_split();
                gpart = c.take<float>(s > 1 ? s * z.nad * z.R * (z.D + z.O) : 0);
            }
        }
        bytes = c.used;
    }
};

template <bool BF16>
int shrink16(const Shrink& p, dim3 grid, cudaStream_t st) {
    const int nt = (p.R + 7) / 8;
#define ATOM_SHRINK(N)                                                                       \
    if (nt <= N) {                                                                           \
        const int smem = 8 * 16 * 8 * N * 4;                                                 \
        if (smem > 48 * 1024)                                                                \
            cudaFuncSetAttribute(shrink16_kernel<BF16, N>,                                   \
                                 cudaFuncAttributeMaxDynamicSharedMemorySize, smem);         \
        shrink16_kernel<BF16, N><<<grid, 256, smem, st>>>(p);                                \
        return check_launch("adapters: low-rank rows");                                      \
    }
    ATOM_SHRINK(1)
    ATOM_SHRINK(2)
    ATOM_SHRINK(4)
    ATOM_SHRINK(8)
    ATOM_SHRINK(16)
#undef ATOM_SHRINK
    return ATOM_ERR_UNSUPPORTED;
}
int shrink(const Shrink& p, cudaStream_t st) {
    const dim3 grid(p.pieces + p.q.nad + 1, 4);
    if (p.dtype == ATOM_BF16) return shrink16<true>(p, grid, st);
    if (p.dtype == ATOM_F16) return shrink16<false>(p, grid, st);
    shrink32_kernel<<<grid, 256, 64 * (p.R + 1) * 4, st>>>(p);
    return check_launch("adapters: low-rank rows");
}

// One direction: out [M, N] = rows [M, K] W' + (low-rank rows) (adapters), where forward has
// rows = x, W' = w^T, and backward rows = dy, W' = w.
struct Ad {
    AdSizes z;
    AdSpace sp;
    cudaStream_t st;
    Requests q;
    const float* scale;
    const void *w, *a, *b;

    int run(const void* rows, long long ld, bool bwd, void* out, long long ldo, void* compact,
            bool low_only) {
        const int K = bwd ? z.O : z.D, N = bwd ? z.D : z.O, k = z.split ? 2 : 1;
        const long long Kp = bwd ? z.Op : z.Dp;
        PrepList l;
        const void* xr = rows;
        long long xld = ld;
        const void* wp = w;
        long long wld = z.D;
        const void* first = bwd ? b : a;         // [nad][R][K] forward, [nad][K][R] backward
        const void* second = bwd ? a : b;        // the product beside the projection
        const long long srows = bwd ? (long long)z.nad * z.R : (long long)z.nad * z.O;
        const int scols = bwd ? z.D : z.R;
        const long long sp_ld = bwd ? z.Dp : z.Rs;
        const void* sec = second;
        long long sec_ld = scols;
        const bool both = z.on && !low_only;
        if (z.split && low_only) {
        } else if (z.split) {
            cudaMemsetAsync(sp.max, 0, 16, st);
            if (z.on) cudaMemsetAsync(sp.ext_rinv, 0, z.M * sizeof(float), st);
            l.add({w, z.O, z.D, z.D, nullptr, 0, 0, nullptr, sp.max + 1, kMax});
            if (z.on) l.add({second, srows, scols, scols, nullptr, 0, 0, nullptr, sp.max + 2, kMax});
            l.add({rows, z.M, K, ld, sp.rows, Kp, z.M * Kp, sp.rinv, nullptr, kRowSplit});
            if (int s = prepare(l, st)) return s;
            l.n = 0;
            l.add({w, z.O, z.D, z.D, sp.w, z.Dp, z.O * z.Dp, nullptr, sp.max + 1, kTensorSplit});
            if (z.on)
                l.add({second, srows, scols, scols, sp.ext, sp_ld, srows * sp_ld, nullptr,
                       sp.max + 2, kTensorSplit});
        } else {
            if (!tma_ready(rows, ld)) {
                l.add({rows, z.M, K, ld, sp.rows, Kp, 0, nullptr, nullptr, kPack});
                xr = sp.rows, xld = Kp;
            }
            if (!low_only && !tma_ready(w, z.D)) {
                l.add({w, z.O, z.D, z.D, sp.w, z.Dp, 0, nullptr, nullptr, kPack});
                wp = sp.w, wld = z.Dp;
            }
            if (both && !tma_ready(second, scols)) {
                l.add({second, srows, scols, scols, sp.ext, sp_ld, 0, nullptr, nullptr, kPack});
                sec = sp.ext, sec_ld = sp_ld;
            }
            if (z.on && !bwd && !tma_ready(first, z.D)) {
                l.add({first, (long long)z.nad * z.R, z.D, z.D, sp.ad, z.Dp, 0, nullptr, nullptr,
                       kPack});
                first = sp.ad;
            }
        }
        if (int s = prepare(l, st)) return s;
        if (z.on) {
            Shrink h;
            memset(&h, 0, sizeof(h));
            h.q = q;
            h.pieces = z.pieces;
            h.rows = z.split ? rows : xr;
            h.ld = z.split ? ld : xld;
            h.K = K;
            h.w = first;
            if (bwd && z.split) {
                h.wa = (long long)z.O * z.R, h.wr = 1, h.wk = z.R;
            } else if (bwd) {
                transpose_kernel<<<dim3(ceil_div(z.Op, 32), ceil_div(z.R, 32), z.nad), 256, 0, st>>>(
                    static_cast<const unsigned short*>(b), z.O, z.R, (int)z.Op,
                    reinterpret_cast<unsigned short*>(sp.ad));
                if (int s = check_launch("adapters: transpose")) return s;
                h.w = sp.ad;
                h.wa = z.R * z.Op, h.wr = z.Op, h.wk = 1;
            } else {
                h.wr = z.split || first != sp.ad ? z.D : z.Dp;
                h.wa = z.R * h.wr, h.wk = 1;
            }
            h.R = z.R, h.Rs = z.Rs;
            h.scale = scale;
            h.other = second;
            h.other_n = low_only ? 0 : (long long)z.R * (bwd ? z.D : z.O);
            h.piece = sp.piece;
            h.tile_req = sp.tile_req;
            h.tiles = z.tiles;
            h.bad = sp.bad;
            h.block = sp.block;
            h.plane = (long long)z.pieces * 256 * z.Rs;
            h.compact = compact;
            h.rinv = sp.ext_rinv;
            h.dtype = z.dtype;
            if (int s = shrink(h, st)) return s;
        }
        if (low_only) return ATOM_OK;
        const Choice c = z.product(bwd);
        Maps maps;
        const long long planes[3] = {z.M * Kp, z.O * z.Dp, srows * sp_ld};
        const long long bplane = (long long)z.pieces * 256 * z.Rs;
        for (int pl = 0; pl < k; ++pl) {
            auto at = [&](const void* base, long long plane) {
                return static_cast<const __half*>(base) + pl * plane;
            };
            const void* r = z.split ? sp.rows : xr;
            if (int s = make_map(&maps.m[pl], at(r, planes[0]), K, z.M, z.split ? Kp : xld, 128))
                return s;
            if (int s = make_map(&maps.m[k + pl], at(z.split ? sp.w : wp, planes[1]), z.D, z.O,
                                 z.split ? z.Dp : wld, bwd ? 64 : c.bn / 2))
                return s;
            if (!z.on) continue;
            if (int s = make_map(&maps.m[2 * k + pl], at(sp.block, bplane), z.R,
                                 (long long)z.pieces * 256, z.Rs, 128))
                return s;
            const long long sl = z.split ? sp_ld : sec_ld;
            if (int s = make_map(&maps.m[3 * k + pl], at(z.split ? sp.ext : sec, planes[2]), scols,
                                 bwd ? z.R : z.O, sl, bwd ? 64 : c.bn / 2, z.nad,
                                 (bwd ? z.R : z.O) * sl))
                return s;
        }
        Args p;
        memset(&p, 0, sizeof(p));
        p.M = z.M, p.N = N, p.groups = 1, p.nphase = 1;
        p.ph[0] = {0, k, k, (K + 63) / 64, 0, bwd ? 1 : 0, c.bn, c.bn / 2};
        p.bf16 = z.dtype == ATOM_BF16;
        p.dtype = z.dtype;
        p.C[0] = out;
        p.ldc = ldo;
        p.used = z.on ? (1u << 4 * k) - 1 : (1u << 2 * k) - 1;
        p.part = sp.part;
        p.rinv = sp.rinv;
        p.bmax = sp.max + 1;
        if (z.on) {
            p.ext = (z.R + 63) / 64;
            p.ext_a = 2 * k, p.ext_b = 3 * k, p.ext_bmn = bwd ? 1 : 0;
            p.tile_req = sp.tile_req;
            p.piece = sp.piece;
            p.bad = sp.bad;
            p.R = z.R;
            p.ext_rinv = sp.ext_rinv;
            p.ext_bmax = sp.max + 2;
        }
        return launch(kStore, c, z.split, maps, p, st);
    }
};

int check_ad(int dtype, int64_t M, int D, int O, int nad, int R, int nreq) {
    ATOM_REQUIRE(dtype >= ATOM_F32 && dtype <= ATOM_F16, "adapted_linear: unknown type %d", dtype);
    ATOM_REQUIRE(M >= 0 && M < (1LL << 31) - 256 && D > 0 && O > 0 && nad >= 0 && nreq >= 0,
                 "adapted_linear: bad sizes");
    ATOM_REQUIRE(D < (1 << 24) && O < (1 << 24), "adapted_linear: widths above 2^24");
    ATOM_REQUIRE(nad < (1 << 14) && nreq < (1 << 22) && (M + 255) / 256 + nreq < (1 << 23),
                 "adapted_linear: sizes above 2^14 adapters, 2^22 requests or 2^23 pieces of 256 "
                 "rows");
    ATOM_REQUIRE(R >= 1 && R <= 128, "adapted_linear: the rank must be 1..128");
    return ATOM_OK;
}

}  // namespace
}  // namespace atom

using namespace atom;

extern "C" int atom_adapted_linear_bytes(int dtype, int64_t M, int D, int O, int n_adapters,
                                         int R, int nreq, size_t* bytes_host) {
    if (int s = check_ad(dtype, M, D, O, n_adapters, R, nreq)) return s;
    ATOM_REQUIRE(bytes_host, "adapted_linear: bytes_host is NULL");
    const AdSizes z(dtype, M, D, O, n_adapters, R, nreq);
    bytes_host[0] = AdSpace(nullptr, z, false).bytes;
    bytes_host[1] = AdSpace(nullptr, z, true).bytes;
    bytes_host[2] = (size_t)M * z.Rs * dtype_size(dtype);
    return ATOM_OK;
}

extern "C" int atom_adapted_linear_fwd(int dtype, const void* x, int64_t ldx, int64_t M, int D,
                                       int O, const void* w, const void* a, const void* b,
                                       const float* scale, int n_adapters, int R,
                                       const int* req_ptr, const int* req_adapter, int nreq,
                                       void* y, int64_t ldy, void* kept, void* ws,
                                       size_t ws_bytes, void* stream) {
    if (int s = check_ad(dtype, M, D, O, n_adapters, R, nreq)) return s;
    if (M == 0) return ATOM_OK;
    ATOM_REQUIRE(x && w && y && ldx >= D && ldy >= O, "adapted_linear: bad operand");
    const AdSizes z(dtype, M, D, O, n_adapters, R, nreq);
    ATOM_REQUIRE(!z.on || (a && b && scale && req_ptr && req_adapter),
                 "adapted_linear: bad operand");
    Ad f{z, AdSpace(ws, z, false), (cudaStream_t)stream,
         {req_ptr, req_adapter, nreq, n_adapters, (int)M}, scale, w, a, b};
    ATOM_REQUIRE(ws && ws_bytes >= f.sp.bytes, "adapted_linear: the workspace needs %zu bytes",
                 f.sp.bytes);
    return f.run(x, ldx, false, y, ldy, kept, false);
}

extern "C" int atom_adapted_linear_bwd(int dtype, const void* x, int64_t ldx, int64_t M, int D,
                                       int O, const void* w, const void* a, const void* b,
                                       const float* scale, int n_adapters, int R,
                                       const int* req_ptr, const int* req_adapter, int nreq,
                                       const void* dy, int64_t lddy, const void* kept, void* dx,
                                       int64_t lddx, void* da, void* db, void* ws,
                                       size_t ws_bytes, void* stream) {
    if (int s = check_ad(dtype, M, D, O, n_adapters, R, nreq)) return s;
    cudaStream_t st = (cudaStream_t)stream;
    const size_t e = dtype_size(dtype);
    const AdSizes z(dtype, M, D, O, n_adapters, R, nreq);
    if (M == 0 || !z.on) {
        if (da) cudaMemsetAsync(da, 0, e * n_adapters * R * D, st);
        if (db) cudaMemsetAsync(db, 0, e * n_adapters * R * O, st);
        if (int s = check_launch("adapters", 0)) return s;
    }
    if (M == 0) return ATOM_OK;
    ATOM_REQUIRE(x && w && dy && ldx >= D && lddy >= O && (!dx || lddx >= D),
                 "adapted_linear: bad operand");
    ATOM_REQUIRE(!z.on || (a && b && scale && req_ptr && req_adapter),
                 "adapted_linear: bad operand");
    Ad f{z, AdSpace(ws, z, true), st, {req_ptr, req_adapter, nreq, n_adapters, (int)M}, scale, w,
         a, b};
    ATOM_REQUIRE(ws && ws_bytes >= f.sp.bytes, "adapted_linear: the workspace needs %zu bytes",
                 f.sp.bytes);
    const bool grads = z.on && (da || db);
    if (grads && db && !kept) {      // S again
        AdSpace fs = f.sp;
        fs.rows = f.sp.x;            // x's copy, where it needs one
        fs.ad = f.sp.bt;
        Ad g = f;
        g.sp = fs;
        if (int s = g.run(x, ldx, false, nullptr, 0, f.sp.S, true)) return s;
    }
    if (int s = f.run(dy, lddy, true, dx, lddx, grads ? f.sp.T : nullptr, !dx)) return s;
    if (!grads) return ATOM_OK;
    Grads p;
    memset(&p, 0, sizeof(p));
    p.piece = f.sp.piece;
    p.pieces = z.pieces, p.nad = n_adapters, p.R = R, p.Rs = z.Rs;
    p.low[0] = f.sp.T, p.low[1] = kept ? kept : f.sp.S;
    p.rows[0] = x, p.rows[1] = dy;
    p.ld[0] = ldx, p.ld[1] = lddy;
    p.width[0] = da ? D : 0, p.width[1] = db ? O : 0;
    p.tiles0 = ceil_div(p.width[0], 128);
    p.out[0] = da, p.out[1] = db;
    p.part = f.sp.gpart;
    p.split = z.grad_split();
    p.dtype = dtype;
    const int tiles = p.tiles0 + ceil_div(p.width[1], 128);
    const long long ny = (long long)n_adapters * ((R + 31) / 32);
    grads_kernel<<<dim3(tiles, (unsigned)ny, p.split), 256, 0, st>>>(p);
    ATOM_CHECK_LAUNCH("adapters: gradients");
    if (p.split > 1) {
        grads_sum_kernel<<<592, 256, 0, st>>>(p);
        ATOM_CHECK_LAUNCH("adapters: gradient sums");
    }
    return ATOM_OK;
}
