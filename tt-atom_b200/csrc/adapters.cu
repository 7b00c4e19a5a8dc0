// Low-rank adapters of many requests beside a shared projection, and their backward pass.
//
//   y = x W^T + S B^T,  S = s (x A^T) row by row with the row's own A, B and s
//
// The requests' rows are cut at every 256th row into pieces: piece t + r holds the rows of request
// r in row tile t (t + r grows along the requests, so it names a piece without a table). The
// shrink pass writes S of each piece as a block of 256 rows, zeros where the rows are not the
// request's, and the shared projection's product (pair_product.cu) then takes each piece of its
// row tile as more of K, S's block times the request's B, in slices of 16 ranks of which four make
// a stage: the adapters cost their own multiplications and no pass over y. The backward pass is the same with T = s (dy B), W and A in
// the place of S, W^T and B, and dA = T^T x, dB = dy^T S summed by pieces in their order.
//
// Zeros in a block keep other requests' rows as they are only where B is finite; an adapter that
// is not is found in the shrink pass, left out, and its own rows are set to NaN.
#include <algorithm>

#include "few_rows.cuh"
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

struct Shrink {
    Requests q;
    int pieces;              // row tiles + requests
    int rb;                  // rows of a piece that a block has (32 .. 256, grid.y = 256 / rb)
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
        for (int t = blockIdx.y * 8 + warp; t < p.tiles; t += 8 * gridDim.y) {
            const int first = last_le(p.q.n, t * 256, [&](int r) { return row_of(p.q, r); });
            const int last = last_le(p.q.n, t * 256 + 255, [&](int r) { return row_of(p.q, r); });
            // a request that begins before the tile reaches into it at most as the last such one
            if (lane == 0) p.tile_req[t] = make_int2(max(first, 0), last + 1);
        }
        return true;
    }
    const int parts = min(4, gridDim.y);
    if (blockIdx.y >= parts) return true;
    int found = 0;
    const long long lo = p.other_n * blockIdx.y / parts, hi = p.other_n * (blockIdx.y + 1) / parts;
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
    for (int i = blockIdx.y; i < 4 && threadIdx.x == 0; i += parts)
        reinterpret_cast<int*>(p.bad + b)[i] = i == blockIdx.y ? found : 0;
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

// 16-bit: a block of 8 warps has 32 rows of a piece, 16 a warp, and the warps split K (all eight
// of them for 16 rows or fewer). Rows and adapters go from memory into the fragments of m16n8k16
// directly: the product does not mind in which order K runs, so each lane reads 8 consecutive
// elements of its row, half for one instruction and half for the next. Bound by reading x: an
// adapter's rows come from L2 and L1, and small blocks, three on an SM, keep enough in flight
// (with 64 rows and one block an SM 8192 x 2048 rows of rank 32 took 30 us).
template <bool BF16, int NT>
__global__ void __launch_bounds__(256, NT <= 4 ? 3 : 1)
    shrink16_kernel(const __grid_constant__ Shrink p) {
    extern __shared__ float red[];       // [8 warps][16][8 NT]
    let_next_start();
    wait_before();
    if (side_work(p)) return;
    const Piece c = find_piece(p);
    if (c.slot < 0) return;
    for (int m0 = c.m0 + blockIdx.y * p.rb, behind = m0 + p.rb; m0 < behind; m0 += 32) {
    const int lo = max(c.lo, m0), hi = min(c.hi, m0 + 32);
    unsigned short* block = static_cast<unsigned short*>(p.block) +
                            ((long long)blockIdx.x * 256 + m0 - c.m0) * p.Rs;
    if (lo >= hi) {                      // Rs is a multiple of 8
        for (int i = threadIdx.x; i < 4 * p.Rs; i += 256)
            reinterpret_cast<uint4*>(block)[i] = make_uint4(0, 0, 0, 0);
        continue;
    }
    const int g0 = (lo - m0) / 16, gp = (hi - 1 - m0) / 16 - g0 + 1, parts = 8 / gp;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t8 = (lane & 3) * 8;
    const int grp = warp % gp, part = warp / gp;
    const int nt = (p.R + 7) / 8;
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
    {
        const int chunks = (p.K + 31) / 32;
        const int ra = m0 + (g0 + grp) * 16 + g, rb = ra + 8;
        const bool oka = ra >= lo && ra < hi, okb = rb >= lo && rb < hi;
        const unsigned short* xa = static_cast<const unsigned short*>(p.rows) + ra * p.ld;
        const unsigned short* xb = xa + 8 * p.ld;
        const unsigned short* w = static_cast<const unsigned short*>(p.w) + c.slot * p.wa + g * p.wr;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        constexpr int U = NT <= 2 ? 3 : NT <= 4 ? 2 : 1;
        const int end = chunks * (part + 1) / parts;
        for (int ch = chunks * part / parts; ch < end; ch += U) {
            uint4 a[U], b[U], v[U][NT];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = (ch + u) * 32 + t8;
                const bool in = k < p.K && ch + u < end;
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
    for (int i = threadIdx.x; i < 32 * p.Rs; i += 256) {
        const int row = i / p.Rs, r = i - row * p.Rs, m = m0 + row;
        float v = 0.f;
        const bool in = m >= lo && m < hi;
        if (in && r < p.R) {
            const float* q = red + ((row / 16 - g0) * 16 + row % 16) * 8 * NT + r;
            for (int k = 0; k < parts; ++k) v += q[k * gp * 128 * NT];
            v *= s;
        }
        store_f(block, i, v, p.dtype);
        if (p.compact && in) store_f(p.compact, (long long)m * p.Rs + r, v, p.dtype);
    }
    __syncthreads();                     // red is free for the next 32 rows
    }
}

// fp32: a warp has 8 rows by 4 ranks, its lanes split K, and the 32 sums are added over the lanes
// by halves; then each row's planes.
__global__ void __launch_bounds__(256, 2) shrink32_kernel(const __grid_constant__ Shrink p) {
    extern __shared__ float out[];       // [32][R + 1]
    let_next_start();
    wait_before();
    if (side_work(p)) return;
    const Piece c = find_piece(p);
    if (c.slot < 0) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pitch = p.R + 1;
    const float s = p.scale[c.slot];
    const bool xvec = p.K % 4 == 0 && p.ld % 4 == 0 && aligned16(p.rows);
    const bool wvec = p.K % 4 == 0 && p.wk == 1 && aligned16(p.w);
    const bool wrow = p.wr == 1 && p.R % 4 == 0 && aligned16(p.w);
    // four consecutive elements a lane, whatever the strides: the sums' order stays the same
    auto four = [&](const float* q, long long step, int k, bool in, bool vec) {
        if (!in) return make_float4(0.f, 0.f, 0.f, 0.f);
        if (vec) return *reinterpret_cast<const float4*>(q + k);
        return make_float4(q[k * step], k + 1 < p.K ? q[(k + 1) * step] : 0.f,
                           k + 2 < p.K ? q[(k + 2) * step] : 0.f,
                           k + 3 < p.K ? q[(k + 3) * step] : 0.f);
    };
    for (int m0 = c.m0 + blockIdx.y * p.rb, behind = m0 + p.rb; m0 < behind; m0 += 32) {
        const int lo = max(c.lo, m0), hi = min(c.hi, m0 + 32);
        __half* block = static_cast<__half*>(p.block) +
                        ((long long)blockIdx.x * 256 + m0 - c.m0) * p.Rs;
        if (lo >= hi) {
            for (int i = threadIdx.x; i < 4 * p.Rs; i += 256) {
                reinterpret_cast<uint4*>(block)[i] = make_uint4(0, 0, 0, 0);
                reinterpret_cast<uint4*>(block + p.plane)[i] = make_uint4(0, 0, 0, 0);
            }
            continue;
        }
        const int groups = (hi - lo + 7) / 8, ranks = (p.R + 3) / 4;
        for (int item = warp; item < groups * ranks; item += 8) {
            const int row0 = lo + item / ranks * 8, r0 = item % ranks * 4;
            const float* x = static_cast<const float*>(p.rows) + row0 * p.ld;
            const float* w = static_cast<const float*>(p.w) + c.slot * p.wa + r0 * p.wr;
            const int nr = min(8, hi - row0), nk = min(4, p.R - r0);
            float acc[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) acc[i] = 0.f;
            for (int k = lane * 4; k < p.K; k += 128) {
                float4 a[8], d[4];
#pragma unroll
                for (int i = 0; i < 8; ++i) a[i] = four(x + i * p.ld, 1, k, i < nr, xvec);
                if (wrow && k + 3 < p.K) {       // the ranks of a K element lie side by side
                    float4 t[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        t[e] = *reinterpret_cast<const float4*>(w + (k + e) * p.wk);
                    d[0] = make_float4(t[0].x, t[1].x, t[2].x, t[3].x);
                    d[1] = make_float4(t[0].y, t[1].y, t[2].y, t[3].y);
                    d[2] = make_float4(t[0].z, t[1].z, t[2].z, t[3].z);
                    d[3] = make_float4(t[0].w, t[1].w, t[2].w, t[3].w);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) d[j] = four(w + j * p.wr, p.wk, k, j < nk, wvec);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        acc[4 * i + j] = fmaf(a[i].x, d[j].x, fmaf(a[i].y, d[j].y,
                                         fmaf(a[i].z, d[j].z, fmaf(a[i].w, d[j].w, acc[4 * i + j]))));
            }
            sum_halves<32>(acc, lane);
            const int i = lane >> 2, j = lane & 3;
            if (i < nr && j < nk) out[(row0 - m0 + i) * pitch + r0 + j] = s * acc[0];
        }
        __syncthreads();
        for (int row = warp; row < 32; row += 8) {
            const int m = m0 + row;
            const bool in = m >= lo && m < hi;
            unsigned mx = 0;
            if (in)
                for (int r = lane; r < p.R; r += 32)
                    mx = max(mx, finite_bits(out[row * pitch + r]));
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
        __syncthreads();                 // out is free for the next 32 rows
    }
}

// dst[a][r][o] = src[a][o][r], 16-bit, dst's rows `pitch` apart and zero-filled.
__global__ void __launch_bounds__(256) transpose_kernel(const unsigned short* src, int O, int R,
                                                        int pitch, unsigned short* dst) {
    let_next_start();
    wait_before();
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

// dA[a] = T^T x and dB[a] = (S^T dy)^T over the pieces of adapter a, in their order: blocks have
// all ranks by 128 columns of x or dy, and the pieces are shared out over blocks (`split`) whose
// sums are added in order by a second pass. Bound by reading x and dy once.
struct Grads {
    const int4* piece;
    int pieces, nad, R, Rs;
    const void* low[2];      // T, S [M][Rs]
    const void* rows[2];     // x, dy
    long long ld[2];
    int width[2];            // D, O
    int tiles0;              // 128-column tiles of the first
    void* out[2];
    float* part;             // split > 1: [split][adapter][R][D + O]
    int split;
    int dtype;
};
// Walks an adapter's rows in a block's share of the pieces, `step` at a time (whole warps).
struct Rows {
    const int4* piece;
    int a, b, behind, step;
    unsigned mine = 0;
    int m = 0, hi = 0;
    __device__ __forceinline__ Rows(const Grads& p, int adapter, int rows)
        : piece(p.piece), a(adapter), step(rows) {
        b = (int)((long long)p.pieces * blockIdx.z / p.split) - 32;
        behind = (int)((long long)p.pieces * (blockIdx.z + 1) / p.split);
    }
    // the next rows m .. min(m + step, hi) - 1; false when there are none
    __device__ __forceinline__ bool next() {
        m += step;
        if (m < hi) return true;
        while (mine == 0) {
            b += 32;
            if (b >= behind) {
                b = behind;
                hi = 0;
                return false;
            }
            const int i = b + (threadIdx.x & 31);
            mine = __ballot_sync(0xffffffffu, i < behind && piece[i].x == a);
        }
        const int4 c = piece[b + __ffs(mine) - 1];
        mine &= mine - 1;
        m = c.y;
        hi = c.z;
        return true;
    }
};
__device__ __forceinline__ void put_grad(const Grads& p, int which, int a, int r, int k, float v) {
    const int W = p.width[which];
    if (r >= p.R || k >= W) return;
    if (p.split > 1)
        p.part[(((long long)blockIdx.z * p.nad + a) * p.R + r) * (p.width[0] + p.width[1]) +
               (which ? p.width[0] : 0) + k] = v;
    else
        store_f(p.out[which], (long long)a * p.R * W + (which ? (long long)k * p.R + r
                                                             : (long long)r * W + k), v, p.dtype);
}

// 16-bit: 32 rows of both operands a stage, four stages by cp.async, both read transposed into
// the fragments of m16n8k16. Each of 8 warps has 16 columns and all ranks.
template <bool BF16, int MT>
__global__ void __launch_bounds__(256) grads16_kernel(const __grid_constant__ Grads p) {
    constexpr int kX = 32 * 272, kT = 32 * (32 * MT + 16), kStages = 4;
    extern __shared__ __align__(16) uint8_t smem[];
    let_next_start();
    wait_before();
    const int which = blockIdx.x >= p.tiles0;
    const int c0 = (blockIdx.x - (which ? p.tiles0 : 0)) * 128, W = p.width[which];
    const unsigned short* rows = static_cast<const unsigned short*>(p.rows[which]);
    const unsigned short* low = static_cast<const unsigned short*>(p.low[which]);
    const long long ld = p.ld[which];
    const int a = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
    Rows it(p, a, 32);
    int loaded = 0;
    bool more = true;
    auto load = [&]() {
        if (more && (more = it.next())) {
            const uint32_t x = base + (loaded % kStages) * (kX + kT), t = x + kX;
            const int n = min(32, it.hi - it.m);
            for (int i = threadIdx.x; i < 32 * 16; i += 256) {
                const int r = i >> 4, c = (i & 15) * 8;
                // bytes past the row's or the matrix's end are zeros
                const int bytes = r < n ? max(0, min(16, 2 * (W - c0 - c))) : 0;
                const void* src = bytes ? rows + (it.m + r) * ld + c0 + c : rows;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(x + r * 272 + c * 2),
                             "l"(src), "r"(bytes) : "memory");
            }
            for (int i = threadIdx.x; i < 32 * 2 * MT; i += 256) {
                const int r = i / (2 * MT), c = (i % (2 * MT)) * 8;
                const int bytes = r < n && c < p.Rs ? 16 : 0;
                const void* src = bytes ? low + (long long)(it.m + r) * p.Rs + c : low;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                                 t + r * (32 * MT + 16) + c * 2), "l"(src), "r"(bytes) : "memory");
            }
            ++loaded;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    float acc[MT][2][4] = {};
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) load();
    for (int done = 0; done < loaded; ++done) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        __syncthreads();
        const uint32_t x = base + (done % kStages) * (kX + kT), t = x + kX;
#pragma unroll
        for (int k = 0; k < 32; k += 16) {
            uint32_t b[4];
            asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                         : "=r"(b[0]), "=r"(b[1]), "=r"(b[2]), "=r"(b[3])
                         : "r"(x + (k + (lane & 7) + ((lane >> 3) & 1) * 8) * 272 +
                               (warp * 16 + (lane >> 4) * 8) * 2) : "memory");
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                uint32_t f[4];
                asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                             : "=r"(f[0]), "=r"(f[1]), "=r"(f[2]), "=r"(f[3])
                             : "r"(t + (k + (lane & 7) + (lane >> 4) * 8) * (32 * MT + 16) +
                                   (i * 16 + ((lane >> 3) & 1) * 8) * 2) : "memory");
                mma16816<BF16>(acc[i][0], f[0], f[1], f[2], f[3], b[0], b[1]);
                mma16816<BF16>(acc[i][1], f[0], f[1], f[2], f[3], b[2], b[3]);
            }
        }
        load();
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    const int k0 = c0 + warp * 16 + (lane & 3) * 2;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                put_grad(p, which, a, i * 16 + (lane >> 2) + (e >> 1) * 8, k0 + j * 8 + (e & 1),
                         acc[i][j][e]);
}

// fp32: 32 ranks by 128 columns a block, 4 x 4 a thread, 32 rows at a time.
__global__ void __launch_bounds__(256) grads32_kernel(const __grid_constant__ Grads p) {
    __shared__ __align__(16) float ts[32][36], xs[32][132];
    let_next_start();
    wait_before();
    const int which = blockIdx.x >= p.tiles0;
    const int c0 = (blockIdx.x - (which ? p.tiles0 : 0)) * 128, W = p.width[which];
    const int chunks = (p.R + 31) / 32;
    const int a = blockIdx.y / chunks, r0 = (blockIdx.y - a * chunks) * 32;
    const float* rows = static_cast<const float*>(p.rows[which]) + c0;
    const float* low = static_cast<const float*>(p.low[which]) + r0;
    const long long ld = p.ld[which];
    const int lane = threadIdx.x & 31, ty = threadIdx.x >> 5;
    float acc[4][4] = {};
    for (Rows it(p, a, 32); it.next();) {
        const int n = min(32, it.hi - it.m);
        float x[16], t[4];
#pragma unroll
        for (int i = 0; i < 16; ++i) {       // warp: rows ty, ty + 8, ..; lanes: columns
            const int r = ty + 8 * (i >> 2), k = lane + 32 * (i & 3);
            x[i] = r < n && c0 + k < W ? rows[(it.m + r) * ld + k] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = ty + 8 * i;
            t[i] = r < n && r0 + lane < p.R ? low[(long long)(it.m + r) * p.Rs + lane] : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 16; ++i) xs[ty + 8 * (i >> 2)][lane + 32 * (i & 3)] = x[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) ts[ty + 8 * i][lane] = t[i];
        __syncthreads();
        for (int k = 0; k < n; ++k) {
            const float4 u = *reinterpret_cast<const float4*>(&ts[k][ty * 4]);
            const float4 v = *reinterpret_cast<const float4*>(&xs[k][lane * 4]);
            const float tt[4] = {u.x, u.y, u.z, u.w}, xx[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(tt[i], xx[j], acc[i][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            put_grad(p, which, a, r0 + ty * 4 + i, c0 + lane * 4 + j, acc[i][j]);
}
__global__ void __launch_bounds__(256) grads_sum_kernel(const __grid_constant__ Grads p) {
    let_next_start();
    wait_before();
    const int W = p.width[0] + p.width[1];
    const long long per = (long long)p.R * W, all = per * p.nad;
    for (long long i = blockIdx.x * 256LL + threadIdx.x; i < all; i += gridDim.x * 256LL) {
        float v = 0.f;
        for (int s = 0; s < p.split; ++s) v += p.part[s * all + i];
        const long long a = i / per, e = i - a * per;
        const int r = (int)(e / W), k = (int)(e - (long long)r * W);
        if (k < p.width[0])
            store_f(p.out[0], (a * p.R + r) * p.width[0] + k, v, p.dtype);
        else
            store_f(p.out[1], (a * p.width[1] + k - p.width[0]) * p.R + r, v, p.dtype);
    }
}
template <bool BF16>
int grads16(const Grads& p, dim3 grid, Chain& st) {
#define ATOM_GRADS(N)                                                                             \
    if (p.R <= 16 * N) {                                                                          \
        constexpr int smem = 4 * (32 * 272 + 32 * (32 * N + 16));                                 \
        if (smem > 48 * 1024)                                                                     \
            cudaFuncSetAttribute(grads16_kernel<BF16, N>,                                         \
                                 cudaFuncAttributeMaxDynamicSharedMemorySize, smem);              \
        return st.launch("adapters: gradients", grads16_kernel<BF16, N>, grid, 256, smem, p);     \
    }
    ATOM_GRADS(1)
    ATOM_GRADS(2)
    ATOM_GRADS(4)
    ATOM_GRADS(8)
#undef ATOM_GRADS
    return ATOM_ERR_UNSUPPORTED;
}

struct AdSizes {
    int dtype;
    long long M;
    int D, O, nad, R, nreq;
    int tiles, pieces, Rs;
    long long Dp, Op;
    bool split, on;
    Choice product;
    AdSizes(int t, long long m, int d, int o, int n, int r, int q, bool bwd)
        : dtype(t), M(m), D(d), O(o), nad(n), R(r), nreq(q), tiles((int)((m + 255) / 256)),
          pieces(tiles + q), Rs((int)up(r, 8)), Dp(up(d, 8)), Op(up(o, 8)), split(t == ATOM_F32),
          on(n > 0 && q > 0),
          product(choose(m, bwd ? d : o, ((bwd ? o : d) + 63) / 64, 1, false, t == ATOM_F32, true)) {}
    int grad_split() const {
        const long long blocks = (long long)nad * (split ? (R + 31) / 32 : 1) *
                                 ((D + 127) / 128 + (O + 127) / 128);
        const long long s = blocks ? (split ? 592 : 1184) / blocks : 1;
        return (int)std::max(1LL, std::min({s, 16LL, (long long)pieces}));
    }
};

struct AdSpace {
    __half *rows, *x, *w, *ad, *ext, *block, *bt;
    float *rinv, *wr, *ext_rinv, *part, *gpart;
    void *S, *T;
    int4 *piece, *bad;
    int2* tile_req;
    float* few_S;
    int* few_slot;
    unsigned* max;           // rows, w, adapters
    size_t bytes;
    AdSpace(void* ws, const AdSizes& z, bool bwd) {
        memset(this, 0, sizeof(*this));
        Cursor c(ws);
        const long long k = z.split ? 2 : 1, e = dtype_size(z.dtype);
        rows = c.take<__half>(k * z.M * (bwd ? z.Op : z.Dp));
        w = c.take<__half>(k * z.O * z.Dp);
        part = c.take<float>(z.product.part);
        if (z.split) {
            rinv = c.take<float>(up(z.M, 32));
            if (!bwd) wr = c.take<float>(up(z.O, 32));
            max = c.take<unsigned>(4);
            ext_rinv = c.take<float>(z.on ? z.M : 0);
        }
        if (z.on) {
            if (!bwd && z.M <= few::kFewRows) {
                few_S = c.take<float>(z.M * z.R);
                few_slot = c.take<int>(z.M);
            }
            piece = c.take<int4>(z.pieces);
            bad = c.take<int4>(z.nad);
            tile_req = c.take<int2>(z.tiles);
            // the low-rank product's adapters, and those of the product beside the projection
            if (!z.split) ad = c.take<__half>((long long)z.nad * z.R * (bwd ? z.Op : z.Dp));
            ext = c.take<__half>(k * z.nad * (bwd ? z.R * z.Dp : (long long)z.O * z.Rs));
            block = c.take<__half>(k * z.pieces * 256 * z.Rs);
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
int shrink16(const Shrink& p, dim3 grid, Chain& st) {
    const int nt = (p.R + 7) / 8;
#define ATOM_SHRINK(N)                                                                       \
    if (nt <= N) {                                                                           \
        const int smem = 8 * 16 * 8 * N * 4;                                                 \
        if (smem > 48 * 1024)                                                                \
            cudaFuncSetAttribute(shrink16_kernel<BF16, N>,                                   \
                                 cudaFuncAttributeMaxDynamicSharedMemorySize, smem);         \
        return st.launch("adapters: low-rank rows", shrink16_kernel<BF16, N>, grid, 256, smem, p); \
    }
    ATOM_SHRINK(1)
    ATOM_SHRINK(2)
    ATOM_SHRINK(4)
    ATOM_SHRINK(8)
    ATOM_SHRINK(16)
#undef ATOM_SHRINK
    return ATOM_ERR_UNSUPPORTED;
}
int shrink(const Shrink& p, Chain& st) {
    const dim3 grid(p.pieces + p.q.nad + 1, 256 / p.rb);
    if (p.dtype == ATOM_BF16) return shrink16<true>(p, grid, st);
    if (p.dtype == ATOM_F16) return shrink16<false>(p, grid, st);
    return st.launch("adapters: low-rank rows", shrink32_kernel, grid, 256, 32 * (p.R + 1) * 4, p);
}

// One direction: out [M, N] = rows [M, K] W' + (low-rank rows) (adapters), where forward has
// rows = x, W' = w^T, and backward rows = dy, W' = w.
struct Ad {
    AdSizes z;
    AdSpace sp;
    Chain st;
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
            // the largest w and adapters, and no scales for rows without low-rank values
            if (int s = st.zero("adapters", sp.max,
                                (char*)(sp.ext_rinv + (z.on ? z.M : 0)) - (char*)sp.max))
                return s;
            if (bwd) l.add({w, z.O, z.D, z.D, nullptr, 0, 0, nullptr, sp.max + 1, kMax, nullptr});
            if (z.on)
                l.add({second, srows, scols, scols, nullptr, 0, 0, nullptr, sp.max + 2, kMax,
                       nullptr});
            l.add({rows, z.M, K, ld, sp.rows, Kp, z.M * Kp, sp.rinv, nullptr, kRowSplit, nullptr});
            if (!bwd)
                l.add({w, z.O, z.D, z.D, sp.w, z.Dp, z.O * z.Dp, sp.wr, nullptr, kRowSplit,
                       nullptr});
            if (int s = prepare(l, st)) return s;
            l.n = 0;
            if (bwd)
                l.add({w, z.O, z.D, z.D, sp.w, z.Dp, z.O * z.Dp, nullptr, sp.max + 1, kTensorSplit,
                       nullptr});
            if (z.on)
                l.add({second, srows, scols, scols, sp.ext, sp_ld, srows * sp_ld, nullptr,
                       sp.max + 2, kTensorSplit, nullptr});
        } else {
            if (!tma_ready(rows, ld)) {
                l.add({rows, z.M, K, ld, sp.rows, Kp, 0, nullptr, nullptr, kPack, nullptr});
                xr = sp.rows, xld = Kp;
            }
            if (!low_only && !tma_ready(w, z.D)) {
                l.add({w, z.O, z.D, z.D, sp.w, z.Dp, 0, nullptr, nullptr, kPack, nullptr});
                wp = sp.w, wld = z.Dp;
            }
            if (both && !tma_ready(second, scols)) {
                l.add({second, srows, scols, scols, sp.ext, sp_ld, 0, nullptr, nullptr, kPack, nullptr});
                sec = sp.ext, sec_ld = sp_ld;
            }
            if (z.on && !bwd && !tma_ready(first, z.D)) {
                l.add({first, (long long)z.nad * z.R, z.D, z.D, sp.ad, z.Dp, 0, nullptr, nullptr,
                       kPack, nullptr});
                first = sp.ad;
            }
        }
        if (int s = prepare(l, st)) return s;
        if (z.on) {
            Shrink h;
            memset(&h, 0, sizeof(h));
            h.q = q;
            h.pieces = z.pieces;
            // Small blocks for large requests, but no more than eight blocks an SM (fp32, whose blocks
            // are larger: two): most of a small request's piece is zeros, and finding its rows costs
            // a block some two microseconds (12,011 rows of 512 requests, fp32: 54 us with 4,800
            // blocks, 25 us with 1,200, SHRINKUS us with 600).
            for (h.rb = 32; h.rb < 256 && z.pieces * (256 / h.rb) > (z.split ? 2 : 8) * 148;
                 h.rb *= 2) {
            }
            h.rows = z.split ? rows : xr;
            h.ld = z.split ? ld : xld;
            h.K = K;
            h.w = first;
            if (bwd && z.split) {
                h.wa = (long long)z.O * z.R, h.wr = 1, h.wk = z.R;
            } else if (bwd) {
                if (int s = st.launch("adapters: transpose", transpose_kernel,
                                      dim3(ceil_div(z.Op, 32), ceil_div(z.R, 32), z.nad), 256, 0,
                                      static_cast<const unsigned short*>(b), z.O, z.R, (int)z.Op,
                                      reinterpret_cast<unsigned short*>(sp.ad)))
                    return s;
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
        const Choice c = z.product;
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
            if (int s = make_slice_map(&maps.m[2 * k + pl], at(sp.block, bplane), z.R,
                                       (long long)z.pieces * 256, z.Rs, 128, false, 0, 0))
                return s;
            const long long sl = z.split ? sp_ld : sec_ld;
            if (int s = make_slice_map(&maps.m[3 * k + pl], at(z.split ? sp.ext : sec, planes[2]),
                                       scols, bwd ? z.R : z.O, sl, c.bn / 2, bwd, z.nad,
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
        p.cinv[0] = sp.wr;
        if (z.split && bwd) p.bmax = sp.max + 1;
        if (z.on) {
            p.ext = (z.R + 15) / 16;
            p.ext_a = 2 * k, p.ext_b = 3 * k, p.ext_bmn = bwd ? 1 : 0;
            p.tile_req = sp.tile_req;
            p.piece = sp.piece;
            p.bad = sp.bad;
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
    const AdSizes z(dtype, M, D, O, n_adapters, R, nreq, false);
    bytes_host[0] = AdSpace(nullptr, z, false).bytes;
    bytes_host[1] = AdSpace(nullptr, AdSizes(dtype, M, D, O, n_adapters, R, nreq, true), true).bytes;
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
    const AdSizes z(dtype, M, D, O, n_adapters, R, nreq, false);
    ATOM_REQUIRE(!z.on || (a && b && scale && req_ptr && req_adapter),
                 "adapted_linear: bad operand");
    Ad f{z, AdSpace(ws, z, false), (cudaStream_t)stream,
         {req_ptr, req_adapter, nreq, n_adapters, (int)M}, scale, w, a, b};
    ATOM_REQUIRE(ws && ws_bytes >= f.sp.bytes, "adapted_linear: the workspace needs %zu bytes",
                 f.sp.bytes);
    if (few::suits(dtype, M, D, x, ldx, w, a)) {
        // a few rows: the low-rank values first, then the projection with them in its epilogue;
        // nothing is kept, the backward pass computes S again
        if (z.on)
            if (int s = few::low_rank({x, ldx, (int)M, D, a, R, scale, req_ptr, req_adapter, nreq,
                                       n_adapters, f.sp.few_S, f.sp.few_slot, dtype}, f.st))
                return s;
        return few::product({x, ldx, (int)M, D, {w, nullptr}, O, 0, y, ldy, dtype,
                             z.on ? f.sp.few_S : nullptr, f.sp.few_slot, b, R}, f.st);
    }
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
    const AdSizes z(dtype, M, D, O, n_adapters, R, nreq, true);
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
    if (few::suits(dtype, M, D, x, ldx, w, a)) kept = nullptr;
    if (grads && db && !kept) {      // S again
        AdSpace fs = f.sp;
        fs.rows = f.sp.x;            // x's copy, where it needs one
        fs.ad = f.sp.bt;
        Ad g = f;
        g.sp = fs;
        if (int s = g.run(x, ldx, false, nullptr, 0, f.sp.S, true)) return s;
        f.st = g.st;
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
    if (!z.split) {                  // the copies that the products read, where they made one
        if (!tma_ready(dy, lddy)) p.rows[1] = f.sp.rows, p.ld[1] = z.Op;
        if (da && !tma_ready(x, ldx)) {
            if (kept || !db) {
                PrepList l;
                l.add({x, M, D, ldx, f.sp.x, z.Dp, 0, nullptr, nullptr, kPack, nullptr});
                if (int s = prepare(l, f.st)) return s;
            }
            p.rows[0] = f.sp.x, p.ld[0] = z.Dp;
        }
    }
    p.width[0] = da ? D : 0, p.width[1] = db ? O : 0;
    p.tiles0 = ceil_div(p.width[0], 128);
    p.out[0] = da, p.out[1] = db;
    p.part = f.sp.gpart;
    p.split = z.grad_split();
    p.dtype = dtype;
    const int tiles = p.tiles0 + ceil_div(p.width[1], 128);
    const dim3 grid(tiles, (unsigned)n_adapters * (z.split ? (R + 31) / 32 : 1), p.split);
    int rc;
    if (dtype == ATOM_BF16) rc = grads16<true>(p, grid, f.st);
    else if (dtype == ATOM_F16) rc = grads16<false>(p, grid, f.st);
    else rc = f.st.launch("adapters: gradients", grads32_kernel, grid, 256, 0, p);
    if (rc) return rc;
    if (p.split > 1)
        return f.st.launch("adapters: gradient sums", grads_sum_kernel, dim3(592), 256, 0, p);
    return ATOM_OK;
}
