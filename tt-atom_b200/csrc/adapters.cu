// Low-rank adapters of many requests beside a shared projection, and their backward pass.
//
//   y = x W^T + S B^T,  S = s (x A^T) row by row with the row's own A, B and s
//
// The requests' rows are cut at every 256th row into pieces: piece t + r holds the rows of request
// r in row tile t (t + r grows along the requests, so it names a piece without a table). Pieces of
// a tile that have one adapter share a block of 256 rows, which the first of them leads. One product
// gives S: each row tile times the adapters of its blocks, 16 ranks a slice, of which rows that are
// not the adapter's become zeros in its block. The shared projection's product (pair_product.cu)
// then takes each block of its row tile as more of K, S times the adapter's B, in slices of 16
// ranks of which four make a stage: the adapters cost their own multiplications and no pass over
// y. The backward pass is the same with T = s (dy B), W and A in the place of S, W^T and B, and
// dA = T^T x, dB = dy^T S summed by pieces in their order.
//
// Zeros in a block keep other requests' rows as they are only where B is finite; an adapter that
// is not is found when the pieces are, read as zeros, and its own rows are set to NaN.
#include <algorithm>

#include "few_rows.cuh"
#include "pair_product.cuh"

namespace atom {
namespace {

using namespace pair;

constexpr int kStages = 4;           // of grads16_kernel
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
// the fragments of m16n8k16. Each of 8 warps has 16 columns and all ranks. 6,007 rows of 2,048 + 2,048
// columns, 8 adapters of 16 ranks: 20 us (2.4 TB/s; floor 7.6), bound by the latency of its stages.
template <bool BF16, int MT>
__global__ void __launch_bounds__(256) grads16_kernel(const __grid_constant__ Grads p) {
    constexpr int kX = 32 * 272, kT = 32 * (32 * MT + 16);
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

// fp32: 32 ranks by 128 columns a block, 4 x 4 a thread, 32 rows at a time. On the FMA pipe: it is
// exact without planes, and 4,000 x 512 columns x 20 ranks take 14 us, 2,124 x 4,150 x 32 take 42.
__global__ void __launch_bounds__(256) grads32_kernel(const __grid_constant__ Grads p) {
    __shared__ __align__(16) float ts[32][36], xs[32][132];
    let_next_start();
    wait_before();
    const int chunks = (p.R + 31) / 32, tile = blockIdx.x / chunks;
    const int a = blockIdx.y, r0 = (blockIdx.x - tile * chunks) * 32;
    const int which = tile >= p.tiles0;
    const int c0 = (tile - (which ? p.tiles0 : 0)) * 128, W = p.width[which];
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
// A thread has a column and four ranks: it reads along rows of columns and writes dB's ranks,
// which lie side by side, together. Bound by the latency of its loads, 16 in flight a thread.
__global__ void __launch_bounds__(256) grads_sum_kernel(const __grid_constant__ Grads p) {
    let_next_start();
    wait_before();
    const int W = p.width[0] + p.width[1], groups = (p.R + 3) / 4;
    const int k = blockIdx.x * 256 + threadIdx.x;
    if (k >= W) return;
    const long long per = (long long)p.R * W, all = per * p.nad;
    const bool first = k < p.width[0], vec = aligned16(p.out[1]);
    for (int i = blockIdx.y; i < p.nad * groups; i += gridDim.y) {
        const int a = i / groups, r0 = (i - a * groups) * 4, n = min(4, p.R - r0);
        const float* part = p.part + a * per + (long long)r0 * W + k;
        float v[4] = {};
        for (int s0 = 0; s0 < p.split; s0 += 4) {    // 16 loads at once
            float t[4][4];
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    t[s][j] = j < n && s0 + s < p.split
                        ? part[(s0 + s) * all + (long long)j * W] : 0.f;
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] += t[s][j];
        }
        const long long at = first ? ((long long)a * p.R + r0) * p.width[0] + k
                                   : ((long long)a * p.width[1] + k - p.width[0]) * p.R + r0;
        const long long step = first ? p.width[0] : 1;
        if (!first && p.R % 4 == 0 && vec) {         // four ranks at once
            if (p.dtype == ATOM_F32)
                *reinterpret_cast<float4*>(static_cast<float*>(p.out[1]) + at) =
                    make_float4(v[0], v[1], v[2], v[3]);
            else
                *reinterpret_cast<uint2*>(static_cast<unsigned short*>(p.out[1]) + at) =
                    make_uint2(pair_w(v[0], v[1], p.dtype), pair_w(v[2], v[3], p.dtype));
            continue;
        }
        void* out = first ? p.out[0] : p.out[1];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < n) store_f(out, at + j * step, v[j], p.dtype);
    }
}
template <bool BF16>
int grads16(const Grads& p, dim3 grid, Chain& st) {
#define ATOM_GRADS(N)                                                                             \
    if (p.R <= 16 * N) {                                                                          \
        constexpr int smem = kStages * (32 * 272 + 32 * (32 * N + 16));                           \
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
    int tiles, pieces, Rs, ext;      // ext: slices of 16 ranks
    long long stages;                // of four slices, in all row tiles' blocks
    long long Dp, Op;
    bool split, on;
    Choice product;
    AdSizes(int t, long long m, int d, int o, int n, int r, int q, bool bwd)
        : dtype(t), M(m), D(d), O(o), nad(n), R(r), nreq(q), tiles((int)((m + 255) / 256)),
          pieces(tiles + q), Rs((int)up(r, 8)), ext((r + 15) / 16),
          stages(first_stage(tiles, q, ext) + 1), Dp(up(d, 8)), Op(up(o, 8)), split(t == ATOM_F32),
          on(n > 0 && q > 0),
          product(choose(m, bwd ? d : o, ((bwd ? o : d) + 63) / 64, 1, false, t == ATOM_F32, true)) {}
    int planes() const { return split ? kPlanes : 1; }
    int grad_split() const {
        const long long blocks = (long long)nad * (split ? (R + 31) / 32 : 1) *
                                 ((D + 127) / 128 + (O + 127) / 128);
        // shares of the rows, for some eight blocks an SM, forward and backward: 6,007 rows, 8 adapters
        // in bf16 took 162, 149, 134 and 145 us with 1, 2, 4 and 8; in fp32, 7,882 rows of 1,146 + 336
        // columns, 2 adapters 287, 247 and 251 us with 8, 16 and 32, and 2,124 of 1,486 + 2,664 344,
        // 336 and 337
        const long long s = blocks ? 1184 / blocks : 1;
        return (int)std::max(1LL, std::min({s, split ? 32LL : 16LL, (long long)pieces}));
    }
};

// One call's buffers. Copies and planes of one direction's operands; the backward pass has x's a
// second time where the forward pass kept no S.
struct AdSpace {
    uint16_t *rows, *x, *w, *first, *first2, *ext, *block;
    float *part, *gpart, *few_S, *few_T, *few_dx;
    void *S, *T;
    int4 *piece, *bad, *tile_req;
    int2* lead;
    int *row_lead, *usable, *few_slot;
    size_t bytes;
    AdSpace(void* ws, const AdSizes& z, bool bwd) {
        memset(this, 0, sizeof(*this));
        Cursor c(ws);
        const long long k = z.planes(), e = dtype_size(z.dtype);
        if (z.M <= few::kFewRows) {
            few_S = c.take<float>(z.M * z.R);
            few_T = c.take<float>(bwd ? z.M * z.R : 0);
            few_slot = c.take<int>(z.M);
            if (bwd) few_dx = c.take<float>(few::down_shares(z.O, z.D) * z.M * z.D);
            bytes = c.used;
            return;
        }
        const long long a_n = (long long)z.nad * z.R * z.Dp, b_n = (long long)z.nad * z.O * z.Rs;
        rows = c.take<uint16_t>(k * z.M * (bwd ? z.Op : z.Dp));
        w = c.take<uint16_t>(k * z.O * z.Dp);
        part = c.take<float>(z.product.part);
        if (z.on) {
            piece = c.take<int4>(z.pieces);
            bad = c.take<int4>(z.nad);
            tile_req = c.take<int4>(z.tiles);
            usable = c.take<int>(z.pieces);
            lead = c.take<int2>(z.pieces);
            row_lead = c.take<int>(z.M);
            first = c.take<uint16_t>(k * (bwd ? b_n : a_n));
            ext = c.take<uint16_t>(k * (bwd ? a_n : b_n));
            block = c.take<uint16_t>(k * z.stages * 256 * 64);
            if (bwd) {
                T = c.take<char>(z.M * z.Rs * e);
                x = c.take<uint16_t>(k * z.M * z.Dp);
                if (!z.split) first2 = c.take<uint16_t>(a_n);
                S = c.take<char>(z.M * z.Rs * e);
                const long long s = z.grad_split();
                gpart = c.take<float>(s > 1 ? s * z.nad * z.R * (z.D + z.O) : 0);
            }
        }
        bytes = c.used;
    }
};

// One direction: out [M, N] = rows [M, K] W' + (low-rank rows) (adapters), where forward has
// rows = x, W' = w^T, and backward rows = dy, W' = w.
struct Ad {
    AdSizes z;
    AdSpace sp;
    Chain st;
    const int *req_ptr, *req_adapter;
    const float* scale;
    const void *w, *a, *b;
    Sums sums{};

    Pieces pieces(const void* other, long long other_n) const {
        return {req_ptr, req_adapter, z.nreq, z.nad, (int)z.M, z.tiles, z.pieces, sp.piece,
                sp.lead, sp.row_lead, sp.tile_req, other, other_n, sp.bad, z.dtype};
    }

    // A direction's operands: rows, the shared matrix, the adapters that make the low-rank rows
    // (first) and those beside the projection (second), each as it lies or as copies.
    struct Operands {
        const void *rows, *w, *first, *second;
        long long ld, w_ld, first_ld, second_ld;
        long long rows_plane, w_plane, first_plane, second_plane;
    };
    Args args(int N) const {
        Args p;
        memset(&p, 0, sizeof(p));
        p.M = z.M, p.N = N, p.groups = 1, p.nphase = 1;
        p.bf16 = z.dtype == ATOM_BF16;
        p.dtype = z.dtype;
        p.ext = z.ext;
        p.nad = z.nad;
        p.tile_req = sp.tile_req;
        p.piece = sp.piece;
        p.usable = sp.usable;
        p.lead = sp.lead;
        p.row_lead = sp.row_lead;
        p.bad = sp.bad;
        return p;
    }

    // The low-rank rows of `rows` [M, K] and a (forward) or b (backward): s rows first^T into
    // `kept` (may be NULL) and, as the product beside the projection takes them, the blocks.
    int low_rows(const Operands& o, bool bwd, void* kept, bool blocks) {
        const int K = bwd ? z.O : z.D, k = z.planes();
        Maps maps;
        for (int pl = 0; pl < k; ++pl) {
            const uint16_t* r = static_cast<const uint16_t*>(o.rows) + pl * o.rows_plane;
            const uint16_t* f = static_cast<const uint16_t*>(o.first) + pl * o.first_plane;
            if (int s = make_map(&maps.m[pl], r, K, z.M, o.ld, 128)) return s;
            if (int s = make_low_map(&maps.m[k + pl], f, bwd ? z.R : K, bwd ? K : z.R, o.first_ld,
                                     bwd, z.nad, (bwd ? K : z.R) * o.first_ld))
                return s;
        }
        Args p = args(128);
        p.ph[0] = {0, k, k, (K + 63) / 64, 0, bwd ? 1 : 0, 0, 0};
        p.used = (1u << 2 * k) - 1;
        p.low_scale = scale;
        p.low_block = !z.split || blocks ? sp.block : nullptr;
        p.low_plane = z.stages * 256 * 64;
        p.low_rows = kept;
        if (!blocks) p.usable = nullptr;
        p.Rs = z.Rs;
        // as many items as pairs of SMs, but no more than a tile may have groups (300 requests in 512
        // rows, an adapter each, 1,024 x 1,024 in bf16: 69 us so, 96 with four a tile, 208 with one;
        // 2,000 rows of 40 requests, rank 64, 512 x 512: 20.5, 20.5 and 26.7)
        const int groups = std::min(16, (z.nreq * p.ext + 7) / 8);
        const int share = std::max(1, std::min(groups, pair_count() / z.tiles));
        return launch(kLow, {128, share, 0}, z.split, maps, p, st, sums);
    }

    int run(const void* rows, long long ld, bool bwd, void* out, long long ldo, void* kept) {
        const int K = bwd ? z.O : z.D, N = bwd ? z.D : z.O, k = z.planes();
        const long long Kp = bwd ? z.Op : z.Dp;
        const void* first = bwd ? b : a;         // forward [nad][R][D], backward [nad][O][R]
        const void* second = bwd ? a : b;
        const long long frows = (long long)z.nad * (bwd ? z.O : z.R);
        const long long srows = (long long)z.nad * (bwd ? z.R : z.O);
        const int fcols = bwd ? z.R : z.D, scols = bwd ? z.D : z.R;
        const long long fp = bwd ? z.Rs : z.Dp, spp = bwd ? z.Dp : z.Rs;
        const bool product = out != nullptr;
        Operands o{rows, w, first, second, ld, z.D, fcols, scols, 0, 0, 0, 0};
        PrepList l;
        const Pieces found = pieces(product ? second : nullptr, (long long)z.R * (bwd ? z.D : z.O));
        auto take = [&](const void*& p, long long& pld, long long& plane, long long n, long long cols,
                        uint16_t* buf, long long pitch) {
            if (!z.split && tma_ready(p, pld)) return;
            plane = n * pitch;
            l.add({p, n, cols, pld, buf, pitch, plane, z.split ? kSplit : kPack});
            p = buf, pld = pitch;
        };
        take(o.rows, o.ld, o.rows_plane, z.M, K, sp.rows, Kp);
        if (product) take(o.w, o.w_ld, o.w_plane, z.O, z.D, sp.w, z.Dp);
        if (z.on) {
            take(o.first, o.first_ld, o.first_plane, frows, fcols, sp.first, fp);
            // (fp32: a's planes serve the gradients as well)
            if (product || z.split)
                take(o.second, o.second_ld, o.second_plane, srows, scols, sp.ext, spp);
        }
        if (int s = prepare(l, st, z.on ? &found : nullptr)) return s;
        if (z.on)
            if (int s = low_rows(o, bwd, kept, product)) return s;
        if (!product) return ATOM_OK;
        const Choice c = z.product;
        Maps maps;
        for (int pl = 0; pl < k; ++pl) {
            auto at = [&](const void* base, long long plane) {
                return static_cast<const uint16_t*>(base) + pl * plane;
            };
            if (int s = make_map(&maps.m[pl], at(o.rows, o.rows_plane), K, z.M, o.ld, 128)) return s;
            if (int s = make_map(&maps.m[k + pl], at(o.w, o.w_plane), z.D, z.O, o.w_ld,
                                 bwd ? 64 : c.bn / 2))
                return s;
            if (!z.on) continue;
            if (int s = make_map(&maps.m[2 * k + pl], at(sp.block, z.stages * 256 * 64), 64,
                                 z.stages * 256, 64, 128))
                return s;
            if (int s = make_slice_map(&maps.m[3 * k + pl], at(o.second, o.second_plane), scols,
                                       bwd ? z.R : z.O, o.second_ld, c.bn / 2, bwd, z.nad,
                                       (bwd ? z.R : z.O) * o.second_ld))
                return s;
        }
        Args p = args(N);
        p.ph[0] = {0, k, k, (K + 63) / 64, 0, bwd ? 1 : 0, c.bn, c.bn / 2};
        p.C[0] = out;
        p.ldc = ldo;
        p.used = z.on ? (1u << 4 * k) - 1 : (1u << 2 * k) - 1;
        p.part = sp.part;
        p.ext_a = 2 * k, p.ext_b = 3 * k, p.ext_bmn = bwd ? 1 : 0;
        if (int s = launch(z.on ? kStoreLow : kStore, c, z.split, maps, p, st, sums)) return s;
        return add_up(sums, st);
    }

    // S alone, in the backward pass: x's own copy (and a's: fp32 has it beside the projection), the
    // pieces as they are
    int low_again(const void* x, long long ldx) {
        const long long an = (long long)z.nad * z.R;
        Operands o{x, nullptr, a, nullptr, ldx, 0, z.D, 0, 0, 0, 0, 0};
        PrepList l;
        if (z.split || !tma_ready(x, ldx)) {
            o.rows = sp.x, o.ld = z.Dp, o.rows_plane = z.M * z.Dp;
            l.add({x, z.M, z.D, ldx, sp.x, z.Dp, o.rows_plane, z.split ? kSplit : kPack});
        }
        if (z.split) {
            o.first = sp.ext, o.first_ld = z.Dp, o.first_plane = an * z.Dp;
        } else if (!tma_ready(a, z.D)) {
            l.add({a, an, z.D, z.D, sp.first2, z.Dp, 0, kPack});
            o.first = sp.first2, o.first_ld = z.Dp;
        }
        if (int s = prepare(l, st)) return s;
        return low_rows(o, false, sp.S, false);
    }
};

int check_ad(int dtype, int64_t M, int D, int O, int nad, int R, int nreq) {
    ATOM_REQUIRE(dtype >= ATOM_F32 && dtype <= ATOM_F16, "adapted_linear: unknown type %d", dtype);
    ATOM_REQUIRE(M >= 0 && M < (1LL << 31) - 256 && D > 0 && O > 0 && nad >= 0 && nreq >= 0,
                 "adapted_linear: bad sizes");
    ATOM_REQUIRE(D < (1 << 24) && O < (1 << 24), "adapted_linear: widths above 2^24");
    ATOM_REQUIRE(R >= 1 && R <= 128, "adapted_linear: the rank must be 1..128");
    ATOM_REQUIRE(nad <= (1 << 14) && nreq <= (1 << 22) &&
                     first_stage((M + 255) / 256, nreq, (R + 15) / 16) < (1 << 23) - 1,
                 "adapted_linear: sizes above 2^14 adapters, 2^22 requests or 2^25 slices of 256 "
                 "rows by 16 ranks");
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
    Ad f{z, AdSpace(ws, z, false), (cudaStream_t)stream, req_ptr, req_adapter, scale, w, a, b};
    ATOM_REQUIRE(ws && ws_bytes >= f.sp.bytes, "adapted_linear: the workspace needs %zu bytes",
                 f.sp.bytes);
    ATOM_REQUIRE(aligned256(ws) && (M <= few::kFewRows || aligned256(kept)),
                 "adapted_linear: ws and kept must be 256-byte aligned");
    if (M <= few::kFewRows) {
        // a few rows: the low-rank values first, then the projection with them in its epilogue;
        // nothing is kept, the backward pass computes S again
        if (z.on)
            if (int s = few::low_rank({x, ldx, (int)M, D, a, R, scale, req_ptr, req_adapter, nreq,
                                       n_adapters, f.sp.few_S, f.sp.few_slot, dtype}, f.st))
                return s;
        few::Args p{};
        p.x = x, p.ldx = ldx, p.M = (int)M, p.K = D, p.N = O;
        p.w[0] = w;
        p.out = y, p.ldo = ldy;
        p.dtype = dtype;
        p.S = z.on ? f.sp.few_S : nullptr, p.slot = f.sp.few_slot, p.b = b, p.R = R;
        return few::product(p, f.st);
    }
    return f.run(x, ldx, false, y, ldy, kept);
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
    Ad f{z, AdSpace(ws, z, true), st, req_ptr, req_adapter, scale, w, a, b};
    ATOM_REQUIRE(ws && ws_bytes >= f.sp.bytes, "adapted_linear: the workspace needs %zu bytes",
                 f.sp.bytes);
    ATOM_REQUIRE(aligned256(ws) && (M <= few::kFewRows || aligned256(kept)),
                 "adapted_linear: ws and kept must be 256-byte aligned");
    const bool grads = z.on && (da || db);
    // (2,048 x 2,048, rank 16, bf16: 20.5 us at 1 row and 31.2 at 16, against 33.2 and 43.2 by tiles;
    // an adapter a row, 16 rows against 17 by tiles: fp32 44 and 121 us, fp16 45 and 53, forward 16 and
    // 72 in fp32, 10 and 27 in 16 bits)
    if (M <= few::kFewRows) {
        const int m = (int)M, shares = few::down_shares(O, D);
        if (z.on) {
            if (int s = few::low_rank({x, ldx, m, D, a, R, scale, req_ptr, req_adapter, nreq,
                                       n_adapters, f.sp.few_S, f.sp.few_slot, dtype}, f.st))
                return s;
            if (int s = few::low_rank_back({dy, lddy, m, O, b, R, scale, f.sp.few_slot, f.sp.few_T,
                                            dtype}, f.st))
                return s;
        }
        if (grads)
            if (int s = few::adapter_grads({f.sp.few_T, f.sp.few_S, f.sp.few_slot, x, dy, ldx, lddy,
                                            m, D, O, R, n_adapters, da, db, dtype}, f.st))
                return s;
        if (!dx) return ATOM_OK;
        if (int s = few::down({{dy, nullptr}, lddy, 0, m, O, {w, nullptr}, D, shares, f.sp.few_dx,
                               dtype}, f.st))
            return s;
        return few::sum({f.sp.few_dx, shares, m, D, dx, lddx, z.on ? f.sp.few_T : nullptr,
                         f.sp.few_slot, a, R, dtype}, f.st);
    }
    if (grads || dx)
        if (int s = f.run(dy, lddy, true, dx, lddx, grads ? f.sp.T : nullptr)) return s;
    const bool again = grads && db && !kept;
    if (again)
        if (int s = f.low_again(x, ldx)) return s;
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
        if (!tma_ready(x, ldx)) {
            if (!again) {
                PrepList l;
                l.add({x, M, D, ldx, f.sp.x, z.Dp, 0, kPack});
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
    const dim3 grid(tiles * (z.split ? (R + 31) / 32 : 1), n_adapters, p.split);
    int rc;
    if (dtype == ATOM_BF16) rc = grads16<true>(p, grid, f.st);
    else if (dtype == ATOM_F16) rc = grads16<false>(p, grid, f.st);
    else rc = f.st.launch("adapters: gradients", grads32_kernel, grid, 256, 0, p);
    if (rc) return rc;
    if (p.split > 1)
        return f.st.launch("adapters: gradient sums", grads_sum_kernel,
                           dim3(ceil_div(p.width[0] + p.width[1], 256),
                                std::min(n_adapters * ((R + 3) / 4), 65535)), 256, 0, p);
    return ATOM_OK;
}
