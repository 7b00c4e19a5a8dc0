// The tensor-core product behind the typed operators: D = sum over phases of A_p B_p^T on CTA
// pairs (tcgen05.mma.cta_group::2), with the operators' epilogues.
//
// Why pairs: a 256 x 256 tile of two SMs reads, per 64-deep K stage, 32 KB into each SM's shared
// memory for 512 clocks of tensor work; a 128 x 256 tile of one SM would read 48 KB for the same
// 512 clocks, more than shared memory can take in and hand to the tensor core at once.
//
// Operands are 16-bit, K-major (rows of K elements) or M/N-major (rows of M/N elements: the
// transposed products of a backward pass, read as they lie), in 128-byte swizzled tiles that
// TMA fetches and zero-fills past the ends. CTA 0 of a pair has rows 0..127 of the tile and half
// of B's, CTA 1 the others. Accumulators are fp32 in tensor memory, two buffers (SPLIT: four), so that the
// epilogue of one tile runs beside the products of the next.
//
// fp32 operands (SPLIT) come as three bf16 planes, hi + mid + lo (typed.cuh), without scales: a result
// does not depend on how large other rows, columns or requests are. A sum is six products: lo hi,
// hi lo, mid mid, mid hi, hi mid and hi hi (what is left out is below 2^-23 of a term). The tensor core
// rounds every addition toward zero, some 2^-24 of the sum a step, so a SPLIT tile is drained into
// registers (added there to nearest) after every stage, and a stage begins with the small products:
// four additions to a large sum. A slot of the ring holds one plane of a stage, lo first, and is free
// again when its products are done.
//
// Bound by the tensor core where K and the tiles are many: the whole training step of 8,192 x 2,048
// x 8,192 in bf16 (2.47 TFLOP in 6 launches) runs at 1.34 PFLOP/s, 95 % of what a library product
// sustains under the power cap; 60,000 x 256 -> 2 x 1,024 with the gate at 1.1, bound by its
// epilogue; a SPLIT sum's six products run at 1.19 PFLOP/s together at 4,011 x 672 x 2,632 forward and
// at 1.49 at 8,192 x 2,048 x 4,096, bound by reading planes from L2 and by the tensor core.
//
// Warp 0 has TMA, warp 1 tensor memory and the products (CTA 0's issues for both), warps 2.. the
// epilogue. Every wait is bounded: on expiry the kernel records a code, lets copies in
// flight land, frees its tensor memory and returns.
#include <cudaTypedefs.h>

#include <algorithm>
#include <cstring>

#include "pair_product.cuh"

#pragma nv_diag_suppress 128      // loops that an instantiation has no way to

namespace atom {
namespace pair {

constexpr long long kWaitCycles = 2000000000LL;      // ~1 s

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ uint32_t peer_addr(uint32_t a, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    return r;
}
__device__ __forceinline__ void mbar_init(uint64_t* b, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(b)), "r"(count));
}
__device__ __forceinline__ bool mbar_try(uint64_t* b, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(smem_u32(b)), "r"(parity) : "memory");
    return ok != 0;
}
// Bounded wait; false once the budget is spent or any CTA has failed. The clock and the error
// word (a trip to L2) are looked at every 256 tries only.
__device__ __forceinline__ bool mbar_wait(uint64_t* b, uint32_t parity, int* err,
                                          long long budget = kWaitCycles) {
    if (mbar_try(b, parity)) return true;
    const long long t0 = clock64();
    for (uint32_t n = 1;; ++n) {
        if (mbar_try(b, parity)) return true;
        if ((n & 255) == 0) {
            if (clock64() - t0 > budget) {
                atomicCAS(err, 0, ATOM_PAIR_WAIT_CODE);
                return false;
            }
            if (*(volatile int*)err != 0) return false;
        }
    }
}
// TMA tile load into this CTA's shared memory, counted on a barrier of the pair's CTA 0.
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y,
                                         uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x),
        "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_load3(uint32_t dst, const CUtensorMap* map, int x, int y,
                                          int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)),
        "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
// Shared-memory matrix descriptor, 128-byte swizzle. K-major: 8-row groups 1024 bytes apart.
// M/N-major: 64-element blocks 8192 bytes apart (one 64-deep stage), 8-deep groups 1024 apart.
__device__ __forceinline__ uint64_t sdesc(uint32_t saddr, int mn) {
    uint64_t d = (uint64_t)((saddr >> 4) & 0x3FFF);
    d |= (uint64_t)(mn ? 8192 >> 4 : 1) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
// A low-rank slice, 16 deep: K-major rows of 32 bytes in 32-byte swizzle (8-row groups 256 bytes
// apart), or M/N-major like a stage's but with 64-element blocks 2048 bytes apart.
__device__ __forceinline__ uint64_t sdesc_slice(uint32_t saddr, int mn) {
    uint64_t d = (uint64_t)((saddr >> 4) & 0x3FFF);
    d |= (uint64_t)(mn ? 2048 >> 4 : 1) << 16;
    d |= (uint64_t)((mn ? 1024 : 256) >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)(mn ? 2 : 6) << 61;
    return d;
}
// kLow's M/N-major slices: 64 rows of 32 bytes in 32-byte swizzle, 16-element blocks 2048 bytes
// apart, 8-deep groups 256 bytes apart.
__device__ __forceinline__ uint64_t sdesc_low(uint32_t saddr) {
    uint64_t d = (uint64_t)((saddr >> 4) & 0x3FFF);
    d |= (uint64_t)(2048 >> 4) << 16;
    d |= (uint64_t)(256 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)6 << 61;
    return d;
}
// Instruction descriptor (kind::f16): D fp32, M = 256 over the pair, N = n.
__device__ __forceinline__ uint32_t idesc(int n, int bf16, int a_mn, int b_mn) {
    return (1u << 4) | ((uint32_t)bf16 << 7) | ((uint32_t)bf16 << 10) | ((uint32_t)a_mn << 15) |
           ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | (16u << 24);
}
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t id,
                                    uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
        "r"(id), "r"(accumulate));
}
// Arrives on the barrier of both CTAs once the products issued so far are done.
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
        " [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t a, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
        "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
        "%30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
          "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
          "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(a));
}
__device__ __forceinline__ void tmem_wait_ld() {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// Keeps the use of loaded values behind the wait.
__device__ __forceinline__ void pin32(float* v) {
#pragma unroll
    for (int i = 0; i < 32; ++i) asm volatile("" : "+f"(v[i]));
}
// True in one lane of a converged warp. The TMA and product warps walk their loops with all
// lanes, so that what they compute stays uniform, and one lane issues.
__device__ __forceinline__ bool elect_one() {
    uint32_t yes;
    asm volatile(
        "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(yes));
    return yes != 0;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

struct Tile {
    int mt, nt, grp, ks;
};
// Work item -> tile. Eight row tiles by all column tiles at a time, so that the pairs at work
// share both operands' tiles in L2.
__device__ __forceinline__ Tile tile_of(const Args& p, long long item) {
    Tile ti;
    uint32_t u = (uint32_t)item;         // 32-bit: every warp divides here, tile by tile
    ti.ks = 0;
    if (p.ksplit > 1) {
        ti.ks = u % (uint32_t)p.ksplit;
        u /= (uint32_t)p.ksplit;
    }
    const uint32_t all = p.mtiles * p.groups, band = 8u * p.ntiles_n;
    const uint32_t b = u / band, r = u - b * band;
    const uint32_t high = min(8u, all - b * 8);
    ti.nt = high == 8 ? r >> 3 : r / high;
    ti.mt = b * 8 + r - ti.nt * high;
    ti.grp = 0;
    if (ti.mt >= p.mtiles) ti.grp = 1, ti.mt -= p.mtiles;
    return ti;
}

__device__ __forceinline__ bool is_finite(const Args& p, int slot) {
    const int4 b = p.bad[slot];
    return (b.x | b.y | b.z | b.w) == 0;
}
// Whether row m (a lane's) belongs to a request whose adapter is not finite.
__device__ __noinline__ bool spoilt_row(const Args& p, int mt, long long m, int lane) {
    const int4 q = p.tile_req[mt];
    bool bad = false;
    for (int r = q.x; r < q.y; r += 32) {
        int4 c = make_int4(-1, 0, 0, 0);
        if (r + lane < q.y) c = p.piece[mt + r + lane];
        unsigned found = __ballot_sync(0xffffffffu, c.x >= 0 && !is_finite(p, c.x));
        for (; found; found &= found - 1) {
            const int i = __ffs(found) - 1;
            const int lo = __shfl_sync(0xffffffffu, c.y, i), hi = __shfl_sync(0xffffffffu, c.z, i);
            bad |= m >= lo && m < hi;
        }
    }
    return bad;
}

// What a warp knows of its tiles' requests: a lane a tile, 32 tiles ahead, so that no tile waits
// for its own (a load takes two microseconds beside the tiles' traffic).
struct Ahead {
    int4 mine;
    __device__ __forceinline__ int4 get(const Args& p, uint32_t k, uint32_t first, uint32_t pairs) {
        if ((k & 31) == 0) {
            const long long t = first + (long long)(k + (threadIdx.x & 31)) * pairs;
            mine = make_int4(0, 0, 0, 0);
            if (t < p.tiles) mine = p.tile_req[tile_of(p, t).mt];
        }
        const int l = k & 31;
        return make_int4(__shfl_sync(0xffffffffu, mine.x, l), __shfl_sync(0xffffffffu, mine.y, l),
                         __shfl_sync(0xffffffffu, mine.z, l), __shfl_sync(0xffffffffu, mine.w, l));
    }
};

// A work item's K stages of one phase.
struct Share {
    int kt, end;
    __device__ __forceinline__ Share(const Args& p, const Tile& ti, int f) {
        const int nk = p.ph[f].nk;
        kt = p.ksplit == 1 ? 0 : (int)((long long)ti.ks * nk / p.ksplit);
        end = p.ksplit == 1 ? nk : (int)((long long)(ti.ks + 1) * nk / p.ksplit);
    }
};
// Walks the low-rank blocks of a row tile in slices of 16 ranks, p.ext of them each, four to a
// stage. The adapters of 32 blocks, one a lane, are asked for when the walk is made and needed when
// it begins.
struct Blocks {
    const Args& p;
    const int* usable;
    int n, j = -1, mine, sub = 0, slot = 0;
    __device__ __forceinline__ Blocks(const Args& q, int tile, const int4& t)
        : p(q), usable(q.usable + tile + t.x), n(t.z) {
        ask(0);
    }
    __device__ __forceinline__ void ask(int k) {
        k += threadIdx.x & 31;
        mine = k < n ? usable[k] : 0;
    }
    // the next slice (at(), slot); false when there is none
    __device__ __forceinline__ bool next() {
        if (sub > 0 && sub < p.ext) {
            ++sub;
            return true;
        }
        if (++j >= n) return false;
        if (j && (j & 31) == 0) ask(j);
        slot = __shfl_sync(0xffffffffu, mine, j & 31);
        sub = 1;
        return true;
    }
    __device__ __forceinline__ int at() const { return (sub - 1) * 16; }     // first rank
};

// Writes down which adapters the product beside the projection takes for a row tile's blocks.
// Adapter nad, past the tensor map's end, reads as zeros: what is not finite leaves the other rows
// as they are. A whole warp.
__device__ __forceinline__ void settle(const Args& p, int mt) {
    const int4 t = p.tile_req[mt];
    bool spoilt = false;
    for (int j = threadIdx.x & 31; j < t.z; j += 32) {
        const int a = p.lead[mt + t.x + j].x;
        const bool ok = is_finite(p, a);
        p.usable[mt + t.x + j] = ok ? a : p.nad;
        spoilt |= !ok;
    }
    spoilt = __any_sync(0xffffffffu, spoilt);
    if ((threadIdx.x & 31) == 0) p.tile_req[mt].w = spoilt;
}

// kLow: groups of a row tile's blocks whose slices of 16 ranks fill 128 columns (a block's slices
// stay together); with few row tiles, `ksplit` work items share a tile's groups.
struct Low {
    const Args& p;
    int mt, first, count, slices, half, each;    // blocks; slices a block; blocks a half, a group
    __device__ __forceinline__ Low(const Args& q, int tile) : p(q), mt(tile) {
        const int4 t = p.tile_req[mt];
        first = t.x;
        count = t.z;
        slices = p.ext;
        half = slices <= 4 ? 4 / slices : 0;
        each = slices <= 4 ? 2 * half : 1;
    }
    __device__ __forceinline__ int groups() const { return (count + each - 1) / each; }
    // slices of group g in half h (64 columns; slice i of a group is i % 4 of half i / 4)
    __device__ __forceinline__ int used(int g, int h) const {
        if (slices > 4) return h ? slices - 4 : 4;
        return max(0, min(half, count - g * each - h * half)) * slices;
    }
    __device__ __forceinline__ int sub(int i) const {           // which of its block's slices i is
        return slices > 4 ? i : (i & 3) % slices;
    }
    // the block of slice i of group g: which one of the tile's, its adapter, the request that leads it
    __device__ __forceinline__ int3 block(int g, int i) const {
        const int j = g * each + (slices > 4 ? 0 : (i >> 2) * half + (i & 3) / slices);
        const int2 l = p.lead[mt + first + j];
        return make_int3(j, l.x, l.y);
    }
};

template <int BN, int EPI, bool SPLIT>
struct Cfg {
    // Epilogue warps: 16 for a wide gate, whose arithmetic is more than its products at small K
    // (60,000 x 256 x 1024 bf16: 78 us with 8, 69 us with 16; two groups of 8 on alternate
    // tiles hold accumulators longer, 80 us), at the cost of a stage's room; 8 elsewhere (plain
    // tiles lose 4 % to the shorter ring).
    static constexpr int EW = EPI == kGate && BN == 256 ? 16 : 8;
    static constexpr int kThreads = 64 + 32 * EW;
    static constexpr int HB = BN / 2;
    static constexpr uint32_t kA = 128 * 128, kB = HB * 128;
    static constexpr uint32_t kSlot = kA + kB;       // a stage (SPLIT: of one plane)
    static constexpr int S = (EW == 16 ? 160 : 192) * 1024 / kSlot;
    static constexpr int kBufs = SPLIT ? 4 : 2;      // accumulators in tensor memory
    static_assert(kBufs * BN <= 512, "tensor memory");
    static constexpr uint32_t kOut = EW * 4096;
    static constexpr uint32_t kSmem = S * kSlot + kOut + 512 + 1024;
    static_assert(kSmem <= 232448, "shared memory");
};

// A warp's way out: 32 x 32 blocks, one row a lane, through a swizzled 4 KB buffer of its own. A
// lane that stored its row directly would touch 32 lines with every 16 bytes: the gate's tiles
// took 13,000 clocks that way, more than their products.
struct Out {
    uint8_t* buf;
    uint32_t turn;
};
__device__ __forceinline__ void stage_f32(uint8_t* buf, int lane, const float* v) {
#pragma unroll
    for (int c = 0; c < 8; ++c)
        *reinterpret_cast<float4*>(buf + lane * 128 + ((c ^ (lane & 7)) << 4)) =
            make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
}
// By TMA, which leaves out what lies past the map's rows and columns.
template <bool DEEP>
__device__ __forceinline__ void send(const uint8_t* b, int lane, const CUtensorMap* map, int x, int y,
                                     int z) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) {
        if constexpr (!DEEP)
            asm volatile(
                "cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                    reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(b)) : "memory");
        else
            asm volatile(
                "cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];"
                ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(b))
                : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
}
template <bool DEEP = false>
__device__ __forceinline__ void store_f32(Out& o, int lane, const CUtensorMap* map, int x, int y, int z,
                                          const float* v) {
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
    stage_f32(o.buf, lane, v);
    send<DEEP>(o.buf, lane, map, x, y, z);
}
// 16-bit blocks, `word(i)` columns 2 i and 2 i + 1, take the two halves of the buffer in turn.
template <typename W>
__device__ __forceinline__ void store_16(Out& o, int lane, const CUtensorMap* map, int x, int y, W word) {
    uint8_t* b = o.buf + (o.turn++ & 1u) * 2048;
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 4; ++c)
        *reinterpret_cast<uint4*>(b + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4)) =
            make_uint4(word(4 * c), word(4 * c + 1), word(4 * c + 2), word(4 * c + 3));
    send<false>(b, lane, map, x, y, 0);
}
// Typed, or (SPLIT) as planes, which uses up v.
template <bool SPLIT>
__device__ __forceinline__ void store_typed(Out& o, int lane, const CUtensorMap* map, int x, int y,
                                            float* v, int dtype) {
    if constexpr (SPLIT) {
#pragma unroll
        for (int k = 0; k < kPlanes; ++k)
            store_16(o, lane, map + k, x, y,
                     [&](int i) { return take_plane(v[2 * i], v[2 * i + 1], k); });
    } else {
        store_16(o, lane, map, x, y, [&](int i) { return pair_w(v[2 * i], v[2 * i + 1], dtype); });
    }
}
// Where rows do not start on 16 bytes, or end inside them: row by row, a column a lane.
__device__ __forceinline__ void store_rows(Out& o, int lane, void* C, long long off, long long ld,
                                           int rows, int cols, const float* v, int dtype) {
    __syncwarp();
    stage_f32(o.buf, lane, v);
    __syncwarp();
    for (int r = 0; r < rows; ++r) {
        const float x = *reinterpret_cast<const float*>(
            o.buf + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
        if (lane < cols) store_f(C, off + r * ld + lane, x, dtype);
    }
}
// Buffers that only these kernels read are kept as the lanes have them: 32 x 32 blocks, 16
// bytes a lane at a time.
__device__ __forceinline__ float* lane_block(float* p, long long m, int n, int Fp, int lane) {
    return p + ((m >> 5) * (Fp >> 5) + (n >> 5)) * 1024 + lane * 4;
}
__device__ __forceinline__ void store_block(float* q, const float* v) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
        *reinterpret_cast<float4*>(q + 128 * j) =
            make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
}
__device__ __forceinline__ void load_block(const float* q, float* v) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float4 x = *reinterpret_cast<const float4*>(q + 128 * j);
        v[4 * j] = x.x, v[4 * j + 1] = x.y, v[4 * j + 2] = x.z, v[4 * j + 3] = x.w;
    }
}
__device__ __forceinline__ void spoil32(float* v) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(0x7FC00000u);
}
// The gate and its gradient. Sigmoids from ex2.approx and rcp.approx, each good to 2 units in the
// last place, beside |g| 2^-24 from the exponent's own rounding.
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// GELU's normal distribution function: its tail is exp(-g^2 / 2) t P(t), t = 1 / (1 + |g| / 8^0.5), with
// P fitted to erfc(x) exp(x^2) / 2 for the least relative error over x < 10.5 (4e-8; 3.2e-7 in fp32
// steps), which a closed gate's value needs; the exponential is the density in the derivative.
__device__ __forceinline__ void normal(float g, float& cdf, float& bell) {
    const float t = __fdividef(1.f, fmaf(0.35355339f, fabsf(g), 1.f));
    bell = __expf(-0.5f * g * g);
    constexpr float kP[9] = {0.141042784f,   0.141195029f, 0.121498309f, 0.101554938f, -0.0138116609f,
                             0.139756203f, -0.24423036f, 0.142591372f, -0.0295966566f};
    float poly = kP[8];
#pragma unroll
    for (int k = 7; k >= 0; --k) poly = fmaf(t, poly, kP[k]);
    const float tail = t * poly * bell;
    cdf = g < 0.f ? tail : 1.f - tail;
}
// Two sigmoids with one reciprocal, 1 / (a b): a multiprocessor has 16 results of ex2 and rcp a
// clock, and a gate needs both for every value. From e = exp(-|g|) <= 1, so that a b is at most 4 and
// a closed gate (e / (1 + e)) keeps its value down to the smallest normal one. A NaN in one of the
// two is in both: they are columns of one row of H, and each of y's sums over that row is NaN anyway.
__device__ __forceinline__ void sigmoid2(float g0, float g1, float& s0, float& s1) {
    const float e0 = exp2_fast(-1.4426950f * fabsf(g0)), e1 = exp2_fast(-1.4426950f * fabsf(g1));
    const float a = 1.f + e0, b = 1.f + e1, r = rcp_fast(a * b);
    s0 = (g0 >= 0.f ? b : e0 * b) * r;
    s1 = (g1 >= 0.f ? a : e1 * a) * r;
}
// h = act(g) u
template <bool GELU>
__device__ __forceinline__ void gate32(float* g, const float* u, int act) {
    if constexpr (!GELU) {
        const bool silu = act == 0;
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            float s0, s1;
            sigmoid2(g[i], g[i + 1], s0, s1);
            g[i] = (silu ? g[i] : 1.f) * s0 * u[i];
            g[i + 1] = (silu ? g[i + 1] : 1.f) * s1 * u[i + 1];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            float c, bell;
            normal(g[i], c, bell);
            g[i] = g[i] * c * u[i];
        }
    }
}
// (g, u, d = dh) -> (dg, du, h)
template <bool GELU>
__device__ __forceinline__ void gate_bwd32(float* g, float* u, float* d, int act) {
    auto out = [&](int i, float a, float da) {
        const float x = u[i];
        g[i] = d[i] * x * da;
        u[i] = d[i] * a;
        d[i] = a * x;
    };
    if constexpr (!GELU) {
        const bool silu = act == 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            // s' = e / (1 + e)^2: of s (1 - s) an open gate's s, rounded, leaves nothing
            const float x = g[i], e = __expf(-fabsf(x)), r = __fdividef(1.f, 1.f + e);
            const float s = x >= 0.f ? r : e * r, ds = e * r * r;
            out(i, silu ? x * s : s, silu ? fmaf(x, ds, s) : ds);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const float x = g[i];
            float c, bell;
            normal(x, c, bell);
            out(i, x * c, c + x * 0.39894228f * bell);
        }
    }
}

// What an epilogue does is in the instance, since a launch begins with fetching its code: with all
// of it in one, the training step of 18,000 x 128 x 512 in fp32 took 8 % longer.
enum Form { kOut = 0, kRows = 1, kPart = 2, kBlocked = 3, kGelu = 1 };     // kGelu: of gates
// The epilogue's last step on 32 columns n.. of the warp's rows m.. (m + lane is this lane's);
// v0 (and v1: the u columns of a gate).
template <int EPI, bool SPLIT, int OUT>
__device__ __forceinline__ void finish32(const CUtensorMap* maps, const Args& p, const Tile& ti, Out& o,
                                         long long m, int n, int lane, float* v0, float* v1) {
    constexpr int P = SPLIT ? kPlanes : 1;
    if (m >= p.M || n >= p.N) return;
    if constexpr (EPI == kStore || EPI == kStoreLow) {
        const int z = ti.ks * p.groups + ti.grp;
        if constexpr (OUT == kBlocked)
            store_block(lane_block(p.blocked, m, n, p.Fp, lane), v0);
        else if constexpr (OUT == kPart)
            store_f32<true>(o, lane, maps + part_map(P), n, (int)m, z, v0);
        else if constexpr (OUT == kOut && SPLIT)
            store_f32(o, lane, maps + out_map(P) + ti.grp, n, (int)m, 0, v0);
        else if constexpr (OUT == kOut)
            store_typed<false>(o, lane, maps + out_map(P) + ti.grp, n, (int)m, v0, p.dtype);
        else if (p.ksplit > 1)
            store_rows(o, lane, p.part, (z * p.M + m) * p.N + n, p.N, (int)min(32LL, p.M - m),
                       p.N - n, v0, ATOM_F32);
        else
            store_rows(o, lane, p.C[ti.grp], m * p.ldc + n, p.ldc, (int)min(32LL, p.M - m),
                       p.N - n, v0, p.dtype);
    } else if constexpr (EPI == kGate) {
        if (p.gu) {
            store_block(lane_block(p.gu, m, n, p.Fp, lane), v0);
            store_block(lane_block(p.gu, m, n, p.Fp, lane) + p.gu_half, v1);
        }
        gate32<OUT == kGelu>(v0, v1, p.act);
        store_typed<SPLIT>(o, lane, maps + out_map(P), n, (int)m, v0, p.dtype);
    } else {
        // v0, v1 = g, u (kGateBwdGU, dh from memory) or v0 = dh (kGateBwdDH, g and u from memory)
        float w[32];
        if constexpr (EPI == kGateBwdGU) {
            load_block(lane_block(p.dh, m, n, p.Fp, lane), w);
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) w[i] = v0[i];
            load_block(lane_block(p.gu, m, n, p.Fp, lane), v0);
            load_block(lane_block(p.gu, m, n, p.Fp, lane) + p.gu_half, v1);
        }
        gate_bwd32<OUT == kGelu>(v0, v1, w, p.act);
        store_typed<SPLIT>(o, lane, maps + out_map(P), n, (int)m, v0, p.dtype);
        store_typed<SPLIT>(o, lane, maps + out_map(P), p.Fp + n, (int)m, v1, p.dtype);
        if (p.H) store_typed<SPLIT>(o, lane, maps + h_map(P), n, (int)m, w, p.dtype);
    }
}

// kLow: a lane's row of the four slices that a warp has of group g, times the adapter's scale: into the
// tile's blocks (zeros where the row is of another one), and into the rows' own places.
template <bool SPLIT>
__device__ __forceinline__ void low_store(const Args& p, const Low& low, int g, int part,
                                          long long m0, int lane, int lead, float (*v)[32]) {
    const int used = low.used(g, part);
    const long long m = m0 + lane;
    const long long stage0 = first_stage(low.mt, low.first, p.ext);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (i >= used) break;
        const int3 block = low.block(g, part * 4 + i);
        const int sub = low.sub(part * 4 + i), c0 = sub * 16, slice = block.x * p.ext + sub;
        const bool in = block.z == lead;
        const float s = p.low_scale[block.y];
        float* x = v[i >> 1] + (i & 1) * 16;
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = in ? x[j] * s : 0.f;
        // the slice's 16 values of this row, in 16-bit elements
        const long long at = ((stage0 + (slice >> 2)) * 256 + (m & 255)) * 64 + (slice & 3) * 16;
#pragma unroll
        for (int h = 0; h < 2; ++h) {                // eight ranks at a time: Rs is a multiple of 8
            const int c = c0 + 8 * h;
            float* y = x + 8 * h;
            uint16_t* q = static_cast<uint16_t*>(p.low_block) + at + 8 * h;
            if constexpr (SPLIT) {
                if (p.low_rows && in && c < p.Rs) {
                    float* r = static_cast<float*>(p.low_rows) + m * p.Rs + c;
                    *reinterpret_cast<float4*>(r) = make_float4(y[0], y[1], y[2], y[3]);
                    *reinterpret_cast<float4*>(r + 4) = make_float4(y[4], y[5], y[6], y[7]);
                }
                if (!p.low_block) continue;
#pragma unroll
                for (int k = 0; k < kPlanes; ++k, q += p.low_plane)
                    *reinterpret_cast<uint4*>(q) =
                        make_uint4(take_plane(y[0], y[1], k), take_plane(y[2], y[3], k),
                                   take_plane(y[4], y[5], k), take_plane(y[6], y[7], k));
                continue;
            }
            const uint4 w = make_uint4(pair_w(y[0], y[1], p.dtype), pair_w(y[2], y[3], p.dtype),
                                       pair_w(y[4], y[5], p.dtype), pair_w(y[6], y[7], p.dtype));
            *reinterpret_cast<uint4*>(q) = w;
            if (p.low_rows && in && c < p.Rs)
                *reinterpret_cast<uint4*>(static_cast<unsigned short*>(p.low_rows) + m * p.Rs + c) = w;
        }
    }
}

template <int BN, int EPI, bool SPLIT, int OUT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Cfg<BN, EPI, SPLIT>::kThreads, 1)
    pair_kernel(const __grid_constant__ MapArray<part_map(SPLIT ? kPlanes : 1) + 1> maps,
                const __grid_constant__ Args p) {
    using CF = Cfg<BN, EPI, SPLIT>;
    constexpr int S = CF::S, P = SPLIT ? kPlanes : 1, kBufs = CF::kBufs;
    // a gate's tile: columns 0 .. BN/2 of the accumulator are g, the others u
    constexpr bool GATED = EPI == kGate || EPI == kGateBwdGU;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* outbuf = smem + S * CF::kSlot;
    uint64_t* full = reinterpret_cast<uint64_t*>(outbuf + CF::kOut);
    uint64_t* empty = full + S;
    uint64_t* accf = empty + S;      // [kBufs] accumulator full
    uint64_t* acce = accf + kBufs;   // [kBufs] and free again (CTA 0's: both CTAs' epilogue warps)
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acce + kBufs);
    int* failed = reinterpret_cast<int*>(tmem_slot + 1);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    uint32_t rank;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const int pairs = gridDim.x >> 1, first = blockIdx.x >> 1;
    let_next_start();
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < kBufs; ++b) {
            mbar_init(&accf[b], 1);
            mbar_init(&acce[b], 2 * CF::EW);
        }
        *failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2 && lane <= part_map(P) && (p.used >> lane & 1))
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.m[lane]))
                     : "memory");
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
            smem_u32(tmem_slot)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    const uint32_t base = smem_u32(smem);
    wait_before();

    if (warp == 0) {
        {
            uint32_t it = 0, slot = 0, turn = 0;
            bool ok = true;
            const uint32_t full0 = peer_addr(smem_u32(full), 0);
            // waits for a free slot and names its barrier of CTA 0
            auto open = [&](uint32_t& dst, uint32_t& bar, uint32_t bytes = CF::kSlot) {
                const uint32_t s = slot;
                if (!mbar_wait(&empty[s], turn ^ 1u, p.err)) return false;
                if (rank == 0 && elect_one())
                    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(
                                     smem_u32(&full[s])), "r"(2 * bytes) : "memory");
                dst = base + s * CF::kSlot;
                bar = full0 + s * 8;
                ++it;
                if (++slot == S) slot = 0, turn ^= 1u;
                return true;
            };
            Ahead ahead;
            uint32_t mine_k = 0;
            for (long long t = first; ok && t < p.tiles; t += pairs, ++mine_k) {
                const Tile ti = tile_of(p, t);
                const int m0 = ti.mt * 256 + rank * 128;
                int4 req = make_int4(0, 0, 0, 0);
                if (EPI == kStoreLow) {
                    req = ahead.get(p, mine_k, first, pairs);
                    if (ti.ks != p.ksplit - 1) req.z = 0;
                }
                Blocks st(p, ti.mt, req);
                if constexpr (EPI == kLow) {
                    Low low(p, ti.mt);
                    const bool mn = p.ph[0].b_mn;
                    for (int g = ti.ks; ok && g < low.groups(); g += p.ksplit) {
                        const int n = low.used(g, 0) + low.used(g, 1), mine = low.used(g, rank);
                        int slot[4], r16[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            slot[i] = i < mine ? low.block(g, 4 * rank + i).y : 0;
                            r16[i] = low.sub(4 * rank + i) * 16;
                        }
                        for (int kt = 0; ok && kt < p.ph[0].nk; ++kt) {
                            const int k0 = kt * 64;
#pragma unroll
                            for (int pl = P - 1; pl >= 0; --pl) {
                                uint32_t dst, bar;
                                if (!(ok = open(dst, bar, CF::kA + n * 1024))) break;
                                if (!elect_one()) continue;
                                tma_load(dst, &maps.m[p.ph[0].a + pl], k0, m0, bar);
#pragma unroll
                                for (int i = 0; i < 4; ++i)
                                    if (i < mine)
                                        tma_load3(dst + CF::kA + i * 2048,
                                                  &maps.m[p.ph[0].b0 + pl], mn ? r16[i] : k0,
                                                  mn ? k0 : r16[i], slot[i], bar);
                            }
                        }
                    }
                    continue;
                }
                for (int f = 0; ok && f < p.nphase; ++f) {
                    const Phase ph = p.ph[f];
                    const Share sh(p, ti, f);
                    const int n0 = ti.nt * ph.bstep + rank * ph.brank;
                    const CUtensorMap* ma = &maps.m[ph.a + P * ti.grp];
                    const CUtensorMap* mb = &maps.m[rank ? ph.b1 : ph.b0];
                    for (int kt = sh.kt; ok && kt < sh.end; ++kt) {
                        const int k0 = kt * 64;
#pragma unroll
                        for (int pl = P - 1; pl >= 0; --pl) {
                            uint32_t da, bar;
                            if (!(ok = open(da, bar))) break;
                            if (!elect_one()) continue;
                            const uint32_t db = da + CF::kA;
                            if (ph.a_mn) {
                                tma_load(da, ma + pl, m0, k0, bar);
                                tma_load(da + 8192, ma + pl, m0 + 64, k0, bar);
                            } else {
                                tma_load(da, ma + pl, k0, m0, bar);
                            }
                            if (ph.b_mn) {
#pragma unroll
                                for (int j = 0; j < CF::HB / 64; ++j)
                                    tma_load(db + j * 8192, mb + pl, n0 + 64 * j, k0, bar);
                            } else {
                                tma_load(db, mb + pl, k0, n0, bar);
                            }
                        }
                    }
                }
                if constexpr (EPI != kStoreLow) continue;
                const int n0 = ti.nt * BN + rank * CF::HB;
                long long y = first_stage(ti.mt, req.x, p.ext) * 256 + rank * 128;
                for (; ok; y += 256) {
                    int slots[4], ks[4], n = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (n == i && st.next()) slots[i] = st.slot, ks[i] = st.at(), ++n;
                    if (n == 0) break;
#pragma unroll
                    for (int pl = P - 1; pl >= 0; --pl) {
                        uint32_t dst, bar;
                        if (!(ok = open(dst, bar, CF::kA + n * (CF::kB / 4)))) break;
                        if (!elect_one()) continue;
                        tma_load(dst, &maps.m[p.ext_a + pl], 0, (int)y, bar);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (i >= n) break;
                            const uint32_t db = dst + CF::kA + i * (CF::kB / 4);
                            const CUtensorMap* mb = &maps.m[p.ext_b + pl];
                            if (p.ext_bmn) {
#pragma unroll
                                for (int j = 0; j < CF::HB / 64; ++j)
                                    tma_load3(db + j * 2048, mb, n0 + 64 * j, ks[i], slots[i], bar);
                            } else {
                                tma_load3(db, mb, ks[i], n0, slots[i], bar);
                            }
                        }
                    }
                }
            }
            // the last slots are read before this CTA may end
            for (uint32_t k = it > S ? it - S : 0; ok && k < it; ++k)
                ok = mbar_wait(&empty[k % S], (k / S) & 1u, p.err);
            if (!ok) *(volatile int*)failed = 1;
        }
    } else if (warp == 1) {
        if (rank == 0) {
            uint32_t slot = 0, turn = 0, round = 0;
            bool ok = true, open = false;
            uint32_t acc = 0, fresh = 0;
            const uint64_t base_k = sdesc(base, 0), base_mn = sdesc(base, 1);
            auto begin = [&]() {         // a free accumulator for the next round
                const uint32_t b = round % kBufs;
                if (!mbar_wait(&acce[b], ((round / kBufs) & 1u) ^ 1u, p.err)) return false;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                acc = tmem + b * BN;
                fresh = 0;
                return open = true;
            };
            auto end = [&]() {
                if (elect_one()) mma_commit(&accf[round % kBufs]);
                ++round;
                open = false;
            };
            // One stage's products (SPLIT: a round of their own). Descriptors only add to their address
            // field: one thread issues a product every ~40 clocks this way, against ~160 building each
            // anew, which had bound the whole kernel (a product of 256 x 256 x 16 takes 128 clocks).
            auto stage = [&](uint64_t a, uint64_t b, uint32_t as, uint32_t bs, uint32_t id,
                             int steps) {
                if (!open && !begin()) return false;
                uint64_t at[P], bt[P], *done[P];
#pragma unroll
                for (int pl = P - 1; pl >= 0; --pl) {
                    if (!mbar_wait(&full[slot], turn, p.err)) return false;
                    at[pl] = a + slot * (CF::kSlot >> 4);
                    bt[pl] = b + slot * (CF::kSlot >> 4);
                    done[pl] = &empty[slot];
                    if (++slot == S) slot = 0, turn ^= 1u;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (elect_one()) {
                    auto product = [&](int i, int j) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (k < steps) {
                                mma(acc, at[i] + k * as, bt[j] + k * bs, id, k ? 1u : fresh);
                                fresh = 1;
                            }
                    };
                    if constexpr (SPLIT) {
                        product(2, 0);
                        product(0, 2);
                        mma_commit(done[2]);
                        product(1, 1);
                        product(1, 0);
                        product(0, 1);
                        mma_commit(done[1]);
                    }
                    product(0, 0);
                    mma_commit(done[0]);
                }
                __syncwarp();
                fresh = 1;
                if constexpr (SPLIT) end();
                return true;
            };
            Ahead ahead;
            uint32_t mine_k = 0;
            for (long long t = first; ok && t < p.tiles; t += pairs, ++mine_k) {
                const Tile ti = tile_of(p, t);
                int left = 0;
                if (EPI == kStoreLow) {
                    left = ahead.get(p, mine_k, first, pairs).z * p.ext;
                    if (ti.ks != p.ksplit - 1) left = 0;
                }
                if constexpr (EPI == kLow) {
                    const int groups = Low(p, ti.mt).groups(), mn = p.ph[0].b_mn;
                    const uint64_t b = mn ? sdesc_low(base + CF::kA) : base_k + (CF::kA >> 4);
                    const uint32_t id = idesc(BN, SPLIT ? 1 : p.bf16, 0, mn);
                    for (int g = ti.ks; ok && g < groups; g += p.ksplit) {
                        for (int kt = 0; ok && kt < p.ph[0].nk; ++kt)
                            ok = stage(base_k, b, 32 >> 4, mn ? 512 >> 4 : 32 >> 4, id, 4);
                        if (ok && open) end();
                    }
                    continue;
                }
                for (int f = 0; ok && f < p.nphase; ++f) {
                    const int a_mn = p.ph[f].a_mn, b_mn = p.ph[f].b_mn;
                    const Share sh(p, ti, f);
                    const uint64_t a = a_mn ? base_mn : base_k;
                    const uint64_t b = (b_mn ? base_mn : base_k) + (CF::kA >> 4);
                    const uint32_t as = a_mn ? 2048 >> 4 : 32 >> 4, bs = b_mn ? 2048 >> 4 : 32 >> 4;
                    const uint32_t id = idesc(BN, SPLIT ? 1 : p.bf16, a_mn, b_mn);
                    for (int kt = sh.kt; ok && kt < sh.end; ++kt) ok = stage(a, b, as, bs, id, 4);
                }
                if constexpr (EPI == kStoreLow) {
                    const uint64_t b = sdesc_slice(base + CF::kA, p.ext_bmn);
                    const uint32_t id = idesc(BN, SPLIT ? 1 : p.bf16, 0, p.ext_bmn);
                    for (; ok && left > 0; left -= 4)
                        ok = stage(base_k, b, 32 >> 4, CF::kB >> 6, id, min(4, left));
                }
                if (ok && open) end();
            }
            if (!ok) *(volatile int*)failed = 1;
        }
    } else {
        const int q = warp & 3, part = (warp - 2) >> 2;     // rows' quarter, columns' share
        const uint32_t lanes = (uint32_t)(q * 32) << 16;
        uint32_t round = 0;
        const uint32_t acce0 = peer_addr(smem_u32(acce), 0);
        // This warp has read the round's accumulators. Relaxed: only tensor memory is handed over,
        // which the fence orders; a release would wait for this warp's stores to memory as well.
        auto drained = [&]() {
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0)
                asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(
                                 acce0 + 8 * (round % kBufs)) : "memory");
            ++round;
        };
        auto filled = [&]() {
            const bool ok = __all_sync(0xffffffffu,
                                       mbar_wait(&accf[round % kBufs], (round / kBufs) & 1u, p.err));
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            return ok;
        };
        // first column of this warp's k-th 32-column chunk (of g, for a gate; u: BN/2 further)
        constexpr int kChunks = (GATED ? BN / 2 : BN) / (CF::EW / 4) / 32;
        const int c0 = part * kChunks * 32;
        bool ok = true;
        Out out{outbuf + (warp - 2) * 4096, 0};
        constexpr int kParts = GATED ? 2 * kChunks : kChunks;
        Ahead ahead;
        uint32_t mine_k = 0;
        for (long long t = first; ok && t < p.tiles; t += pairs, ++mine_k) {
            const Tile ti = tile_of(p, t);
            const long long m = (long long)ti.mt * 256 + rank * 128 + q * 32;
            const int nb = ti.nt * (GATED ? BN / 2 : BN) + c0;
            int4 req = make_int4(0, 0, 0, 0);
            if (EPI == kStoreLow) req = ahead.get(p, mine_k, first, pairs);
            const bool spoilt = EPI == kStoreLow && req.w && spoilt_row(p, ti.mt, m + lane, lane);
            if (EPI == kLow && warp == 2 && rank == 0 && ti.ks == 0 && p.usable)
                settle(p, ti.mt);
            if constexpr (EPI == kLow && !SPLIT) {
                const int lead = m + lane < p.M ? p.row_lead[m + lane] : -1;
                Low low_(p, ti.mt);
                for (int g = ti.ks; g < low_.groups(); g += p.ksplit) {
                    if (!(ok = filled())) break;
                    const uint32_t ta = tmem + lanes + (round % kBufs) * BN + c0;
                    float v[2][32];
                    tmem_ld32(ta, v[0]);
                    tmem_ld32(ta + 32, v[1]);
                    tmem_wait_ld();
                    pin32(v[0]);
                    pin32(v[1]);
                    drained();
                    low_store<SPLIT>(p, low_, g, part, m, lane, lead, v);
                }
            } else if constexpr (!SPLIT) {
                if (!(ok = filled())) break;
                const uint32_t ta = tmem + lanes + (round % kBufs) * BN + c0;
#pragma unroll 1
                for (int k = 0; k < kChunks; ++k) {
                    float v0[32], v1[32];
                    tmem_ld32(ta + 32 * k, v0);
                    if (GATED) tmem_ld32(ta + BN / 2 + 32 * k, v1);
                    tmem_wait_ld();
                    pin32(v0);
                    if (GATED) pin32(v1);
                    if (k == kChunks - 1) drained();
                    if (EPI == kStoreLow && spoilt) spoil32(v0);
                    finish32<EPI, SPLIT, OUT>(maps.m, p, ti, out, m, nb + 32 * k, lane, v0, v1);
                }
            } else {
                // the tile's rounds summed in registers
                float v[kParts][32];
                auto clear = [&]() {
#pragma unroll
                    for (int k = 0; k < kParts; ++k)
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[k][i] = 0.f;
                };
                clear();
                auto column = [&](int k) {
                    return GATED ? (k / kChunks) * (BN / 2) + (k % kChunks) * 32 : 32 * k;
                };
                auto add = [&](int rounds) {
                    for (int r = 0; r < rounds; ++r) {
                        if (!filled()) return false;
                        const uint32_t ta = tmem + lanes + (round % kBufs) * BN + c0;
                        float x[2][32];
#pragma unroll
                        for (int k = 0; k < kParts; ++k) tmem_ld32(ta + column(k), x[k]);
                        tmem_wait_ld();
#pragma unroll
                        for (int k = 0; k < kParts; ++k) pin32(x[k]);
                        drained();
#pragma unroll
                        for (int k = 0; k < kParts; ++k)
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[k][i] += x[k][i];
                    }
                    return true;
                };
                static_assert(!SPLIT || kParts == 2, "parts of a SPLIT tile");
                if constexpr (EPI == kLow) {
                    const int lead = m + lane < p.M ? p.row_lead[m + lane] : -1;
                    Low low_(p, ti.mt);
                    for (int g = ti.ks; g < low_.groups(); g += p.ksplit) {
                        clear();
                        if (!(ok = add(p.ph[0].nk))) break;
                        low_store<SPLIT>(p, low_, g, part, m, lane, lead, v);
                    }
                    if (!ok) break;
                    continue;
                }
                int stages = 0;
                for (int f = 0; f < p.nphase; ++f) {
                    const Share sh(p, ti, f);
                    stages += sh.end - sh.kt;
                }
                if (EPI == kStoreLow && ti.ks == p.ksplit - 1) stages += (req.z * p.ext + 3) >> 2;
                if (!(ok = add(stages))) break;
#pragma unroll
                for (int k = 0; k < kChunks; ++k) {
                    float u[32];         // kGateBwdDH: room for the u that it reads
                    if (EPI == kStoreLow && spoilt) spoil32(v[k]);
                    finish32<EPI, SPLIT, OUT>(maps.m, p, ti, out, m, nb + 32 * k, lane, v[k],
                                              GATED ? v[kChunks + k] : u);
                }
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        if (!ok && lane == 0) *(volatile int*)failed = 1;
    }
    __syncthreads();
    if (*(volatile int*)failed) {        // copies and products in flight end within microseconds
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000) {
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    cluster_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}


// C[g][m, n] = sum over the splits, in order. Split products are small (fewer tiles than pairs of
// SMs), so 32-bit indexes do.
__global__ void __launch_bounds__(256) reduce_kernel(const __grid_constant__ Sums sums) {
    let_next_start();
    wait_before();
    const Sums::Item& p = sums.it[blockIdx.y];
    const uint32_t N = p.N, all = p.M * N * p.groups;
    const uint32_t step = N % 4 ? 1 : 4;
    for (uint32_t i = (blockIdx.x * 256u + threadIdx.x) * step; i < all; i += gridDim.x * 256u * step) {
        float v[4] = {};
        if (step == 4) {
#pragma unroll 4
            for (int s = 0; s < p.ksplit; ++s) {
                const float4 x = *reinterpret_cast<const float4*>(p.part + (long long)s * all + i);
                v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
            }
        } else {
#pragma unroll 4
            for (int s = 0; s < p.ksplit; ++s) v[0] += p.part[(long long)s * all + i];
        }
        const uint32_t row = i / N, n = i - row * N, g = row >= p.M;
        const long long at = (row - g * p.M) * p.ldc + n;
        for (uint32_t j = 0; j < step; ++j) store_f(p.C[g], at + j, v[j], sums.dtype);
    }
}
int add_up(Sums& sums, Chain& st) {
    long long blocks = 0;
    for (int i = 0; i < sums.n; ++i) {
        const Sums::Item& p = sums.it[i];
        blocks = std::max(blocks, ((long long)p.M * p.N * p.groups / (p.N % 4 ? 1 : 4) + 255) / 256);
    }
    if (sums.n == 0) return ATOM_OK;
    const int s = st.launch("pair product sums", reduce_kernel,
                            dim3((unsigned)std::min(blocks, 1184LL), sums.n), 256, 0, sums);
    sums.n = 0;
    return s;
}

// Operand preparation. A warp has eight float4 a lane: one row of up to 1024 columns, two, four or
// eight narrower ones, so that narrow rows keep as much in flight, or 1024 columns of a wider one.
// Planes and packed rows are zero past the row's end up to the pitch. Bound by memory: planes of
// 18,000 x 1,536 values take 42 us, 6.6 TB/s read and written.
constexpr int kNV = 8;
__host__ __device__ inline int prep_slots(const PrepItem& it) {      // float4 a lane of one row
    return it.dld <= 128 ? 1 : it.dld <= 256 ? 2 : it.dld <= 512 ? 4 : 8;
}
__host__ __device__ inline int prep_chunks(const PrepItem& it) {     // warps a row
    return (int)((it.dld + 1023) / 1024);
}
__device__ __forceinline__ void prep_split(const PrepItem& it, int blocks) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int nv = prep_slots(it), rows = kNV / nv, shift = 31 - __clz(nv), chunks = prep_chunks(it);
    const int cols = (int)it.cols, dld = (int)it.dld;
    const long long units = (it.rows + rows - 1) / rows * chunks;
    const bool four = aligned16(it.src) && it.ld % 4 == 0 && cols % 4 == 0;
    for (long long u = blockIdx.x * 8LL + warp; u < units; u += blocks * 8LL) {
        const long long r0 = chunks == 1 ? u * rows : u / chunks;
        const int c0 = chunks == 1 ? 0 : (int)(u - r0 * chunks) * 1024;
        const float* src = static_cast<const float*>(it.src) + r0 * it.ld;
        float4 x[kNV];
        // slot j: row r0 + j / nv, columns c0 + 4 (j % nv * 32 + lane) ..
#pragma unroll
        for (int j = 0; j < kNV; ++j) {
            const int i = j >> shift, c = c0 + (((j & (nv - 1)) << 5) + lane) * 4;
            const int end = r0 + i < it.rows ? cols : 0;
            const float* q = src + i * it.ld + c;
            if (four)
                x[j] = c < end ? *reinterpret_cast<const float4*>(q) : make_float4(0.f, 0.f, 0.f, 0.f);
            else
                x[j] = make_float4(c < end ? q[0] : 0.f, c + 1 < end ? q[1] : 0.f,
                                   c + 2 < end ? q[2] : 0.f, c + 3 < end ? q[3] : 0.f);
        }
#pragma unroll
        for (int j = 0; j < kNV; ++j) {
            const int i = j >> shift, c = c0 + (((j & (nv - 1)) << 5) + lane) * 4;
            if (r0 + i >= it.rows || c >= dld) continue;
            uint16_t* q = static_cast<uint16_t*>(it.dst) + (r0 + i) * dld + c;
#pragma unroll
            for (int k = 0; k < kPlanes; ++k, q += it.plane)
                *reinterpret_cast<uint2*>(q) =
                    make_uint2(take_plane(x[j].x, x[j].y, k), take_plane(x[j].z, x[j].w, k));
        }
    }
}

// 16-bit rows to an aligned pitch; eight single loads in flight, then eight stores.
__device__ __forceinline__ void prep_pack(const PrepItem& it, int blocks) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int cols = (int)it.cols, dld = (int)it.dld;
    for (long long r = blockIdx.x * 8LL + warp; r < it.rows; r += blocks * 8LL) {
        const unsigned short* src = static_cast<const unsigned short*>(it.src) + r * it.ld;
        unsigned short* dst = static_cast<unsigned short*>(it.dst) + r * dld;
        for (int c0 = 0; c0 < dld; c0 += 256) {
            unsigned short v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = c0 + j * 32 + lane < cols ? src[c0 + j * 32 + lane] : 0;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c0 + j * 32 + lane < dld) dst[c0 + j * 32 + lane] = v[j];
        }
    }
}

// Finds pieces: a piece a warp, a row tile a warp, then four blocks an adapter.
__device__ __forceinline__ void find_pieces(const Pieces& p) {
    __shared__ unsigned seen[8][1 << 14 >> 5];       // adapters, of a warp's tile
    const int lane = threadIdx.x & 31, w = blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lookups = (p.pieces + p.tiles + 7) / 8;
    // rows are kept within 0 .. M whatever the table holds
    auto begins = [&](int r) { return min(::max(p.ptr[r], 0), p.M); };
    if (blockIdx.x < lookups) {
        if (w < p.pieces) {
            // t + r grows with r at each request's first tile t: the last request at or before w
            const int r = last_le(p.n, w, [&](int i) { return begins(i) / 256 + i; });
            int4 c = make_int4(-1, 0, 0, 0);
            if (r >= 0 && w - r < p.tiles) {
                const int m0 = (w - r) * 256, a = p.adapter[r];
                c.y = ::max(begins(r), m0);
                c.z = min(begins(r + 1), m0 + 256);
                if (c.y < c.z && a >= 0 && a < p.nad) c.x = a;
            }
            // The requests of a tile that share an adapter share a block: the first of them among
            // 256 numbers leads it (156 rows of 153 requests, 3 adapters, 16 ranks, forward
            // and backward: 115 us with a block a request, 65 us so).
            int lead = r;
            const int t = w - r;
            if (c.x >= 0) {
                int got = r;
#pragma unroll
                for (int j = 7; j >= 0; --j) {
                    const int q = (r & ~255) + 32 * j + lane;
                    if (q < r && p.adapter[q] == c.x &&
                        ::max(begins(q), t * 256) < min(begins(q + 1), t * 256 + 256))
                        got = q;
                }
                lead = __reduce_min_sync(0xffffffffu, got);
            }
            if (lane == 0) p.piece[w] = c;
            for (int m = c.y + lane; m < c.z; m += 32) p.row_lead[m] = c.x < 0 ? -1 : lead;
        } else if (w < p.pieces + p.tiles) {
            const int t = w - p.pieces;
            const int first = last_le(p.n, t * 256, begins);
            const int last = last_le(p.n, t * 256 + 255, begins);
            const int head = begins(0), tail = begins(p.n);
            for (int m = t * 256 + lane; m < min(p.M, t * 256 + 256); m += 32)
                if (m < head || m >= tail) p.row_lead[m] = -1;
            // The tile's blocks in order: of each 256 numbers, the first requests with an adapter. (A
            // request that begins before the tile reaches into it at most as the last such one.)
            unsigned* bits = seen[threadIdx.x >> 5];
            int n = 0;
            for (int r0 = ::max(first, 0) & ~31; r0 <= last; r0 += 32) {
                const int r = r0 + lane;
                if (r0 <= ::max(first, 0) || (r0 & 255) == 0) {
                    __syncwarp();
                    for (int i = lane; i < (p.nad + 31) / 32; i += 32) bits[i] = 0;
                    __syncwarp();
                }
                int a = -1;
                if (r >= first && r >= 0 && r <= last && p.adapter[r] < p.nad &&
                    ::max(begins(r), t * 256) < min(begins(r + 1), t * 256 + 256))
                    a = p.adapter[r];
                const unsigned same = __match_any_sync(0xffffffffu, a);
                const bool leads = a >= 0 && __ffs(same) - 1 == lane && !(bits[a >> 5] >> (a & 31) & 1);
                const unsigned all = __ballot_sync(0xffffffffu, leads);
                if (leads) {
                    atomicOr(&bits[a >> 5], 1u << (a & 31));
                    p.lead[t + ::max(first, 0) + n + __popc(all & ((1u << lane) - 1))] =
                        make_int2(a, r);
                }
                n += __popc(all);
                __syncwarp();
            }
            if (lane == 0) p.tile_req[t] = make_int4(::max(first, 0), last + 1, n, 0);
        }
        return;
    }
    const int a = (blockIdx.x - lookups) >> 2, part = (blockIdx.x - lookups) & 3;
    if (!p.other || a >= p.nad) return;
    int found = 0;
    const long long lo = p.other_n * part / 4, hi = p.other_n * (part + 1) / 4;
    const long long at = (long long)a * p.other_n;
    if (p.dtype == ATOM_F32) {
        const unsigned* v = static_cast<const unsigned*>(p.other) + at;
#pragma unroll 16
        for (long long i = lo + threadIdx.x; i < hi; i += 256)
            found |= (v[i] & 0x7F800000u) == 0x7F800000u;
    } else {
        const unsigned short top = p.dtype == ATOM_BF16 ? 0x7F80 : 0x7C00;
        const unsigned short* v = static_cast<const unsigned short*>(p.other) + at;
        long long i = lo + threadIdx.x;
        if ((reinterpret_cast<uintptr_t>(v + lo) & 15) == 0) {
            const unsigned two = top * 0x10001u;
            const long long n8 = (hi - lo) / 8;
#pragma unroll 8
            for (long long j = threadIdx.x; j < n8; j += 256) {
                const uint4 x = *reinterpret_cast<const uint4*>(v + lo + 8 * j);
                const unsigned w4[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    found |= (w4[k] & top) == top || ((w4[k] & two) >> 16) == top;
            }
            i = lo + 8 * n8 + threadIdx.x;
        }
        for (; i < hi; i += 256) found |= (v[i] & top) == top;
    }
    found = __syncthreads_or(found);
    if (threadIdx.x == 0) reinterpret_cast<int*>(p.bad + a)[part] = found;
}

// SPLIT: planes, else 16-bit copies. FINDS: and an adapters call's pieces. Small operands are prepared
// in the time of a launch and of their code's first fetch, so each has an instance.
template <bool SPLIT, bool FINDS>
__global__ void __launch_bounds__(256, 3)
    prep_kernel(const __grid_constant__ PrepList l, const __grid_constant__ Pieces pieces) {
    let_next_start();
    wait_before();
    if constexpr (FINDS)
        if (blockIdx.y == l.n) {
            find_pieces(pieces);
            return;
        }
    const int blocks = l.blocks[blockIdx.y];
    if (blockIdx.x >= blocks) return;
    if constexpr (SPLIT) prep_split(l.it[blockIdx.y], blocks);
    else prep_pack(l.it[blockIdx.y], blocks);
}

int prepare(PrepList& l, Chain& st, const Pieces* pieces) {
    if (l.n == 0 && !pieces) return ATOM_OK;
    int grid = 1;
    bool split = false;              // a list is of one type
    for (int i = 0; i < l.n; ++i) {
        const PrepItem& it = l.it[i];
        split = it.mode == kSplit;
        const int rows = split ? kNV / prep_slots(it) : 1, chunks = split ? prep_chunks(it) : 1;
        const long long warps = (it.rows + rows - 1) / rows * chunks;
        l.blocks[i] = (int)std::max(1LL, std::min((warps + 7) / 8, (long long)kPrepBlocks));
        grid = std::max(grid, l.blocks[i]);
    }
    Pieces none{};
    if (pieces)
        grid = std::max(grid, (pieces->pieces + pieces->tiles + 7) / 8 +
                                  (pieces->other ? 4 * pieces->nad : 0));
    const int s = st.launch("operand preparation",
                            split ? pieces ? prep_kernel<true, true> : prep_kernel<true, false>
                                  : pieces ? prep_kernel<false, true> : prep_kernel<false, false>,
                            dim3(grid, l.n + (pieces != nullptr)), 256, 0, l,
                            pieces ? *pieces : none);
    l.n = 0;
    return s;
}

static PFN_cuTensorMapEncodeTiled_v12000 encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) !=
                cudaSuccess || q != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    }();
    return fn;
}

static int encode_map(CUtensorMap* m, const void* p, bool f32, long long cols, long long rows,
                      long long depth, long long ld, long long ldz, int box_cols, int box_rows,
                      CUtensorMapSwizzle swizzle) {
    const auto encode = encoder();
    if (!encode) {
        set_error("cuTensorMapEncodeTiled unavailable");
        return ATOM_ERR_CUDA;
    }
    const int e = f32 ? 4 : 2;
    cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)depth};
    cuuint64_t strides[2] = {(cuuint64_t)ld * e, (cuuint64_t)ldz * e};
    cuuint32_t box[3] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = encode(m, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : CU_TENSOR_MAP_DATA_TYPE_UINT16, depth ? 3 : 2,
                              const_cast<void*>(p), dims, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("cuTensorMapEncodeTiled failed (%d): %lld x %lld, ld %lld", (int)r, rows, cols, ld);
        return ATOM_ERR_ARG;
    }
    return ATOM_OK;
}
int make_map(CUtensorMap* m, const void* p, long long cols, long long rows, long long ld,
             int box_rows) {
    return encode_map(m, p, false, cols, rows, 0, ld, 0, 64, box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}
int make_slice_map(CUtensorMap* m, const void* p, long long cols, long long rows, long long ld,
                   int box_rows, bool mn, int depth, long long ldz) {
    return mn ? encode_map(m, p, false, cols, rows, depth, ld, ldz, 64, 16,
                           CU_TENSOR_MAP_SWIZZLE_128B)
              : encode_map(m, p, false, cols, rows, depth, ld, ldz, 16, box_rows,
                           CU_TENSOR_MAP_SWIZZLE_32B);
}
int make_low_map(CUtensorMap* m, const void* p, long long cols, long long rows, long long ld, bool mn,
                 int depth, long long ldz) {
    return mn ? encode_map(m, p, false, cols, rows, depth, ld, ldz, 16, 64,
                           CU_TENSOR_MAP_SWIZZLE_32B)
              : encode_map(m, p, false, cols, rows, depth, ld, ldz, 64, 16,
                           CU_TENSOR_MAP_SWIZZLE_128B);
}
int make_out_map(CUtensorMap* m, const void* p, int dtype, long long cols, long long rows,
                 long long ld) {
    const bool f32 = dtype == ATOM_F32;
    return encode_map(m, p, f32, cols, rows, 0, ld, 0, 32, 32,
                      f32 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

int pair_count() {
    static std::atomic<int> count[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 74;
    int n = count[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) n = 148;
        count[dev].store(n, std::memory_order_relaxed);
    }
    return n / 2;
}

// The tile width and split that a count of clocks prefers: rounds of work items over the SM
// pairs, each a tile's stages (512 clocks of tensor work at width 256, 256 at 128 but fed no
// faster than ~300; SPLIT 24 products of 64) and its fill and drain, and for a split the pass
// over the partial sums. Width 256 against 128: 60,000 x 256 x 1,024 bf16 forward 91 and 103 us,
// 8,192 x 2,048 x 8,192 559 and 622; splits against none: 18,000 x 128 x 512 fp32 backward 159 and
// 582 us, 200 x 1,024 x 4,096 bf16 forward 16.7 and 19.7.
Choice choose(long long M, int N, int nk, int groups, bool gated, bool split, bool may_split) {
    const int pairs = pair_count();
    const long long mt = (M + 255) / 256 * groups;
    Choice best{128, 1, 0};
    double least = 1e30;
    for (int bn : {256, 128}) {
        if (split && bn == 256) continue;
        const int w = gated ? bn / 2 : bn;
        const long long tiles = mt * ((N + w - 1) / w);
        const double stage = split ? 1600 : bn == 256 ? 530 : 310;
        for (int ks = 1; ks <= 32 && ks * 2 <= nk + 1; ++ks) {
            if (ks > 1 && (!may_split || tiles >= pairs)) break;
            const double fill = 2500 + (split || bn == 256 ? 1200 : 600);
            double t = (double)((tiles * ks + pairs - 1) / pairs) * ((nk + ks - 1) / ks * stage) + fill;
            if (ks > 1) t += 5000 + (double)ks * groups * M * N * 8 / 2500;
            if (t < least * 0.999) {
                least = t;
                best = {bn, ks, ks > 1 ? (size_t)ks * groups * M * N : 0};
            }
        }
    }
    return best;
}

template <int BN, int EPI, bool SPLIT, int OUT>
static int run(const Maps& maps, const Args& p, Chain& st, Sums& sums) {
    using CF = Cfg<BN, EPI, SPLIT>;
    static std::atomic<bool> set[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !set[dev].load(std::memory_order_relaxed)) {
        const cudaError_t e = cudaFuncSetAttribute(
            pair_kernel<BN, EPI, SPLIT, OUT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
            (int)CF::kSmem);
        if (e != cudaSuccess) {
            set_error("pair product: cannot reserve %u bytes of shared memory: %s", CF::kSmem,
                      cudaGetErrorString(e));
            return ATOM_ERR_CUDA;
        }
        if (dev >= 0 && dev < 64) set[dev].store(true, std::memory_order_relaxed);
    }
    const long long pairs = pair_count();
    const int grid = 2 * (int)(p.tiles < pairs ? p.tiles : pairs);
    MapArray<part_map(SPLIT ? kPlanes : 1) + 1> its;
    memcpy(&its, &maps, sizeof(its));
    if (int s = st.launch("pair product", pair_kernel<BN, EPI, SPLIT, OUT>, dim3(grid), CF::kThreads,
                          CF::kSmem, its, p))
        return s;
    if (EPI != kLow && p.ksplit > 1) {
        sums.dtype = p.dtype;
        sums.it[sums.n++] = {p.part, (uint32_t)p.M, (uint32_t)p.N, (uint32_t)p.groups, p.ksplit,
                             {p.C[0], p.C[1]}, p.ldc};
    }
    return ATOM_OK;
}

int launch(int epilogue, const Choice& c, bool split, Maps& maps, Args& p, Chain& st, Sums& sums) {
    const bool gated = epilogue == kGate || epilogue == kGateBwdGU;
    const int w = gated ? c.bn / 2 : c.bn;
    p.mtiles = ceil_div(p.M, 256);
    p.ntiles_n = ceil_div(p.N, w);
    p.ksplit = c.ksplit;
    p.tiles = (long long)p.mtiles * p.groups * p.ntiles_n * p.ksplit;
    p.err = device_error_word();
    if (!p.err) {
        set_error("pair product: no error word on this device");
        return ATOM_ERR_CUDA;
    }
    if (p.tiles >= (1LL << 31)) {
        set_error("pair product: too many tiles");
        return ATOM_ERR_CAPACITY;
    }
    if (p.tiles == 0) return ATOM_OK;
    if (epilogue == kLow)
        return split ? run<128, kLow, true, kOut>(maps, p, st, sums)
                     : run<128, kLow, false, kOut>(maps, p, st, sums);
    if ((epilogue == kStore || epilogue == kStoreLow) && !p.blocked) {
        // TMA stores clip at 16 bytes, so columns have to end there too
        const int planes = split ? kPlanes : 1, part = part_map(planes), out = out_map(planes);
        const int e = p.ksplit > 1 ? 4 : dtype_size(p.dtype);
        p.tma = p.N * e % 16 == 0;
        for (int g = 0; g < p.groups && p.ksplit == 1; ++g)
            p.tma = p.tma && aligned16(p.C[g]) && p.ldc * e % 16 == 0;
        if (p.tma && p.ksplit > 1) {
            p.used |= 1u << part;
            if (int s = encode_map(&maps.m[part], p.part, true, p.N, p.M, p.ksplit * p.groups,
                                   p.N, p.M * p.N, 32, 32, CU_TENSOR_MAP_SWIZZLE_128B))
                return s;
        }
        for (int g = 0; p.tma && p.ksplit == 1 && g < p.groups; ++g) {
            p.used |= 1u << (out + g);
            if (int s = make_out_map(&maps.m[out + g], p.C[g], p.dtype, p.N, p.M, p.ldc))
                return s;
        }
    }
    const int form = gated || epilogue == kGateBwdDH ? (p.act == 2 ? kGelu : kOut)
                     : p.blocked                     ? kBlocked
                     : !p.tma                        ? kRows
                     : p.ksplit > 1                  ? kPart : kOut;
#define ATOM_PAIR(E, O)                                            \
    if (epilogue == E && form == O) {                              \
        if (split) return run<128, E, true, O>(maps, p, st, sums);       \
        return c.bn == 256 ? run<256, E, false, O>(maps, p, st, sums)    \
                           : run<128, E, false, O>(maps, p, st, sums);   \
    }
    ATOM_PAIR(kStore, kOut)
    ATOM_PAIR(kStore, kRows)
    ATOM_PAIR(kStore, kPart)
    ATOM_PAIR(kStore, kBlocked)
    ATOM_PAIR(kStoreLow, kOut)
    ATOM_PAIR(kStoreLow, kRows)
    ATOM_PAIR(kStoreLow, kPart)
    ATOM_PAIR(kGate, kOut)
    ATOM_PAIR(kGate, kGelu)
    ATOM_PAIR(kGateBwdGU, kOut)
    ATOM_PAIR(kGateBwdGU, kGelu)
    ATOM_PAIR(kGateBwdDH, kOut)
    ATOM_PAIR(kGateBwdDH, kGelu)
#undef ATOM_PAIR
    return ATOM_ERR_UNSUPPORTED;
}

// Test hook: one thread waits, as the products do, on a barrier that nothing arrives on.
__global__ void wait_selftest_kernel(long long budget, int* err) {
    __shared__ uint64_t b;
    mbar_init(&b, 1);
    mbar_wait(&b, 0, err, budget);
}

}  // namespace pair
}  // namespace atom

extern "C" int atom_pair_wait_selftest(int64_t budget_cycles, void* stream) {
    using namespace atom;
    ATOM_REQUIRE(budget_cycles > 0 && budget_cycles <= pair::kWaitCycles,
                 "atom_pair_wait_selftest: budget_cycles must be in [1, %lld]", pair::kWaitCycles);
    int* err = device_error_word();
    ATOM_REQUIRE(err, "atom_pair_wait_selftest: no device error word");
    pair::wait_selftest_kernel<<<1, 1, 0, (cudaStream_t)stream>>>(budget_cycles, err);
    return check_launch("atom_pair_wait_selftest");
}
