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
// of B's, CTA 1 the others. Accumulators are fp32 in tensor memory, two buffers, so that the
// epilogue of one tile runs beside the products of the next.
//
// fp32 operands (SPLIT) come as two fp16 planes: x = (hi + lo 2^-11) / s with s a power of two
// per row or per tensor (22 significant bits for what lies within 2^-28 of the largest entry),
// and hi hi + 2^-11 (hi lo + lo hi) is kept in two accumulators. The tensor core rounds every
// addition toward zero, some 2^-24 of the sum a step, so a SPLIT tile is drained into registers
// (added there to nearest) every kRound stages: 8 additions, which holds an fp32 result near 5e-7
// of itself (2-norm) at any K; one accumulator at K = 1024 is 3.5e-6 off, 16 additions 9.7e-7.
//
// 320 threads: warp 0 TMA, warp 1 tensor memory and the products (CTA 0's issues for both), warps
// 2..9 the epilogue. Every wait is bounded: on expiry the kernel records a code, lets copies in
// flight land, frees its tensor memory and returns.
#include <cudaTypedefs.h>

#include "pair_product.cuh"

namespace atom {
namespace pair {

constexpr int kThreads = 320;
constexpr int kRound = 2;                            // stages between two drains of a SPLIT tile
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
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(smem_u32(b)), "r"(parity) : "memory");
    return ok != 0;
}
// Bounded wait; false once the budget is spent or any CTA has failed.
__device__ __forceinline__ bool mbar_wait(uint64_t* b, uint32_t parity, int* err) {
    if (mbar_try(b, parity)) return true;
    const long long t0 = clock64();
    while (!mbar_try(b, parity)) {
        if (clock64() - t0 > kWaitCycles) {
            atomicCAS(err, 0, ATOM_PAIR_WAIT_CODE);
            return false;
        }
        if (*(volatile int*)err != 0) return false;
    }
    return true;
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
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

struct Tile {
    int mt, nt, grp, ks;
};
// Work item -> tile. Eight row tiles by all column tiles at a time, so that the pairs at work
// share both operands' tiles in L2.
__device__ __forceinline__ Tile tile_of(const Args& p, long long t) {
    Tile ti;
    ti.ks = (int)(t % p.ksplit);
    int u = (int)(t / p.ksplit);
    const int all = p.mtiles * p.groups, band = 8 * p.ntiles_n;
    const int b = u / band, r = u - b * band;
    const int high = min(8, all - b * 8);
    ti.mt = b * 8 + r % high;
    ti.nt = r / high;
    ti.grp = ti.mt / p.mtiles;
    ti.mt -= ti.grp * p.mtiles;
    return ti;
}

__device__ __forceinline__ bool is_finite(const Args& p, int slot) {
    const int4 b = p.bad[slot];
    return (b.x | b.y | b.z | b.w) == 0;
}
// Whether row m (a lane's) belongs to a request whose adapter is not finite.
__device__ __forceinline__ bool spoilt_row(const Args& p, const Tile& ti, long long m, int lane) {
    const int2 q = p.tile_req[ti.mt];
    bool bad = false;
    for (int r = q.x; r < q.y; r += 32) {
        int4 c = make_int4(-1, 0, 0, 0);
        if (r + lane < q.y) c = p.piece[ti.mt + r + lane];
        unsigned found = __ballot_sync(0xffffffffu, c.x >= 0 && !is_finite(p, c.x));
        for (; found; found &= found - 1) {
            const int i = __ffs(found) - 1;
            const int lo = __shfl_sync(0xffffffffu, c.y, i), hi = __shfl_sync(0xffffffffu, c.z, i);
            bad |= m >= lo && m < hi;
        }
    }
    return bad;
}

// Walks the stages of a tile: the phases' (this split's share), then the low-rank blocks'.
struct Stages {
    const Args& p;
    Tile ti;
    int ph = 0, kt, kend;
    int r, rend, sub = 0, slot = -1;
    bool ext = false;
    __device__ __forceinline__ Stages(const Args& q, const Tile& t) : p(q), ti(t) {
        range();
        r = rend = 0;
        if (p.ext && ti.ks == p.ksplit - 1) {
            const int2 q2 = p.tile_req[ti.mt];
            r = q2.x;
            rend = q2.y;
        }
    }
    __device__ __forceinline__ void range() {
        const int nk = p.ph[ph].nk;
        kt = (int)((long long)ti.ks * nk / p.ksplit);
        kend = (int)((long long)(ti.ks + 1) * nk / p.ksplit);
    }
    // moves to the next stage; false when there is none
    __device__ __forceinline__ bool phase_stage() {
        while (kt >= kend) {
            if (++ph >= p.nphase) return false;
            range();
        }
        return true;
    }
    __device__ __forceinline__ bool ext_stage() {
        if (sub > 0) return true;                       // in the middle of a request's stages
        while (r < rend) {
            slot = p.piece[ti.mt + r].x;
            if (slot >= 0 && is_finite(p, slot)) return true;
            ++r;
        }
        return false;
    }
    __device__ __forceinline__ void ext_next() {
        if (++sub == p.ext) {
            sub = 0;
            ++r;
        }
    }
};

template <int BN, bool SPLIT>
struct Cfg {
    static constexpr int HB = BN / 2;
    static constexpr uint32_t kA = 128 * 128, kB = HB * 128;
    static constexpr uint32_t kStage = (SPLIT ? 2 : 1) * (kA + kB);
    static constexpr int S = SPLIT ? 4 : (BN == 256 ? 6 : 8);
    static constexpr int kAcc = SPLIT ? 2 * BN : BN;    // tensor-memory columns of one buffer
    static constexpr uint32_t kSmem = S * kStage + 512 + 1024;
    static_assert(kSmem <= 232448 && 2 * kAcc <= 512, "shared / tensor memory");
};

// 32 values of one row from column n on, as far as the row goes.
__device__ __forceinline__ void store32(void* C, long long off, const float* v, int left,
                                        int dtype, int vec) {
    if (dtype == ATOM_F32) {
        float* q = static_cast<float*>(C) + off;
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
            if (vec && i + 4 <= left) {
                *reinterpret_cast<float4*>(q + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (i + j < left) q[i + j] = v[i + j];
            }
        }
        return;
    }
    unsigned short* q = static_cast<unsigned short*>(C) + off;
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (dtype == ATOM_BF16) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[i + 2 * j], v[i + 2 * j + 1]);
                w[j] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __half2 h = __floats2half2_rn(v[i + 2 * j], v[i + 2 * j + 1]);
                w[j] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        if (vec && i + 8 <= left) {
            *reinterpret_cast<uint4*>(q + i) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (i + j < left) q[i + j] = (unsigned short)(w[j >> 1] >> (16 * (j & 1)));
        }
    }
}
__device__ __forceinline__ void spoil32(float* v) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(0x7FC00000u);
}
__device__ __forceinline__ void load32(const float* q, float* v) {
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
        const float4 x = *reinterpret_cast<const float4*>(q + i);
        v[i] = x.x, v[i + 1] = x.y, v[i + 2] = x.z, v[i + 3] = x.w;
    }
}

// Activation and derivative: fast intrinsics (a few 2^-23) for 16-bit results, the accurate
// functions for fp32 ones.
template <bool EXACT>
__device__ __forceinline__ float act_of(float g, int act) {
    if (act == 2) return g * 0.5f * erfcf(-0.70710678f * g);
    const float s = EXACT ? sigmoid_f(g) : sigmoid_gate(g);
    return act == 1 ? s : g * s;
}
template <bool EXACT>
__device__ __forceinline__ void act_both(float g, int act, float& a, float& da) {
    if (act == 2) {
        const float phi = 0.5f * erfcf(-0.70710678f * g);
        a = g * phi;
        da = phi + g * 0.39894228f * (EXACT ? expf(-0.5f * g * g) : __expf(-0.5f * g * g));
        return;
    }
    const float s = EXACT ? sigmoid_f(g) : sigmoid_gate(g);
    a = act == 1 ? s : g * s;
    da = act == 1 ? s * (1.f - s) : s * (1.f + g * (1.f - s));
}
// The epilogue's last step on 32 columns n.. of row m; v0 (and v1: the u columns of a gate).
template <int EPI, bool SPLIT>
__device__ __forceinline__ void finish32(const Args& p, const Tile& ti, long long m, int n,
                                         float* v0, float* v1, unsigned& mx0, unsigned& mx1) {
    if (m >= p.M || n >= p.N) return;
    const int left = p.N - n;
    if constexpr (EPI == kStore) {
        if (p.ksplit > 1) {
            float* q = p.part + ((long long)(ti.ks * p.groups + ti.grp) * p.M + m) * p.N + n;
            store32(q, 0, v0, left, ATOM_F32, p.N % 4 == 0);
        } else {
            store32(p.C[ti.grp], m * p.ldc + n, v0, left, p.dtype, p.vec);
        }
    } else if constexpr (EPI == kGate) {
        if (p.gu) {
            float* q = p.gu + m * 2 * p.Fp + n;
            store32(q, 0, v0, 32, ATOM_F32, 1);
            store32(q, p.Fp, v1, 32, ATOM_F32, 1);
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) v0[i] = act_of<SPLIT>(v0[i], p.act) * v1[i];
        store32(p.C[0], m * p.ldc + n, v0, 32, p.dtype, 1);
    } else {
        // v0, v1 = g, u (kGateBwdGU, dh from memory) or v0 = dh (kGateBwdDH, g and u from memory)
        float w[32];
        if constexpr (EPI == kGateBwdGU) {
            load32(p.dh + m * p.Fp + n, w);
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (i >= left) w[i] = 0.f;      // past the row nothing was written
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) w[i] = v0[i];
            load32(p.gu + m * 2 * p.Fp + n, v0);
            load32(p.gu + m * 2 * p.Fp + p.Fp + n, v1);
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            float a, da;
            act_both<SPLIT>(v0[i], p.act, a, da);
            const float u = v1[i], d = w[i];
            v0[i] = d * u * da;
            v1[i] = d * a;
            w[i] = a * u;
            if (SPLIT && i < left) {
                mx0 = max(mx0, max(finite_bits(v0[i]), finite_bits(v1[i])));
                mx1 = max(mx1, finite_bits(w[i]));
            }
        }
        store32(p.C[0], m * 2 * p.Fp + n, v0, 32, p.dtype, 1);
        store32(p.C[0], m * 2 * p.Fp + p.Fp + n, v1, 32, p.dtype, 1);
        if (p.H) store32(p.H, m * p.Fp + n, w, 32, p.dtype, 1);
    }
}

template <int BN, int EPI, bool SPLIT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    pair_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args p) {
    using CF = Cfg<BN, SPLIT>;
    constexpr int S = CF::S;
    // a gate's tile: columns 0 .. BN/2 of the accumulator are g, the others u
    constexpr bool GATED = EPI == kGate || EPI == kGateBwdGU;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S * CF::kStage);
    uint64_t* empty = full + S;
    uint64_t* accf = empty + S;      // [2] accumulator buffer full
    uint64_t* acce = accf + 2;       // [2] and free again (CTA 0's: both CTAs' epilogue warps)
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acce + 2);
    int* failed = reinterpret_cast<int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t rank;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const int pairs = gridDim.x >> 1, first = blockIdx.x >> 1;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&accf[b], 1);
            mbar_init(&acce[b], 16);
        }
        *failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
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

    if (warp == 0) {
        if (lane == 0) {
            uint32_t it = 0;
            bool ok = true;
            // waits for a free stage and names its barrier of CTA 0
            auto open = [&](uint32_t& dst, uint32_t& bar) {
                const uint32_t s = it % S, ph = (it / S) & 1u;
                if (!mbar_wait(&empty[s], ph ^ 1u, p.err)) return false;
                if (rank == 0)
                    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(
                                     smem_u32(&full[s])), "r"(2 * CF::kStage) : "memory");
                dst = base + s * CF::kStage;
                bar = peer_addr(smem_u32(&full[s]), 0);
                ++it;
                return true;
            };
            for (long long t = first; ok && t < p.tiles; t += pairs) {
                Stages st(p, tile_of(p, t));
                const int m0 = st.ti.mt * 256 + rank * 128;
                for (; st.phase_stage(); ++st.kt) {
                    uint32_t dst, bar;
                    if (!(ok = open(dst, bar))) break;
                    const Phase& f = p.ph[st.ph];
                    const int k0 = st.kt * 64, n0 = st.ti.nt * f.bstep + rank * f.brank;
#pragma unroll
                    for (int pl = 0; pl < (SPLIT ? 2 : 1); ++pl) {
                        const CUtensorMap* ma = &maps.m[f.a + pl + (SPLIT ? 2 : 1) * st.ti.grp];
                        const uint32_t da = dst + pl * CF::kA;
                        if (f.a_mn) {
                            tma_load(da, ma, m0, k0, bar);
                            tma_load(da + 8192, ma, m0 + 64, k0, bar);
                        } else {
                            tma_load(da, ma, k0, m0, bar);
                        }
                        const CUtensorMap* mb = &maps.m[(rank ? f.b1 : f.b0) + pl];
                        const uint32_t db = dst + (SPLIT ? 2 : 1) * CF::kA + pl * CF::kB;
                        if (f.b_mn) {
#pragma unroll
                            for (int j = 0; j < CF::HB / 64; ++j)
                                tma_load(db + j * 8192, mb, n0 + 64 * j, k0, bar);
                        } else {
                            tma_load(db, mb, k0, n0, bar);
                        }
                    }
                }
                for (; ok && p.ext && st.ext_stage(); st.ext_next()) {
                    uint32_t dst, bar;
                    if (!(ok = open(dst, bar))) break;
                    const int y = (st.ti.mt + st.r) * 256 + rank * 128, k0 = st.sub * 64;
                    const int n0 = st.ti.nt * BN + rank * CF::HB;
#pragma unroll
                    for (int pl = 0; pl < (SPLIT ? 2 : 1); ++pl) {
                        tma_load(dst + pl * CF::kA, &maps.m[p.ext_a + pl], k0, y, bar);
                        const uint32_t db = dst + (SPLIT ? 2 : 1) * CF::kA + pl * CF::kB;
                        const CUtensorMap* mb = &maps.m[p.ext_b + pl];
                        if (p.ext_bmn) {
#pragma unroll
                            for (int j = 0; j < CF::HB / 64; ++j)
                                tma_load3(db + j * 8192, mb, n0 + 64 * j, k0, st.slot, bar);
                        } else {
                            tma_load3(db, mb, k0, n0, st.slot, bar);
                        }
                    }
                }
            }
            // the last stages are read before this CTA may end
            for (uint32_t k = it > S ? it - S : 0; ok && k < it; ++k)
                ok = mbar_wait(&empty[k % S], (k / S) & 1u, p.err);
            if (!ok) *(volatile int*)failed = 1;
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            uint32_t it = 0, round = 0;
            bool ok = true, open = false;
            uint32_t acc = 0, fresh = 0;
            auto begin = [&]() {         // a free accumulator buffer for the next round
                const uint32_t b = round & 1u;
                if (!mbar_wait(&acce[b], ((round >> 1) & 1u) ^ 1u, p.err)) return false;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                acc = tmem + b * CF::kAcc;
                fresh = 0;
                return open = true;
            };
            auto end = [&]() {
                mma_commit(&accf[round & 1u]);
                ++round;
                open = false;
            };
            auto stage = [&](int a_mn, int b_mn, int steps) {
                const uint32_t s = it % S, ph = (it / S) & 1u;
                if (!mbar_wait(&full[s], ph, p.err)) return false;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t id = idesc(BN, SPLIT ? 0 : p.bf16, a_mn, b_mn);
                const uint32_t a = base + s * CF::kStage, b = a + (SPLIT ? 2 : 1) * CF::kA;
                const uint32_t as = a_mn ? 2048 : 32, bs = b_mn ? 2048 : 32;
                for (int k = 0; k < steps; ++k) {
                    const uint64_t ad = sdesc(a + k * as, a_mn), bd = sdesc(b + k * bs, b_mn);
                    mma(acc, ad, bd, id, fresh);
                    if constexpr (SPLIT) {
                        const uint64_t al = sdesc(a + CF::kA + k * as, a_mn);
                        const uint64_t bl = sdesc(b + CF::kB + k * bs, b_mn);
                        mma(acc + BN, ad, bl, id, fresh);
                        mma(acc + BN, al, bd, id, 1u);
                    }
                    fresh = 1;
                }
                mma_commit(&empty[s]);
                ++it;
                return true;
            };
            for (long long t = first; ok && t < p.tiles; t += pairs) {
                Stages st(p, tile_of(p, t));
                int n = 0;
                for (; ok && st.phase_stage(); ++st.kt, ++n) {
                    if (SPLIT && open && n == kRound) end(), n = 0;
                    ok = (open || begin()) && stage(p.ph[st.ph].a_mn, p.ph[st.ph].b_mn, 4);
                }
                if (SPLIT && ok && open) end(), n = 0;
                for (; ok && p.ext && st.ext_stage(); st.ext_next(), ++n) {
                    if (SPLIT && open && n == kRound) end(), n = 0;
                    ok = (open || begin()) &&
                         stage(0, p.ext_bmn, (min(64, p.R - 64 * st.sub) + 15) >> 4);
                }
                if (ok && open) end();
            }
            if (!ok) *(volatile int*)failed = 1;
        }
    } else {
        const int q = warp & 3, half = (warp - 2) >> 2;
        const uint32_t lanes = (uint32_t)(q * 32) << 16;
        uint32_t round = 0;
        unsigned mx0 = 0, mx1 = 0;
        auto drained = [&]() {           // this warp has read the round's accumulators
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0)
                asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(
                                 peer_addr(smem_u32(&acce[round & 1u]), 0)) : "memory");
            ++round;
        };
        auto filled = [&]() {
            const bool ok = __all_sync(0xffffffffu,
                                       mbar_wait(&accf[round & 1u], (round >> 1) & 1u, p.err));
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            return ok;
        };
        // first column of this warp's k-th 32-column chunk (of g, for a gate; u: BN/2 further)
        constexpr int kChunks = (GATED ? BN / 4 : BN / 2) / 32;
        const int c0 = half * kChunks * 32;
        bool ok = true;
        for (long long t = first; ok && t < p.tiles; t += pairs) {
            const Tile ti = tile_of(p, t);
            const long long m = (long long)ti.mt * 256 + rank * 128 + q * 32 + lane;
            const int nb = ti.nt * (GATED ? BN / 2 : BN) + c0;
            const bool spoilt = EPI == kStore && p.ext && spoilt_row(p, ti, m, lane);
            if constexpr (!SPLIT) {
                if (!(ok = filled())) break;
                const uint32_t ta = tmem + lanes + (round & 1u) * CF::kAcc + c0;
#pragma unroll 1
                for (int k = 0; k < kChunks; ++k) {
                    float v0[32], v1[32];
                    tmem_ld32(ta + 32 * k, v0);
                    if (GATED) tmem_ld32(ta + BN / 2 + 32 * k, v1);
                    tmem_wait_ld();
                    pin32(v0);
                    if (GATED) pin32(v1);
                    if (k == kChunks - 1) drained();
                    if (EPI == kStore && spoilt) spoil32(v0);
                    finish32<EPI, SPLIT>(p, ti, m, nb + 32 * k, v0, v1, mx0, mx1);
                }
            } else {
                // per chunk pair: the tile's rounds summed in registers
                float v[GATED ? 2 * kChunks : kChunks][32];
#pragma unroll
                for (int k = 0; k < (GATED ? 2 * kChunks : kChunks); ++k)
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[k][i] = 0.f;
                auto add = [&](float f) {
                    const uint32_t ta = tmem + lanes + (round & 1u) * CF::kAcc + c0;
#pragma unroll
                    for (int k = 0; k < (GATED ? 2 * kChunks : kChunks); ++k) {
                        const uint32_t col =
                            GATED ? (k / kChunks) * (BN / 2) + (k % kChunks) * 32 : 32 * k;
                        float x[32], y[32];
                        tmem_ld32(ta + col, x);
                        tmem_ld32(ta + BN + col, y);
                        tmem_wait_ld();
                        pin32(x);
                        pin32(y);
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            v[k][i] = fmaf(f, fmaf(y[i], 1.f / 2048.f, x[i]), v[k][i]);
                    }
                    drained();
                };
                const float sb = pow2_inv(pow2_scale(*p.bmax));
                const float sa = p.rinv ? (m < p.M ? p.rinv[m] : 0.f)
                                        : pow2_inv(pow2_scale(*p.amax));
                int stages = 0;
                for (int f = 0; f < p.nphase; ++f)
                    stages += (int)((long long)(ti.ks + 1) * p.ph[f].nk / p.ksplit) -
                              (int)((long long)ti.ks * p.ph[f].nk / p.ksplit);
                for (int k = 0; ok && k < stages; k += kRound)
                    if ((ok = filled())) add(1.f);
                if (!ok) break;
#pragma unroll
                for (int k = 0; k < (GATED ? 2 * kChunks : kChunks); ++k)
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[k][i] = v[k][i] * sa * sb;
                if (p.ext) {
                    Stages st(p, ti);
                    int es = 0;
                    for (; st.ext_stage(); st.ext_next()) ++es;
                    const float f = (m < p.M ? p.ext_rinv[m] : 0.f) *
                                    pow2_inv(pow2_scale(*p.ext_bmax));
                    for (int k = 0; ok && k < es; k += kRound)
                        if ((ok = filled())) add(f);
                    if (!ok) break;
                }
#pragma unroll
                for (int k = 0; k < kChunks; ++k) {
                    float u[32];         // kGateBwdDH: room for the u that it reads
                    if (EPI == kStore && spoilt) spoil32(v[k]);
                    finish32<EPI, SPLIT>(p, ti, m, nb + 32 * k, v[k], GATED ? v[kChunks + k] : u,
                                         mx0, mx1);
                }
            }
        }
        if constexpr (SPLIT && (EPI == kGateBwdGU || EPI == kGateBwdDH)) {
            if (p.hmax) {
                mx0 = __reduce_max_sync(0xffffffffu, mx0);
                mx1 = __reduce_max_sync(0xffffffffu, mx1);
                if (lane == 0) {
                    atomicMax(p.hmax, mx0);
                    atomicMax(p.hmax + 1, mx1);
                }
            }
        }
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


// C[g][m, n] = sum over the splits, in order.
__global__ void __launch_bounds__(256) reduce_kernel(Args p) {
    const long long per = p.M * p.N, all = per * p.groups;
    const bool four = p.N % 4 == 0;
    for (long long i = (blockIdx.x * 256LL + threadIdx.x) * 4; i < all; i += gridDim.x * 1024LL) {
        float v[4] = {};
        const int n = (int)min(4LL, all - i);
        for (int s = 0; s < p.ksplit; ++s) {
            const float* q = p.part + s * all + i;
            if (four) {
                const float4 x = *reinterpret_cast<const float4*>(q);
                v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
            } else {
                for (int j = 0; j < n; ++j) v[j] += q[j];
            }
        }
        for (int j = 0; j < n; ++j) {
            const long long e = i + j;
            const int g = (int)(e / per);
            const long long r = e - g * per;
            store_f(p.C[g], r / p.N * p.ldc + r % p.N, v[j], p.dtype);
        }
    }
}

// One warp a row. Planes are zero past the row's end up to the pitch.
__global__ void __launch_bounds__(256) prep_kernel(const __grid_constant__ PrepList l) {
    const PrepItem& it = l.it[blockIdx.y];
    const int lane = threadIdx.x & 31;
    unsigned top = 0;
    for (long long r = blockIdx.x * 8LL + (threadIdx.x >> 5); r < it.rows; r += gridDim.x * 8LL) {
        if (it.mode == kPack) {
            const unsigned short* src = static_cast<const unsigned short*>(it.src) + r * it.ld;
            unsigned short* dst = static_cast<unsigned short*>(it.dst) + r * it.dld;
            for (long long c = lane; c < it.dld; c += 32) dst[c] = c < it.cols ? src[c] : 0;
            continue;
        }
        const float* src = static_cast<const float*>(it.src) + r * it.ld;
        const bool four = (reinterpret_cast<uintptr_t>(src) & 15) == 0 && it.cols % 4 == 0;
        float s = 1.f;
        if (it.mode == kTensorSplit) {
            s = pow2_scale(*it.max);
        } else {
            unsigned mx = 0;
            if (four) {
                for (long long c = 4 * lane; c < it.cols; c += 128) {
                    const float4 x = *reinterpret_cast<const float4*>(src + c);
                    mx = max(max(mx, max(finite_bits(x.x), finite_bits(x.y))),
                             max(finite_bits(x.z), finite_bits(x.w)));
                }
            } else {
                for (long long c = lane; c < it.cols; c += 32) mx = max(mx, finite_bits(src[c]));
            }
            mx = __reduce_max_sync(0xffffffffu, mx);
            top = max(top, mx);
            if (it.mode == kMax) continue;
            s = pow2_scale(mx);
            if (lane == 0) it.rinv[r] = pow2_inv(s);
        }
        __half* hi = static_cast<__half*>(it.dst) + r * it.dld;
        __half* lo = hi + it.plane;
        for (long long c = 4 * lane; c < it.dld; c += 128) {
            float x[4];
            if (four && c < it.cols) {
                const float4 v = *reinterpret_cast<const float4*>(src + c);
                x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = c + j < it.cols ? src[c + j] : 0.f;
            }
            __half h[4], g[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) split_half(x[j] * s, h[j], g[j]);
            *reinterpret_cast<uint2*>(hi + c) = *reinterpret_cast<uint2*>(h);
            *reinterpret_cast<uint2*>(lo + c) = *reinterpret_cast<uint2*>(g);
        }
    }
    if (it.max && (it.mode == kMax || it.mode == kRowSplit) && lane == 0 && top)
        atomicMax(it.max, top);
}

int prepare(const PrepList& l, cudaStream_t st) {
    if (l.n == 0) return ATOM_OK;
    long long rows = 1;
    for (int i = 0; i < l.n; ++i) rows = rows < l.it[i].rows ? l.it[i].rows : rows;
    const long long blocks = (rows + 7) / 8;
    prep_kernel<<<dim3((unsigned)(blocks < 1184 ? blocks : 1184), l.n), 256, 0, st>>>(l);
    return check_launch("operand preparation");
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

int make_map(CUtensorMap* m, const void* p, long long cols, long long rows, long long ld,
             int box_rows, int depth, long long ldz) {
    const auto encode = encoder();
    if (!encode) {
        set_error("cuTensorMapEncodeTiled unavailable");
        return ATOM_ERR_CUDA;
    }
    cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)depth};
    cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)ldz * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, depth ? 3 : 2,
                              const_cast<void*>(p), dims, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("cuTensorMapEncodeTiled failed (%d): %lld x %lld, ld %lld", (int)r, rows, cols, ld);
        return ATOM_ERR_ARG;
    }
    return ATOM_OK;
}

static int sm_count() {
    int dev = 0, n = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    return n;
}

// The tile width and split that a count of clocks prefers: rounds of work items over the SM
// pairs, each a tile's stages (512 clocks of tensor work at width 256, 256 at 128 but fed no
// faster than ~300; SPLIT 12 products of 64) and its fill and drain, and for a split the pass
// over the partial sums.
Choice choose(long long M, int N, int nk, int groups, bool gated, bool split, bool may_split) {
    const int pairs = sm_count() / 2;
    const long long mt = (M + 255) / 256 * groups;
    Choice best{128, 1, 0};
    double least = 1e30;
    for (int bn : {256, 128}) {
        if (split && bn == 256) continue;
        const int w = gated ? bn / 2 : bn;
        const long long tiles = mt * ((N + w - 1) / w);
        const double stage = split ? 800 : bn == 256 ? 530 : 310;
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

template <int BN, int EPI, bool SPLIT>
static int run(const Maps& maps, const Args& p, cudaStream_t st) {
    using CF = Cfg<BN, SPLIT>;
    static bool set[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !set[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(
            pair_kernel<BN, EPI, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
            (int)CF::kSmem);
        if (e != cudaSuccess) {
            set_error("pair product: cannot reserve %u bytes of shared memory: %s", CF::kSmem,
                      cudaGetErrorString(e));
            return ATOM_ERR_CUDA;
        }
        if (dev >= 0 && dev < 64) set[dev] = true;
    }
    const long long pairs = sm_count() / 2;
    const int grid = 2 * (int)(p.tiles < pairs ? p.tiles : pairs);
    pair_kernel<BN, EPI, SPLIT><<<grid, kThreads, CF::kSmem, st>>>(maps, p);
    if (int s = check_launch("pair product")) return s;
    if (p.ksplit > 1) {
        const long long blocks = (p.M * p.N * p.groups + 1023) / 1024;
        reduce_kernel<<<(unsigned)(blocks < 1184 ? blocks : 1184), 256, 0, st>>>(p);
        return check_launch("pair product sums");
    }
    return ATOM_OK;
}

int launch(int epilogue, const Choice& c, bool split, const Maps& maps, Args& p, cudaStream_t st) {
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
#define ATOM_PAIR(E)                                            \
    if (epilogue == E) {                                        \
        if (split) return run<128, E, true>(maps, p, st);       \
        return c.bn == 256 ? run<256, E, false>(maps, p, st)    \
                           : run<128, E, false>(maps, p, st);   \
    }
    ATOM_PAIR(kStore)
    ATOM_PAIR(kGate)
    ATOM_PAIR(kGateBwdGU)
    ATOM_PAIR(kGateBwdDH)
#undef ATOM_PAIR
    return ATOM_ERR_UNSUPPORTED;
}

}  // namespace pair
}  // namespace atom
