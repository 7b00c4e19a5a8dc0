// The gated feed-forward block Y = (act(X Wg^T) * (X Wu^T)) Wd^T and its backward pass.
#include "typed.cuh"

namespace atom {

// 64 x 64 tile, 16 deep, 4 x 4 outputs a thread.
__global__ void __launch_bounds__(256) plain_product_kernel(PlainProduct p) {
    __shared__ float As[16][64 + 1], Bs[16][64 + 1];
    const long long m0 = (long long)blockIdx.y * 64, n0 = (long long)blockIdx.x * 64;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float acc[4][4] = {};
    const long long kp = (p.K + 15) / 16 * 16;
    for (long long kk = 0; kk < (p.A2 ? 2 * kp : kp); kk += 16) {
        const void* A = kk < kp ? p.A : p.A2;
        const void* B = kk < kp ? p.B : p.B2;
        const long long k0 = kk < kp ? kk : kk - kp;
        for (int i = threadIdx.x; i < 1024; i += 256) {
            const int r = p.ak == 1 ? i >> 4 : i & 63, k = p.ak == 1 ? i & 15 : i >> 6;
            const int rb = p.bk == 1 ? i >> 4 : i & 63, kb = p.bk == 1 ? i & 15 : i >> 6;
            As[k][r] = m0 + r < p.M && k0 + k < p.K
                           ? load_f(A, (m0 + r) * p.am + (k0 + k) * p.ak, p.ta) : 0.f;
            Bs[kb][rb] = n0 + rb < p.N && k0 + kb < p.K
                             ? load_f(B, (n0 + rb) * p.bn + (k0 + kb) * p.bk, p.tb) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[i][j] = fmaf(As[k][ty + 16 * i], Bs[k][tx + 16 * j], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const long long m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
            if (m >= p.M || n >= p.N) continue;
            store_f(p.C, m * p.ldc + n, acc[i][j], p.tc);
        }
}

int plain_product(const PlainProduct& p, cudaStream_t st) {
    if (p.M == 0 || p.N == 0) return ATOM_OK;
    ATOM_REQUIRE(ceil_div(p.M, 64) < 65536, "too many rows");
    plain_product_kernel<<<dim3(ceil_div(p.N, 64), ceil_div(p.M, 64)), 256, 0, st>>>(p);
    return check_launch("plain product");
}

// H = act(G) U; with dH: dG and dU in place of G and U.
__global__ void gate_kernel(float* G, float* U, const float* dH, float* H, long long n, int act) {
    for (long long i = blockIdx.x * 256LL + threadIdx.x; i < n; i += gridDim.x * 256LL) {
        float a, da;
        const float u = U[i];
        act_grad(G[i], act, a, da);
        H[i] = a * u;
        if (dH) {
            G[i] = dH[i] * u * da;
            U[i] = dH[i] * a;
        }
    }
}

static int gate(float* G, float* U, const float* dH, float* H, long long n, int act,
                cudaStream_t st) {
    const long long blocks = (n + 255) / 256;
    gate_kernel<<<(int)(blocks < 4096 ? blocks : 4096), 256, 0, st>>>(G, U, dH, H, n, act);
    return check_launch("gate");
}

}  // namespace atom

using namespace atom;

static int check_ff(int dtype, int64_t M, int D, int F, int O, int act) {
    ATOM_REQUIRE(dtype >= ATOM_F32 && dtype <= ATOM_F16, "gated_ff: unknown type %d", dtype);
    ATOM_REQUIRE(M >= 0 && M < (1LL << 31) && D > 0 && F > 0 && O > 0, "gated_ff: bad sizes");
    ATOM_REQUIRE(D < (1 << 24) && F < (1 << 24) && O < (1 << 24), "gated_ff: widths above 2^24");
    ATOM_REQUIRE(act >= 0 && act <= 2, "gated_ff: act must be 0, 1 or 2");
    return ATOM_OK;
}

struct FfSpace {
    float *G, *U, *H, *dH;
    FfSpace(Cursor& c, int64_t M, int F, bool bwd) {
        G = c.take<float>(M * F);
        U = c.take<float>(M * F);
        H = c.take<float>(M * F);
        dH = bwd ? c.take<float>(M * F) : nullptr;
    }
};

extern "C" int atom_gated_ff_bytes(int dtype, int64_t M, int D, int F, int O, size_t* bytes_host) {
    if (int s = check_ff(dtype, M, D, F, O, 0)) return s;
    ATOM_REQUIRE(bytes_host, "gated_ff: bytes_host is NULL");
    Cursor f(nullptr), b(nullptr);
    FfSpace(f, M, F, false);
    FfSpace(b, M, F, true);
    bytes_host[0] = f.used;
    bytes_host[1] = b.used;
    bytes_host[2] = 256;
    return ATOM_OK;
}

extern "C" int atom_gated_ff_fwd(int dtype, const void* x, int64_t ldx, int64_t M, int D, int F,
                                 int O, const void* wg, const void* wu, const void* wd, int act,
                                 void* y, int64_t ldy, void* kept, void* ws, size_t ws_bytes,
                                 void* stream) {
    if (int s = check_ff(dtype, M, D, F, O, act)) return s;
    if (M == 0) return ATOM_OK;
    ATOM_REQUIRE(x && wg && wu && wd && y && ldx >= D && ldy >= O, "gated_ff: bad operand");
    Cursor c(ws);
    FfSpace sp(c, M, F, false);
    ATOM_REQUIRE(ws && ws_bytes >= c.used, "gated_ff: the workspace needs %zu bytes", c.used);
    cudaStream_t st = (cudaStream_t)stream;
    const int t = dtype;
    if (int s = plain_product({x, ldx, 1, t, wg, D, 1, t, sp.G, F, 0, M, F, D}, st)) return s;
    if (int s = plain_product({x, ldx, 1, t, wu, D, 1, t, sp.U, F, 0, M, F, D}, st)) return s;
    if (int s = gate(sp.G, sp.U, nullptr, sp.H, M * F, act, st)) return s;
    return plain_product({sp.H, F, 1, 0, wd, F, 1, t, y, ldy, t, M, O, F}, st);
}

extern "C" int atom_gated_ff_bwd(int dtype, const void* x, int64_t ldx, int64_t M, int D, int F,
                                 int O, const void* wg, const void* wu, const void* wd, int act,
                                 const void* dy, int64_t lddy, const void* kept, void* dx,
                                 int64_t lddx, void* dwg, void* dwu, void* dwd, void* ws,
                                 size_t ws_bytes, void* stream) {
    if (int s = check_ff(dtype, M, D, F, O, act)) return s;
    cudaStream_t st = (cudaStream_t)stream;
    const int t = dtype;
    if (M > 0) {
        ATOM_REQUIRE(x && wg && wu && wd && dy && ldx >= D && lddy >= O && (!dx || lddx >= D),
                     "gated_ff: bad operand");
        Cursor c(ws);
        FfSpace sp(c, M, F, true);
        ATOM_REQUIRE(ws && ws_bytes >= c.used, "gated_ff: the workspace needs %zu bytes", c.used);
        if (int s = plain_product({x, ldx, 1, t, wg, D, 1, t, sp.G, F, 0, M, F, D}, st))
            return s;
        if (int s = plain_product({x, ldx, 1, t, wu, D, 1, t, sp.U, F, 0, M, F, D}, st))
            return s;
        if (int s = plain_product({dy, lddy, 1, t, wd, 1, F, t, sp.dH, F, 0, M, F, O}, st))
            return s;
        if (int s = gate(sp.G, sp.U, sp.dH, sp.H, M * F, act, st)) return s;
        if (dx) {
            if (int s = plain_product({sp.G, F, 1, 0, wg, 1, D, t, dx, lddx, t, M, D, F, sp.U, wu},
                                      st))
                return s;
        }
        if (dwg)
            if (int s = plain_product({sp.G, 1, F, 0, x, 1, ldx, t, dwg, D, t, F, D, M}, st))
                return s;
        if (dwu)
            if (int s = plain_product({sp.U, 1, F, 0, x, 1, ldx, t, dwu, D, t, F, D, M}, st))
                return s;
        if (dwd)
            if (int s = plain_product({dy, 1, lddy, t, sp.H, 1, F, 0, dwd, F, t, O, F, M}, st))
                return s;
        return ATOM_OK;
    }
    const size_t e = dtype_size(dtype);
    for (void* p : {dwg, dwu}) if (p) cudaMemsetAsync(p, 0, e * F * D, st);
    if (dwd) cudaMemsetAsync(dwd, 0, e * O * F, st);
    return check_launch("gated_ff", 0);
}
