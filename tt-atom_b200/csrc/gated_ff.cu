// The gated feed-forward block Y = (act(X Wg^T) * (X Wu^T)) Wd^T and its backward pass, as pair
// products (pair_product.cu) with the gate in their epilogues:
//   forward   [G | U] tiles -> H = act(G) U;  Y = H Wd^T
//   backward  dH = dY Wd, then [G | U] again with dH in the epilogue -> dG, dU, H (or, with the
//             forward's G and U kept, dH tiles with G and U in the epilogue);
//             dX = [dG | dU] [Wg; Wu],  dWg, dWu = [dG | dU]^T X,  dWd = dY^T H
// The transposed products read their operands as they lie (M/N-major tiles), so nothing is
// transposed in memory.
#include <algorithm>
#include <initializer_list>

#include "few_rows.cuh"
#include "pair_product.cuh"

namespace atom {
namespace {

using namespace pair;

// A 16-bit operand ready for TMA (fp32: the first of its planes, `plane` elements apart).
struct Operand {
    const void* p = nullptr;
    long long rows = 0, cols = 0, ld = 0, plane = 0;
    Operand columns(long long c0, long long n) const {
        Operand o = *this;
        o.p = static_cast<const uint16_t*>(p) + c0;
        o.cols = n;
        return o;
    }
};

// Whether a call's rows are streamed past: 16 at most, where a tile of 256 would be all but empty
// (1,024 x 4,096 in bf16, forward: 8.7 us at 1 row and 11.1 at 16 against 21.6 and 17.1 by tiles;
// fp32, 16 rows against 17 by tiles: 41 and 55 us forward, 92 and 104 backward, at 256 x 1,024 14 and
// 20, 34 and 45). A 16-bit backward pass multiplies on
// the FMA pipe there: from 7 rows on, or 80 million products of rows and weights, tiles are faster
// (1,024 x 4,096: 31 against 43 us at 1 row, 39 and 39 at 6, 63 and 36 at 16; 2,048 x 8,192: 92 and
// 91 at 1 row, 97 and 83 at 2).
bool few_rows(int dtype, long long M, int D, int F, int O, bool bwd) {
    if (M > few::kFewRows) return false;
    return !bwd || dtype == ATOM_F32 || (M <= 6 && M * F * (2LL * D + O) <= 80000000);
}

struct FfSizes {
    int dtype;
    long long M;
    int D, F, O;
    long long Dp, Fp, Op;       // widths of packed rows
    bool split, few;
    Choice gate{}, down{}, dh{}, dx{}, dwgu{}, dwd{};
    FfSizes(int t, long long m, int d, int f, int o, bool bwd)
        : dtype(t), M(m), D(d), F(f), O(o), Dp(up(d, 8)), Fp(up(f, 32)), Op(up(o, 8)),
          split(t == ATOM_F32), few(few_rows(t, m, d, f, o, bwd)) {
        if (few) return;
        gate = choose(M, F, nk(D), 1, true, split, false);
        if (!bwd) {
            down = choose(M, O, nk(F), 1, false, split, true);
        } else {
            dh = choose(M, F, nk(O), 1, false, split, false);
            dx = choose(M, D, 2 * nk(F), 1, false, split, true);
            dwgu = choose(F, D, nk(M), 2, false, split, true);
            dwd = choose(O, F, nk(M), 1, false, split, true);
        }
    }
    int nk(long long k) const { return (int)((k + 63) / 64); }
    int planes() const { return split ? kPlanes : 1; }
};

// One call's buffers. 16-bit operands are packed only where TMA cannot read them; fp32 ones
// always become planes.
struct FfSpace {
    uint16_t *x, *wg, *wu, *wd, *dy, *H, *dgu;
    float *dh, *part, *part_gu, *part_d;
    float *few_H, *few_dh, *few_dx, *few_grads;
    size_t bytes;
    FfSpace(void* ws, const FfSizes& z, bool bwd) {
        memset(this, 0, sizeof(*this));
        Cursor c(ws);
        const long long M = z.M, k = z.planes();
        if (z.few) {
            if (bwd) {
                few_dh = c.take<float>(few::down_shares(z.O, z.F, 32) * M * z.F);
                few_dx = c.take<float>(few::down_shares(z.F, z.D) * M * z.D);
                few_grads = c.take<float>(3 * M * z.F);
            } else if (z.split) {
                few_H = c.take<float>(M * z.Fp);
            } else {
                H = c.take<uint16_t>(M * z.Fp);
            }
            bytes = c.used;
            return;
        }
        x = c.take<uint16_t>(k * M * z.Dp);
        wg = c.take<uint16_t>(k * z.F * z.Dp);
        wu = c.take<uint16_t>(k * z.F * z.Dp);
        wd = c.take<uint16_t>(k * z.O * z.Fp);
        H = c.take<uint16_t>(k * M * z.Fp);
        if (bwd) {
            dy = c.take<uint16_t>(k * M * z.Op);
            dh = c.take<float>(up(M, 32) * z.Fp);
            dgu = c.take<uint16_t>(k * M * 2 * z.Fp);
        }
        part = c.take<float>(bwd ? z.dx.part : z.down.part);
        part_gu = c.take<float>(z.dwgu.part);
        part_d = c.take<float>(z.dwd.part);
        bytes = c.used;
    }
};

// Fills a map (and, for further planes, the next ones).
int put(Maps& maps, int i, const Operand& o, bool mn, int box_rows, int planes) {
    for (int pl = 0; pl < planes; ++pl)
        if (int s = make_map(&maps.m[i + pl], static_cast<const uint16_t*>(o.p) + pl * o.plane, o.cols,
                             o.rows, o.ld, mn ? 64 : box_rows))
            return s;
    return ATOM_OK;
}

struct Ff {
    FfSizes z;
    FfSpace sp;
    Chain st;
    int act;
    Operand x, wg, wu, wd, dy;
    PrepList list;
    Sums sums{};

    // an operand of this call: as it lies, or through the list's packing / planes
    Operand take(const void* p, long long rows, long long cols, long long ld, uint16_t* buf,
                 long long pitch) {
        if (!z.split && tma_ready(p, ld)) return {p, rows, cols, ld, 0};
        const long long plane = rows * pitch;
        list.add({p, rows, cols, ld, buf, pitch, plane, z.split ? kSplit : kPack});
        return {buf, rows, cols, pitch, plane};
    }
    // What the products read, in one launch; dyp: a backward pass, which reads x for G and U and for
    // the weights' gradients alone.
    int inputs(const void* xp, long long ldx, const void* g, const void* u, const void* d,
               const void* dyp = nullptr, long long lddy = 0, bool reads_x = true) {
        if (reads_x) x = take(xp, z.M, z.D, ldx, sp.x, z.Dp);
        wg = take(g, z.F, z.D, z.D, sp.wg, z.Dp);
        wu = take(u, z.F, z.D, z.D, sp.wu, z.Dp);
        wd = take(d, z.O, z.F, z.F, sp.wd, up(z.F, 8));
        if (dyp) dy = take(dyp, z.M, z.O, lddy, sp.dy, z.Op);
        return prepare(list, st);
    }
    Args args(long long M, int N) const {
        Args p;
        memset(&p, 0, sizeof(p));
        p.M = M;
        p.N = N;
        p.groups = 1;
        p.nphase = 1;
        p.bf16 = z.dtype == ATOM_BF16;
        p.act = act;
        p.Fp = (int)z.Fp;
        p.dtype = z.dtype;
        p.part = sp.part;
        p.used = 0;
        return p;
    }
    void output(Args& p, void* C, long long ldc) const {
        p.C[0] = C;
        p.ldc = ldc;
    }
    // a gate epilogue's output (dgu or, forward, H; and H beside dgu); fp32: planes
    int gate_output(Maps& maps, Args& p, uint16_t* C, long long width, uint16_t* H) const {
        p.gu_half = up(z.M, 32) * z.Fp;
        p.H = H != nullptr;
        const int n = z.planes(), t = z.split ? ATOM_BF16 : z.dtype;
        for (int k = 0; k < n; ++k) {
            p.used |= 1u << (out_map(n) + k) | (unsigned)p.H << (h_map(n) + k);
            if (int s = make_out_map(&maps.m[out_map(n) + k], C + k * z.M * width, t, width, z.M, width))
                return s;
            if (!H) continue;
            if (int s = make_out_map(&maps.m[h_map(n) + k], H + k * z.M * z.Fp, t, z.Fp, z.M, z.Fp))
                return s;
        }
        return ATOM_OK;
    }
    // [G | U] tiles of X
    int gates(int epilogue, Args& p, uint16_t* C, long long width, uint16_t* H) {
        const Choice c = z.gate;
        const int k = z.planes();
        Maps maps;
        if (int s = put(maps, 0, x, false, 128, k)) return s;
        if (int s = put(maps, k, wg, false, c.bn / 2, k)) return s;
        if (int s = put(maps, 2 * k, wu, false, c.bn / 2, k)) return s;
        p.ph[0] = {0, k, 2 * k, z.nk(z.D), 0, 0, c.bn / 2, 0};
        p.used = (1u << 3 * k) - 1;
        if (int s = gate_output(maps, p, C, width, H)) return s;
        return launch(epilogue, c, z.split, maps, p, st, sums);
    }
    int forward(void* y, long long ldy, float* kept) {
        Args p = args(z.M, z.F);
        p.gu = kept;
        if (int s = gates(kGate, p, sp.H, z.Fp, nullptr)) return s;
        const Operand h{sp.H, z.M, z.F, z.Fp, z.M * z.Fp};
        const Choice c = z.down;
        const int k = z.planes();
        Maps maps;
        if (int s = put(maps, 0, h, false, 128, k)) return s;
        if (int s = put(maps, k, wd, false, c.bn / 2, k)) return s;
        Args q = args(z.M, z.O);
        q.ph[0] = {0, k, k, z.nk(z.F), 0, 0, c.bn, c.bn / 2};
        output(q, y, ldy);
        if (int s = launch(kStore, c, z.split, maps, q, st, sums)) return s;
        return add_up(sums, st);
    }
    int backward(const float* kept, void* dx, long long lddx, void* dwg, void* dwu, void* dwd) {
        const int k = z.planes();
        uint16_t *dgu = sp.dgu, *H = dwd ? sp.H : nullptr;
        {   // dH, and dG, dU, H either in its epilogue or in that of G and U
            const Choice c = z.dh;
            Maps maps;
            if (int s = put(maps, 0, dy, false, 128, k)) return s;
            if (int s = put(maps, k, wd, true, 64, k)) return s;
            Args p = args(z.M, z.F);
            p.ph[0] = {0, k, k, z.nk(z.O), 0, 1, c.bn, c.bn / 2};
            p.used = (1u << 2 * k) - 1;
            if (kept) {
                p.gu = const_cast<float*>(kept);
                if (int s = gate_output(maps, p, dgu, 2 * z.Fp, H)) return s;
                if (int s = launch(kGateBwdDH, c, z.split, maps, p, st, sums)) return s;
            } else {
                p.blocked = sp.dh;
                if (int s = launch(kStore, c, z.split, maps, p, st, sums)) return s;
                Args q = args(z.M, z.F);
                q.dh = sp.dh;
                if (int s = gates(kGateBwdGU, q, dgu, 2 * z.Fp, H)) return s;
            }
        }
        const Operand g{dgu, z.M, 2 * z.Fp, 2 * z.Fp, z.M * 2 * z.Fp};
        const Operand h{sp.H, z.M, z.F, z.Fp, z.M * z.Fp};
        if (dx) {
            const Choice c = z.dx;
            Maps maps;
            if (int s = put(maps, 0, g.columns(0, z.F), false, 128, k)) return s;
            if (int s = put(maps, k, g.columns(z.Fp, z.F), false, 128, k)) return s;
            if (int s = put(maps, 2 * k, wg, true, 64, k)) return s;
            if (int s = put(maps, 3 * k, wu, true, 64, k)) return s;
            Args p = args(z.M, z.D);
            p.nphase = 2;
            p.ph[0] = {0, 2 * k, 2 * k, z.nk(z.F), 0, 1, c.bn, c.bn / 2};
            p.ph[1] = {k, 3 * k, 3 * k, z.nk(z.F), 0, 1, c.bn, c.bn / 2};
            output(p, dx, lddx);
            if (int s = launch(kStore, c, z.split, maps, p, st, sums)) return s;
        }
        if (dwg || dwu) {
            Choice c = z.dwgu;
            const bool two = dwg && dwu;
            Maps maps;
            if (int s = put(maps, 0, g.columns(dwg ? 0 : z.Fp, z.F), true, 64, k)) return s;
            if (two)
                if (int s = put(maps, k, g.columns(z.Fp, z.F), true, 64, k)) return s;
            if (int s = put(maps, 2 * k, x, true, 64, k)) return s;
            Args p = args(z.F, z.D);
            p.groups = two ? 2 : 1;
            p.ph[0] = {0, 2 * k, 2 * k, z.nk(z.M), 1, 1, c.bn, c.bn / 2};
            p.part = sp.part_gu;
            output(p, dwg ? dwg : dwu, z.D);
            p.C[1] = dwu;
            if (int s = launch(kStore, c, z.split, maps, p, st, sums)) return s;
        }
        if (dwd) {
            const Choice c = z.dwd;
            Maps maps;
            if (int s = put(maps, 0, dy, true, 64, k)) return s;
            if (int s = put(maps, k, h, true, 64, k)) return s;
            Args p = args(z.O, z.F);
            p.ph[0] = {0, k, k, z.nk(z.M), 1, 1, c.bn, c.bn / 2};
            p.part = sp.part_d;
            output(p, dwd, z.F);
            if (int s = launch(kStore, c, z.split, maps, p, st, sums)) return s;
        }
        return add_up(sums, st);
    }
};

// A few rows: two products forward, which keep nothing; back, dH, then G and U again with dG, dU
// and H from them in fp32, dX and the weights' outer products.
int few_forward(Ff& f, const void* x, long long ldx, const void* wg, const void* wu, const void* wd,
                void* y, long long ldy) {
    const FfSizes& z = f.z;
    void* h = z.split ? (void*)f.sp.few_H : f.sp.H;
    few::Args p{};
    p.x = x, p.ldx = ldx, p.M = (int)z.M, p.K = z.D, p.N = z.F;
    p.w[0] = wg, p.w[1] = wu;
    p.act = f.act;
    p.out = h, p.ldo = z.Fp;
    p.dtype = z.dtype;
    if (int s = few::product(p, f.st)) return s;
    few::Args q{};
    q.x = h, q.ldx = z.Fp, q.M = (int)z.M, q.K = z.F, q.N = z.O;
    q.w[0] = wd;
    q.out = y, q.ldo = ldy;
    q.dtype = z.dtype;
    return few::product(q, f.st);
}
int few_backward(Ff& f, const void* x, long long ldx, const void* wg, const void* wu,
                 const void* wd, const void* dy, long long lddy, void* dx, long long lddx,
                 void* dwg, void* dwu, void* dwd) {
    const FfSizes& z = f.z;
    const int M = (int)z.M, t = z.dtype;
    const int s1 = few::down_shares(z.O, z.F, 32), s2 = few::down_shares(z.F, z.D);
    if (int s = few::down({{dy, nullptr}, lddy, 0, M, z.O, {wd, nullptr}, z.F, s1, f.sp.few_dh, t},
                          f.st))
        return s;
    few::Args p{};
    p.x = x, p.ldx = ldx, p.M = M, p.K = z.D, p.N = z.F;
    p.w[0] = wg, p.w[1] = wu;
    p.act = f.act;
    p.dtype = t;
    p.dh = f.sp.few_dh, p.dh_parts = s1, p.grads = f.sp.few_grads;
    if (int s = few::product(p, f.st)) return s;
    const long long n = (long long)M * z.F;
    const float *dg = f.sp.few_grads, *du = dg + n, *h = du + n;
    if (dx) {
        if (int s = few::down({{dg, du}, z.F, 1, M, z.F, {wg, wu}, z.D, s2, f.sp.few_dx, t}, f.st))
            return s;
        if (int s = few::sum({f.sp.few_dx, s2, M, z.D, dx, lddx, nullptr, nullptr, nullptr, 0, t},
                             f.st))
            return s;
    }
    few::OuterArgs o{};
    o.M = M, o.dtype = t;
    if (dwg) o.it[o.n++] = {dg, z.F, 1, z.F, x, ldx, 0, z.D, dwg};
    if (dwu) o.it[o.n++] = {du, z.F, 1, z.F, x, ldx, 0, z.D, dwu};
    if (dwd) o.it[o.n++] = {dy, lddy, 0, z.O, h, z.F, 1, z.F, dwd};
    return few::outer(o, f.st);
}

int check_ff(int dtype, int64_t M, int D, int F, int O, int act) {
    ATOM_REQUIRE(dtype >= ATOM_F32 && dtype <= ATOM_F16, "gated_ff: unknown type %d", dtype);
    ATOM_REQUIRE(M >= 0 && M < (1LL << 31) && D > 0 && F > 0 && O > 0, "gated_ff: bad sizes");
    ATOM_REQUIRE(D < (1 << 24) && F < (1 << 24) && O < (1 << 24), "gated_ff: widths above 2^24");
    ATOM_REQUIRE(act >= 0 && act <= 2, "gated_ff: act must be 0, 1 or 2");
    return ATOM_OK;
}

}  // namespace
}  // namespace atom

using namespace atom;

extern "C" int atom_gated_ff_bytes(int dtype, int64_t M, int D, int F, int O, size_t* bytes_host) {
    if (int s = check_ff(dtype, M, D, F, O, 0)) return s;
    ATOM_REQUIRE(bytes_host, "gated_ff: bytes_host is NULL");
    const FfSizes z(dtype, M, D, F, O, false);
    bytes_host[0] = FfSpace(nullptr, z, false).bytes;
    bytes_host[1] = FfSpace(nullptr, FfSizes(dtype, M, D, F, O, true), true).bytes;
    bytes_host[2] = (size_t)up(M, 32) * 2 * z.Fp * sizeof(float);
    return ATOM_OK;
}

extern "C" int atom_gated_ff_fwd(int dtype, const void* x, int64_t ldx, int64_t M, int D, int F,
                                 int O, const void* wg, const void* wu, const void* wd, int act,
                                 void* y, int64_t ldy, void* kept, void* ws, size_t ws_bytes,
                                 void* stream) {
    if (int s = check_ff(dtype, M, D, F, O, act)) return s;
    if (M == 0) return ATOM_OK;
    ATOM_REQUIRE(x && wg && wu && wd && y && ldx >= D && ldy >= O, "gated_ff: bad operand");
    const FfSizes z(dtype, M, D, F, O, false);
    Ff f{z, FfSpace(ws, z, false), (cudaStream_t)stream, act};
    ATOM_REQUIRE(ws && ws_bytes >= f.sp.bytes, "gated_ff: the workspace needs %zu bytes",
                 f.sp.bytes);
    ATOM_REQUIRE(aligned256(ws) && (M <= few::kFewRows || aligned256(kept)),
                 "gated_ff: ws and kept must be 256-byte aligned");
    if (z.few) return few_forward(f, x, ldx, wg, wu, wd, y, ldy);
    if (int s = f.inputs(x, ldx, wg, wu, wd)) return s;
    return f.forward(y, ldy, static_cast<float*>(kept));
}

extern "C" int atom_gated_ff_bwd(int dtype, const void* x, int64_t ldx, int64_t M, int D, int F,
                                 int O, const void* wg, const void* wu, const void* wd, int act,
                                 const void* dy, int64_t lddy, const void* kept, void* dx,
                                 int64_t lddx, void* dwg, void* dwu, void* dwd, void* ws,
                                 size_t ws_bytes, void* stream) {
    if (int s = check_ff(dtype, M, D, F, O, act)) return s;
    cudaStream_t st = (cudaStream_t)stream;
    if (M == 0) {
        const size_t e = dtype_size(dtype);
        for (void* p : {dwg, dwu})
            if (p) cudaMemsetAsync(p, 0, e * F * D, st);
        if (dwd) cudaMemsetAsync(dwd, 0, e * O * F, st);
        return check_launch("gated_ff", 0);
    }
    ATOM_REQUIRE(x && wg && wu && wd && dy && ldx >= D && lddy >= O && (!dx || lddx >= D),
                 "gated_ff: bad operand");
    const FfSizes z(dtype, M, D, F, O, true);
    Ff f{z, FfSpace(ws, z, true), st, act};
    ATOM_REQUIRE(ws && ws_bytes >= f.sp.bytes, "gated_ff: the workspace needs %zu bytes",
                 f.sp.bytes);
    ATOM_REQUIRE(aligned256(ws) && (M <= few::kFewRows || aligned256(kept)),
                 "gated_ff: ws and kept must be 256-byte aligned");
    if (z.few)
        return few_backward(f, x, ldx, wg, wu, wd, dy, lddy, dx, lddx, dwg, dwu, dwd);
    if (M <= few::kFewRows) kept = nullptr;          // the forward pass kept nothing
    if (int s = f.inputs(x, ldx, wg, wu, wd, dy, lddy, !kept || dwg || dwu)) return s;
    return f.backward(static_cast<const float*>(kept), dx, lddx, dwg, dwu, dwd);
}
