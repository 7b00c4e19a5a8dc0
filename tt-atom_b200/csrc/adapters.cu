// Low-rank adapters of many requests beside a shared projection, and their backward pass.
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

struct Requests {
    const int* ptr;
    const int* adapter;
    int n, nad;
    long long M;
};
// Rows of request r, kept within 0 .. M whatever the table holds.
__device__ __forceinline__ void request_rows(const Requests& q, int r, int& lo, int& hi) {
    const int top = (int)q.M;
    lo = min(max(q.ptr[r], 0), top);
    hi = min(max(q.ptr[r + 1], lo), top);
}

// out[m, r] = sum_k rows[m, k] W_a[r, k] with W_a = w + a * stride, element (r, k) at r*wr + k*wk
__global__ void shrink_kernel(Requests q, const void* rows, long long ld, int K, const void* w,
                              long long wr, long long wk, int R, float* out, int dtype) {
    int lo, hi;
    request_rows(q, blockIdx.x, lo, hi);
    const int a = q.adapter[blockIdx.x];
    const bool none = a < 0 || a >= q.nad;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (long long i = blockIdx.y * 8LL + warp; i < (long long)(hi - lo) * R; i += gridDim.y * 8LL) {
        const long long m = lo + i / R;
        const int r = (int)(i % R);
        float v = 0.f;
        if (!none)
            for (int k = lane; k < K; k += 32)
                v += load_f(rows, m * ld + k, dtype) *
                     load_f(w, (long long)a * R * K + r * wr + k * wk, dtype);
        v = warp_sum(v);
        if (lane == 0) out[m * R + r] = v;
    }
}

// out[m, n] += scale_a sum_r T[m, r] W_a(r, n); base fp32 [M, N], out typed
__global__ void expand_kernel(Requests q, const float* T, const void* w, long long wr,
                              long long wn, int R, int N, const float* scale, float* base,
                              int dtype) {
    int lo, hi;
    request_rows(q, blockIdx.x, lo, hi);
    const int a = q.adapter[blockIdx.x];
    if (a < 0 || a >= q.nad) return;
    for (long long m = lo + blockIdx.y; m < hi; m += gridDim.y)
        for (int n = threadIdx.x; n < N; n += blockDim.x) {
            float v = 0.f;
            for (int r = 0; r < R; ++r)
                v += T[m * R + r] * load_f(w, (long long)a * R * N + r * wr + n * wn, dtype);
            base[m * N + n] += scale[a] * v;
        }
}

__global__ void cast_kernel(const float* src, int N, void* dst, long long ld, long long M,
                            int dtype) {
    const long long n = M * N;
    for (long long i = blockIdx.x * 256LL + threadIdx.x; i < n; i += gridDim.x * 256LL)
        store_f(dst, i / N * ld + i % N, src[i], dtype);
}

// out[a](r, k) = scale_a sum_{m of a} T[m, r] rows[m, k], element (r, k) at r*orr + k*ok
__global__ void outer_kernel(Requests q, const float* T, const void* rows, long long ld, int K,
                             int R, const float* scale, void* out, long long orr, long long ok,
                             int dtype) {
    const int a = blockIdx.x;
    const int k = blockIdx.y * 128 + threadIdx.x;
    if (k >= K) return;
    for (int r = 0; r < R; ++r) {
        float v = 0.f;
        for (int j = 0; j < q.n; ++j) {
            if (q.adapter[j] != a) continue;
            int lo, hi;
            request_rows(q, j, lo, hi);
            for (long long m = lo; m < hi; ++m)
                v += T[m * R + r] * load_f(rows, m * ld + k, dtype);
        }
        store_f(out, (long long)a * R * K + r * orr + k * ok, scale[a] * v, dtype);
    }
}

}  // namespace atom

using namespace atom;

static int check_ad(int dtype, int64_t M, int D, int O, int nad, int R, int nreq) {
    ATOM_REQUIRE(dtype >= ATOM_F32 && dtype <= ATOM_F16, "adapted_linear: unknown type %d", dtype);
    ATOM_REQUIRE(M >= 0 && M < (1LL << 31) && D > 0 && O > 0 && nad >= 0 && nreq >= 0,
                 "adapted_linear: bad sizes");
    ATOM_REQUIRE(D < (1 << 24) && O < (1 << 24), "adapted_linear: widths above 2^24");
    ATOM_REQUIRE(R >= 1 && R <= 128, "adapted_linear: the rank must be 1..128");
    return ATOM_OK;
}

extern "C" int atom_adapted_linear_bytes(int dtype, int64_t M, int D, int O, int n_adapters,
                                         int R, int nreq, size_t* bytes_host) {
    if (int s = check_ad(dtype, M, D, O, n_adapters, R, nreq)) return s;
    ATOM_REQUIRE(bytes_host, "adapted_linear: bytes_host is NULL");
    Cursor f(nullptr), b(nullptr);
    f.take<float>(M * O);
    f.take<float>(M * R);
    b.take<float>(M * D);
    b.take<float>(M * R);
    b.take<float>(M * R);
    bytes_host[0] = f.used;
    bytes_host[1] = b.used;
    bytes_host[2] = 256;
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
    const bool adapted = nreq > 0 && n_adapters > 0;
    ATOM_REQUIRE(!adapted || (a && b && scale && req_ptr && req_adapter),
                 "adapted_linear: bad operand");
    cudaStream_t st = (cudaStream_t)stream;
    Cursor c(ws);
    float* base = c.take<float>(M * O);
    float* S = c.take<float>(M * R);
    ATOM_REQUIRE(ws && ws_bytes >= c.used, "adapted_linear: the workspace needs %zu bytes", c.used);
    if (int s = plain_product({x, ldx, 1, dtype, w, D, 1, dtype, base, O, 0, M, O, D}, st))
        return s;
    Requests q{req_ptr, req_adapter, nreq, n_adapters, M};
    if (adapted) {
        shrink_kernel<<<dim3(nreq, 16), 256, 0, st>>>(q, x, ldx, D, a, D, 1, R, S, dtype);
        ATOM_CHECK_LAUNCH("adapters shrink");
        expand_kernel<<<dim3(nreq, 16), 128, 0, st>>>(q, S, b, 1, R, R, O, scale, base, dtype);
        ATOM_CHECK_LAUNCH("adapters expand");
    }
    cast_kernel<<<1024, 256, 0, st>>>(base, O, y, ldy, M, dtype);
    return check_launch("adapters cast");
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
    if (M == 0 || nreq == 0 || n_adapters == 0) {
        if (da) cudaMemsetAsync(da, 0, e * n_adapters * R * D, st);
        if (db) cudaMemsetAsync(db, 0, e * n_adapters * R * O, st);
        if (int s = check_launch("adapters", 0)) return s;
    }
    if (M == 0) return ATOM_OK;
    ATOM_REQUIRE(x && w && dy && ldx >= D && lddy >= O && (!dx || lddx >= D),
                 "adapted_linear: bad operand");
    const bool adapted = nreq > 0 && n_adapters > 0;
    ATOM_REQUIRE(!adapted || (a && b && scale && req_ptr && req_adapter),
                 "adapted_linear: bad operand");
    Cursor c(ws);
    float* base = c.take<float>(M * D);
    float* S = c.take<float>(M * R);
    float* T = c.take<float>(M * R);
    ATOM_REQUIRE(ws && ws_bytes >= c.used, "adapted_linear: the workspace needs %zu bytes", c.used);
    Requests q{req_ptr, req_adapter, nreq, n_adapters, M};
    if (adapted) {
        shrink_kernel<<<dim3(nreq, 16), 256, 0, st>>>(q, dy, lddy, O, b, 1, R, R, T, dtype);
        ATOM_CHECK_LAUNCH("adapters shrink");
        if (db) {
            shrink_kernel<<<dim3(nreq, 16), 256, 0, st>>>(q, x, ldx, D, a, D, 1, R, S, dtype);
            ATOM_CHECK_LAUNCH("adapters shrink");
            outer_kernel<<<dim3(n_adapters, ceil_div(O, 128)), 128, 0, st>>>(
                q, S, dy, lddy, O, R, scale, db, 1, R, dtype);
            ATOM_CHECK_LAUNCH("adapters outer");
        }
        if (da) {
            outer_kernel<<<dim3(n_adapters, ceil_div(D, 128)), 128, 0, st>>>(
                q, T, x, ldx, D, R, scale, da, D, 1, dtype);
            ATOM_CHECK_LAUNCH("adapters outer");
        }
    }
    if (!dx) return ATOM_OK;
    if (int s = plain_product({dy, lddy, 1, dtype, w, 1, D, dtype, base, D, 0, M, D, O}, st))
        return s;
    if (adapted) {
        expand_kernel<<<dim3(nreq, 16), 128, 0, st>>>(q, T, a, D, 1, R, D, scale, base, dtype);
        ATOM_CHECK_LAUNCH("adapters expand");
    }
    cast_kernel<<<1024, 256, 0, st>>>(base, D, dx, lddx, M, dtype);
    return check_launch("adapters cast");
}
