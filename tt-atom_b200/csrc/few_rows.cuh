// Products of a few rows: streaming a weight matrix past rows that fit registers.
#pragma once

#include "typed.cuh"

namespace atom {
namespace few {

// One tensor-core tile's rows. (fp32 with 32, measured against planes: 75 us for 62 at
// 22 x 752 x 1280 backward, 248 for 196 at 27 x 1173 x 6032.)
constexpr int kFewRows = 16;

struct Args {
    const void* x;           // [M, K]
    long long ldx;
    int M, K;
    const void* w[2];        // [N, K]; w[1]: the u matrix of a gate, or NULL
    int N;
    int act;
    void* out;               // [M, N]
    long long ldo;
    int dtype;
    // low-rank part: out += S[m, :] . b[slot[m]][n, :]
    const float* S;          // [M][R], scaled, or NULL
    const int* slot;         // [M], -1: none
    const void* b;           // [adapters][N][R]
    int R;
    // a gate's backward pass: dh as partial sums, and dg, du, h [3][M][N] instead of out
    const float* dh;         // [dh_parts][M][N], or NULL
    int dh_parts;
    float* grads;
};
int product(const Args& p, Chain& st);

// S[m, r] = scale x[m] . a[slot][r], and each row's adapter.
struct LowArgs {
    const void* x;
    long long ldx;
    int M, K;
    const void* a;           // [adapters][R][K]
    int R;
    const float* scale;
    const int* ptr;
    const int* adapter;
    int nreq, nad;
    float* S;
    int* slot;
    int dtype;
};
int low_rank(const LowArgs& p, Chain& st);
// T[m, r] = scale dy[m] . b[slot][:, r] for the rows' adapters.
struct LowBackArgs {
    const void* dy;
    long long ld;
    int M, O;
    const void* b;           // [adapters][O][R]
    int R;
    const float* scale;
    const int* slot;
    float* T;
    int dtype;
};
int low_rank_back(const LowBackArgs& p, Chain& st);

// part[s][m, n] = sum over a share of k of a[m, k] w[k, n] (and of a second pair): the products
// whose sum runs along the weights' rows, down their columns.
struct DownArgs {
    const void* a[2];        // [M, K], fp32 where a32, else typed; a[1] may be NULL
    long long lda;
    int a32, M, K;
    const void* w[2];        // [K, N]
    int N, shares;
    float* part;
    int dtype;
};
int down_shares(int K, int N, int most = 592);
int down(const DownArgs& p, Chain& st);
// out[m, n] = the shares' sum (+ T[m, :] . a[slot[m]][:, n])
struct SumArgs {
    const float* part;
    int shares, M, N;
    void* out;
    long long ldo;
    const float* T;
    const int* slot;
    const void* a;
    int R, dtype;
};
int sum(const SumArgs& p, Chain& st);

// out[i, j] = sum over the rows m of p[m, i] q[m, j], up to three of them a launch.
struct OuterItem {
    const void* p;
    long long ldp;
    int p32, I;              // p32: fp32 whatever the type
    const void* q;
    long long ldq;
    int q32, J;
    void* out;
};
struct OuterArgs {
    OuterItem it[3];
    int n, M, dtype, first[4];
};
int outer(OuterArgs p, Chain& st);
// dA[a][r, d] = sum over a's rows of T[m, r] x[m, d]; dB[a][o, r] the same of S and dy.
struct GradArgs {
    const float *T, *S;
    const int* slot;
    const void *x, *dy;
    long long ldx, lddy;
    int M, D, O, R, nad;
    void *da, *db;
    int dtype;
};
int adapter_grads(const GradArgs& p, Chain& st);

}  // namespace few
}  // namespace atom
