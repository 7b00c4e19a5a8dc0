// Products of a few rows (up to kFewRows): streaming a weight matrix past rows that fit registers.
#pragma once

#include "typed.cuh"

namespace atom {
namespace few {

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
};
// Whether the matrices suit: 16-byte loads along rows of K.
bool suits(int dtype, long long M, int K, const void* x, long long ldx, const void* w0,
           const void* w1);
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

}  // namespace few
}  // namespace atom
