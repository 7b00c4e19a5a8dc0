// Host side of the pair products (pair_product.cu): operands, tile choice, launches.
#pragma once

#include <cuda.h>

#include "typed.cuh"

namespace atom {
namespace pair {

// Tensor maps of a product whose operands have `planes` planes (16-bit: one): up to four operands,
// the outputs (two groups, or a gate's planes), H, partial sums.
constexpr int out_map(int planes) { return 4 * planes; }
constexpr int h_map(int planes) { return 5 * planes; }
constexpr int part_map(int planes) { return 6 * planes; }
template <int N>
struct MapArray {
    CUtensorMap m[N];
};
using Maps = MapArray<part_map(kPlanes) + 1>;

// One run of K stages: operands by map index (SPLIT: the other planes' maps are the next ones).
struct Phase {
    int a, b0, b1;           // A; B of CTA 0 and of CTA 1
    int nk;                  // 64-deep stages
    int a_mn, b_mn;          // 1: M/N-major
    int bstep, brank;        // B's first row: column tile * bstep + CTA * brank
};

// kLow: the requests' low-rank rows themselves: of each row tile, times the adapters of its pieces,
// 16 columns a slice (ph[0].b0: the adapters' map). kStoreLow: kStore with low-rank blocks beside the
// phases.
enum Epilogue { kStore = 0, kGate = 1, kGateBwdGU = 2, kGateBwdDH = 3, kLow = 4, kStoreLow = 5 };

// A row tile's first stage of low-rank blocks, by its number and its first request's: tiles need at
// most a stage more than a quarter of their pieces' slices.
__host__ __device__ inline long long first_stage(long long tile, long long request, int ext) {
    return (tile + request) * ext / 4 + tile;
}

struct Args {
    long long M;             // rows of the output (of one group)
    int N;                   // its columns (gate epilogues: F)
    int mtiles, ntiles_n;    // tiles of one group
    int groups;              // outputs stacked along M: A's map index and C of group g
    long long tiles;         // all work items
    int ksplit;
    int nphase;
    Phase ph[2];
    int bf16;                // operand type of the products: 1 bf16, 0 fp16
    void* C[2];
    long long ldc;
    int dtype;               // C's type
    int tma;                 // kStore: C (the partial sums) by TMA
    unsigned used;           // maps to prefetch
    float* blocked;          // kStore: fp32 to 32 x 32 lane blocks instead of C
    float* part;             // ksplit > 1: [split][group][M][N] fp32
    int act;
    float* gu;               // gate: kept g, and u gu_half further, lane blocks, or NULL
    long long gu_half;
    float* dh;               // kGateBwdGU: lane blocks
    int H;                   // gate backward: H wanted (its map; dG | dU: the output's, u at Fp)
    int Fp;
    // Low-rank blocks beside the phases: a row tile's requests that share an adapter have one, led
    // by the first of them, of `ext` slices of 16 ranks, zero in the other rows. A tile's blocks lie
    // slice by slice, four to a stage of 256 rows x 64, from stage first_stage() on.
    int ext;                 // slices a block, 0: none
    int nad;                 // adapters
    int ext_a, ext_b, ext_bmn;
    int4* tile_req;          // of a row tile: its requests' first and behind, its blocks; and, from
                             // kLow on, whether one's adapter is not finite
    const int4* piece;       // t + r, of request r in tile t: adapter or -1 (none), its rows
    const int2* lead;        // t + first + j, of tile t's j-th block: its adapter, the request that
                             // leads it
    const int* row_lead;     // per row: the request whose block it is in, -1: none
    int* usable;             // from kLow on: as lead, but nad where the adapter is not finite
    const int4* bad;         // of an adapter: not all zero = not finite, its rows become NaN
    const float* low_scale;  // kLow: per adapter
    void* low_block;         // kLow: [stage][256][64] 16-bit (SPLIT: planes low_plane apart), or NULL
    long long low_plane;
    void* low_rows;          // kLow: [M][Rs] typed, or NULL
    int Rs;
    int* err;
};

// Tile width, K splits and the partial sums' floats of one product.
struct Choice {
    int bn, ksplit;
    size_t part;
};
Choice choose(long long M, int N, int nk, int groups, bool gated, bool split, bool may_split);

// Tensor map of a 16-bit matrix [rows, cols] with rows ld elements apart (16-byte aligned); boxes
// of 64 x box_rows.
int make_map(CUtensorMap* m, const void* p, long long cols, long long rows, long long ld,
             int box_rows);
// The same for low-rank slices, of `depth` matrices `ldz` elements apart where depth > 0: boxes of
// 16 x box_rows, or of 64 x 16 where K runs along the rows (mn).
int make_slice_map(CUtensorMap* m, const void* p, long long cols, long long rows, long long ld,
                   int box_rows, bool mn, int depth, long long ldz);
// kLow's adapters [depth][rows = R][cols = K], or [depth][rows = K][cols = R] (mn).
int make_low_map(CUtensorMap* m, const void* p, long long cols, long long rows, long long ld, bool mn,
                 int depth, long long ldz);
// Map of an output [rows, cols] that is written in blocks of 32 x 32.
int make_out_map(CUtensorMap* m, const void* p, int dtype, long long cols, long long rows,
                 long long ld);

int pair_count();            // CTA pairs that the current device runs at a time

// The outputs of products whose K was split, to be added up in one launch.
struct Sums {
    struct Item {
        const float* part;
        uint32_t M, N, groups;
        int ksplit;
        void* C[2];
        long long ldc;
    } it[3];
    int n = 0, dtype = 0;
};
int add_up(Sums& sums, Chain& st);

// Launches the product: tiles, C's maps (kStore) etc. are filled in from M, N, C and the choice. The
// sums of a split K go into the list.
int launch(int epilogue, const Choice& c, bool split, Maps& maps, Args& p, Chain& st, Sums& sums);

// Operand preparation, up to 6 matrices a launch: 16-bit copies (kPack) or an fp32 matrix's planes
// (kSplit).
enum Prep { kPack = 0, kSplit = 1 };
struct PrepItem {
    const void* src;
    long long rows, cols, ld;
    void* dst;               // [rows][dld], planes `plane` elements apart
    long long dld, plane;
    int mode;
};
constexpr int kPrepBlocks = 1184;            // of one launch and item, at most
struct PrepList {
    PrepItem it[6];
    int n = 0, blocks[6];
    void add(const PrepItem& i) { it[n++] = i; }
};

// The pieces of an adapters call's requests (adapters.cu), found in a preparation launch beside its
// matrices.
struct Pieces {
    const int *ptr, *adapter;
    int n, nad, M;           // requests, adapters, rows
    int tiles, pieces;       // row tiles; and requests
    int4* piece;             // adapter or -1, first row, behind the last row
    int2* lead;              // as in Args, like the next two
    int* row_lead;
    int4* tile_req;
    const void* other;       // the matrix of each adapter beside the projection: `other_n` values
    long long other_n;
    int4* bad;               // per adapter: a quarter of them is not finite
    int dtype;
};
int prepare(PrepList& l, Chain& st, const Pieces* pieces = nullptr);      // empties the list

inline bool tma_ready(const void* p, long long ld) { return aligned16(p) && ld % 8 == 0; }
inline long long up(long long n, long long k) { return (n + k - 1) / k * k; }

}  // namespace pair
}  // namespace atom
