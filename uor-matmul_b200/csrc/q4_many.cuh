// q4_many.cuh -- products of many rows with 4-bit weights (q4_many.cu).
#pragma once
#include "q4.cuh"

namespace uor {

enum ManyMode {
    MANY_DENSE = 0,  // y[i][j] = x[i] . w[j]
    MANY_UP = 1,     // h[p][j] = silu(x[p] . gate[j]) (x[p] . up[j]) of the expert that sorted row p belongs to
    MANY_DOWN = 2    // part[pair][j] = h[p] . w[j], pair the one behind sorted row p
};

constexpr int MANY_MAX_EXPERTS = 1024;

struct ManyParams {
    Q4Dev w;
    const void* x;        // rows of the reduction's length: 16-byte aligned, contiguous within a row
    int64_t x_rs;
    int64_t x_rows;
    int mode;
    int n;                // outputs of a matrix: w.rows, f or d
    int experts;          // 1 for dense
    const int* offsets;   // [experts + 1] first sorted row of each expert; null for dense
    const int* perm;      // the pair behind each sorted row
    int m;                // dense: rows of x
    MatOut y;             // dense, without splits
    float* part;          // dense with splits: [splits][m][n]; down: [splits][pairs][n]
    int64_t part_rows;    // m or pairs
    void* h;              // up: [sorted rows][h_rs]
    int64_t h_rs;
    // Set by the launch:
    int max_cols;         // rows of x in a tile, a multiple of 64
    int row_tiles, splits, kb_per_split, groups;
    int* status;
    uint64_t budget_ns;
};

// The reduction is cut `splits` ways when a launch would otherwise leave processors idle; the
// caller provides `part` for many_splits' answer and adds the parts.
int many_splits(const uor_b200_ctx* ctx, const ManyParams& p);
// Status; early: after a kernel of the same call, and may begin while that one still runs. Codes and x have to be TMA-readable (16-byte aligned rows).
int many_launch(uor_b200_ctx* ctx, int elem, ManyParams p, bool early);

}  // namespace uor
