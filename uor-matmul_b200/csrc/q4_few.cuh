// q4_few.cuh -- products of few rows with 4-bit weights (q4_few.cu).
#pragma once
#include "q4.cuh"

namespace uor {

// What one launch of the few-rows kernel computes.
enum FewKind {
    FEW_DENSE = 0,  // y[i][j] = x[i] . w[j]
    FEW_UP = 1,     // h[pair][j] = silu(x[t] . gate[j]) (x[t] . up[j]) of each chosen expert
    FEW_PART = 2    // part[pair][j] = h[pair] . w[j]
};

constexpr int FEW_MAX_PAIRS = 1024;    // tokens * top_k with experts
constexpr int FEW_MAX_EXPERTS = 1024;  // a word of bits to a lane

struct FewParams {
    Q4Dev w;
    int kind;
    const void* x;       // rows of the reduction's length, contiguous
    int64_t x_rs;
    int64_t m;           // dense: rows of x
    int n;               // outputs of a matrix: w.rows, f or d
    MatOut y;            // dense
    Mat ids;             // experts
    int tokens, top_k, experts;
    void* h;             // up: [tokens * top_k][h_rs], every eight in the operands' order
    int64_t h_rs;        // n rounded up to 8
    float* part;         // part: [tokens * top_k][n]
    int codes_align;     // 16 if every row of codes begins at a multiple of 16 bytes
    int x_vec;           // rows of x begin at multiples of 16 bytes
    // Set by the launch:
    int panel;           // chunks whose activations are resident
    int k_shift;         // log2 of the warps that share a tile's reduction
    int chunks, panels, groups, tiles;
    int group_shift;     // log2 of the group, or -1
    int quants_vec;      // a chunk's scales, and its zero points, are one vector each
};

// early: the launch may begin while the one before it runs; it reads what that wrote (the inner
// activations) only after its end.
int few_launch(uor_b200_ctx* ctx, int elem, FewParams p, bool early);

// The same for what lies well (q4_lean.cu): whether it does, and then the launch's status.
bool lean_launch(uor_b200_ctx* ctx, int elem, FewParams p, bool early, int* status);

}  // namespace uor
