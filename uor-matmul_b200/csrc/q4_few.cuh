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

// Of up to 4 tokens an inner activation is kept as two of the 16-bit type, a rounded one and what
// that left, in two columns of the down product: the tensor instruction's eight have room for both,
// so the result lacks h's rounding for little (8 of 64 experts of 2048x1024: 1 token 19.9 -> 20.2
// us, 4 41.8 -> 42.5). More tokens take more eights of columns (5: 48.2 -> 52.6, 8: 68.9 -> 75.7)
// and average the rounding over more outputs; there h is rounded once.
inline int few_twice(int64_t tokens) { return tokens <= 4 ? 1 : 0; }

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
    void* h;             // up: [tokens * top_k][1 + twice][h_rs], every eight in the operands' order
    int twice;           // experts: 1 if an inner activation is two of the 16-bit type, see few_twice
    int64_t h_rs;        // n rounded up to 8
    float* part;         // part: [tokens * top_k][n]
    int codes_align;     // 16 if every row of codes begins at a multiple of 16 bytes
    int x_vec;           // rows of x begin at multiples of 16 bytes
    // Set by the launch:
    int columns;         // of a pass: 8 or 16
    int panel;           // chunks whose activations are resident
    int k_shift;         // log2 of the warps that share a tile's reduction
    int chunks, panels, groups, tiles;
    int group_shift;     // log2 of the group, or -1
    int quants_vec;      // a chunk's scales, and its zero points, are one vector each
};

// early: the launch may begin while the one before it runs; it reads what that wrote (the inner
// activations) only after its end.
int few_launch(uor_b200_ctx* ctx, int elem, FewParams& p, bool early);

// The same for what lies well (q4_lean.cu): whether it does, and then the launch's status.
bool lean_launch(uor_b200_ctx* ctx, int elem, FewParams& p, bool early, int* status);

}  // namespace uor
