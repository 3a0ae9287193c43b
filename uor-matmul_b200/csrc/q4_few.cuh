// q4_few.cuh -- products of few rows with 4-bit weights (q4_few.cu).
#pragma once
#include "q4.cuh"

namespace uor {

// What one launch of the few-rows kernel computes.
enum FewMode {
    FEW_DENSE = 0,  // y[i][j] = x[i] . w[j]
    FEW_UP = 1,     // h[pair][j] = silu(x[t] . gate[j]) (x[t] . up[j]) of each chosen expert
    FEW_DOWN = 2    // y[t][j] = sum over the token's choices of weight (h[pair] . w[j])
};

struct FewParams {
    Q4Dev w;
    const void* x;       // rows of the reduction's length, contiguous
    int64_t x_rs;
    int64_t m;           // dense: rows of x
    int n;               // outputs: w.rows, f or d
    MatOut y;            // dense and down
    Mat ids, weights;    // experts
    int tokens, top_k, experts;
    void* h;             // up: [tokens * top_k][h_rs], every eight in the operands' order
    int64_t h_rs;        // n rounded up to 8
    int codes_align;     // 16 if every row of codes begins at a multiple of 16 bytes
    int x_vec;           // rows of x begin at multiples of 16 bytes
    // Set by the launch:
    int panel;           // chunks whose activations are resident
    int group_shift;     // log2 of the group, or -1
    int quants_vec;      // a chunk's scales, and its zero points, are one vector each
};

constexpr int FEW_MAX_PAIRS = 256;  // tokens * top_k of the experts' modes
constexpr int FEW_MAX_TOKENS = 8;

int few_launch(uor_b200_ctx* ctx, int elem, FewMode mode, FewParams p, bool after_up);

}  // namespace uor
