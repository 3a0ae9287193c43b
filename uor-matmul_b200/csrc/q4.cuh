// q4.cuh -- 4-bit weights with group scales: the device-side descriptor and conversions.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstddef>
#include <cstdint>
#include "internal.h"

namespace uor {

// uor_b200_q4 after staging: device pointers and checked extents.
struct Q4Dev {
    const uint8_t* codes;
    const void* scales;
    const uint8_t* zeros;  // null: every zero point is 8
    int64_t row_bytes, groups_rs;
    int rows, cols, group;
    int scale_type;        // uor_b200_dtype: F32, BF16 or F16
};

// A strided matrix on the device; the element type is known from elsewhere.
struct Mat {
    const void* p;
    int64_t rs, cs;
};
struct MatOut {
    void* p;
    int64_t rs, cs;
    int type;  // uor_b200_dtype: F32, BF16 or F16
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// An element of a buffer whose type is a run-time tag.
__device__ __forceinline__ float load_f32(const void* p, int64_t i, int type) {
    if (type == UOR_B200_F32) return static_cast<const float*>(p)[i];
    if (type == UOR_B200_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_f32(void* p, int64_t i, int type, float v) {
    if (type == UOR_B200_F32)
        static_cast<float*>(p)[i] = v;
    else if (type == UOR_B200_BF16)
        static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else
        static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// What a sum of codes' products is multiplied by in the end. bfloat16 activations reach f32's own
// range, and a group's codes, before the scale that makes weights of them, would carry their sum
// past it: there a code is held as 2^-12 of itself, exactly, so that 128 positions of 15 times the
// largest activation still fit. Powers of two change no rounding but among f32's denormals: results
// below 2^-114 keep 2^-137 absolute. Multiplied in the end, it costs nothing that was measured.
template <typename T>
struct CodeUnit {
    static constexpr float VALUE = 1.0f;
};
template <>
struct CodeUnit<__nv_bfloat16> {
    static constexpr float VALUE = 4096.0f;
};

__device__ __forceinline__ float silu(float v) { return v / (1.0f + expf(-v)); }

// What follows a product before its rounding (uor_b200_q4_linear): act(v + bias[j]) + residual[i][j].
// Where `on` is 0 there is none of it.
struct Epilogue {
    int on;
    int act;             // uor_b200_activation
    const void* bias;    // null: none
    int bias_type;
    Mat residual;        // of the output's type; p null: none
};
// v / (1 + e), e = exp(-u), without the exact quotient's branch, at which a thread's elements would
// wait for one another; both sides are a quarter, since the fast quotient is 0 beyond 2^126.
__device__ __forceinline__ float over_one_and(float v, float e) { return __fdividef(0.25f * v, fmaf(0.25f, e, 0.25f)); }
__device__ __forceinline__ float activate(float v, int act) {
    switch (act) {
    case UOR_B200_RELU: return v < 0.0f ? 0.0f : v;
    case UOR_B200_GELU: return 0.5f * v * erfcf(-0.70710678118654752f * v);  // 1 + erf, its tail included
    case UOR_B200_GELU_TANH:  // (1 + tanh z) / 2 = 1 / (1 + exp(-2 z))
        return over_one_and(v, expf(-1.5957691216057308f * fmaf(0.044715f * v * v, v, v)));
    case UOR_B200_SILU: return over_one_and(v, expf(-v));
    default: return v;
    }
}
// The output at (i, j) from its product. What it reads is asked for before anything waits for it.
__device__ __forceinline__ float follow_up(const Epilogue& e, int type, int64_t i, int64_t j, float v) {
    const float bias = e.bias ? load_f32(e.bias, j, e.bias_type) : 0.0f;
    const float residual = e.residual.p ? load_f32(e.residual.p, i * e.residual.rs + j * e.residual.cs, type) : 0.0f;
    if (e.bias) v += bias;
    v = activate(v, e.act);
    return e.residual.p ? v + residual : v;
}

// y (m x n) = x (m x k of elem) dequant(w)^T, and what follows it.
int run_q4_gemm(uor_b200_ctx* ctx, int elem, const Mat& x, int64_t m, const Q4Dev& w, const Epilogue& e, const MatOut& y,
                uor_b200_route* route);

// The experts' gated feed-forward layer (uor_b200_expert_q4_ffn).
struct FfnArgs {
    int elem;
    int64_t tokens;
    int top_k, experts, d, f;
    Mat x, ids, weights;
    Q4Dev up, down;
    MatOut y;
};
int run_expert_ffn(uor_b200_ctx* ctx, const FfnArgs& a, uor_b200_route* route);

// The router and its gradient (expert_route.cu).
struct RouterArgs {
    uor_b200_router r;
    int64_t tokens;
    int elem;
    Mat logits;
    const float* bias;
    MatOut ids, weights;            // forward
    Mat in_ids, dweights;           // backward
    MatOut dlogits;
    // Set by the launch:
    bool vec, vec_out;              // rows of logits (of dlogits) are whole vectors
    int group_size;
    int lane_shift;                 // log2 of the lanes that hold a group, or -1 where they do not hold one alone
};
int run_expert_route(uor_b200_ctx* ctx, const RouterArgs& a, uor_b200_route* route);
int run_expert_route_backward(uor_b200_ctx* ctx, const RouterArgs& a, uor_b200_route* route);

}  // namespace uor
