// q4_gemm.cu -- products with 4-bit weights and group scales.
//
// y[i][j] = sum_p x[i][p] scale[j][p / g] (code[j][p] - zero[j][p / g]). The plainest kernel: a
// warp per output, lanes over the reduction's bytes, f32 sums, a shuffle tree at the end.
#include "q4.cuh"
#include "q4_few.cuh"

namespace uor {

// One lane's share of sum_p x[p cs] w[row][p].
template <typename T>
__device__ __forceinline__ float q4_dot(const T* x, int64_t cs, const Q4Dev& w, int64_t row, int lane) {
    const uint8_t* codes = w.codes + row * w.row_bytes;
    float sum = 0;
    for (int b = lane; b < (w.cols + 1) / 2; b += 32) {
        const int g = 2 * b / w.group;
        const float scale = load_f32(w.scales, row * w.groups_rs + g, w.scale_type);
        const int zero = w.zeros ? w.zeros[row * w.groups_rs + g] & 15 : 8;
        const int code = codes[b];
        float part = to_f32(x[2 * b * cs]) * static_cast<float>((code & 15) - zero);
        if (2 * b + 1 < w.cols)
            part = fmaf(to_f32(x[(2 * b + 1) * cs]), static_cast<float>((code >> 4) - zero), part);
        sum = fmaf(part, scale, sum);
    }
    return sum;
}

__device__ __forceinline__ float warp_sum(float v) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <typename T>
__global__ void q4_simple(Mat x, Q4Dev w, MatOut y, int64_t m) {
    const int lane = threadIdx.x & 31;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int64_t i = at / w.rows, j = at % w.rows;
    if (i >= m) return;
    const float s = warp_sum(q4_dot(static_cast<const T*>(x.p) + i * x.rs, x.cs, w, j, lane));
    if (lane == 0) store_f32(y.p, i * y.rs + j * y.cs, y.type, s);
}

template <typename T>
__global__ void ffn_up_simple(FfnArgs a, T* h) {
    const int lane = threadIdx.x & 31;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int64_t pair = at / a.f, j = at % a.f, t = pair / a.top_k;
    if (t >= a.tokens) return;
    const int64_t e = static_cast<const int32_t*>(a.ids.p)[t * a.ids.rs + pair % a.top_k * a.ids.cs];
    if (e < 0 || e >= a.experts) return;
    const T* x = static_cast<const T*>(a.x.p) + t * a.x.rs;
    const float gate = warp_sum(q4_dot(x, a.x.cs, a.up, e * 2 * a.f + j, lane));
    const float up = warp_sum(q4_dot(x, a.x.cs, a.up, e * 2 * a.f + a.f + j, lane));
    if (lane == 0) h[pair * a.f + j] = from_f32<T>(silu(gate) * up);
}

template <typename T>
__global__ void ffn_down_simple(FfnArgs a, const T* h) {
    const int lane = threadIdx.x & 31;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int64_t t = at / a.d, j = at % a.d;
    if (t >= a.tokens) return;
    float total = 0;
    for (int s = 0; s < a.top_k; ++s) {
        const int64_t e = static_cast<const int32_t*>(a.ids.p)[t * a.ids.rs + s * a.ids.cs];
        if (e < 0 || e >= a.experts) continue;
        const float weight = static_cast<const float*>(a.weights.p)[t * a.weights.rs + s * a.weights.cs];
        const float v = warp_sum(q4_dot(h + (t * a.top_k + s) * a.f, 1, a.down, e * a.d + j, lane));
        total = fmaf(weight, v, total);
    }
    if (lane == 0) store_f32(a.y.p, t * a.y.rs + j * a.y.cs, a.y.type, total);
}

// What the few-rows kernel's vector loads may rely on.
static void few_align(FewParams* p) {
    const uint64_t codes = reinterpret_cast<uint64_t>(p->w.codes) | static_cast<uint64_t>(p->w.row_bytes);
    p->codes_align = codes % 16 == 0 ? 16 : 1;
    p->x_vec = (reinterpret_cast<uint64_t>(p->x) | static_cast<uint64_t>(p->x_rs * 2)) % 16 == 0;
}

static unsigned blocks_for(int64_t warps) { return static_cast<unsigned>((warps + 7) / 8); }

int run_q4_gemm(uor_b200_ctx* ctx, int elem, const Mat& x, int64_t m, const Q4Dev& w, const MatOut& y,
                uor_b200_route* route) {
    route->kernel = UOR_B200_KERNEL_Q4;
    if (m <= 8 && x.cs == 1 && w.cols > 0) {
        FewParams p{};
        p.w = w;
        p.x = x.p;
        p.x_rs = x.rs;
        p.m = m;
        p.n = w.rows;
        p.y = y;
        few_align(&p);
        return few_launch(ctx, elem, FEW_DENSE, p, false);
    }
    const unsigned grid = blocks_for(m * w.rows);
    if (elem == UOR_B200_BF16)
        q4_simple<__nv_bfloat16><<<grid, 256, 0, ctx->stream>>>(x, w, y, m);
    else
        q4_simple<__half><<<grid, 256, 0, ctx->stream>>>(x, w, y, m);
    return cuda_status(cudaGetLastError());
}

template <typename T>
static int ffn_typed(uor_b200_ctx* ctx, const FfnArgs& a) {
    int st = UOR_B200_OK;
    T* h = static_cast<T*>(ctx_buffer(ctx, SLOT_WS, static_cast<size_t>(a.tokens) * a.top_k * a.f * 2, &st));
    if (!h) return st;
    if (a.top_k && a.f)
        ffn_up_simple<T><<<blocks_for(a.tokens * a.top_k * a.f), 256, 0, ctx->stream>>>(a, h);
    ffn_down_simple<T><<<blocks_for(a.tokens * a.d), 256, 0, ctx->stream>>>(a, h);
    return cuda_status(cudaGetLastError());
}

int run_expert_ffn(uor_b200_ctx* ctx, const FfnArgs& a, uor_b200_route* route) {
    route->kernel = UOR_B200_KERNEL_Q4;
    if (a.tokens <= FEW_MAX_TOKENS && a.tokens * a.top_k <= FEW_MAX_PAIRS && a.top_k > 0 && a.f > 0 && a.x.cs == 1) {
        int st = UOR_B200_OK;
        FewParams p{};
        p.h = ctx_buffer(ctx, SLOT_WS, static_cast<size_t>(a.tokens) * a.top_k * ((a.f + 7) / 8 * 8) * 2, &st);
        if (!p.h) return st;
        p.h_rs = (a.f + 7) / 8 * 8;
        p.w = a.up;
        p.x = a.x.p;
        p.x_rs = a.x.rs;
        p.n = a.f;
        p.ids = a.ids;
        p.weights = a.weights;
        p.tokens = static_cast<int>(a.tokens);
        p.top_k = a.top_k;
        p.experts = a.experts;
        few_align(&p);
        if ((st = few_launch(ctx, a.elem, FEW_UP, p, false))) return st;
        p.w = a.down;
        p.x = p.h;
        p.x_rs = p.h_rs;
        p.n = a.d;
        p.y = a.y;
        few_align(&p);
        return few_launch(ctx, a.elem, FEW_DOWN, p, true);
    }
    return a.elem == UOR_B200_BF16 ? ffn_typed<__nv_bfloat16>(ctx, a) : ffn_typed<__half>(ctx, a);
}

}  // namespace uor
