// expert_route.cu -- the experts' router and the gradient of its logits.
//
// A warp per token. Lane l holds the experts l, l + 32, ...; a key is ordered as an unsigned
// integer (the float's bits, negative ones complemented), so that the largest key is one
// warp-wide integer maximum and the lowest index among its equals one minimum. What is closed
// (a logit or key of -inf or NaN) is key 0, below every open one.
#include "q4.cuh"

namespace uor {

namespace {

constexpr unsigned FULL = 0xffffffffu;

__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t b = __float_as_uint(v);
    return b ^ (b & 0x80000000u ? FULL : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// The key of an open value, or 0.
__device__ __forceinline__ uint32_t open_key(float v) { return v > -INFINITY ? order_key(v) : 0u; }

__device__ __forceinline__ float warp_sum(float v) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
    return v;
}

// exp(l - top) with the infinities' differences as limits have them: equal ones give 1.
__device__ __forceinline__ float exp_below(float l, float top) { return l == top ? 1.0f : expf(l - top); }

__device__ __forceinline__ float sigmoid(float l) { return 1.0f / (1.0f + expf(-l)); }

// The chosen experts' shares of their scores' sum; lane s holds choice s (open: whether it is
// one). They are taken relative to the largest chosen logit, so that scores which underflow
// still have shares: exp(l) / exp(m) for the softmax, and, as sigmoid(l) = exp(min(l, 0)) /
// (1 + exp(-|l|)), that over exp(m) for the sigmoid. A sigmoid's m ends at -700: below it (the
// lowest finite logit, which masks carry) a score is 0 in any precision and has no share.
__device__ __forceinline__ float chosen_share(float l, bool open, bool softmax) {
    const uint32_t k = __reduce_max_sync(FULL, open ? open_key(l) : 0u);
    const float top = k ? key_value(k) : 0.0f;
    float w = 0;
    if (open)
        w = softmax ? exp_below(l, top)
                    : expf(fminf(l, 0.0f) - fmaxf(fminf(top, 0.0f), -700.0f)) / (1.0f + expf(-fabsf(l)));
    const float sum = warp_sum(w);
    return sum > 0 ? w / sum : 0.0f;
}

// A row's largest open logit and the sum of exp(l - top) over the open ones.
template <int VPL>
__device__ __forceinline__ void softmax_of(const float (&l)[VPL], float* top, float* total) {
    uint32_t k = 0;
#pragma unroll
    for (int i = 0; i < VPL; ++i) k = max(k, open_key(l[i]));
    k = __reduce_max_sync(FULL, k);
    *top = k ? key_value(k) : 0.0f;
    float s = 0;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
        if (l[i] > -INFINITY) s += exp_below(l[i], *top);
    *total = warp_sum(s);
}

template <typename T, int VPL>
__device__ __forceinline__ void load_row(float (&l)[VPL], const Mat& m, int64_t t, int experts, int lane) {
    const T* p = static_cast<const T*>(m.p) + t * m.rs;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const int e = lane + 32 * i;
        l[i] = e < experts ? to_f32(p[e * m.cs]) : -INFINITY;
    }
}

// The largest of the warp's keys and the lowest expert that has it.
template <int VPL>
__device__ __forceinline__ uint32_t warp_best(const uint32_t (&key)[VPL], int lane, int* expert) {
    uint32_t k = 0;
    int at = 0;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
        if (key[i] > k) k = key[i], at = lane + 32 * i;
    const uint32_t best = __reduce_max_sync(FULL, k);
    *expert = static_cast<int>(__reduce_min_sync(FULL, k == best ? static_cast<unsigned>(at) : FULL));
    return best;
}

template <typename T, int VPL>
__global__ void route_kernel(RouterArgs a) {
    const int lane = threadIdx.x & 31;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (t >= a.tokens) return;
    const int experts = a.r.experts, top_k = a.r.top_k;
    float l[VPL];
    load_row<T>(l, a.logits, t, experts, lane);
    float top = 0, total = 1;
    if (a.r.score == UOR_B200_SOFTMAX) softmax_of(l, &top, &total);
    uint32_t key[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const int e = lane + 32 * i;
        float s = a.r.score == UOR_B200_SOFTMAX ? exp_below(l[i], top) / total : sigmoid(l[i]);
        if (a.bias && e < experts) s += a.bias[e];
        key[i] = l[i] > -INFINITY ? open_key(s) : 0u;
    }
    if (a.r.top_groups < a.r.groups) {
        // Lane g keeps group g's score; a group without two open experts has -inf's.
        const int size = experts / a.r.groups;
        uint32_t mine = 0;
        for (int g = 0; g < static_cast<int>(a.r.groups); ++g) {
            uint32_t in[VPL];
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                const int e = lane + 32 * i;
                in[i] = e >= g * size && e < (g + 1) * size ? key[i] : 0u;
            }
            int e1, e2;
            const uint32_t k1 = warp_best(in, lane, &e1);
            uint32_t sum = k1;
            if (size > 1) {
#pragma unroll
                for (int i = 0; i < VPL; ++i)
                    if (lane + 32 * i == e1) in[i] = 0;
                const uint32_t k2 = warp_best(in, lane, &e2);
                sum = k1 && k2 ? open_key(key_value(k1) + key_value(k2)) : 0u;
            }
            if (lane == g) mine = sum + 1;  // 1: a group of -inf, which is behind every other
        }
        uint32_t keep = 0;
        for (int s = 0; s < static_cast<int>(a.r.top_groups); ++s) {
            const uint32_t best = __reduce_max_sync(FULL, mine);
            const unsigned g = __reduce_min_sync(FULL, mine == best ? static_cast<unsigned>(lane) : FULL);
            keep |= 1u << g;
            if (lane == static_cast<int>(g)) mine = 0;
        }
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int e = lane + 32 * i;
            if (e < experts && !(keep >> (e / size) & 1)) key[i] = 0;
        }
    }
    // Lane s keeps choice s.
    int expert = -1;
    for (int s = 0; s < top_k; ++s) {
        int e;
        const uint32_t best = warp_best(key, lane, &e);
        if (!best) break;
#pragma unroll
        for (int i = 0; i < VPL; ++i)
            if (lane + 32 * i == e) key[i] = 0;
        if (lane == s) expert = e;
    }
    float v = -INFINITY, w = 0;
    if (expert >= 0) v = to_f32(static_cast<const T*>(a.logits.p)[t * a.logits.rs + expert * a.logits.cs]);
    if (a.r.renormalize)
        w = chosen_share(v, expert >= 0, a.r.score == UOR_B200_SOFTMAX);
    else if (expert >= 0)
        w = a.r.score == UOR_B200_SOFTMAX ? exp_below(v, top) / total : sigmoid(v);
    if (lane < top_k) {
        static_cast<int32_t*>(a.ids.p)[t * a.ids.rs + lane * a.ids.cs] = expert;
        static_cast<float*>(a.weights.p)[t * a.weights.rs + lane * a.weights.cs] = w * a.r.scale;
    }
}

// With s the scores, g the weights' gradient times the scale, w_j = s_j / sum_i s_i the chosen
// experts' shares (0 for the others):
//   renormalised: dl_j = w_j (g_j - sum_i g_i w_i), and that times (1 - s_j) for the sigmoid;
//   otherwise:    softmax dl = s (g - sum_i g_i s_i), sigmoid dl = g s (1 - s).
// Only the softmax without renormalisation has gradients beyond the chosen experts.
template <typename T, int VPL>
__global__ void route_backward_kernel(RouterArgs a) {
    const int lane = threadIdx.x & 31;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (t >= a.tokens) return;
    const int experts = a.r.experts, top_k = a.r.top_k;
    const bool softmax = a.r.score == UOR_B200_SOFTMAX, whole = softmax && !a.r.renormalize;
    int expert = -1;
    float g = 0, v = -INFINITY;
    if (lane < top_k) {
        expert = static_cast<const int32_t*>(a.in_ids.p)[t * a.in_ids.rs + lane * a.in_ids.cs];
        if (expert < 0 || expert >= experts) expert = -1;
    }
    if (expert >= 0) {
        v = to_f32(static_cast<const T*>(a.logits.p)[t * a.logits.rs + expert * a.logits.cs]);
        if (!(v > -INFINITY)) expert = -1;
    }
    if (expert >= 0)
        g = static_cast<const float*>(a.dweights.p)[t * a.dweights.rs + lane * a.dweights.cs] * a.r.scale;
    float l[VPL], d[VPL];
    float top = 0, total = 1, inner = 0;
#pragma unroll
    for (int i = 0; i < VPL; ++i) d[i] = 0;
    if (whole) {
        load_row<T>(l, a.logits, t, experts, lane);
        softmax_of(l, &top, &total);
        inner = warp_sum(expert >= 0 ? g * (exp_below(v, top) / total) : 0.0f);
    } else if (a.r.renormalize) {
        const float w = chosen_share(v, expert >= 0, softmax);
        const float dot = warp_sum(g * w);
        g = w * (g - dot);
        if (!softmax && expert >= 0) g *= sigmoid(-v);
    } else if (expert >= 0) {
        g *= sigmoid(v) * sigmoid(-v);
    }
    for (int j = 0; j < top_k; ++j) {
        const int e = __shfl_sync(FULL, expert, j);
        const float add = __shfl_sync(FULL, g, j);
#pragma unroll
        for (int i = 0; i < VPL; ++i)
            if (lane + 32 * i == e) d[i] += add;
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const int e = lane + 32 * i;
        if (e >= experts) continue;
        if (whole) d[i] = l[i] > -INFINITY ? exp_below(l[i], top) / total * (d[i] - inner) : 0.0f;
        store_f32(a.dlogits.p, t * a.dlogits.rs + e * a.dlogits.cs, a.dlogits.type, d[i]);
    }
}

template <typename T>
int launch(uor_b200_ctx* ctx, const RouterArgs& a, bool backward) {
    const unsigned grid = static_cast<unsigned>((a.tokens + 7) / 8);
    auto go = [&](auto vpl) {
        constexpr int V = decltype(vpl)::value;
        if (backward)
            route_backward_kernel<T, V><<<grid, 256, 0, ctx->stream>>>(a);
        else
            route_kernel<T, V><<<grid, 256, 0, ctx->stream>>>(a);
    };
    const int v = (static_cast<int>(a.r.experts) + 31) / 32;
    if (v <= 1) go(std::integral_constant<int, 1>());
    else if (v <= 2) go(std::integral_constant<int, 2>());
    else if (v <= 4) go(std::integral_constant<int, 4>());
    else if (v <= 8) go(std::integral_constant<int, 8>());
    else if (v <= 16) go(std::integral_constant<int, 16>());
    else go(std::integral_constant<int, 32>());
    return cuda_status(cudaGetLastError());
}

int run(uor_b200_ctx* ctx, const RouterArgs& a, bool backward, uor_b200_route* route) {
    route->kernel = UOR_B200_KERNEL_ROUTER;
    if (a.elem == UOR_B200_F32) return launch<float>(ctx, a, backward);
    if (a.elem == UOR_B200_BF16) return launch<__nv_bfloat16>(ctx, a, backward);
    return launch<__half>(ctx, a, backward);
}

}  // namespace

int run_expert_route(uor_b200_ctx* ctx, const RouterArgs& a, uor_b200_route* route) {
    return run(ctx, a, false, route);
}
int run_expert_route_backward(uor_b200_ctx* ctx, const RouterArgs& a, uor_b200_route* route) {
    return run(ctx, a, true, route);
}

}  // namespace uor
