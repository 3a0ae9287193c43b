// expert_route.cu -- the experts' router and the gradient of its logits.
//
// A warp per token, a run of neighbouring experts per lane: a row is read (and its gradient
// written) as vectors, a group of experts is a run of lanes, and among equal keys the lowest lane
// has the lowest expert. A key is ordered as an unsigned integer (the float's bits, negative
// ones complemented), so that the largest of a warp is one integer reduction. What is closed (a
// logit or key of -inf or NaN) is key 0, below every open one.
//
// Bound by instructions: a token's 256 logits are 1 KB, and some 900 instructions of its warp.
// 16384 x 256 with groups and a bias: 18.0 us (0.99 TB/s); with a lane's experts 32 apart and every
// choice a reduction over them, 52. Its gradient, two rows of memory and eight values: 10.6 us
// (3.3 TB/s); with every element computed rather than scattered over zeros, 14.6.
#include <cstring>

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

// 1 / (1 + exp(-l)) within 3 units: the reciprocal's and the exponential's own, and an addition's.
// The divisor is taken as a fourth, exactly: past 2^126 (logits below -87.3) the quick division
// gives 0, where the score is a denormal still.
__device__ __forceinline__ float sigmoid(float l) { return 0.25f * __fdividef(1.0f, fmaf(0.25f, expf(-l), 0.25f)); }

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

// This lane's logits, experts lane * VPL on; -inf past the last.
template <typename T, int VPL>
__device__ __forceinline__ void load_row(float (&l)[VPL], const Mat& m, bool vec, int64_t t, int experts, int lane) {
    const T* p = static_cast<const T*>(m.p) + t * m.rs;
    const int e0 = lane * VPL;
    constexpr int BYTES = VPL * sizeof(T);
    if (BYTES >= 4 && vec && e0 + VPL <= experts) {
        constexpr int WORDS = BYTES >= 4 ? BYTES / 4 : 1;
        uint32_t w[WORDS];
        if constexpr (WORDS % 4 == 0) {
#pragma unroll
            for (int i = 0; i < WORDS; i += 4) {
                const uint4 v = reinterpret_cast<const uint4*>(p + e0)[i / 4];
                w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
            }
        } else if constexpr (WORDS == 2) {
            const uint2 v = *reinterpret_cast<const uint2*>(p + e0);
            w[0] = v.x, w[1] = v.y;
        } else {
            w[0] = *reinterpret_cast<const uint32_t*>(p + e0);
        }
        T v[VPL];
        memcpy(v, w, BYTES < WORDS * 4 ? BYTES : WORDS * 4);
#pragma unroll
        for (int i = 0; i < VPL; ++i) l[i] = to_f32(v[i]);
        return;
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i) l[i] = e0 + i < experts ? to_f32(p[(e0 + i) * m.cs]) : -INFINITY;
}

// The two largest of two ordered pairs.
__device__ __forceinline__ void merge2(uint32_t& a1, uint32_t& a2, uint32_t b1, uint32_t b2) {
    a2 = max(min(a1, b1), max(a2, b2));
    a1 = max(a1, b1);
}

// The groups that stay open, a bit each. A group's order is its score's key plus one: a group of
// -inf is behind every other, and before none. Groups are runs of whole lanes, as many as a power
// of two, or else looked at one after another.
template <int VPL>
__device__ __forceinline__ uint32_t open_groups(const uint32_t (&key)[VPL], const RouterArgs& a, int lane) {
    const int groups = a.r.groups, size = a.group_size;
    uint32_t mine = 0;  // lane g: group g's
    if (a.lane_shift >= 0) {
        const int lanes = 1 << a.lane_shift;
        uint32_t k1 = 0, k2 = 0;
#pragma unroll
        for (int i = 0; i < VPL; ++i) merge2(k1, k2, key[i], 0);
        for (int o = 1; o < lanes; o <<= 1) {
            const uint32_t b1 = __shfl_xor_sync(FULL, k1, o), b2 = __shfl_xor_sync(FULL, k2, o);
            merge2(k1, k2, b1, b2);
        }
        const uint32_t sum = size == 1 ? k1 : k2 ? open_key(key_value(k1) + key_value(k2)) : 0u;
        mine = __shfl_sync(FULL, sum, lane * lanes & 31) + 1;
    } else {
        for (int g = 0; g < groups; ++g) {
            uint32_t k1 = 0, k2 = 0;
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                const int e = lane * VPL + i;
                if (e >= g * size && e < (g + 1) * size) merge2(k1, k2, key[i], 0);
            }
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t b1 = __shfl_xor_sync(FULL, k1, o), b2 = __shfl_xor_sync(FULL, k2, o);
                merge2(k1, k2, b1, b2);
            }
            const uint32_t sum = size == 1 ? k1 : k2 ? open_key(key_value(k1) + key_value(k2)) : 0u;
            if (lane == g) mine = sum + 1;
        }
    }
    int ahead = 0;  // groups before this lane's
    for (int g = 0; g < groups; ++g) {
        const uint32_t other = __shfl_sync(FULL, mine, g);
        ahead += other > mine || (other == mine && g < lane);
    }
    return __ballot_sync(FULL, lane < groups && ahead < static_cast<int>(a.r.top_groups));
}

// The expert of this lane's choice (lane s: the s-th largest key's), or -1. The top_k-th of the
// lanes' own largest keys bounds the choices from below, so few keys are left to order, a lane to
// each: by how many are ahead of it. Where equal keys leave more than that, the choices are taken
// one after another.
template <int VPL>
__device__ __forceinline__ int choose(uint32_t (&key)[VPL], int top_k, int lane, uint2* candidates) {
    const int e0 = lane * VPL;
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < VPL; ++i) mine = max(mine, key[i]);
    uint32_t bound = 1;
    if (VPL > 1) {
        uint32_t left = mine;
        for (int s = 0; s < top_k; ++s) {
            const uint32_t k = __reduce_max_sync(FULL, left);
            bound = max(k, 1u);
            if (k == 0) break;
            const unsigned at = __ballot_sync(FULL, left == k);
            if (lane == __ffs(at) - 1) left = 0;
        }
    }
    int count = 0, my_at = 0;  // candidates; where this lane's begin
#pragma unroll
    for (int i = 0; i < VPL; ++i) count += key[i] >= bound;
    int upto = count;
    if (VPL > 1) {
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(FULL, upto, o);
            if (lane >= o) upto += v;
        }
    } else {
        upto = __popc(__ballot_sync(FULL, count) & (0xFFFFFFFFu >> (31 - lane)));
    }
    my_at = upto - count;
    const int all = __shfl_sync(FULL, upto, 31);
    int expert = -1;
    if (all <= 32) {
        if (count) {
#pragma unroll
            for (int i = 0; i < VPL; ++i)
                if (key[i] >= bound) candidates[my_at++] = make_uint2(key[i], e0 + i);
        }
        __syncwarp();
        // In the experts' order, so that of equal ones those before this one are ahead of it.
        const uint2 c = lane < all ? candidates[lane] : make_uint2(0, 0);
        int ahead = 0;
        for (int o = 0; o < all; ++o) {
            const uint32_t other = __shfl_sync(FULL, c.x, o);
            ahead += other > c.x || (other == c.x && o < lane);
        }
        __syncwarp();
        if (lane < all && ahead < top_k) candidates[ahead].y = c.y;
        __syncwarp();
        if (lane < min(top_k, all)) expert = static_cast<int>(candidates[lane].y);
        return expert;
    }
    for (int s = 0; s < top_k; ++s) {  // a choice's lane takes out its key, the first among equals
        const uint32_t k = __reduce_max_sync(FULL, mine);
        if (!k) break;
        const int from = __ffs(__ballot_sync(FULL, mine == k)) - 1;
        int at = 0;
        if (lane == from) {
            bool found = false;
            mine = 0;
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                if (!found && key[i] == k) {
                    found = true;
                    key[i] = 0;
                    at = e0 + i;
                }
                mine = max(mine, key[i]);
            }
        }
        at = __shfl_sync(FULL, at, from);
        if (lane == s) expert = at;
    }
    return expert;
}

template <typename T, int VPL>
__global__ void __launch_bounds__(256) route_kernel(const __grid_constant__ RouterArgs a) {
    const int lane = threadIdx.x & 31;
    __shared__ uint2 candidates[8][32];
    const int64_t t = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (t >= a.tokens) return;
    const int experts = a.r.experts, top_k = a.r.top_k, e0 = lane * VPL;
    const bool softmax = a.r.score == UOR_B200_SOFTMAX;
    float l[VPL];
    load_row<T>(l, a.logits, a.vec, t, experts, lane);
    float top = 0, total = 1;
    uint32_t key[VPL];
    if (softmax) {
        softmax_of(l, &top, &total);
        const float share = 1.0f / total;
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            float s = exp_below(l[i], top) * share;
            if (a.bias) s += a.bias[min(e0 + i, experts - 1)];
            key[i] = l[i] > -INFINITY ? open_key(s) : 0u;
        }
    } else {
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            float s = sigmoid(l[i]);
            if (a.bias) s += a.bias[min(e0 + i, experts - 1)];
            key[i] = l[i] > -INFINITY ? open_key(s) : 0u;
        }
    }
    if (a.r.top_groups < a.r.groups) {
        const uint32_t open = open_groups(key, a, lane);
        const int size = a.group_size;
        if (a.lane_shift >= 0) {
            if (!(open >> (lane >> a.lane_shift) & 1)) {
#pragma unroll
                for (int i = 0; i < VPL; ++i) key[i] = 0;
            }
        } else {
#pragma unroll
            for (int i = 0; i < VPL; ++i)
                if (e0 + i < experts && !(open >> ((e0 + i) / size) & 1)) key[i] = 0;
        }
    }
    // Lane s keeps choice s.
    const int expert = choose(key, top_k, lane, candidates[threadIdx.x >> 5]);
    float v = -INFINITY, w = 0;
    if (expert >= 0) v = to_f32(static_cast<const T*>(a.logits.p)[t * a.logits.rs + expert * a.logits.cs]);
    if (a.r.renormalize)
        w = chosen_share(v, expert >= 0, softmax);
    else if (expert >= 0)
        w = softmax ? exp_below(v, top) / total : sigmoid(v);
    if (lane < top_k) {
        static_cast<int32_t*>(a.ids.p)[t * a.ids.rs + lane * a.ids.cs] = expert;
        static_cast<float*>(a.weights.p)[t * a.weights.rs + lane * a.weights.cs] = w * a.r.scale;
    }
}

// With s the scores, g the weights' gradient times the scale, w_j = s_j / sum_i s_i the chosen
// experts' shares (0 for the others):
//   renormalised: dl_j = w_j (g_j - sum_i g_i w_i), and that times (1 - s_j) for the sigmoid;
//   otherwise:    softmax dl = s (g - sum_i g_i s_i), sigmoid dl = g s (1 - s).
// Only the softmax without renormalisation has gradients beyond the chosen experts; elsewhere
// these alone are written, over a row of zeros.
template <typename T, int VPL>
__global__ void __launch_bounds__(256) route_backward_kernel(const __grid_constant__ RouterArgs a) {
    const int lane = threadIdx.x & 31;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (t >= a.tokens) return;
    const int experts = a.r.experts, top_k = a.r.top_k, e0 = lane * VPL;
    const bool softmax = a.r.score == UOR_B200_SOFTMAX, whole = softmax && !a.r.renormalize;
    int expert = -1;
    float g = 0, v = -INFINITY;
    if (lane < top_k) {
        expert = static_cast<const int32_t*>(a.in_ids.p)[t * a.in_ids.rs + lane * a.in_ids.cs];
        g = static_cast<const float*>(a.dweights.p)[t * a.dweights.rs + lane * a.dweights.cs] * a.r.scale;
        if (expert < 0 || expert >= experts) expert = -1;
    }
    T* row = static_cast<T*>(a.dlogits.p) + t * a.dlogits.rs;
    const int64_t cs = a.dlogits.cs;
    constexpr int BYTES = VPL * sizeof(T);
    const bool vec_row = BYTES % 16 == 0 && a.vec_out, vec = vec_row && e0 + VPL <= experts;
    if (!whole) {  // while the chosen logits travel
        if (!vec_row) {  // the lanes side by side, all of them
            for (int e = lane; e < experts; e += 32) row[e * cs] = from_f32<T>(0.0f);
        } else if (vec) {
#pragma unroll
            for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4*>(row + e0)[i] = make_uint4(0, 0, 0, 0);
        } else {  // the lane whose run the row ends in
            for (int e = e0; e < experts; ++e) row[e * cs] = from_f32<T>(0.0f);
        }
    }
    if (expert >= 0) {
        v = to_f32(static_cast<const T*>(a.logits.p)[t * a.logits.rs + expert * a.logits.cs]);
        if (!(v > -INFINITY)) expert = -1;
    }
    if (expert < 0) g = 0;
    if (!whole) {
        if (a.r.renormalize) {
            const float w = chosen_share(v, expert >= 0, softmax);
            const float dot = warp_sum(g * w);
            g = w * (g - dot);
            if (!softmax && expert >= 0) g *= sigmoid(-v);
        } else if (expert >= 0) {
            g *= sigmoid(v) * sigmoid(-v);
        }
        // An expert chosen more than once gets the sum, in the choices' order.
        const unsigned same = __match_any_sync(FULL, expert);
        if (__any_sync(FULL, expert >= 0 && (same & (same - 1)))) {
            float sum = 0;
            for (int j = 0; j < top_k; ++j) {
                const float other = __shfl_sync(FULL, g, j);
                if (same >> j & 1) sum += other;
            }
            g = sum;
        }
        __syncwarp();  // the zeros are written
        if (expert >= 0) row[expert * cs] = from_f32<T>(g);
        return;
    }
    float l[VPL], d[VPL];
    float top = 0, total = 1;
    load_row<T>(l, a.logits, a.vec, t, experts, lane);
    softmax_of(l, &top, &total);
    const float inner = warp_sum(expert >= 0 ? g * (exp_below(v, top) / total) : 0.0f);
#pragma unroll
    for (int i = 0; i < VPL; ++i) d[i] = -inner;
    for (int j = 0; j < top_k; ++j) {
        const int e = __shfl_sync(FULL, expert, j);
        const float add = __shfl_sync(FULL, g, j);
#pragma unroll
        for (int i = 0; i < VPL; ++i)
            if (e0 + i == e) d[i] += add;
    }
    const float share = 1.0f / total;
    T out[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) out[i] = from_f32<T>(l[i] > -INFINITY ? exp_below(l[i], top) * share * d[i] : 0.0f);
    if (vec) {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) {
            uint4 w;
            memcpy(&w, reinterpret_cast<const char*>(out) + i * 16, 16);
            reinterpret_cast<uint4*>(row + e0)[i] = w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < VPL; ++i)
            if (e0 + i < experts) row[(e0 + i) * cs] = out[i];
    }
}

template <typename T>
int launch(uor_b200_ctx* ctx, RouterArgs& a, bool backward) {
    const unsigned grid = static_cast<unsigned>((a.tokens + 7) / 8);
    auto go = [&](auto vpl) {
        constexpr int V = decltype(vpl)::value;
        if (backward)
            route_backward_kernel<T, V><<<grid, 256, 0, ctx->stream>>>(a);
        else
            route_kernel<T, V><<<grid, 256, 0, ctx->stream>>>(a);
    };
    const int v = (static_cast<int>(a.r.experts) + 31) / 32;
    const int vpl = v <= 1 ? 1 : v <= 2 ? 2 : v <= 4 ? 4 : v <= 8 ? 8 : v <= 16 ? 16 : 32;
    a.group_size = static_cast<int>(a.r.experts / a.r.groups);
    const int lanes = a.group_size / vpl;
    a.lane_shift = a.group_size % vpl == 0 && (lanes & (lanes - 1)) == 0 ? __builtin_ctz(lanes) : -1;
    if (v <= 1) go(std::integral_constant<int, 1>());
    else if (v <= 2) go(std::integral_constant<int, 2>());
    else if (v <= 4) go(std::integral_constant<int, 4>());
    else if (v <= 8) go(std::integral_constant<int, 8>());
    else if (v <= 16) go(std::integral_constant<int, 16>());
    else go(std::integral_constant<int, 32>());
    return cuda_status(cudaGetLastError());
}

int run(uor_b200_ctx* ctx, RouterArgs a, bool backward, uor_b200_route* route) {
    route->kernel = UOR_B200_KERNEL_ROUTER;
    const uint64_t size = a.elem == UOR_B200_F32 ? 4 : 2;
    a.vec = a.logits.cs == 1 && (reinterpret_cast<uint64_t>(a.logits.p) | static_cast<uint64_t>(a.logits.rs) * size) % 16 == 0;
    a.vec_out = a.dlogits.cs == 1 && (reinterpret_cast<uint64_t>(a.dlogits.p) | static_cast<uint64_t>(a.dlogits.rs) * size) % 16 == 0;
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
