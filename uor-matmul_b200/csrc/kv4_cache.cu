// kv4_cache.cu -- tokens into and out of the 4-bit cache of keys and values.
//
// A prompt's rows are read once, the rotated queries and the codes written. A warp has one row and steps
// through its heads, a lane eight neighbouring channels of a head, so that its cosines and sines are read
// once a row. A group's extremes meet by shuffles.
//
// A rotated value is the exact x cos - y sin rounded to f32 and then to 16 bits; a code that comes out one
// off would be a whole step of the range off, so both are computed as their definition has them. The
// products are exact in 64 bits, where this processor multiplies at half its 32-bit rate. (In 32 bits, by
// two fused multiply-adds with a bound of what they leave open and doubles where that matters: the same
// time.) A code is a multiplication by the scale's reciprocal but where that comes near a half; its eight
// and their exceptions are one branch.
//
// 8192 tokens, 32 heads of queries, 8 of keys and values, 128 channels, all rotated: 91 us, 2.5 TB/s, and
// 13 us to read them back. Bound by what a processor's 20 warps have under way: half of its cycles issue,
// 270 instructions for 512 values (16 warps of 128 registers: 103 us; 24 of 80, which spill, 90; two heads
// at a time with nothing ahead of them 96). One token: 3.8 us, a launch's own time.
#include "kv4.cuh"

#include <cstring>

namespace uor {

namespace {

constexpr int WARPS = 4;

// The row's sequence: the last one that begins at or before it, found by a warp 32 at a time; -1 where
// it has none.
__device__ __forceinline__ int sequence_of(const BatchDev& b, int row, int lane) {
    int lo = 0, hi = b.seqs;  // the answer is in lo .. hi - 1
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + lane * step;
        const uint32_t less = __ballot_sync(0xffffffffu, at < hi && b.starts[at] <= row);
        if (!less) return -1;
        lo += (31 - __clz(less)) * step;
        hi = min(hi, lo + step);
    }
    return b.starts[lo] <= row && row < b.starts[lo + 1] ? lo : -1;
}

template <typename T>
struct Half;
template <>
struct Half<__nv_bfloat16> {
    static constexpr float MOST = 3.3895313892515355e38f;
    __device__ static __forceinline__ uint32_t pair(float a, float b) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        uint32_t r;
        memcpy(&r, &v, 4);
        return r;
    }
    // The next smaller one of a positive value.
    __device__ static __forceinline__ float below(float v) { return __uint_as_float(__float_as_uint(v) - 0x10000u); }
    __device__ static __forceinline__ float first(uint32_t w) { return __uint_as_float(w << 16); }
    __device__ static __forceinline__ float second(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
};
template <>
struct Half<__half> {
    static constexpr float MOST = 65504.0f;
    __device__ static __forceinline__ float below(float v) { return __half2float(__ushort_as_half(__half_as_ushort(__float2half_rn(v)) - 1)); }
    __device__ static __forceinline__ uint32_t pair(float a, float b) {
        const __half2 v = __floats2half2_rn(a, b);
        uint32_t r;
        memcpy(&r, &v, 4);
        return r;
    }
    __device__ static __forceinline__ float first(uint32_t w) {
        return __half2float(__ushort_as_half(static_cast<unsigned short>(w & 0xFFFFu)));
    }
    __device__ static __forceinline__ float second(uint32_t w) {
        return __half2float(__ushort_as_half(static_cast<unsigned short>(w >> 16)));
    }
};

// f32(x c - y s): the products are exact in 64 bits, their difference is rounded there once.
__device__ __forceinline__ float turned(float x, double c, float y, double s) {
    return __double2float_rn(__fma_rn(x, c, -__dmul_rn(y, s)));
}

__device__ __noinline__ uint32_t code_slow(float t, float scale) {
    return static_cast<uint32_t>(fminf(fmaxf(rintf(__fadd_rn(__fdiv_rn(t, scale), 7.5f)), 0.0f), 15.0f));
}
// Eight codes: the integers nearest to (r - mid) / scale + 7.5, the quotient and the sum each rounded,
// within 0 .. 15. inverse: 1 / scale, or 0 for one so small that it has none.
__device__ __forceinline__ uint32_t codes_of(const float (&r)[8], float mid, float scale, float inverse) {
    uint32_t codes = 0, hard = inverse == 0.0f ? 0xFFu : 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        // 1.5 2^23 more leaves the nearest integer in the lowest bits; within 0 .. 15 before, which it is but for rounding
        const float z = fminf(fmaxf(__fmaf_rn(__fsub_rn(r[i], mid), inverse, 7.5f), 0.0f), 15.0f), n = __fadd_rn(z, 12582912.0f);
        if (fabsf(z - __fsub_rn(n, 12582912.0f)) > 0.4999f) hard |= 1u << i;
        codes |= (__float_as_uint(n) & 15u) << (4 * i);
    }
    if (hard) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (hard >> i & 1) codes = (codes & ~(15u << (4 * i))) | code_slow(__fsub_rn(r[i], mid), scale) << (4 * i);
    }
    return codes;
}

// Eight channels of 16 bits from `p`; vec: as one vector.
__device__ __forceinline__ uint4 load8(const void* p, bool vec) {
    if (vec) return *static_cast<const uint4*>(p);
    const auto* s = static_cast<const uint16_t*>(p);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = s[2 * i] | static_cast<uint32_t>(s[2 * i + 1]) << 16;
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store8(void* p, uint4 v, bool vec) {
    if (vec) {
        *static_cast<uint4*>(p) = v;
        return;
    }
    auto* s = static_cast<uint16_t*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) s[2 * i] = static_cast<uint16_t>(w[i]), s[2 * i + 1] = static_cast<uint16_t>(w[i] >> 16);
}

// How a lane's eight channels turn.
enum Turn {
    TURN_NONE = 0,
    TURN_HALVES = 1,  // with eight of the other half of the rotated channels
    TURN_PAIRS = 2,   // among themselves
    TURN_ANY = 3      // some of them, or with channels that do not lie so: one by one
};

// VEC: every row of heads begins at a multiple of 16 bytes.
template <typename T, bool VEC>
__global__ void __launch_bounds__(WARPS * 32, 5) append_kernel(const __grid_constant__ AppendArgs a, int slices) {
    const int lane = threadIdx.x & 31;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * WARPS + (threadIdx.x >> 5);
    const int row = static_cast<int>(item / slices), slice = static_cast<int>(item - static_cast<int64_t>(row) * slices);
    const BatchDev& b = a.batch;
    if (row >= b.rows) return;
    const int s = sequence_of(b, row, lane);
    if (s < 0) return;
    const Sequence seq(b, s);
    const int at = seq.at + row - seq.first;
    if (at < 0 || at >= b.capacity) return;
    uint8_t* block = kv_block(a.kv, b, s, 0, at);
    if (!block) return;

    const int dim = a.kv.dim, units = dim / 8, abreast = 32 / units;
    const int sub = lane / units, channel = (lane - sub * units) * 8;
    const bool mine = sub < abreast;
    const int t = at & 15, g = channel >> a.kv.group_shift, per_group = 1 << (a.kv.group_shift - 3);
    // The rotation of this lane's channels.
    int turn = TURN_NONE, other = 0;
    double c[8], sn[8];
    if (channel < a.turned && mine) {
        const float *cos = a.cos + at * a.turn_rs, *sin = a.sin + at * a.turn_rs;
        const int half = a.turned / 2;
        if (a.interleaved && a.turned % 8 == 0) {
            turn = TURN_PAIRS;
#pragma unroll
            for (int i = 0; i < 4; ++i) c[i] = cos[channel / 2 + i], sn[i] = sin[channel / 2 + i];
        } else if (!a.interleaved && half % 8 == 0) {
            turn = TURN_HALVES;
            const bool low = channel < half;
            other = low ? half : -half;
            const int i0 = low ? channel : channel - half;
#pragma unroll
            for (int i = 0; i < 8; ++i) c[i] = cos[i0 + i], sn[i] = low ? sin[i0 + i] : -sin[i0 + i];
        } else {
            turn = TURN_ANY;
        }
    }
    // Heads: the queries', the keys', the values'.
    const int heads = a.q_heads + 2 * a.kv.heads, each = (heads + slices * abreast - 1) / (slices * abreast) * abreast;
    const int last = min(heads, (slice + 1) * each);
    auto place = [&](int h, const Rows** from, int* local) {
        const bool q = h < a.q_heads, k = h < a.q_heads + a.kv.heads;
        *from = q ? &a.q : k ? &a.k : &a.v;
        *local = q ? h : k ? h - a.q_heads : h - a.q_heads - a.kv.heads;
    };
    // The next heads are on their way while these are worked on.
    uint4 x, y;
    auto load = [&](int h, uint4& own, uint4& with) {
        own = with = make_uint4(0, 0, 0, 0);
        if (!mine || h >= last) return;
        const Rows* from;
        int local;
        place(h, &from, &local);
        const uint16_t* p = static_cast<const uint16_t*>(from->p) + row * from->rs + local * dim + channel;
        own = load8(p, VEC || from->vec);
        if (turn == TURN_HALVES && h < a.q_heads + a.kv.heads) with = load8(p + other, VEC || from->vec);
    };
    load(slice * each + sub, x, y);
    uint4 next_x, next_y;
    for (int h0 = slice * each; h0 < last; h0 += abreast, x = next_x, y = next_y) {
        load(h0 + abreast + sub, next_x, next_y);
        const int h = h0 + sub;
        const bool live = mine && h < last;
        const bool query = h < a.q_heads, value = h >= a.q_heads + a.kv.heads;
        uint32_t w[4] = {x.x, x.y, x.z, x.w};
        float r[8];
        if (live && !value && turn != TURN_NONE) {
            if (turn == TURN_HALVES) {
                const uint32_t v[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w[i] = Half<T>::pair(turned(Half<T>::first(w[i]), c[2 * i], Half<T>::first(v[i]), sn[2 * i]),
                                         turned(Half<T>::second(w[i]), c[2 * i + 1], Half<T>::second(v[i]), sn[2 * i + 1]));
            } else if (turn == TURN_PAIRS) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float even = Half<T>::first(w[i]), odd = Half<T>::second(w[i]);
                    w[i] = Half<T>::pair(turned(even, c[i], odd, sn[i]), turned(odd, c[i], even, -sn[i]));
                }
            } else {
                const Rows* from;
                int local;
                place(h, &from, &local);
                const T* head = static_cast<const T*>(from->p) + row * from->rs + local * dim;
                const float *cos = a.cos + at * a.turn_rs, *sin = a.sin + at * a.turn_rs;
                const int half = a.turned / 2;
#pragma unroll
                for (int i = 0; i < 4; ++i) r[2 * i] = Half<T>::first(w[i]), r[2 * i + 1] = Half<T>::second(w[i]);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int ch = channel + i;
                    if (ch >= a.turned) break;
                    const bool low = a.interleaved ? ch % 2 == 0 : ch < half;
                    const int pair = a.interleaved ? ch / 2 : low ? ch : ch - half;
                    const int with = a.interleaved ? ch ^ 1 : low ? ch + half : ch - half;
                    r[i] = turned(r[i], cos[pair], to_f32(head[with]), low ? sin[pair] : -sin[pair]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = Half<T>::pair(r[2 * i], r[2 * i + 1]);
            }
        }
        __syncwarp();  // queries may turn in place: no lane writes what another still reads
        if (live && query) {
            store8(static_cast<uint16_t*>(a.q_out.p) + row * a.q_out.rs + h * dim + channel, make_uint4(w[0], w[1], w[2], w[3]),
                   VEC || a.q_out.vec);
        }
        if (h0 + abreast <= a.q_heads) continue;  // of the whole warp
        // Extremes of the group, by all lanes: those of other kinds take part and are not used.
        float high, low;
#pragma unroll
        for (int i = 0; i < 4; ++i) r[2 * i] = Half<T>::first(w[i]), r[2 * i + 1] = Half<T>::second(w[i]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            r[i] = r[i] != r[i] ? 0.0f : fminf(fmaxf(r[i], -Half<T>::MOST), Half<T>::MOST);
            high = i ? fmaxf(high, r[i]) : r[0];
            low = i ? fminf(low, r[i]) : r[0];
        }
        for (int o = 1; o < per_group; o <<= 1) {
            high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
            low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
        }
        if (!live || query) continue;
        const float mid = to_f32(from_f32<T>(__fadd_rn(high * 0.5f, low * 0.5f)));
        float scale = to_f32(from_f32<T>(__fdiv_rn(__fsub_rn(high * 0.5f, low * 0.5f), 7.5f)));
        // half of the largest float and 7.5 halves of the scale: what is held stays within the type
        if (fmaf(3.75f, scale, 0.5f * fabsf(mid)) > 0.5f * Half<T>::MOST) scale = Half<T>::below(scale);
        const float inverse = scale > 0x1p-120f ? __frcp_rn(scale) : 0.0f;
        const uint32_t codes = scale > 0.0f ? codes_of(r, mid, scale, inverse) : 0u;
        const int head = h - a.q_heads - (value ? a.kv.heads : 0);
        uint8_t* to = block + head * a.kv.head_bytes;
        if (value) {
            *reinterpret_cast<uint16_t*>(to + kv_value_half(dim, a.kv.groups, t, channel)) = static_cast<uint16_t>(codes);
            *reinterpret_cast<uint16_t*>(to + kv_value_half(dim, a.kv.groups, t, channel + 4)) = static_cast<uint16_t>(codes >> 16);
        } else {
            *reinterpret_cast<uint32_t*>(to + kv_key_word(dim, t, channel)) = codes;
        }
        if ((channel & ((1 << a.kv.group_shift) - 1)) == 0) {
            const uint32_t both = Half<T>::pair(scale, mid);
            auto* p = reinterpret_cast<uint16_t*>(to + kv_scale(dim, a.kv.groups, t, g, value));
            p[0] = static_cast<uint16_t>(both);
            p[2] = static_cast<uint16_t>(both >> 16);
        }
    }
}

// A lane reads eight channels of a key and of a value and writes what they stand for.
template <typename T, typename O>
__global__ void __launch_bounds__(WARPS * 32) read_kernel(const __grid_constant__ ReadArgs a, int slices) {
    const int lane = threadIdx.x & 31;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * WARPS + (threadIdx.x >> 5);
    const int row = static_cast<int>(item / slices), slice = static_cast<int>(item - static_cast<int64_t>(row) * slices);
    const BatchDev& b = a.batch;
    if (row >= b.rows) return;
    const int s = sequence_of(b, row, lane);
    if (s < 0) return;
    const Sequence seq(b, s);
    const int at = seq.at + row - seq.first;
    if (at < 0 || at >= b.capacity) return;
    const uint8_t* block = kv_block(a.kv, b, s, 0, at);
    if (!block) return;
    const int dim = a.kv.dim, units = dim / 8, abreast = 32 / units;
    const int sub = lane / units, channel = (lane - sub * units) * 8, t = at & 15, g = channel >> a.kv.group_shift;
    if (sub >= abreast) return;
    const int each = (a.kv.heads + slices * abreast - 1) / (slices * abreast) * abreast, last = min(a.kv.heads, (slice + 1) * each);
    for (int h0 = slice * each + sub; h0 < last; h0 += 2 * abreast) {
        uint32_t codes[2][2];
        uint16_t quants[2][2][2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if (h0 + u * abreast >= last) break;
            const uint8_t* from = block + (h0 + u * abreast) * a.kv.head_bytes;
            codes[u][0] = *reinterpret_cast<const uint32_t*>(from + kv_key_word(dim, t, channel));
            codes[u][1] = *reinterpret_cast<const uint16_t*>(from + kv_value_half(dim, a.kv.groups, t, channel)) |
                          static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(from + kv_value_half(dim, a.kv.groups, t, channel + 4)))
                              << 16;
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const auto* p = reinterpret_cast<const uint16_t*>(from + kv_scale(dim, a.kv.groups, t, g, v));
                quants[u][v][0] = p[0], quants[u][v][1] = p[2];
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if (h0 + u * abreast >= last) break;
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const float scale = Half<T>::first(quants[u][v][0]), mid = Half<T>::first(quants[u][v][1]);
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = __fmaf_rn(scale, static_cast<float>(codes[u][v] >> (4 * i) & 15) - 7.5f, mid);
                const Rows& to = v ? a.v : a.k;
                O* p = static_cast<O*>(to.p) + row * to.rs + (h0 + u * abreast) * dim + channel;
                if constexpr (sizeof(O) == 2) {
                    store8(p, make_uint4(Half<T>::pair(x[0], x[1]), Half<T>::pair(x[2], x[3]), Half<T>::pair(x[4], x[5]), Half<T>::pair(x[6], x[7])),
                           to.vec);
                } else if (to.vec) {
                    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
                    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) p[i] = x[i];
                }
            }
        }
    }
}

// A row's heads are cut over several warps where the rows alone leave processors idle.
int slices_for(const uor_b200_ctx* ctx, int64_t rows, int heads, int abreast) {
    const int64_t warps = static_cast<int64_t>(ctx->sm_count) * 16, most = (heads + abreast - 1) / abreast;
    const int64_t want = (warps + rows - 1) / rows;
    return static_cast<int>(want < most ? want : most);
}

}  // namespace

int run_kv4_append(uor_b200_ctx* ctx, const AppendArgs& a, uor_b200_route* route) {
    route->kernel = UOR_B200_KERNEL_KV4;
    const int slices = slices_for(ctx, a.batch.rows, a.q_heads + 2 * a.kv.heads, 32 / (a.kv.dim / 8));
    const int64_t blocks = (static_cast<int64_t>(a.batch.rows) * slices + WARPS - 1) / WARPS;
    if (blocks > INT32_MAX) return UOR_B200_UNSUPPORTED;
    const bool vec = a.k.vec && a.v.vec && (a.q_heads == 0 || (a.q.vec && a.q_out.vec));
    auto* kernel = a.elem == UOR_B200_BF16 ? (vec ? append_kernel<__nv_bfloat16, true> : append_kernel<__nv_bfloat16, false>)
                                           : (vec ? append_kernel<__half, true> : append_kernel<__half, false>);
    kernel<<<static_cast<unsigned>(blocks), WARPS * 32, 0, ctx->stream>>>(a, slices);
    return UOR_B200_OK;
}

int run_kv4_read(uor_b200_ctx* ctx, const ReadArgs& a, uor_b200_route* route) {
    route->kernel = UOR_B200_KERNEL_KV4;
    const int slices = slices_for(ctx, a.batch.rows, a.kv.heads, 32 / (a.kv.dim / 8));
    const int64_t blocks = (static_cast<int64_t>(a.batch.rows) * slices + WARPS - 1) / WARPS;
    if (blocks > INT32_MAX) return UOR_B200_UNSUPPORTED;
    auto* kernel = a.elem == UOR_B200_BF16 ? (a.out == UOR_B200_F32 ? read_kernel<__nv_bfloat16, float> : read_kernel<__nv_bfloat16, __nv_bfloat16>)
                                           : (a.out == UOR_B200_F32 ? read_kernel<__half, float> : read_kernel<__half, __half>);
    kernel<<<static_cast<unsigned>(blocks), WARPS * 32, 0, ctx->stream>>>(a, slices);
    return UOR_B200_OK;
}

}  // namespace uor
