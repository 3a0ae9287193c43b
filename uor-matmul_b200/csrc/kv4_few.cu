// kv4_few.cu -- attention over the 4-bit cache where few rows read it: decoding steps and drafts.
//
// Bound by the cache's reading. Each warp takes blocks of 16 tokens in turn through a ring of its own
// in shared memory, with its own softmax statistics and sums, and meets the block's other warps only
// where a sequence's share ends. The scores are mma.m16n8k16 with the queries as the 16 rows, so that
// their accumulators are what the values' product takes as its columns: there the values are the rows.
//
// Codes become 16-bit floats by their bits alone: u = 1 + code / 16 is an exponent or-ed to them. With
// x = mid + scale (code - 7.5) and code - 7.5 = 16 u - 23.5, of a group of channels
//   q . k / 16 = scale (q . u) + (mid - 23.5 scale) sum(q) / 16
//   sum_j p_j v_j = 16 sum_j (p_j scale_j) u_j - 23.5 sum_j p_j scale_j + sum_j p_j mid_j,
// so that no key or value is rounded: products of codes are exact, scales multiply in f32. p scale goes
// to the tensor cores as two bfloat16 (a rounded one and what that left, 2^-17 together), whatever the
// cache's type is: float16 would lose the small ones.
//
// The work is cut evenly: tiles of 64 tokens of every sequence, head and eight (or sixteen) rows are
// numbered by the lengths, which the device alone knows, and each block of threads has as many of them
// as any other. What a sequence's share is cut into is joined by a second kernel in the order of the
// tokens; so is nothing that one block had whole.
#include "kv4.cuh"

#include <cfloat>
#include <cstring>
#include <type_traits>

namespace uor {

namespace {

constexpr int WARPS = 4, THREADS = 32 * WARPS, STAGES = 4;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct FewAttend {
    AttendArgs a;
    float* part;   // [2 grid][8 NT][dim]
    float2* stat;  // [2 grid][8 NT]: maximum, sum
    int4* split;   // [grid]: sequence, head, row tile and parts of what block i begins and does not end
};

__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(mask), "r"(bits));
    return r;
}
// A word's nibbles i and 4 + i as 1 + code / 16, i = 0 .. 3.
template <typename T>
__device__ __forceinline__ void unpack(uint32_t w, uint32_t (&u)[4]) {
    if constexpr (std::is_same<T, __half>::value) {
        u[0] = and_or(w << 6, 0x03C003C0u, 0x3C003C00u), u[1] = and_or(w << 2, 0x03C003C0u, 0x3C003C00u);
        u[2] = and_or(w >> 2, 0x03C003C0u, 0x3C003C00u), u[3] = and_or(w >> 6, 0x03C003C0u, 0x3C003C00u);
    } else {
        u[0] = and_or(w << 3, 0x00780078u, 0x3F803F80u), u[1] = and_or(w >> 1, 0x00780078u, 0x3F803F80u);
        u[2] = and_or(w >> 5, 0x00780078u, 0x3F803F80u), u[3] = and_or(w >> 9, 0x00780078u, 0x3F803F80u);
    }
}
template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <typename T>
__device__ __forceinline__ float2 two(uint32_t w) {
    if constexpr (std::is_same<T, __half>::value) {
        __half2 v;
        memcpy(&v, &w, 4);
        return __half22float2(v);
    }
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <typename T>
__device__ __forceinline__ uint32_t pack(float a, float b) {
    uint32_t r;
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 v = __floats2half2_rn(a, b);
        memcpy(&r, &v, 4);
    } else {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        memcpy(&r, &v, 4);
    }
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void cp_async(uint32_t to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// N words from shared memory at a multiple of N words.
template <int N>
__device__ __forceinline__ void words(const uint8_t* p, uint32_t (&w)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const uint4 v = reinterpret_cast<const uint4*>(p)[i];
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const uint2 v = reinterpret_cast<const uint2*>(p)[i];
            w[2 * i] = v.x, w[2 * i + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    }
}

// Which blocks of 16 tokens the rows of a sequence see: sink_blocks first ones, then those from
// first_block on; and its work.
struct Share {
    int rows, row_tiles, sink_blocks, first_block, blocks, tiles;
    __device__ __forceinline__ Share(const Sequence& s, const AttendArgs& a, int tile_rows) {
        rows = s.count * a.share;
        row_tiles = (rows + tile_rows - 1) / tile_rows;
        const int low = a.window ? max(0, s.at - a.window + 1) : 0, ends = (s.keys + 15) >> 4;
        first_block = low < s.keys ? low >> 4 : ends;
        sink_blocks = a.window ? min((min(a.sinks, s.keys) + 15) >> 4, first_block) : 0;
        blocks = sink_blocks + ends - first_block;
        tiles = max(1, (blocks + WARPS - 1) / WARPS);  // of one head and row tile
    }
    __device__ __forceinline__ int block_at(int i) const { return i < sink_blocks ? i : first_block + i - sink_blocks; }
    __device__ __forceinline__ int64_t work(int heads) const { return static_cast<int64_t>(row_tiles) * heads * tiles; }
};

__device__ __forceinline__ void store4(void* p, float4 v, int type) {
    if (type == UOR_B200_F32) {
        auto* f = static_cast<float*>(p);
        if (reinterpret_cast<uintptr_t>(p) % 16 == 0) {
            *reinterpret_cast<float4*>(f) = v;
        } else {
            f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
        }
        return;
    }
    const uint32_t a = type == UOR_B200_BF16 ? pack<__nv_bfloat16>(v.x, v.y) : pack<__half>(v.x, v.y);
    const uint32_t b = type == UOR_B200_BF16 ? pack<__nv_bfloat16>(v.z, v.w) : pack<__half>(v.z, v.w);
    if (reinterpret_cast<uintptr_t>(p) % 8 == 0) {
        *static_cast<uint2*>(p) = make_uint2(a, b);
    } else {
        auto* h = static_cast<uint16_t*>(p);
        h[0] = static_cast<uint16_t>(a), h[1] = static_cast<uint16_t>(a >> 16);
        h[2] = static_cast<uint16_t>(b), h[3] = static_cast<uint16_t>(b >> 16);
    }
}

// Channels ch .. ch + 3 of row r of a sequence's head, from a sum that the weights' sum l divides; m:
// the scores' maximum in powers of two.
__device__ __forceinline__ void finish(const AttendArgs& a, const Sequence& seq, int head, int r, int ch, float4 sum, float m, float l) {
    const int row = seq.first + r / a.share, col = head * a.share + r % a.share;
    const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
    const int es = a.out == UOR_B200_F32 ? 4 : 2;
    store4(static_cast<char*>(a.y.p) + (row * a.y.rs + static_cast<int64_t>(col) * a.kv.dim + ch) * es,
           make_float4(sum.x * inverse, sum.y * inverse, sum.z * inverse, sum.w * inverse), a.out);
    if (ch == 0 && a.lse.p) static_cast<float*>(a.lse.p)[row * a.lse.rs + col] = (m + log2f(l)) * LN2;
}

// NT: rows in eights.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(THREADS) few_kernel(const __grid_constant__ FewAttend p) {
    constexpr int N32 = D / 32, ROWS = 8 * NT;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int64_t scan[WARPS];
    __shared__ float2 stat[WARPS][ROWS];
    const AttendArgs& a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int groups = a.kv.groups, per_group = 1 << (a.kv.group_shift - 5), block_bytes = kv_block_bytes(D, groups);
    uint8_t* ring = smem + warp * STAGES * block_bytes;
    const uint32_t ring_at = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
    int64_t* before = reinterpret_cast<int64_t*>(smem + WARPS * STAGES * block_bytes);  // [seqs + 1] tiles before each sequence's
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    int64_t total = 0;
    for (int s0 = 0; s0 < a.batch.seqs; s0 += THREADS) {
        const int s = s0 + threadIdx.x;
        int64_t mine = s < a.batch.seqs ? Share(Sequence(a.batch, s), a, ROWS).work(a.kv.heads) : 0;
        const int64_t own = mine;
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, mine, o);
            if (lane >= o) mine += v;
        }
        __syncthreads();
        if (lane == 31) scan[warp] = mine;
        __syncthreads();
        int64_t at = total + mine - own;
        for (int w = 0; w < WARPS; ++w) {
            if (w < warp) at += scan[w];
            total += scan[w];
        }
        if (s < a.batch.seqs) before[s] = at;
    }
    if (threadIdx.x == 0) before[a.batch.seqs] = total;
    if (threadIdx.x == 0) p.split[blockIdx.x] = make_int4(0, 0, 0, 0);
    __syncthreads();
    const int64_t each = (total + gridDim.x - 1) / gridDim.x;
    int64_t x = blockIdx.x * each;
    const int64_t end = min(total, x + each);
    const float to_log2 = a.scale * 16.0f * LOG2E;

    while (x < end) {
        int lo = 0, hi = a.batch.seqs;  // before[lo] <= x < before[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (before[mid] <= x) lo = mid;
            else hi = mid;
        }
        while (before[lo + 1] <= x) ++lo;  // past sequences without work
        const Sequence seq(a.batch, lo);
        const Share share(seq, a, ROWS);
        const int64_t rel = x - before[lo];
        const int item = static_cast<int>(rel / share.tiles), tile0 = static_cast<int>(rel - static_cast<int64_t>(item) * share.tiles);
        const int tile1 = static_cast<int>(min(static_cast<int64_t>(share.tiles), tile0 + end - x));
        const int row_tile = item / a.kv.heads, head = item - row_tile * a.kv.heads;

        // This warp's blocks: first, first + WARPS, ..
        const int first = tile0 * WARPS + warp, upto = min(share.blocks, tile1 * WARPS);
        const int count = first < upto ? (upto - first + WARPS - 1) / WARPS : 0;
        int pages = -1;
        uint32_t bad = 0;  // stages whose block lies on no page
        auto load = [&](int j) {
            const int stage = j % STAGES;
            if (j < count) {
                if ((j & 31) == 0) {  // the pages of the next 32
                    const int b = first + (j + lane) * WARPS;
                    pages = j + lane < count
                                ? a.batch.table[lo * a.batch.table_rs + (share.block_at(b) * KV_BLOCK >> a.kv.page_shift)]
                                : -1;
                }
                const int page = __shfl_sync(0xffffffffu, pages, j & 31);
                if (static_cast<uint32_t>(page) < a.kv.pages) {
                    const int in_page = share.block_at(first + j * WARPS) & ((1 << (a.kv.page_shift - 4)) - 1);
                    const uint8_t* from = a.kv.pool + page * a.kv.page_bytes + head * a.kv.head_bytes +
                                          static_cast<int64_t>(in_page) * block_bytes;
                    const uint32_t to = ring_at + stage * block_bytes;
                    for (int i = lane * 16; i < block_bytes; i += 512) cp_async(to + i, from + i);
                    bad &= ~(1u << stage);
                } else {
                    bad |= 1u << stage;
                }
            }
            cp_commit();
        };
#pragma unroll
        for (int j = 0; j < STAGES - 1; ++j) load(j);

        // The queries of this row tile as the scores' rows, and a sixteenth of their sums by 32 channels.
        uint32_t q[NT][N32][4];
        float q_sum[NT][N32];
        int at[NT];  // the rows' positions
        int nearest = INT32_MAX, farthest = -1;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = row_tile * ROWS + n * 8 + g;
            const bool there = r < share.rows;
            at[n] = there ? seq.at + r / a.share : -1;
            if (there) nearest = min(nearest, at[n]), farthest = max(farthest, at[n]);
            const uint16_t* from = static_cast<const uint16_t*>(a.q.p) + (seq.first + (there ? r / a.share : 0)) * a.q.rs +
                                   static_cast<int64_t>(head * a.share + (there ? r % a.share : 0)) * D + 8 * c;
#pragma unroll
            for (int i = 0; i < N32; ++i) {
                uint32_t w[4] = {0, 0, 0, 0};
                if (there) {
                    if (a.q.vec) {
                        const uint4 v = *reinterpret_cast<const uint4*>(from + 32 * i);
                        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; ++k) w[k] = from[32 * i + 2 * k] | static_cast<uint32_t>(from[32 * i + 2 * k + 1]) << 16;
                    }
                }
                float sum = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float2 v = two<T>(w[k]);
                    sum += v.x + v.y;
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                q_sum[n][i] = sum * 0.0625f;
                // channels (0, 4), (1, 5), (2, 6), (3, 7), as the nibbles come
                q[n][i][0] = __byte_perm(w[0], w[2], 0x5410), q[n][i][1] = __byte_perm(w[0], w[2], 0x7632);
                q[n][i][2] = __byte_perm(w[1], w[3], 0x5410), q[n][i][3] = __byte_perm(w[1], w[3], 0x7632);
            }
        }
        nearest = __reduce_min_sync(0xffffffffu, nearest);
        farthest = __reduce_max_sync(0xffffffffu, farthest);

        float o[NT][N32][2][4], o_mid[NT][4], weights[NT][N32], m[NT], l[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n] = -INFINITY, l[n] = 0;
            o_mid[n][0] = o_mid[n][1] = o_mid[n][2] = o_mid[n][3] = 0;
#pragma unroll
            for (int i = 0; i < N32; ++i) {
                weights[n][i] = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) o[n][i][0][k] = o[n][i][1][k] = 0;
            }
        }

        for (int j = 0; j < count; ++j) {
            cp_wait<STAGES - 2>();
            __syncwarp();
            load(j + STAGES - 1);
            const int stage = j % STAGES;
            if (bad >> stage & 1) continue;
            uint8_t* block = ring + stage * block_bytes;
            const int token = share.block_at(first + j * WARPS) * KV_BLOCK;
            if (token + KV_BLOCK > seq.keys) {
                // What lies behind the last token may be anything: its weights are 0, and so are the
                // values' scales and middles that they multiply.
                for (int i = lane; i < 8 * groups; i += 32) {
                    uint32_t* v = reinterpret_cast<uint32_t*>(block + 16 * D + 64 * groups + i * 8);
                    const int t = token + i / groups * 2;
                    const uint32_t keep = (t < seq.keys ? 0xFFFFu : 0u) | (t + 1 < seq.keys ? 0xFFFF0000u : 0u);
                    v[0] &= keep, v[1] &= keep;
                }
                __syncwarp();
            }
            // Scores / 16: rows g (and 8 + g), tokens 2 c, 2 c + 1, 8 + 2 c, 9 + 2 c.
            float score[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) score[n][0] = score[n][1] = score[n][2] = score[n][3] = 0;
            {
                uint32_t w[2][N32];
                words<N32>(block + (g * 4 + c) * N32 * 4, w[0]);
                words<N32>(block + ((8 + g) * 4 + c) * N32 * 4, w[1]);
                float acc[2][4], sums[NT];
#pragma unroll
                for (int i = 0; i < N32; ++i) {
                    if ((i & (per_group - 1)) == 0) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) acc[0][k] = acc[1][k] = 0;
#pragma unroll
                        for (int n = 0; n < NT; ++n) sums[n] = 0;
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) sums[n] += q_sum[n][i];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t u[4];
                        unpack<T>(w[h][i], u);
                        mma<T>(acc[h], q[0][i][0], NT == 2 ? q[NT - 1][i][0] : 0, q[0][i][1], NT == 2 ? q[NT - 1][i][1] : 0, u[0], u[1]);
                        mma<T>(acc[h], q[0][i][2], NT == 2 ? q[NT - 1][i][2] : 0, q[0][i][3], NT == 2 ? q[NT - 1][i][3] : 0, u[2], u[3]);
                    }
                    if ((i & (per_group - 1)) == per_group - 1) {
                        const uint8_t* params = block + 8 * D + (i >> (a.kv.group_shift - 5)) * 8;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint2 v = *reinterpret_cast<const uint2*>(params + (h * 4 + c) * groups * 8);
                            const float2 scale = two<T>(v.x), mid = two<T>(v.y);
                            const float low0 = fmaf(scale.x, -23.5f, mid.x), low1 = fmaf(scale.y, -23.5f, mid.y);
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                score[n][2 * h] = fmaf(scale.x, acc[h][2 * n], fmaf(low0, sums[n], score[n][2 * h]));
                                score[n][2 * h + 1] = fmaf(scale.y, acc[h][2 * n + 1], fmaf(low1, sums[n], score[n][2 * h + 1]));
                            }
                        }
                    }
                }
            }
            const int last = token + KV_BLOCK - 1;
            const bool open = last <= nearest && last < seq.keys &&
                              (a.window == 0 || token > farthest - a.window || last < a.sinks);
            float top[NT];
            bool higher = false;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    score[n][k] *= to_log2;
                    if (!open) {
                        const int t = token + (k >> 1) * 8 + 2 * c + (k & 1);
                        const bool seen = t <= at[n] && t < seq.keys && (a.window == 0 || t > at[n] - a.window || t < a.sinks);
                        if (!seen) score[n][k] = -INFINITY;
                    }
                }
                top[n] = fmaxf(fmaxf(score[n][0], score[n][1]), fmaxf(score[n][2], score[n][3]));
                // sums may run 2^8 past the maximum that they were begun with
                higher |= top[n] > m[n] + 8.0f;
            }
            if (__any_sync(0xffffffffu, higher)) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    top[n] = fmaxf(top[n], __shfl_xor_sync(0xffffffffu, top[n], 1));
                    top[n] = fmaxf(top[n], __shfl_xor_sync(0xffffffffu, top[n], 2));
                    const float next = fmaxf(m[n], top[n]);
                    const float by = m[n] == -INFINITY ? 0.0f : ex2(m[n] - next);
                    m[n] = next;
                    l[n] *= by;
                    const float by0 = __shfl_sync(0xffffffffu, by, 8 * c), by1 = __shfl_sync(0xffffffffu, by, 8 * c + 4);
                    o_mid[n][0] *= by0, o_mid[n][1] *= by1;
#pragma unroll
                    for (int i = 0; i < N32; ++i) {
                        weights[n][i] *= by;
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            o[n][i][h][0] *= by0, o[n][i][h][1] *= by1, o[n][i][h][2] *= by0, o[n][i][h][3] *= by1;
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float base = m[n] == -INFINITY ? 0.0f : m[n];
#pragma unroll
                for (int k = 0; k < 4; ++k) score[n][k] = ex2(score[n][k] - base);
                l[n] += (score[n][0] + score[n][1]) + (score[n][2] + score[n][3]);
            }
            // The middles' part: their groups are the rows.
            {
                const uint8_t* params = block + 16 * D + 64 * groups;
                const uint32_t mid0 = g < groups ? *reinterpret_cast<const uint32_t*>(params + (c * groups + g) * 8 + 4) : 0;
                const uint32_t mid1 = g < groups ? *reinterpret_cast<const uint32_t*>(params + ((4 + c) * groups + g) * 8 + 4) : 0;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint32_t b0 = pack<T>(score[n][0], score[n][1]), b1 = pack<T>(score[n][2], score[n][3]);
                    mma<T>(o_mid[n], mid0, 0, mid1, 0, b0, b1);
                    const float2 r0 = two<T>(b0), r1 = two<T>(b1);
                    mma<T>(o_mid[n], mid0, 0, mid1, 0, pack<T>(score[n][0] - r0.x, score[n][1] - r0.y),
                           pack<T>(score[n][2] - r1.x, score[n][3] - r1.y));
                }
                uint32_t w[2][N32];
                words<N32>(block + 8 * D + 64 * groups + (g * 4 + c) * N32 * 4, w[0]);
                words<N32>(block + 8 * D + 64 * groups + ((8 + g) * 4 + c) * N32 * 4, w[1]);
                using B = __nv_bfloat16;
                uint32_t high[NT][2], low[NT][2];
#pragma unroll
                for (int i = 0; i < N32; ++i) {
                    if ((i & (per_group - 1)) == 0) {
                        const int gi = i >> (a.kv.group_shift - 5);
                        const float2 s0 = two<T>(*reinterpret_cast<const uint32_t*>(params + (c * groups + gi) * 8));
                        const float2 s1 = two<T>(*reinterpret_cast<const uint32_t*>(params + ((4 + c) * groups + gi) * 8));
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const float w0 = score[n][0] * s0.x, w1 = score[n][1] * s0.y, w2 = score[n][2] * s1.x, w3 = score[n][3] * s1.y;
                            weights[n][i] += (w0 + w1) + (w2 + w3);
                            high[n][0] = pack<B>(w0, w1), high[n][1] = pack<B>(w2, w3);
                            const float2 r0 = two<B>(high[n][0]), r1 = two<B>(high[n][1]);
                            low[n][0] = pack<B>(w0 - r0.x, w1 - r0.y), low[n][1] = pack<B>(w2 - r1.x, w3 - r1.y);
                        }
                    }
                    uint32_t u0[4], u1[4];
                    unpack<B>(w[0][i], u0);
                    unpack<B>(w[1][i], u1);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            mma<B>(o[n][i][h], u0[2 * h], u0[2 * h + 1], u1[2 * h], u1[2 * h + 1], high[n][0], high[n][1]);
                            mma<B>(o[n][i][h], u0[2 * h], u0[2 * h + 1], u1[2 * h], u1[2 * h + 1], low[n][0], low[n][1]);
                        }
                }
            }
        }
        cp_wait<0>();
        __syncthreads();  // the rings are read out: the sums take their place
        float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            l[n] += __shfl_xor_sync(0xffffffffu, l[n], 1);
            l[n] += __shfl_xor_sync(0xffffffffu, l[n], 2);
            if (c == 0) stat[warp][n * 8 + g] = make_float2(m[n], l[n]);
            float w0 = 0, w1 = 0, mid0 = 0, mid1 = 0;
#pragma unroll
            for (int i = 0; i < N32; ++i) {
                if ((i & (per_group - 1)) == 0) {
                    float w = weights[n][i];
                    w += __shfl_xor_sync(0xffffffffu, w, 1);
                    w += __shfl_xor_sync(0xffffffffu, w, 2);
                    w0 = __shfl_sync(0xffffffffu, w, 8 * c), w1 = __shfl_sync(0xffffffffu, w, 8 * c + 4);
                    const int gi = i >> (a.kv.group_shift - 5);
                    mid0 = __shfl_sync(0xffffffffu, o_mid[n][0], gi * 4 + c), mid1 = __shfl_sync(0xffffffffu, o_mid[n][1], gi * 4 + c);
                }
                auto value = [&](float v, float w, float mid) { return fmaf(16.0f, v, fmaf(-23.5f, w, mid)); };
                float* to = sums + ((warp * ROWS + n * 8 + 2 * c) * D + 32 * i + 4 * g);
                const auto& v = o[n][i];
                *reinterpret_cast<float4*>(to) = make_float4(value(v[0][0], w0, mid0), value(v[0][2], w0, mid0), value(v[1][0], w0, mid0), value(v[1][2], w0, mid0));
                *reinterpret_cast<float4*>(to + D) = make_float4(value(v[0][1], w1, mid1), value(v[0][3], w1, mid1), value(v[1][1], w1, mid1), value(v[1][3], w1, mid1));
            }
        }
        __syncthreads();
        const bool whole = tile0 == 0 && tile1 == share.tiles;
        const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (tile0 == 0);
        for (int v = threadIdx.x; v < ROWS * D / 4; v += THREADS) {
            const int r = v / (D / 4), ch = (v - r * (D / 4)) * 4;
            float most = -INFINITY;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) most = fmaxf(most, stat[w][r].x);
            float4 sum = make_float4(0, 0, 0, 0);
            float all = 0;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float2 s = stat[w][r];
                const float by = s.x == -INFINITY ? (s.y == 0.0f ? 0.0f : 1.0f) : ex2(s.x - most);
                const float4 add = *reinterpret_cast<const float4*>(sums + (w * ROWS + r) * D + ch);
                if (s.y != 0.0f) sum.x = fmaf(by, add.x, sum.x), sum.y = fmaf(by, add.y, sum.y), sum.z = fmaf(by, add.z, sum.z), sum.w = fmaf(by, add.w, sum.w);
                all = fmaf(by, s.y, all);
            }
            if (whole) {
                if (row_tile * ROWS + r < share.rows) finish(a, seq, head, row_tile * ROWS + r, ch, sum, most, all);
            } else {
                *reinterpret_cast<float4*>(p.part + (slot * ROWS + r) * D + ch) = sum;
                if (ch == 0) p.stat[slot * ROWS + r] = make_float2(most, all);
            }
        }
        if (!whole && tile0 == 0 && threadIdx.x == 0) {
            const int64_t item_end = x + share.tiles;  // of its tiles, numbered with all
            p.split[blockIdx.x] = make_int4(lo, head, row_tile, static_cast<int>((item_end - 1) / each - blockIdx.x + 1));
        }
        x += tile1 - tile0;
        __syncthreads();  // before the next copies into the rings
    }
}

// What several blocks had a part of each, in the order of the tokens.
__global__ void __launch_bounds__(THREADS) join_kernel(const __grid_constant__ FewAttend p, int tile_rows) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int4 it = p.split[blockIdx.x];
    if (it.w == 0) return;
    const AttendArgs& a = p.a;
    const Sequence seq(a.batch, it.x);
    const int dim = a.kv.dim, rows = seq.count * a.share, quads = dim / 4;
    auto slot = [&](int i) { return 2 * (static_cast<int64_t>(blockIdx.x) + i) + (i == 0); };
    for (int v = threadIdx.x; v < tile_rows * quads; v += THREADS) {
        const int r = v / quads, ch = (v - r * quads) * 4, row = it.z * tile_rows + r;
        if (row >= rows) continue;
        float most = -INFINITY;
        for (int i = 0; i < it.w; ++i) most = fmaxf(most, p.stat[slot(i) * tile_rows + r].x);
        float4 sum = make_float4(0, 0, 0, 0);
        float all = 0;
#pragma unroll 4
        for (int i = 0; i < it.w; ++i) {
            const float2 s = p.stat[slot(i) * tile_rows + r];
            const float4 add = *reinterpret_cast<const float4*>(p.part + (slot(i) * tile_rows + r) * dim + ch);
            const float by = s.x == -INFINITY ? (s.y == 0.0f ? 0.0f : 1.0f) : ex2(s.x - most);
            if (s.y != 0.0f) sum.x = fmaf(by, add.x, sum.x), sum.y = fmaf(by, add.y, sum.y), sum.z = fmaf(by, add.z, sum.z), sum.w = fmaf(by, add.w, sum.w);
            all = fmaf(by, s.y, all);
        }
        finish(a, seq, it.y, row, ch, sum, most, all);
    }
}

template <typename T, int D, int NT>
int launch_few(uor_b200_ctx* ctx, const AttendArgs& a, uor_b200_route* route) {
    auto* kernel = few_kernel<T, D, NT>;
    const int smem = WARPS * STAGES * a.kv.block_bytes + (a.batch.seqs + 1) * 8;
    static int resident[64][9] = {};  // blocks of a processor, by groups
    int& per_sm = resident[ctx->device & 63][a.kv.groups];
    if (!per_sm) {
        const int ring = WARPS * STAGES * a.kv.block_bytes;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) != cudaSuccess ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, THREADS, ring + 1024) != cudaSuccess || per_sm < 1)
            return UOR_B200_DEVICE_ERROR;
    }
    const int64_t grid = static_cast<int64_t>(ctx->sm_count) * per_sm;
    const size_t parts = static_cast<size_t>(2 * grid) * 8 * NT;
    int st = UOR_B200_OK;
    auto* ws = static_cast<uint8_t*>(ctx_buffer(ctx, SLOT_WS, parts * (D * 4 + 8) + grid * 16, &st));
    if (!ws) return st;
    FewAttend p{};
    p.a = a;
    p.part = reinterpret_cast<float*>(ws);
    p.stat = reinterpret_cast<float2*>(ws + parts * D * 4);
    p.split = reinterpret_cast<int4*>(ws + parts * (D * 4 + 8));
    route->tile_m = 8 * NT, route->tile_n = KV_BLOCK * WARPS, route->tile_k = D;
    route->ctas = static_cast<uint32_t>(grid);
    kernel<<<static_cast<unsigned>(grid), THREADS, smem, ctx->stream>>>(p);
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(static_cast<unsigned>(grid));
    c.blockDim = dim3(THREADS);
    c.stream = ctx->stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &attr;
    c.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&c, join_kernel, p, 8 * NT));
}

template <typename T, int D>
int by_rows(uor_b200_ctx* ctx, const AttendArgs& a, uor_b200_route* route) {
    // Rows of one head that a sequence has on average.
    const int64_t rows = static_cast<int64_t>(a.batch.rows) * a.share / a.batch.seqs;
    return rows > 8 ? launch_few<T, D, 2>(ctx, a, route) : launch_few<T, D, 1>(ctx, a, route);
}
template <typename T>
int by_dim(uor_b200_ctx* ctx, const AttendArgs& a, uor_b200_route* route) {
    switch (a.kv.dim) {
    case 64: return by_rows<T, 64>(ctx, a, route);
    case 96: return by_rows<T, 96>(ctx, a, route);
    case 128: return by_rows<T, 128>(ctx, a, route);
    case 192: return by_rows<T, 192>(ctx, a, route);
    default: return by_rows<T, 256>(ctx, a, route);
    }
}

}  // namespace

int run_kv4_attention(uor_b200_ctx* ctx, const AttendArgs& a, uor_b200_route* route) {
    route->kernel = UOR_B200_KERNEL_KV4;
    return a.elem == UOR_B200_BF16 ? by_dim<__nv_bfloat16>(ctx, a, route) : by_dim<__half>(ctx, a, route);
}

}  // namespace uor
