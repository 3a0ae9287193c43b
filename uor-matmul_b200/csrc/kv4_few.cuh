// kv4_few.cuh -- attention over the 4-bit cache where few rows read it: decoding steps and drafts.
//
// Bound by the cache's reading. Each warp takes blocks of 16 tokens in turn through a ring of its own
// in shared memory, with its own softmax statistics and sums, and meets the block's other warps only
// where a sequence's share ends. Keys and values are the 16 rows of mma.m16n8k16, the queries its eight
// columns; the weights are turned by movmatrix from the one's result to the other's operand.
//
// Beside that it is issue slots that count: a block of 2560 bytes (128 channels, groups of 32) comes in
// 111 cycles. Codes become 16-bit floats by their bits alone: u = 1 + code / 16 is an exponent or-ed to
// them. With x = mid + scale (code - 7.5) and code - 7.5 = 16 u - 23.5, of a group of channels
//   q . k / 16 = scale (q . u - 23.5 / 16 sum(q)) + mid sum(q) / 16
//   sum_j p_j v_j = 16 sum_j (p_j scale_j) u_j - 23.5 sum_j p_j scale_j + sum_j p_j mid_j,
// so that no key or value is rounded: products of codes are exact, keys' scales multiply in f32. The
// middles' terms are products of their own; in the keys' one sum(q) / 16 is two or three 16-bit parts that
// lie behind one another in the reduction.
//
// Queries are brought below 2 by a power of two, which makes float16 of either type (what lies 2^-14
// below a row's largest keeps 2^-25 of it). Float16's ten bits hold two codes: for a bfloat16 result they
// come as 1 + code / 1024 of the even channels, of which one multiplication makes what the odd ones are
// at once, 1 + code / 64, with queries 4 times as large; that is five instructions of the integer pipe for
// eight codes and two of another, not eight. (With the even ones as they come and queries 64 times as
// large, 3 us of 167 less, the sums' roundings reached 2e-5 of lse, now 1.5e-6.) For the others u is
// 1 + code / 16.
//
// Weights times scales, for a bfloat16 result, are rounded twice, as weights and values that were each
// brought to 16 bits would be; sum_j p_j scale_j is of the same rounded numbers, so the cancellation costs
// nothing. For f32 and float16 results (EXACT) they are two 16-bit numbers, a rounded one and what that
// left (2^-17 together), and values' codes are code - 7.5, an addition more for each pair: the tensor
// cores' sums of u, five times as large as what is left of them, cut off more than that (1.4e-5 of the
// result, not 2.5e-6). Weights are bfloat16 whatever the cache's type is: float16 would lose the small
// ones. (64 contexts of 8192: 169 us with one, 204 with two. A float16 result is 2e-4 off its 64 bits with
// two, its own rounding; with one 1.8e-3.)
//
// The work is cut evenly: tiles of 64 tokens of every item (a sequence, head and eight or sixteen rows)
// are numbered by the lengths, which the device alone knows, and each block of threads has as many of them
// as any other. What an item is cut into is joined by a second kernel in a fixed order; nothing is that one
// block had whole. Cutting the last third of the work smaller and letting blocks take it as they come free
// evened their ends out (83 to 165 us after the start) but cost as much in beginnings: 178 us, not 167.
//
// 64 contexts of 8192, 8 heads of 128 channels with 8 queries each, bfloat16: 169 us, 4.0 TB/s of codes
// and scales; 388 instructions a block of 16 tokens and warp, 60 % of all issue slots (a tenth more on
// processors with four blocks than on average; the half-rate integer pipe is as busy). One token in 4096:
// 12.5 us, of which the sequences' scan takes 1.8, a table entry and then a block's arrival 2, three blocks
// to a warp and their sums 4.5, and the second kernel 2.5 behind the last block.
#pragma once
#include "kv4_math.cuh"

#include <algorithm>

namespace uor {

namespace {

constexpr int WARPS = 4, THREADS = 32 * WARPS, STAGES = 4;
constexpr int JOINERS = 256;  // threads of a block that joins
// Tiles that a block takes at least, unless an item has fewer: what it saves in its own time a smaller
// share costs in parts to join (one token, 4096 in the cache, 8 heads: 13.3 us with one, 12.4 with two
// to four, 13.5 with six).
constexpr int LEAST = 3;


struct FewAttend {
    AttendArgs a;
    float* part;   // [2 grid][8 NT][dim]
    float2* stat;  // [2 grid][8 NT]: maximum, sum
    // [grid]: sequence, head, row tile and parts of what block i begins and does not end; and the block
    // that began what block i begins with, i where that is itself.
    int4* split;
    int* from;
};

__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {  // of numbers that are mostly small
    return (a | b) >> 32 ? a / b : static_cast<int64_t>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b));
}

// A word's nibbles i and 4 + i, i = 0 .. 3: of values as bfloat16 1 + code / 16, or (EXACT) code - 7.5; of keys as float16 the
// same, or (FAST) 1 + code / 64.
template <bool EXACT>
__device__ __forceinline__ void unpack_values(uint32_t w, uint32_t (&u)[4]) {
    constexpr uint32_t BASE = EXACT ? 0x41804180u : 0x3F803F80u;  // 16, or 1
    u[0] = and_or(w << 3, 0x00780078u, BASE), u[1] = and_or(w >> 1, 0x00780078u, BASE);
    u[2] = and_or(w >> 5, 0x00780078u, BASE), u[3] = and_or(w >> 9, 0x00780078u, BASE);
    if constexpr (EXACT) {
#pragma unroll
        for (int i = 0; i < 4; ++i) asm("add.rn.bf16x2 %0, %0, %1;" : "+r"(u[i]) : "r"(0xC1BCC1BCu));  // -23.5
    }
}
template <bool FAST>
__device__ __forceinline__ void unpack_keys(uint32_t w, uint32_t (&u)[4]) {
    if constexpr (FAST) {
        const uint32_t v = w >> 8;
        u[0] = and_or(w, 0x000F000Fu, 0x3C003C00u), u[1] = and_or(w, 0x00F000F0u, 0x3C003C00u);
        u[2] = and_or(v, 0x000F000Fu, 0x3C003C00u), u[3] = and_or(v, 0x00F000F0u, 0x3C003C00u);
        // 1 + code / 1024, times 16, less 15
        asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(u[0]) : "r"(0x4C004C00u), "r"(0xCB80CB80u));
        asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(u[2]) : "r"(0x4C004C00u), "r"(0xCB80CB80u));
    } else {
        u[0] = and_or(w << 6, 0x03C003C0u, 0x3C003C00u), u[1] = and_or(w << 2, 0x03C003C0u, 0x3C003C00u);
        u[2] = and_or(w >> 2, 0x03C003C0u, 0x3C003C00u), u[3] = and_or(w >> 6, 0x03C003C0u, 0x3C003C00u);
    }
}
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

// d += a b.
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
// An 8 x 8 matrix of 16-bit elements, two neighbours of a row to a lane, turned over.
__device__ __forceinline__ uint32_t turn(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// One 16-bit float.
template <typename T>
__device__ __forceinline__ float one(uint16_t v) {
    if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half(v));
    return __uint_as_float(static_cast<uint32_t>(v) << 16);
}
__device__ __forceinline__ uint32_t mul_bf16(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

__device__ __forceinline__ float weight(float2 s, float most) { return s.x == -INFINITY ? (s.y == 0.0f ? 0.0f : 1.0f) : ex2(s.x - most); }
// A sum and its statistics with one part more.
__device__ __forceinline__ void take(float4& sum, float2& both, const float4& add, float2 s) {
    const float most = fmaxf(both.x, s.x), by = weight(both, most), of = weight(s, most);
    if (both.y != 0.0f) sum.x *= by, sum.y *= by, sum.z *= by, sum.w *= by;
    if (s.y != 0.0f) sum.x = fmaf(of, add.x, sum.x), sum.y = fmaf(of, add.y, sum.y), sum.z = fmaf(of, add.z, sum.z), sum.w = fmaf(of, add.w, sum.w);
    both = make_float2(most, fmaf(of, s.y, by * both.y));
}

// NT: rows in eights. GP: 32s of channels in a group. EXACT: weights in two parts, for f32 and float16 results.
template <typename T, int D, int GP, int NT, bool EXACT>
__global__ void __launch_bounds__(THREADS, D <= 128 && NT == 1 ? 4 : 1) few_kernel(const __grid_constant__ FewAttend p) {
    constexpr int N32 = D / 32, ROWS = 8 * NT, G = N32 / GP;
    constexpr int block_bytes = kv_block_bytes(D, G);
    using B = __nv_bfloat16;
    static_assert(EXACT || std::is_same<T, B>::value, "float16 results take two parts");
    constexpr float UNIT = EXACT ? 1.0f : 16.0f;  // of the values' products
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int64_t scan[WARPS];
    __shared__ float2 stat[WARPS][ROWS];
    const AttendArgs& a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    uint8_t* ring = smem + warp * STAGES * block_bytes;
    const uint32_t ring_at = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
    int64_t* before = reinterpret_cast<int64_t*>(smem + WARPS * STAGES * block_bytes);  // [seqs + 1] tiles before each sequence's, padded
    // The middles' product: reduction positions 2 c, 2 c + 1 (and 8 + them) are a pair of groups of a
    // part of sum(q); pairs beyond the groups and parts beyond the third are 0.
    constexpr int PAIRS = (G + 1) / 2, SPAN = PAIRS == 1 ? 1 : PAIRS == 2 ? 2 : 4;  // lanes of a part
    const int pair0 = c % SPAN, part0 = c / SPAN, part1 = part0 + 4 / SPAN;
    const int mid_at0 = min(2 * pair0, G - 1) * 8 + 4, mid_at1 = min(2 * pair0 + 1, G - 1) * 8 + 4;
    const uint32_t odd = g & 1, mid_half = odd ? 0x7632 : 0x5410;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // Items and their tiles, each thread's cut off at 2^20 (starts that do not rise may count rows often);
    // where they matter there are few.
    constexpr int MANY = 1 << 20;
    int64_t total = 0;
    int items = 0, work = 0, own_items = 0, own_tiles = 0;
    for (int s = threadIdx.x; s < a.batch.seqs; s += THREADS) {
        const Share share(Sequence(a.batch, s), a, ROWS, WARPS);
        own_items = share.row_tiles * a.kv.heads, own_tiles = share.tiles;
        items = min(MANY, items + min(MANY, own_items));
        work = static_cast<int>(min(static_cast<int64_t>(MANY * 16), work + static_cast<int64_t>(own_items) * own_tiles));
    }
    items = __reduce_add_sync(0xffffffffu, items), work = __reduce_add_sync(0xffffffffu, work);
    if (lane == 0) scan[warp] = static_cast<int64_t>(work) << 32 | items;
    __syncthreads();
    items = 0;
    for (int w = 0; w < WARPS; ++w) items += static_cast<int>(scan[w]), total += scan[w] >> 32;
    const int blocks = gridDim.x;
    // Where there are two blocks to an item, an item's tiles count as many as whole blocks of them have, so
    // that no block has parts of two: a part's beginning and end cost as much as four tiles (29 x 5 drafted
    // tokens 23.9 -> 18.1 us, 8 contexts of 8192 40.2 -> 36.0, 32 of them 95.4 -> 97.3).
    const bool padded = 2 * items <= blocks && total < MANY * 16;
    const int pad = padded ? max(LEAST, static_cast<int>(quotient(total + blocks - items - 1, blocks - items))) : 1;
    auto whole_pads = [&](int tiles) { return (tiles + pad - 1) / pad * pad; };
    total = 0;
    for (int s0 = 0; s0 < a.batch.seqs; s0 += THREADS) {
        const int s = s0 + threadIdx.x;
        if (a.batch.seqs > THREADS) {
            own_items = 0;
            if (s < a.batch.seqs) {
                const Share share(Sequence(a.batch, s), a, ROWS, WARPS);
                own_items = share.row_tiles * a.kv.heads, own_tiles = share.tiles;
            }
        }
        const int64_t own = static_cast<int64_t>(own_items) * whole_pads(own_tiles);
        int64_t mine = own;
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
    if (threadIdx.x == 0) {
        before[a.batch.seqs] = total;
        p.split[blockIdx.x] = make_int4(0, 0, 0, 0);
        p.from[blockIdx.x] = blockIdx.x;
    }
    __syncthreads();
    // Tiles of a block.
    const int64_t each = padded ? pad : max(static_cast<int64_t>(LEAST), quotient(total + blocks - 1, blocks));
    int64_t x = blockIdx.x * each;
    const int64_t end = min(total, x + each);

    while (x < end) {
        int lo = 0, hi = a.batch.seqs;  // before[lo] <= x < before[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (before[mid] <= x) lo = mid;
            else hi = mid;
        }
        while (before[lo + 1] <= x) ++lo;  // past sequences without work
        const Sequence seq(a.batch, lo);
        const Share share(seq, a, ROWS, WARPS);
        const int64_t rel = x - before[lo];
        const int padded_tiles = whole_pads(share.tiles);
        const int item = static_cast<int>(quotient(rel, padded_tiles)), from = static_cast<int>(rel - static_cast<int64_t>(item) * padded_tiles);
        const int to = static_cast<int>(min(static_cast<int64_t>(padded_tiles), from + end - x));
        // padded: as many tiles as the item's other blocks have, or one less
        const int span = padded ? (share.tiles - 1) / (padded_tiles / pad) + 1 : 1;
        const int tile0 = padded ? from / pad * span : from, tile1 = padded ? min(share.tiles, tile0 + span) : to;
        const int row_tile = item / a.kv.heads, head = item - row_tile * a.kv.heads;

        // This warp's blocks: first, first + WARPS, ..
        const int first = tile0 * WARPS + warp, upto = min(share.blocks, tile1 * WARPS);
        const int count = first < upto ? (upto - first + WARPS - 1) / WARPS : 0;
        int places = -1;  // where in the pool the blocks of 32 steps lie, one to a lane; -1: on none of its pages
        uint32_t bad = 0;  // stages of those
        auto load = [&](int j) {
            const int stage = j % STAGES;
            if (j < count) {
                if ((j & 31) == 0) {
                    places = -1;
                    if (j + lane < count) {
                        const int b = share.block_at(first + (j + lane) * WARPS), in_page = a.kv.page_shift - 4;
                        const int page = a.batch.table[lo * a.batch.table_rs + (b >> in_page)];
                        if (static_cast<uint32_t>(page) < a.kv.pages)
                            places = ((page * a.kv.heads + head) << in_page) + (b & ((1 << in_page) - 1));
                    }
                }
                const int place = __shfl_sync(0xffffffffu, places, j & 31);
                bad = place < 0 ? bad | 1u << stage : bad & ~(1u << stage);
                if (place >= 0) {
                    const uint8_t* from = a.kv.pool + static_cast<int64_t>(place) * block_bytes + lane * 16;
                    const uint32_t to = ring_at + stage * block_bytes + lane * 16;
#pragma unroll
                    for (int i = 0; i < block_bytes; i += 512)
                        if (i + 512 <= block_bytes || lane * 16 < block_bytes - i) cp_async(to + i, from + i);
                }
            }
            cp_commit();
        };
#pragma unroll
        for (int j = 0; j < STAGES - 1; ++j) load(j);

        // The queries of this row tile as the scores' columns, each row brought below 2; by groups what
        // the codes' offsets add to them; and the parts of their sums as the middles' product has them.
        uint32_t q[NT][N32][4], q_mid[NT][2];
        uint64_t offset[NT][G], to_log2[NT];  // of columns 2 c and 2 c + 1
        int at[NT][2];                        // their rows' positions
        int nearest = INT32_MAX, farthest = -1;
        auto columns = [&](float v) { return pair_of(__shfl_sync(0xffffffffu, v, 8 * c), __shfl_sync(0xffffffffu, v, 8 * c + 4)); };
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = row_tile * ROWS + n * 8 + g;
            const bool there = r < share.rows;
            const int position = there ? seq.at + r / a.share : -1;
            if (there) nearest = min(nearest, position), farthest = max(farthest, position);
            at[n][0] = __shfl_sync(0xffffffffu, position, 8 * c), at[n][1] = __shfl_sync(0xffffffffu, position, 8 * c + 4);
            const uint16_t* from = static_cast<const uint16_t*>(a.q.p) + (seq.first + (there ? r / a.share : 0)) * a.q.rs +
                                   static_cast<int64_t>(head * a.share + (there ? r % a.share : 0)) * D + 8 * c;
            float most = 0;
#pragma unroll
            for (int i = 0; i < N32; ++i) {
#pragma unroll
                for (int k = 0; k < 4; ++k) q[n][i][k] = 0;
                if (there) {
                    if (a.q.vec) {
                        const uint4 v = *reinterpret_cast<const uint4*>(from + 32 * i);
                        q[n][i][0] = v.x, q[n][i][1] = v.y, q[n][i][2] = v.z, q[n][i][3] = v.w;
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            q[n][i][k] = from[32 * i + 2 * k] | static_cast<uint32_t>(from[32 * i + 2 * k + 1]) << 16;
                    }
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float2 v = two<T>(q[n][i][k]);
                    most = fmaxf(most, fmaxf(fabsf(v.x), fabsf(v.y)));
                }
            }
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const uint32_t power = min(max(__float_as_uint(most) >> 23, 1u), 253u);  // most is 1 to 2 times 2^(power - 127)
            const float down = __uint_as_float((254 - power) << 23), up = __uint_as_float(power << 23);
            to_log2[n] = columns(up * (a.scale * (16.0f * LOG2E)));
            float sum = 0, by_code = 0, of0[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < N32; ++i) {
                float v[8];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float2 w = two<T>(q[n][i][k]);
                    v[2 * k] = w.x * down, v[2 * k + 1] = w.y * down;
                }
                constexpr float by = EXACT ? 1.0f : 4.0f;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    // channels (0, 4), (1, 5), (2, 6), (3, 7), as the nibbles come
                    q[n][i][k] = pack<__half>(v[k] * by, v[k + 4] * by);
                    sum += v[k] + v[k + 4];
                    by_code = fmaf(-(by + 7.5f / 16.0f), v[k] + v[k + 4], by_code);
                }
                if (i % GP == GP - 1) {
#pragma unroll
                    for (int o = 1; o < 4; o <<= 1) {
                        sum += __shfl_xor_sync(0xffffffffu, sum, o);
                        by_code += __shfl_xor_sync(0xffffffffu, by_code, o);
                    }
                    offset[n][i / GP] = columns(by_code);
                    if (i / GP / 2 == pair0) of0[i / GP & 1] = sum * 0.0625f;
                    sum = by_code = 0;
                }
            }
            // parts: rounded, what that left rounded, and what that left
            uint32_t part[3];
#pragma unroll
            for (int k = 0; k < 3; ++k) {
                part[k] = pack<T>(of0[0], of0[1]);
                const float2 v = two<T>(part[k]);
                of0[0] -= v.x, of0[1] -= v.y;
                // of what is not finite nothing is left
                if (!(fabsf(v.x) < INFINITY)) of0[0] = 0;
                if (!(fabsf(v.y) < INFINITY)) of0[1] = 0;
            }
            auto at_part = [&](int k) { return k == 0 ? part[0] : k == 1 ? part[1] : k == 2 ? part[2] : 0u; };
            q_mid[n][0] = pair0 < PAIRS ? at_part(part0) : 0u;
            q_mid[n][1] = pair0 < PAIRS ? at_part(part1) : 0u;
        }
        nearest = min(__reduce_min_sync(0xffffffffu, nearest), seq.keys - 1);
        farthest = __reduce_max_sync(0xffffffffu, farthest);
        const int behind = a.window ? farthest - a.window : -1;  // the last position that some row's window has left

        // Of columns 2 c and 2 c + 1: the maximum that the sums are of, its negative, how far past it a
        // score may be, the sums.
        float o[NT][N32][2][4], rest[NT][4], m[NT][2], bar[NT][2];
        uint64_t base[NT], l[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n][0] = m[n][1] = bar[n][0] = bar[n][1] = -INFINITY;
            base[n] = l[n] = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                rest[n][k] = 0;
#pragma unroll
                for (int i = 0; i < N32; ++i) o[n][i][0][k] = o[n][i][1][k] = 0;
            }
        }

        // Scores / 16 of a block: tokens g (first half) and 8 + g, columns 2 c and 2 c + 1.
        uint64_t score[NT][2];
        auto scores = [&](const uint8_t* block) {
            const uint8_t* params = block + 8 * D + (g >> 1) * G * 8;
            uint32_t w[2][N32], mid[2];
            words<N32>(block + (g * 4 + c) * N32 * 4, w[0]);
            words<N32>(block + ((8 + g) * 4 + c) * N32 * 4, w[1]);
#pragma unroll
            for (int h = 0; h < 2; ++h)
                mid[h] = __byte_perm(*reinterpret_cast<const uint32_t*>(params + h * 32 * G + mid_at0),
                                     *reinterpret_cast<const uint32_t*>(params + h * 32 * G + mid_at1), mid_half);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float sums[4] = {0, 0, 0, 0};
                mma<T>(sums, mid[0], mid[1], mid[0], mid[1], q_mid[n][0], q_mid[n][1]);
                score[n][0] = pair_of(sums[0], sums[1]), score[n][1] = pair_of(sums[2], sums[3]);
            }
            float acc[NT][4];
#pragma unroll
            for (int i = 0; i < N32; ++i) {
                uint32_t u0[4], u1[4];
                unpack_keys<!EXACT>(w[0][i], u0);
                unpack_keys<!EXACT>(w[1][i], u1);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if (i % GP == 0) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0;
                    mma<__half>(acc[n], u0[0], u1[0], u0[1], u1[1], q[n][i][0], q[n][i][1]);
                    mma<__half>(acc[n], u0[2], u1[2], u0[3], u1[3], q[n][i][2], q[n][i][3]);
                }
                if (i % GP == GP - 1) {
                    const float s0 = one<T>(*reinterpret_cast<const uint16_t*>(params + i / GP * 8 + odd * 2));
                    const float s1 = one<T>(*reinterpret_cast<const uint16_t*>(params + 32 * G + i / GP * 8 + odd * 2));
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        score[n][0] = fma2(pair_of(s0, s0), add2(pair_of(acc[n][0], acc[n][1]), offset[n][i / GP]), score[n][0]);
                        score[n][1] = fma2(pair_of(s1, s1), add2(pair_of(acc[n][2], acc[n][3]), offset[n][i / GP]), score[n][1]);
                    }
                }
            }
        };

        for (int j = 0; j < count; ++j) {
            cp_wait<STAGES - 2>();
            __syncwarp();  // the copies of every lane are there, and every lane is done with the block before
            load(j + STAGES - 1);
            const int stage = j % STAGES;
            uint8_t* block = ring + stage * block_bytes;
            if (bad >> stage & 1) continue;
            const int token = share.block_at(first + j * WARPS) * KV_BLOCK;
            scores(block);
            // In powers of two, past the maximum at hand.
            float x[NT][4];
            const int last = token + KV_BLOCK - 1;
            const bool masked = last > nearest || (token <= behind && last >= a.sinks);
            bool higher = false;
            if (last >= seq.keys) {
                // What lies behind the last token may be anything: its weights are 0, and so are the
                // values' scales and middles that they multiply.
                for (int i = lane; i < 8 * G; i += 32) {
                    uint32_t* v = reinterpret_cast<uint32_t*>(block + 16 * D + 64 * G + i * 8);
                    const int t = token + i / G * 2;
                    const uint32_t keep = (t < seq.keys ? 0xFFFFu : 0u) | (t + 1 < seq.keys ? 0xFFFF0000u : 0u);
                    v[0] &= keep, v[1] &= keep;
                }
                __syncwarp();
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                parts_of(fma2(score[n][0], to_log2[n], base[n]), x[n][0], x[n][1]);
                parts_of(fma2(score[n][1], to_log2[n], base[n]), x[n][2], x[n][3]);
                if (masked) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int t = token + (k >> 1) * 8 + g, row = at[n][k & 1];
                        const bool seen = t <= row && t < seq.keys && (a.window == 0 || t > row - a.window || t < a.sinks);
                        if (!seen) x[n][k] = -INFINITY;
                    }
                }
                higher |= fmaxf(x[n][0], x[n][2]) > bar[n][0] || fmaxf(x[n][1], x[n][3]) > bar[n][1];
            }
            if (__any_sync(0xffffffffu, higher)) {  // sums may run 2^8 past the maximum that they were begun with
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float by[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float top = fmaxf(x[n][k], x[n][2 + k]);
#pragma unroll
                        for (int v = 4; v < 32; v <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, v));
                        const float before_ = m[n][k] == -INFINITY ? 0.0f : m[n][k], next = fmaxf(m[n][k], top + before_);
                        const float now = next == -INFINITY ? 0.0f : next;
                        by[k] = m[n][k] == -INFINITY ? 0.0f : ex2(m[n][k] - next);
                        x[n][k] += before_ - now, x[n][2 + k] += before_ - now;
                        m[n][k] = next;
                        bar[n][k] = next == -INFINITY ? -INFINITY : 8.0f;
                    }
                    base[n] = pair_of(m[n][0] == -INFINITY ? 0.0f : -m[n][0], m[n][1] == -INFINITY ? 0.0f : -m[n][1]);
                    l[n] = mul2(l[n], pair_of(by[0], by[1]));
                    rest[n][0] *= by[0], rest[n][1] *= by[1];
#pragma unroll
                    for (int i = 0; i < N32; ++i)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            o[n][i][h][0] *= by[0], o[n][i][h][1] *= by[1], o[n][i][h][2] *= by[0], o[n][i][h][3] *= by[1];
                }
            }
            const uint8_t* params = block + 16 * D + 64 * G;
            // The middles' part: their groups are the rows, as they are of -23.5 times the weights' sums.
            const uint32_t mid0 = g < G ? *reinterpret_cast<const uint32_t*>(params + (c * G + g) * 8 + 4) : 0;
            const uint32_t mid1 = g < G ? *reinterpret_cast<const uint32_t*>(params + ((4 + c) * G + g) * 8 + 4) : 0;
            // Weights rounded, of tokens 2 c, 2 c + 1 and 8 more, column g; EXACT: what that left, and both.
            uint32_t p0[NT], p1[NT];
            float both[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int k = 0; k < 4; ++k) x[n][k] = ex2(x[n][k]);
                l[n] = add2(l[n], add2(pair_of(x[n][0], x[n][1]), pair_of(x[n][2], x[n][3])));
                const uint32_t r0 = pack<T>(x[n][0], x[n][1]), r1 = pack<T>(x[n][2], x[n][3]);
                p0[n] = turn(r0), p1[n] = turn(r1);
                mma<T>(rest[n], mid0, 0, mid1, 0, p0[n], p1[n]);
                if constexpr (EXACT) {
                    const float2 v0 = two<T>(r0), v1 = two<T>(r1);
                    const uint32_t left0 = turn(pack<T>(x[n][0] - v0.x, x[n][1] - v0.y)), left1 = turn(pack<T>(x[n][2] - v1.x, x[n][3] - v1.y));
                    mma<T>(rest[n], mid0, 0, mid1, 0, left0, left1);
                    parts_of(add2(pair_of<T>(p0[n]), pair_of<T>(left0)), both[n][0], both[n][1]);
                    parts_of(add2(pair_of<T>(p1[n]), pair_of<T>(left1)), both[n][2], both[n][3]);
                }
            }
            uint32_t w[2][N32];
            words<N32>(block + 8 * D + 64 * G + (g * 4 + c) * N32 * 4, w[0]);
            words<N32>(block + 8 * D + 64 * G + ((8 + g) * 4 + c) * N32 * 4, w[1]);
            uint32_t high[NT][2], low[NT][2];
#pragma unroll
            for (int i = 0; i < N32; ++i) {
                if (i % GP == 0) {
                    [[maybe_unused]] const uint32_t minus = g == i / GP ? 0xC1BCC1BCu : 0u;  // -23.5 in the group's row
                    const uint32_t s0 = *reinterpret_cast<const uint32_t*>(params + (c * G + i / GP) * 8);
                    const uint32_t s1 = *reinterpret_cast<const uint32_t*>(params + ((4 + c) * G + i / GP) * 8);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        if constexpr (!EXACT) {
                            high[n][0] = mul_bf16(p0[n], s0), high[n][1] = mul_bf16(p1[n], s1);
                        } else {
                            float v[4];
                            parts_of(mul2(pair_of(both[n][0], both[n][1]), pair_of<T>(s0)), v[0], v[1]);
                            parts_of(mul2(pair_of(both[n][2], both[n][3]), pair_of<T>(s1)), v[2], v[3]);
                            high[n][0] = pack<B>(v[0], v[1]), high[n][1] = pack<B>(v[2], v[3]);
                            const float2 r0 = two<B>(high[n][0]), r1 = two<B>(high[n][1]);
                            low[n][0] = pack<B>(v[0] - r0.x, v[1] - r0.y), low[n][1] = pack<B>(v[2] - r1.x, v[3] - r1.y);
                        }
                        if constexpr (!EXACT) mma<B>(rest[n], minus, 0, minus, 0, high[n][0], high[n][1]);
                    }
                }
                uint32_t u0[4], u1[4];
                unpack_values<EXACT>(w[0][i], u0);
                unpack_values<EXACT>(w[1][i], u1);
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        mma<B>(o[n][i][h], u0[2 * h], u0[2 * h + 1], u1[2 * h], u1[2 * h + 1], high[n][0], high[n][1]);
                        if constexpr (EXACT)
                            mma<B>(o[n][i][h], u0[2 * h], u0[2 * h + 1], u1[2 * h], u1[2 * h + 1], low[n][0], low[n][1]);
                    }
            }
        }
        cp_wait<0>();
        __syncthreads();  // the rings are read out: the sums take their place
        float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float all[2];
            parts_of(l[n], all[0], all[1]);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
#pragma unroll
                for (int v = 4; v < 32; v <<= 1) all[k] += __shfl_xor_sync(0xffffffffu, all[k], v);
                if (g == 0) stat[warp][n * 8 + 2 * c + k] = make_float2(m[n][k], all[k]);
            }
            float mid0 = 0, mid1 = 0;
#pragma unroll
            for (int i = 0; i < N32; ++i) {
                if (i % GP == 0) {
                    mid0 = __shfl_sync(0xffffffffu, rest[n][0], (i / GP) * 4 + c);
                    mid1 = __shfl_sync(0xffffffffu, rest[n][1], (i / GP) * 4 + c);
                }
                float* to = sums + ((warp * ROWS + n * 8 + 2 * c) * D + 32 * i + 4 * g);
                const auto& v = o[n][i];
                *reinterpret_cast<float4*>(to) = make_float4(fmaf(UNIT, v[0][0], mid0), fmaf(UNIT, v[0][2], mid0),
                                                             fmaf(UNIT, v[1][0], mid0), fmaf(UNIT, v[1][2], mid0));
                *reinterpret_cast<float4*>(to + D) = make_float4(fmaf(UNIT, v[0][1], mid1), fmaf(UNIT, v[0][3], mid1),
                                                                 fmaf(UNIT, v[1][1], mid1), fmaf(UNIT, v[1][3], mid1));
            }
        }
        __syncthreads();
        const bool whole = from == 0 && to == padded_tiles;
        const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (from == 0);
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
        if (!whole && threadIdx.x == 0) {
            const int64_t begun = x - from;  // its first tile's number
            if (from == 0)
                p.split[blockIdx.x] = make_int4(lo, head, row_tile, static_cast<int>(quotient(begun + padded_tiles - 1, each)) - blockIdx.x + 1);
            else
                p.from[blockIdx.x] = static_cast<int>(quotient(begun, each));
        }
        x += to - from;
        __syncthreads();  // before the next copies into the rings
    }
}

// What several blocks had a part of each. As many blocks as had one join it, each some of its outputs;
// a block's threads take those, four channels each, beside one another and the parts in turn, and what
// they have is added in a fixed order.
__global__ void __launch_bounds__(JOINERS) join_kernel(const __grid_constant__ FewAttend p, int tile_rows) {
    __shared__ float4 sums[JOINERS];
    __shared__ float2 stats[JOINERS];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const AttendArgs& a = p.a;
    const int quads = a.kv.dim / 4, from = p.from[blockIdx.x];
    for (int k = 0; k < 2; ++k) {  // what the block ended, what it began
        const int me = blockIdx.x, begin = k ? me : from;
        if (k == 0 && begin == me) continue;
        int4 it = p.split[begin];
        it.w = min(it.w, static_cast<int>(gridDim.x) - begin);
        if (it.w <= 0) continue;
        const Sequence seq(a.batch, it.x);
        const int outs = min(tile_rows, seq.count * a.share - it.z * tile_rows) * quads, each = (outs + it.w - 1) / it.w;
        const int first = (me - begin) * each, upto = min(outs, first + each);
        int abreast = 1;  // parts that are read beside one another
        while (abreast < it.w && abreast < 32) abreast <<= 1;
        const int width = JOINERS / abreast, column = threadIdx.x & (width - 1), row = threadIdx.x / width;
        auto slot = [&](int i) { return 2 * (static_cast<int64_t>(begin) + i) + (i == 0); };
        for (int o = first; o < upto; o += width) {
            const int out = o + column, r = out / quads, ch = (out - r * quads) * 4;
            float2 both = make_float2(-INFINITY, 0);
            float4 sum = make_float4(0, 0, 0, 0);
            if (out < upto) {
#pragma unroll 4
                for (int i = row; i < it.w; i += abreast)
                    take(sum, both, *reinterpret_cast<const float4*>(p.part + (slot(i) * tile_rows + r) * a.kv.dim + ch), p.stat[slot(i) * tile_rows + r]);
            }
            sums[threadIdx.x] = sum, stats[threadIdx.x] = both;
            __syncthreads();
            if (row == 0 && out < upto) {
                for (int i = 1; i < min(abreast, it.w); ++i) take(sum, both, sums[i * width + column], stats[i * width + column]);
                finish(a, seq, it.y, it.z * tile_rows + r, ch, sum, both.x, both.y);
            }
            __syncthreads();
        }
    }
}

template <typename T, int D, int GP, int NT, bool EXACT>
int launch_few(uor_b200_ctx* ctx, const AttendArgs& a, uor_b200_route* route) {
    auto* kernel = few_kernel<T, D, GP, NT, EXACT>;
    constexpr int RINGS = WARPS * STAGES * kv_block_bytes(D, D / 32 / GP);
    const int smem = RINGS + (a.batch.seqs + 1) * 8;
    static int resident[64] = {};  // blocks of a processor
    int& per_sm = resident[ctx->device & 63];
    if (!per_sm) {
        int found = 0;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, RINGS + 4097 * 8) != cudaSuccess ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&found, kernel, THREADS, RINGS + 1024) != cudaSuccess || found < 1)
            return UOR_B200_DEVICE_ERROR;
        per_sm = found;
    }
    // As many blocks as the table's whole length gives work.
    const int64_t tiles = std::max(1, (a.batch.capacity + KV_BLOCK * WARPS - 1) / (KV_BLOCK * WARPS));
    const int64_t items = (a.batch.seqs + static_cast<int64_t>(a.batch.rows) * a.share / (8 * NT)) * a.kv.heads;
    const int64_t most = static_cast<int64_t>(ctx->sm_count) * per_sm;
    if (items > INT32_MAX) return UOR_B200_UNSUPPORTED;
    const int64_t grid = std::min(most, items >= most ? most : items * ((tiles + LEAST - 1) / LEAST));
    const size_t parts = static_cast<size_t>(2 * grid) * 8 * NT;
    int st = UOR_B200_OK;
    auto* ws = static_cast<uint8_t*>(ctx_buffer(ctx, SLOT_WS, parts * (D * 4 + 8) + grid * 20, &st));
    if (!ws) return st;
    FewAttend p{};
    p.a = a;
    p.part = reinterpret_cast<float*>(ws);
    p.stat = reinterpret_cast<float2*>(ws + parts * D * 4);
    p.split = reinterpret_cast<int4*>(ws + parts * (D * 4 + 8));
    p.from = reinterpret_cast<int*>(p.split + grid);
    route->tile_m = 8 * NT, route->tile_n = KV_BLOCK * WARPS, route->tile_k = D;
    route->ctas = static_cast<uint32_t>(grid);
    kernel<<<static_cast<unsigned>(grid), THREADS, smem, ctx->stream>>>(p);
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(static_cast<unsigned>(grid));
    c.blockDim = dim3(JOINERS);
    c.stream = ctx->stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &attr;
    c.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&c, join_kernel, p, 8 * NT));
}

template <typename T, int D, int GP, bool EXACT>
int by_rows(uor_b200_ctx* ctx, const AttendArgs& a, uor_b200_route* route) {
    // Rows of one head that a sequence has on average.
    const int64_t rows = static_cast<int64_t>(a.batch.rows) * a.share / a.batch.seqs;
    return rows > 8 ? launch_few<T, D, GP, 2, EXACT>(ctx, a, route) : launch_few<T, D, GP, 1, EXACT>(ctx, a, route);
}
template <typename T, int D, bool EXACT>
int by_group(uor_b200_ctx* ctx, const AttendArgs& a, uor_b200_route* route) {
    switch (a.kv.group_shift) {
    case 5: return by_rows<T, D, 1, EXACT>(ctx, a, route);
    case 6:
        if constexpr (D % 64 == 0) return by_rows<T, D, 2, EXACT>(ctx, a, route);
        break;
    case 7:
        if constexpr (D % 128 == 0) return by_rows<T, D, 4, EXACT>(ctx, a, route);
        break;
    case 8:
        if constexpr (D % 256 == 0) return by_rows<T, D, 8, EXACT>(ctx, a, route);
        break;
    }
    return UOR_B200_UNSUPPORTED;
}

}  // namespace

template <typename T, bool EXACT>
int kv4_few(uor_b200_ctx* ctx, const AttendArgs& a, uor_b200_route* route) {
    switch (a.kv.dim) {
    case 64: return by_group<T, 64, EXACT>(ctx, a, route);
    case 96: return by_group<T, 96, EXACT>(ctx, a, route);
    case 128: return by_group<T, 128, EXACT>(ctx, a, route);
    case 192: return by_group<T, 192, EXACT>(ctx, a, route);
    default: return by_group<T, 256, EXACT>(ctx, a, route);
    }
}

}  // namespace uor
