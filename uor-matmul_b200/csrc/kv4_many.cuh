// kv4_many.cuh -- attention over the 4-bit cache where many rows read it: prompts and their pieces.
//
// Bound by the tensor cores: 4 D operations for every pair of a row and a token that it sees. A work item
// is a tile of 256 rows (128 of heads past 128 channels), tokens by the heads that share keys, against
// the tokens that they see, 128 (64) at a time. One CTA a processor takes items in turn from a counter,
// the longest of a sequence first.
//
// The roles of a CTA: a warpgroup turns codes into 16-bit floats, in shared memory as the tensor cores
// read them, mid + scale (code - 7.5) rounded once; one thread issues the tcgen05.mma, of each half of
// the rows in turn; a warpgroup for each half has a row to a thread, whose scores it reads from tensor
// memory, and where it puts the weights in their place, as the next product's A side. While one half's
// exponentials run the other half's products do. Sums keep the maximum that they were begun with until
// it is passed by 2^8; only then a row's sums in tensor memory are multiplied.
//
// Why this shape: a tile of tokens' codes cost as much of the issue slots as its exponentials for 128
// rows, so they serve 256; the two halves' scores and sums take all of tensor memory's 512 columns at 128
// channels. Of 128 tokens the products are 2097 cycles; their operands' reads from shared memory 1536,
// the codes' decoding 512 of writes, 32768 exponentials 2048 of the special units.
//
// Every wait is bounded; a role that gives up records it, and all leave at the item's end.
#pragma once
#include "kv4_math.cuh"
#include "ptx.cuh"

namespace uor {

namespace {

constexpr int THREADS = 512;
constexpr int REGS_SOFTMAX = 200, REGS_DECODE = 80, REGS_CONTROL = 32;
static_assert(2 * REGS_SOFTMAX + REGS_DECODE + REGS_CONTROL <= 4 * 128, "registers of the launch");
constexpr int DECODERS = 4;       // warps
constexpr uint32_t NAP_NS = 1000;  // a wait's sleep between looks; an arrival ends it at once

struct ManyAttend {
    AttendArgs a;
    const int64_t* before;  // [seqs + 1] items before each sequence's
    unsigned* next;         // the item that is taken next
    int* status;
    uint64_t budget_ns;
};

template <int D>
struct Shape {
    static constexpr int HALVES = D <= 128 ? 2 : 1;      // of 128 rows
    static constexpr int TOKENS = D <= 128 ? 128 : 64;   // of a step
    static constexpr int BLOCKS = TOKENS / KV_BLOCK;
    static constexpr int ATOMS = (D + 63) / 64;          // of 64 channels, the 128 bytes that a swizzle spans
    static constexpr int KSTAGES = 2, VSTAGES = D <= 192 ? 2 : 1, RING = 3;
    static constexpr int Q_ATOM = 128 * 128, Q_HALF = ATOMS * Q_ATOM;
    static constexpr int T_ATOM = TOKENS * 128, T_BYTES = ATOMS * T_ATOM;  // a step's keys, or values
    static constexpr int S_AT = 0, O_AT = HALVES * TOKENS;  // tensor-memory columns: scores, sums
    static constexpr int BARS = 1 + 2 * KSTAGES + 2 * VSTAGES + 3 * HALVES + 1;
    static constexpr int FIXED = HALVES * Q_HALF + KSTAGES * T_BYTES + VSTAGES * T_BYTES;
    static_assert(O_AT + HALVES * D <= 512, "tensor memory");
    static int smem(int groups) { return 1024 + FIXED + DECODERS * RING * kv_block_bytes(D, groups) + BARS * 8 + 4 * BLOCKS + 64; }
};

// What one item is; the same for all roles.
struct Item {
    int seq, head, tile;
};

// Eight codes of a word less 7.5: of channels (0, 4), (1, 5), (2, 6), (3, 7), or of a pair of tokens four
// channels each. 16 + code (64 + code in float16) is an exponent or-ed to the code's bits.
template <typename T>
__device__ __forceinline__ void centred(uint32_t w, uint32_t (&x)[4]) {
    if constexpr (std::is_same<T, __half>::value) {
        x[0] = and_or(w << 4, 0x00F000F0u, 0x54005400u), x[1] = and_or(w, 0x00F000F0u, 0x54005400u);
        x[2] = and_or(w >> 4, 0x00F000F0u, 0x54005400u), x[3] = and_or(w >> 8, 0x00F000F0u, 0x54005400u);
#pragma unroll
        for (int i = 0; i < 4; ++i) asm("add.rn.f16x2 %0, %0, %1;" : "+r"(x[i]) : "r"(0xD478D478u));  // -71.5
    } else {
        x[0] = and_or(w << 3, 0x00780078u, 0x41804180u), x[1] = and_or(w >> 1, 0x00780078u, 0x41804180u);
        x[2] = and_or(w >> 5, 0x00780078u, 0x41804180u), x[3] = and_or(w >> 9, 0x00780078u, 0x41804180u);
#pragma unroll
        for (int i = 0; i < 4; ++i) asm("add.rn.bf16x2 %0, %0, %1;" : "+r"(x[i]) : "r"(0xC1BCC1BCu));  // -23.5
    }
}
template <typename T>
__device__ __forceinline__ uint32_t fma_half2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    if constexpr (std::is_same<T, __half>::value)
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    else
        asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
__device__ __forceinline__ void sts128(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// The items before each sequence's, and the first to be taken.
__global__ void __launch_bounds__(1024) items_kernel(const __grid_constant__ AttendArgs a, int tile_rows, int tile_blocks, int64_t* before,
                                                     unsigned* next) {
    __shared__ int64_t sums[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    int64_t total = 0;
    for (int s0 = 0; s0 < a.batch.seqs; s0 += 1024) {
        const int s = s0 + threadIdx.x;
        const Share share = s < a.batch.seqs ? Share(Sequence(a.batch, s), a, tile_rows, tile_blocks) : Share();
        int64_t mine = s < a.batch.seqs ? static_cast<int64_t>(share.row_tiles) * a.kv.heads : 0;
        const int64_t own = mine;
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, mine, o);
            if (lane >= o) mine += v;
        }
        __syncthreads();
        if (lane == 31) sums[warp] = mine;
        __syncthreads();
        int64_t at = total + mine - own;
        for (int w = 0; w < 32; ++w) {
            if (w < warp) at += sums[w];
            total += sums[w];
        }
        if (s < a.batch.seqs) before[s] = at;
    }
    if (threadIdx.x == 0) before[a.batch.seqs] = total, *next = 0;
}

template <typename T, int D>
__global__ void __launch_bounds__(THREADS, 1) many_kernel(const __grid_constant__ ManyAttend p) {
    using Z = Shape<D>;
    constexpr int N32 = D / 32;
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Item items[2];
    __shared__ uint32_t tmem_slot;
    const AttendArgs& a = p.a;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* keys_at = smem + Z::HALVES * Z::Q_HALF;
    uint8_t* values_at = keys_at + Z::KSTAGES * Z::T_BYTES;
    uint8_t* rings = values_at + Z::VSTAGES * Z::T_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(rings + DECODERS * Z::RING * a.kv.block_bytes);
    uint8_t* there = reinterpret_cast<uint8_t*>(bars + Z::BARS);  // [4][BLOCKS]: whether a step's blocks are
    const uint32_t qfull = smem_u32(bars), kfull = qfull + 8, kempty = kfull + 8 * Z::KSTAGES;
    const uint32_t vfull = kempty + 8 * Z::KSTAGES, vempty = vfull + 8 * Z::VSTAGES;
    const uint32_t sfull = vempty + 8 * Z::VSTAGES, pfull = sfull + 8 * Z::HALVES, ofull = pfull + 8 * Z::HALVES;
    const uint32_t drain = ofull + 8 * Z::HALVES;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wg = warp >> 2;

    if (threadIdx.x == 0) {
        mbar_init(qfull, 4 * Z::HALVES);
        for (int i = 0; i < Z::KSTAGES; ++i) mbar_init(kfull + 8 * i, DECODERS), mbar_init(kempty + 8 * i, 1);
        for (int i = 0; i < Z::VSTAGES; ++i) mbar_init(vfull + 8 * i, DECODERS), mbar_init(vempty + 8 * i, 1);
        for (int i = 0; i < Z::HALVES; ++i) mbar_init(sfull + 8 * i, 1), mbar_init(pfull + 8 * i, 4), mbar_init(ofull + 8 * i, 1);
        mbar_init(drain, 1);
        fence_barrier_init();
    }
    if (warp == 13) tmem_alloc(smem_u32(&tmem_slot), 512);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // Takes an item; none left: seq is -1.
    auto take = [&](int slot) {
        const int64_t x = atomicAdd(p.next, 1u), total = p.before[a.batch.seqs];
        Item it{-1, 0, 0};
        if (x < total) {
            int lo = 0, hi = a.batch.seqs;  // before[lo] <= x < before[hi]
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (p.before[mid] <= x) lo = mid;
                else hi = mid;
            }
            while (p.before[lo + 1] <= x) ++lo;  // past sequences without rows
            const int rel = static_cast<int>(x - p.before[lo]), tiles = static_cast<int>(p.before[lo + 1] - p.before[lo]) / a.kv.heads;
            it.seq = lo, it.tile = tiles - 1 - rel / a.kv.heads, it.head = rel % a.kv.heads;
        }
        items[slot] = it;
    };
    if (warp == 14 && lane == 0) take(0);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    // A role's items, one after another: all leave an item together.
    bool ok = true;
    uint32_t steps_done = 0;  // of the items before this one
    auto end = [&](int steps) {
        steps_done += steps;
        tc_fence_before();
        __syncwarp();
        const bool on = bar_and_all(1, THREADS, ok);
        tc_fence_after();
        return on;
    };
    auto steps_of = [&](const Share& share) { return (share.blocks + Z::BLOCKS - 1) / Z::BLOCKS; };
    if (wg < Z::HALVES) {
        regs_up<REGS_SOFTMAX>();
        for (int n = 0;; ++n) {
            const Item it = items[n & 1];
            if (it.seq < 0) break;
            const Sequence seq(a.batch, it.seq);
            const Share share(seq, a, 128 * Z::HALVES, Z::BLOCKS);
            const int steps = steps_of(share);
            // A row to a thread.
            const int half = wg, t = threadIdx.x & 127;
            const uint32_t lanes = static_cast<uint32_t>(t & ~31) << 16;
            const uint32_t scores = tmem + lanes + Z::S_AT + half * Z::TOKENS, sums = tmem + lanes + Z::O_AT + half * D;
            const int r = it.tile * 128 * Z::HALVES + half * 128 + t;
            const bool live = r < share.rows;
            const int at = live ? seq.at + r / a.share : -1;
            const int row = seq.first + (live ? r / a.share : 0), col = it.head * a.share + (live ? r % a.share : 0);
            // The row's query, its channels in each eight as the keys' words have them, and negated
            // where the scale is, so that the largest score is the largest product.
            {
                const uint16_t* from = static_cast<const uint16_t*>(a.q.p) + row * a.q.rs + static_cast<int64_t>(col) * D;
                const uint32_t to = smem_u32(smem) + half * Z::Q_HALF + t * 128, flip = a.scale < 0 ? 0x80008000u : 0u;
#pragma unroll 4
                for (int i = 0; i < D / 8; ++i) {
                    uint32_t w[4] = {0, 0, 0, 0};
                    if (live) {
                        if (a.q.vec) {
                            const uint4 v = *reinterpret_cast<const uint4*>(from + 8 * i);
                            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
                        } else {
#pragma unroll
                            for (int k = 0; k < 4; ++k) w[k] = from[8 * i + 2 * k] | static_cast<uint32_t>(from[8 * i + 2 * k + 1]) << 16;
                        }
#pragma unroll
                        for (int k = 0; k < 4; ++k) w[k] ^= flip;
                    }
                    sts128(to + (i >> 3) * Z::Q_ATOM + (((i & 7) ^ (t & 7)) << 4), __byte_perm(w[0], w[2], 0x5410), __byte_perm(w[0], w[2], 0x7632),
                           __byte_perm(w[1], w[3], 0x5410), __byte_perm(w[1], w[3], 0x7632));
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(qfull);
            }
            // Positions of this half's rows.
            const int first_row = it.tile * 128 * Z::HALVES + half * 128, last_row = min(first_row + 127, share.rows - 1);
            const int nearest = min(seq.at + first_row / a.share, seq.keys - 1);
            const int behind = a.window ? seq.at + last_row / a.share - a.window : -1;
            const float k = fmaxf(fabsf(a.scale) * LOG2E, 1e-38f);  // of a scale of 0 still what -inf becomes -inf by
            const uint64_t kk = pair_of(k, k);
            float m = -INFINITY;
            uint64_t l = 0;
            for (int j = 0; j < steps; ++j) {
                const uint32_t g = steps_done + j;
                if (!mbar_wait_warp_hint(sfull + 8 * half, g & 1, p.budget_ns, p.status, KERR_TIMEOUT_EPILOGUE, NAP_NS)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                // Where some token of the step is hidden from some row.
                const int b0 = j * Z::BLOCKS, b1 = b0 + Z::BLOCKS - 1;
                bool hidden = b1 >= share.blocks;
                if (!hidden) {
                    const int low = share.block_at(b0) * KV_BLOCK, high = share.block_at(b1) * KV_BLOCK + KV_BLOCK - 1;
                    hidden = high > nearest || (a.window && low <= behind && !(b1 < share.sink_blocks && high < a.sinks));
                    if constexpr (Z::BLOCKS == 8) hidden |= *reinterpret_cast<const uint64_t*>(there + (g & 3) * 8) != 0x0101010101010101ull;
                    else hidden |= *reinterpret_cast<const uint32_t*>(there + (g & 3) * 4) != 0x01010101u;
                }
                // 32 tokens' scores travel at a time, the next while these are used. They are read twice, for
                // their maximum and for their weights: 128 of them do not fit the registers.
                uint32_t s[2][32];
                auto hide = [&](uint32_t (&v)[32], int c) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int b = b0 + c / KV_BLOCK + e, token = share.block_at(b) * KV_BLOCK;
                        const bool block = b < share.blocks && there[(g & 3) * Z::BLOCKS + c / KV_BLOCK + e];
                        const int upto = block ? min(at, seq.keys - 1) : -1;
                        const int window = a.window ? at - a.window : -1;
#pragma unroll
                        for (int i = 0; i < KV_BLOCK; ++i) {
                            const int position = token + i;
                            if (!(position <= upto && (position > window || position < a.sinks))) v[e * KV_BLOCK + i] = __float_as_uint(-INFINITY);
                        }
                    }
                };
                tmem_ld32(scores, s[0]);
                float part[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < Z::TOKENS; c += 32) {
                    auto& v = s[c / 32 & 1];
                    tmem_ld_wait();
                    tmem_ld32(scores + (c + 32) % Z::TOKENS, s[c / 32 + 1 & 1]);
                    if (hidden) hide(v, c);
#pragma unroll
                    for (int i = 0; i < 32; ++i) part[i & 3] = fmaxf(part[i & 3], __uint_as_float(v[i]));
                }
                const float top = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])) * k;
                const bool higher = top > m + 8.0f;
                if (__any_sync(0xffffffffu, higher)) {
                    const float next = higher ? top : m;
                    const float by = m == -INFINITY ? 0.0f : ex2(m - next);
                    m = next;
                    l = mul2(l, pair_of(by, by));
                    if (j) {  // the sums so far, once the product before this one is in them
                        if (!mbar_wait_warp_hint(ofull + 8 * half, (g - 1) & 1, p.budget_ns, p.status, KERR_TIMEOUT_EPILOGUE, NAP_NS)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
#pragma unroll
                        for (int c = 0; c < D; c += 16) {
                            uint32_t v[16];
                            tmem_ld16(sums + c, v);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * by);
                            tmem_st16(sums + c, v);
                        }
                    }
                }
                const float minus = m == -INFINITY ? 0.0f : -m;
                const uint64_t mm = pair_of(minus, minus);
                uint64_t l2 = 0;
#pragma unroll
                for (int c = 0; c < Z::TOKENS; c += 32) {
                    auto& v = s[c / 32 & 1];
                    tmem_ld_wait();
                    if (c + 32 < Z::TOKENS) tmem_ld32(scores + c + 32, s[c / 32 + 1 & 1]);
                    if (hidden) hide(v, c);
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        float x, y;
                        parts_of(fma2(pair_of(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), kk, mm), x, y);
                        x = ex2(x), y = ex2(y);
                        if (i & 2) l2 = add2(l2, pair_of(x, y));
                        else l = add2(l, pair_of(x, y));
                        w[i / 2] = pack<T>(x, y);
                    }
                    tmem_st16(scores + c / 2, w);  // over scores that were read
                }
                l = add2(l, l2);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(pfull + 8 * half);
            }
            if (ok && steps &&
                !mbar_wait_warp_hint(ofull + 8 * half, (steps_done + steps - 1) & 1, p.budget_ns, p.status, KERR_TIMEOUT_EPILOGUE, NAP_NS))
                ok = false;
            if (ok) {
                tc_fence_after();
                float l0, l1;
                parts_of(l, l0, l1);
                const float all = l0 + l1, inverse = all == 0.0f ? 0.0f : 1.0f / all;
                uint16_t* to = static_cast<uint16_t*>(a.y.p) + row * a.y.rs + static_cast<int64_t>(col) * D;
#pragma unroll 2
                for (int c = 0; c < D; c += 16) {
                    uint32_t v[16];
                    if (steps) {
                        tmem_ld16(sums + c, v);
                        tmem_ld_wait();
                    }
                    uint32_t w[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        w[i] = all == 0.0f ? 0u : pack<T>(__uint_as_float(v[2 * i]) * inverse, __uint_as_float(v[2 * i + 1]) * inverse);
                    if (live) {
                        if (a.y.vec) {
                            reinterpret_cast<uint4*>(to + c)[0] = make_uint4(w[0], w[1], w[2], w[3]);
                            reinterpret_cast<uint4*>(to + c)[1] = make_uint4(w[4], w[5], w[6], w[7]);
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; ++i) to[c + i] = static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1)));
                        }
                    }
                }
                if (live && a.lse.p) static_cast<float*>(a.lse.p)[row * a.lse.rs + col] = (m + log2f(all)) * LN2;
                tc_fence_before();
            }
            if (!end(steps)) break;
        }
    } else if (wg == 2) {
        regs_down<REGS_DECODE>();
        for (int n = 0;; ++n) {
            const Item it = items[n & 1];
            if (it.seq < 0) break;
            const Sequence seq(a.batch, it.seq);
            const Share share(seq, a, 128 * Z::HALVES, Z::BLOCKS);
            const int steps = steps_of(share);
            // Blocks w, w + 4 of each step, through a ring of this warp's own.
            constexpr int EACH = Z::BLOCKS / DECODERS;
            const int w = warp & 3, block_bytes = a.kv.block_bytes, groups = a.kv.groups, to_group = a.kv.group_shift - 5;
            uint8_t* ring = rings + w * Z::RING * block_bytes;
            const uint32_t ring_at = smem_u32(ring);
            const int count = steps * EACH;  // of blocks; some behind the last
            int places = -1;
            auto index = [&](int i) { return i / EACH * Z::BLOCKS + w + i % EACH * DECODERS; };
            auto place_of = [&](int i) { return __shfl_sync(0xffffffffu, places, i & 31); };
            uint32_t gone = 0;  // of the ring's blocks
            auto load = [&](int i) {
                if (i < count) {
                    if ((i & 31) == 0) {
                        places = -1;
                        const int b = index(i + lane);
                        if (i + lane < count && b < share.blocks) {
                            const int block = share.block_at(b), in_page = a.kv.page_shift - 4;
                            const int page = a.batch.table[it.seq * a.batch.table_rs + (block >> in_page)];
                            if (static_cast<uint32_t>(page) < a.kv.pages)
                                places = ((page * a.kv.heads + it.head) << in_page) + (block & ((1 << in_page) - 1));
                        }
                    }
                    const int place = place_of(i), slot = i % Z::RING;
                    gone = place < 0 ? gone | 1u << slot : gone & ~(1u << slot);
                    if (place >= 0) {
                        const uint8_t* from = a.kv.pool + static_cast<int64_t>(place) * block_bytes;
                        for (int b = lane * 16; b < block_bytes; b += 512) cp_async(ring_at + slot * block_bytes + b, from + b);
                    }
                }
                cp_commit();
            };
#pragma unroll
            for (int i = 0; i < Z::RING - 1; ++i) load(i);
            const int t = lane >> 2, c = lane & 3;
            for (int j = 0; j < steps && ok; ++j) {
                const uint32_t g = steps_done + j, ks = g % Z::KSTAGES, vs = g % Z::VSTAGES;
                if (!mbar_wait_warp_hint(kempty + 8 * ks, (g / Z::KSTAGES & 1) ^ 1, p.budget_ns, p.status, KERR_TIMEOUT_PRODUCER, NAP_NS)) {
                    ok = false;
                    break;
                }
                // keys: all of the step's blocks of this warp, then its values
#pragma unroll
                for (int e = 0; e < EACH; ++e) {
                    const int i = j * EACH + e, slot = i % Z::RING, in_step = w + e * DECODERS;
                    cp_wait<Z::RING - 2>();
                    __syncwarp();
                    // With two blocks a step the first one's values are decoded before its slot is wanted
                    // again; see below.
                    const uint8_t* block = ring + slot * block_bytes;
                    const bool missing = gone >> slot & 1;
                    if (lane == 0) there[(g & 3) * Z::BLOCKS + in_step] = !missing;
                    const int token = missing ? 0 : share.block_at(index(i)) * KV_BLOCK;
                    const uint32_t to = smem_u32(keys_at) + ks * Z::T_BYTES;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int tok = h * 8 + t, row = in_step * KV_BLOCK + tok;
                        uint32_t v[N32];
                        words<N32>(block + (tok * 4 + c) * N32 * 4, v);
                        const uint32_t odd = (tok & 1) ? 0x3232 : 0x1010;
                        const bool none = missing || token + tok >= seq.keys;  // what lies there may be anything
                        uint32_t scale = 0, mid = 0;
#pragma unroll
                        for (int n32 = 0; n32 < N32; ++n32) {
                            if ((n32 & ((1 << to_group) - 1)) == 0) {
                                const uint2 q = *reinterpret_cast<const uint2*>(block + 8 * D + ((tok >> 1) * groups + (n32 >> to_group)) * 8);
                                scale = none ? 0u : __byte_perm(q.x, 0, odd), mid = none ? 0u : __byte_perm(q.y, 0, odd);
                            }
                            uint32_t x[4];
                            centred<T>(v[n32], x);
#pragma unroll
                            for (int b = 0; b < 4; ++b) x[b] = fma_half2<T>(scale, x[b], mid);
                            sts128(to + (n32 >> 1) * Z::T_ATOM + row * 128 + ((((n32 & 1) * 4 + c) ^ (row & 7)) << 4), x[0], x[1], x[2], x[3]);
                        }
                    }
                    if (e == 0 && EACH == 2) load(i + Z::RING - 1);
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(kfull + 8 * ks);
                if (!mbar_wait_warp_hint(vempty + 8 * vs, (g / Z::VSTAGES & 1) ^ 1, p.budget_ns, p.status, KERR_TIMEOUT_PRODUCER, NAP_NS)) {
                    ok = false;
                    break;
                }
#pragma unroll
                for (int e = 0; e < EACH; ++e) {
                    const int i = j * EACH + e, slot = i % Z::RING, in_step = w + e * DECODERS;
                    const uint8_t* block = ring + slot * block_bytes;
                    const bool missing = gone >> slot & 1;
                    const int token = missing ? 0 : share.block_at(index(i)) * KV_BLOCK;
                    const uint32_t to = smem_u32(values_at) + vs * Z::T_BYTES;
                    // Two tokens, 8 h + 2 c and the next, by eight channels of every 32.
                    const int h = lane >> 4, eight = lane >> 2 & 3;
                    const int tok = 8 * h + 2 * c, row = in_step * KV_BLOCK + tok;
                    const uint8_t* codes = block + 8 * D + 64 * groups + ((h * 8 + 2 * eight) * 4 + c) * N32 * 4;
                    uint32_t v[2][N32];
                    words<N32>(codes, v[0]);
                    words<N32>(codes + 4 * N32 * 4, v[1]);
                    const uint32_t keep = missing ? 0u : (token + tok < seq.keys ? 0xFFFFu : 0u) | (token + tok + 1 < seq.keys ? 0xFFFF0000u : 0u);
                    uint32_t scale = 0, mid = 0;
#pragma unroll
                    for (int n32 = 0; n32 < N32; ++n32) {
                        if ((n32 & ((1 << to_group) - 1)) == 0) {
                            const uint2 q = *reinterpret_cast<const uint2*>(block + 16 * D + 64 * groups + ((tok >> 1) * groups + (n32 >> to_group)) * 8);
                            scale = q.x & keep, mid = q.y & keep;
                        }
                        uint32_t x[2][4];
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            centred<T>(v[b][n32], x[b]);
#pragma unroll
                            for (int k = 0; k < 4; ++k) x[b][k] = fma_half2<T>(scale, x[b][k], mid);
                        }
                        const uint32_t dst = to + (n32 >> 1) * Z::T_ATOM + row * 128;
                        const uint32_t chunk = (n32 & 1) * 4 + eight;
                        sts128(dst + ((chunk ^ (row & 7)) << 4), __byte_perm(x[0][0], x[0][1], 0x5410), __byte_perm(x[0][2], x[0][3], 0x5410),
                               __byte_perm(x[1][0], x[1][1], 0x5410), __byte_perm(x[1][2], x[1][3], 0x5410));
                        sts128(dst + 128 + ((chunk ^ ((row + 1) & 7)) << 4), __byte_perm(x[0][0], x[0][1], 0x7632), __byte_perm(x[0][2], x[0][3], 0x7632),
                               __byte_perm(x[1][0], x[1][1], 0x7632), __byte_perm(x[1][2], x[1][3], 0x7632));
                    }
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(vfull + 8 * vs);
                load((j + 1) * EACH - 1 + Z::RING - 1);
            }
            cp_wait<0>();
            if (!end(steps)) break;
        }
    } else {
        regs_down<REGS_CONTROL>();
        for (int n = 0;; ++n) {
            const Item it = items[n & 1];
            if (it.seq < 0) break;
            int steps = 0;
            if (warp == 12) {
                const Sequence seq(a.batch, it.seq);
                steps = steps_of(Share(seq, a, 128 * Z::HALVES, Z::BLOCKS));
                if (lane == 0) {
                    constexpr uint32_t QK = idesc_f16(128, Z::TOKENS, BF16), PV = idesc_f16(128, D, BF16, true);
                    auto values = [&](int half, uint32_t g, bool first) {  // sums += weights values of step g
                        const uint32_t v = smem_u32(values_at) + g % Z::VSTAGES * Z::T_BYTES;
#pragma unroll
                        for (int i = 0; i < Z::TOKENS / 16; ++i)
                            mma_f16_ts(tmem + Z::O_AT + half * D, tmem + Z::S_AT + half * Z::TOKENS + i * 8, smem_desc_sw128(v + i * 2048, Z::T_ATOM, 1024), PV,
                                       !(first && i == 0));
                        mma_commit(ofull + 8 * half);
                        if (half == Z::HALVES - 1) mma_commit(vempty + 8 * (g % Z::VSTAGES));
                    };
                    if (steps) ok = mbar_wait(qfull, n & 1, p.budget_ns, p.status, KERR_TIMEOUT_MMA_FULL);
                    for (int j = 0; j <= steps && ok && steps; ++j) {
                        const uint32_t g = steps_done + j;
                        if (j < steps) ok = mbar_wait(kfull + 8 * (g % Z::KSTAGES), g / Z::KSTAGES & 1, p.budget_ns, p.status, KERR_TIMEOUT_MMA_FULL);
                        for (int half = 0; half < Z::HALVES && ok; ++half) {
                            if (j) {
                                ok = mbar_wait(pfull + 8 * half, (g - 1) & 1, p.budget_ns, p.status, KERR_TIMEOUT_MMA_ACC) &&
                                     mbar_wait(vfull + 8 * ((g - 1) % Z::VSTAGES), (g - 1) / Z::VSTAGES & 1, p.budget_ns, p.status, KERR_TIMEOUT_MMA_FULL);
                                if (!ok) break;
                                tc_fence_after();
                                values(half, g - 1, j == 1);
                            }
                            if (j < steps) {
                                tc_fence_after();
                                const uint32_t q = smem_u32(smem) + half * Z::Q_HALF, k = smem_u32(keys_at) + g % Z::KSTAGES * Z::T_BYTES;
#pragma unroll
                                for (int i = 0; i < D / 16; ++i)
                                    mma_f16(tmem + Z::S_AT + half * Z::TOKENS, smem_desc_sw128(q + i / 4 * Z::Q_ATOM + i % 4 * 32, 16, 1024),
                                            smem_desc_sw128(k + i / 4 * Z::T_ATOM + i % 4 * 32, 16, 1024), QK, i != 0);
                                mma_commit(sfull + 8 * half);
                                if (half == Z::HALVES - 1) mma_commit(kempty + 8 * (g % Z::KSTAGES));
                            }
                        }
                    }
                    if (!ok) {  // what was issued ends before the memory goes
                        mma_commit(drain);
                        mbar_wait(drain, 0, p.budget_ns, p.status, KERR_TIMEOUT_DRAIN);
                    }
                }
                __syncwarp();
            } else if (warp == 14 && lane == 0) {
                take((n + 1) & 1);
            }
            if (!end(steps)) break;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 13) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <typename T, int D>
int launch_many(uor_b200_ctx* ctx, const AttendArgs& a, uor_b200_route* route) {
    using Z = Shape<D>;
    auto* kernel = many_kernel<T, D>;
    const int smem = Z::smem(a.kv.groups);
    static bool ready[64] = {};
    if (!ready[ctx->device & 63]) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Z::smem(D / 32)) != cudaSuccess) return UOR_B200_DEVICE_ERROR;
        ready[ctx->device & 63] = true;
    }
    int st = UOR_B200_OK;
    auto* ws = static_cast<uint8_t*>(ctx_buffer(ctx, SLOT_WS, (a.batch.seqs + 2) * 8, &st));
    if (!ws) return st;
    ManyAttend p{};
    p.a = a;
    auto* before = reinterpret_cast<int64_t*>(ws);
    p.before = before;
    p.next = reinterpret_cast<unsigned*>(before + a.batch.seqs + 1);
    p.status = ctx->d_status;
    p.budget_ns = ctx->budget_ns;
    items_kernel<<<1, 1024, 0, ctx->stream>>>(a, 128 * Z::HALVES, Z::BLOCKS, before, p.next);
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(ctx->sm_count);
    c.blockDim = dim3(THREADS);
    c.dynamicSmemBytes = smem;
    c.stream = ctx->stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &attr;
    c.numAttrs = 1;
    route->tile_m = 128 * Z::HALVES, route->tile_n = Z::TOKENS, route->tile_k = D;
    route->ctas = static_cast<uint32_t>(ctx->sm_count);
    return cuda_status(cudaLaunchKernelEx(&c, kernel, p));
}

}  // namespace

template <typename T>
int kv4_many(uor_b200_ctx* ctx, const AttendArgs& a, uor_b200_route* route) {
    switch (a.kv.dim) {
    case 64: return launch_many<T, 64>(ctx, a, route);
    case 96: return launch_many<T, 96>(ctx, a, route);
    case 128: return launch_many<T, 128>(ctx, a, route);
    case 192: return launch_many<T, 192>(ctx, a, route);
    default: return launch_many<T, 256>(ctx, a, route);
    }
}

}  // namespace uor
