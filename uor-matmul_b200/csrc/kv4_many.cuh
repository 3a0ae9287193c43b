// kv4_many.cuh -- attention over the 4-bit cache where many rows read it: prompts and their pieces.
//
// A work item is a tile of 256 rows (128 of heads past 128 channels, or where items are few) by the heads that share keys, against
// the tokens that they see, 64 at a time. One CTA a processor takes items in turn from a counter, the
// longest of a sequence first.
//
// The mathematics. With x = mid + scale (code - 7.5), of each group of channels
//   q . k = sum q (scale (code - 7.5)) + mid sum(q).
// A scale has eight bits (eleven in float16) and code - 7.5 four: their product is exactly two numbers of
// the 16-bit type, what it is rounded to and what that leaves, and the middles multiply the groups' sums of
// queries, two parts each, in a product of their own. So scores are f32's own, and so is lse. (Keys rounded
// once to 16 bits, and half the products: 8192 of 8192 in 692 us, but lse 3e-5 to 4e-4 off in bfloat16, 4e-6
// to 5e-5 in float16; now 4e-7.) Values and weights are rounded once to 16 bits, as their type has
// them. Queries are brought below 2 by a power of two, for the sums' sake in float16.
//
// The roles of a CTA: a warpgroup turns keys' codes, and another values', into 16-bit floats in shared
// memory as the tensor cores read them, from rings of blocks that bulk copies fill; a thread for each half
// of the rows issues its tcgen05.mma; a warpgroup for each half has a row to a thread, whose scores it
// reads from tensor memory, and where it puts the weights in their place, as the next product's A side.
// Scores of odd and even steps have columns of their own, so that the next step's are at hand when a
// step's weights are done (8192 of 8192, keys rounded once: 927 us -> 705). Sums keep the maximum that they
// were begun with until it is passed by 2^8; only then a row's sums in tensor memory are multiplied.
//
// Why this shape. A step's codes cost as many issue slots as the exponentials of 128 rows, so they serve
// 256; the two halves' scores and sums take all of tensor memory's 512 columns at 128 channels. A query tile
// comes from shared memory for both parts of the keys at once (898 us -> 845): read for each, the
// operands' 12 KB for 64 cycles of products pass its 128 bytes a cycle.
//
// 8192 of 8192 tokens, 32 heads over 8 of 128 channels, bfloat16: 845 us, 651 TFLOP/s of the 4 D operations
// of each pair. A step of 64 tokens takes 1.9 us at the 1.56 GHz that the processors run at under it, 2900
// cycles: 1600 of products, shared memory some 2000 for their operands, the decoded values and the rings.
// 2048 of 4096: 189 us; six sequences of up to 300 of 2500: 67 us, where items are few and uneven.
//
// Every wait is bounded; a role that gives up records it, and all leave at the item's end.
#pragma once
#include "kv4_math.cuh"
#include "ptx.cuh"

namespace uor {

namespace {

constexpr int THREADS = 640;
constexpr int REGS_SOFTMAX = 136, REGS_DECODE = 80, REGS_CONTROL = 40;
static_assert(2 * REGS_SOFTMAX + 2 * REGS_DECODE + REGS_CONTROL <= 5 * 96, "registers of the launch");
constexpr int DECODERS = 4;  // warps for the keys, and for the values

struct ManyAttend {
    AttendArgs a;
    const int64_t* before;  // [seqs + 1] items before each sequence's
    unsigned long long* next;  // the item that is taken next
    int* status;
    uint64_t budget_ns;
};

template <int D, int H>
struct Shape {
    static constexpr int HALVES = H;                     // of 128 rows
    static constexpr int TOKENS = 64;                    // of a step
    static constexpr int BLOCKS = TOKENS / KV_BLOCK;
    static constexpr int ATOMS = (D + 63) / 64;          // of 64 channels, the 128 bytes that a swizzle spans
    static constexpr int KSTAGES = D <= 128 ? 2 : 1, VSTAGES = D <= 128 ? 3 : D <= 192 ? 2 : 1;
    static constexpr int RING = D <= 192 ? 3 : 2;        // blocks' keys, or values, under way of each decoding warp
    static constexpr int THERE = 8;                      // steps that the decoders' notes are kept for
    static constexpr int Q_ATOM = 128 * 128, Q_SUMS = ATOMS * Q_ATOM, Q_HALF = Q_SUMS + 128 * 32;
    static constexpr int T_ATOM = TOKENS * 128, T_BYTES = ATOMS * T_ATOM;  // a step's values
    // A step's keys without their middles, rounded, what that left, and the middles.
    static constexpr int K_MIDS = 2 * T_BYTES, K_BYTES = K_MIDS + TOKENS * 32;
    static constexpr int S_AT = 0, O_AT = 2 * HALVES * TOKENS;  // tensor-memory columns: scores, sums
    static constexpr int BARS = HALVES + 3 + 2 * KSTAGES + 2 * VSTAGES + 6 * HALVES + 2 + 2 * DECODERS * RING;
    static constexpr int FIXED = HALVES * Q_HALF + KSTAGES * K_BYTES + VSTAGES * T_BYTES;
    static_assert(BLOCKS == DECODERS, "a block of a step to each decoding warp");
    static_assert(O_AT + HALVES * D <= 512, "tensor memory");
    static int smem(int groups) { return 1024 + FIXED + DECODERS * RING * kv_block_bytes(D, groups) + BARS * 8 + THERE * BLOCKS; }
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
// x: the product of scale and x, rounded; left: exactly what that left, four bits at most.
template <typename T>
__device__ __forceinline__ void product(uint32_t scale, uint32_t& x, uint32_t& left) {
    uint32_t p, minus;
    if constexpr (std::is_same<T, __half>::value)
        asm("mul.rn.f16x2 %0, %2, %3;\n neg.f16x2 %1, %0;" : "=&r"(p), "=r"(minus) : "r"(scale), "r"(x));
    else
        asm("mul.rn.bf16x2 %0, %2, %3;\n neg.bf16x2 %1, %0;" : "=&r"(p), "=r"(minus) : "r"(scale), "r"(x));
    left = fma_half2<T>(scale, x, minus);
    x = p;
}
// Into the tensor cores' operands, which no thread reads: reads of the rings may pass it.
__device__ __forceinline__ void sts128(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d));
}

// mbar_wait whose looks are few instructions: the roles wait for one another most of the time, and looks
// take issue slots from those that work. The status is looked at every 512th time.
__device__ __forceinline__ bool wait_on(uint32_t bar, uint32_t parity, uint64_t budget_ns, int* status, int code) {
    uint64_t t0 = 0;  // the timer is slow to read: only by those who wait long
    while (true) {
        uint32_t done;
        asm volatile(
            "{\n .reg .pred p, q;\n .reg .u32 n;\n mov.u32 n, 512;\nAGAIN:\n"
            " mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n @p bra DONE;\n"
            " sub.u32 n, n, 1;\n setp.ne.u32 q, n, 0;\n @q bra AGAIN;\nDONE:\n selp.u32 %0, 1, 0, p;\n}\n"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (done) return true;
        if (*(volatile int*)status != 0) return false;
        const uint64_t now = globaltimer();
        if (t0 == 0) t0 = now;
        if (now - t0 > budget_ns) {
            atomicCAS(status, 0, code);
            return false;
        }
    }
}
__device__ __forceinline__ bool wait_on_warp(uint32_t bar, uint32_t parity, uint64_t budget_ns, int* status, int code) {
    uint64_t t0 = 0;
    for (uint32_t looks = 1;; ++looks) {
        uint32_t done = 0;
        asm volatile(
            "{\n .reg .pred p, first;\n setp.eq.u32 first, %3, 0;\n setp.ne.u32 p, 0, 0;\n"
            " @first mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
            : "=r"(done)
            : "r"(bar), "r"(parity), "r"(threadIdx.x & 31)
            : "memory");
        if (__any_sync(0xffffffffu, done)) return true;
        if ((looks & 511) == 0) {
            const uint64_t now = globaltimer();
            if (t0 == 0) t0 = now;
            const bool late = now - t0 > budget_ns;
            if (late) atomicCAS(status, 0, code);
            if (__any_sync(0xffffffffu, late || *(volatile int*)status != 0)) return false;
        }
    }
}
// A wait of the way out, when a role has given up: for what is under way, whatever the status.
__device__ __forceinline__ void wait_out(uint32_t bar, uint32_t parity, uint64_t budget_ns) {
    const uint64_t t0 = globaltimer();
    while (!mbar_try_wait(bar, parity) && globaltimer() - t0 <= budget_ns) {
    }
}
// Contiguous bytes (a multiple of 16, at multiples of 16) into shared memory, counted on a barrier.
__device__ __forceinline__ void bulk_load(uint32_t to, const void* from, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "l"(from), "r"(bytes), "r"(bar)
                 : "memory");
}

// The items before each sequence's, and the first to be taken.
__global__ void __launch_bounds__(1024) items_kernel(const __grid_constant__ AttendArgs a, int tile_rows, int tile_blocks, int64_t* before,
                                                     unsigned long long* next) {
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

template <typename T, int D, int H>
__global__ void __launch_bounds__(THREADS, 1) many_kernel(const __grid_constant__ ManyAttend p) {
    using Z = Shape<D, H>;
    constexpr int N32 = D / 32;
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Item items[2];
    __shared__ uint32_t tmem_slot;
    const AttendArgs& a = p.a;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* keys_at = smem + Z::HALVES * Z::Q_HALF;
    uint8_t* values_at = keys_at + Z::KSTAGES * Z::K_BYTES;
    uint8_t* rings = values_at + Z::VSTAGES * Z::T_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(rings + DECODERS * Z::RING * a.kv.block_bytes);
    uint8_t* there = reinterpret_cast<uint8_t*>(bars + Z::BARS);  // [THERE][BLOCKS]: whether a step's blocks are
    const uint32_t qfull = smem_u32(bars), ifull = qfull + 8 * Z::HALVES, iempty = ifull + 16, kfull = iempty + 8, kempty = kfull + 8 * Z::KSTAGES;
    const uint32_t vfull = kempty + 8 * Z::KSTAGES, vempty = vfull + 8 * Z::VSTAGES;
    // Scores, weights and sums of odd and even steps have signals of their own: a role may be two steps ahead
    // of another, and a signal's parity tells one filling from the next alone.
    const uint32_t sfull = vempty + 8 * Z::VSTAGES, pfull = sfull + 16 * Z::HALVES, ofull = pfull + 16 * Z::HALVES;
    const uint32_t drain = ofull + 16 * Z::HALVES;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wg = warp >> 2;

    if (threadIdx.x == 0) {
        for (int i = 0; i < Z::HALVES; ++i) mbar_init(qfull + 8 * i, 4);
        for (int i = 0; i < 2; ++i) mbar_init(ifull + 8 * i, 1);
        mbar_init(iempty, 5 * Z::HALVES + 2 * DECODERS);
        for (int i = 0; i < Z::KSTAGES; ++i) mbar_init(kfull + 8 * i, DECODERS), mbar_init(kempty + 8 * i, Z::HALVES);
        for (int i = 0; i < Z::VSTAGES; ++i) mbar_init(vfull + 8 * i, DECODERS), mbar_init(vempty + 8 * i, Z::HALVES);
        for (int i = 0; i < 2 * Z::HALVES; ++i) mbar_init(sfull + 8 * i, 1), mbar_init(pfull + 8 * i, 4), mbar_init(ofull + 8 * i, 1);
        for (int i = 0; i < 2 + 2 * DECODERS * Z::RING; ++i) mbar_init(drain + 8 * i, 1);
        fence_barrier_init();
    }
    if (warp == 17) tmem_alloc(smem_u32(&tmem_slot), 512);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // Takes an item; none left: seq is -1.
    auto take = [&](int slot) {
        const int64_t x = static_cast<int64_t>(atomicAdd(p.next, 1ull)), total = p.before[a.batch.seqs];
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
        return it.seq >= 0;
    };
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    // A role's items, one after another; every role goes on to the next as soon as it can. The lanes that
    // ask agree.
    bool ok = true;
    uint32_t steps_done = 0;  // of the items before this one
    auto item_at = [&](int n, Item* it) {
        if (!ok || !wait_on(ifull + 8 * (n & 1), n >> 1 & 1, p.budget_ns, p.status, KERR_TIMEOUT_PRODUCER)) return false;
        *it = items[n & 1];
        return it->seq >= 0;
    };
    auto next_item = [&](int n, Item* it) {
        return static_cast<bool>(__all_sync(0xffffffffu, item_at(n, it)));
    };
    // The next item is taken when all know theirs and the decoders, who are ahead, are through with it: taken
    // sooner, the last and shortest items would lie in line behind long ones.
    auto wants_next = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(iempty);
    };
    if (wg < Z::HALVES) {
        regs_up<REGS_SOFTMAX>();
        Item it;
        for (int n = 0; next_item(n, &it); ++n) {
            const Sequence seq(a.batch, it.seq);
            const Share share(seq, a, 128 * Z::HALVES, Z::BLOCKS, it.tile);
            const int steps = share.tiles;
            wants_next();
            // A row to a thread.
            const int half = wg, t = threadIdx.x & 127;
            const uint32_t lanes = static_cast<uint32_t>(t & ~31) << 16;
            const uint32_t scores_at = tmem + lanes + Z::S_AT + half * 2 * Z::TOKENS, sums = tmem + lanes + Z::O_AT + half * D;
            const int r = it.tile * 128 * Z::HALVES + half * 128 + t;
            const bool live = r < share.rows;
            const int at = live ? seq.at + r / a.share : -1;
            const int row = seq.first + (live ? r / a.share : 0), col = it.head * a.share + (live ? r % a.share : 0);
            // The row's query below 2 by a power of two, its channels in each eight as the keys' words have
            // them, and negated where the scale is, so that the largest score is the largest product; and
            // its groups' sums, that the middles multiply, in two parts.
            float up;
            {
                const uint16_t* from = static_cast<const uint16_t*>(a.q.p) + row * a.q.rs + static_cast<int64_t>(col) * D;
                const uint32_t to = smem_u32(smem) + half * Z::Q_HALF + t * 128, sums_to = smem_u32(smem) + half * Z::Q_HALF + Z::Q_SUMS + (t >> 3) * 256 + (t & 7) * 16;
                auto eight = [&](int i, uint32_t (&w)[4]) {
                    w[0] = w[1] = w[2] = w[3] = 0;
                    if (!live) return;
                    if (a.q.vec) {
                        const uint4 v = *reinterpret_cast<const uint4*>(from + 8 * i);
                        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; ++k) w[k] = from[8 * i + 2 * k] | static_cast<uint32_t>(from[8 * i + 2 * k + 1]) << 16;
                    }
                };
                float most = 0;
#pragma unroll 8
                for (int i = 0; i < D / 8; ++i) {
                    uint32_t w[4];
                    eight(i, w);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float2 v = two<T>(w[k]);
                        most = fmaxf(most, fmaxf(fabsf(v.x), fabsf(v.y)));
                    }
                }
                const uint32_t power = min(max(__float_as_uint(most) >> 23, 1u), 253u);  // most is 1 to 2 times 2^(power - 127)
                const float down = __uint_as_float((254 - power) << 23 | (a.scale < 0 ? 0x80000000u : 0u));
                up = __uint_as_float(power << 23);
                float sum = 0;
#pragma unroll 4
                for (int i = 0; i < D / 8; ++i) {
                    uint32_t w[4];
                    eight(i, w);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float2 v = two<T>(w[k]);
                        const float x = v.x * down, y = v.y * down;
                        sum += x + y;
                        w[k] = pack<T>(x, y);
                    }
                    sts128(to + (i >> 3) * Z::Q_ATOM + (((i & 7) ^ (t & 7)) << 4), __byte_perm(w[0], w[2], 0x5410), __byte_perm(w[0], w[2], 0x7632),
                           __byte_perm(w[1], w[3], 0x5410), __byte_perm(w[1], w[3], 0x7632));
                    const int per = 1 << (a.kv.group_shift - 3);
                    if ((i & (per - 1)) == per - 1) {
                        const int group = i / per;
                        const uint32_t high = pack<T>(sum, 0.0f) & 0xFFFFu;
                        const float held = two<T>(high).x;  // of what is not finite nothing is left
                        const uint32_t low = fabsf(held) < INFINITY ? pack<T>(sum - held, 0.0f) & 0xFFFFu : 0u;
                        asm volatile("st.shared.u16 [%0], %1;" ::"r"(sums_to + group * 2), "h"(static_cast<uint16_t>(high)));
                        asm volatile("st.shared.u16 [%0], %1;" ::"r"(sums_to + 128 + group * 2), "h"(static_cast<uint16_t>(low)));
                        sum = 0;
                    }
                }
                for (int group = a.kv.groups; group < 8; ++group) {
                    asm volatile("st.shared.u16 [%0], %1;" ::"r"(sums_to + group * 2), "h"(static_cast<uint16_t>(0)));
                    asm volatile("st.shared.u16 [%0], %1;" ::"r"(sums_to + 128 + group * 2), "h"(static_cast<uint16_t>(0)));
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(qfull + 8 * half);
            }
            // Positions of this half's rows.
            const int first_row = it.tile * 128 * Z::HALVES + half * 128, last_row = min(first_row + 127, share.rows - 1);
            const int nearest = min(seq.at + first_row / a.share, seq.keys - 1);
            const int behind = a.window ? seq.at + last_row / a.share - a.window : -1;
            const float k = fmaxf(fabsf(a.scale) * LOG2E * up, 1e-38f);  // of a scale of 0 still what -inf becomes -inf by
            const uint64_t kk = pair_of(k, k);
            float m = -INFINITY;
            uint64_t l = 0;
            for (int j = 0; j < steps; ++j) {
                const uint32_t g = steps_done + j;
                const uint32_t side = 2 * half + (g & 1), scores = scores_at + (g & 1) * Z::TOKENS;  // scores of odd and even steps
                if (!wait_on_warp(sfull + 8 * side, g >> 1 & 1, p.budget_ns, p.status, KERR_TIMEOUT_EPILOGUE)) {
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
                    hidden |= *reinterpret_cast<const uint32_t*>(there + g % Z::THERE * Z::BLOCKS) != 0x01010101u;
                }
                uint32_t s[Z::TOKENS];
                tmem_ld32(scores, *reinterpret_cast<uint32_t(*)[32]>(s));
                tmem_ld32(scores + 32, *reinterpret_cast<uint32_t(*)[32]>(s + 32));
                tmem_ld_wait();
                if (hidden) {
#pragma unroll
                    for (int e = 0; e < Z::BLOCKS; ++e) {
                        const int b = b0 + e, token = share.block_at(b) * KV_BLOCK;
                        const bool block = b < share.blocks && there[g % Z::THERE * Z::BLOCKS + e];
                        const int upto = block ? min(at, seq.keys - 1) : -1;
                        const int window = a.window ? at - a.window : -1;
#pragma unroll
                        for (int i = 0; i < KV_BLOCK; ++i) {
                            const int position = token + i;
                            if (!(position <= upto && (position > window || position < a.sinks))) s[e * KV_BLOCK + i] = __float_as_uint(-INFINITY);
                        }
                    }
                }
                float part[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < Z::TOKENS; ++i) part[i & 3] = fmaxf(part[i & 3], __uint_as_float(s[i]));
                const float top = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])) * k;
                const bool higher = top > m + 8.0f;
                if (__any_sync(0xffffffffu, higher)) {
                    const float next = higher ? top : m;
                    const float by = m == -INFINITY ? 0.0f : ex2(m - next);
                    m = next;
                    l = mul2(l, pair_of(by, by));
                    if (j) {  // the sums so far, once the product before this one is in them
                        if (!wait_on_warp(ofull + 8 * (side ^ 1), (g - 1) >> 1 & 1, p.budget_ns, p.status, KERR_TIMEOUT_EPILOGUE)) {
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
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        float x, y;
                        parts_of(fma2(pair_of(__uint_as_float(s[c + i]), __uint_as_float(s[c + i + 1])), kk, mm), x, y);
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
                if (lane == 0) mbar_arrive(pfull + 8 * side);
            }
            if (ok && steps &&
                !wait_on_warp(ofull + 8 * (2 * half + ((steps_done + steps - 1) & 1)), (steps_done + steps - 1) >> 1 & 1, p.budget_ns, p.status, KERR_TIMEOUT_EPILOGUE))
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
            steps_done += steps;
            if (!ok) break;
        }
    } else if (wg == 2 || wg == 3) {
        regs_down<REGS_DECODE>();
        uint32_t turn = 0;  // the parity of each of the ring's signals
        Item it;
        for (int n = 0; next_item(n, &it); ++n) {
            const Sequence seq(a.batch, it.seq);
            const Share share(seq, a, 128 * Z::HALVES, Z::BLOCKS, it.tile);
            const int steps = share.tiles;
            // The keys, or the values, of block w of each step, through a ring of this warp's own.
            const bool keys = wg == 2;
            const uint32_t raw = drain + 16 + (warp - 8) * 8 * Z::RING;  // signals of the ring's copies
            const int w = warp & 3, block_bytes = a.kv.block_bytes, part_bytes = block_bytes / 2, groups = a.kv.groups;
            const int to_group = a.kv.group_shift - 5;
            uint8_t* ring = rings + (warp - 8) * Z::RING * part_bytes;
            const uint8_t* pool = a.kv.pool + (keys ? 0 : part_bytes);
            auto index = [&](int i) { return i * Z::BLOCKS + w; };
            int places = -1;                 // where in the pool 32 of them lie, one to a lane; -1: nowhere
            uint32_t gone = 0, asked = 0;    // of the ring's: those that are nowhere; those under way
            auto load = [&](int i, int slot) {
                if (i >= steps) return;
                if ((i & 31) == 0) {
                    places = -1;
                    const int b = index(i + lane);
                    if (b < share.blocks) {
                        const int block = share.block_at(b), in_page = a.kv.page_shift - 4;
                        const int page = a.batch.table[it.seq * a.batch.table_rs + (block >> in_page)];
                        if (static_cast<uint32_t>(page) < a.kv.pages)
                            places = ((page * a.kv.heads + it.head) << in_page) + (block & ((1 << in_page) - 1));
                    }
                }
                const int place = __shfl_sync(0xffffffffu, places, i & 31);
                gone = place < 0 ? gone | 1u << slot : gone & ~(1u << slot);
                asked |= 1u << slot;
                if (lane == 0) {
                    mbar_expect_tx(raw + 8 * slot, place < 0 ? 0 : part_bytes);
                    if (place >= 0) bulk_load(smem_u32(ring + slot * part_bytes), pool + static_cast<int64_t>(place) * block_bytes, part_bytes, raw + 8 * slot);
                }
            };
            for (int i = 0; i < Z::RING; ++i) load(i, i);
            const int t = lane >> 2, c = lane & 3;
            const uint32_t full = keys ? kfull : vfull, empty = keys ? kempty : vempty, stages = keys ? Z::KSTAGES : Z::VSTAGES;
            uint32_t stage = steps_done % stages, filled = steps_done / stages & 1, g = steps_done;
            int slot = 0;
#pragma unroll 1
            for (int i = 0; i < steps; ++i) {
                if (!wait_on_warp(empty + 8 * stage, filled ^ 1, p.budget_ns, p.status, KERR_TIMEOUT_PRODUCER)) {
                    ok = false;
                    break;
                }
                if (!wait_on_warp(raw + 8 * slot, turn >> slot & 1, p.budget_ns, p.status, KERR_TIMEOUT_MMA_FULL)) {
                    ok = false;
                    break;
                }
                turn ^= 1u << slot;
                asked &= ~(1u << slot);
                uint8_t* part = ring + slot * part_bytes;
                const bool missing = gone >> slot & 1;
                const int token = missing ? seq.keys : share.block_at(index(i)) * KV_BLOCK;
                if (token + KV_BLOCK > seq.keys) {
                    // What lies behind the last token may be anything: by a scale and a middle of 0 it is 0.
                    for (int b = lane; b < 8 * groups; b += 32) {
                        auto* q = reinterpret_cast<uint32_t*>(part + 8 * D + b * 8);
                        const int first = token + b / groups * 2;
                        const uint32_t keep = (first < seq.keys ? 0xFFFFu : 0u) | (first + 1 < seq.keys ? 0xFFFF0000u : 0u);
                        q[0] &= keep, q[1] &= keep;
                    }
                    __syncwarp();
                }
                const int row = w * KV_BLOCK;
                if (keys) {
                    // Tokens t and 8 + t, channels 8 c .. 8 c + 7 of every 32.
                    if (lane == 0) there[g % Z::THERE * Z::BLOCKS + w] = !missing;
                    const uint32_t odd = (t & 1) ? 0x3232 : 0x1010;
#pragma unroll 1
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t to = smem_u32(keys_at) + stage * Z::K_BYTES + (row + h * 8 + t) * 128;
                        uint32_t v[N32];
                        uint32_t q[N32];
                        const uint8_t* params = part + 8 * D + (h * 4 + (t >> 1)) * groups * 8;
                        words<N32>(part + ((h * 8 + t) * 4 + c) * N32 * 4, v);
#pragma unroll
                        for (int n = 0; n < N32; ++n) q[n] = *reinterpret_cast<const uint32_t*>(params + (n >> to_group) * 8);
                        // the token's middles of groups 2 c and 2 c + 1, once for each part of the queries' sums
                        const uint32_t m0 = 2 * c < groups ? *reinterpret_cast<const uint32_t*>(params + 2 * c * 8 + 4) : 0u;
                        const uint32_t m1 = 2 * c + 1 < groups ? *reinterpret_cast<const uint32_t*>(params + (2 * c + 1) * 8 + 4) : 0u;
                        const uint32_t mids = __byte_perm(m0, m1, (t & 1) ? 0x7632 : 0x5410);
                        const uint32_t mids_to = smem_u32(keys_at) + stage * Z::K_BYTES + Z::K_MIDS + (2 * w + h) * 256 + t * 16 + c * 4;
                        asm volatile("st.shared.u32 [%0], %1;" ::"r"(mids_to), "r"(mids));
                        asm volatile("st.shared.u32 [%0], %1;" ::"r"(mids_to + 128), "r"(mids));
#pragma unroll
                        for (int n = 0; n < N32; ++n) {
                            const uint32_t scale = __byte_perm(q[n], 0, odd);
                            uint32_t x[4], left[4];
                            centred<T>(v[n], x);
#pragma unroll
                            for (int b = 0; b < 4; ++b) product<T>(scale, x[b], left[b]);
                            const uint32_t piece = to + (n >> 1) * Z::T_ATOM + ((((n & 1) * 4 + c) ^ t) << 4);
                            sts128(piece, x[0], x[1], x[2], x[3]);
                            sts128(piece + Z::T_BYTES, left[0], left[1], left[2], left[3]);
                        }
                    }
                } else {
                    // Two tokens, 8 h + 2 c and the next, by eight channels of every 32.
                    const int h = lane >> 4, eight = lane >> 2 & 3, tok = 8 * h + 2 * c;
                    const uint32_t to = smem_u32(values_at) + stage * Z::T_BYTES + (row + tok) * 128;
                    uint32_t v[2][N32];
                    uint2 q[N32];
                    words<N32>(part + ((h * 8 + 2 * eight) * 4 + c) * N32 * 4, v[0]);
                    words<N32>(part + ((h * 8 + 2 * eight + 1) * 4 + c) * N32 * 4, v[1]);
#pragma unroll
                    for (int n = 0; n < N32; ++n) q[n] = *reinterpret_cast<const uint2*>(part + 8 * D + ((tok >> 1) * groups + (n >> to_group)) * 8);
#pragma unroll
                    for (int n = 0; n < N32; ++n) {
                        uint32_t x[2][4];
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            centred<T>(v[b][n], x[b]);
#pragma unroll
                            for (int k = 0; k < 4; ++k) x[b][k] = fma_half2<T>(q[n].x, x[b][k], q[n].y);
                        }
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const uint32_t half = k ? 0x7632 : 0x5410;
                            sts128(to + (n >> 1) * Z::T_ATOM + k * 128 + ((((n & 1) * 4 + eight) ^ ((2 * c + k) & 7)) << 4), __byte_perm(x[0][0], x[0][1], half),
                                   __byte_perm(x[0][2], x[0][3], half), __byte_perm(x[1][0], x[1][1], half), __byte_perm(x[1][2], x[1][3], half));
                        }
                    }
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(full + 8 * stage);
                if (++stage == stages) stage = 0, filled ^= 1;
                ++g;
                load(i + Z::RING, slot);
                if (++slot == Z::RING) slot = 0;
            }
            if (!ok)  // copies under way end before the memory goes
                for (int i = 0; i < Z::RING; ++i)
                    if (asked >> i & 1) wait_out(raw + 8 * i, turn >> i & 1, p.budget_ns);
            steps_done += steps;
            if (!ok) break;
            wants_next();
        }
    } else {
        regs_down<REGS_CONTROL>();
        if (warp >= 20 - Z::HALVES) {
            // A thread for each half's products: one for both spent more time on its waits than they took.
            const int half = warp - (20 - Z::HALVES);
            if (elect_one()) {
                Item it;
                constexpr uint32_t QK = idesc_f16(128, Z::TOKENS, BF16), PV = idesc_f16(128, D, BF16, true);
                const uint64_t q_at = smem_desc_sw128(smem_u32(smem), 16, 1024), k_at = smem_desc_sw128(smem_u32(keys_at), 16, 1024);
                const uint64_t qs_at = smem_desc_plain(smem_u32(smem) + Z::Q_SUMS, 128, 256), ks_at = smem_desc_plain(smem_u32(keys_at) + Z::K_MIDS, 128, 256);
                const uint64_t v_at = smem_desc_sw128(smem_u32(values_at), Z::T_ATOM, 1024);
                auto scores = [&](uint32_t g) {
                    const uint32_t side = 2 * half + (g & 1), ks = g % Z::KSTAGES;
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        const uint64_t k0 = k_at + (ks * Z::K_BYTES + i / 4 * Z::T_ATOM + i % 4 * 32) / 16;
                        mma_f16_twice(tmem + Z::S_AT + side * Z::TOKENS, q_at + ((half * Z::Q_HALF + i / 4 * Z::Q_ATOM + i % 4 * 32) >> 4), k0,
                                      k0 + Z::T_BYTES / 16, QK, i != 0);
                    }
                    mma_f16(tmem + Z::S_AT + side * Z::TOKENS, qs_at + (half * Z::Q_HALF >> 4), ks_at + ks * Z::K_BYTES / 16, QK, true);
                    mma_commit(sfull + 8 * side);
                };
                auto values = [&](uint32_t g, bool first) {  // sums (+)= weights values
                    const uint32_t side = 2 * half + (g & 1), vs = g % Z::VSTAGES;
#pragma unroll
                    for (int i = 0; i < Z::TOKENS / 16; ++i)
                        mma_f16_ts(tmem + Z::O_AT + half * D, tmem + Z::S_AT + side * Z::TOKENS + i * 8, v_at + (vs * Z::T_BYTES + i * 2048) / 16, PV,
                                   i != 0 || !first);
                    mma_commit(ofull + 8 * side);
                };
                for (int n = 0; item_at(n, &it); ++n) {
                    mbar_arrive(iempty);
                    const Sequence seq(a.batch, it.seq);
                    const int steps = Share(seq, a, 128 * Z::HALVES, Z::BLOCKS, it.tile).tiles;
                    ok = wait_on(qfull + 8 * half, n & 1, p.budget_ns, p.status, KERR_TIMEOUT_MMA_FULL);
                    // Scores are a step ahead of the weights: while a half's weights of one step are made, the
                    // next step's scores are at hand.
                    for (int j = -1; j <= steps && ok && steps; ++j) {
                        const uint32_t g = steps_done + j;  // scores of step j + 1 after values of step j - 1
                        if (j >= 1) {
                            const uint32_t vs = (g - 1) % Z::VSTAGES;
                            ok = wait_on(vfull + 8 * vs, (g - 1) / Z::VSTAGES & 1, p.budget_ns, p.status, KERR_TIMEOUT_MMA_FULL) &&
                                 wait_on(pfull + 8 * (2 * half + ((g - 1) & 1)), (g - 1) >> 1 & 1, p.budget_ns, p.status, KERR_TIMEOUT_MMA_ACC);
                            if (!ok) break;
                            tc_fence_after();
                            values(g - 1, j == 1);
                            mma_commit(vempty + 8 * vs);
                        }
                        if (j + 1 < steps) {
                            const uint32_t ks = (g + 1) % Z::KSTAGES;
                            ok = wait_on(kfull + 8 * ks, (g + 1) / Z::KSTAGES & 1, p.budget_ns, p.status, KERR_TIMEOUT_MMA_FULL);
                            if (!ok) break;
                            tc_fence_after();
                            scores(g + 1);
                            mma_commit(kempty + 8 * ks);
                        }
                    }
                    steps_done += steps;
                }
                if (!ok) {  // what was issued ends before the memory goes
                    mma_commit(drain + 8 * half);
                    wait_out(drain + 8 * half, 0, p.budget_ns);
                }
            }
        } else if (warp == 16 && elect_one()) {
            // Behind the last item is one that says so.
            for (int n = 0; !n || wait_on(iempty, n & 1 ^ 1, p.budget_ns, p.status, KERR_TIMEOUT_PRODUCER); ++n) {
                const bool more = take(n & 1);
                mbar_arrive(ifull + 8 * (n & 1));
                if (!more) break;
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 17) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <typename T, int D, int H>
int launch_many(uor_b200_ctx* ctx, const AttendArgs& a, uor_b200_route* route) {
    using Z = Shape<D, H>;
    auto* kernel = many_kernel<T, D, H>;
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
    p.next = reinterpret_cast<unsigned long long*>(before + a.batch.seqs + 1);
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

template <typename T, int D>
int by_halves(uor_b200_ctx* ctx, const AttendArgs& a, uor_b200_route* route) {
    const int64_t mean = (static_cast<int64_t>(a.batch.rows) * a.share + a.batch.seqs - 1) / a.batch.seqs;
    // Tiles of 128 rows where there are processors enough for them all: 1.6 us a step for one half, 1.85 for
    // two (512 new tokens of 4096, 4 queries to each of 8 heads: 108 : 126 us, 1024: 184 : 128).
    return a.batch.seqs * a.kv.heads * ((mean + 127) / 128) <= ctx->sm_count ? launch_many<T, D, 1>(ctx, a, route)
                                                                             : launch_many<T, D, 2>(ctx, a, route);
}

}  // namespace

template <typename T>
int kv4_many(uor_b200_ctx* ctx, const AttendArgs& a, uor_b200_route* route) {
    switch (a.kv.dim) {
    case 64: return by_halves<T, 64>(ctx, a, route);
    case 96: return by_halves<T, 96>(ctx, a, route);
    case 128: return by_halves<T, 128>(ctx, a, route);
    case 192: return launch_many<T, 192, 1>(ctx, a, route);
    default: return launch_many<T, 256, 1>(ctx, a, route);
    }
}

}  // namespace uor
