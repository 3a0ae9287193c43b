// q4_many.cu -- products of many rows with 4-bit weights and group scales.
//
// Bound by the tensor cores: 2 m n k operations on 16-bit floats. A work item is a tile of 256
// weight rows by up to 256 activation rows, on a pair of CTAs (tcgen05.mma.cta_group::2): each
// CTA holds 128 of the weight rows and brings half of the activation rows. The weights are the
// instruction's M side, so that a thread of the epilogue owns one weight row and a group's scale
// is one number per thread.
//
// The roles of a CTA: a warp brings 128-position stages of activations by TMA, another the codes;
// a warpgroup turns each code into a 16-bit float, exactly (code - zero), and stores it to tensor
// memory, where the instruction takes its A side from; one thread of the pair issues the
// tcgen05.mma, for one half of the tile's columns and then the other; a warpgroup for each half
// holds its sums. A group's products are summed in tensor memory, and at the group's end the
// warpgroup adds scale x sum to its f32 registers, while the instructions run on in the two
// other accumulators. So no weight is rounded: rounding scale x code to 16 bits would cost as
// much precision as rounding the output does.
//
// Why this shape. With the weights in shared memory and one CTA per 128 x 256 tile, the operands'
// reads, the TMA's and the decoders' writes came to 104 KB per 64 positions, 830 cycles at 128
// bytes a cycle, for 512 cycles of multiplication (2048 x 8192 x 8192: 366 us, 295 us without
// decoding and scaling); here they are 40 KB. Beside that it is issue slots that count: decoding
// takes 13 instructions per eight codes and a sum half a one per column, waits and bookkeeping as
// much again, so a tile has as many columns as the sums' registers allow (192 of them, with
// two decoding warpgroups: 287 us), there is one commit per 128 positions and half, waits sleep,
// and no arrival carries a release at cluster scope, which held its warp for 2000 cycles.
// Tensor memory's 512 columns hold three accumulators of 128 and two stages of weights of 64.
//
// 2048 x 8192 x 8192: 264 us, 1040 TFLOP/s (289 us back to back for a second, at the power cap's
// clocks). A stage of 128 positions takes 0.89 us, its multiplication 1024 cycles, 0.52; a tile's way
// out and start 9.4 us, in which the three accumulators fill and the tensor cores stop.
//
// Every wait is bounded; a role that gives up records it, and every other role leaves after it.
#include "q4_many.cuh"

#include <cstring>
#include <type_traits>

#include "ptx.cuh"

namespace uor {

namespace {

constexpr int BM = 128;        // weight rows of a CTA's half of a tile
constexpr int BK = 128;        // reduction positions of a stage
constexpr int ATOM = 64;       // positions in the 128 bytes that the activations' swizzle spans
constexpr int MAX_COLS = 256;  // activation rows of a tile
constexpr int HALF = 128;      // columns of an accumulator: half a tile's
constexpr int X_BOX = 32;      // activation rows of one TMA copy
constexpr int X_BOX_BYTES = X_BOX * ATOM * 2;
constexpr int HALF_BYTES = HALF / 2 * ATOM * 2;      // a CTA's rows of a half, per atom
constexpr int ATOM_BYTES = 2 * HALF_BYTES;
constexpr int X_BYTES = ATOM_BYTES * BK / ATOM;
constexpr int C_BYTES = BM * BK / 2;
constexpr int STAGES = 4, CSTAGES = 4, ASTAGES = 2, ACCS = 3;
constexpr int A_COLS = BK / 2;                       // tensor-memory columns of a stage of weights
constexpr int A_FIRST = ACCS * HALF;
constexpr int DECODERS = 4, SUMMERS = 4;             // warps of a CTA; of a CTA and a half
constexpr int OUT_COLS = 32;                         // columns that leave at a time
constexpr int EXCHANGE = BM * OUT_COLS * 4 + HALF * 4;  // bytes, per half: sums, and their rows' pairs
// Signals of filled accumulators, per half: as many as can be filled before the first is read, and
// one, since a warpgroup waits for its own half's alone and must not mistake a later filling.
constexpr int FULLS = ACCS + 1;
constexpr int BARS = 2 * STAGES + 2 * CSTAGES + ASTAGES + 2 * FULLS + ACCS + 1;
constexpr int SMEM = STAGES * X_BYTES + CSTAGES * C_BYTES + 2 * EXCHANGE + (BARS + 1) * 8 + (MANY_MAX_EXPERTS + 1) * 4 + 1024;
constexpr uint32_t NAP_NS = 1000;  // a wait's sleep between looks; an arrival ends it at once
// Warpgroup 0: TMA, MMA; 1: decoders; 2 and 3: sums. Registers: 128 a thread at launch.
constexpr int THREADS = 512;
constexpr int REGS_CONTROL = 32, REGS_DECODE = 80, REGS_SUM = 200;
static_assert(SMEM <= 232448, "shared memory of a block");
static_assert(A_FIRST + ASTAGES * A_COLS <= 512, "tensor memory");
static_assert(REGS_CONTROL + REGS_DECODE + 2 * REGS_SUM <= 4 * 128, "registers of the launch");

struct Item {
    int cols, half;           // existing activation rows; an instruction's columns
    int halves;               // instructions' columns in the tile: one or two
    int64_t p0;               // first activation row
    int64_t row0;             // first weight row
    int j0;                   // first output
    int kb0, kbs;             // stages of the reduction
    int split;
};

__device__ __forceinline__ int tiles_of(int count, int max_cols) { return (count + max_cols - 1) / max_cols; }

// Item u: row tiles run fastest, then the experts' tiles of activations, then the splits.
__device__ __forceinline__ bool item_at(int u, const ManyParams& p, const int* first_tile, int rank, Item* it) {
    const int rt = u % p.row_tiles;
    const int rest = u / p.row_tiles;
    const int tiles = first_tile[p.experts];
    const int tt = rest % tiles;
    it->split = rest / tiles;
    int lo = 0, hi = p.experts;  // the expert with first_tile[lo] <= tt < first_tile[lo + 1]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first_tile[mid] <= tt) lo = mid;
        else hi = mid;
    }
    const int begin = p.offsets ? p.offsets[lo] : 0;
    const int count = p.offsets ? p.offsets[lo + 1] - begin : p.m;
    const int parts = tiles_of(count, p.max_cols);
    const int size = ((count + parts - 1) / parts + 63) & ~63;  // even shares, in whole instructions
    const int i = tt - first_tile[lo];
    it->cols = min(size, count - i * size);
    it->halves = it->cols > 32 ? 2 : 1;
    it->half = it->halves == 2 ? (it->cols + 63) / 64 * 32 : 32;
    it->p0 = begin + static_cast<int64_t>(i) * size;
    const int outputs = p.mode == MANY_UP ? BM / 2 : BM;  // of a CTA
    it->j0 = (2 * rt + rank) * outputs;
    it->row0 = static_cast<int64_t>(lo) * (p.mode == MANY_UP ? 2 * p.n : p.n) + it->j0;
    it->kb0 = it->split * p.kb_per_split;
    it->kbs = min(p.kb_per_split, (p.w.cols + BK - 1) / BK - it->kb0);
    return it->cols > 0 && it->kbs > 0;
}

// Eight codes of a word, in order, less their zero point, in CodeUnits, as 16-bit floats.
template <typename T>
__device__ __forceinline__ uint4 decode8(uint32_t w, uint32_t zero) {
    constexpr uint32_t HIGH = std::is_same<T, __half>::value ? 0x64u : 0x3Du;  // 1024, or 128 of 2^-12
    const uint32_t lo = w & 0x0F0F0F0Fu, hi = (w >> 4) & 0x0F0F0F0Fu;
    const uint32_t a = __byte_perm(lo, hi, 0x5140), b = __byte_perm(lo, hi, 0x7362);
    auto less = [&](uint32_t v) {
        if constexpr (std::is_same<T, __half>::value) {
            __half2 x, z;
            memcpy(&x, &v, 4);
            memcpy(&z, &zero, 4);
            x = __hsub2(x, z);
            memcpy(&v, &x, 4);
        } else {
            __nv_bfloat162 x, z;
            memcpy(&x, &v, 4);
            memcpy(&z, &zero, 4);
            x = __hsub2(x, z);
            memcpy(&v, &x, 4);
        }
        return v;
    };
    return make_uint4(less(__byte_perm(a, HIGH, 0x4140)), less(__byte_perm(a, HIGH, 0x4342)),
                      less(__byte_perm(b, HIGH, 0x4140)), less(__byte_perm(b, HIGH, 0x4342)));
}
template <typename T>
__device__ __forceinline__ uint32_t zero_pair(uint32_t z) {
    return (std::is_same<T, __half>::value ? 0x64006400u : 0x3D003D00u) | (z << 16) | z;
}

// Steps along a row's scales (or zero points) by a piece of a group at a time.
struct GroupWalk {
    int at, pos;
    __device__ __forceinline__ GroupWalk(int k, const ManyParams& p) : at(k / p.w.group), pos(k - k / p.w.group * p.w.group) {}
    __device__ __forceinline__ int index(const ManyParams& p) const { return min(at, p.groups - 1); }
    __device__ __forceinline__ void step(int by, const ManyParams& p) {
        pos += by;
        while (pos >= p.w.group) pos -= p.w.group, ++at;
    }
};

// acc += v * s on two floats at once.
__device__ __forceinline__ void fma2(uint64_t& acc, uint32_t lo, uint32_t hi, uint64_t s) {
    asm("{\n .reg .b64 v;\n mov.b64 v, {%1, %2};\n fma.rn.f32x2 %0, v, %3, %0;\n}\n" : "+l"(acc) : "r"(lo), "r"(hi), "l"(s));
}
__device__ __forceinline__ float half_of(uint64_t v, int i) {
    return __uint_as_float(static_cast<uint32_t>(i ? v >> 32 : v));
}

// The sums of `cols` activation rows from row i0 on, [column][row] in shared memory, to where
// this launch's outputs go (pairs: the ones behind them); 128 threads, `r` this one. Each stores eight neighbouring outputs of a
// column (four with gates and ups), as one vector where they lie so.
template <typename T>
__device__ __noinline__ void sums_out(const ManyParams& p, const Item& it, const float* swap, const int* pairs, int64_t i0, int cols,
                                      int r) {
    if (p.mode == MANY_UP) {
        // Rows 0 .. 63 are gates, 64 .. 127 the same outputs' ups.
        const int j = (r & 15) * 4, valid = min(4, p.n - it.j0 - j);
        T* to = static_cast<T*>(p.h) + i0 * p.h_rs + it.j0 + j;
        for (int c = r >> 4; c < cols && valid > 0; c += 8) {
            const float4 g = *reinterpret_cast<const float4*>(swap + c * BM + j);
            const float4 u = *reinterpret_cast<const float4*>(swap + c * BM + j + 64);
            const T v[4] = {from_f32<T>(silu(g.x) * u.x), from_f32<T>(silu(g.y) * u.y), from_f32<T>(silu(g.z) * u.z),
                            from_f32<T>(silu(g.w) * u.w)};
            if (valid == 4) {  // rows of h begin at multiples of 16 bytes
                uint2 bits;
                memcpy(&bits, v, 8);
                *reinterpret_cast<uint2*>(to + c * p.h_rs) = bits;
            } else {
                for (int k = 0; k < valid; ++k) to[c * p.h_rs + k] = k == 0 ? v[0] : k == 1 ? v[1] : v[2];
            }
        }
        return;
    }
    const int j = (r & 15) * 8, valid = min(8, p.n - it.j0 - j);
    const bool parts = p.mode == MANY_DOWN || p.splits > 1;
    const int type = parts ? UOR_B200_F32 : p.y.type;
    const int64_t rs = parts ? p.n : p.y.rs, step = parts ? 1 : p.y.cs;
    void* to = parts ? p.part + it.split * p.part_rows * p.n : p.y.p;
    for (int c = r >> 4; c < cols && valid > 0; c += 8) {
        const float4 a = *reinterpret_cast<const float4*>(swap + c * BM + j);
        const float4 b = *reinterpret_cast<const float4*>(swap + c * BM + j + 4);
        const int64_t i = p.mode == MANY_DOWN ? pairs[c] : i0 + c;
        const int64_t at = i * rs + (it.j0 + j) * step;
        char* first = static_cast<char*>(to) + at * (type == UOR_B200_F32 ? 4 : 2);
        if (valid == 8 && step == 1 && reinterpret_cast<uint64_t>(first) % 16 == 0) {
            if (type == UOR_B200_F32) {
                reinterpret_cast<float4*>(first)[0] = a;
                reinterpret_cast<float4*>(first)[1] = b;
            } else {
                uint4 w;
                if (type == UOR_B200_BF16) {
                    const __nv_bfloat162 t[4] = {__floats2bfloat162_rn(a.x, a.y), __floats2bfloat162_rn(a.z, a.w),
                                                 __floats2bfloat162_rn(b.x, b.y), __floats2bfloat162_rn(b.z, b.w)};
                    memcpy(&w, t, 16);
                } else {
                    const __half2 t[4] = {__floats2half2_rn(a.x, a.y), __floats2half2_rn(a.z, a.w), __floats2half2_rn(b.x, b.y),
                                          __floats2half2_rn(b.z, b.w)};
                    memcpy(&w, t, 16);
                }
                *reinterpret_cast<uint4*>(first) = w;
            }
        } else {
            for (int k = 0; k < valid; ++k) store_f32(to, at + k * step, type, swap[c * BM + j + k]);
        }
    }
}

template <int N>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

template <typename T, int SEG>
__global__ void __launch_bounds__(THREADS, 1)
    many_kernel(const __grid_constant__ CUtensorMap tm_codes, const __grid_constant__ CUtensorMap tm_x,
                const __grid_constant__ ManyParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* codes_at = smem + STAGES * X_BYTES;
    float* exchange = reinterpret_cast<float*>(codes_at + CSTAGES * C_BYTES);
    uint64_t* bars = reinterpret_cast<uint64_t*>(exchange + 2 * (EXCHANGE / 4));
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + BARS);
    int* first_tile = reinterpret_cast<int*>(bars + BARS + 1);
    // xfull, afull and tempty count on the leader, for both CTAs. done: a stage's products are
    // complete, which frees its activations and its weights. tfull: a group's are, of one half.
    const uint32_t xfull = smem_u32(bars), done = xfull + 8 * STAGES;
    const uint32_t cfull = done + 8 * STAGES, cempty = cfull + 8 * CSTAGES;
    const uint32_t afull = cempty + 8 * CSTAGES;
    const uint32_t tfull = afull + 8 * ASTAGES, tempty = tfull + 8 * 2 * FULLS, drain = tempty + 8 * ACCS;
    constexpr int GROUPS = BK / SEG;  // of a stage
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wg = warp >> 2;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const int pair = static_cast<int>(cluster_id_x()), pairs = static_cast<int>(nclusters_x());

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(xfull + 8 * s, 1);
            mbar_init(done + 8 * s, 1);
        }
        for (int s = 0; s < CSTAGES; ++s) {
            mbar_init(cfull + 8 * s, 1);
            mbar_init(cempty + 8 * s, DECODERS);
        }
        for (int s = 0; s < ASTAGES; ++s) mbar_init(afull + 8 * s, 2 * DECODERS);
        for (int b = 0; b < 2 * FULLS; ++b) mbar_init(tfull + 8 * b, 1);
        for (int b = 0; b < ACCS; ++b) mbar_init(tempty + 8 * b, 2 * SUMMERS);
        mbar_init(drain, 1);
        fence_barrier_init();
        tma_prefetch_desc(&tm_codes);
        tma_prefetch_desc(&tm_x);
    }
    if (warp == 3) tmem_alloc_pair(smem_u32(tmem_slot), 512);
    // So far nothing of the kernel before this one was read; every thread waits for it now.
    // With experts the next kernel begins as this one's blocks leave (8 of 2048 x 1024: 42.5 -> 41.8
    // us); before the adding of parts that costs (1024 x 2048, 17 rows: 14.1 -> 15.0).
    if (p.mode != MANY_DENSE) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (warp == 4) {  // tiles of activations before each expert's
        int before = 0;
        for (int e0 = 0; e0 <= p.experts; e0 += 32) {
            const int e = e0 + lane;
            int t = 0;
            if (e < p.experts) t = tiles_of(p.offsets ? p.offsets[e + 1] - p.offsets[e] : p.m, p.max_cols);
            int sum = t;
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += v;
            }
            if (e <= p.experts) first_tile[e] = before + sum - t;
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // both CTAs' barriers exist before either signals the other
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int items = p.row_tiles * first_tile[p.experts] * p.splits;
    Item it;

    if (wg == 0) {
        regs_down<REGS_CONTROL>();
        if (warp == 0) {  // activations: this CTA's half of the tile's
            if (elect_one()) {
                const uint64_t policy = l2_policy_evict_last();
                uint32_t n = 0, armed = 0, armed_phase = 0;  // n: stages so far
                bool ok = true;
                for (int u = pair; u < items && ok; u += pairs) {
                    if (!item_at(u, p, first_tile, rank, &it)) continue;
                    const int boxes = (it.half / 2 + X_BOX - 1) / X_BOX;  // of a half
                    const int row = static_cast<int>(it.p0) + static_cast<int>(rank) * (it.half / 2);
                    for (int kb = 0; kb < it.kbs; ++kb, ++n) {
                        const uint32_t s = n % STAGES, phase = n / STAGES & 1;
                        if (!mbar_wait_hint(done + 8 * s, phase ^ 1, p.budget_ns, p.status, KERR_TIMEOUT_PRODUCER, NAP_NS)) {
                            ok = false;
                            break;
                        }
                        if (leader) {
                            mbar_expect_tx(xfull + 8 * s, 2 * (BK / ATOM) * it.halves * boxes * X_BOX_BYTES);
                            armed |= 1u << s;
                            armed_phase = (armed_phase & ~(1u << s)) | phase << s;
                        }
                        const uint32_t full = mapa_shared(xfull + 8 * s, 0);
                        const uint32_t dst = smem_u32(smem + s * X_BYTES);
                        for (int a = 0; a < BK / ATOM; ++a)
                            for (int h = 0; h < it.halves; ++h)
                                for (int b = 0; b < boxes; ++b)
                                    tma_load_2d_pair(dst + a * ATOM_BYTES + h * HALF_BYTES + b * X_BOX_BYTES, &tm_x, full,
                                                     (it.kb0 + kb) * BK + a * ATOM, row + h * it.half + b * X_BOX, policy);
                    }
                }
                if (!ok && leader)
                    for (int i = 0; i < STAGES; ++i)
                        if (armed >> i & 1)
                            mbar_wait(xfull + 8 * i, armed_phase >> i & 1, p.budget_ns, p.status, KERR_TIMEOUT_DRAIN);
            }
            __syncwarp();
        } else if (warp == 2) {  // codes
            if (elect_one()) {
                const uint64_t policy = l2_policy_evict_last();
                int s = 0;
                uint32_t phase = 0, armed = 0, armed_phase = 0;
                bool ok = true;
                for (int u = pair; u < items && ok; u += pairs) {
                    if (!item_at(u, p, first_tile, rank, &it)) continue;
                    const int second = static_cast<int>(it.row0) + (p.mode == MANY_UP ? p.n : 64);
                    for (int kb = 0; kb < it.kbs; ++kb) {
                        if (!mbar_wait_hint(cempty + 8 * s, phase ^ 1, p.budget_ns, p.status, KERR_TIMEOUT_PRODUCER, NAP_NS)) {
                            ok = false;
                            break;
                        }
                        mbar_expect_tx(cfull + 8 * s, C_BYTES);
                        armed |= 1u << s;
                        armed_phase = (armed_phase & ~(1u << s)) | phase << s;
                        const uint32_t dst = smem_u32(codes_at + s * C_BYTES);
                        const int byte = (it.kb0 + kb) * (BK / 2);
                        tma_load_2d(dst, &tm_codes, cfull + 8 * s, byte, static_cast<int>(it.row0), policy);
                        tma_load_2d(dst + C_BYTES / 2, &tm_codes, cfull + 8 * s, byte, second, policy);
                        if (++s == CSTAGES) s = 0, phase ^= 1;
                    }
                }
                if (!ok)
                    for (int i = 0; i < CSTAGES; ++i)
                        if (armed >> i & 1)
                            mbar_wait(cfull + 8 * i, armed_phase >> i & 1, p.budget_ns, p.status, KERR_TIMEOUT_DRAIN);
            }
            __syncwarp();
        } else if (warp == 1 && leader) {  // the tensor cores of both CTAs
            if (elect_one()) {
                uint32_t n = 0, b = 0, turn = 0;  // stages so far; the next accumulator, its round's parity
                uint32_t filled[2] = {0, 0};      // accumulators of each half so far
                bool ok = true;
                for (int u = pair; u < items && ok; u += pairs) {
                    if (!item_at(u, p, first_tile, rank, &it)) continue;
                    const uint32_t idesc = idesc_f16(2 * BM, it.half, std::is_same<T, __nv_bfloat16>::value);
                    for (int kb = 0; kb < it.kbs && ok; ++kb, ++n) {
                        const uint32_t s = n % STAGES, a = n % ASTAGES;
                        ok = mbar_wait(xfull + 8 * s, n / STAGES & 1, p.budget_ns, p.status, KERR_TIMEOUT_MMA_FULL) &&
                             mbar_wait(afull + 8 * a, n / ASTAGES & 1, p.budget_ns, p.status, KERR_TIMEOUT_MMA_FULL);
                        const uint32_t sx = smem_u32(smem + s * X_BYTES), sa = tmem + A_FIRST + a * A_COLS;
#pragma unroll
                        for (int g = 0; g < GROUPS; ++g) {
                            if (g && (it.kb0 + kb) * BK + g * SEG >= p.w.cols) break;
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                if (h >= it.halves || !ok) break;
                                ok = mbar_wait(tempty + 8 * b, turn ^ 1, p.budget_ns, p.status, KERR_TIMEOUT_MMA_ACC);
                                if (!ok) break;
                                tc_fence_after();
#pragma unroll
                                for (int i = 0; i < SEG / 16; ++i) {
                                    const int k16 = g * (SEG / 16) + i;
                                    mma_f16_pair_ts(tmem + b * HALF, sa + k16 * 8,
                                                    smem_desc_sw128(sx + k16 / 4 * ATOM_BYTES + h * HALF_BYTES + k16 % 4 * 32, 16, 1024),
                                                    idesc, i != 0);
                                }
                                mma_commit_pair(tfull + 8 * (h * FULLS + filled[h]++ % FULLS), 0x3);
                                if (++b == ACCS) b = 0, turn ^= 1;
                            }
                        }
                        if (ok) mma_commit_pair(done + 8 * s, 0x3);
                    }
                }
                if (!ok && (n || b || turn)) {
                    mma_commit_pair(drain, 0x1);
                    mbar_wait(drain, 0, p.budget_ns, p.status, KERR_TIMEOUT_DRAIN);
                }
            }
            __syncwarp();
        }
    } else if (wg == 1) {
        regs_down<REGS_DECODE>();
        // A thread turns its row's codes into the operand's row, lane r of tensor memory.
        const int r = threadIdx.x & 127;
        const uint32_t to = tmem + (static_cast<uint32_t>(r & ~31) << 16) + A_FIRST;
        const int turn = ((r >> 1) & 3) << 4;  // the 64-byte swizzle's
        const uint8_t* from = codes_at + r * (BK / 2);
        int q = 0;
        uint32_t qphase = 0, n = 0;  // n: stages so far
        bool ok = true;
        for (int u = pair; u < items && ok; u += pairs) {
            if (!item_at(u, p, first_tile, rank, &it)) continue;
            const int64_t row = min(it.row0 + (r < 64 ? r : r - 64 + (p.mode == MANY_UP ? p.n : 64)), static_cast<int64_t>(p.w.rows) - 1);
            const uint8_t* zeros = p.w.zeros ? p.w.zeros + row * p.w.groups_rs : nullptr;
            constexpr int PIECES = BK / SEG;  // zero points of a stage
            uint32_t next[PIECES];
#pragma unroll
            for (int i = 0; i < PIECES; ++i) next[i] = 8;
            GroupWalk walk(it.kb0 * BK, p);
            auto fetch = [&]() {
                if (!zeros) return;
#pragma unroll
                for (int i = 0; i < PIECES; ++i) {
                    next[i] = zeros[walk.index(p)];
                    walk.step(SEG, p);
                }
            };
            fetch();
            for (int kb = 0; kb < it.kbs; ++kb, ++n) {
                if (!mbar_wait_warp_hint(cfull + 8 * q, qphase, p.budget_ns, p.status, KERR_TIMEOUT_MMA_FULL, NAP_NS)) {
                    ok = false;
                    break;
                }
                uint4 c[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) c[i] = *reinterpret_cast<const uint4*>(from + q * C_BYTES + ((i << 4) ^ turn));
                uint32_t z[PIECES];
#pragma unroll
                for (int i = 0; i < PIECES; ++i) z[i] = zero_pair<T>(next[i] & 15u);
                fetch();
                // the stage that used this one's columns is ASTAGES back
                const uint32_t a = n % ASTAGES, before = n - ASTAGES;
                if (n >= ASTAGES && !mbar_wait_warp_hint(done + 8 * (before % STAGES), before / STAGES & 1, p.budget_ns, p.status,
                                                         KERR_TIMEOUT_PRODUCER, NAP_NS)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t w[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
                    uint32_t v[16];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint4 d = decode8<T>(w[k], z[i * 32 / SEG]);
                        v[4 * k] = d.x, v[4 * k + 1] = d.y, v[4 * k + 2] = d.z, v[4 * k + 3] = d.w;
                    }
                    tmem_st16(to + a * A_COLS + i * 16, v);
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                // The codes are given back only now that they have been used. Given back behind their
                // reads alone, which a global access that misses can hold up for microseconds, the next
                // copy overtook those: its first rows stood in for this stage's, some passes in a
                // hundred over weights just laid out.
                if (lane == 0) {
                    mbar_arrive(cempty + 8 * q);
                    mbar_arrive_pair(mapa_shared(afull + 8 * a, 0));
                }
                if (++q == CSTAGES) q = 0, qphase ^= 1;
            }
        }
    } else {
        regs_up<REGS_SUM>();
        const int r = threadIdx.x & 127, part = wg - 2;  // part: which half of a tile's columns
        const uint32_t lanes = tmem + (static_cast<uint32_t>(r & ~31) << 16);
        const bool wide = p.w.scale_type == UOR_B200_F32, bf16 = p.w.scale_type == UOR_B200_BF16;
        const int per_group = p.w.group / SEG;
        uint32_t g = 0, filled = 0;  // accumulators filled before this item's; of this half so far
        bool ok = true;
        for (int u = pair; u < items && ok; u += pairs) {
            if (!item_at(u, p, first_tile, rank, &it)) continue;
            const int64_t row = min(it.row0 + (r < 64 ? r : r - 64 + (p.mode == MANY_UP ? p.n : 64)), static_cast<int64_t>(p.w.rows) - 1);
            const int k0 = it.kb0 * BK, first = k0 / p.w.group;
            const int steps = (min(p.w.cols - k0, it.kbs * BK) + SEG - 1) / SEG;
            int repeat = per_group - (k0 - first * p.w.group) / SEG;  // steps with the scale at hand
            const char* scale_at = static_cast<const char*>(p.w.scales) + (row * p.w.groups_rs + first) * (wide ? 4 : 2);
            auto load = [&]() -> uint32_t {
                return wide ? *reinterpret_cast<const uint32_t*>(scale_at) : *reinterpret_cast<const uint16_t*>(scale_at);
            };
            auto value = [&](uint32_t raw) {
                return wide ? raw
                       : bf16 ? raw << 16
                              : __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(raw))));
            };
            uint64_t acc[HALF / 2];
#pragma unroll
            for (int i = 0; i < HALF / 2; ++i) acc[i] = 0;
            const int mine = part < it.halves ? it.half : 0;  // this warpgroup's columns
            // asked for long before it is needed: the pair behind this half's column r
            const int row_pair = p.mode == MANY_DOWN && r < mine && part * it.half + r < it.cols ? p.perm[it.p0 + part * it.half + r] : 0;
            uint32_t next = load();
            // Accumulators are filled in turn, those of both halves: this one's are every
            // `halves`-th from its own first on.
            uint32_t at = g + part;
            for (int i = 0; i < steps && mine; ++i, at += it.halves, ++filled) {
                const uint32_t sb = value(next), b = at % ACCS;
                const uint64_t scale = static_cast<uint64_t>(sb) << 32 | sb;
                if (--repeat == 0 && i + 1 < steps) {
                    repeat = per_group;
                    scale_at += wide ? 4 : 2;
                    next = load();
                }
                if (!mbar_wait_warp_hint(tfull + 8 * (part * FULLS + filled % FULLS), filled / FULLS & 1, p.budget_ns, p.status, KERR_TIMEOUT_EPILOGUE, NAP_NS)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                // Columns travel 48 at a time: a read takes some 250 cycles, however many are under way.
                __syncwarp();
#pragma unroll
                for (int h = 0; h < HALF; h += 48) {
                    uint32_t v[3][16];
#pragma unroll
                    for (int c = 0; c < 3; ++c)
                        if (h + c * 16 < HALF && h + c * 16 < mine) tmem_ld16(lanes + b * HALF + h + c * 16, v[c]);
                    tmem_ld_wait();
                    if (h + 48 >= HALF || h + 48 >= mine) {  // the last: the accumulator is free
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0 && h < mine) mbar_arrive_pair(mapa_shared(tempty + 8 * b, 0));
                    }
#pragma unroll
                    for (int c = 0; c < 3; ++c)
                        if (h + c * 16 < HALF && h + c * 16 < mine) {
#pragma unroll
                            for (int k = 0; k < 8; ++k) fma2(acc[h / 2 + c * 8 + k], v[c][2 * k], v[c][2 * k + 1], scale);
                        }
                    if (h + 48 >= mine) break;
                }
            }
            g += steps * it.halves;
            // The warpgroup stores together or not at all: a warp that gave up meets the others here.
            ok = bar_and_all(1 + part, 128, ok);
            if (!ok) break;
            item_at(u, p, first_tile, rank, &it);  // again: nothing of it is kept above
            // Sums leave through shared memory 32 columns at a time, [column][row], so that a
            // thread stores neighbouring outputs of one column at once.
            const int left = min(mine, it.cols - part * it.half);  // this warpgroup's existing columns
            float* swap = exchange + part * (EXCHANGE / 4);
            int* pairs_at = reinterpret_cast<int*>(swap + BM * OUT_COLS);
            pairs_at[r] = row_pair;
#pragma unroll
            for (int c = 0; c < HALF; c += OUT_COLS)
                if (c < left) {
#pragma unroll
                    for (int i = 0; i < OUT_COLS; ++i) swap[i * BM + r] = CodeUnit<T>::VALUE * half_of(acc[(c + i) / 2], i & 1);
                    asm volatile("bar.sync %0, 128;" ::"r"(1 + part) : "memory");
                    sums_out<T>(p, it, swap, pairs_at + c, it.p0 + part * it.half + c, min(OUT_COLS, left - c), r);
                    asm volatile("bar.sync %0, 128;" ::"r"(1 + part) : "memory");
                }
        }
    }

    tc_fence_before();
    __syncthreads();
    cluster_sync();  // neither CTA leaves while the other may still signal it
    if (warp == 3) {
        tc_fence_after();
        tmem_dealloc_pair(tmem, 512);
    }
}

int resident_pairs(const uor_b200_ctx* ctx);

// A launch's tile width and splits. An expert's rows are spread evenly over their tiles; for one
// matrix the width is chosen by the time of whole waves of tiles.
void plan(const uor_b200_ctx* ctx, ManyParams* p) {
    const int outputs = p->mode == MANY_UP ? BM : 2 * BM;
    const int clusters = resident_pairs(ctx);
    p->row_tiles = (p->n + outputs - 1) / outputs;
    const int kbs = (p->w.cols + BK - 1) / BK;
    p->splits = 1;
    p->max_cols = MAX_COLS;
    int64_t tiles = p->experts;
    if (p->mode == MANY_DENSE) {
        double best = 0;
        for (int width = MAX_COLS; width >= 128 && p->m > 128; width -= 64) {
            const int64_t tt = (p->m + width - 1) / width;
            const int64_t each = ((p->m + tt - 1) / tt + 63) & ~63ll;
            const int64_t waves = (tt * p->row_tiles + clusters - 1) / clusters;
            // decoding and scaling take as long beside narrow tiles as beside wide ones
            const double cost = static_cast<double>(waves) * (each + 128);
            if (best == 0 || cost < best) best = cost, p->max_cols = width;
        }
        tiles = (p->m + p->max_cols - 1) / p->max_cols;
    }
    if (p->mode != MANY_UP) {
        // Eight stages to a split at least.
        int64_t want = clusters / (tiles * p->row_tiles);
        const int64_t most = kbs / 8;
        if (want > most) want = most;
        if (want > 8) want = 8;
        if (want > 1) p->splits = static_cast<int>(want);
    }
    p->kb_per_split = (kbs + p->splits - 1) / p->splits;
    p->splits = (kbs + p->kb_per_split - 1) / p->kb_per_split;
}

// The pairs that run at one time. All instances have the same resources.
int resident_pairs(const uor_b200_ctx* ctx) {
    static int most[64] = {};
    int& n = most[ctx->device & 63];
    if (n) return n;
    auto* kernel = many_kernel<__nv_bfloat16, 128>;
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(ctx->sm_count / 2 * 2);
    c.blockDim = dim3(THREADS);
    c.dynamicSmemBytes = SMEM;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    c.attrs = &attr;
    c.numAttrs = 1;
    int found = 0;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&found, kernel, &c) != cudaSuccess || found < 1) {
        cudaGetLastError();
        found = ctx->sm_count / 2;
    }
    return n = found;
}

template <typename T, int SEG>
int launch_many(uor_b200_ctx* ctx, ManyParams& p, bool early) {
    CUtensorMap tm_codes, tm_x;
    const uint64_t rows = static_cast<uint64_t>(p.w.rows);
    if (!make_tmap_u8_sw64(&tm_codes, p.w.codes, (p.w.cols + 1) / 2, rows, p.w.row_bytes, BK / 2, 64) ||
        !make_tmap_u16(&tm_x, p.x, p.w.cols, p.x_rows, p.x_rs * 2, ATOM, X_BOX))
        return UOR_B200_DEVICE_ERROR;
    auto* kernel = many_kernel<T, SEG>;
    static bool ready[64] = {};
    if (!ready[ctx->device & 63]) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess)
            return UOR_B200_DEVICE_ERROR;
        ready[ctx->device & 63] = true;
    }
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(2 * resident_pairs(ctx));
    c.blockDim = dim3(THREADS);
    c.dynamicSmemBytes = SMEM;
    c.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    c.attrs = attr;
    c.numAttrs = early ? 2 : 1;
    return cuda_status(cudaLaunchKernelEx(&c, kernel, tm_codes, tm_x, p));
}

template <typename T>
int by_segment(uor_b200_ctx* ctx, ManyParams& p, bool early) {
    if (p.w.group % 128 == 0) return launch_many<T, 128>(ctx, p, early);
    if (p.w.group % 64 == 0) return launch_many<T, 64>(ctx, p, early);
    return launch_many<T, 32>(ctx, p, early);
}

}  // namespace

int many_splits(const uor_b200_ctx* ctx, const ManyParams& p) {
    ManyParams q = p;
    plan(ctx, &q);
    return q.splits;
}

int many_launch(uor_b200_ctx* ctx, int elem, ManyParams p, bool early) {
    plan(ctx, &p);
    p.groups = (p.w.cols + p.w.group - 1) / p.w.group;
    p.status = ctx->d_status;
    p.budget_ns = ctx->budget_ns;
    return elem == UOR_B200_BF16 ? by_segment<__nv_bfloat16>(ctx, p, early) : by_segment<__half>(ctx, p, early);
}

}  // namespace uor
