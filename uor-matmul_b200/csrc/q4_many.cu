// q4_many.cu -- products of many rows with 4-bit weights and group scales.
//
// Bound by the tensor cores: 2 m n k operations on 16-bit floats. A work item is a tile of 256
// weight rows by up to 192 activation rows, on a pair of CTAs (tcgen05.mma.cta_group::2): each
// CTA holds 128 of the weight rows and brings half of the activation rows. The weights are the
// instruction's M side, so that a thread of the epilogue owns one weight row and a group's scale
// is one number per thread.
//
// The roles of a CTA: a warp brings 64-position stages of activations by TMA, another the codes of
// 128 positions; two warpgroups turn each code into a 16-bit float, exactly (code - zero), and
// store it to tensor memory, where the instruction takes its A side from; one thread of the pair
// issues the tcgen05.mma; two warpgroups hold the sums. A group's products are summed in tensor
// memory, and at the group's end these warpgroups add scale x sum to their f32 registers, while the
// next group runs in the other of two accumulators. So no weight is rounded: rounding scale x
// code to 16 bits would cost as much precision as rounding the output does.
//
// Why this shape. With the weights in shared memory and one CTA per 128 x 256 tile, the operands'
// reads, the TMA's and the decoders' writes came to 104 KB a stage, 830 cycles at 128 bytes a
// cycle, for 512 cycles of multiplication (2048 x 8192 x 8192: 366 us, 295 us without decoding
// and scaling). Here a stage moves 4 x 3 KB of operands, 12 KB of TMA and 8 KB of codes for 384.
// Tensor memory's 512 columns hold two accumulators of 192 and four stages of weights of 32.
//
// Every wait is bounded; a role that gives up records it, and every other role leaves after it.
#include "q4_many.cuh"

#include <cstring>
#include <type_traits>

#include "ptx.cuh"

namespace uor {

namespace {

constexpr int BM = 128;        // weight rows of a CTA's half of a tile
constexpr int BK = 64;         // reduction positions of a stage: 128 bytes of a row
constexpr int CODES_K = 128;   // of a stage of codes
constexpr int MAX_COLS = 192;  // activation rows of a tile
constexpr int X_BOX = 32;      // activation rows of one TMA copy
constexpr int X_BOX_BYTES = X_BOX * BK * 2;
constexpr int X_BYTES = MAX_COLS / 2 * BK * 2;
constexpr int C_BYTES = BM * CODES_K / 2;
constexpr int XSTAGES = 8, CSTAGES = 6, ASTAGES = 4;
constexpr int A_COLS = BK / 2;                       // tensor-memory columns of a stage of weights
constexpr int A_FIRST = 2 * MAX_COLS;
constexpr int DECODERS = 8, SUMMERS = 8;             // warps of a CTA
constexpr int PART = MAX_COLS / 2;                   // columns of a summing warpgroup
constexpr int EXCHANGE = BM * 8 * 4;                 // bytes, per summing warpgroup
constexpr int BARS = 2 * XSTAGES + 2 * CSTAGES + 2 * ASTAGES + 5;
constexpr int SMEM = XSTAGES * X_BYTES + CSTAGES * C_BYTES + 2 * EXCHANGE + (BARS + 1) * 8 + (MANY_MAX_EXPERTS + 1) * 4 + 1024;
// Warpgroup 0: TMA, MMA; 1 and 2: decoders; 3 and 4: sums. Registers: 96 a thread at launch.
constexpr int THREADS = 640;
constexpr int REGS_CONTROL = 48, REGS_DECODE = 48, REGS_SUM = 160;
static_assert(SMEM <= 232448, "shared memory of a block");
static_assert(A_FIRST + ASTAGES * A_COLS == 512, "tensor memory");
static_assert(REGS_CONTROL + 2 * REGS_DECODE + 2 * REGS_SUM <= 5 * 96, "registers of the launch");

struct Item {
    int expert, cols, n;      // cols: existing activation rows; n: the instruction's
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
    const int size = ((count + parts - 1) / parts + 31) & ~31;  // even shares, in whole instructions
    const int i = tt - first_tile[lo];
    it->expert = lo;
    it->cols = min(size, count - i * size);
    it->n = (it->cols + 31) & ~31;
    it->p0 = begin + static_cast<int64_t>(i) * size;
    const int outputs = p.mode == MANY_UP ? BM / 2 : BM;  // of a CTA
    it->j0 = (2 * rt + rank) * outputs;
    it->row0 = static_cast<int64_t>(lo) * (p.mode == MANY_UP ? 2 * p.n : p.n) + it->j0;
    it->kb0 = it->split * p.kb_per_split;
    it->kbs = min(p.kb_per_split, (p.w.cols + BK - 1) / BK - it->kb0);
    return it->cols > 0 && it->kbs > 0;
}

// Eight codes of a word, in order, less their zero point, as 16-bit floats.
template <typename T>
__device__ __forceinline__ uint4 decode8(uint32_t w, uint32_t zero) {
    constexpr uint32_t HIGH = std::is_same<T, __half>::value ? 0x64u : 0x43u;  // 1024 or 128
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
    return (std::is_same<T, __half>::value ? 0x64006400u : 0x43004300u) | (z << 16) | z;
}

// acc += v * s on two floats at once.
__device__ __forceinline__ void fma2(uint64_t& acc, uint32_t lo, uint32_t hi, uint64_t s) {
    asm("{\n .reg .b64 v;\n mov.b64 v, {%1, %2};\n fma.rn.f32x2 %0, v, %3, %0;\n}\n" : "+l"(acc) : "r"(lo), "r"(hi), "l"(s));
}
__device__ __forceinline__ float half_of(uint64_t v, int i) {
    return __uint_as_float(static_cast<uint32_t>(i ? v >> 32 : v));
}

// Four inner activations from their gates' and ups' sums.
template <typename T>
__device__ __noinline__ void up_out(const float* gate, int valid, T* to) {
    const float4 g = *reinterpret_cast<const float4*>(gate), u = *reinterpret_cast<const float4*>(gate + 64);
    const float v[4] = {silu(g.x) * u.x, silu(g.y) * u.y, silu(g.z) * u.z, silu(g.w) * u.w};
    if (valid == 4) {  // rows of h begin at multiples of 16 bytes
        T t[4] = {from_f32<T>(v[0]), from_f32<T>(v[1]), from_f32<T>(v[2]), from_f32<T>(v[3])};
        uint2 bits;
        memcpy(&bits, t, 8);
        *reinterpret_cast<uint2*>(to) = bits;
    } else {
        for (int i = 0; i < valid; ++i) to[i] = from_f32<T>(i == 0 ? v[0] : i == 1 ? v[1] : v[2]);
    }
}

// Eight neighbouring outputs of activation row i from output j on, to where this launch's go.
__device__ __noinline__ void out(const ManyParams& p, const Item& it, int64_t i, int j, const float* from, int valid) {
    const float4 a = *reinterpret_cast<const float4*>(from), b = *reinterpret_cast<const float4*>(from + 4);
    void* to = p.part;
    int64_t at, step = 1;
    int type = UOR_B200_F32;
    if (p.mode == MANY_DOWN || p.splits > 1) {
        at = (it.split * p.part_rows + (p.mode == MANY_DOWN ? p.perm[i] : i)) * p.n + j;
    } else {
        to = p.y.p;
        type = p.y.type;
        step = p.y.cs;
        at = i * p.y.rs + j * step;
    }
    const int size = type == UOR_B200_F32 ? 4 : 2;
    char* c = static_cast<char*>(to) + at * size;
    if (valid == 8 && step == 1 && reinterpret_cast<uint64_t>(c) % 16 == 0) {
        if (type == UOR_B200_F32) {
            reinterpret_cast<float4*>(c)[0] = a;
            reinterpret_cast<float4*>(c)[1] = b;
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
            *reinterpret_cast<uint4*>(c) = w;
        }
    } else {
        for (int k = 0; k < valid; ++k) store_f32(to, at + k * step, type, from[k]);
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
    uint8_t* codes_at = smem + XSTAGES * X_BYTES;
    float* exchange = reinterpret_cast<float*>(codes_at + CSTAGES * C_BYTES);
    uint64_t* bars = reinterpret_cast<uint64_t*>(exchange + 2 * BM * 8);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + BARS);
    int* first_tile = reinterpret_cast<int*>(bars + BARS + 1);
    const uint32_t xfull = smem_u32(bars), xempty = xfull + 8 * XSTAGES;  // xfull: the leader's, both CTAs' bytes
    const uint32_t cfull = xempty + 8 * XSTAGES, cempty = cfull + 8 * CSTAGES;
    const uint32_t afull = cempty + 8 * CSTAGES, aempty = afull + 8 * ASTAGES;  // afull: the leader's
    const uint32_t tfull = aempty + 8 * ASTAGES, tempty = tfull + 16, drain = tempty + 16;  // tempty: the leader's
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wg = warp >> 2;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const int pair = static_cast<int>(cluster_id_x()), pairs = static_cast<int>(nclusters_x());

    if (threadIdx.x == 0) {
        for (int s = 0; s < XSTAGES; ++s) {
            mbar_init(xfull + 8 * s, 1);
            mbar_init(xempty + 8 * s, 1);
        }
        for (int s = 0; s < CSTAGES; ++s) {
            mbar_init(cfull + 8 * s, 1);
            mbar_init(cempty + 8 * s, DECODERS);
        }
        for (int s = 0; s < ASTAGES; ++s) {
            mbar_init(afull + 8 * s, DECODERS);  // one warpgroup of each CTA
            mbar_init(aempty + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(tfull + 8 * b, 1);
            mbar_init(tempty + 8 * b, 2 * SUMMERS);
        }
        mbar_init(drain, 1);
        fence_barrier_init();
        tma_prefetch_desc(&tm_codes);
        tma_prefetch_desc(&tm_x);
    }
    if (warp == 3) tmem_alloc_pair(smem_u32(tmem_slot), 512);
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
                int s = 0;
                uint32_t phase = 0, armed = 0, armed_phase = 0;
                bool ok = true;
                for (int u = pair; u < items && ok; u += pairs) {
                    if (!item_at(u, p, first_tile, rank, &it)) continue;
                    const int boxes = (it.n / 2 + X_BOX - 1) / X_BOX;
                    const int row = static_cast<int>(it.p0) + static_cast<int>(rank) * (it.n / 2);
                    for (int kb = 0; kb < it.kbs; ++kb) {
                        if (!mbar_wait(xempty + 8 * s, phase ^ 1, p.budget_ns, p.status, KERR_TIMEOUT_PRODUCER)) {
                            ok = false;
                            break;
                        }
                        if (leader) {
                            mbar_expect_tx(xfull + 8 * s, 2 * boxes * X_BOX_BYTES);
                            armed |= 1u << s;
                            armed_phase = (armed_phase & ~(1u << s)) | phase << s;
                        }
                        const uint32_t full = mapa_shared(xfull + 8 * s, 0);
                        const uint32_t dst = smem_u32(smem + s * X_BYTES);
                        for (int b = 0; b < boxes; ++b)
                            tma_load_2d_pair(dst + b * X_BOX_BYTES, &tm_x, full, (it.kb0 + kb) * BK, row + b * X_BOX, policy);
                        if (++s == XSTAGES) s = 0, phase ^= 1;
                    }
                }
                if (!ok && leader)
                    for (int i = 0; i < XSTAGES; ++i)
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
                    for (int kb = 0; kb < it.kbs; kb += 2) {
                        if (!mbar_wait(cempty + 8 * s, phase ^ 1, p.budget_ns, p.status, KERR_TIMEOUT_PRODUCER)) {
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
            int s = 0, a = 0, b = 0;
            uint32_t phase = 0, aphase = 0, bphase = 0;
            bool ok = true, issued = false;
            constexpr int PER_STAGE = SEG >= BK ? 1 : BK / SEG;  // groups' pieces in a stage
            constexpr int MMAS = BK / 16 / PER_STAGE;
            for (int u = pair; u < items && ok; u += pairs) {
                if (!item_at(u, p, first_tile, rank, &it)) continue;
                const uint32_t idesc = idesc_f16(2 * BM, it.n, std::is_same<T, __nv_bfloat16>::value);
                for (int kb = 0; kb < it.kbs && ok; ++kb) {
                    if (!mbar_wait_warp(xfull + 8 * s, phase, p.budget_ns, p.status, KERR_TIMEOUT_MMA_FULL) ||
                        !mbar_wait_warp(afull + 8 * a, aphase, p.budget_ns, p.status, KERR_TIMEOUT_MMA_FULL)) {
                        ok = false;
                        break;
                    }
                    const uint32_t sx = smem_u32(smem + s * X_BYTES), sa = tmem + A_FIRST + a * A_COLS;
                    const bool first = SEG != 128 || (kb & 1) == 0;
                    const bool last = SEG != 128 || (kb & 1) == 1 || kb == it.kbs - 1;
                    for (int h = 0; h < PER_STAGE; ++h) {
                        if (h && (it.kb0 + kb) * BK + h * SEG >= p.w.cols) break;
                        if (first && !mbar_wait_warp(tempty + 8 * b, bphase ^ 1, p.budget_ns, p.status, KERR_TIMEOUT_MMA_ACC)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        if (elect_one()) {
#pragma unroll
                            for (int i = 0; i < MMAS; ++i)
                                mma_f16_pair_ts(tmem + b * MAX_COLS, sa + (h * MMAS + i) * 8,
                                                smem_desc_sw128(sx + (h * MMAS + i) * 32, 16, 1024), idesc, !first || i != 0);
                            if (last) mma_commit_pair(tfull + 8 * b, 0x3);
                            issued = true;
                        }
                        __syncwarp();
                        if (last) {
                            b ^= 1;
                            if (b == 0) bphase ^= 1;
                        }
                    }
                    if (!ok) break;
                    if (elect_one()) {
                        mma_commit_pair(xempty + 8 * s, 0x3);
                        mma_commit_pair(aempty + 8 * a, 0x3);
                    }
                    __syncwarp();
                    if (++s == XSTAGES) s = 0, phase ^= 1;
                    if (++a == ASTAGES) a = 0, aphase ^= 1;
                }
            }
            if (!ok) {
                if (elect_one() && issued) {
                    mma_commit_pair(drain, 0x1);
                    mbar_wait(drain, 0, p.budget_ns, p.status, KERR_TIMEOUT_DRAIN);
                }
                __syncwarp();
            }
        }
    } else if (wg <= 2) {
        regs_down<REGS_DECODE>();
        // A thread turns its row's codes into the operand's row, lane r of tensor memory. The two
        // warpgroups take the two stages of each stage of codes.
        const int r = threadIdx.x & 127, odd = wg - 1;
        const uint32_t to = tmem + (static_cast<uint32_t>(r & ~31) << 16) + A_FIRST;
        const uint8_t* from = codes_at + r * (CODES_K / 2);
        const int turn = (r >> 1) & 3;  // the 64-byte swizzle's
        int q = 0;
        uint32_t qphase = 0, n = 0;  // n: stages of weights so far
        const int groups = (p.w.cols + p.w.group - 1) / p.w.group;
        bool ok = true;
        for (int u = pair; u < items && ok; u += pairs) {
            if (!item_at(u, p, first_tile, rank, &it)) continue;
            const int64_t row = min(it.row0 + (r < 64 ? r : r - 64 + (p.mode == MANY_UP ? p.n : 64)), static_cast<int64_t>(p.w.rows) - 1);
            const uint8_t* zeros = p.w.zeros ? p.w.zeros + row * p.w.groups_rs : nullptr;
            constexpr int PIECE = SEG < BK ? SEG : BK;  // positions under one zero point
            constexpr int PIECES = BK / PIECE;
            uint32_t next[PIECES];
            auto fetch = [&](int kb) {  // this row's zero points of stage kb
#pragma unroll
                for (int i = 0; i < PIECES; ++i)
                    next[i] = zeros ? zeros[min(((it.kb0 + kb) * BK + i * PIECE) / p.w.group, groups - 1)] & 15u : 8u;
            };
            fetch(odd);
            for (int kb = odd; kb - odd < it.kbs; kb += 2) {
                if (!mbar_wait_warp(cfull + 8 * q, qphase, p.budget_ns, p.status, KERR_TIMEOUT_MMA_FULL)) {
                    ok = false;
                    break;
                }
                const uint4 c0 = *reinterpret_cast<const uint4*>(from + q * C_BYTES + (((2 * odd) ^ turn) << 4));
                const uint4 c1 = *reinterpret_cast<const uint4*>(from + q * C_BYTES + (((2 * odd + 1) ^ turn) << 4));
                __syncwarp();
                if (lane == 0) mbar_arrive(cempty + 8 * q);
                if (++q == CSTAGES) q = 0, qphase ^= 1;
                if (kb >= it.kbs) break;  // the last stage of codes was half a one
                const uint32_t z0 = zero_pair<T>(next[0]), z1 = zero_pair<T>(next[PIECES - 1]);
                if (zeros) fetch(kb + 2);
                const uint32_t a = (n + kb) % ASTAGES, aphase = (n + kb) / ASTAGES & 1;
                if (!mbar_wait_warp(aempty + 8 * a, aphase ^ 1, p.budget_ns, p.status, KERR_TIMEOUT_PRODUCER)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                uint32_t v[16];
                auto put = [&](const uint4& c, uint32_t z, int at) {
                    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint4 d = decode8<T>(w[i], z);
                        v[4 * i] = d.x, v[4 * i + 1] = d.y, v[4 * i + 2] = d.z, v[4 * i + 3] = d.w;
                    }
                    __syncwarp();
                    tmem_st16(to + a * A_COLS + at, v);
                };
                put(c0, z0, 0);
                put(c1, z1, 16);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_pair(mapa_shared(afull + 8 * a, 0));
            }
            n += it.kbs;
        }
    } else {
        regs_up<REGS_SUM>();
        const int r = threadIdx.x & 127, part = wg - 3;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(r & ~31) << 16) + part * PART;
        const int groups = (p.w.cols + p.w.group - 1) / p.w.group;
        int b = 0;
        uint32_t bphase = 0;
        bool ok = true;
        for (int u = pair; u < items && ok; u += pairs) {
            if (!item_at(u, p, first_tile, rank, &it)) continue;
            const int64_t row = min(it.row0 + (r < 64 ? r : r - 64 + (p.mode == MANY_UP ? p.n : 64)), static_cast<int64_t>(p.w.rows) - 1);
            const int64_t scales = row * p.w.groups_rs;
            const int from = it.kb0 * BK, to = min(p.w.cols, from + it.kbs * BK);
            auto scale_at = [&](int k) { return load_f32(p.w.scales, scales + min(k / p.w.group, groups - 1), p.w.scale_type); };
            uint64_t acc[PART / 2];
#pragma unroll
            for (int i = 0; i < PART / 2; ++i) acc[i] = 0;
            const int mine = it.n - part * PART;  // this warpgroup's columns
            float next = scale_at(from);
            for (int k = from; k < to; k += SEG) {
                const uint32_t sb = __float_as_uint(next);
                const uint64_t scale = static_cast<uint64_t>(sb) << 32 | sb;
                if (k + SEG < to) next = scale_at(k + SEG);
                if (!mbar_wait_warp(tfull + 8 * b, bphase, p.budget_ns, p.status, KERR_TIMEOUT_EPILOGUE)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                // Sixteen columns travel while the sixteen before them are added.
                uint32_t v[2][16];
                __syncwarp();
                if (mine > 0) tmem_ld16(lanes + b * MAX_COLS, v[0]);
#pragma unroll
                for (int c = 0; c < PART / 16; ++c) {
                    if (c * 16 < mine) {
                        tmem_ld_wait();
                        if (c + 1 < PART / 16 && (c + 1) * 16 < mine) tmem_ld16(lanes + b * MAX_COLS + (c + 1) * 16, v[(c + 1) & 1]);
#pragma unroll
                        for (int i = 0; i < 8; ++i) fma2(acc[c * 8 + i], v[c & 1][2 * i], v[c & 1][2 * i + 1], scale);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_pair(mapa_shared(tempty + 8 * b, 0));
                b ^= 1;
                if (b == 0) bphase ^= 1;
            }
            // The warpgroup stores together or not at all: a warp that gave up meets the others here.
            ok = bar_and_all(1 + part, 128, ok);
            if (!ok) break;
            // Sums leave through shared memory eight columns at a time, [column][row], so that a
            // thread stores neighbouring outputs of one column at once.
            const int left = it.cols - part * PART;  // this warpgroup's existing columns
            float* swap = exchange + part * (BM * 8);
            const int col = r >> 4;  // the column of eight that this thread stores
            if (p.mode == MANY_UP) {
                // Rows 0 .. 63 are gates, 64 .. 127 the same outputs' ups.
                const int j = (r & 15) * 4;
                const float* gate = swap + col * BM + j;
                T* to = static_cast<T*>(p.h) + (it.p0 + part * PART + col) * p.h_rs + it.j0 + j;
                const int valid = min(4, p.n - it.j0 - j);
#pragma unroll
                for (int c = 0; c < PART; c += 8)
                    if (c < left) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) swap[i * BM + r] = half_of(acc[(c + i) / 2], i & 1);
                        asm volatile("bar.sync %0, 128;" ::"r"(1 + part) : "memory");
                        if (c + col < left && valid > 0) up_out(gate, valid, to + c * p.h_rs);
                        asm volatile("bar.sync %0, 128;" ::"r"(1 + part) : "memory");
                    }
            } else {
                const int j = (r & 15) * 8;
                const float* from = swap + col * BM + j;
                const int valid = min(8, p.n - it.j0 - j);
#pragma unroll
                for (int c = 0; c < PART; c += 8)
                    if (c < left) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) swap[i * BM + r] = half_of(acc[(c + i) / 2], i & 1);
                        asm volatile("bar.sync %0, 128;" ::"r"(1 + part) : "memory");
                        if (c + col < left && valid > 0) out(p, it, it.p0 + part * PART + c + col, it.j0 + j, from, valid);
                        asm volatile("bar.sync %0, 128;" ::"r"(1 + part) : "memory");
                    }
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
        for (int width = MAX_COLS; width >= 96 && p->m > MAX_COLS; width -= 32) {
            const int64_t tt = (p->m + width - 1) / width;
            const int64_t each = ((p->m + tt - 1) / tt + 31) & ~31ll;
            const int64_t waves = (tt * p->row_tiles + clusters - 1) / clusters;
            const double cost = static_cast<double>(waves) * (each + 24);  // a tile's fixed part
            if (best == 0 || cost < best) best = cost, p->max_cols = width;
        }
        tiles = (p->m + p->max_cols - 1) / p->max_cols;
    }
    if (p->mode != MANY_UP) {
        // Whole stages of codes to a split, and eight of them at least.
        int64_t want = clusters / (tiles * p->row_tiles);
        const int64_t most = kbs / 16;
        if (want > most) want = most;
        if (want > 8) want = 8;
        if (want > 1) p->splits = static_cast<int>(want);
    }
    p->kb_per_split = ((kbs + p->splits - 1) / p->splits + 1) & ~1;
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
int launch_many(uor_b200_ctx* ctx, ManyParams& p) {
    CUtensorMap tm_codes, tm_x;
    const uint64_t rows = static_cast<uint64_t>(p.w.rows);
    if (!make_tmap_u8_sw64(&tm_codes, p.w.codes, (p.w.cols + 1) / 2, rows, p.w.row_bytes, CODES_K / 2, 64) ||
        !make_tmap_u16(&tm_x, p.x, p.w.cols, p.x_rows, p.x_rs * 2, BK, X_BOX))
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
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    c.attrs = &attr;
    c.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&c, kernel, tm_codes, tm_x, p));
}

template <typename T>
int by_segment(uor_b200_ctx* ctx, ManyParams& p) {
    if (p.w.group % 128 == 0) return launch_many<T, 128>(ctx, p);
    if (p.w.group % 64 == 0) return launch_many<T, 64>(ctx, p);
    return launch_many<T, 32>(ctx, p);
}

}  // namespace

int many_splits(const uor_b200_ctx* ctx, const ManyParams& p) {
    ManyParams q = p;
    plan(ctx, &q);
    return q.splits;
}

int many_launch(uor_b200_ctx* ctx, int elem, ManyParams p) {
    plan(ctx, &p);
    p.status = ctx->d_status;
    p.budget_ns = ctx->budget_ns;
    return elem == UOR_B200_BF16 ? by_segment<__nv_bfloat16>(ctx, p) : by_segment<__half>(ctx, p);
}

}  // namespace uor
