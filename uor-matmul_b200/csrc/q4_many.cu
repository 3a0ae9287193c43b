// q4_many.cu -- products of many rows with 4-bit weights and group scales.
//
// Bound by the tensor cores: 2 m n k operations on 16-bit floats. A work item is a tile of 128
// weight rows by up to 256 activation rows; the weights are the instruction's M side, so that a
// thread of the epilogue owns one weight row and a group's scale is one number per thread.
//
// The roles of a CTA: a warp brings 64-position stages of activations by TMA, another the codes of
// 128 positions; a warpgroup (two where tiles have at most 128 columns) turns each code into a
// 16-bit float, exactly (code - zero), in the swizzled layout of the operand; one thread issues
// the tcgen05.mma; two warpgroups (one) hold the sums. A group's products are summed in tensor
// memory, and at the group's end these warpgroups add scale x sum to their f32 registers, while the
// next group runs in the other half of tensor memory. So no weight is rounded: rounding scale x
// code to 16 bits would cost as much precision as rounding the output does. That costs the reads
// of tensor memory: a multiply-add per group, row and column, two in one instruction.
//
// Every wait is bounded; a role that gives up records it, and every other role leaves after it.
#include "q4_many.cuh"

#include <cstring>
#include <type_traits>

#include "ptx.cuh"

namespace uor {

namespace {

constexpr int BM = 128;        // weight rows of a tile
constexpr int BK = 64;         // reduction positions of a stage: 128 bytes of a row
constexpr int CODES_K = 128;   // of a stage of codes
constexpr int A_BYTES = BM * BK * 2;
constexpr int C_BYTES = BM * CODES_K / 2;
constexpr int THREADS = 512;

template <bool WIDE>
struct Shape {
    static constexpr int COLS = WIDE ? 256 : 128;
    static constexpr int STAGES = WIDE ? 4 : 5;
    static constexpr int CSTAGES = WIDE ? 2 : 4;
    static constexpr int X_BYTES = COLS * BK * 2;
    static constexpr int STAGE_BYTES = X_BYTES + A_BYTES;
    static constexpr int DECODERS = WIDE ? 4 : 8;  // warps
    static constexpr int SUMMERS = WIDE ? 8 : 4;
    static constexpr int EXCHANGE = (WIDE ? 2 : 1) * BM * 8 * 4;
    static constexpr int SMEM = STAGES * STAGE_BYTES + CSTAGES * C_BYTES + EXCHANGE + (MANY_MAX_EXPERTS + 1) * 4 + 256 + 1024;
};
static_assert(Shape<true>::SMEM <= 232448 && Shape<false>::SMEM <= 232448, "shared memory of a block");

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
__device__ __forceinline__ bool item_at(int u, const ManyParams& p, const int* first_tile, Item* it) {
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
    const int size = ((count + parts - 1) / parts + 15) & ~15;  // even shares, in whole instructions
    const int i = tt - first_tile[lo];
    it->expert = lo;
    it->cols = min(size, count - i * size);
    it->n = (it->cols + 15) & ~15;
    it->p0 = begin + static_cast<int64_t>(i) * size;
    const int outputs = p.mode == MANY_UP ? BM / 2 : BM;
    it->j0 = rt * outputs;
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

template <typename T, int SEG, bool WIDE>
__global__ void __launch_bounds__(THREADS, 1)
    many_kernel(const __grid_constant__ CUtensorMap tm_codes, const __grid_constant__ CUtensorMap tm_x,
                const __grid_constant__ ManyParams p) {
    using S = Shape<WIDE>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* codes_at = smem + S::STAGES * S::STAGE_BYTES;
    float* exchange = reinterpret_cast<float*>(codes_at + S::CSTAGES * C_BYTES);
    uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(exchange) + S::EXCHANGE);
    int* first_tile = reinterpret_cast<int*>(bars + 32);
    const uint32_t xfull = smem_u32(bars), afull = xfull + 8 * S::STAGES, empty = afull + 8 * S::STAGES;
    const uint32_t cfull = empty + 8 * S::STAGES, cempty = cfull + 8 * S::CSTAGES;
    const uint32_t tfull = cempty + 8 * S::CSTAGES, tempty = tfull + 16, drain = tempty + 16;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 31);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wg = warp >> 2;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; ++s) {
            mbar_init(xfull + 8 * s, 1);
            mbar_init(afull + 8 * s, S::DECODERS);
            mbar_init(empty + 8 * s, 1);
        }
        for (int s = 0; s < S::CSTAGES; ++s) {
            mbar_init(cfull + 8 * s, 1);
            mbar_init(cempty + 8 * s, S::DECODERS);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(tfull + 8 * b, 1);
            mbar_init(tempty + 8 * b, S::SUMMERS);
        }
        mbar_init(drain, 1);
        fence_barrier_init();
        tma_prefetch_desc(&tm_codes);
        tma_prefetch_desc(&tm_x);
    }
    if (warp == 3) tmem_alloc(smem_u32(tmem_slot), 2 * S::COLS);
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
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int items = p.row_tiles * first_tile[p.experts] * p.splits;
    Item it;

    if (wg == 0) {
        regs_down<32>();
        if (warp == 0) {  // activations
            if (elect_one()) {
                const uint64_t policy = l2_policy_evict_last();
                int s = 0;
                uint32_t phase = 0, armed = 0, armed_phase = 0;
                bool ok = true;
                for (int u = blockIdx.x; u < items && ok; u += gridDim.x) {
                    if (!item_at(u, p, first_tile, &it)) continue;
                    const int boxes = (it.n + 63) / 64;
                    for (int kb = 0; kb < it.kbs; ++kb) {
                        if (!mbar_wait(empty + 8 * s, phase ^ 1, p.budget_ns, p.status, KERR_TIMEOUT_PRODUCER)) {
                            ok = false;
                            break;
                        }
                        mbar_expect_tx(xfull + 8 * s, boxes * 64 * BK * 2);
                        armed |= 1u << s;
                        armed_phase = (armed_phase & ~(1u << s)) | phase << s;
                        const uint32_t dst = smem_u32(smem + s * S::STAGE_BYTES);
                        for (int b = 0; b < boxes; ++b)
                            tma_load_2d(dst + b * (64 * BK * 2), &tm_x, xfull + 8 * s, (it.kb0 + kb) * BK,
                                        static_cast<int>(it.p0) + b * 64, policy);
                        if (++s == S::STAGES) s = 0, phase ^= 1;
                    }
                }
                if (!ok)
                    for (int i = 0; i < S::STAGES; ++i)
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
                for (int u = blockIdx.x; u < items && ok; u += gridDim.x) {
                    if (!item_at(u, p, first_tile, &it)) continue;
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
                        if (++s == S::CSTAGES) s = 0, phase ^= 1;
                    }
                }
                if (!ok)
                    for (int i = 0; i < S::CSTAGES; ++i)
                        if (armed >> i & 1)
                            mbar_wait(cfull + 8 * i, armed_phase >> i & 1, p.budget_ns, p.status, KERR_TIMEOUT_DRAIN);
            }
            __syncwarp();
        } else if (warp == 1) {  // the tensor cores
            int s = 0, b = 0;
            uint32_t phase = 0, bphase = 0;
            bool ok = true, issued = false;
            constexpr int PER_STAGE = SEG >= BK ? 1 : BK / SEG;  // groups' pieces in a stage
            constexpr int MMAS = BK / 16 / PER_STAGE;
            for (int u = blockIdx.x; u < items && ok; u += gridDim.x) {
                if (!item_at(u, p, first_tile, &it)) continue;
                const uint32_t idesc = idesc_f16(BM, it.n, std::is_same<T, __nv_bfloat16>::value);
                for (int kb = 0; kb < it.kbs && ok; ++kb) {
                    if (!mbar_wait_warp(xfull + 8 * s, phase, p.budget_ns, p.status, KERR_TIMEOUT_MMA_FULL) ||
                        !mbar_wait_warp(afull + 8 * s, phase, p.budget_ns, p.status, KERR_TIMEOUT_MMA_FULL)) {
                        ok = false;
                        break;
                    }
                    const uint32_t sx = smem_u32(smem + s * S::STAGE_BYTES), sa = sx + S::X_BYTES;
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
                            for (int i = 0; i < MMAS; ++i) {
                                const int at = (h * MMAS + i) * 32;
                                mma_f16(tmem + b * S::COLS, smem_desc_sw128(sa + at, 16, 1024), smem_desc_sw128(sx + at, 16, 1024),
                                        idesc, !first || i != 0);
                            }
                            if (last) mma_commit(tfull + 8 * b);
                            issued = true;
                        }
                        __syncwarp();
                        if (last) {
                            b ^= 1;
                            if (b == 0) bphase ^= 1;
                        }
                    }
                    if (!ok) break;
                    if (elect_one()) mma_commit(empty + 8 * s);
                    __syncwarp();
                    if (++s == S::STAGES) s = 0, phase ^= 1;
                }
            }
            if (!ok) {
                if (elect_one() && issued) {
                    mma_commit(drain);
                    mbar_wait(drain, 0, p.budget_ns, p.status, KERR_TIMEOUT_DRAIN);
                }
                __syncwarp();
            }
        }
    } else if (wg == 1 || (!WIDE && wg == 3)) {
        if constexpr (WIDE) regs_down<80>();
        else regs_down<104>();
        // A thread turns its row's codes into the operand: all of a stage's 64 positions, or half.
        const int r = threadIdx.x & 127;
        constexpr int SPAN = WIDE ? BK : BK / 2;
        const int k0 = WIDE || wg == 1 ? 0 : SPAN;
        int s = 0, q = 0;
        uint32_t phase = 0, qphase = 0;
        const int groups = (p.w.cols + p.w.group - 1) / p.w.group;
        bool ok = true;
        for (int u = blockIdx.x; u < items && ok; u += gridDim.x) {
            if (!item_at(u, p, first_tile, &it)) continue;
            const int64_t row = min(it.row0 + (r < 64 ? r : r - 64 + (p.mode == MANY_UP ? p.n : 64)), static_cast<int64_t>(p.w.rows) - 1);
            const uint8_t* zeros = p.w.zeros ? p.w.zeros + row * p.w.groups_rs : nullptr;
            // this row's zero point at position k
            auto zero_at = [&](int k) {
                return zeros ? static_cast<uint32_t>(zeros[min(k / p.w.group, groups - 1)]) & 15u : 8u;
            };
            constexpr int PIECE = SEG < SPAN ? SEG : SPAN;  // positions under one zero point
            constexpr int PIECES = SPAN / PIECE;
            uint32_t z[PIECES], next[PIECES];
#pragma unroll
            for (int i = 0; i < PIECES; ++i) next[i] = zero_at(it.kb0 * BK + k0 + i * PIECE);
            for (int kb = 0; kb < it.kbs; ++kb) {
#pragma unroll
                for (int i = 0; i < PIECES; ++i) {
                    z[i] = zero_pair<T>(next[i]);
                    if (zeros) next[i] = zero_at((it.kb0 + kb + 1) * BK + k0 + i * PIECE);
                }
                if ((kb & 1) == 0 &&
                    !mbar_wait_warp(cfull + 8 * q, qphase, p.budget_ns, p.status, KERR_TIMEOUT_MMA_FULL)) {
                    ok = false;
                    break;
                }
                const uint8_t* from = codes_at + q * C_BYTES + r * (CODES_K / 2) + ((kb & 1) * BK + k0) / 2;
                uint4 c[SPAN / 32];
#pragma unroll
                for (int i = 0; i < SPAN / 32; ++i) c[i] = reinterpret_cast<const uint4*>(from)[i];
                if ((kb & 1) == 1 || kb == it.kbs - 1) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(cempty + 8 * q);
                    if (++q == S::CSTAGES) q = 0, qphase ^= 1;
                }
                if (!mbar_wait_warp(empty + 8 * s, phase ^ 1, p.budget_ns, p.status, KERR_TIMEOUT_PRODUCER)) {
                    ok = false;
                    break;
                }
                uint8_t* to = smem + s * S::STAGE_BYTES + S::X_BYTES + r * (BK * 2);
#pragma unroll
                for (int i = 0; i < SPAN / 8; ++i) {
                    const uint32_t w = i % 4 == 0 ? c[i / 4].x : i % 4 == 1 ? c[i / 4].y : i % 4 == 2 ? c[i / 4].z : c[i / 4].w;
                    *reinterpret_cast<uint4*>(to + (((k0 / 8 + i) ^ (r & 7)) << 4)) = decode8<T>(w, z[i * 8 / PIECE]);
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(afull + 8 * s);
                if (++s == S::STAGES) s = 0, phase ^= 1;
            }
        }
    } else {
        if constexpr (WIDE) regs_up<200>();
        else regs_up<208>();
        const int r = threadIdx.x & 127, part = WIDE ? wg - 2 : 0;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(r & ~31) << 16) + part * 128;
        const int groups = (p.w.cols + p.w.group - 1) / p.w.group;
        int b = 0;
        uint32_t bphase = 0;
        bool ok = true;
        for (int u = blockIdx.x; u < items && ok; u += gridDim.x) {
            if (!item_at(u, p, first_tile, &it)) continue;
            const int64_t row = min(it.row0 + (r < 64 ? r : r - 64 + (p.mode == MANY_UP ? p.n : 64)), static_cast<int64_t>(p.w.rows) - 1);
            const int64_t scales = row * p.w.groups_rs;
            const int from = it.kb0 * BK, to = min(p.w.cols, from + it.kbs * BK);
            auto scale_at = [&](int k) { return load_f32(p.w.scales, scales + min(k / p.w.group, groups - 1), p.w.scale_type); };
            uint64_t acc[64];
#pragma unroll
            for (int i = 0; i < 64; ++i) acc[i] = 0;
            const int mine = it.n - part * 128;  // this warpgroup's columns
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
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (c * 32 < mine) {
                        uint32_t v[32];
                        __syncwarp();
                        tmem_ld32(lanes + b * S::COLS + c * 32, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; ++i) fma2(acc[c * 16 + i], v[2 * i], v[2 * i + 1], scale);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(tempty + 8 * b);
                b ^= 1;
                if (b == 0) bphase ^= 1;
            }
            // The warpgroup stores together or not at all: a warp that gave up meets the others here.
            ok = bar_and_all(1 + part, 128, ok);
            if (!ok) break;
            // Sums leave through shared memory eight columns at a time, [column][row], so that a
            // thread stores neighbouring outputs of one column at once.
            const int left = it.cols - part * 128;  // this warpgroup's existing columns
            float* swap = exchange + part * (BM * 8);
            const int col = r >> 4;  // the column of eight that this thread stores
            if (p.mode == MANY_UP) {
                // Rows 0 .. 63 are gates, 64 .. 127 the same outputs' ups.
                const int j = (r & 15) * 4;
                const float* gate = swap + col * BM + j;
                T* to = static_cast<T*>(p.h) + (it.p0 + part * 128 + col) * p.h_rs + it.j0 + j;
                const int valid = min(4, p.n - it.j0 - j);
#pragma unroll
                for (int c = 0; c < 128; c += 8)
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
                for (int c = 0; c < 128; c += 8)
                    if (c < left) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) swap[i * BM + r] = half_of(acc[(c + i) / 2], i & 1);
                        asm volatile("bar.sync %0, 128;" ::"r"(1 + part) : "memory");
                        if (c + col < left && valid > 0) out(p, it, it.p0 + part * 128 + c + col, it.j0 + j, from, valid);
                        asm volatile("bar.sync %0, 128;" ::"r"(1 + part) : "memory");
                    }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 3) {
        tc_fence_after();
        tmem_dealloc(tmem, 2 * S::COLS);
    }
}

// A launch's tile width and splits. Rows of x are spread evenly over their tiles, so a tile is
// as wide as the rows allow up to 256 (or 128, where none needs more: the second warpgroup of
// decoders then halves the time a stage's codes take). For one matrix the width is chosen by the
// time of whole waves of tiles.
void plan(const uor_b200_ctx* ctx, ManyParams* p) {
    const int outputs = p->mode == MANY_UP ? BM / 2 : BM;
    p->row_tiles = (p->n + outputs - 1) / outputs;
    const int kbs = (p->w.cols + BK - 1) / BK;
    p->splits = 1;
    p->max_cols = p->row_bound <= 128 ? 128 : 256;
    int64_t tiles = p->experts;
    if (p->mode == MANY_DENSE) {
        if (p->m > 256) {
            double best = 0;
            for (int width = 256; width >= 160; width -= 16) {
                const int64_t tt = (p->m + width - 1) / width;
                const int64_t each = ((p->m + tt - 1) / tt + 15) & ~15ll;
                const int64_t waves = (tt * p->row_tiles + ctx->sm_count - 1) / ctx->sm_count;
                const double cost = static_cast<double>(waves) * (each + 24);  // a tile's fixed part
                if (best == 0 || cost < best) best = cost, p->max_cols = width;
            }
        }
        tiles = (p->m + p->max_cols - 1) / p->max_cols;
    }
    if (p->mode != MANY_UP) {
        // Whole stages of codes to a split, and eight of them at least.
        int64_t want = ctx->sm_count / (tiles * p->row_tiles);
        const int64_t most = kbs / 16;
        if (want > most) want = most;
        if (want > 8) want = 8;
        if (want > 1) p->splits = static_cast<int>(want);
    }
    p->kb_per_split = ((kbs + p->splits - 1) / p->splits + 1) & ~1;
    p->splits = (kbs + p->kb_per_split - 1) / p->kb_per_split;
}

template <typename T, int SEG, bool WIDE>
int launch_many(uor_b200_ctx* ctx, ManyParams& p) {
    CUtensorMap tm_codes, tm_x;
    const uint64_t rows = static_cast<uint64_t>(p.w.rows);
    if (!make_tmap_u8(&tm_codes, p.w.codes, (p.w.cols + 1) / 2, rows, p.w.row_bytes, CODES_K / 2, 64, false) ||
        !make_tmap_u16(&tm_x, p.x, p.w.cols, p.x_rows, p.x_rs * 2, BK, 64))
        return UOR_B200_DEVICE_ERROR;
    auto* kernel = many_kernel<T, SEG, WIDE>;
    static bool ready[64] = {};
    if (!ready[ctx->device & 63]) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<WIDE>::SMEM) != cudaSuccess)
            return UOR_B200_DEVICE_ERROR;
        ready[ctx->device & 63] = true;
    }
    kernel<<<ctx->sm_count, THREADS, Shape<WIDE>::SMEM, ctx->stream>>>(tm_codes, tm_x, p);
    return cuda_status(cudaGetLastError());
}

template <typename T, int SEG>
int by_width(uor_b200_ctx* ctx, ManyParams& p) {
    return p.max_cols > 128 ? launch_many<T, SEG, true>(ctx, p) : launch_many<T, SEG, false>(ctx, p);
}

template <typename T>
int by_segment(uor_b200_ctx* ctx, ManyParams& p) {
    if (p.w.group % 128 == 0) return by_width<T, 128>(ctx, p);
    if (p.w.group % 64 == 0) return by_width<T, 64>(ctx, p);
    return by_width<T, 32>(ctx, p);
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
