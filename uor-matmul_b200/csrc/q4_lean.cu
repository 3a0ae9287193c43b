// q4_lean.cu -- products of few rows with 4-bit weights that lie well: rows of codes at multiples of
// four bytes, in whole eights, groups of 32, 64 or 128 positions, activations that fit in a block's
// shared memory.
//
// q4_few.cu's product and its split, but for the way of the codes: each lane reads its operands'
// words straight from memory into registers, one chunk ahead, so that there are no copies to
// place, to wait for and to read back. What bounds these products is latency: four warps a
// scheduler, 128 registers of each under way, keep a third to half of the issue slots busy (an
// operand's word takes 11 instructions to unpack), and a launch has its few microseconds of start:
// activations are asked for first, and nothing is divided on the device. One row: 4096 x 4096 in
// 6.3 us, 8192 x 8192 with zero points in 15.7 (2.3 TB/s), 17.0 by way of shared memory. 13 x 5003
// x 4008 with a scale and a zero point per 32 positions: 21.9, of which the bytes are 2.1; two
// chunks of 16 scales do not fit the registers beside 16 columns, and 220 bytes a thread are spilled.
#include "ptx.cuh"
#include "q4_mma.cuh"

namespace uor {

namespace {

// A chunk's codes of this lane's two rows: word SEG / 32 s + j is the j-th of segment s. WIDE: a
// segment's words are one vector, else rows begin at multiples of four bytes only.
template <int SEG, bool WIDE>
struct Codes {
    static constexpr int WORDS = SEG / 32, SEGS = CHUNK / SEG;
    uint32_t w[2][8];

    // at0, at1: the chunk's rows at this lane's first word; bytes: what is left of a row from there.
    __device__ __forceinline__ void load(const uint8_t* at0, const uint8_t* at1, int bytes, int c) {
        if (bytes >= CHUNK / 2) {
            read<false>(w[0], at0, bytes, c);
            read<false>(w[1], at1, bytes, c);
        } else {
            read<true>(w[0], at0, bytes, c);
            read<true>(w[1], at1, bytes, c);
        }
    }
    template <bool TAIL>
    __device__ static __forceinline__ void read(uint32_t (&w)[8], const uint8_t* at, int bytes, int c) {
#pragma unroll
        for (int s = 0; s < SEGS; ++s) {
            const uint8_t* from = at + s * (SEG / 2);
            uint32_t* to = w + s * WORDS;
            const int left = bytes - s * (SEG / 2) - c * 4 * WORDS;
            if (TAIL && left < 4 * WORDS) {
#pragma unroll
                for (int j = 0; j < WORDS; ++j) to[j] = 4 * j < left ? __ldg(reinterpret_cast<const uint32_t*>(from) + j) : 0;
            } else if constexpr (!WIDE) {
#pragma unroll
                for (int j = 0; j < WORDS; ++j) to[j] = __ldg(reinterpret_cast<const uint32_t*>(from) + j);
            } else if constexpr (WORDS == 4) {
                const uint4 x = __ldg(reinterpret_cast<const uint4*>(from));
                to[0] = x.x, to[1] = x.y, to[2] = x.z, to[3] = x.w;
            } else if constexpr (WORDS == 2) {
                const uint2 x = __ldg(reinterpret_cast<const uint2*>(from));
                to[0] = x.x, to[1] = x.y;
            } else {
                to[0] = __ldg(reinterpret_cast<const uint32_t*>(from));
            }
        }
    }
};

template <typename T, typename S, int SEG, int NT, bool WIDE>
__global__ void __launch_bounds__(Block<NT>::THREADS, NT == 1 ? 2 : 1) lean_kernel(const __grid_constant__ FewParams p) {
    constexpr int WARPS = Block<NT>::WARPS, THREADS = Block<NT>::THREADS, COLS = 8 * NT;
    constexpr int WORDS = SEG / 32, SEGS = CHUNK / SEG;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Found found;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int kind = p.kind, chunks = p.chunks;
    if (kind != FEW_DENSE) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    int e = 0, listed;
    int64_t x0 = 0;
    if (kind == FEW_DENSE) {
        x0 = static_cast<int64_t>(blockIdx.y) * COLS;
        listed = static_cast<int>(min(static_cast<int64_t>(COLS), p.m - x0));
    } else {
        listed = find_pairs<WARPS>(p, found);
        if (listed < 0) return;
        e = found.chosen;
        if (kind == FEW_PART) listed <<= p.twice;
    }
    const int kw = 1 << p.k_shift, k_warp = warp & (kw - 1), t_warp = warp >> p.k_shift, abreast = WARPS >> p.k_shift;
    float* red = reinterpret_cast<float*>(smem);
    const uint32_t x_all = smem_u32(smem) + Block<NT>::RED;
    const bool zeros = p.w.zeros != nullptr;
    const int row_len = p.w.cols / 2, tile_step = gridDim.x * abreast;
    const int units = chunks > k_warp ? (chunks - k_warp + kw - 1) >> p.k_shift : 0;  // chunks of a tile for this warp
    bool waited = kind != FEW_PART;

    for (int c0 = blockIdx.z * COLS; c0 < listed; c0 += gridDim.z * COLS) {
        const int rows_x = min(COLS, listed - c0), pieces = chunks * 32;
        auto x_row_at = [&](int r) {
            return static_cast<const T*>(p.x) + x_row_of(p, found, x0, c0 + r) * p.x_rs;
        };
        auto x_get = [&](const T* row, int piece) {  // 16-byte piece of an activation row
            uint4 x = make_uint4(0, 0, 0, 0);
            if (piece * 8 < p.w.cols) x = *reinterpret_cast<const uint4*>(row + piece * 8);
            return x;
        };
        auto x_put = [&](int r, int piece, uint4 x) {
            sts128(x_all + (r * chunks * 2 + (piece >> 4)) * X_BYTES + x_piece<SEG>(r, piece & 15), kind == FEW_PART ? x : in_pairs(x));
        };
        uint4 x8[2];  // of a single row
        const bool asked = waited && rows_x == 1;
        if (asked) {
            const T* row = x_row_at(0);
#pragma unroll
            for (int b = 0; b < 2; ++b) x8[b] = x_get(row, threadIdx.x + b * THREADS);
        }
        // The next unit to read: its tile and chunk, its rows of codes at this lane's words, and
        // its rows' first scales.
        int lt = blockIdx.x * abreast + t_warp, lu = 0;
        const uint8_t *at0 = nullptr, *at1 = nullptr, *z0 = nullptr, *z1 = nullptr;
        const S *s0 = nullptr, *s1 = nullptr;
        auto settle = [&]() {
            const Tile tile = tile_at(p, e, lt);
            const int64_t r0 = tile.row(g), r1 = tile.row(g + 8);
            const int k = k_warp * (CHUNK / 2) + c * 4 * WORDS;
            at0 = p.w.codes + r0 * p.w.row_bytes + k;
            at1 = p.w.codes + r1 * p.w.row_bytes + k;
            s0 = static_cast<const S*>(p.w.scales) + r0 * p.w.groups_rs + k_warp * SEGS;
            s1 = static_cast<const S*>(p.w.scales) + r1 * p.w.groups_rs + k_warp * SEGS;
            if (zeros) {
                z0 = p.w.zeros + r0 * p.w.groups_rs + k_warp * SEGS;
                z1 = p.w.zeros + r1 * p.w.groups_rs + k_warp * SEGS;
            }
        };
        Codes<SEG, WIDE> now, next;
        Quants<T, S, SEG> q_now, q_next;
        auto read = [&](Codes<SEG, WIDE>& codes, Quants<T, S, SEG>& q) {
            const int chunk = k_warp + (lu << p.k_shift), step = lu << p.k_shift;
            codes.load(at0 + step * (CHUNK / 2), at1 + step * (CHUNK / 2), row_len - chunk * (CHUNK / 2), c);
            q.load_at(s0 + step * SEGS, s1 + step * SEGS, z0 + step * SEGS, z1 + step * SEGS, zeros, p.quants_vec != 0, p.groups - chunk * SEGS);
            if (++lu == units) {
                lu = 0;
                lt += tile_step;
                if (lt < p.tiles) settle();
            }
        };
        if (units && lt < p.tiles) {
            settle();
            read(next, q_next);
        }
        if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");
        waited = true;
        if (asked) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
                if (static_cast<int>(threadIdx.x) + b * THREADS < pieces) x_put(0, threadIdx.x + b * THREADS, x8[b]);
        }
        // Three rows' reads at a time; where a row has fewer pieces than the block threads, other
        // threads take other rows.
        const int beside = pieces < THREADS ? THREADS / pieces : 1, turn = pieces < THREADS ? threadIdx.x / pieces : 0;
        for (int r0 = 3 * turn; r0 < rows_x && turn < beside; r0 += 3 * beside) {
            const T* row[3];
#pragma unroll
            for (int b = 0; b < 3; ++b) row[b] = x_row_at(min(r0 + b, rows_x - 1));
            for (int piece = threadIdx.x - turn * pieces + (asked ? 2 * THREADS : 0); piece < pieces; piece += THREADS) {
                uint4 x[3];
#pragma unroll
                for (int b = 0; b < 3; ++b)
                    if (r0 + b < rows_x) x[b] = x_get(row[b], piece);
#pragma unroll
                for (int b = 0; b < 3; ++b)
                    if (r0 + b < rows_x) x_put(r0 + b, piece, x[b]);
            }
        }
        __syncthreads();

        int x_row[NT];
        uint32_t x_base[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            x_row[n] = min(n * 8 + g, rows_x - 1);
            x_base[n] = x_all + (x_row[n] * chunks + k_warp) * (2 * X_BYTES);
        }
        int buffer = 0;
        for (int t0 = blockIdx.x * abreast; t0 < p.tiles; t0 += tile_step) {
            float total[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) total[n][0] = total[n][1] = total[n][2] = total[n][3] = 0;
            if (t0 + t_warp < p.tiles) {
                uint32_t xs[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) xs[n] = x_base[n];
                for (int u = 0; u < units; ++u) {
                    now = next;
                    q_now = q_next;
                    if (lt < p.tiles) read(next, q_next);
                    q_now.mask();
                    const int left = p.w.cols - (k_warp + (u << p.k_shift)) * CHUNK;
#pragma unroll
                    for (int s = 0; s < SEGS; ++s) {
                        if (s && s * SEG >= left) break;
                        const float scale0 = q_now.scale(0, s), scale1 = q_now.scale(1, s);
                        const auto zero0 = Decode<T>::zero(q_now.zero(0, s, zeros)), zero1 = Decode<T>::zero(q_now.zero(1, s, zeros));
                        float acc[NT][4];
#pragma unroll
                        for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0;
#pragma unroll
                        for (int j = 0; j < WORDS; ++j) {
                            uint32_t a0[4], a1[4];
                            Decode<T>::unpack(now.w[0][s * WORDS + j], zero0, a0[0], a0[2], a1[0], a1[2]);
                            Decode<T>::unpack(now.w[1][s * WORDS + j], zero1, a0[1], a0[3], a1[1], a1[3]);
                            const int in_sub = s % (SUB / SEG);  // the segment within its 128 positions
                            const int piece = SEG == 128 ? 4 * c + j : SEG == 64 ? 8 * in_sub + 2 * c + j : 4 * in_sub + c;
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                const uint4 x = lds<uint4>(xs[n] + s * SEG / SUB * X_BYTES + x_piece<SEG>(x_row[n], piece));
                                Decode<T>::mma(acc[n], a0, x.x, x.y);
                                Decode<T>::mma(acc[n], a1, x.z, x.w);
                            }
                        }
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            total[n][0] = fmaf(scale0, acc[n][0], total[n][0]);
                            total[n][1] = fmaf(scale0, acc[n][1], total[n][1]);
                            total[n][2] = fmaf(scale1, acc[n][2], total[n][2]);
                            total[n][3] = fmaf(scale1, acc[n][3], total[n][3]);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) xs[n] += (2 * X_BYTES) << p.k_shift;
                }
            }
            float* joined = red + buffer * (WARPS * NT * 128);
            buffer ^= 1;
#pragma unroll
            for (int n = 0; n < NT; ++n)
                reinterpret_cast<float4*>(joined)[(warp * NT + n) * 32 + lane] = make_float4(total[n][0], total[n][1], total[n][2], total[n][3]);
            __syncthreads();
            tiles_out<T, NT>(p, found, joined, e, t0, c0, rows_x, x0);
        }
        __syncthreads();
    }
}

template <typename T, typename S, int SEG, int NT, bool WIDE>
int launch_lean(uor_b200_ctx* ctx, FewParams& p, int cols, bool early) {
    using B = Block<NT>;
    p.columns = 8 * NT;
    p.k_shift = __builtin_ctz(B::WARPS);
    while (p.k_shift > 0 && 1 << (p.k_shift - 1) >= p.chunks) --p.k_shift;
    const int rows = p.kind == FEW_UP ? 8 : ROWS;
    p.tiles = (p.n + rows - 1) / rows;
    int64_t across = p.kind == FEW_DENSE ? (p.m + 8 * NT - 1) / (8 * NT) : static_cast<int64_t>(p.tokens) * p.top_k;
    if (p.kind != FEW_DENSE && across > p.experts) across = p.experts;
    const auto blocks_y = static_cast<unsigned>(across);
    // An expert of twice the mean has a block for each of its column tiles (8 experts of 512 x 768,
    // 16 pairs each: 27 -> 21 us), and the dealing below counts those that the mean fills.
    const int shares = few_shares(p, 8 * NT, 2);
    across *= few_shares(p, 8 * NT, 1);
    // Tiles are dealt to about as many blocks as run at one time.
    const int64_t resident = static_cast<int64_t>(ctx->sm_count) * (NT == 1 ? 2 : 1);
    auto bundles_at = [&](int shift) { return (p.tiles + (B::WARPS >> shift) - 1) / (B::WARPS >> shift); };
    // A warp with one chunk of a tile spends as long on joining it: two, where tiles abound.
    while (p.k_shift > 0 && p.chunks >> p.k_shift < 2 && bundles_at(p.k_shift - 1) * across >= resident * (NT == 1 ? 1 : 4)) --p.k_shift;
    const int64_t bundles = bundles_at(p.k_shift);
    const int64_t each = NT == 1 && bundles * across * 2 < resident * 3 ? 1 : (bundles * across + resident - 1) / resident;
    auto* kernel = lean_kernel<T, S, SEG, NT, WIDE>;
    static bool ready[64] = {};
    if (!ready[ctx->device & 63]) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, B::RED + B::X_MOST) != cudaSuccess)
            return UOR_B200_DEVICE_ERROR;
        ready[ctx->device & 63] = true;
    }
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(static_cast<unsigned>((bundles + each - 1) / each), blocks_y, shares);
    c.blockDim = dim3(B::THREADS);
    c.dynamicSmemBytes = B::RED + static_cast<size_t>(cols) * p.chunks * 2 * X_BYTES;
    c.stream = ctx->stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &attr;
    c.numAttrs = early ? 1 : 0;
    return cuda_status(cudaLaunchKernelEx(&c, kernel, p));
}

template <typename T, typename S, int SEG, bool WIDE>
bool try_lean(uor_b200_ctx* ctx, FewParams& p, bool early, int* status) {
    constexpr int N = CHUNK / SEG;
    constexpr int VEC = N * sizeof(S) < 16 ? N * sizeof(S) : 16;
    const uint64_t scales = reinterpret_cast<uint64_t>(p.w.scales) | static_cast<uint64_t>(p.w.groups_rs) * sizeof(S);
    const uint64_t zeros = p.w.zeros ? reinterpret_cast<uint64_t>(p.w.zeros) | static_cast<uint64_t>(p.w.groups_rs) : 0;
    p.quants_vec = scales % VEC == 0 && zeros % N == 0;
    p.chunks = (p.w.cols + CHUNK - 1) / CHUNK;
    p.groups = (p.w.cols + SEG - 1) / SEG;
    const int64_t most = few_columns(p);
    // Activations too many for two blocks of eight warps may fit one of sixteen (8192 x 8192 with 6
    // rows 41 -> 20 us, 2048 x 7168 with 8 17 -> 8.3).
    const bool two = most > 8 || most * p.chunks * 2 * X_BYTES > Block<1>::X_MOST;
    const int cols = static_cast<int>(two ? (most < 16 ? most : 16) : most);
    if (static_cast<int64_t>(cols) * p.chunks * 2 * X_BYTES > (two ? Block<2>::X_MOST : Block<1>::X_MOST)) return false;
    *status = two ? launch_lean<T, S, SEG, 2, WIDE>(ctx, p, cols, early) : launch_lean<T, S, SEG, 1, WIDE>(ctx, p, cols, early);
    return true;
}

template <typename T, typename S>
bool by_group(uor_b200_ctx* ctx, FewParams& p, bool early, int* status) {
    const uint64_t rows = reinterpret_cast<uint64_t>(p.w.codes) | static_cast<uint64_t>(p.w.row_bytes);
    if (rows % 4) return false;
    if (p.w.group == 128)
        return rows % 16 ? try_lean<T, S, 128, false>(ctx, p, early, status) : try_lean<T, S, 128, true>(ctx, p, early, status);
    if (p.w.group == 64)
        return rows % 8 ? try_lean<T, S, 64, false>(ctx, p, early, status) : try_lean<T, S, 64, true>(ctx, p, early, status);
    return p.w.group == 32 && try_lean<T, S, 32, true>(ctx, p, early, status);
}

template <typename T>
bool by_scales(uor_b200_ctx* ctx, int elem, FewParams& p, bool early, int* status) {
    if (p.w.scale_type == elem) return by_group<T, T>(ctx, p, early, status);
    return p.w.scale_type == UOR_B200_F32 && by_group<T, float>(ctx, p, early, status);
}

}  // namespace

bool lean_launch(uor_b200_ctx* ctx, int elem, FewParams& p, bool early, int* status) {
    if (!p.x_vec || p.w.cols % 8) return false;
    return elem == UOR_B200_BF16 ? by_scales<__nv_bfloat16>(ctx, elem, p, early, status) : by_scales<__half>(ctx, elem, p, early, status);
}

}  // namespace uor
