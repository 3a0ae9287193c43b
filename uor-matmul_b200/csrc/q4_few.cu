// q4_few.cu -- products of few rows with 4-bit weights and group scales.
//
// Bound by the weights' bytes, read once: 4 bits and a share of a scale each. A CTA takes tiles of
// 16 rows of weights, one after another, and its warps split a tile's reduction into chunks of 256
// positions (128 bytes of a row), neighbouring warps taking neighbouring chunks. Each warp keeps a
// ring of chunks of codes in flight with cp.async, in shared memory of its own and across the
// tiles, so no warp waits for another but where a tile's sums are joined. A chunk's scales and
// zero points travel in registers one chunk ahead; the activations are laid out in shared memory
// once, while the first chunks travel.
//
// The products run on the tensor cores (mma.m16n8k16) with the weights as the 16 rows and up to 8
// or 16 activation rows as the columns, since CUDA cores could not multiply at the rate the codes
// arrive at from four rows on. A code is exact as a 16-bit float: its bits under the exponent of
// 128 (bfloat16, in units of 2^-12) or 1024 (float16), less the same plus the zero point: the old
// conversion of small integers by a float whose unit they are. So the sum of a group is
// exact but for its f32 additions, and the group's scale multiplies it in f32: no weight is ever
// rounded. The reduction's order within a group is free, so a lane's 16 bytes are taken as they
// lie: word j of lane c holds positions 32 c + 8 j .. + 7, and the instruction's operands are its
// nibbles (0, 4), (1, 5) | (2, 6), (3, 7). The activations lie in shared memory in that order:
// every eight as 0 4 1 5 2 6 3 7.
//
// 8 x 5003 x 4008 in groups of 96: 27.0 us, with zero points 29.7. Beside the memory it is
// instructions and their latency, 47 % of the issue slots with four warps a scheduler: 11 to unpack
// eight weights of bfloat16 (three shifts, four and-or, four subtractions), so addresses, scales and
// their types are kept out of the loop. Three blocks of eight warps leave 80 registers a thread, of
// which every instance spills 8 to 168 bytes.
//
// With experts a CTA finds the pairs (token, choice) of one of them by looking through all ids:
// its columns are these pairs' activation rows.
#include "q4_few.cuh"

#include "ptx.cuh"
#include "q4_mma.cuh"

namespace uor {

namespace {

constexpr int STAGES = 2;
constexpr int HALF_BYTES = ROWS * SUB / 2;     // of a stage's codes, per SUB
constexpr int PITCH_ANY = 144;                 // of a row's codes whose addresses are not aligned

template <bool ANY>
constexpr int stage_bytes() {
    return ANY ? ROWS * PITCH_ANY : 2 * HALF_BYTES;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Where 16-byte piece c of a row's 64 bytes of codes lies: eight rows' reads of any width meet no
// bank twice.
__device__ __forceinline__ int code_at(int row, int c) {
    return row * 64 + ((c ^ ((row & 2) | ((row >> 2) & 1))) << 4);
}
// One warp's ring of chunks of codes.
template <typename T, typename S, int SEG, bool ANY>
struct Ring {
    static constexpr int NSEG = SUB / SEG;
    uint32_t base;               // shared address of stage 0
    const uint8_t* row[ANY ? 2 : 4];  // this lane's rows of codes: its pieces' (lane / 8 + 4 v), or g and g + 8
    int row_len;

    __device__ __forceinline__ void set(const FewParams& p, int lane, const Tile& t) {
        if constexpr (ANY) {
            row[0] = p.w.codes + t.row(lane >> 2) * p.w.row_bytes, row[1] = p.w.codes + t.row((lane >> 2) + 8) * p.w.row_bytes;
        } else {
#pragma unroll
            for (int v = 0; v < 4; ++v) row[v] = p.w.codes + t.row((lane >> 3) + 4 * v) * p.w.row_bytes + 16 * (lane & 7);
        }
    }

    __device__ __forceinline__ void load(int stage, int chunk, int lane) const {
        const uint32_t at = base + stage * stage_bytes<ANY>();
        const int from = chunk * (CHUNK / 2);
        const int left = row_len - chunk * (CHUNK / 2);  // bytes of the row from here
        if constexpr (!ANY) {
            const int c = lane & 7;
            const uint32_t dst = at + (c >> 2) * HALF_BYTES;
            if (left >= CHUNK / 2) {
#pragma unroll
                for (int v = 0; v < 4; ++v) cp_async16(dst + code_at((lane >> 3) + 4 * v, c & 3), row[v] + from, 16);
            } else {
                const int n = max(0, min(16, left - 16 * c));
#pragma unroll
                for (int v = 0; v < 4; ++v)
                    cp_async16(dst + code_at((lane >> 3) + 4 * v, c & 3), n ? row[v] + from : row[v] - 16 * c, n);
            }
        } else {
            // the 33 aligned words that cover 128 bytes from any address; none past the row's end
#pragma unroll 1
            for (int v = 0; v < 2; ++v) {
                const uint8_t* s = row[v] + from;
                const int past = static_cast<int>(reinterpret_cast<uint64_t>(s) & 3);
                const int have = min(CHUNK / 2, left) + past;
                for (int w = lane & 3; 4 * w < have; w += 4)
                    cp_async4(at + ((lane >> 2) + 8 * v) * PITCH_ANY + 4 * w, s - past + 4 * w, min(4, have - 4 * w));
            }
        }
    }

    // sum += the products of one half of the chunk (`sub`). xs: the half's activations of this
    // lane's columns of the instructions (rows x_row of them); left: positions that exist;
    // m0, m1: how far past a word the lane's two rows of codes begin, in bits.
    template <int NT>
    __device__ __forceinline__ void compute(int stage, int sub, int lane, const Quants<T, S, SEG>& q, bool zeros, int m0, int m1,
                                            const uint32_t (&xs)[NT], const int (&x_row)[NT], int left, float (&sum)[NT][4]) const {
        const uint32_t codes = base + stage * stage_bytes<ANY>() + (ANY ? sub * 64 : sub * HALF_BYTES);
        const int g = lane >> 2, c = lane & 3;
#pragma unroll
        for (int s = 0; s < NSEG; ++s) {
            if (NSEG > 1 && s * SEG >= left) break;
            const float scale0 = q.scale(0, sub * NSEG + s), scale1 = q.scale(1, sub * NSEG + s);
            const auto zero0 = Decode<T>::zero(q.zero(0, sub * NSEG + s, zeros));
            const auto zero1 = Decode<T>::zero(q.zero(1, sub * NSEG + s, zeros));
            constexpr int WORDS = SEG / 32;
            uint32_t w0[4], w1[4];
            if constexpr (ANY) {
                const int word = SEG == 128 ? 4 * c : SEG == 64 ? 8 * s + 2 * c : 4 * s + c;
                const uint32_t a0 = codes + g * PITCH_ANY + 4 * word, a1 = a0 + 8 * PITCH_ANY;
                uint32_t n0 = lds<uint32_t>(a0), n1 = lds<uint32_t>(a1);
#pragma unroll
                for (int j = 0; j < WORDS; ++j) {
                    const uint32_t f0 = lds<uint32_t>(a0 + 4 * j + 4), f1 = lds<uint32_t>(a1 + 4 * j + 4);
                    w0[j] = __funnelshift_r(n0, f0, m0), w1[j] = __funnelshift_r(n1, f1, m1);
                    n0 = f0, n1 = f1;
                }
            } else if constexpr (SEG == 128) {
                const uint32_t a = codes + code_at(g, c);
                const uint4 v0 = lds<uint4>(a), v1 = lds<uint4>(a + 8 * 64);
                w0[0] = v0.x, w0[1] = v0.y, w0[2] = v0.z, w0[3] = v0.w;
                w1[0] = v1.x, w1[1] = v1.y, w1[2] = v1.z, w1[3] = v1.w;
            } else if constexpr (SEG == 64) {
                const uint32_t a = codes + code_at(g, 2 * s + (c >> 1)) + (c & 1) * 8;
                const uint2 v0 = lds<uint2>(a), v1 = lds<uint2>(a + 8 * 64);
                w0[0] = v0.x, w0[1] = v0.y, w1[0] = v1.x, w1[1] = v1.y;
            } else {
                const uint32_t a = codes + code_at(g, s) + c * 4;
                w0[0] = lds<uint32_t>(a), w1[0] = lds<uint32_t>(a + 8 * 64);
            }
            float acc[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0;
#pragma unroll
            for (int j = 0; j < WORDS; ++j) {
                uint32_t a0[4], a1[4];
                Decode<T>::unpack(w0[j], zero0, a0[0], a0[2], a1[0], a1[2]);
                Decode<T>::unpack(w1[j], zero1, a0[1], a0[3], a1[1], a1[3]);
                const int piece = SEG == 128 ? 4 * c + j : SEG == 64 ? 8 * s + 2 * c + j : 4 * s + c;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint4 x = lds<uint4>(xs[n] + sub * X_BYTES + x_piece<SEG>(x_row[n], piece));
                    Decode<T>::mma(acc[n], a0, x.x, x.y);
                    Decode<T>::mma(acc[n], a1, x.z, x.w);
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                sum[n][0] = fmaf(scale0, acc[n][0], sum[n][0]);
                sum[n][1] = fmaf(scale0, acc[n][1], sum[n][1]);
                sum[n][2] = fmaf(scale1, acc[n][2], sum[n][2]);
                sum[n][3] = fmaf(scale1, acc[n][3], sum[n][3]);
            }
        }
    }
};

template <typename T, typename S, int SEG, int NT, bool ANY>
__global__ void __launch_bounds__(Block<NT>::THREADS, NT == 1 ? 3 : 1) few_kernel(const __grid_constant__ FewParams p) {
    constexpr int WARPS = Block<NT>::WARPS, THREADS = Block<NT>::THREADS, COLS = 8 * NT;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Found found;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int chunks = p.chunks, kind = p.kind;
    if (kind != FEW_DENSE) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // The columns: activation rows from x0 on, or of the listed pairs of expert e.
    int e = 0, listed = 0;
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

    // `kw` warps share a tile's reduction, so WARPS / kw tiles are under way at once.
    const int kw = 1 << p.k_shift, k_warp = warp & (kw - 1), t_warp = warp >> p.k_shift, abreast = WARPS >> p.k_shift;
    const int tiles = p.tiles;
    Ring<T, S, SEG, ANY> ring;
    ring.base = smem_u32(smem) + warp * (STAGES * stage_bytes<ANY>());
    ring.row_len = (p.w.cols + 1) / 2;
    float* red = reinterpret_cast<float*>(smem + WARPS * STAGES * stage_bytes<ANY>());
    const uint32_t x_all = smem_u32(smem) + WARPS * STAGES * stage_bytes<ANY>() + Block<NT>::RED;
    const int groups = p.groups;
    const bool zeros = p.w.zeros != nullptr;
    const int panel = p.panel, panels = p.panels;  // chunks whose activations are resident
    const int tile_step = gridDim.x * abreast;
    bool waited = kind != FEW_PART;

    for (int c0 = blockIdx.z * COLS; c0 < listed; c0 += gridDim.z * COLS) {
        const int rows_x = min(COLS, listed - c0);
        int x_row[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) x_row[n] = min(n * 8 + (lane >> 2), rows_x - 1);
        int buffer = 0;
        // A warp's units: of each of its tiles in turn, of each panel, chunks k_warp, k_warp + kw, ..
        int lt = blockIdx.x * abreast + t_warp, lpanel = 0, lc = k_warp, lstage = 0;  // the next to load
        auto settle = [&]() {  // past the end of a panel or a tile
            while (lt < tiles && lc >= min(chunks, (lpanel + 1) * panel)) {
                if (++lpanel == panels) {
                    lpanel = 0;
                    lt += tile_step;
                    if (lt < tiles) ring.set(p, lane, tile_at(p, e, lt));
                }
                lc = lpanel * panel + k_warp;
            }
        };
        auto load = [&]() {
            if (lt < tiles) {
                ring.load(lstage, lc, lane);
                lc += kw;
                settle();
            }
            lstage = lstage + 1 == STAGES ? 0 : lstage + 1;
            cp_commit();
        };
        if (lt < tiles) ring.set(p, lane, tile_at(p, e, lt));
        settle();
        // The weights depend on nothing before this launch; the inner activations do.
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s) load();
        if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");
        waited = true;
        int stage = 0;
        for (int t0 = blockIdx.x * abreast; t0 < tiles; t0 += tile_step) {
            const int t = t0 + t_warp;
            const Tile tile = tile_at(p, e, t);
            const int64_t r0 = tile.row(lane >> 2), r1 = tile.row((lane >> 2) + 8);
            const int64_t quants0 = r0 * p.w.groups_rs, quants1 = r1 * p.w.groups_rs;
            int m0 = 0, m1 = 0;
            if constexpr (ANY) {
                m0 = 8 * static_cast<int>((reinterpret_cast<uint64_t>(p.w.codes) + r0 * p.w.row_bytes) & 3);
                m1 = 8 * static_cast<int>((reinterpret_cast<uint64_t>(p.w.codes) + r1 * p.w.row_bytes) & 3);
            }
            float total[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) total[n][0] = total[n][1] = total[n][2] = total[n][3] = 0;
            for (int pn = 0; pn < panels; ++pn) {
                const int first = pn * panel, last = min(chunks, first + panel);
                const int units = t < tiles && last - first > k_warp ? (last - first - k_warp + kw - 1) >> p.k_shift : 0;
                Quants<T, S, SEG> now, next;
                if (units) now.load(p, quants0, quants1, first + k_warp, groups);
                if (panels > 1 || t0 == static_cast<int>(blockIdx.x) * abreast) {
                    __syncthreads();  // every warp is done with the activations before these
                    const int pieces = (last - first) * 32;
                    for (int v0 = threadIdx.x; v0 < rows_x * pieces; v0 += 4 * THREADS) {
                        uint4 x8[4];
#pragma unroll
                        for (int b = 0; b < 4; ++b) {
                            const int v = min(v0 + b * THREADS, rows_x * pieces - 1);
                            const int r = rows_x == 1 ? 0 : v / pieces, k = first * CHUNK + (v - r * pieces) * 8;
                            const int64_t row = x_row_of(p, found, x0, c0 + r);
                            // rows of inner activations end in whole eights
                            const int left = kind == FEW_PART ? (k < p.x_rs ? 8 : 0) : p.w.cols - k;
                            x8[b] = load_x8(static_cast<const T*>(p.x) + row * p.x_rs + (left > 0 ? k : 0), left, p.x_vec != 0);
                        }
#pragma unroll
                        for (int b = 0; b < 4; ++b) {
                            const int v = v0 + b * THREADS;
                            const int r = rows_x == 1 ? 0 : v / pieces, piece = v - r * pieces;
                            if (v < rows_x * pieces)
                                sts128(x_all + (r * panel * 2 + (piece >> 4)) * X_BYTES + x_piece<SEG>(r, piece & 15),
                                       kind == FEW_PART ? x8[b] : in_pairs(x8[b]));
                        }
                    }
                    __syncthreads();
                }
                uint32_t xs[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) xs[n] = x_all + (x_row[n] * panel + k_warp) * (2 * X_BYTES);
                int c = first + k_warp;
                for (int i = 0; i < units; ++i, c += kw) {
                    cp_wait<STAGES - 2>();
                    __syncwarp();
                    load();
                    if (i + 1 < units) next.load(p, quants0, quants1, c + kw, groups);
                    const int left = p.w.cols - c * CHUNK;
                    now.mask();
                    ring.compute(stage, 0, lane, now, zeros, m0, m1, xs, x_row, left, total);
                    if (left > SUB) ring.compute(stage, 1, lane, now, zeros, m0, m1, xs, x_row, left - SUB, total);
                    stage = stage + 1 == STAGES ? 0 : stage + 1;
#pragma unroll
                    for (int n = 0; n < NT; ++n) xs[n] += kw * (2 * X_BYTES);
                    now = next;
                }
            }
            // Join the warps' sums, [warp][column eight][lane][4], in the warps' order.
            float* joined = red + buffer * (WARPS * NT * 128);
            buffer ^= 1;
#pragma unroll
            for (int n = 0; n < NT; ++n)
                reinterpret_cast<float4*>(joined)[(warp * NT + n) * 32 + lane] = make_float4(total[n][0], total[n][1], total[n][2], total[n][3]);
            __syncthreads();
            tiles_out<T, NT>(p, found, joined, e, t0, c0, rows_x, x0);
        }
        cp_wait<0>();
        __syncthreads();
    }
}

template <typename T, typename S, int SEG, int NT, bool ANY>
int launch_few(uor_b200_ctx* ctx, FewParams& p, bool early) {
    using B = Block<NT>;
    p.columns = 8 * NT;
    const int chunks = p.chunks = (p.w.cols + CHUNK - 1) / CHUNK;
    p.groups = (p.w.cols + p.w.group - 1) / p.w.group;
    int64_t cols = few_columns(p);  // of a block, at most
    if (cols > 8 * NT) cols = 8 * NT;
    p.group_shift = (p.w.group & (p.w.group - 1)) == 0 ? __builtin_ctz(p.w.group) : -1;
    constexpr int N = CHUNK / SEG;
    constexpr int VEC = N * sizeof(S) < 16 ? N * sizeof(S) : 16;
    p.quants_vec = p.w.group == SEG && (sizeof(S) == 2 || p.w.scale_type == UOR_B200_F32) &&
                   (reinterpret_cast<uint64_t>(p.w.scales) | static_cast<uint64_t>(p.w.groups_rs) * sizeof(S)) % VEC == 0 &&
                   (reinterpret_cast<uint64_t>(p.w.zeros) | (p.w.zeros ? static_cast<uint64_t>(p.w.groups_rs) : 0)) % N == 0;
    p.panel = static_cast<int>(B::X_MOST / (cols * 2 * X_BYTES));
    if (p.panel > chunks) p.panel = chunks;
    p.panels = (chunks + p.panel - 1) / p.panel;
    p.k_shift = __builtin_ctz(B::WARPS);
    while (p.k_shift > 0 && 1 << (p.k_shift - 1) >= p.panel) --p.k_shift;
    constexpr int FIXED = B::WARPS * STAGES * stage_bytes<ANY>() + B::RED;
    auto* kernel = few_kernel<T, S, SEG, NT, ANY>;
    static bool ready[64] = {};
    if (!ready[ctx->device & 63]) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, FIXED + B::X_MOST) != cudaSuccess)
            return UOR_B200_DEVICE_ERROR;
        ready[ctx->device & 63] = true;
    }
    // Tiles are dealt to about as many blocks as run at one time.
    const int rows = p.kind == FEW_UP ? 8 : ROWS, abreast = B::WARPS >> p.k_shift;
    p.tiles = (p.n + rows - 1) / rows;
    const int64_t bundles = (p.tiles + abreast - 1) / abreast;
    int64_t across = p.kind == FEW_DENSE ? (p.m + 8 * NT - 1) / (8 * NT) : static_cast<int64_t>(p.tokens) * p.top_k;
    if (p.kind != FEW_DENSE && across > p.experts) across = p.experts;
    const auto blocks_y = static_cast<unsigned>(across);
    // An expert of twice the mean has a block for each of its column tiles (8 experts of 512 x 768,
    // 16 pairs each: 27 -> 21 us), and the dealing below counts those that the mean fills.
    const int shares = few_shares(p, 8 * NT, 2);
    across *= few_shares(p, 8 * NT, 1);
    const int64_t resident = static_cast<int64_t>(ctx->sm_count) * (NT == 1 ? 3 : 1);
    const int64_t each = (bundles * across + resident - 1) / resident;
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(static_cast<unsigned>((bundles + each - 1) / each), blocks_y, shares);
    c.blockDim = dim3(B::THREADS);
    c.dynamicSmemBytes = FIXED + cols * p.panel * 2 * X_BYTES;
    c.stream = ctx->stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &attr;
    c.numAttrs = early ? 1 : 0;
    return cuda_status(cudaLaunchKernelEx(&c, kernel, p));
}

// The segment is what one scale covers within 128 positions: the largest of 128, 64 and 32 that
// divides the group.
template <typename T, typename S, int NT, bool ANY>
int by_segment(uor_b200_ctx* ctx, FewParams& p, bool early) {
    if (p.w.group % 128 == 0) return launch_few<T, S, 128, NT, ANY>(ctx, p, early);
    if (p.w.group % 64 == 0) return launch_few<T, S, 64, NT, ANY>(ctx, p, early);
    return launch_few<T, S, 32, NT, ANY>(ctx, p, early);
}

// Eight columns, or sixteen where there are more rows than eight. Rows of codes that do not all
// begin at multiples of 16 bytes are copied by words and shifted into place; scales that are
// neither float nor of the activations' type are converted as they are read.
template <typename T, typename S, bool ANY>
int by_columns(uor_b200_ctx* ctx, FewParams& p, bool early) {
    // Where the activations leave room for one or two blocks of eight warps, one of sixteen hides
    // more (5003 x 4008 with 8 rows 47 -> 27 us, 300 x 12000 with 4 31 -> 13); one row would pay for
    // fifteen others' columns.
    const int64_t bytes = few_columns(p) * ((p.w.cols + CHUNK - 1) / CHUNK) * 2 * X_BYTES;
    return few_columns(p) > 8 || (few_columns(p) > 1 && bytes > Block<1>::X_MOST / 4) ? by_segment<T, S, 2, ANY>(ctx, p, early) : by_segment<T, S, 1, ANY>(ctx, p, early);
}
template <typename T>
int by_codes(uor_b200_ctx* ctx, int elem, FewParams& p, bool early) {
    if (p.codes_align != 16) return by_columns<T, float, true>(ctx, p, early);
    if (p.w.scale_type == elem) return by_columns<T, T, false>(ctx, p, early);
    return by_columns<T, float, false>(ctx, p, early);
}

}  // namespace

int few_launch(uor_b200_ctx* ctx, int elem, FewParams& p, bool early) {
    int st = UOR_B200_OK;
    if (lean_launch(ctx, elem, p, early, &st)) return st;
    return elem == UOR_B200_BF16 ? by_codes<__nv_bfloat16>(ctx, elem, p, early) : by_codes<__half>(ctx, elem, p, early);
}

}  // namespace uor
