// q4_gemm.cu -- 4-bit weights with group scales and the experts' layer: which kernels a call runs,
// and the small ones around the products (rows brought together, choices sorted, parts added).
#include <cstring>

#include "q4.cuh"
#include "q4_few.cuh"
#include "q4_many.cuh"

namespace uor {

namespace {

// A kernel that begins while the one before it in the call still runs: it waits for that one's
// results here, and lets the next begin as its blocks leave.
__device__ __forceinline__ void follow() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

constexpr int THREADS = 256;
constexpr int ROWS_EACH = 4;

// Rows of x, strided anyhow, as contiguous ones of `pitch` elements; row i is x's row
// perm[i] / top_k where there is a permutation, and then only offsets[experts] rows exist.
// Eight elements to a thread, four times side by side.
__global__ void __launch_bounds__(THREADS) rows_kernel(Mat x, int cols, int pitch, int64_t rows, const int* perm, int top_k,
                                                       const int* total, bool vec, uint16_t* to) {
    follow();
    const int per_row = pitch / 8;
    const int64_t exist = total ? min(static_cast<int64_t>(*total), rows) : rows;
    int64_t i[ROWS_EACH];
    int c[ROWS_EACH];
    const uint16_t* from[ROWS_EACH];
    // one long division a block: the rest is within 32 bits
    const int64_t begin = static_cast<int64_t>(blockIdx.x) * (ROWS_EACH * THREADS), i0 = begin / per_row;
    const uint32_t c0 = static_cast<uint32_t>(begin - i0 * per_row) + threadIdx.x;
#pragma unroll
    for (int b = 0; b < ROWS_EACH; ++b) {
        const uint32_t at = c0 + b * THREADS, down = at / static_cast<uint32_t>(per_row);
        i[b] = i0 + down;
        c[b] = static_cast<int>(at - down * per_row) * 8;
        const int64_t row = i[b] >= exist ? 0 : perm ? perm[i[b]] / top_k : i[b];
        from[b] = static_cast<const uint16_t*>(x.p) + row * x.rs;
    }
    uint4 v[ROWS_EACH];
#pragma unroll
    for (int b = 0; b < ROWS_EACH; ++b) {
        if (i[b] >= exist) continue;
        if (vec && c[b] + 8 <= cols) {
            v[b] = *reinterpret_cast<const uint4*>(from[b] + c[b]);
        } else {
            uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c[b] + e < cols) w[e >> 1] |= static_cast<uint32_t>(from[b][(c[b] + e) * x.cs]) << (16 * (e & 1));
            v[b] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
#pragma unroll
    for (int b = 0; b < ROWS_EACH; ++b)
        if (i[b] < exist) *reinterpret_cast<uint4*>(to + i[b] * pitch + c[b]) = v[b];
}

// Rows of codes at any address and distance as rows of `pitch` bytes, a multiple of 16.
__global__ void codes_kernel(const uint8_t* codes, int64_t row_bytes, int64_t rows, int row_len, int pitch, uint8_t* to) {
    const int per_row = pitch / 16;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    const int64_t i = at / per_row;
    if (i >= rows) return;
    const int c = static_cast<int>(at - i * per_row) * 16;
    const uint8_t* from = codes + i * row_bytes + c;
    uint32_t w[4] = {0, 0, 0, 0};
    if (c + 19 <= row_len) {  // five aligned words hold the sixteen bytes, and end within the row
        const int past = static_cast<int>(reinterpret_cast<uint64_t>(from) & 3);
        const uint32_t* a = reinterpret_cast<const uint32_t*>(from - past);
        uint32_t v[5];
#pragma unroll
        for (int b = 0; b < 4; ++b) v[b] = a[b];
        v[4] = past ? a[4] : 0;
#pragma unroll
        for (int b = 0; b < 4; ++b) w[b] = __funnelshift_r(v[b], v[b + 1], 8 * past);
    } else {
#pragma unroll
        for (int b = 0; b < 16; ++b)
            if (c + b < row_len) w[b >> 2] |= static_cast<uint32_t>(from[b]) << (8 * (b & 3));
    }
    *reinterpret_cast<uint4*>(to + i * pitch + c) = make_uint4(w[0], w[1], w[2], w[3]);
}

constexpr int SORT_THREADS = 1024, SORT_BATCH = 8;

// The pairs (token, choice) of one expert per block, in their own order, behind those of the
// experts before it: offsets[e] counts the pairs of lower experts. Ids outside the experts have
// no place. Every warp counts and then places a run of pairs of its own, 32 abreast and eight
// times 32 under way (8192 pairs among 32 experts: 5.8 us).
__global__ void __launch_bounds__(SORT_THREADS) sort_kernel(Mat ids, int pairs, int top_k, int experts, int* offsets, int* perm) {
    constexpr int WARPS = SORT_THREADS / 32;
    __shared__ int warp_less[WARPS], warp_same[WARPS];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int e = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int run = (pairs + SORT_THREADS - 1) / SORT_THREADS * 32;
    const int first = min(pairs, warp * run), last = min(pairs, first + run);
    auto read = [&](int at, int (&v)[SORT_BATCH]) {
#pragma unroll
        for (int b = 0; b < SORT_BATCH; ++b) {
            const int i = at + b * 32 + lane, t = i / top_k;
            v[b] = i < last ? static_cast<const int32_t*>(ids.p)[t * ids.rs + (i - t * top_k) * ids.cs] : -1;
        }
    };
    int less = 0, same = 0, v[SORT_BATCH];
    for (int at = first; at < last; at += 32 * SORT_BATCH) {
        read(at, v);
#pragma unroll
        for (int b = 0; b < SORT_BATCH; ++b) {
            less += v[b] >= 0 && v[b] < e;
            same += v[b] == e;
        }
    }
    less = __reduce_add_sync(0xffffffffu, less);
    same = __reduce_add_sync(0xffffffffu, same);
    if (lane == 0) warp_less[warp] = less, warp_same[warp] = same;
    __syncthreads();
    const int begin = __reduce_add_sync(0xffffffffu, warp_less[lane]), all = __reduce_add_sync(0xffffffffu, warp_same[lane]);
    int to = begin + __reduce_add_sync(0xffffffffu, lane < warp ? warp_same[lane] : 0);
    if (threadIdx.x == 0) {
        offsets[e] = begin;
        if (e == experts - 1) offsets[experts] = begin + all;
    }
    if (!same) return;
    for (int at = first; at < last; at += 32 * SORT_BATCH) {
        if (last - first > 32 * SORT_BATCH) read(at, v);  // else they are at hand
#pragma unroll
        for (int b = 0; b < SORT_BATCH; ++b) {
            const uint32_t mine = __ballot_sync(0xffffffffu, v[b] == e);
            if (v[b] == e) perm[to + __popc(mine & ((1u << lane) - 1))] = at + b * 32 + lane;
            to += __popc(mine);
        }
    }
}
static_assert(SORT_THREADS == 1024, "a lane for each warp's counts");

// Four neighbouring outputs of a row; one by one where they do not lie as a vector.
__device__ __forceinline__ void store4(const MatOut& y, int64_t i, int j, int n, const float (&v)[4]) {
    const int64_t at = i * y.rs + j * y.cs;
    char* to = static_cast<char*>(y.p) + at * (y.type == UOR_B200_F32 ? 4 : 2);
    if (j + 4 <= n && y.cs == 1 && reinterpret_cast<uint64_t>(to) % (y.type == UOR_B200_F32 ? 16 : 8) == 0) {
        if (y.type == UOR_B200_F32) {
            *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
        } else if (y.type == UOR_B200_BF16) {
            const __nv_bfloat162 t[2] = {__floats2bfloat162_rn(v[0], v[1]), __floats2bfloat162_rn(v[2], v[3])};
            memcpy(to, t, 8);
        } else {
            const __half2 t[2] = {__floats2half2_rn(v[0], v[1]), __floats2half2_rn(v[2], v[3])};
            memcpy(to, t, 8);
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (j + k < n) store_f32(y.p, at + k * y.cs, y.type, v[k]);
}
// Four neighbouring f32 of a row of n, zeros past its end.
__device__ __forceinline__ float4 load4(const float* row, int j, int n, bool vec) {
    if (vec && j + 4 <= n) return *reinterpret_cast<const float4*>(row + j);
    return make_float4(j < n ? row[j] : 0.0f, j + 1 < n ? row[j + 1] : 0.0f, j + 2 < n ? row[j + 2] : 0.0f,
                       j + 3 < n ? row[j + 3] : 0.0f);
}

// y[i][j] = the parts' sum, in their order (no parts: 0). A block's x takes 1024 outputs of a
// row, its y strides the rows.
__global__ void add_parts_kernel(const float* part, int splits, int64_t rows, int n, MatOut y) {
    follow();
    const int j = (blockIdx.x * blockDim.x + threadIdx.x) * 4;
    if (j >= n) return;
    for (int64_t i = blockIdx.y; i < rows; i += gridDim.y) {
        float v[4] = {0, 0, 0, 0};
        for (int s = 0; s < splits; ++s) {
            const float4 a = load4(part + (s * rows + i) * n, j, n, n % 4 == 0);
            v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w;
        }
        store4(y, i, j, n, v);
    }
}

// y[t][j] = the token's choices' products, each times its weight, in the choices' order. once: a
// token's second choice of an expert has no product of its own, it is the first's. AT: choices that
// are read at a time; four where there are no more, which halves the registers (2048 tokens, 4
// choices of 2048: 35 -> 21 us).
template <int AT>
__global__ void __launch_bounds__(256) combine_kernel(const float* part, int splits, bool once, const __grid_constant__ FfnArgs a) {
    const int j = (blockIdx.x * blockDim.x + threadIdx.x) * 4;
    if (j >= a.d) return;  // with nothing read or written, there is nothing to wait for
    const int64_t step = a.tokens * a.top_k;
    const auto* ids = static_cast<const int32_t*>(a.ids.p);
    const auto* weights = static_cast<const float*>(a.weights.p);
    bool waited = false;
    for (int64_t t = blockIdx.y; t < a.tokens; t += gridDim.y) {
        float v[4] = {0, 0, 0, 0};
        for (int s0 = 0; s0 < a.top_k; s0 += AT) {
            int e[AT], from[AT];
            float w[AT];
            float4 sum[AT];
#pragma unroll
            for (int b = 0; b < AT; ++b) {
                e[b] = s0 + b < a.top_k ? ids[t * a.ids.rs + (s0 + b) * a.ids.cs] : -1;
                w[b] = s0 + b < a.top_k ? weights[t * a.weights.rs + (s0 + b) * a.weights.cs] : 0.0f;
                if (e[b] >= a.experts) e[b] = -1;
            }
#pragma unroll
            for (int b = 0; b < AT; ++b) {
                from[b] = s0 + b;
                if (once && e[b] >= 0) {
#pragma unroll
                    for (int o = b - 1; o >= 0; --o)
                        if (e[o] == e[b]) from[b] = s0 + o;
                    for (int o = s0 - 1; o >= 0; --o)
                        if (ids[t * a.ids.rs + o * a.ids.cs] == e[b]) from[b] = o;
                }
            }
            if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");
            waited = true;
#pragma unroll
            for (int b = 0; b < AT; ++b)
                if (e[b] >= 0) sum[b] = load4(part + (t * a.top_k + from[b]) * a.d, j, a.d, a.d % 4 == 0);
#pragma unroll
            for (int b = 0; b < AT; ++b) {
                if (e[b] < 0) continue;
                for (int c = 1; c < splits; ++c) {
                    const float4 more = load4(part + (c * step + t * a.top_k + from[b]) * a.d, j, a.d, a.d % 4 == 0);
                    sum[b].x += more.x, sum[b].y += more.y, sum[b].z += more.z, sum[b].w += more.w;
                }
                v[0] = fmaf(w[b], sum[b].x, v[0]), v[1] = fmaf(w[b], sum[b].y, v[1]);
                v[2] = fmaf(w[b], sum[b].z, v[2]), v[3] = fmaf(w[b], sum[b].w, v[3]);
            }
        }
        store4(a.y, t, j, a.d, v);
    }
}

// Four outputs to a thread, a row to a block's y.
dim3 blocks_of_rows(int64_t rows, int n) {
    return dim3((n + 4 * THREADS - 1) / (4 * THREADS), static_cast<unsigned>(rows < 65535 ? rows : 65535));
}
// A launch of THREADS to a block; early: it may begin while the kernel before it still runs, whose
// results it waits for itself.
template <typename... P, typename... A>
int launch(uor_b200_ctx* ctx, dim3 grid, bool early, void (*kernel)(P...), const A&... args) {
    cudaLaunchConfig_t c = {};
    c.gridDim = grid;
    c.blockDim = dim3(THREADS);
    c.stream = ctx->stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &attr;
    c.numAttrs = early ? 1 : 0;
    return cuda_status(cudaLaunchKernelEx(&c, kernel, static_cast<P>(args)...));
}
unsigned blocks_for(int64_t threads) { return static_cast<unsigned>((threads + THREADS - 1) / THREADS); }

int up_to(int v, int by) { return (v + by - 1) / by * by; }

bool rows_aligned(const void* p, int64_t stride_bytes) {
    return (reinterpret_cast<uint64_t>(p) | static_cast<uint64_t>(stride_bytes)) % 16 == 0;
}

// What the kernels with TMA read must lie in rows of whole 16 bytes that do not overlap.
bool x_in_place(const Mat& x, int cols) { return x.cs == 1 && rows_aligned(x.p, x.rs * 2) && x.rs >= cols; }
bool codes_in_place(const Q4Dev& w) {
    return rows_aligned(w.codes, w.row_bytes) && w.row_bytes >= (w.cols + 1) / 2 && w.row_bytes < (int64_t(1) << 40);
}

// A call's pieces of the context's workspace.
class Pieces {
  public:
    size_t add(size_t bytes) {
        const size_t at = total_;
        total_ += (bytes + 1023) / 1024 * 1024;
        return at;
    }
    uint8_t* get(uor_b200_ctx* ctx, int* st) { return static_cast<uint8_t*>(ctx_buffer(ctx, SLOT_WS, total_, st)); }

  private:
    size_t total_ = 0;
};

size_t codes_copy_bytes(const Q4Dev& w) {
    return codes_in_place(w) ? 0 : static_cast<size_t>(w.rows) * up_to((w.cols + 1) / 2, 16);
}
void copy_codes(uor_b200_ctx* ctx, Q4Dev* w, uint8_t* to) {
    if (codes_in_place(*w)) return;
    const int pitch = up_to((w->cols + 1) / 2, 16);
    codes_kernel<<<blocks_for(static_cast<int64_t>(w->rows) * (pitch / 16)), THREADS, 0, ctx->stream>>>(
        w->codes, w->row_bytes, w->rows, (w->cols + 1) / 2, pitch, to);
    w->codes = to;
    w->row_bytes = pitch;
}
// early: after a kernel of the same call, and may begin while that one still runs.
void copy_rows(uor_b200_ctx* ctx, const Mat& x, int cols, int64_t rows, const int* perm, int top_k, const int* total, void* to,
               bool early) {
    const int pitch = up_to(cols, 8);
    launch(ctx, dim3(blocks_for((rows * (pitch / 8) + ROWS_EACH - 1) / ROWS_EACH)), early, rows_kernel, x, cols, pitch, rows, perm,
           top_k, total, x.cs == 1 && rows_aligned(x.p, x.rs * 2), static_cast<uint16_t*>(to));
}

// What the few-rows kernel's vector loads may rely on.
void few_align(FewParams* p) {
    p->codes_align = rows_aligned(p->w.codes, p->w.row_bytes) ? 16 : 1;
    p->x_vec = rows_aligned(p->x, p->x_rs * 2);
}

// few: after the few-rows kernel, which wrote a token's products with an expert once.
int launch_combine(uor_b200_ctx* ctx, const float* part, int splits, const FfnArgs& a, bool few) {
    return launch(ctx, blocks_of_rows(a.tokens, a.d), true, a.top_k <= 4 ? combine_kernel<4> : combine_kernel<8>, part, splits, few,
                  a);
}

// The few-rows kernel's 16 columns at a time against the tensor-memory kernel's 256 (which starts
// slower, takes rows as TMA can read them, and with experts has them sorted and copied first).
// Times in us, few : many.
//
// Dense: while the activations of a pass stay in shared memory, few rows are the weights' reading
// (8192 x 8192 with 6 rows 20 : 30, 4096 x 4096 with 12 9 : 16, 5003 x 4008 at odd addresses with 8
// 27 : 34), and else not (8192 x 8192 with 8 53 : 30, 4096 x 4096 with 16 25 : 17). Small products
// fit the processors many passes abreast: 2048 x 2048 with 64 rows 9.4 : 15.0, 128 14.6 : 17.8,
// 256 40 : 18.5; 768 x 768 with 512 rows 12 : 17, 1024 20 : 17; 1000 x 1001 with 128 rows 11.5 : 34,
// 512 30 : 35. That is up to 2^25 weights and passes together.
bool few_rows(int64_t m, const Q4Dev& w) {
    const int64_t passes = (m + 15) / 16, cols = m < 16 ? m : 16;
    return m <= 2 || (cols * w.cols <= 57344 && (passes == 1 || (passes <= 65535 && passes * w.rows * w.cols <= int64_t(1) << 25)));
}

// Experts: their weights times the passes over them, half a pass empty on average, against a start
// of some 36 us and then the same weights once. 8 experts of 2048 x 1024 with 8 pairs each
// 30 : 40, 12 43 : 41; 16 of 1024 x 512 with 12 35 : 37, 24 53 : 40; 8 of 512 x 768 with 48
// 38 : 53, 96 71 : 61; 4 of 512 x 128 with 128 23 : 48. With 4 pairs an expert, 32 of 2048 x 1024
// still run 75 : 100, with 8 121 : 105.
bool few_experts(const FfnArgs& a) {
    const int64_t pairs = a.tokens * a.top_k;
    return pairs <= FEW_MAX_PAIRS && (a.tokens <= 16 || pairs <= 4 * static_cast<int64_t>(a.experts) ||
                                      static_cast<int64_t>(a.d) * a.f <= 192000000 / (pairs + a.experts));
}

int zeros_out(uor_b200_ctx* ctx, int64_t rows, int n, const MatOut& y) {
    return launch(ctx, blocks_of_rows(rows, n), false, add_parts_kernel, nullptr, 0, rows, n, y);
}

}  // namespace

int run_q4_gemm(uor_b200_ctx* ctx, int elem, const Mat& x, int64_t m, const Q4Dev& w, const MatOut& y,
                uor_b200_route* route) {
    route->kernel = UOR_B200_KERNEL_Q4;
    if (w.cols == 0) return zeros_out(ctx, m, w.rows, y);
    int st = UOR_B200_OK;
    const bool few = few_rows(m, w);
    Pieces pieces;
    // The few-rows kernel reads any row whose elements follow one another.
    const bool own_rows = few ? x.cs != 1 : !x_in_place(x, w.cols);
    const size_t x_at = pieces.add(own_rows ? static_cast<size_t>(m) * up_to(w.cols, 8) * 2 : 0);
    ManyParams many{};
    many.w = w;
    many.mode = MANY_DENSE;
    many.n = w.rows;
    many.experts = 1;
    many.m = static_cast<int>(m);
    many.y = y;
    many.part_rows = m;
    const int splits = few ? 1 : many_splits(ctx, many);
    const size_t codes_at = pieces.add(few ? 0 : codes_copy_bytes(w));
    const size_t part_at = pieces.add(splits > 1 ? static_cast<size_t>(splits) * m * w.rows * 4 : 0);
    uint8_t* ws = pieces.get(ctx, &st);
    if (!ws) return st;
    Mat rows = x;
    if (own_rows) {
        copy_rows(ctx, x, w.cols, m, nullptr, 1, nullptr, ws + x_at, false);
        rows = Mat{ws + x_at, up_to(w.cols, 8), 1};
    }
    if (few) {
        FewParams p{};
        p.kind = FEW_DENSE;
        p.w = w;
        p.x = rows.p;
        p.x_rs = rows.rs;
        p.m = m;
        p.n = w.rows;
        p.y = y;
        few_align(&p);
        st = few_launch(ctx, elem, p, false);
        route->tile_m = 16, route->tile_n = p.columns, route->tile_k = 256;
        return st;
    }
    copy_codes(ctx, &many.w, ws + codes_at);
    many.x = rows.p;
    many.x_rs = rows.rs;
    many.x_rows = m;
    many.part = reinterpret_cast<float*>(ws + part_at);
    route->tile_m = 256, route->tile_n = 256, route->tile_k = 128;
    route->k_chunks = splits;
    if ((st = many_launch(ctx, elem, many, own_rows || codes_copy_bytes(w) > 0))) return st;
    if (splits > 1) {
        return launch(ctx, blocks_of_rows(m, w.rows), true, add_parts_kernel, many.part, splits, m, w.rows, y);
    }
    return UOR_B200_OK;
}

int run_expert_ffn(uor_b200_ctx* ctx, const FfnArgs& a, uor_b200_route* route) {
    route->kernel = UOR_B200_KERNEL_Q4;
    if (a.top_k == 0 || a.f == 0) return zeros_out(ctx, a.tokens, a.d, a.y);
    int st = UOR_B200_OK;
    const int64_t pairs = a.tokens * a.top_k;
    const int h_rs = up_to(a.f, 8), x_rs = up_to(a.d, 8);
    Pieces pieces;
    const bool few = few_experts(a);
    const size_t h_at = pieces.add(static_cast<size_t>(pairs) * h_rs * (few && few_twice(a.tokens) ? 4 : 2));
    if (few) {
        const size_t x_at = pieces.add(a.x.cs == 1 ? 0 : static_cast<size_t>(a.tokens) * x_rs * 2);
        const size_t part_at = pieces.add(static_cast<size_t>(pairs) * a.d * 4);
        uint8_t* ws = pieces.get(ctx, &st);
        if (!ws) return st;
        FewParams p{};
        p.kind = FEW_UP;
        p.h = ws + h_at;
        p.h_rs = h_rs;
        p.twice = few_twice(a.tokens);
        p.w = a.up;
        p.x = a.x.p;
        p.x_rs = a.x.rs;
        if (a.x.cs != 1) {
            copy_rows(ctx, a.x, a.d, a.tokens, nullptr, 1, nullptr, ws + x_at, false);
            p.x = ws + x_at;
            p.x_rs = x_rs;
        }
        p.n = a.f;
        p.ids = a.ids;
        p.tokens = static_cast<int>(a.tokens);
        p.top_k = a.top_k;
        p.experts = a.experts;
        few_align(&p);
        if ((st = few_launch(ctx, a.elem, p, false))) return st;
        route->tile_m = 16, route->tile_n = p.columns, route->tile_k = 256;  // the up product's
        p.kind = FEW_PART;
        p.w = a.down;
        p.x = p.h;
        p.x_rs = h_rs;
        p.n = a.d;
        p.part = reinterpret_cast<float*>(ws + part_at);
        few_align(&p);
        if ((st = few_launch(ctx, a.elem, p, true))) return st;
        return launch_combine(ctx, p.part, 1, a, true);
    }

    ManyParams up{};
    up.w = a.up;
    up.mode = MANY_UP;
    up.n = a.f;
    up.experts = a.experts;
    up.x_rs = x_rs;
    up.x_rows = pairs;
    up.h_rs = h_rs;
    ManyParams down = up;
    down.w = a.down;
    down.mode = MANY_DOWN;
    down.n = a.d;
    down.x_rs = h_rs;
    down.part_rows = pairs;
    const int splits = many_splits(ctx, down);
    const size_t x_at = pieces.add(static_cast<size_t>(pairs) * x_rs * 2);
    const size_t part_at = pieces.add(static_cast<size_t>(splits) * pairs * a.d * 4);
    const size_t up_at = pieces.add(codes_copy_bytes(a.up)), down_at = pieces.add(codes_copy_bytes(a.down));
    const size_t offsets_at = pieces.add((a.experts + 1) * sizeof(int)), perm_at = pieces.add(pairs * sizeof(int));
    uint8_t* ws = pieces.get(ctx, &st);
    if (!ws) return st;
    int* offsets = reinterpret_cast<int*>(ws + offsets_at);
    int* perm = reinterpret_cast<int*>(ws + perm_at);
    sort_kernel<<<a.experts, SORT_THREADS, 0, ctx->stream>>>(a.ids, static_cast<int>(pairs), a.top_k, a.experts, offsets, perm);
    copy_rows(ctx, a.x, a.d, pairs, perm, a.top_k, offsets + a.experts, ws + x_at, true);
    copy_codes(ctx, &up.w, ws + up_at);
    copy_codes(ctx, &down.w, ws + down_at);
    up.offsets = down.offsets = offsets;
    up.perm = down.perm = perm;
    up.x = ws + x_at;
    up.h = ws + h_at;
    down.x = ws + h_at;
    down.part = reinterpret_cast<float*>(ws + part_at);
    route->tile_m = 256, route->tile_n = 256, route->tile_k = 128;
    if ((st = many_launch(ctx, a.elem, up, true)) || (st = many_launch(ctx, a.elem, down, true))) return st;
    return launch_combine(ctx, down.part, splits, a, false);
}

}  // namespace uor
