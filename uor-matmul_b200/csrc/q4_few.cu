// q4_few.cu -- products of few rows with 4-bit weights and group scales.
//
// Bound by the weights' bytes, read once: 4 bits and a share of a scale each. A CTA takes 16 rows
// of weights and its eight warps split the reduction into chunks of 128 positions (64 bytes of a
// row), warp w taking chunks w, w + 8, ...: side by side they read 512 contiguous bytes of each
// row. Each warp keeps a ring of chunks of codes and activations in flight with cp.async, in
// shared memory of its own, so no warp waits for another until the sums are joined at the end.
//
// The products run on the tensor cores (mma.m16n8k16) with the weights as the 16 rows and up to 8
// activation rows as the columns, since CUDA cores could not multiply at the rate the codes
// arrive at from four rows on. A code is exact as a 16-bit float: its bits under the exponent of
// 128 (bfloat16) or 1024 (float16), less the same plus the zero point. So the sum of a group is
// exact but for its f32 additions, and the group's scale multiplies it in f32: no weight is ever
// rounded. The reduction's order within a group is free, so a lane's 16 bytes are taken as they
// lie: word j of lane c holds positions 32 c + 8 j .. + 7, the instruction's operands are its
// nibbles (0, 4), (1, 5) | (2, 6), (3, 7), and the activations are paired to match.
#include "q4_few.cuh"

#include "ptx.cuh"

namespace uor {

namespace {

constexpr int WARPS = 8;
constexpr int STAGES = 4;
constexpr int ROWS = 16;
constexpr int CHUNK = 128;                     // positions of the reduction per ring stage
constexpr int CODE_BYTES = ROWS * CHUNK / 2;   // of a stage
constexpr int X_BYTES = CHUNK * 2;             // of a stage, per activation row

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

// Four nibbles' pairs as two 16-bit floats each: (code - zero) of positions (s, s + 4).
template <typename T>
struct Decode;
template <>
struct Decode<__nv_bfloat16> {
    static constexpr uint32_t MAGIC = 0x43004300u;  // 128
    __device__ static __forceinline__ uint32_t less(uint32_t v, uint32_t zero) {
        __nv_bfloat162 a, b;
        memcpy(&a, &v, 4);
        memcpy(&b, &zero, 4);
        a = __hsub2(a, b);
        memcpy(&v, &a, 4);
        return v;
    }
    __device__ static __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <>
struct Decode<__half> {
    static constexpr uint32_t MAGIC = 0x64006400u;  // 1024
    __device__ static __forceinline__ uint32_t less(uint32_t v, uint32_t zero) {
        __half2 a, b;
        memcpy(&a, &v, 4);
        memcpy(&b, &zero, 4);
        a = __hsub2(a, b);
        memcpy(&v, &a, 4);
        return v;
    }
    __device__ static __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};

// Where 16-byte piece c of a row's 64 bytes of codes lies: eight rows' reads of any width meet no
// bank twice.
__device__ __forceinline__ int code_at(int row, int c) {
    return row * 64 + ((c ^ ((row & 2) | ((row >> 2) & 1))) << 4);
}
// The same for 16-byte piece p of an activation row's 256 bytes, read by lane c of segment s as
// piece 4 c + j (SEG 128), 8 s + 2 c + j (64) or 4 s + c (32).
template <int SEG>
__device__ __forceinline__ int x_at(int row, int p) {
    const int odd = row & 1;
    const int q = SEG == 128 ? p ^ ((p >> 2) & 2) ^ odd : SEG == 64 ? p ^ odd : p ^ (odd << 2);
    return row * X_BYTES + (q << 4);
}

// 16 bytes from any address, of which `left` exist.
__device__ __forceinline__ uint4 load16_anywhere(const uint8_t* p, int left) {
    uint32_t w[4] = {0, 0, 0, 0};
    for (int i = 0; i < 16; ++i)
        if (i < left) w[i >> 2] |= static_cast<uint32_t>(p[i]) << (8 * (i & 3));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

struct Unit {
    const uint8_t* codes;  // of the tile's row 0 (rows follow by the stride, the second eight by `half`)
    int64_t scale0;        // scale index of the tile's row 0
    int chunk;
};

// One warp's ring.
template <typename T, int SEG, int NT>
struct Ring {
    static constexpr int NSEG = CHUNK / SEG;
    uint32_t base;   // shared address
    int stage_bytes, rows_x, lane;

    __device__ __forceinline__ uint32_t stage(int i) const { return base + (i % STAGES) * stage_bytes; }

    // Row r of a tile, as an offset in rows: the last valid row stands in for those past it.
    __device__ static __forceinline__ int64_t row_of(int r, int valid, int64_t half) {
        return r < 8 ? min(r, valid - 1) : half + min(r - 8, valid - 1);
    }

    __device__ __forceinline__ void load_codes(int i, const uint8_t* tile, int chunk, const FewParams& p, int lo, int hi,
                                               int64_t half) const {
        const uint32_t at = stage(i);
        const int row_len = (p.w.cols + 1) / 2;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            const int r = (lane >> 2) + 8 * v, c = lane & 3;
            const int64_t row = v == 0 ? min(r, lo - 1) : half + min(r - 8, hi - 1);
            const int byte = chunk * (CHUNK / 2) + c * 16;
            const int left = max(0, min(16, row_len - byte));
            const uint8_t* src = tile + row * p.w.row_bytes + (left ? byte : 0);
            const uint32_t dst = at + code_at(r, c);
            if (p.codes_align == 16) {
                cp_async16(dst, src, left);
            } else if (p.codes_align == 4) {
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int n = max(0, min(4, left - 4 * b));
                    cp_async4(dst + 4 * b, n ? src + 4 * b : src, n);
                }
            } else {
                const uint4 w = load16_anywhere(src, left);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w)
                             : "memory");
            }
        }
    }

    // x_row(r): the activation row behind column r.
    template <typename F>
    __device__ __forceinline__ void load_x(int i, int chunk, const FewParams& p, F x_row) const {
        const uint32_t at = stage(i) + CODE_BYTES;
        for (int v = lane; v < rows_x * 16; v += 32) {
            const int r = v >> 4, c = v & 15;
            const int k = chunk * CHUNK + c * 8;
            const int left = max(0, min(8, p.w.cols - k));
            const T* src = static_cast<const T*>(p.x) + x_row(r) * p.x_rs + (left ? k : 0);
            const uint32_t dst = at + x_at<SEG>(r, c);
            if (p.x_vec) {
                cp_async16(dst, src, left * 2);
            } else {
                uint32_t w[4] = {0, 0, 0, 0};
                const uint16_t* s = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
                for (int b = 0; b < 8; ++b)
                    if (b < left) w[b >> 1] |= static_cast<uint32_t>(s[b]) << (16 * (b & 1));
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                             : "memory");
            }
        }
    }

    // This lane's scales and zero points (its rows lane / 4 and + 8) of a chunk's segments.
    struct Scales {
        float s[NSEG][2];
        uint32_t z[NSEG][2];
    };
    __device__ __forceinline__ void load_scales(Scales& q, int64_t scale0, int chunk, const FewParams& p, int lo, int hi,
                                                int64_t half) const {
        const int groups = (p.w.cols + p.w.group - 1) / p.w.group;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            const int r = lane >> 2;
            const int64_t row = v == 0 ? min(r, lo - 1) : half + min(r, hi - 1);
            const int64_t at = scale0 + row * p.w.groups_rs;
#pragma unroll
            for (int s = 0; s < NSEG; ++s) {
                const int g = min((chunk * CHUNK + s * SEG) / p.w.group, groups - 1);
                q.s[s][v] = load_f32(p.w.scales, at + g, p.w.scale_type);
                const uint32_t z = p.w.zeros ? p.w.zeros[at + g] & 15u : 8u;
                q.z[s][v] = Decode<T>::MAGIC | (z << 16) | z;
            }
        }
    }

    // sum[nt] += the chunk's products: column n of the instruction is activation row 8 nt + n.
    __device__ __forceinline__ void compute(int i, const Scales& q, int segs, float (&sum)[NT][4]) const {
        const uint32_t codes = stage(i), xs = codes + CODE_BYTES;
        const int g = lane >> 2, c = lane & 3;
#pragma unroll
        for (int s = 0; s < NSEG; ++s) {
            if (s >= segs) break;
            constexpr int WORDS = SEG / 32;
            uint32_t w[2][4];
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const int r = g + 8 * v;
                if (SEG == 128)
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(w[v][0]), "=r"(w[v][1]), "=r"(w[v][2]), "=r"(w[v][3])
                                 : "r"(codes + code_at(r, c)));
                else if (SEG == 64)
                    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];"
                                 : "=r"(w[v][0]), "=r"(w[v][1])
                                 : "r"(codes + code_at(r, 2 * s + (c >> 1)) + (c & 1) * 8));
                else
                    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[v][0]) : "r"(codes + code_at(r, s) + c * 4));
            }
            float acc[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0;
#pragma unroll
            for (int j = 0; j < WORDS; ++j) {
                uint32_t a[2][4];
#pragma unroll
                for (int v = 0; v < 2; ++v)
#pragma unroll
                    for (int h = 0; h < 4; ++h)
                        a[v][h] = Decode<T>::less(((w[v][j] >> (4 * h)) & 0x000F000Fu) | Decode<T>::MAGIC, q.z[s][v]);
                const uint32_t a0[4] = {a[0][0], a[1][0], a[0][1], a[1][1]};
                const uint32_t a1[4] = {a[0][2], a[1][2], a[0][3], a[1][3]};
                const int piece = SEG == 128 ? 4 * c + j : SEG == 64 ? 8 * s + 2 * c + j : 4 * s + c;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    uint32_t x0, x1, x2, x3;
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(x0), "=r"(x1), "=r"(x2), "=r"(x3)
                                 : "r"(xs + x_at<SEG>(min(nt * 8 + g, rows_x - 1), piece)));
                    Decode<T>::mma(acc[nt], a0, __byte_perm(x0, x2, 0x5410), __byte_perm(x0, x2, 0x7632));
                    Decode<T>::mma(acc[nt], a1, __byte_perm(x1, x3, 0x5410), __byte_perm(x1, x3, 0x7632));
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                sum[nt][0] = fmaf(q.s[s][0], acc[nt][0], sum[nt][0]);
                sum[nt][1] = fmaf(q.s[s][0], acc[nt][1], sum[nt][1]);
                sum[nt][2] = fmaf(q.s[s][1], acc[nt][2], sum[nt][2]);
                sum[nt][3] = fmaf(q.s[s][1], acc[nt][3], sum[nt][3]);
            }
        }
    }
};

__device__ __forceinline__ int id_at(const FewParams& p, int pair) {
    return static_cast<const int32_t*>(p.ids.p)[pair / p.top_k * p.ids.rs + pair % p.top_k * p.ids.cs];
}

// The joined sums of a tile: [warp][nt][lane][4] in shared memory, added in the warps' order.
template <int NT>
__device__ __forceinline__ float joined(const float* red, int row, int col) {
    const int lane = (row & 7) * 4 + ((col & 7) >> 1), nt = col >> 3, r = (row >> 3) * 2 + (col & 1);
    float v = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) v += red[((w * NT + nt) * 32 + lane) * 4 + r];
    return v;
}

template <typename T, int SEG, int NT, int MODE>
__global__ void __launch_bounds__(WARPS * 32) few_kernel(const FewParams p) {
    using R = Ring<T, SEG, NT>;
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr bool DOWN = MODE == FEW_DOWN;
    __shared__ int id_of[MODE == FEW_DENSE ? 1 : FEW_MAX_PAIRS];
    __shared__ int expert_of[DOWN ? FEW_MAX_PAIRS : 1];        // the chosen experts, each once
    __shared__ float weight_of[DOWN ? FEW_MAX_PAIRS * 8 : 1];  // by expert and token
    __shared__ int pair_of[DOWN ? FEW_MAX_PAIRS * 8 : 1];
    __shared__ unsigned chosen_by[DOWN ? FEW_MAX_PAIRS : 1];   // an expert's tokens, a bit each
    __shared__ int rank_of[DOWN ? FEW_MAX_PAIRS : 1];
    __shared__ int count[WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int chunks = (p.w.cols + CHUNK - 1) / CHUNK;
    const int pairs = p.tokens * p.top_k;
    R ring;
    ring.lane = lane;

    int64_t row0 = 0, half = 8, x0 = 0;  // the tile's first row of weights; from it to its ninth
    int lo, hi;                          // valid rows of the tile's two halves
    int units;
    if (MODE == FEW_DENSE) {
        row0 = static_cast<int64_t>(blockIdx.x) * ROWS;
        lo = min(8, p.n - static_cast<int>(row0));
        hi = max(1, min(8, p.n - static_cast<int>(row0) - 8));
        if (p.n - row0 <= 8) half = 0;  // no second half: the first stands in
        x0 = static_cast<int64_t>(blockIdx.y) * (8 * NT);
        ring.rows_x = static_cast<int>(min(static_cast<int64_t>(8 * NT), p.m - x0));
        units = chunks;
    } else if (MODE == FEW_UP) {
        // CTA y takes the expert of pair y, unless an earlier pair has the same one.
        const int j0 = blockIdx.x * 8;
        if (threadIdx.x < pairs) id_of[threadIdx.x] = id_at(p, threadIdx.x);
        __syncthreads();
        const int e = id_of[blockIdx.y];
        if (e < 0 || e >= p.experts) return;
        if (__syncthreads_or(threadIdx.x < blockIdx.y && id_of[threadIdx.x] == e)) return;
        row0 = static_cast<int64_t>(e) * 2 * p.n + j0;
        half = p.n;
        lo = hi = min(8, p.n - j0);
        ring.rows_x = p.tokens;
        units = chunks;
    } else {
        // The experts in the order of their first choice, with their tokens' weights; an expert
        // that a token chose twice has both weights.
        const int i = threadIdx.x, t = i / p.top_k, slot = i % p.top_k;
        float w = 0;
        int e = -1;
        if (i < pairs) {
            e = id_at(p, i);
            if (e < 0 || e >= p.experts) e = -1;
            w = static_cast<const float*>(p.weights.p)[t * p.weights.rs + slot * p.weights.cs];
            id_of[i] = e;
            weight_of[i] = w;  // by pair until they are summed
            chosen_by[i] = 0;
        }
        __syncthreads();
        int first = i;  // the first pair of this pair's expert
        if (e >= 0)
            for (int o = i - 1; o >= 0; --o)
                if (id_of[o] == e) first = o;
        const bool head = e >= 0 && first == i;
        const unsigned vote = __ballot_sync(0xffffffffu, head);
        if (lane == 0) count[warp] = __popc(vote);
        bool mine = e >= 0;  // the token's first choice of this expert sums its weights
        for (int s = 0; s < p.top_k && i < pairs; ++s) {
            const int o = t * p.top_k + s;
            if (id_of[o] != e || o == i) continue;
            if (o < i) mine = false;
            if (mine) w += weight_of[o];
        }
        __syncthreads();
        int before = 0, listed = 0;
        for (int v = 0; v < WARPS; ++v) {
            if (v < warp) before += count[v];
            listed += count[v];
        }
        if (head) {
            const int a = before + __popc(vote & ((1u << lane) - 1));
            rank_of[i] = a;
            expert_of[a] = e;
        }
        if (i < FEW_MAX_PAIRS)
            for (int r = 0; r < 8; ++r) pair_of[i * 8 + r] = 0;
        __syncthreads();
        if (mine) {
            const int a = rank_of[first];
            weight_of[a * 8 + t] = w;
            pair_of[a * 8 + t] = i;
            atomicOr(&chosen_by[a], 1u << t);
        }
        __syncthreads();
        row0 = static_cast<int64_t>(blockIdx.x) * ROWS;
        lo = min(8, p.n - static_cast<int>(row0));
        hi = max(1, min(8, p.n - static_cast<int>(row0) - 8));
        if (p.n - row0 <= 8) half = 0;
        ring.rows_x = p.tokens;
        units = chunks * listed;
    }
    ring.stage_bytes = CODE_BYTES + ring.rows_x * X_BYTES;
    ring.base = smem_u32(smem) + warp * STAGES * ring.stage_bytes;

    const int mine = units > warp ? (units - warp + WARPS - 1) / WARPS : 0;
    auto unit_chunk = [&](int i) { return MODE == FEW_DOWN ? (warp + i * WARPS) % chunks : warp + i * WARPS; };
    auto unit_row = [&](int i) {
        return MODE == FEW_DOWN ? static_cast<int64_t>(expert_of[(warp + i * WARPS) / chunks]) * p.n + row0 : row0;
    };
    auto codes = [&](int i) {
        ring.load_codes(i, p.w.codes + unit_row(i) * p.w.row_bytes, unit_chunk(i), p, lo, hi, half);
    };
    auto x = [&](int i) {
        if (MODE == FEW_DOWN) {
            const int a = (warp + i * WARPS) / chunks;
            ring.load_x(i, unit_chunk(i), p, [&](int r) { return static_cast<int64_t>(pair_of[a * 8 + r]); });
        } else {
            ring.load_x(i, unit_chunk(i), p, [&](int r) { return x0 + r; });
        }
    };
    float total[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) total[nt][0] = total[nt][1] = total[nt][2] = total[nt][3] = 0;

    // The weights depend on nothing before this launch, the inner activations on the one before,
    // which lets this one begin as soon as its own blocks have.
    if (MODE == FEW_UP) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    for (int s = 0; s < STAGES - 1; ++s)
        if (s < mine) codes(s);
    if (MODE == FEW_DOWN) asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int s = 0; s < STAGES - 1; ++s) {
        if (s < mine) x(s);
        cp_commit();
    }
    typename R::Scales now, next;
    if (mine) ring.load_scales(now, unit_row(0) * p.w.groups_rs, unit_chunk(0), p, lo, hi, half);
    for (int i = 0; i < mine; ++i) {
        cp_wait<STAGES - 2>();
        __syncwarp();
        if (i + STAGES - 1 < mine) {
            codes(i + STAGES - 1);
            x(i + STAGES - 1);
        }
        cp_commit();
        if (i + 1 < mine) ring.load_scales(next, unit_row(i + 1) * p.w.groups_rs, unit_chunk(i + 1), p, lo, hi, half);
        const int segs = min(R::NSEG, (p.w.cols - unit_chunk(i) * CHUNK + SEG - 1) / SEG);
        if (MODE == FEW_DOWN) {
            float part[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) part[nt][0] = part[nt][1] = part[nt][2] = part[nt][3] = 0;
            ring.compute(i, now, segs, part);
            const int a = (warp + i * WARPS) / chunks, t = (lane & 3) * 2;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (chosen_by[a] >> (t + (r & 1)) & 1)
                    total[0][r] = fmaf(weight_of[a * 8 + t + (r & 1)], part[0][r], total[0][r]);
        } else {
            ring.compute(i, now, segs, total);
        }
        now = next;
    }
    cp_wait<0>();
    __syncthreads();
    float* red = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
        reinterpret_cast<float4*>(red)[(warp * NT + nt) * 32 + lane] =
            make_float4(total[nt][0], total[nt][1], total[nt][2], total[nt][3]);
    __syncthreads();
    if (MODE == FEW_UP) {
        const int e = id_of[blockIdx.y];
        for (int v = threadIdx.x; v < 8 * pairs; v += blockDim.x) {
            const int r = v & 7, i = v >> 3, t = i / p.top_k;
            if (r < lo && id_of[i] == e)
                static_cast<T*>(p.h)[static_cast<int64_t>(i) * p.n + blockIdx.x * 8 + r] =
                    from_f32<T>(silu(joined<NT>(red, r, t)) * joined<NT>(red, r + 8, t));
        }
    } else {
        for (int v = threadIdx.x; v < ROWS * ring.rows_x; v += blockDim.x) {
            const int r = v & 15, t = v >> 4;
            if (row0 + r < p.n)
                store_f32(p.y.p, (x0 + t) * p.y.rs + (row0 + r) * p.y.cs, p.y.type, joined<NT>(red, r, t));
        }
    }
}

template <typename T, int SEG, int NT, int MODE>
int launch_few(uor_b200_ctx* ctx, const FewParams& p, bool after_up) {
    const int rows_x = MODE == FEW_DENSE ? static_cast<int>(p.m < 8 * NT ? p.m : 8 * NT) : p.tokens;
    const int ring = WARPS * STAGES * (CODE_BYTES + rows_x * X_BYTES), red = WARPS * NT * 32 * 16;
    const int bytes = ring > red ? ring : red;
    auto* kernel = few_kernel<T, SEG, NT, MODE>;
    static bool ready[64] = {};
    if (!ready[ctx->device & 63]) {
        const int most = WARPS * STAGES * (CODE_BYTES + 8 * NT * X_BYTES);
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess)
            return UOR_B200_DEVICE_ERROR;
        ready[ctx->device & 63] = true;
    }
    cudaLaunchConfig_t c = {};
    c.blockDim = dim3(WARPS * 32);
    c.dynamicSmemBytes = bytes;
    c.stream = ctx->stream;
    if (MODE == FEW_DENSE)
        c.gridDim = dim3((p.n + ROWS - 1) / ROWS, static_cast<unsigned>((p.m + 8 * NT - 1) / (8 * NT)));
    else if (MODE == FEW_UP)
        c.gridDim = dim3((p.n + 7) / 8, p.tokens * p.top_k);
    else
        c.gridDim = dim3((p.n + ROWS - 1) / ROWS);
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &early;
    c.numAttrs = after_up ? 1 : 0;
    return cuda_status(cudaLaunchKernelEx(&c, kernel, p));
}

template <typename T, int SEG>
int by_mode(uor_b200_ctx* ctx, FewMode mode, const FewParams& p, bool after_up) {
    if (mode == FEW_UP) return launch_few<T, SEG, 1, FEW_UP>(ctx, p, after_up);
    if (mode == FEW_DOWN) return launch_few<T, SEG, 1, FEW_DOWN>(ctx, p, after_up);
    return launch_few<T, SEG, 1, FEW_DENSE>(ctx, p, after_up);
}

// The segment is what one scale covers within a chunk: the largest of 128, 64 and 32 that
// divides the group.
template <typename T>
int by_segment(uor_b200_ctx* ctx, FewMode mode, const FewParams& p, bool after_up) {
    if (p.w.group % 128 == 0) return by_mode<T, 128>(ctx, mode, p, after_up);
    if (p.w.group % 64 == 0) return by_mode<T, 64>(ctx, mode, p, after_up);
    return by_mode<T, 32>(ctx, mode, p, after_up);
}

}  // namespace

int few_launch(uor_b200_ctx* ctx, int elem, FewMode mode, const FewParams& p, bool after_up) {
    return elem == UOR_B200_BF16 ? by_segment<__nv_bfloat16>(ctx, mode, p, after_up)
                                 : by_segment<__half>(ctx, mode, p, after_up);
}

}  // namespace uor
