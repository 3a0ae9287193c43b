// q4_few.cu -- products of few rows with 4-bit weights and group scales.
//
// Bound by the weights' bytes, read once: 4 bits and a share of a scale each. A CTA takes 16 rows
// of weights and its eight warps split the reduction into chunks of 256 positions (128 bytes of a
// row), warp w taking chunks w, w + 8, ...: side by side they read 1 KB of each row. Each warp
// keeps a ring of chunks of codes in flight with cp.async, in shared memory of its own, so no
// warp waits for another until the sums are joined at the end. The scales and zero points of the
// tile, and the activations, are laid out in shared memory while the first chunks travel.
//
// The products run on the tensor cores (mma.m16n8k16) with the weights as the 16 rows and up to 8
// activation rows as the columns, since CUDA cores could not multiply at the rate the codes
// arrive at from four rows on. A code is exact as a 16-bit float: its bits under the exponent of
// 128 (bfloat16) or 1024 (float16), less the same plus the zero point. So the sum of a group is
// exact but for its f32 additions, and the group's scale multiplies it in f32: no weight is ever
// rounded. The reduction's order within a group is free, so a lane's 16 bytes are taken as they
// lie: word j of lane c holds positions 32 c + 8 j .. + 7, and the instruction's operands are its
// nibbles (0, 4), (1, 5) | (2, 6), (3, 7). The activations lie in shared memory in that order:
// every eight as 0 4 1 5 2 6 3 7.
//
// What is left beside the memory is instructions: 11 to unpack eight weights of bfloat16 (three
// shifts, four and-or, four subtractions), so addresses, scales and their types are kept out of
// the loop.
#include "q4_few.cuh"

#include <type_traits>

#include "ptx.cuh"

namespace uor {

namespace {

constexpr int WARPS = 8;
constexpr int STAGES = 2;
constexpr int ROWS = 16;
constexpr int SUB = 128;                       // positions of the reduction in 64 bytes of a row
constexpr int CHUNK = 2 * SUB;                 // positions per ring stage
constexpr int HALF_BYTES = ROWS * SUB / 2;     // of a stage's codes, per SUB
constexpr int PITCH_ANY = 144;                 // of a row's codes whose addresses are not aligned
constexpr int X_BYTES = SUB * 2;               // of a SUB, per activation row
constexpr int X_MOST = 64 * 1024;              // resident activations of a CTA

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

__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(mask), "r"(bits));
    return r;
}

// A word's eight codes less their zero point, as pairs of 16-bit floats: positions (0, 4),
// (1, 5), (2, 6), (3, 7).
template <typename T>
struct Decode;
template <>
struct Decode<__nv_bfloat16> {
    // 128 + code, less 128 + zero.
    struct Zero {
        __nv_bfloat162 v;
    };
    static constexpr uint32_t ZERO_8 = 0x43084308u;
    // Of byte i of a word of zero points.
    __device__ static __forceinline__ uint32_t zero_bits(uint32_t w, int i) { return __byte_perm(w, 0x43, 0x4040 + 0x101 * i); }
    __device__ static __forceinline__ Zero zero(uint32_t b) {
        Zero r;
        memcpy(&r.v, &b, 4);
        return r;
    }
    __device__ static __forceinline__ uint32_t one(uint32_t w, const Zero& z) {
        const uint32_t b = and_or(w, 0x000F000Fu, 0x43004300u);
        __nv_bfloat162 v;
        memcpy(&v, &b, 4);
        v = __hsub2(v, z.v);
        uint32_t r;
        memcpy(&r, &v, 4);
        return r;
    }
    __device__ static __forceinline__ void unpack(uint32_t w, const Zero& z, uint32_t& p0, uint32_t& p1, uint32_t& p2,
                                                  uint32_t& p3) {
        p0 = one(w, z), p1 = one(w >> 4, z), p2 = one(w >> 8, z), p3 = one(w >> 12, z);
    }
    __device__ static __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <>
struct Decode<__half> {
    // 1024 + code, less 1024 + zero; and, of the nibble above it, (1024 + 16 code) / 16 less
    // 64 + zero, which spares the shift.
    struct Zero {
        __half2 low, high;
    };
    static constexpr uint32_t ZERO_8 = 0x64086408u;
    __device__ static __forceinline__ uint32_t zero_bits(uint32_t w, int i) { return __byte_perm(w, 0x64, 0x4040 + 0x101 * i); }
    __device__ static __forceinline__ Zero zero(uint32_t b) {
        Zero r;
        memcpy(&r.low, &b, 4);
        r.high = __hsub2(__float2half2_rn(960.0f), r.low);  // -(64 + zero)
        return r;
    }
    __device__ static __forceinline__ uint32_t low(uint32_t w, const Zero& z) {
        const uint32_t b = and_or(w, 0x000F000Fu, 0x64006400u);
        __half2 v;
        memcpy(&v, &b, 4);
        v = __hsub2(v, z.low);
        uint32_t r;
        memcpy(&r, &v, 4);
        return r;
    }
    __device__ static __forceinline__ uint32_t high(uint32_t w, const Zero& z) {
        const uint32_t b = and_or(w, 0x00F000F0u, 0x64006400u);
        __half2 v;
        memcpy(&v, &b, 4);
        v = __hfma2(v, __float2half2_rn(0.0625f), z.high);
        uint32_t r;
        memcpy(&r, &v, 4);
        return r;
    }
    __device__ static __forceinline__ void unpack(uint32_t w, const Zero& z, uint32_t& p0, uint32_t& p1, uint32_t& p2,
                                                  uint32_t& p3) {
        p0 = low(w, z), p1 = high(w, z), p2 = low(w >> 8, z), p3 = high(w >> 8, z);
    }
    __device__ static __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
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
// The same for 16-byte piece p of an activation row's 256 bytes of a chunk, read by lane c of
// segment s as piece 4 c + j (SEG 128), 8 s + 2 c + j (64) or 4 s + c (32).
template <int SEG>
__device__ __forceinline__ int x_piece(int row, int p) {
    const int odd = row & 1;
    return (SEG == 128 ? p ^ ((p >> 2) & 2) ^ odd : SEG == 64 ? p ^ odd : p ^ (odd << 2)) << 4;
}

// Eight activations from positions k .. k + 7 of a row, `left` of them existing.
template <typename T>
__device__ __forceinline__ uint4 load_x8(const T* p, int left, bool vec) {
    if (vec && left >= 8) return *reinterpret_cast<const uint4*>(p);
    uint32_t w[4] = {0, 0, 0, 0};
    const uint16_t* s = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int b = 0; b < 8; ++b)
        if (b < left) w[b >> 1] |= static_cast<uint32_t>(s[b]) << (16 * (b & 1));
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// The same in the order of the operands.
__device__ __forceinline__ uint4 in_pairs(uint4 w) {
    return make_uint4(__byte_perm(w.x, w.z, 0x5410), __byte_perm(w.x, w.z, 0x7632), __byte_perm(w.y, w.w, 0x5410),
                      __byte_perm(w.y, w.w, 0x7632));
}

__device__ __forceinline__ int id_at(const FewParams& p, int pair) {
    return static_cast<const int32_t*>(p.ids.p)[pair / p.top_k * p.ids.rs + pair % p.top_k * p.ids.cs];
}

// Reads of shared memory at its 32-bit addresses, as loads the compiler may order by itself.
template <typename V>
__device__ __forceinline__ V lds(uint32_t at) {
    return *static_cast<const V*>(__cvta_shared_to_generic(at));
}

__device__ __forceinline__ void sts128(uint32_t at, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// A tile's joined sum: [warp][lane][4] in shared memory, added in the warps' order.
__device__ __forceinline__ float joined(const float* red, int row, int col) {
    const int at = ((row & 7) * 4 + (col >> 1)) * 4 + (row >> 3) * 2 + (col & 1);
    float v = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) v += red[w * 128 + at];
    return v;
}

// The scales and zero points of a chunk for this lane's two rows (lane / 4 of each half of the
// tile), as they lie in memory. S: T where the scales are of that type, float otherwise.
template <typename T, typename S, int SEG>
struct Quants {
    static constexpr int N = CHUNK / SEG;
    static constexpr int SW = N * sizeof(S) / 4, ZW = (N + 3) / 4;
    uint32_t s[2][SW], z[2][ZW];

    template <int WORDS>
    __device__ static __forceinline__ void copy(uint32_t (&to)[WORDS], const void* from) {
        if constexpr (WORDS % 4 == 0) {
#pragma unroll
            for (int i = 0; i < WORDS; i += 4) {
                const uint4 v = static_cast<const uint4*>(from)[i / 4];
                to[i] = v.x, to[i + 1] = v.y, to[i + 2] = v.z, to[i + 3] = v.w;
            }
        } else if constexpr (WORDS == 2) {
            const uint2 v = *static_cast<const uint2*>(from);
            to[0] = v.x, to[1] = v.y;
        } else {
            to[0] = *static_cast<const uint32_t*>(from);
        }
    }

    // row0, row1: scale indexes of the rows' first groups. Where every row's scales begin at a
    // multiple of a chunk's and a group is a segment, a chunk's are one vector.
    __device__ __forceinline__ void load(const FewParams& p, int64_t row0, int64_t row1, int chunk, int groups) {
        if (p.quants_vec && (chunk + 1) * N <= groups) {
            copy(s[0], static_cast<const S*>(p.w.scales) + row0 + chunk * N);
            copy(s[1], static_cast<const S*>(p.w.scales) + row1 + chunk * N);
            if (p.w.zeros) {
                if constexpr (N == 2) {
                    z[0][0] = *reinterpret_cast<const uint16_t*>(p.w.zeros + row0 + chunk * N);
                    z[1][0] = *reinterpret_cast<const uint16_t*>(p.w.zeros + row1 + chunk * N);
                } else {
                    copy(z[0], p.w.zeros + row0 + chunk * N);
                    copy(z[1], p.w.zeros + row1 + chunk * N);
                }
            }
            return;
        }
#pragma unroll
        for (int v = 0; v < 2; ++v) {
#pragma unroll
            for (int i = 0; i < ZW; ++i) z[v][i] = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int at = chunk * CHUNK + i * SEG;
                const int64_t q = (v ? row1 : row0) + min(p.group_shift >= 0 ? at >> p.group_shift : at / p.w.group, groups - 1);
                if constexpr (sizeof(S) == 4) {
                    s[v][i] = __float_as_uint(load_f32(p.w.scales, q, p.w.scale_type));
                } else {
                    const uint32_t raw = static_cast<const uint16_t*>(p.w.scales)[q];
                    s[v][i / 2] = i & 1 ? s[v][i / 2] | raw << 16 : raw;
                }
                if (p.w.zeros) z[v][i / 4] |= static_cast<uint32_t>(p.w.zeros[q]) << (8 * (i & 3));
            }
        }
    }
    __device__ __forceinline__ float scale(int v, int i) const {
        if constexpr (sizeof(S) == 4) return __uint_as_float(s[v][i]);
        if constexpr (std::is_same<S, __nv_bfloat16>::value)
            return __uint_as_float(i & 1 ? s[v][i / 2] & 0xFFFF0000u : s[v][i / 2] << 16);
        else
            return __half2float(__ushort_as_half(static_cast<unsigned short>(i & 1 ? s[v][i / 2] >> 16 : s[v][i / 2])));
    }
    __device__ __forceinline__ uint32_t zero(int v, int i, bool given) const {
        return given ? Decode<T>::zero_bits(z[v][i / 4] & 0x0F0F0F0Fu, i & 3) : Decode<T>::ZERO_8;
    }
};

// One warp's ring of chunks of codes.
template <typename T, typename S, int SEG, bool ANY>
struct Ring {
    static constexpr int NSEG = SUB / SEG;
    uint32_t base;               // shared address of stage 0
    const uint8_t* row[ANY ? 2 : 4];  // this lane's rows of codes: its pieces' (lane / 8 + 4 v), or g and g + 8
    int64_t step;                // from one expert's codes to the next's, in bytes
    int row_len;

    __device__ __forceinline__ void init(const FewParams& p, int lane, int64_t row0, int64_t half, int lo, int hi) {
        auto at = [&](int r) {  // the last valid row stands in for those past it
            const int64_t i = r < 8 ? row0 + min(r, lo - 1) : row0 + half + min(r - 8, hi - 1);
            return p.w.codes + i * p.w.row_bytes;
        };
        if constexpr (ANY) {
            row[0] = at(lane >> 2), row[1] = at((lane >> 2) + 8);
        } else {
#pragma unroll
            for (int v = 0; v < 4; ++v) row[v] = at((lane >> 3) + 4 * v) + 16 * (lane & 7);
        }
        step = static_cast<int64_t>(p.n) * p.w.row_bytes;
        row_len = (p.w.cols + 1) / 2;
    }

    __device__ __forceinline__ void load(int stage, int chunk, int expert, int lane) const {
        const uint32_t at = base + stage * stage_bytes<ANY>();
        const int64_t from = expert * step + chunk * (CHUNK / 2);
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
    // lane's column of the instruction (row x_row of them); left: positions that exist.
    __device__ __forceinline__ void compute(int stage, int sub, int expert, int lane, const Quants<T, S, SEG>& q, bool zeros,
                                            uint32_t xs, int x_row, int left, float (&sum)[4]) const {
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
                const int m0 = 8 * static_cast<int>((reinterpret_cast<uint64_t>(row[0]) + expert * step) & 3);
                const int m1 = 8 * static_cast<int>((reinterpret_cast<uint64_t>(row[1]) + expert * step) & 3);
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
            float acc[4] = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < WORDS; ++j) {
                uint32_t a0[4], a1[4];
                Decode<T>::unpack(w0[j], zero0, a0[0], a0[2], a1[0], a1[2]);
                Decode<T>::unpack(w1[j], zero1, a0[1], a0[3], a1[1], a1[3]);
                const int piece = SEG == 128 ? 4 * c + j : SEG == 64 ? 8 * s + 2 * c + j : 4 * s + c;
                const uint4 x = lds<uint4>(xs + x_piece<SEG>(x_row, piece));
                Decode<T>::mma(acc, a0, x.x, x.y);
                Decode<T>::mma(acc, a1, x.z, x.w);
            }
            sum[0] = fmaf(scale0, acc[0], sum[0]);
            sum[1] = fmaf(scale0, acc[1], sum[1]);
            sum[2] = fmaf(scale1, acc[2], sum[2]);
            sum[3] = fmaf(scale1, acc[3], sum[3]);
        }
    }
};

// An activation's place among its eight in the operands' order.
__device__ __forceinline__ int paired(int r) { return r < 4 ? 2 * r : 2 * r - 7; }

template <typename T, typename S, int SEG, int MODE, bool ANY>
__global__ void __launch_bounds__(WARPS * 32, 3) few_kernel(const FewParams p) {
    using R = Ring<T, S, SEG, ANY>;
    constexpr bool DOWN = MODE == FEW_DOWN;
    extern __shared__ __align__(128) uint8_t smem[];
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

    int64_t row0 = 0, half = 8, x0 = 0;  // the tile's first row of weights; from it to its ninth
    int lo, hi;                          // valid rows of the tile's two halves
    int rows_x = p.tokens, units = chunks;
    if (MODE == FEW_UP) {
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
    } else {
        row0 = static_cast<int64_t>(blockIdx.x) * ROWS;
        lo = min(8, p.n - static_cast<int>(row0));
        hi = max(1, min(8, p.n - static_cast<int>(row0) - 8));
        if (p.n - row0 <= 8) half = 0;  // no second half: the first row stands in
        if (MODE == FEW_DENSE) {
            x0 = static_cast<int64_t>(blockIdx.y) * 8;
            rows_x = static_cast<int>(min(static_cast<int64_t>(8), p.m - x0));
        }
    }
    if (DOWN) {
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
        __syncthreads();
        if (mine) {
            const int a = rank_of[first];
            weight_of[a * 8 + t] = w;
            pair_of[a * 8 + t] = i;
            atomicOr(&chosen_by[a], 1u << t);
        }
        __syncthreads();
        units = chunks * listed;
    }

    R ring;
    ring.init(p, lane, row0, half, lo, hi);
    ring.base = smem_u32(smem) + warp * (STAGES * stage_bytes<ANY>());
    // Behind the rings the activations: resident rows of a panel of the reduction, or a chunk of
    // them with each stage.
    const int panel = DOWN ? units : min(units, p.panel);
    const uint32_t x_all = smem_u32(smem) + WARPS * STAGES * stage_bytes<ANY>();
    const uint32_t x_ring = x_all + warp * (STAGES * rows_x * 2 * X_BYTES);
    const int x_row = min(lane >> 2, rows_x - 1);
    const int groups = (p.w.cols + p.w.group - 1) / p.w.group;
    const int64_t quants0 = (row0 + min(lane >> 2, lo - 1)) * p.w.groups_rs;
    const int64_t quants1 = (row0 + half + min(lane >> 2, hi - 1)) * p.w.groups_rs;
    const int64_t quants_step = static_cast<int64_t>(p.n) * p.w.groups_rs;
    const bool zeros = p.w.zeros != nullptr;
    float total[4] = {0, 0, 0, 0};

    if (MODE == FEW_UP) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (DOWN && units == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
    // This warp's units of a panel: first + warp, first + warp + 8, ... A unit is a chunk, or with
    // several experts the chunks of one after those of another.
    for (int first = 0; first < units; first += panel) {
        const int here = min(panel, units - first);
        const int mine = here > warp ? (here - warp + WARPS - 1) / WARPS : 0;
        int lstage = 0, le = 0, lc = first + warp;  // the next unit to load
        if constexpr (DOWN) le = lc / chunks, lc = lc % chunks;
        auto load_codes = [&]() { ring.load(lstage, lc, DOWN ? expert_of[le] : 0, lane); };
        auto load_x = [&]() {
            if constexpr (DOWN) {
                for (int v = lane; v < rows_x * 32; v += 32) {
                    const int r = v >> 5, piece = v & 31, k = lc * CHUNK + piece * 8;
                    if (!(chosen_by[le] >> r & 1)) continue;
                    const bool in = k < p.x_rs;
                    cp_async16(x_ring + ((lstage * rows_x + r) * 2 + (piece >> 4)) * X_BYTES + x_piece<SEG>(r, piece & 15),
                               static_cast<const T*>(p.x) + pair_of[le * 8 + r] * p.x_rs + (in ? k : 0), in ? 16 : 0);
                }
            }
        };
        auto advance = [&]() {
            lstage = lstage + 1 == STAGES ? 0 : lstage + 1;
            lc += WARPS;
            if constexpr (DOWN) {
                while (lc >= chunks) lc -= chunks, ++le;
            }
        };
        if (first) __syncthreads();  // every warp is done with the panel before this one
        const int c0 = lc, e0 = le;
        for (int s = 0; s < STAGES - 1; ++s) {
            if (s < mine) load_codes(), advance();
            if (!DOWN) cp_commit();
        }
        Quants<T, S, SEG> now, next;
        if (mine) now.load(p, quants0 + (DOWN ? expert_of[e0] * quants_step : 0), quants1 + (DOWN ? expert_of[e0] * quants_step : 0), c0, groups);
        if (DOWN) {
            // The weights depend on nothing before this launch, the inner activations on the
            // launch before it.
            asm volatile("griddepcontrol.wait;" ::: "memory");
            lc = c0, le = e0, lstage = 0;
            for (int s = 0; s < STAGES - 1; ++s) {
                if (s < mine) load_x(), advance();
                cp_commit();
            }
        } else {
            const int pieces = here * 32;
            for (int v0 = threadIdx.x; v0 < rows_x * pieces; v0 += 4 * blockDim.x) {
                uint4 x8[4];
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int v = min(v0 + b * static_cast<int>(blockDim.x), rows_x * pieces - 1);
                    const int r = rows_x == 1 ? 0 : v / pieces, k = first * CHUNK + (v - r * pieces) * 8;
                    x8[b] = load_x8(static_cast<const T*>(p.x) + (x0 + r) * p.x_rs + k, p.w.cols - k, p.x_vec != 0);
                }
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int v = v0 + b * static_cast<int>(blockDim.x);
                    const int r = rows_x == 1 ? 0 : v / pieces, piece = v - r * pieces;
                    if (v < rows_x * pieces)
                        sts128(x_all + (r * panel * 2 + (piece >> 4)) * X_BYTES + x_piece<SEG>(r, piece & 15), in_pairs(x8[b]));
                }
            }
        }
        __syncthreads();
        int stage = 0, e = 0, c = first + warp;
        if constexpr (DOWN) e = c / chunks, c = c % chunks;
        uint32_t xs = x_all + (x_row * panel + warp) * (2 * X_BYTES);
        for (int i = 0; i < mine; ++i) {
            cp_wait<STAGES - 2>();
            __syncwarp();
            if (i + STAGES - 1 < mine) load_codes(), load_x(), advance();
            cp_commit();
            int e2 = e, c2 = c + WARPS;  // the unit after this one
            if constexpr (DOWN) {
                while (c2 >= chunks) c2 -= chunks, ++e2;
            }
            if (i + 1 < mine) {
                const int64_t to = DOWN ? expert_of[e2] * quants_step : 0;
                next.load(p, quants0 + to, quants1 + to, c2, groups);
            }
            const int left = p.w.cols - c * CHUNK;
            if constexpr (DOWN) {
                float part[4] = {0, 0, 0, 0};
                const uint32_t x2 = x_ring + (stage * rows_x + x_row) * (2 * X_BYTES);
                ring.compute(stage, 0, expert_of[e], lane, now, zeros, x2, x_row, left, part);
                if (left > SUB) ring.compute(stage, 1, expert_of[e], lane, now, zeros, x2 + X_BYTES, x_row, left - SUB, part);
                const int t = (lane & 3) * 2;
                const unsigned chosen = chosen_by[e] >> t;
                const float2 w = *reinterpret_cast<const float2*>(&weight_of[e * 8 + t]);
                if (chosen & 1) total[0] = fmaf(w.x, part[0], total[0]), total[2] = fmaf(w.x, part[2], total[2]);
                if (chosen & 2) total[1] = fmaf(w.y, part[1], total[1]), total[3] = fmaf(w.y, part[3], total[3]);
            } else {
                ring.compute(stage, 0, 0, lane, now, zeros, xs, x_row, left, total);
                if (left > SUB) ring.compute(stage, 1, 0, lane, now, zeros, xs + X_BYTES, x_row, left - SUB, total);
            }
            stage = stage + 1 == STAGES ? 0 : stage + 1;
            xs += WARPS * (2 * X_BYTES);
            c = c2, e = e2;
            now = next;
        }
        cp_wait<0>();
    }
    __syncthreads();
    float* red = reinterpret_cast<float*>(smem);
    reinterpret_cast<float4*>(red)[warp * 32 + lane] = make_float4(total[0], total[1], total[2], total[3]);
    __syncthreads();
    if (MODE == FEW_UP) {
        // Eight inner activations in the operands' order, zeros behind the last.
        const int e = id_of[blockIdx.y];
        for (int v = threadIdx.x; v < 8 * pairs; v += blockDim.x) {
            const int r = v & 7, i = v >> 3, t = i / p.top_k;
            if (id_of[i] == e)
                static_cast<T*>(p.h)[static_cast<int64_t>(i) * p.h_rs + blockIdx.x * 8 + paired(r)] =
                    from_f32<T>(r < lo ? silu(joined(red, r, t)) * joined(red, r + 8, t) : 0.0f);
        }
    } else {
        const int v = threadIdx.x, r = v & 15, t = v >> 4;
        if (t < rows_x && row0 + r < p.n)
            store_f32(p.y.p, (x0 + t) * p.y.rs + (row0 + r) * p.y.cs, p.y.type, joined(red, r, t));
    }
}

template <typename T, typename S, int SEG, int MODE, bool ANY>
int launch_few(uor_b200_ctx* ctx, FewParams& p, bool after_up) {
    const int chunks = (p.w.cols + CHUNK - 1) / CHUNK;
    const int rows_x = MODE == FEW_DENSE ? static_cast<int>(p.m < 8 ? p.m : 8) : p.tokens;
    p.group_shift = (p.w.group & (p.w.group - 1)) == 0 ? __builtin_ctz(p.w.group) : -1;
    constexpr int N = CHUNK / SEG;
    constexpr int VEC = N * sizeof(S) < 16 ? N * sizeof(S) : 16;
    p.quants_vec = p.w.group == SEG && (sizeof(S) == 2 || p.w.scale_type == UOR_B200_F32) &&
                   (reinterpret_cast<uint64_t>(p.w.scales) | static_cast<uint64_t>(p.w.groups_rs) * sizeof(S)) % VEC == 0 &&
                   (reinterpret_cast<uint64_t>(p.w.zeros) | (p.w.zeros ? static_cast<uint64_t>(p.w.groups_rs) : 0)) % N == 0;
    int x_bytes = WARPS * STAGES * rows_x * 2 * X_BYTES;
    if (MODE != FEW_DOWN) {
        p.panel = X_MOST / (rows_x * 2 * X_BYTES);
        if (p.panel > chunks) p.panel = chunks;
        x_bytes = rows_x * p.panel * 2 * X_BYTES;
    }
    auto* kernel = few_kernel<T, S, SEG, MODE, ANY>;
    constexpr int RINGS = WARPS * STAGES * stage_bytes<ANY>();
    static bool ready[64] = {};
    if (!ready[ctx->device & 63]) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, RINGS + X_MOST) != cudaSuccess)
            return UOR_B200_DEVICE_ERROR;
        ready[ctx->device & 63] = true;
    }
    cudaLaunchConfig_t c = {};
    c.blockDim = dim3(WARPS * 32);
    c.dynamicSmemBytes = RINGS + x_bytes;
    c.stream = ctx->stream;
    if (MODE == FEW_DENSE)
        c.gridDim = dim3((p.n + ROWS - 1) / ROWS, static_cast<unsigned>((p.m + 7) / 8));
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

template <typename T, typename S, int SEG, bool ANY>
int by_mode(uor_b200_ctx* ctx, FewMode mode, FewParams& p, bool after_up) {
    if (mode == FEW_UP) return launch_few<T, S, SEG, FEW_UP, ANY>(ctx, p, after_up);
    if (mode == FEW_DOWN) return launch_few<T, S, SEG, FEW_DOWN, ANY>(ctx, p, after_up);
    return launch_few<T, S, SEG, FEW_DENSE, ANY>(ctx, p, after_up);
}

// The segment is what one scale covers within 128 positions: the largest of 128, 64 and 32 that
// divides the group.
template <typename T, typename S, bool ANY>
int by_segment(uor_b200_ctx* ctx, FewMode mode, FewParams& p, bool after_up) {
    if (p.w.group % 128 == 0) return by_mode<T, S, 128, ANY>(ctx, mode, p, after_up);
    if (p.w.group % 64 == 0) return by_mode<T, S, 64, ANY>(ctx, mode, p, after_up);
    return by_mode<T, S, 32, ANY>(ctx, mode, p, after_up);
}

// Rows of codes that do not all begin at multiples of 16 bytes are copied by words and shifted
// into place; scales that are neither float nor of the activations' type are converted as they
// are read.
template <typename T>
int by_codes(uor_b200_ctx* ctx, int elem, FewMode mode, FewParams& p, bool after_up) {
    if (p.codes_align != 16) return by_segment<T, float, true>(ctx, mode, p, after_up);
    if (p.w.scale_type == elem) return by_segment<T, T, false>(ctx, mode, p, after_up);
    return by_segment<T, float, false>(ctx, mode, p, after_up);
}

}  // namespace

int few_launch(uor_b200_ctx* ctx, int elem, FewMode mode, FewParams p, bool after_up) {
    return elem == UOR_B200_BF16 ? by_codes<__nv_bfloat16>(ctx, elem, mode, p, after_up) : by_codes<__half>(ctx, elem, mode, p, after_up);
}

}  // namespace uor
