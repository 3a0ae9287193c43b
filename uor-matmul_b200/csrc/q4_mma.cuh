// q4_mma.cuh -- what the kernels for few rows share: codes as operands of mma.m16n8k16, the order
// of the activations beside them, scales and zero points, the pairs of an expert.
#pragma once
#include <cstring>
#include <type_traits>

#include "q4_few.cuh"

namespace uor {

namespace {

constexpr int ROWS = 16;
constexpr int SUB = 128;                       // positions of the reduction in 64 bytes of a row
constexpr int CHUNK = 2 * SUB;                 // positions that a warp takes at a time
constexpr int X_BYTES = SUB * 2;               // of a SUB, per activation row

__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(mask), "r"(bits));
    return r;
}

// A word's eight codes less their zero point, in CodeUnits, as pairs of 16-bit floats: positions
// (0, 4), (1, 5), (2, 6), (3, 7).
template <typename T>
struct Decode;
template <>
struct Decode<__nv_bfloat16> {
    // 128 + code, less 128 + zero, both of 2^-12.
    struct Zero {
        __nv_bfloat162 v;
    };
    static constexpr uint32_t ZERO_8 = 0x3D083D08u;
    // Of byte i of a word of zero points.
    __device__ static __forceinline__ uint32_t zero_bits(uint32_t w, int i) { return __byte_perm(w, 0x3D, 0x4040 + 0x101 * i); }
    __device__ static __forceinline__ Zero zero(uint32_t b) {
        Zero r;
        memcpy(&r.v, &b, 4);
        return r;
    }
    __device__ static __forceinline__ uint32_t one(uint32_t w, const Zero& z) {
        const uint32_t b = and_or(w, 0x000F000Fu, 0x3D003D00u);
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

// Where 16-byte piece p of an activation row's 256 bytes of a SUB lies, so that eight rows' reads
// meet no bank twice; lane c of
// segment s reads it as piece 4 c + j (SEG 128), 8 s + 2 c + j (64) or 4 s + c (32).
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

// Reads of shared memory at its 32-bit addresses, as loads the compiler may order by itself.
template <typename V>
__device__ __forceinline__ V lds(uint32_t at) {
    return *static_cast<const V*>(__cvta_shared_to_generic(at));
}

__device__ __forceinline__ void sts128(uint32_t at, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
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
    // The same from the rows' addresses of the chunk's first scale and zero point, of which `left`
    // exist; vec: they are vectors.
    __device__ __forceinline__ void load_at(const S* s0, const S* s1, const uint8_t* z0, const uint8_t* z1, bool zeros, bool vec, int left) {
        if (vec && left >= N) {
            copy(s[0], s0);
            copy(s[1], s1);
            if (zeros) {
                if constexpr (N == 2) {
                    z[0][0] = *reinterpret_cast<const uint16_t*>(z0);
                    z[1][0] = *reinterpret_cast<const uint16_t*>(z1);
                } else {
                    copy(z[0], z0);
                    copy(z[1], z1);
                }
            }
            return;
        }
        if (left >= N) {
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const S* from = v ? s1 : s0;
                const uint8_t* zfrom = v ? z1 : z0;
#pragma unroll
                for (int i = 0; i < SW; ++i) {
                    if constexpr (sizeof(S) == 4) {
                        s[v][i] = reinterpret_cast<const uint32_t*>(from)[i];
                    } else {
                        const uint32_t lo = reinterpret_cast<const uint16_t*>(from)[2 * i], hi = reinterpret_cast<const uint16_t*>(from)[2 * i + 1];
                        s[v][i] = lo | hi << 16;
                    }
                }
                if (zeros) {
#pragma unroll
                    for (int i = 0; i < ZW; ++i) {
                        z[v][i] = 0;
#pragma unroll
                        for (int b = 0; b < 4 && 4 * i + b < N; ++b) z[v][i] |= static_cast<uint32_t>(zfrom[4 * i + b]) << (8 * b);
                    }
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
                const int at = min(i, left - 1);
                if constexpr (sizeof(S) == 4) {
                    s[v][i] = reinterpret_cast<const uint32_t*>(v ? s1 : s0)[at];
                } else {
                    const uint32_t raw = reinterpret_cast<const uint16_t*>(v ? s1 : s0)[at];
                    s[v][i / 2] = i & 1 ? s[v][i / 2] | raw << 16 : raw;
                }
                if (zeros) z[v][i / 4] |= static_cast<uint32_t>((v ? z1 : z0)[at]) << (8 * (i & 3));
            }
        }
    }
    // Zero points' low four bits, once for the chunk.
    __device__ __forceinline__ void mask() {
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
            for (int i = 0; i < ZW; ++i) z[v][i] &= 0x0F0F0F0Fu;
    }
    __device__ __forceinline__ float scale(int v, int i) const {
        if constexpr (sizeof(S) == 4) return __uint_as_float(s[v][i]);
        if constexpr (std::is_same<S, __nv_bfloat16>::value)
            return __uint_as_float(i & 1 ? s[v][i / 2] & 0xFFFF0000u : s[v][i / 2] << 16);
        else
            return __half2float(__ushort_as_half(static_cast<unsigned short>(i & 1 ? s[v][i / 2] >> 16 : s[v][i / 2])));
    }
    __device__ __forceinline__ uint32_t zero(int v, int i, bool given) const {
        return given ? Decode<T>::zero_bits(z[v][i / 4], i & 3) : Decode<T>::ZERO_8;
    }
};

// A tile of weights: its rows r are row0 + r (half 8), or eight rows from row0 on and eight from
// row0 + half on; `lo` and `hi` of the halves' rows are valid, and the last valid one stands in for
// those past it.
struct Tile {
    int64_t row0, half;
    int lo, hi;
    __device__ __forceinline__ int64_t row(int r) const {
        return r < 8 ? row0 + min(r, lo - 1) : row0 + half + min(r - 8, hi - 1);
    }
};

// Tile t of expert e's matrix (of the one matrix: e 0).
__device__ __forceinline__ Tile tile_at(const FewParams& p, int e, int t) {
    t = min(t, p.tiles - 1);
    Tile w;
    if (p.kind == FEW_UP) {
        w.row0 = static_cast<int64_t>(e) * 2 * p.n + t * 8;
        w.half = p.n;
        w.lo = w.hi = min(8, p.n - t * 8);
    } else {
        const int left = p.n - t * ROWS;
        w.row0 = static_cast<int64_t>(e) * p.n + t * ROWS;
        w.half = left > 8 ? 8 : 0;  // no second half: the first row stands in
        w.lo = min(8, left);
        w.hi = max(1, min(8, left - 8));
    }
    return w;
}

// NT: columns in eights. A block has 8 warps a column eight.
template <int NT>
struct Block {
    static constexpr int WARPS = 8 * NT, THREADS = 32 * WARPS;
    static constexpr int RED = 2 * WARPS * NT * 128 * 4;  // joined sums, twice
    static constexpr int X_MOST = NT == 1 ? 64 * 1024 : 112 * 1024;  // resident activations
};

// An activation's place among its eight in the operands' order.
__device__ __forceinline__ int paired(int r) { return r < 4 ? 2 * r : 2 * r - 7; }

// The pairs of one expert, found by the block.
struct Found {
    uint32_t bits[FEW_MAX_EXPERTS / 32];                // the chosen experts
    uint16_t id_of[FEW_MAX_PAIRS], list[FEW_MAX_PAIRS];  // the pairs' experts; this one's pairs
    int counts[32], chosen;
};

// Block y takes the y-th of the chosen experts: found.chosen, and its pairs in found.list. Their
// count, or -1 where there is no such expert.
template <int WARPS>
__device__ __forceinline__ int find_pairs(const FewParams& p, Found& found) {
    constexpr int THREADS = 32 * WARPS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto& bits = found.bits;
    auto& id_of = found.id_of;
    auto& list = found.list;
    const int pairs = p.tokens * p.top_k;
    if (threadIdx.x < FEW_MAX_EXPERTS / 32) bits[threadIdx.x] = 0;
    if (threadIdx.x == 0) found.chosen = -1;
    __syncthreads();
    for (int i = threadIdx.x; i < pairs; i += THREADS) {
        const int t = i / p.top_k;
        const int id = static_cast<const int32_t*>(p.ids.p)[t * p.ids.rs + (i - t * p.top_k) * p.ids.cs];
        const bool in = id >= 0 && id < p.experts;
        id_of[i] = in ? static_cast<uint16_t>(id) : 0xFFFF;
        if (in) atomicOr(&bits[id >> 5], 1u << (id & 31));
    }
    __syncthreads();
    if (warp == 0) {
        const uint32_t w = bits[lane];
        int before = __popc(w);
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += v;
        }
        before -= __popc(w);
        const int nth = static_cast<int>(blockIdx.y) - before;
        if (nth >= 0 && nth < __popc(w)) {
            uint32_t left = w;
            for (int b = 0; b < nth; ++b) left &= left - 1;
            found.chosen = lane * 32 + __ffs(left) - 1;
        }
    }
    __syncthreads();
    const int e = found.chosen;
    if (e < 0) return -1;
    // its pairs, in order: a run of pairs to a thread. A token that chose it more than once is
    // there with its first choice alone, so there are at most as many columns as tokens.
    auto lists = [&](int i) {
        if (id_of[i] != e) return false;
        for (int o = i - i % p.top_k; o < i; ++o)
            if (id_of[o] == e) return false;
        return true;
    };
    const int run = (pairs + THREADS - 1) / THREADS, from = min(pairs, static_cast<int>(threadIdx.x) * run);
    const int to = min(pairs, from + run);
    int mine = 0;
    for (int i = from; i < to; ++i) mine += lists(i);
    int upto = mine;
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) found.counts[warp] = upto;
    __syncthreads();
    int at = upto - mine, listed = 0;
    for (int w = 0; w < WARPS; ++w) {
        if (w < warp) at += found.counts[w];
        listed += found.counts[w];
    }
    for (int i = from; i < to; ++i)
        if (lists(i)) list[at++] = static_cast<uint16_t>(i);
    __syncthreads();
    return listed;
}

// The activation row behind column c: of a dense block's first x0, the token's of a listed pair, or
// a pair's inner activations.
__device__ __forceinline__ int64_t x_row_of(const FewParams& p, const Found& found, int64_t x0, int c) {
    if (p.kind == FEW_DENSE) return x0 + c;
    if (p.kind == FEW_UP) return found.list[c] / p.top_k;
    return (static_cast<int64_t>(found.list[c >> p.twice]) << p.twice) + (c & p.twice);
}

// The columns that a launch's largest block may have.
inline int64_t few_columns(const FewParams& p) { return p.kind == FEW_DENSE ? p.m : p.kind == FEW_UP ? p.tokens : p.tokens << p.twice; }

// The blocks that share an expert's columns, `width` at a time: as many as `spread` times the mean
// of them needs, where the largest expert may have that many.
inline int few_shares(const FewParams& p, int width, int spread) {
    if (p.kind == FEW_DENSE) return 1;
    const int64_t most = (few_columns(p) + width - 1) / width, all = static_cast<int64_t>(p.experts) * width;
    const int64_t mean = (spread * few_columns(p) * p.top_k + all - 1) / all;
    return static_cast<int>(mean < 1 ? 1 : mean < most ? mean : most);
}

// The tiles t0, t0 + 1, .. that a block's warps hold side by side: their sums, [warp][column
// eight][lane][4] in shared memory, added in the warps' order and put where the launch's go.
// Columns c0 .. c0 + cols - 1 of the block's.
template <typename T, int NT>
__device__ __forceinline__ void tiles_out(const FewParams& p, const Found& found, const float* joined, int e, int t0, int c0,
                                          int cols, int64_t x0) {
    const int kw = 1 << p.k_shift, abreast = Block<NT>::WARPS >> p.k_shift;
    const int row_bits = p.kind == FEW_UP ? 3 : 4, rows = 1 << row_bits;  // outputs of a tile
    const int twice = p.kind == FEW_PART ? p.twice : 0;  // a pair's two columns are one output
    for (int v = threadIdx.x; v < (abreast * rows * cols) >> twice; v += Block<NT>::THREADS) {
        const int r = v & (rows - 1), rest = v >> row_bits;
        const int out_col = abreast == 1 ? rest : rest / abreast, ab = rest - out_col * abreast, col = out_col << twice;
        const int out = (t0 + ab) * rows + r;
        auto sum = [&](int row, int c = 0) {
            const float* at = joined + (ab * kw * NT + (col >> 3)) * 128 + ((row & 7) * 4 + ((col & 7) >> 1)) * 4 + (row >> 3) * 2 + ((col + c) & 1);
            float s = 0;
            for (int w = 0; w < kw; ++w) s += at[w * NT * 128];
            return CodeUnit<T>::VALUE * s;
        };
        if (p.kind == FEW_UP) {
            // eight inner activations in the operands' order, zeros behind the last; in a second
            // row what the first one's rounding left
            if (t0 + ab < p.tiles) {
                const float h = out < p.n ? silu(sum(r)) * sum(r + 8) : 0.0f;
                const T high = from_f32<T>(h);
                T* to = static_cast<T*>(p.h) + (static_cast<int64_t>(found.list[c0 + col]) << p.twice) * p.h_rs + (t0 + ab) * 8 + paired(r);
                to[0] = high;
                if (p.twice) to[p.h_rs] = from_f32<T>(fabsf(to_f32(high)) < INFINITY ? h - to_f32(high) : 0.0f);
            }
        } else if (out < p.n) {
            if (p.kind == FEW_PART)
                p.part[static_cast<int64_t>(found.list[(c0 + col) >> twice]) * p.n + out] = twice ? sum(r) + sum(r, 1) : sum(r);
            else
                store_f32(p.y.p, (x0 + col) * p.y.rs + out * p.y.cs, p.y.type, sum(r));
        }
    }
}

}  // namespace

}  // namespace uor
