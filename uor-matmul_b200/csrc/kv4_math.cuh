// kv4_math.cuh -- what the attention kernels over the 4-bit cache share: pairs of floats, copies, and
// which blocks the rows of a sequence see.
#pragma once
#include "kv4.cuh"

#include <cstring>
#include <type_traits>

namespace uor {

namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(mask), "r"(bits));
    return r;
}
template <typename T>
__device__ __forceinline__ float2 two(uint32_t w) {
    if constexpr (std::is_same<T, __half>::value) {
        __half2 v;
        memcpy(&v, &w, 4);
        return __half22float2(v);
    }
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <typename T>
__device__ __forceinline__ uint32_t pack(float a, float b) {
    uint32_t r;
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 v = __floats2half2_rn(a, b);
        memcpy(&r, &v, 4);
    } else {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        memcpy(&r, &v, 4);
    }
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void cp_async(uint32_t to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// N words from shared memory at a multiple of N words.
template <int N>
__device__ __forceinline__ void words(const uint8_t* p, uint32_t (&w)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const uint4 v = reinterpret_cast<const uint4*>(p)[i];
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const uint2 v = reinterpret_cast<const uint2*>(p)[i];
            w[2 * i] = v.x, w[2 * i + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    }
}

// Two floats at once.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void parts_of(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
template <typename T>
__device__ __forceinline__ uint64_t pair_of(uint32_t w) {
    const float2 v = two<T>(w);
    return pair_of(v.x, v.y);
}
// Which blocks of 16 tokens the rows of a sequence see: sink_blocks first ones, then those from
// first_block on; and its work.
struct Share {
    int rows, row_tiles, sink_blocks, first_block, blocks, tiles;
    Share() = default;
    // tile_rows: rows of a tile; tile_blocks: blocks of a step of its work.
    __device__ __forceinline__ Share(const Sequence& s, const AttendArgs& a, int tile_rows, int tile_blocks) {
        rows = s.count * a.share;
        row_tiles = (rows + tile_rows - 1) / tile_rows;
        blocks_of(s.at, s.keys, a);
        tiles = max(1, (blocks + tile_blocks - 1) / tile_blocks);  // of one head and row tile
    }
    // Of one row tile alone.
    __device__ __forceinline__ Share(const Sequence& s, const AttendArgs& a, int tile_rows, int tile_blocks, int tile) {
        rows = s.count * a.share;
        row_tiles = (rows + tile_rows - 1) / tile_rows;
        const int last = s.at + min((tile + 1) * tile_rows - 1, rows - 1) / a.share;
        blocks_of(s.at + tile * tile_rows / a.share, max(0, min(s.keys, last + 1)), a);
        tiles = (blocks + tile_blocks - 1) / tile_blocks;
    }
    // From the first row's position on, keys 0 .. keys - 1.
    __device__ __forceinline__ void blocks_of(int at, int keys, const AttendArgs& a) {
        const int low = a.window ? max(0, at - a.window + 1) : 0, ends = (keys + 15) >> 4;
        first_block = low < keys ? low >> 4 : ends;
        sink_blocks = a.window ? min((min(a.sinks, keys) + 15) >> 4, first_block) : 0;
        blocks = sink_blocks + ends - first_block;
    }
    __device__ __forceinline__ int block_at(int i) const { return i < sink_blocks ? i : first_block + i - sink_blocks; }
    __device__ __forceinline__ int64_t work(int heads) const { return static_cast<int64_t>(row_tiles) * heads * tiles; }
};

}  // namespace

}  // namespace uor
