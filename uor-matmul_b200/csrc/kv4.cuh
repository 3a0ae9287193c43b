// kv4.cuh -- the 4-bit cache of keys and values: its layout, the device-side descriptors, launches.
#pragma once
#include "q4.cuh"

namespace uor {

// A page holds, per head, page_size / 16 blocks. A block is 16 tokens' keys and values in the order in
// which the attention's matrix instructions take them, so that a warp reads its operands' words as
// whole vectors (words are 32 bits, D channels in 32s, G groups):
//   keys' codes     16 D / 2 bytes. Word (t * 4 + c) * (D / 32) + n: token t's channels 32 n + 8 c + i,
//                   nibble i.
//   keys' params    64 G bytes. Eight bytes (t / 2 * G + g): scale of the even token, of the odd one,
//                   middle of the even one, of the odd one; 16 bits each.
//   values' codes   16 D / 2 bytes. Word ((t / 8 * 8 + r) * 4 + t / 2 % 4) * (D / 32) + n: channels
//                   32 n + 4 r + i of the even token in nibble i, of the odd one in nibble 4 + i.
//   values' params  as the keys'.
// A token's 16-bit pieces are its own: tokens are appended in any order and by any thread.
constexpr int KV_BLOCK = 16;

struct KvDev {
    uint8_t* pool;
    int64_t page_bytes, head_bytes;
    int64_t pages;
    int page_shift;    // log2 of the tokens of a page
    int heads, dim, groups;
    int group_shift;   // log2 of the group
    int block_bytes;   // 16 D + 128 G
};

__host__ __device__ constexpr int kv_block_bytes(int dim, int groups) { return 16 * dim + 128 * groups; }

// Byte offsets in a block.
__device__ __forceinline__ int kv_key_word(int dim, int t, int channel) {  // of the word with 8 channels
    return ((t * 4 + (channel >> 3 & 3)) * (dim >> 5) + (channel >> 5)) * 4;
}
__device__ __forceinline__ int kv_value_half(int dim, int groups, int t, int channel) {  // of 4 channels
    return 8 * dim + 64 * groups + ((((t >> 3) * 8 + (channel >> 2 & 7)) * 4 + (t >> 1 & 3)) * (dim >> 5) + (channel >> 5)) * 4 +
           (t & 1) * 2;
}
__device__ __forceinline__ int kv_scale(int dim, int groups, int t, int g, bool values) {  // the middle: 4 further
    return 8 * dim + (values ? 8 * dim + 64 * groups : 0) + ((t >> 1) * groups + g) * 8 + (t & 1) * 2;
}

struct BatchDev {
    const int32_t *starts, *lengths, *table;
    int64_t table_rs;
    int seqs;
    int rows;          // of the call's matrices
    int capacity;      // positions that the table reaches, below 2^30
};

// Sequence s of a batch, whatever its arrays hold: rows first .. first + count - 1 lie within the
// call's, its first row is at position `at`, and its keys are those at 0 .. keys - 1.
struct Sequence {
    int first, count, at, keys;
    __device__ __forceinline__ Sequence(const BatchDev& b, int s) {
        first = min(max(b.starts[s], 0), b.rows);
        count = min(max(b.starts[s + 1], first), b.rows) - first;
        const int length = max(b.lengths[s], 0);
        at = length - count;
        keys = min(length, b.capacity);
    }
};

// The block with position p (>= 0, below the capacity) of sequence s and a head; null where its page
// is none of the pool's.
__device__ __forceinline__ uint8_t* kv_block(const KvDev& kv, const BatchDev& b, int s, int head, int p) {
    const int page = b.table[s * b.table_rs + (p >> kv.page_shift)];
    if (static_cast<uint32_t>(page) >= kv.pages) return nullptr;
    return kv.pool + page * kv.page_bytes + head * kv.head_bytes +
           static_cast<int64_t>((p & ((1 << kv.page_shift) - 1)) >> 4) * kv.block_bytes;
}

// Rows of heads side by side.
struct Rows {
    void* p;
    int64_t rs;  // elements
    bool vec;    // rows begin at multiples of 16 bytes
};

struct AppendArgs {
    int elem;
    KvDev kv;
    BatchDev batch;
    Rows q, q_out, k, v;
    int q_heads;      // 0: no queries
    const float *cos, *sin;
    int64_t turn_rs;
    int turned;       // channels that are rotated
    bool interleaved;
};
int run_kv4_append(uor_b200_ctx* ctx, const AppendArgs& a, uor_b200_route* route);

struct ReadArgs {
    int elem, out;
    KvDev kv;
    BatchDev batch;
    Rows k, v;
};
int run_kv4_read(uor_b200_ctx* ctx, const ReadArgs& a, uor_b200_route* route);

struct AttendArgs {
    int elem, out;
    KvDev kv;
    BatchDev batch;
    Rows q, y, lse;   // lse.p null: not wanted
    int share;        // query heads to a head of the cache
    float scale;
    int window, sinks;
};
// Few rows (kv4_few.cuh). EXACT: for f32 and float16 results.
template <typename T, bool EXACT>
int kv4_few(uor_b200_ctx* ctx, const AttendArgs& a, uor_b200_route* route);
// Many rows, 16-bit results (kv4_many.cuh).
template <typename T>
int kv4_many(uor_b200_ctx* ctx, const AttendArgs& a, uor_b200_route* route);
int run_kv4_attention(uor_b200_ctx* ctx, const AttendArgs& a, uor_b200_route* route);

}  // namespace uor
