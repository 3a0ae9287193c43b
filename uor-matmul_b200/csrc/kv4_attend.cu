// kv4_attend.cu -- which kernel an attention over the 4-bit cache runs.
#include "kv4.cuh"

namespace uor {

int run_kv4_attention(uor_b200_ctx* ctx, const AttendArgs& a, uor_b200_route* route) {
    route->kernel = UOR_B200_KERNEL_KV4;
    // The many-rows kernel has a row tile's whole context to one processor, 1.85 us for 64 tokens; the
    // few-rows kernel cuts contexts up and takes 210 tiles of 16 rows by 64 tokens in a microsecond, all
    // processors together. Both grow with the contexts alike, so the rows decide. bfloat16, 8 heads of 128
    // channels with 4 queries each, few : many: 1 sequence with 17 new tokens in 4096 25 : 121 us; 8 with 16
    // 78 : 126, with 32 151 : 126; 16 with 16 in 1000 58 : 46. f32 results need the exact weights that the
    // few-rows kernel alone has.
    const int64_t rows = static_cast<int64_t>(a.batch.rows) * a.share, mean = (rows + a.batch.seqs - 1) / a.batch.seqs;
    const int64_t lines = static_cast<int64_t>(a.batch.seqs) * a.kv.heads, tile = a.kv.dim <= 128 ? 256 : 128;
    const int64_t waves = (lines * ((mean + tile - 1) / tile) + ctx->sm_count - 1) / ctx->sm_count;
    if (a.out != UOR_B200_F32 && mean > 16 && lines * ((mean + 15) / 16) > 390 * waves)
        return a.elem == UOR_B200_BF16 ? kv4_many<__nv_bfloat16>(ctx, a, route) : kv4_many<__half>(ctx, a, route);
    if (a.elem == UOR_B200_F16) return kv4_few<__half, true>(ctx, a, route);
    return a.out == UOR_B200_F32 ? kv4_few<__nv_bfloat16, true>(ctx, a, route) : kv4_few<__nv_bfloat16, false>(ctx, a, route);
}

}  // namespace uor
