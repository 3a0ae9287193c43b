// kv4_attend.cu -- which kernel an attention over the 4-bit cache runs.
#include "kv4.cuh"

namespace uor {

int run_kv4_attention(uor_b200_ctx* ctx, const AttendArgs& a, uor_b200_route* route) {
    route->kernel = UOR_B200_KERNEL_KV4;
    if (a.out == UOR_B200_F32)
        return a.elem == UOR_B200_BF16 ? kv4_few<__nv_bfloat16, true>(ctx, a, route) : kv4_few<__half, true>(ctx, a, route);
    // Rows of one head that a sequence has on average.
    const int64_t rows = static_cast<int64_t>(a.batch.rows) * a.share / a.batch.seqs;
    if (rows > 64) return a.elem == UOR_B200_BF16 ? kv4_many<__nv_bfloat16>(ctx, a, route) : kv4_many<__half>(ctx, a, route);
    return a.elem == UOR_B200_BF16 ? kv4_few<__nv_bfloat16, false>(ctx, a, route) : kv4_few<__half, false>(ctx, a, route);
}

}  // namespace uor
