// capi_kv4.cu -- the C ABI of the 4-bit cache of keys and values and its attention: validation and
// dispatch. Device pointers only: a cache lives on its device.
#include <climits>
#include <cmath>
#include "internal.h"
#include "kv4.cuh"
#include "staging.h"

using namespace uor;

namespace {

constexpr size_t MOST = static_cast<size_t>(INT_MAX) / 2;

bool half_type(uint32_t t) { return t == UOR_B200_BF16 || t == UOR_B200_F16; }
bool multiple_of(const void* p, size_t by) { return reinterpret_cast<uintptr_t>(p) % by == 0; }
int log2_of(uint32_t v) { return 31 - __builtin_clz(v); }
bool power_of_two(uint32_t v) { return v && (v & (v - 1)) == 0; }

bool shape_ok(const uor_b200_kv4* c) {
    return power_of_two(c->page_size) && c->page_size >= 16 && c->page_size <= 4096 && c->heads >= 1 && c->heads <= 1024 &&
           (c->dim == 64 || c->dim == 96 || c->dim == 128 || c->dim == 192 || c->dim == 256) && power_of_two(c->group) &&
           c->group >= 32 && c->dim % c->group == 0 && half_type(c->elem);
}

int check_cache(const uor_b200_kv4* c, KvDev* kv) {
    if (!c) return UOR_B200_INVALID_ARGUMENT;
    if (!shape_ok(c) || c->pages > INT_MAX) return UOR_B200_UNSUPPORTED;
    kv->groups = static_cast<int>(c->dim / c->group);
    kv->block_bytes = kv_block_bytes(static_cast<int>(c->dim), kv->groups);
    kv->head_bytes = static_cast<int64_t>(c->page_size / KV_BLOCK) * kv->block_bytes;
    kv->page_bytes = kv->head_bytes * c->heads;
    size_t all;
    if (__builtin_mul_overflow(c->pages, static_cast<size_t>(kv->page_bytes), &all) || all > c->pool_len)
        return UOR_B200_DOES_NOT_FIT;
    if (c->pages * c->heads * (c->page_size / KV_BLOCK) > INT_MAX) return UOR_B200_UNSUPPORTED;  // blocks are numbered in 31 bits
    if (all && (!c->pool || !multiple_of(c->pool, 16))) return UOR_B200_INVALID_ARGUMENT;
    kv->pool = c->pool;
    kv->pages = static_cast<int64_t>(c->pages);
    kv->page_shift = log2_of(c->page_size);
    kv->heads = static_cast<int>(c->heads);
    kv->dim = static_cast<int>(c->dim);
    kv->group_shift = log2_of(c->group);
    return UOR_B200_OK;
}

int check_batch(const uor_b200_batch* b, size_t rows, const uor_b200_kv4* c, BatchDev* d) {
    if (!b) return UOR_B200_INVALID_ARGUMENT;
    const size_t capacity = b->table_cols <= MOST ? b->table_cols * c->page_size : SIZE_MAX;
    if (b->seqs > 4096 || rows > MOST || capacity > MOST || b->table_rs > static_cast<size_t>(PTRDIFF_MAX) / 4096)
        return UOR_B200_UNSUPPORTED;
    if (b->seqs) {
        const size_t reach = b->table_cols ? (b->seqs - 1) * b->table_rs + b->table_cols : 0;
        if (b->starts_len < b->seqs + 1 || b->lengths_len < b->seqs || b->table_len < reach) return UOR_B200_DOES_NOT_FIT;
        if (!b->starts || !b->lengths || (reach && !b->table)) return UOR_B200_INVALID_ARGUMENT;
        if (!multiple_of(b->starts, 4) || !multiple_of(b->lengths, 4) || !multiple_of(b->table, 4))
            return UOR_B200_INVALID_ARGUMENT;
    }
    d->starts = b->starts;
    d->lengths = b->lengths;
    d->table = b->table;
    d->table_rs = static_cast<int64_t>(b->table_rs);
    d->seqs = static_cast<int>(b->seqs);
    d->rows = static_cast<int>(rows);
    d->capacity = static_cast<int>(capacity);
    return UOR_B200_OK;
}

// A matrix whose rows' elements lie side by side.
template <typename V>
int place_rows(const V* v, size_t es, Rows* r) {
    Operand o;
    const int st = place_view(v->data, v->len, v->rows, v->cols, v->rs, v->cs, es, &o);
    if (st) return st;
    if (v->rows && v->cols && !multiple_of(v->data, es)) return UOR_B200_INVALID_ARGUMENT;
    if (v->cols > 1 && v->cs != 1) return UOR_B200_UNSUPPORTED;
    r->p = const_cast<uint8_t*>(o.origin);
    r->rs = v->rs;
    r->vec = (reinterpret_cast<uintptr_t>(o.origin) | static_cast<uintptr_t>(v->rs) * es) % 16 == 0;
    return UOR_B200_OK;
}
int place_out(const uor_b200_view_mut* v, size_t es, Rows* r) {
    const int st = place_rows(v, es, r);
    if (st) return st;
    return self_aliases(v->rows, v->cols, v->rs, v->cs) ? UOR_B200_OUTPUT_ALIASES : UOR_B200_OK;
}

int check_call(const uor_b200_call* call) {
    if (!call || !(call->flags & UOR_B200_DEVICE_POINTERS)) return UOR_B200_INVALID_ARGUMENT;
    if (call->encode == UOR_B200_NEAREST) return UOR_B200_OK;
    return call->encode > UOR_B200_WRAPPING ? UOR_B200_INVALID_ARGUMENT : UOR_B200_UNSUPPORTED;
}

int check_rotation(const uor_b200_rotation* t, const BatchDev& b, int dim, AppendArgs* a) {
    if (!t || t->dims == 0) return UOR_B200_OK;
    if (t->dims % 2 || t->dims > static_cast<uint32_t>(dim) || t->interleaved > 1) return UOR_B200_INVALID_ARGUMENT;
    if (t->rs > static_cast<size_t>(PTRDIFF_MAX)) return UOR_B200_UNSUPPORTED;
    size_t last = 0;
    if (t->positions < static_cast<size_t>(b.capacity)) return UOR_B200_DOES_NOT_FIT;
    if (t->positions && (__builtin_mul_overflow(t->positions - 1, t->rs, &last) ||
                         __builtin_add_overflow(last, static_cast<size_t>(t->dims / 2), &last) || last > t->len))
        return UOR_B200_DOES_NOT_FIT;
    if (last && (!t->cos || !t->sin || !multiple_of(t->cos, 4) || !multiple_of(t->sin, 4))) return UOR_B200_INVALID_ARGUMENT;
    a->cos = t->cos;
    a->sin = t->sin;
    a->turn_rs = static_cast<int64_t>(t->rs);
    a->turned = static_cast<int>(t->dims);
    a->interleaved = t->interleaved != 0;
    return UOR_B200_OK;
}

uor_b200_route* clear_route(const uor_b200_call* call, uor_b200_route* local) {
    uor_b200_route* r = call && call->route ? call->route : local;
    *r = uor_b200_route{};
    return r;
}

}  // namespace

extern "C" {

size_t uor_b200_kv4_page_bytes(const uor_b200_kv4* c) {
    if (!c || !shape_ok(c)) return 0;
    return static_cast<size_t>(c->page_size / KV_BLOCK) * c->heads *
           static_cast<size_t>(kv_block_bytes(static_cast<int>(c->dim), static_cast<int>(c->dim / c->group)));
}

int uor_b200_kv4_append(uor_b200_dtype elem, const uor_b200_kv4* cache, const uor_b200_batch* batch, const uor_b200_view* k,
                        const uor_b200_view* v, const uor_b200_view* q, const uor_b200_view_mut* q_out,
                        const uor_b200_rotation* rotation, const uor_b200_call* call) {
    if (!k || !v || (!q) != (!q_out)) return UOR_B200_INVALID_ARGUMENT;
    if (!half_type(elem)) return UOR_B200_UNSUPPORTED;
    AppendArgs a{};
    a.elem = elem;
    int st;
    if ((st = check_call(call)) || (st = check_cache(cache, &a.kv))) return st;
    if (cache->elem != static_cast<uint32_t>(elem)) return UOR_B200_UNSUPPORTED;
    const size_t rows = k->rows, wide = static_cast<size_t>(cache->heads) * cache->dim;
    if (k->cols != wide || v->rows != rows || v->cols != wide) return UOR_B200_NONCONFORMANT;
    if (q && (q->rows != rows || q_out->rows != rows || q_out->cols != q->cols || q->cols % cache->dim)) return UOR_B200_NONCONFORMANT;
    if ((st = check_batch(batch, rows, cache, &a.batch)) || (st = place_rows(k, 2, &a.k)) || (st = place_rows(v, 2, &a.v))) return st;
    if (q) {
        if (q->cols / cache->dim > 65536) return UOR_B200_UNSUPPORTED;
        if ((st = place_rows(q, 2, &a.q)) || (st = place_out(q_out, 2, &a.q_out))) return st;
        if (a.q.p == a.q_out.p && a.q.rs != a.q_out.rs && rows > 1 && q->cols) return UOR_B200_INVALID_ARGUMENT;
        a.q_heads = static_cast<int>(q->cols / cache->dim);
    }
    if ((st = check_rotation(rotation, a.batch, a.kv.dim, &a))) return st;
    uor_b200_route local;
    uor_b200_route* route = clear_route(call, &local);
    if (rows == 0 || batch->seqs == 0 || a.batch.capacity == 0) return UOR_B200_OK;

    uor_b200_ctx* ctx = resolve_ctx(call, &st);
    if (!ctx) return st;
    std::lock_guard<std::mutex> lock(ctx->mu);
    DeviceTurn turn(ctx);
    if ((st = run_kv4_append(ctx, a, route))) return st;
    return finish_call(ctx, call);
}

int uor_b200_kv4_read(uor_b200_dtype out, const uor_b200_kv4* cache, const uor_b200_batch* batch, const uor_b200_view_mut* k,
                      const uor_b200_view_mut* v, const uor_b200_call* call) {
    if (!k || !v) return UOR_B200_INVALID_ARGUMENT;
    ReadArgs a{};
    int st;
    if ((st = check_call(call)) || (st = check_cache(cache, &a.kv))) return st;
    if (static_cast<uint32_t>(out) != cache->elem && out != UOR_B200_F32) return UOR_B200_UNSUPPORTED;
    const size_t rows = k->rows, wide = static_cast<size_t>(cache->heads) * cache->dim;
    if (k->cols != wide || v->rows != rows || v->cols != wide) return UOR_B200_NONCONFORMANT;
    if ((st = check_batch(batch, rows, cache, &a.batch)) || (st = place_out(k, dtype_size(out), &a.k)) ||
        (st = place_out(v, dtype_size(out), &a.v)))
        return st;
    a.elem = static_cast<int>(cache->elem);
    a.out = out;
    uor_b200_route local;
    uor_b200_route* route = clear_route(call, &local);
    if (rows == 0 || batch->seqs == 0 || a.batch.capacity == 0) return UOR_B200_OK;

    uor_b200_ctx* ctx = resolve_ctx(call, &st);
    if (!ctx) return st;
    std::lock_guard<std::mutex> lock(ctx->mu);
    DeviceTurn turn(ctx);
    if ((st = run_kv4_read(ctx, a, route))) return st;
    return finish_call(ctx, call);
}

int uor_b200_kv4_attention(uor_b200_dtype elem, uor_b200_dtype out, const uor_b200_kv4* cache, const uor_b200_batch* batch,
                           const uor_b200_view* q, float scale, uint32_t window, uint32_t sinks, const uor_b200_view_mut* y,
                           const uor_b200_view_mut* lse, const uor_b200_call* call) {
    if (!q || !y) return UOR_B200_INVALID_ARGUMENT;
    if (!half_type(elem) || (out != elem && out != UOR_B200_F32)) return UOR_B200_UNSUPPORTED;
    if (!std::isfinite(scale)) return UOR_B200_INVALID_ARGUMENT;
    AttendArgs a{};
    int st;
    if ((st = check_call(call)) || (st = check_cache(cache, &a.kv))) return st;
    if (cache->elem != static_cast<uint32_t>(elem)) return UOR_B200_UNSUPPORTED;
    const size_t rows = q->rows, wide = static_cast<size_t>(cache->heads) * cache->dim;
    if (q->cols == 0 || q->cols % wide || y->rows != rows || y->cols != q->cols ||
        (lse && (lse->rows != rows || lse->cols != q->cols / cache->dim)))
        return UOR_B200_NONCONFORMANT;
    size_t heads_rows;  // rows of one head of the cache: 31 bits hold them
    if (__builtin_mul_overflow(rows, q->cols / wide, &heads_rows) || heads_rows > MOST) return UOR_B200_UNSUPPORTED;
    if ((st = check_batch(batch, rows, cache, &a.batch)) || (st = place_rows(q, 2, &a.q)) ||
        (st = place_out(y, dtype_size(out), &a.y)) || (lse && (st = place_out(lse, 4, &a.lse))))
        return st;
    a.elem = elem;
    a.out = out;
    a.share = static_cast<int>(q->cols / wide);
    a.scale = scale;
    // past every position one is as good as another
    a.window = static_cast<int>(window > MOST ? MOST : window);
    a.sinks = static_cast<int>(window == 0 ? 0 : sinks > MOST ? MOST : sinks);
    uor_b200_route local;
    uor_b200_route* route = clear_route(call, &local);
    if (rows == 0 || batch->seqs == 0) return UOR_B200_OK;

    uor_b200_ctx* ctx = resolve_ctx(call, &st);
    if (!ctx) return st;
    std::lock_guard<std::mutex> lock(ctx->mu);
    DeviceTurn turn(ctx);
    if ((st = run_kv4_attention(ctx, a, route))) return st;
    return finish_call(ctx, call);
}

}  // extern "C"
