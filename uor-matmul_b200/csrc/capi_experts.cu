// capi_experts.cu -- the C ABI of 4-bit weights with group scales and of the experts' layer:
// validation, staging of host buffers, dispatch.
#include <climits>
#include "internal.h"
#include "q4.cuh"
#include "staging.h"

using namespace uor;

namespace {

constexpr size_t MOST = static_cast<size_t>(INT_MAX) / 2;

bool half_type(uor_b200_dtype t) { return t == UOR_B200_BF16 || t == UOR_B200_F16; }

// Kernels read and write whole elements: a device address that is no multiple of their size faults
// there. Host arrays are copied, from any address.
bool at_element(const void* p, size_t rows, size_t cols, size_t es, bool device) {
    return !device || rows == 0 || cols == 0 || reinterpret_cast<uintptr_t>(p) % es == 0;
}

int place(const uor_b200_view* v, size_t es, bool device, Operand* o) {
    const int st = place_view(v->data, v->len, v->rows, v->cols, v->rs, v->cs, es, o);
    if (st) return st;
    return at_element(v->data, v->rows, v->cols, es, device) ? UOR_B200_OK : UOR_B200_INVALID_ARGUMENT;
}
int place(const uor_b200_view_mut* v, size_t es, bool device, Operand* o) {
    const int st = place_view(v->data, v->len, v->rows, v->cols, v->rs, v->cs, es, o);
    if (st) return st;
    if (self_aliases(v->rows, v->cols, v->rs, v->cs)) return UOR_B200_OUTPUT_ALIASES;
    return at_element(v->data, v->rows, v->cols, es, device) ? UOR_B200_OK : UOR_B200_INVALID_ARGUMENT;
}

// Whether (rows - 1) * stride + row elements are within len.
bool reaches(size_t rows, size_t stride, size_t row, size_t len) {
    if (rows == 0 || row == 0) return true;
    size_t last;
    if (__builtin_mul_overflow(rows - 1, stride, &last) || __builtin_add_overflow(last, row, &last))
        return false;
    return last <= len;
}

int check_q4(const uor_b200_q4* w, bool device) {
    if (!w) return UOR_B200_INVALID_ARGUMENT;
    if (w->group == 0 || w->group % 32 || w->group > MOST) return UOR_B200_INVALID_ARGUMENT;
    const auto type = static_cast<uor_b200_dtype>(w->scale_type);
    if (type != UOR_B200_F32 && !half_type(type)) return UOR_B200_UNSUPPORTED;
    if (w->rows > MOST || w->cols > MOST) return UOR_B200_UNSUPPORTED;
    const size_t groups = (w->cols + w->group - 1) / w->group;
    if (!reaches(w->rows, w->row_bytes, (w->cols + 1) / 2, w->codes_len) ||
        !reaches(w->rows, w->groups_rs, groups, w->scales_len) ||
        (w->zeros && !reaches(w->rows, w->groups_rs, groups, w->zeros_len)))
        return UOR_B200_DOES_NOT_FIT;
    if (w->row_bytes > static_cast<size_t>(PTRDIFF_MAX) || w->groups_rs > static_cast<size_t>(PTRDIFF_MAX))
        return UOR_B200_DOES_NOT_FIT;
    if (w->rows && w->cols && (!w->codes || !w->scales)) return UOR_B200_INVALID_ARGUMENT;
    return at_element(w->scales, w->rows, w->cols, dtype_size(type), device) ? UOR_B200_OK : UOR_B200_INVALID_ARGUMENT;
}

// Host operands travel to one device buffer together, each at a 256-byte boundary.
class Inputs {
  public:
    Inputs(uor_b200_ctx* ctx, bool device) : ctx_(ctx), device_(device) {}
    // Queues `bytes` at p; the device address is ready after copy().
    void add(const void* p, size_t bytes, const void** dev) {
        *dev = p;
        if (device_ || !p || !bytes) return;
        part_[n_++] = {p, bytes, total_, dev};
        total_ += (bytes + 255) / 256 * 256;
    }
    void add(const Operand& o, const void** dev) {
        if (device_ || o.rows == 0 || o.cols == 0) {
            *dev = o.origin;
            return;
        }
        back_[n_] = -o.lo * static_cast<ptrdiff_t>(o.es);
        add(o.origin + o.lo * static_cast<ptrdiff_t>(o.es), static_cast<size_t>(o.hi - o.lo + 1) * o.es, dev);
    }
    int copy() {
        if (!n_) return UOR_B200_OK;
        int st = UOR_B200_OK;
        auto* base = static_cast<uint8_t*>(ctx_buffer(ctx_, SLOT_A, total_, &st));
        if (!base) return st;
        for (int i = 0; i < n_; ++i) {
            if (cudaMemcpyAsync(base + part_[i].at, part_[i].host, part_[i].bytes, cudaMemcpyHostToDevice,
                                ctx_->stream) != cudaSuccess)
                return UOR_B200_DEVICE_ERROR;
            *part_[i].dev = base + part_[i].at + back_[i];
        }
        return UOR_B200_OK;
    }

  private:
    struct Part {
        const void* host;
        size_t bytes, at;
        const void** dev;
    };
    uor_b200_ctx* ctx_;
    bool device_;
    Part part_[12];
    ptrdiff_t back_[12] = {};
    int n_ = 0;
    size_t total_ = 0;
};

void add_q4(Inputs* in, const uor_b200_q4* w, Q4Dev* q) {
    const size_t groups = (w->cols + w->group - 1) / w->group;
    const size_t codes = w->rows && w->cols ? (w->rows - 1) * w->row_bytes + (w->cols + 1) / 2 : 0;
    const size_t scales = w->rows && w->cols ? (w->rows - 1) * w->groups_rs + groups : 0;
    q->row_bytes = static_cast<int64_t>(w->row_bytes);
    q->groups_rs = static_cast<int64_t>(w->groups_rs);
    q->rows = static_cast<int>(w->rows);
    q->cols = static_cast<int>(w->cols);
    q->group = static_cast<int>(w->group);
    q->scale_type = static_cast<int>(w->scale_type);
    in->add(w->codes, codes, reinterpret_cast<const void**>(&q->codes));
    in->add(w->scales, scales * dtype_size(static_cast<uor_b200_dtype>(w->scale_type)), &q->scales);
    in->add(w->zeros, scales, reinterpret_cast<const void**>(&q->zeros));
}

int check_call(const uor_b200_call* call, bool* device) {
    *device = call && (call->flags & UOR_B200_DEVICE_POINTERS);
    if (!call || call->encode == UOR_B200_NEAREST) return UOR_B200_OK;
    return call->encode > UOR_B200_WRAPPING ? UOR_B200_INVALID_ARGUMENT : UOR_B200_UNSUPPORTED;
}

uor_b200_route* clear_route(const uor_b200_call* call, uor_b200_route* local) {
    uor_b200_route* r = call && call->route ? call->route : local;
    *r = uor_b200_route{};
    return r;
}

int check_router(const uor_b200_router* r) {
    if (!r || r->score > UOR_B200_SIGMOID || r->renormalize > 1) return UOR_B200_INVALID_ARGUMENT;
    if (r->experts == 0 || r->top_k == 0 || r->groups == 0 || r->top_groups == 0) return UOR_B200_INVALID_ARGUMENT;
    if (r->experts > 1024 || r->top_k > 32 || r->groups > 32) return UOR_B200_UNSUPPORTED;
    if (r->experts % r->groups || r->top_groups > r->groups ||
        r->top_k > r->experts / r->groups * r->top_groups)
        return UOR_B200_INVALID_ARGUMENT;
    return UOR_B200_OK;
}

bool logits_type(uor_b200_dtype t) { return t == UOR_B200_F32 || half_type(t); }

}  // namespace

extern "C" {

int uor_b200_q4_gemm(uor_b200_dtype elem, uor_b200_dtype out, const uor_b200_view* a, const uor_b200_q4* w,
                     const uor_b200_view_mut* c, const uor_b200_call* call) {
    return uor_b200_q4_linear(elem, out, a, w, nullptr, 0, UOR_B200_F32, UOR_B200_IDENTITY, nullptr, c, call);
}

int uor_b200_q4_linear(uor_b200_dtype elem, uor_b200_dtype out, const uor_b200_view* a, const uor_b200_q4* w, const void* bias,
                       size_t bias_len, uor_b200_dtype bias_type, uint32_t activation, const uor_b200_view* residual,
                       const uor_b200_view_mut* c, const uor_b200_call* call) {
    if (!a || !c || activation > UOR_B200_SILU) return UOR_B200_INVALID_ARGUMENT;
    if (bias && bias_type != elem && bias_type != UOR_B200_F32) return UOR_B200_UNSUPPORTED;
    if (!half_type(elem) || (out != elem && out != UOR_B200_F32)) return UOR_B200_UNSUPPORTED;
    bool dev = false;
    Operand A, C;
    int st;
    if ((st = check_call(call, &dev)) || (st = check_q4(w, dev)) || (st = place(a, 2, dev, &A))) return st;
    if (a->cols != w->cols || c->rows != a->rows || c->cols != w->rows) return UOR_B200_NONCONFORMANT;
    if ((st = place(c, dtype_size(out), dev, &C))) return st;
    Operand R;
    if (residual) {
        if (residual->rows != c->rows || residual->cols != c->cols) return UOR_B200_NONCONFORMANT;
        if ((st = place(residual, dtype_size(out), dev, &R))) return st;
        // C itself, element by element, or no part of it
        if (R.origin == C.origin && ((R.rows > 1 && R.rs != C.rs) || (R.cols > 1 && R.cs != C.cs))) return UOR_B200_INVALID_ARGUMENT;
    }
    if (bias && bias_len < w->rows) return UOR_B200_DOES_NOT_FIT;
    if (bias && !at_element(bias, a->rows, w->rows, dtype_size(bias_type), dev)) return UOR_B200_INVALID_ARGUMENT;
    uor_b200_route local;
    uor_b200_route* route = clear_route(call, &local);
    if (a->rows == 0 || w->rows == 0) return UOR_B200_OK;
    if (a->rows > MOST) return UOR_B200_UNSUPPORTED;

    uor_b200_ctx* ctx = resolve_ctx(call, &st);
    if (!ctx) return st;
    std::lock_guard<std::mutex> lock(ctx->mu);
    DeviceTurn turn(ctx);
    Inputs in(ctx, dev);
    Mat x{nullptr, A.rs, A.cs};
    Q4Dev q{};
    in.add(A, &x.p);
    add_q4(&in, w, &q);
    Epilogue e{};
    e.act = static_cast<int>(activation);
    e.bias_type = bias_type;
    if (bias) in.add(bias, w->rows * dtype_size(bias_type), &e.bias);
    if (residual) {
        e.residual = Mat{nullptr, R.rs, R.cs};
        in.add(R, &e.residual.p);
    }
    e.on = bias || residual || activation != UOR_B200_IDENTITY;
    OutStage cs;
    if ((st = in.copy()) || (st = stage_out_begin(ctx, C, dev, false, &cs))) return st;
    if ((st = run_q4_gemm(ctx, elem, x, static_cast<int64_t>(a->rows), q, e, MatOut{cs.dev_origin, C.rs, C.cs, out},
                          route)))
        return st;
    if ((st = stage_out_end(ctx, cs))) return st;
    return dev ? finish_call(ctx, call) : uor_b200_ctx_sync(ctx);
}

int uor_b200_expert_route(uor_b200_dtype elem, const uor_b200_router* router, const uor_b200_view* logits,
                          const float* bias, size_t bias_len, const uor_b200_view_mut* ids,
                          const uor_b200_view_mut* weights, const uor_b200_call* call) {
    if (!logits || !ids || !weights) return UOR_B200_INVALID_ARGUMENT;
    if (!logits_type(elem)) return UOR_B200_UNSUPPORTED;
    bool dev = false;
    Operand L, I, W;
    int st;
    if ((st = check_call(call, &dev)) || (st = check_router(router)) || (st = place(logits, dtype_size(elem), dev, &L)))
        return st;
    const size_t t = logits->rows;
    if (logits->cols != router->experts || ids->rows != t || ids->cols != router->top_k || weights->rows != t ||
        weights->cols != router->top_k)
        return UOR_B200_NONCONFORMANT;
    if ((st = place(ids, 4, dev, &I)) || (st = place(weights, 4, dev, &W))) return st;
    if (bias && bias_len < router->experts) return UOR_B200_DOES_NOT_FIT;
    if (!at_element(bias, t, router->experts, sizeof(float), dev)) return UOR_B200_INVALID_ARGUMENT;
    uor_b200_route local;
    uor_b200_route* route = clear_route(call, &local);
    if (t == 0) return UOR_B200_OK;
    if (t > MOST) return UOR_B200_UNSUPPORTED;

    uor_b200_ctx* ctx = resolve_ctx(call, &st);
    if (!ctx) return st;
    std::lock_guard<std::mutex> lock(ctx->mu);
    DeviceTurn turn(ctx);
    Inputs in(ctx, dev);
    RouterArgs r{};
    r.r = *router;
    r.tokens = static_cast<int64_t>(t);
    r.elem = elem;
    r.logits = Mat{nullptr, L.rs, L.cs};
    in.add(L, &r.logits.p);
    in.add(bias, router->experts * sizeof(float), reinterpret_cast<const void**>(&r.bias));
    OutStage is, ws;
    if ((st = in.copy()) || (st = stage_out_begin(ctx, I, dev, false, &is)) ||
        (st = stage_out_begin(ctx, W, dev, false, &ws, SLOT_AUX)))
        return st;
    r.ids = MatOut{is.dev_origin, I.rs, I.cs, UOR_B200_I32};
    r.weights = MatOut{ws.dev_origin, W.rs, W.cs, UOR_B200_F32};
    if ((st = run_expert_route(ctx, r, route))) return st;
    if ((st = stage_out_end(ctx, is)) || (st = stage_out_end(ctx, ws))) return st;
    return dev ? finish_call(ctx, call) : uor_b200_ctx_sync(ctx);
}

int uor_b200_expert_route_backward(uor_b200_dtype elem, const uor_b200_router* router,
                                   const uor_b200_view* logits, const uor_b200_view* ids,
                                   const uor_b200_view* dweights, const uor_b200_view_mut* dlogits,
                                   const uor_b200_call* call) {
    if (!logits || !ids || !dweights || !dlogits) return UOR_B200_INVALID_ARGUMENT;
    if (!logits_type(elem)) return UOR_B200_UNSUPPORTED;
    bool dev = false;
    Operand L, I, G, D;
    int st;
    if ((st = check_call(call, &dev)) || (st = check_router(router)) || (st = place(logits, dtype_size(elem), dev, &L)))
        return st;
    const size_t t = logits->rows;
    if (logits->cols != router->experts || ids->rows != t || ids->cols != router->top_k || dweights->rows != t ||
        dweights->cols != router->top_k || dlogits->rows != t || dlogits->cols != router->experts)
        return UOR_B200_NONCONFORMANT;
    if ((st = place(ids, 4, dev, &I)) || (st = place(dweights, 4, dev, &G)) || (st = place(dlogits, dtype_size(elem), dev, &D)))
        return st;
    uor_b200_route local;
    uor_b200_route* route = clear_route(call, &local);
    if (t == 0) return UOR_B200_OK;
    if (t > MOST) return UOR_B200_UNSUPPORTED;

    uor_b200_ctx* ctx = resolve_ctx(call, &st);
    if (!ctx) return st;
    std::lock_guard<std::mutex> lock(ctx->mu);
    DeviceTurn turn(ctx);
    Inputs in(ctx, dev);
    RouterArgs r{};
    r.r = *router;
    r.tokens = static_cast<int64_t>(t);
    r.elem = elem;
    r.logits = Mat{nullptr, L.rs, L.cs};
    r.in_ids = Mat{nullptr, I.rs, I.cs};
    r.dweights = Mat{nullptr, G.rs, G.cs};
    in.add(L, &r.logits.p);
    in.add(I, &r.in_ids.p);
    in.add(G, &r.dweights.p);
    OutStage ds;
    if ((st = in.copy()) || (st = stage_out_begin(ctx, D, dev, false, &ds))) return st;
    r.dlogits = MatOut{ds.dev_origin, D.rs, D.cs, elem};
    if ((st = run_expert_route_backward(ctx, r, route))) return st;
    if ((st = stage_out_end(ctx, ds))) return st;
    return dev ? finish_call(ctx, call) : uor_b200_ctx_sync(ctx);
}

int uor_b200_expert_q4_ffn(uor_b200_dtype elem, uor_b200_dtype out, size_t experts, const uor_b200_view* x,
                           const uor_b200_view* ids, const uor_b200_view* weights, const uor_b200_q4* up,
                           const uor_b200_q4* down, const uor_b200_view_mut* y, const uor_b200_call* call) {
    if (!x || !ids || !weights || !y || experts == 0) return UOR_B200_INVALID_ARGUMENT;
    if (!half_type(elem) || (out != elem && out != UOR_B200_F32)) return UOR_B200_UNSUPPORTED;
    bool dev = false;
    Operand X, I, W, Y;
    int st;
    if ((st = check_call(call, &dev)) || (st = check_q4(up, dev)) || (st = check_q4(down, dev)) || (st = place(x, 2, dev, &X)) ||
        (st = place(ids, 4, dev, &I)) || (st = place(weights, 4, dev, &W)))
        return st;
    const size_t t = x->rows, d = x->cols, f = down->cols, k = ids->cols;
    if (experts > 1024) return UOR_B200_UNSUPPORTED;
    if (up->cols != d || up->rows != experts * 2 * f || down->rows != experts * d || ids->rows != t ||
        weights->rows != t || weights->cols != k || y->rows != t || y->cols != d)
        return UOR_B200_NONCONFORMANT;
    if ((st = place(y, dtype_size(out), dev, &Y))) return st;
    uor_b200_route local;
    uor_b200_route* route = clear_route(call, &local);
    if (t == 0 || d == 0) return UOR_B200_OK;
    size_t pairs;
    if (t > MOST || __builtin_mul_overflow(t, k, &pairs) || pairs > MOST) return UOR_B200_UNSUPPORTED;

    uor_b200_ctx* ctx = resolve_ctx(call, &st);
    if (!ctx) return st;
    std::lock_guard<std::mutex> lock(ctx->mu);
    DeviceTurn turn(ctx);
    Inputs in(ctx, dev);
    FfnArgs a{};
    a.elem = elem;
    a.tokens = static_cast<int64_t>(t);
    a.top_k = static_cast<int>(k);
    a.experts = static_cast<int>(experts);
    a.d = static_cast<int>(d);
    a.f = static_cast<int>(f);
    a.x = Mat{nullptr, X.rs, X.cs};
    a.ids = Mat{nullptr, I.rs, I.cs};
    a.weights = Mat{nullptr, W.rs, W.cs};
    in.add(X, &a.x.p);
    in.add(I, &a.ids.p);
    in.add(W, &a.weights.p);
    add_q4(&in, up, &a.up);
    add_q4(&in, down, &a.down);
    OutStage ys;
    if ((st = in.copy()) || (st = stage_out_begin(ctx, Y, dev, false, &ys))) return st;
    a.y = MatOut{ys.dev_origin, Y.rs, Y.cs, out};
    if ((st = run_expert_ffn(ctx, a, route))) return st;
    if ((st = stage_out_end(ctx, ys))) return st;
    return dev ? finish_call(ctx, call) : uor_b200_ctx_sync(ctx);
}

}  // extern "C"
