// Entry points of the product with an epilogue and of a layer of experts (lux_gpu_quant_vtbl): argument checks, then the launches on the
// context's stream.
#include <algorithm>
#include <cstdlib>

#include "experts_plan.h"
#include "internal.h"

namespace luxcuda {

namespace {

size_t dtype_size(int dt) { return dt == LUX_DTYPE_FLOAT32 ? 4 : dt == LUX_DTYPE_BFLOAT16 ? 2 : 0; }

LuxBackendError invalid(const char* what) {
    set_last_error("%s", what);
    return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
}
bool overlap(const void* a, size_t na, const void* b, size_t nb) {
    return na && nb && (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}
bool act_ok(int act) { return act >= LUX_CUDA_ACT_NONE && act <= LUX_CUDA_ACT_GELU_TANH; }

// A call's buffers: handles in, then what each has to hold and on what boundary it has to begin.
struct Operand {
    LuxBackendBuffer* handle;
    bool needed;
    size_t bytes = 0, align = 1;
    bool written = false;
    Buffer* b = nullptr;
    void* ptr() const { return b ? b->ptr : nullptr; }
};
LuxBackendError resolve(const Context* c, Operand* o, int n, const char* call) {
    for (int i = 0; i < n; i++) {
        o[i].b = o[i].handle ? as_buf(o[i].handle) : nullptr;
        if (o[i].handle ? !o[i].b : o[i].needed) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
        if (o[i].b && o[i].b->dev != c->dev) {
            set_last_error("%s: a buffer of another device", call);
            return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
        }
    }
    return LUX_BACKEND_OK;
}
// in_place: the written operand that may be the read operand `of` itself
LuxBackendError check(const Operand* o, int n, const char* call, int in_place = -1, int of = -1) {
    for (int i = 0; i < n; i++) {
        if (!o[i].b) continue;
        if (o[i].bytes > o[i].b->bytes) {
            set_last_error("%s: a buffer is smaller than its shape needs", call);
            return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
        }
        if ((uintptr_t)o[i].b->ptr & (o[i].align - 1)) {
            set_last_error("%s: a buffer is not aligned (x, wq, scales, biases: 16 bytes; others: their elements)", call);
            return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
        }
    }
    for (int w = 0; w < n; w++)
        for (int i = 0; i < n && o[w].written && o[w].b; i++) {
            if (i == w || !o[i].b || (w == in_place && i == of && o[w].b->ptr == o[i].b->ptr)) continue;
            if (overlap(o[w].b->ptr, o[w].bytes, o[i].b->ptr, o[i].bytes)) {
                set_last_error("%s: what is written overlaps another buffer", call);
                return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
            }
        }
    return LUX_BACKEND_OK;
}
void note_use(Context* c, const Operand* o, int n) {
    for (int i = 0; i < n; i++)
        if (o[i].b) o[i].b->last_stream = c->stream;
}
// after a launch whose dependents start behind its wait: what it writes
void note_outputs(Context* c, const Operand* o, int n) {
    note_early_chain_launch(c, false);
    for (int i = 0; i < n; i++)
        if (o[i].b && o[i].written) c->chain_out.add(o[i].b->ptr, o[i].bytes);
}

// A workspace of the context of at least `bytes`: never made or grown while the stream is being recorded; an outgrown one stays for the graphs
// that were recorded with it.
LuxBackendError grow_workspace(Context* c, Block** ws, std::vector<Block*>* retired, size_t bytes, const char* call) {
    if (*ws && (*ws)->size >= bytes) return LUX_BACKEND_OK;
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(c->stream, &cap) == cudaSuccess && cap != cudaStreamCaptureStatusNone) {
        set_last_error("%s: this shape needs a larger workspace (%zu bytes); run it once outside the graph capture first", call, bytes);
        return LUX_BACKEND_ERROR_NOT_SUPPORTED;
    }
    // (twice the old one at least, where there is room: what is kept for graphs then stays below the one in use)
    cudaError_t e = cudaSuccess;
    Block* b = *ws ? c->dev->acquire(std::max(bytes, 2 * (*ws)->size), c->stream, &e) : nullptr;
    if (!b) b = c->dev->acquire(bytes, c->stream, &e);
    if (!b) return map_cuda_error(e, call);
    if (*ws) retired->push_back(*ws);
    *ws = b;
    return LUX_BACKEND_OK;
}

LuxBackendError check_format(const char* call, int K, int bits, int group) {
    if (bits != 4 && bits != 8) {
        set_last_error("%s: bits must be 4 or 8 (got %d)", call, bits);
        return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    }
    if (group != 32 && group != 64 && group != 128) {
        set_last_error("%s: group must be 32, 64 or 128 (got %d)", call, group);
        return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    }
    if (K <= 0 || K % group) {
        set_last_error("%s: K=%d must be a positive multiple of group=%d", call, K, group);
        return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    }
    return LUX_BACKEND_OK;
}

LuxBackendError qmatmul_epi(LuxBackendContext* ctx, const lux_qmm_epi_params* params, LuxBackendBuffer* x, LuxBackendBuffer* wq, LuxBackendBuffer* scales,
                            LuxBackendBuffer* biases, LuxBackendBuffer* bias, LuxBackendBuffer* residual, LuxBackendBuffer* y) {
    Context* c = as_ctx(ctx);
    if (!c || !params) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    const lux_qmm_epi_params p = *params;
    enum { X, WQ, SCALES, BIASES, BIAS, RES, Y, COUNT };
    Operand o[COUNT] = {{x, true}, {wq, true}, {scales, true}, {biases, true}, {bias, false}, {residual, false}, {y, true}};
    if (LuxBackendError e = resolve(c, o, COUNT, "qmatmul_epi")) return e;
    if (p.M < 0 || p.N < 0) return invalid("qmatmul_epi: M or N is negative");
    if (LuxBackendError e = check_format("qmatmul_epi", p.K, p.bits, p.group)) return e;
    const size_t ys = dtype_size(p.y_dtype), rs = dtype_size(p.r_dtype), M = p.M, N = p.N, K = p.K;
    if (!ys || (o[RES].b && !rs) || !act_ok(p.act)) return invalid("qmatmul_epi: dtypes must be FLOAT32 or BFLOAT16, act one of LUX_CUDA_ACT_*");
    o[X].bytes = M * K * 2, o[WQ].bytes = N * (K * p.bits / 8), o[SCALES].bytes = o[BIASES].bytes = N * (K / p.group) * 2;
    o[BIAS].bytes = N * 4, o[RES].bytes = M * N * rs, o[Y].bytes = M * N * ys;
    o[X].align = o[WQ].align = o[SCALES].align = o[BIASES].align = 16, o[BIAS].align = 4, o[RES].align = rs ? rs : 1, o[Y].align = ys;
    o[Y].written = true;
    if (LuxBackendError e = check(o, COUNT, "qmatmul_epi", Y, rs == ys ? RES : -1)) return e;
    if (!M || !N) return LUX_BACKEND_OK;
    std::lock_guard<std::mutex> lk(c->mu);
    DeviceGuard g(c->dev->device());
    QmmArgs a{o[X].ptr(), (const uint32_t*)o[WQ].ptr(), o[SCALES].ptr(), o[BIASES].ptr(), o[Y].ptr(), p.M, p.K, p.N, p.bits, p.group,
              (int)LUX_DTYPE_BFLOAT16, (int)LUX_DTYPE_BFLOAT16, p.y_dtype};
    a.epi = true;
    a.bias = (const float*)o[BIAS].ptr();
    a.residual = o[RES].ptr();
    a.act = p.act;
    a.r_bf16 = rs == 2;
    a.error = c->err_dev;
    const LuxBackendError r = qmatmul_epi_on_stream(c, a);
    note_use(c, o, COUNT);
    return r;
}

LuxBackendError moe_route(LuxBackendContext* ctx, const lux_moe_route_params* params, LuxBackendBuffer* logits, LuxBackendBuffer* bias, LuxBackendBuffer* ids,
                          LuxBackendBuffer* weights, LuxBackendBuffer* order, LuxBackendBuffer* pos, LuxBackendBuffer* offsets) {
    Context* c = as_ctx(ctx);
    if (!c || !params) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    const lux_moe_route_params p = *params;
    enum { LOGITS, BIAS, IDS, WEIGHTS, ORDER, POS, OFFSETS, COUNT };
    Operand o[COUNT] = {{logits, false}, {bias, false}, {ids, true}, {weights, logits != nullptr}, {order, true}, {pos, true}, {offsets, true}};
    if (LuxBackendError e = resolve(c, o, COUNT, "moe_route")) return e;
    const bool own_ids = o[LOGITS].b != nullptr;
    if (p.experts < 1 || p.experts > LUX_CUDA_MAX_EXPERTS || p.top_k < 1 || p.top_k > LUX_CUDA_MAX_TOP_K || (own_ids && p.top_k > p.experts))
        return invalid("moe_route: experts or top_k out of range");
    if (p.tokens > (uint64_t)INT32_MAX / p.top_k) return invalid("moe_route: tokens * top_k must be below 2^31");
    const size_t ld = p.ld ? p.ld : (size_t)p.experts, ls = own_ids ? dtype_size(p.logits_dtype) : 4, pairs = p.tokens * p.top_k;
    if (!ls || ld < (size_t)p.experts || ld > (1ull << 31)) return invalid("moe_route: logits must be FLOAT32 or BFLOAT16, with a row stride of at least experts");
    if (own_ids && p.score != LUX_CUDA_SCORE_SOFTMAX && p.score != LUX_CUDA_SCORE_SIGMOID) return invalid("moe_route: unknown score");
    if (o[BIAS].b && (!own_ids || p.score != LUX_CUDA_SCORE_SIGMOID)) return invalid("moe_route: a bias goes with logits and SCORE_SIGMOID only");
    o[LOGITS].bytes = p.tokens ? ((p.tokens - 1) * ld + p.experts) * ls : 0, o[LOGITS].align = ls;
    o[BIAS].bytes = (size_t)p.experts * 4;
    o[IDS].bytes = o[ORDER].bytes = o[POS].bytes = pairs * 4, o[WEIGHTS].bytes = own_ids ? pairs * 4 : 0;
    o[OFFSETS].bytes = ((size_t)p.experts + 1) * 4;
    for (int i = BIAS; i < COUNT; i++) o[i].align = 4;
    o[ORDER].written = o[POS].written = o[OFFSETS].written = true;
    o[IDS].written = o[WEIGHTS].written = own_ids;
    if (LuxBackendError e = check(o, COUNT, "moe_route")) return e;
    std::lock_guard<std::mutex> lk(c->mu);
    DeviceGuard g(c->dev->device());
    MoeRouteArgs a{o[LOGITS].ptr(), (const float*)o[BIAS].ptr(), (int*)o[IDS].ptr(), (float*)o[WEIGHTS].ptr(), (int*)o[ORDER].ptr(), (int*)o[POS].ptr(),
                   (int*)o[OFFSETS].ptr(), nullptr, (size_t)p.tokens, ld, p.experts, p.top_k, p.score, p.renorm, ls == 2, p.scale};
    if (moe_route_blocks(a, c->dev->sm_count) > 1) {
        if (LuxBackendError e = grow_workspace(c, &c->moe_ws, nullptr, moe_route_workspace_bytes(), "moe_route")) return e;
        a.hist = (int*)c->moe_ws->ptr;
    }
    int launches = 0;
    LUX_CUDA_TRY(launch_moe_route(a, c->dev->sm_count, c->stream, chain_is_open(c), &launches));
    c->launches += launches;
    c->last_kernel = "moe_route";
    note_outputs(c, o, COUNT);
    note_use(c, o, COUNT);
    return LUX_BACKEND_OK;
}

LuxBackendError qmatmul_experts(LuxBackendContext* ctx, const lux_experts_params* params, LuxBackendBuffer* x, LuxBackendBuffer* order, LuxBackendBuffer* offsets,
                                LuxBackendBuffer* wq, LuxBackendBuffer* scales, LuxBackendBuffer* biases, LuxBackendBuffer* bias, LuxBackendBuffer* y) {
    Context* c = as_ctx(ctx);
    if (!c || !params) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    const lux_experts_params p = *params;
    enum { X, ORDER, OFFSETS, WQ, SCALES, BIASES, BIAS, Y, COUNT };
    Operand o[COUNT] = {{x, true}, {order, false}, {offsets, true}, {wq, true}, {scales, true}, {biases, true}, {bias, false}, {y, true}};
    if (LuxBackendError e = resolve(c, o, COUNT, "qmatmul_experts")) return e;
    if (p.experts < 1 || p.experts > LUX_CUDA_MAX_EXPERTS || p.N < 0 || p.rows > INT32_MAX || p.x_rows > INT32_MAX) return invalid("qmatmul_experts: experts, N or rows out of range");
    if (LuxBackendError e = check_format("qmatmul_experts", p.K, p.bits, p.group)) return e;
    const size_t ys = dtype_size(p.y_dtype), E = p.experts, N = p.N, K = p.K, n_out = p.gated ? N / 2 : N;
    if (!ys || !act_ok(p.act)) return invalid("qmatmul_experts: y must be FLOAT32 or BFLOAT16, act one of LUX_CUDA_ACT_*");
    if (E * N > INT32_MAX) return invalid("qmatmul_experts: experts * N must be below 2^31");
    if (p.gated && N % 16) return invalid("qmatmul_experts: gated needs N a multiple of 16");
    if (o[ORDER].b && (p.top_k < 1 || p.top_k > LUX_CUDA_MAX_TOP_K)) return invalid("qmatmul_experts: top_k out of range");
    o[X].bytes = p.x_rows * K * 2, o[ORDER].bytes = p.rows * 4, o[OFFSETS].bytes = (E + 1) * 4;
    o[WQ].bytes = E * N * (K * p.bits / 8), o[SCALES].bytes = o[BIASES].bytes = E * N * (K / p.group) * 2, o[BIAS].bytes = E * N * 4, o[Y].bytes = p.rows * n_out * ys;
    o[X].align = o[WQ].align = o[SCALES].align = o[BIASES].align = 16, o[ORDER].align = o[OFFSETS].align = o[BIAS].align = 4, o[Y].align = ys;
    o[Y].written = true;
    if (LuxBackendError e = check(o, COUNT, "qmatmul_experts")) return e;
    if (!p.rows || !N) return LUX_BACKEND_OK;
    std::lock_guard<std::mutex> lk(c->mu);
    DeviceGuard g(c->dev->device());
    ExpertsArgs a{o[X].ptr(), (const int*)o[ORDER].ptr(), (const int*)o[OFFSETS].ptr(), (const uint32_t*)o[WQ].ptr(), o[SCALES].ptr(), o[BIASES].ptr(),
                  (const float*)o[BIAS].ptr(), o[Y].ptr(), (size_t)p.rows, (size_t)p.x_rows, p.experts, p.K, p.N, p.bits, p.group, p.top_k, p.act,
                  p.gated != 0, p.y_dtype, c->err_dev};
    // Few rows an expert: the decode kernel, which reads weights as fast as they come; many: the prefill GEMM.  LUXCUDA_EXPERTS = "few" | "many"
    // (experiments)
    const char* force = getenv("LUXCUDA_EXPERTS");
    const bool many = qmm_experts_supported(a), few = qmv_experts_supported(a, c->dev->sm_count);
    if (!many && !few) {
        set_last_error("qmatmul_experts: experts=%d K=%d N=%d in groups of %d is past the kernels' 32-bit index ranges", p.experts, p.K, p.N, p.group);
        return LUX_BACKEND_ERROR_NOT_SUPPORTED;
    }
    const bool use_many = many && (!few || (force ? force[0] == 'm' : experts_have_many_rows({a.rows, a.experts, a.K, a.N, a.bits, a.order != nullptr}, c->dev->sm_count)));
    const size_t room = use_many ? qmm_experts_workspace_bytes(a) : 0;
    if (room)
        if (LuxBackendError le = grow_workspace(c, &c->gather_ws, &c->gather_ws_retired, room, "qmatmul_experts")) return le;
    const char* name = "";
    const cudaError_t e = use_many ? launch_qmm_experts(a, room ? c->gather_ws->ptr : nullptr, c->dev->sm_count, c->stream, chain_is_open(c), &name)
                                   : launch_qmv_experts(a, c->dev->sm_count, c->stream, chain_is_open(c), &name);
    if (room) c->launches++;
    if (e != cudaSuccess) return map_cuda_error(e, name);
    c->launches++;
    c->last_kernel = name;
    note_outputs(c, o, COUNT);
    note_use(c, o, COUNT);
    return LUX_BACKEND_OK;
}

LuxBackendError moe_combine(LuxBackendContext* ctx, const lux_moe_combine_params* params, LuxBackendBuffer* y, LuxBackendBuffer* pos, LuxBackendBuffer* weights,
                            LuxBackendBuffer* residual, LuxBackendBuffer* out) {
    Context* c = as_ctx(ctx);
    if (!c || !params) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    const lux_moe_combine_params p = *params;
    enum { Y, POS, WEIGHTS, RES, OUT, COUNT };
    Operand o[COUNT] = {{y, true}, {pos, true}, {weights, false}, {residual, false}, {out, true}};
    if (LuxBackendError e = resolve(c, o, COUNT, "moe_combine")) return e;
    const size_t ys = dtype_size(p.y_dtype), os = dtype_size(p.out_dtype);
    if (!ys || !os) return invalid("moe_combine: dtypes must be FLOAT32 or BFLOAT16");
    if (p.top_k < 1 || p.top_k > LUX_CUDA_MAX_TOP_K || p.tokens > (uint64_t)INT32_MAX / p.top_k || p.dim > INT32_MAX || p.y_rows > INT32_MAX)
        return invalid("moe_combine: tokens, dim, top_k or y_rows out of range");
    o[Y].bytes = p.y_rows * p.dim * ys, o[POS].bytes = o[WEIGHTS].bytes = p.tokens * p.top_k * 4, o[RES].bytes = o[OUT].bytes = p.tokens * p.dim * os;
    o[Y].align = ys, o[POS].align = o[WEIGHTS].align = 4, o[RES].align = o[OUT].align = os;
    o[OUT].written = true;
    if (LuxBackendError e = check(o, COUNT, "moe_combine", OUT, RES)) return e;
    if (!p.tokens || !p.dim) return LUX_BACKEND_OK;
    int vec = 8;  // columns that lie together on a boundary of theirs in every row
    auto fits = [&](int i, size_t es) { return !o[i].b || ((uintptr_t)o[i].b->ptr & (std::min<size_t>(vec * es, 16) - 1)) == 0; };
    while (vec > 1 && !(p.dim % vec == 0 && fits(Y, ys) && fits(RES, os) && fits(OUT, os))) vec /= 2;
    const MoeCombineArgs a{o[Y].ptr(), (const int*)o[POS].ptr(), (const float*)o[WEIGHTS].ptr(), o[RES].ptr(), o[OUT].ptr(), (size_t)p.tokens, (size_t)p.dim, (size_t)p.y_rows,
                           p.top_k, ys == 2, os == 2, vec};
    std::lock_guard<std::mutex> lk(c->mu);
    DeviceGuard g(c->dev->device());
    LUX_CUDA_TRY(launch_moe_combine(a, c->dev->sm_count, c->stream, chain_is_open(c)));
    c->launches++;
    c->last_kernel = "moe_combine";
    note_outputs(c, o, COUNT);
    note_use(c, o, COUNT);
    return LUX_BACKEND_OK;
}

}  // namespace

void fill_moe_entries(lux_gpu_quant_vtbl* t) {
    t->qmatmul_epi = qmatmul_epi;
    t->moe_route = moe_route;
    t->qmatmul_experts = qmatmul_experts;
    t->moe_combine = moe_combine;
}

}  // namespace luxcuda
