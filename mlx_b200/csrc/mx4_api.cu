// Entry points of the microscaled 4-bit format and of the row step between two blocks (lux_gpu_quant_vtbl): argument checks, then
// one launch each on the context's stream.
#include "internal.h"
#include "mx4.cuh"

namespace luxcuda {

namespace {

size_t dtype_size(int dt) { return dt == LUX_DTYPE_FLOAT32 ? 4 : dt == LUX_DTYPE_BFLOAT16 ? 2 : 0; }

LuxBackendError invalid(const char* what) {
    set_last_error("%s", what);
    return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
}
bool aligned(const Buffer* b, size_t n) { return ((uintptr_t)b->ptr & (n - 1)) == 0; }
bool overlap(const void* a, size_t na, const void* b, size_t nb) {
    return na && nb && (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}
constexpr int kMaxK = INT32_MAX - 511;  // rounded up to what any kernel takes at a time it is still an int
size_t mx4_scale_bytes(int rows, int K, int format) {
    if (rows < 0 || K <= 0 || K > kMaxK || K % 32 || (format != LUX_CUDA_MX4_E8M0 && format != LUX_CUDA_MX4_E4M3)) return 0;
    return ((size_t)rows + 127) / 128 * mx4_tiles_k(K, format) * 512;
}
LuxBackendError check_format(int rows, int K, int format) {
    if (format != LUX_CUDA_MX4_E8M0 && format != LUX_CUDA_MX4_E4M3) {
        set_last_error("mx4: format must be LUX_CUDA_MX4_E8M0 or LUX_CUDA_MX4_E4M3 (got %d)", format);
        return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    }
    if (rows < 0 || K <= 0 || K > kMaxK || K % 32) {
        set_last_error("mx4: K=%d must be a positive multiple of 32, at most 2^31 - 512, the number of rows (%d) not negative", K, rows);
        return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    }
    return LUX_BACKEND_OK;
}
// codes and scales of [rows][K]: large enough, and where the copy engine can fetch them
LuxBackendError check_operand(const Context* c, const Buffer* codes, const Buffer* scales, int rows, int K, int format) {
    if (codes->dev != c->dev || scales->dev != c->dev) return invalid("mx4: a buffer of another device");
    if ((size_t)rows * K / 2 > codes->bytes || mx4_scale_bytes(rows, K, format) > scales->bytes) return invalid("mx4: codes or scales are smaller than their shape needs");
    if (!aligned(codes, 16) || !aligned(scales, 16)) return invalid("mx4: codes and scales must be 16-byte aligned");
    return LUX_BACKEND_OK;
}

LuxBackendError mx4_quantize(LuxBackendContext* ctx, LuxBackendBuffer* in, LuxBackendBuffer* codes, LuxBackendBuffer* scales, int rows, int K, size_t ld,
                             int format, LuxBackendDtype in_dtype, float pre) {
    Context* c = as_ctx(ctx);
    Buffer *bi = as_buf(in), *bc = as_buf(codes), *bs = as_buf(scales);
    if (!c || !bi || !bc || !bs) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    LuxBackendError e = check_format(rows, K, format);
    if (e == LUX_BACKEND_OK) e = check_operand(c, bc, bs, rows, K, format);
    if (e != LUX_BACKEND_OK) return e;
    const size_t is = dtype_size(in_dtype);
    if (!ld) ld = K;
    if (!is || ld < (size_t)K || ld > SIZE_MAX / 8 / ((size_t)rows + 1)) return invalid("mx4_quantize: in must be FLOAT32 or BFLOAT16, with a row stride of at least K");
    const size_t in_bytes = rows ? ((size_t)(rows - 1) * ld + K) * is : 0, code_bytes = (size_t)rows * K / 2, scale_bytes = mx4_scale_bytes(rows, K, format);
    if (bi->dev != c->dev || in_bytes > bi->bytes || !aligned(bi, is)) return invalid("mx4_quantize: in is of another device, too small or not aligned to its elements");
    if (overlap(bi->ptr, in_bytes, bc->ptr, code_bytes) || overlap(bi->ptr, in_bytes, bs->ptr, scale_bytes) || overlap(bc->ptr, code_bytes, bs->ptr, scale_bytes))
        return invalid("mx4_quantize: in, codes and scales overlap");
    if (!rows) return LUX_BACKEND_OK;
    std::lock_guard<std::mutex> lk(c->mu);
    DeviceGuard g(c->dev->device());
    // behind a chain kernel: at work beside it where neither touches what the other writes, else after it
    const bool chained = chain_is_open(c), known = !chained || c->chain_in_known;
    const bool ahead = chained && mx4_quantize_is_short(rows, K, c->dev->sm_count) && !chain_writes(c, bi->ptr, in_bytes) && !chain_writes(c, bc->ptr, code_bytes) &&
                       !chain_writes(c, bs->ptr, scale_bytes) && !chain_reads(c, bc->ptr, code_bytes) && !chain_reads(c, bs->ptr, scale_bytes);
    LUX_CUDA_TRY(launch_mx4_quantize(bi->ptr, (uint32_t*)bc->ptr, (uint8_t*)bs->ptr, rows, K, ld, format, (int)in_dtype, pre, c->stream, chained, ahead));
    c->launches++;
    note_early_chain_launch(c, chained);
    c->chain_out.add(bc->ptr, code_bytes);
    c->chain_out.add(bs->ptr, scale_bytes);
    c->chain_in.add(bi->ptr, in_bytes);
    c->chain_in_known = known;
    bi->last_stream = bc->last_stream = bs->last_stream = c->stream;
    return LUX_BACKEND_OK;
}

LuxBackendError mx4_dequantize(LuxBackendContext* ctx, LuxBackendBuffer* codes, LuxBackendBuffer* scales, LuxBackendBuffer* out, int rows, int K, int format,
                               LuxBackendDtype out_dtype, float post) {
    Context* c = as_ctx(ctx);
    Buffer *bc = as_buf(codes), *bs = as_buf(scales), *bo = as_buf(out);
    if (!c || !bc || !bs || !bo) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    LuxBackendError e = check_format(rows, K, format);
    if (e == LUX_BACKEND_OK) e = check_operand(c, bc, bs, rows, K, format);
    if (e != LUX_BACKEND_OK) return e;
    const size_t os = dtype_size(out_dtype);
    if (!os) return invalid("mx4_dequantize: out must be FLOAT32 or BFLOAT16");
    const size_t out_bytes = (size_t)rows * K * os;
    if (bo->dev != c->dev || out_bytes > bo->bytes || !aligned(bo, os)) return invalid("mx4_dequantize: out is of another device, too small or not aligned to its elements");
    if (overlap(bo->ptr, out_bytes, bc->ptr, (size_t)rows * K / 2) || overlap(bo->ptr, out_bytes, bs->ptr, mx4_scale_bytes(rows, K, format)))
        return invalid("mx4_dequantize: out overlaps codes or scales");
    if (!rows) return LUX_BACKEND_OK;
    std::lock_guard<std::mutex> lk(c->mu);
    DeviceGuard g(c->dev->device());
    LUX_CUDA_TRY(launch_mx4_dequantize((const uint32_t*)bc->ptr, (const uint8_t*)bs->ptr, bo->ptr, rows, K, format, (int)out_dtype, post, c->stream));
    c->launches++;
    bc->last_stream = bs->last_stream = bo->last_stream = c->stream;
    return LUX_BACKEND_OK;
}

LuxBackendError mx4_matmul(LuxBackendContext* ctx, LuxBackendBuffer* x_codes, LuxBackendBuffer* x_scales, LuxBackendBuffer* w_codes, LuxBackendBuffer* w_scales,
                           LuxBackendBuffer* y, int M, int K, int N, int format, LuxBackendDtype y_dtype, float alpha) {
    Context* c = as_ctx(ctx);
    Buffer *bx = as_buf(x_codes), *bxs = as_buf(x_scales), *bw = as_buf(w_codes), *bws = as_buf(w_scales), *by = as_buf(y);
    if (!c || !bx || !bxs || !bw || !bws || !by) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    LuxBackendError e = check_format(M, K, format);
    if (e == LUX_BACKEND_OK) e = check_format(N, K, format);
    if (e == LUX_BACKEND_OK) e = check_operand(c, bx, bxs, M, K, format);
    if (e == LUX_BACKEND_OK) e = check_operand(c, bw, bws, N, K, format);
    if (e != LUX_BACKEND_OK) return e;
    const size_t ys = dtype_size(y_dtype);
    if (!ys) return invalid("mx4_matmul: y must be FLOAT32 or BFLOAT16");
    const size_t y_bytes = (size_t)M * N * ys;
    if (by->dev != c->dev || y_bytes > by->bytes || !aligned(by, ys)) return invalid("mx4_matmul: y is of another device, too small or not aligned to its elements");
    if (overlap(by->ptr, y_bytes, bx->ptr, (size_t)M * K / 2) || overlap(by->ptr, y_bytes, bw->ptr, (size_t)N * K / 2) ||
        overlap(by->ptr, y_bytes, bxs->ptr, mx4_scale_bytes(M, K, format)) || overlap(by->ptr, y_bytes, bws->ptr, mx4_scale_bytes(N, K, format)))
        return invalid("mx4_matmul: y overlaps an operand");
    if (!M || !N) return LUX_BACKEND_OK;
    std::lock_guard<std::mutex> lk(c->mu);
    DeviceGuard g(c->dev->device());
    Mx4MatmulArgs a{(const uint32_t*)bx->ptr, (const uint8_t*)bxs->ptr, (const uint32_t*)bw->ptr, (const uint8_t*)bws->ptr, by->ptr, M, K, N, format, (int)y_dtype,
                    alpha, c->err_dev, false};
    // behind a chain kernel the weights may be fetched while it drains, unless it writes them
    const bool early = chain_is_open(c) && !chain_writes(c, a.wq, (size_t)N * K / 2) && !chain_writes(c, a.ws, mx4_scale_bytes(N, K, format));
    a.x_stable = early && !chain_writes(c, a.xq, (size_t)M * K / 2) && !chain_writes(c, a.xs, mx4_scale_bytes(M, K, format));
    const char* name = "";
    const cudaError_t r = launch_mx4_matmul(a, c->dev->sm_count, c->stream, early, &name);
    if (r != cudaSuccess) return map_cuda_error(r, name);
    c->launches++;
    note_chain_launch(c, by->ptr, y_bytes);
    c->chain_in.add(a.xq, (size_t)M * K / 2);
    c->chain_in.add(a.xs, mx4_scale_bytes(M, K, format));
    c->chain_in.add(a.wq, (size_t)N * K / 2);
    c->chain_in.add(a.ws, mx4_scale_bytes(N, K, format));
    c->chain_in_known = true;
    c->last_kernel = name;
    bx->last_stream = bxs->last_stream = bw->last_stream = bws->last_stream = by->last_stream = c->stream;
    return LUX_BACKEND_OK;
}

LuxBackendError block_norm(LuxBackendContext* ctx, const lux_block_norm_params* params, LuxBackendBuffer* h, LuxBackendBuffer* gate, LuxBackendBuffer* r,
                           LuxBackendBuffer* post_w, LuxBackendBuffer* post_b, LuxBackendBuffer* pre_w, LuxBackendBuffer* pre_b, LuxBackendBuffer* r_out,
                           LuxBackendBuffer* out, LuxBackendBuffer* out_scales) {
    Context* c = as_ctx(ctx);
    if (!c || !params) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    const lux_block_norm_params p = *params;
    enum { H, GATE, R, POST_W, POST_B, PRE_W, PRE_B, R_OUT, OUT, SCALES, COUNT };
    LuxBackendBuffer* const handles[COUNT] = {h, gate, r, post_w, post_b, pre_w, pre_b, r_out, out, out_scales};
    Buffer* b[COUNT];
    for (int i = 0; i < COUNT; i++) {
        b[i] = handles[i] ? as_buf(handles[i]) : nullptr;
        if (handles[i] && !b[i]) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
        if (b[i] && b[i]->dev != c->dev) return invalid("block_norm: a buffer of another device");
    }
    const size_t xs = dtype_size(p.x_dtype), rs = dtype_size(p.r_dtype), os = dtype_size(p.out_dtype);
    const bool mx = p.out_format != 0;
    auto norm_ok = [](int k) { return k == LUX_CUDA_NORM_NONE || k == LUX_CUDA_NORM_RMS || k == LUX_CUDA_NORM_LAYER; };
    if (!xs || !rs || (b[OUT] && !mx && !os)) return invalid("block_norm: dtypes must be FLOAT32 or BFLOAT16");
    if (!norm_ok(p.post_norm) || !norm_ok(p.pre_norm) || p.gate_act < LUX_CUDA_GATE_IDENTITY || p.gate_act > LUX_CUDA_GATE_TANH)
        return invalid("block_norm: unknown norm or gate function");
    if (!b[H] && !b[R]) return invalid("block_norm: neither h nor r");
    if (!b[R_OUT] && !b[OUT]) return invalid("block_norm: neither r_out nor out");
    if (!b[H] && (b[GATE] || b[POST_W] || b[POST_B] || p.post_norm)) return invalid("block_norm: gate or post norm without h");
    if ((b[POST_W] && p.post_norm == LUX_CUDA_NORM_NONE) || (b[PRE_W] && p.pre_norm == LUX_CUDA_NORM_NONE) ||
        (b[POST_B] && p.post_norm != LUX_CUDA_NORM_LAYER) || (b[PRE_B] && p.pre_norm != LUX_CUDA_NORM_LAYER))
        return invalid("block_norm: a weight without a norm, or a bias without a layer norm");
    if (mx && (!b[OUT] || !b[SCALES] || (p.out_format != LUX_CUDA_MX4_E8M0 && p.out_format != LUX_CUDA_MX4_E4M3) || p.dim % 32))
        return invalid("block_norm: out_format needs out, out_scales, a known format and dim a multiple of 32");
    if (!mx && b[SCALES]) return invalid("block_norm: out_scales without out_format");
    const size_t h_ld = p.h_ld ? p.h_ld : p.dim, gate_ld = p.gate_ld ? p.gate_ld : p.dim;
    if (!p.dim || p.dim > INT32_MAX || p.rows > INT32_MAX || h_ld < p.dim || gate_ld < p.dim || h_ld > (1ull << 31) || gate_ld > (1ull << 31))
        return invalid("block_norm: rows, dim or a row stride out of range");
    if (mx)
        if (LuxBackendError e = check_format((int)p.rows, (int)p.dim, p.out_format)) return e;
    if (!p.rows) return LUX_BACKEND_OK;
    const size_t gate_rows = p.gate_rows < p.rows ? p.gate_rows : 0;  // (from here on below 2^31: all rows share one beyond)
    const size_t gate_n = gate_rows ? (p.rows + gate_rows - 1) / gate_rows : 1;
    const size_t bytes[COUNT] = {((p.rows - 1) * h_ld + p.dim) * xs, ((gate_n - 1) * gate_ld + p.dim) * xs, p.rows * p.dim * rs, p.dim * 4, p.dim * 4, p.dim * 4,
                                 p.dim * 4, p.rows * p.dim * rs, mx ? p.rows * p.dim / 2 : p.rows * p.dim * os,
                                 mx ? mx4_scale_bytes((int)p.rows, (int)p.dim, p.out_format) : 0};
    const size_t element[COUNT] = {xs, xs, rs, 4, 4, 4, 4, rs, mx ? (size_t)16 : os, 16};
    for (int i = 0; i < COUNT; i++) {
        if (!b[i]) continue;
        if (bytes[i] > b[i]->bytes) return invalid("block_norm: a buffer is smaller than its shape needs");
        if (!aligned(b[i], element[i])) return invalid("block_norm: a buffer is not aligned to its elements (codes and scales: to 16 bytes)");
    }
    for (int o = R_OUT; o < COUNT; o++)
        for (int i = 0; i < COUNT && b[o]; i++) {
            if (!b[i] || i == o || (o == R_OUT && i == R && b[i]->ptr == b[o]->ptr)) continue;
            if (overlap(b[o]->ptr, bytes[o], b[i]->ptr, bytes[i])) return invalid("block_norm: what is written overlaps another buffer");
        }
    auto ptr = [&](int i) { return b[i] ? b[i]->ptr : nullptr; };
    auto vec = [&](int i, size_t ld, size_t es) { return !b[i] || (aligned(b[i], 16) && (ld * es % 16 == 0 || p.rows == 1)); };
    BlockNormArgs a;
    a.h = ptr(H); a.gate = ptr(GATE); a.r = ptr(R);
    a.post_w = (const float*)ptr(POST_W); a.post_b = (const float*)ptr(POST_B); a.pre_w = (const float*)ptr(PRE_W); a.pre_b = (const float*)ptr(PRE_B);
    a.r_out = ptr(R_OUT); a.out = ptr(OUT); a.out_scales = (uint8_t*)ptr(SCALES);
    a.rows = p.rows; a.dim = p.dim; a.h_ld = h_ld; a.gate_ld = gate_ld; a.gate_rows = gate_rows;
    a.post_kind = p.post_norm; a.pre_kind = p.pre_norm; a.gate_act = p.gate_act; a.out_format = p.out_format;
    a.x_bf16 = xs == 2; a.r_bf16 = rs == 2; a.out_bf16 = os == 2;
    a.vec = vec(H, h_ld, xs) && vec(GATE, gate_ld, xs) && vec(R, p.dim, rs) && vec(R_OUT, p.dim, rs) && (mx || vec(OUT, p.dim, os));
    for (int i = POST_W; i <= PRE_B; i++) a.vec = a.vec && vec(i, 0, 4);
    a.eps = p.eps; a.res_scale = p.res_scale; a.branch_scale = p.branch_scale; a.out_pre = p.out_pre; a.inv_dim = (float)(1.0 / (double)p.dim); a.error = c->err_dev;
    std::lock_guard<std::mutex> lk(c->mu);
    DeviceGuard g(c->dev->device());
    const bool chained = chain_is_open(c);
    LUX_CUDA_TRY(launch_block_norm(a, c->dev->sm_count, c->stream, chained));
    c->launches++;
    note_early_chain_launch(c, chained);
    for (int o = R_OUT; o < COUNT; o++)
        if (b[o]) c->chain_out.add(b[o]->ptr, bytes[o]);
    for (int i = 0; i < COUNT; i++)
        if (b[i]) b[i]->last_stream = c->stream;
    return LUX_BACKEND_OK;
}

}  // namespace

void fill_mx4_entries(lux_gpu_quant_vtbl* t) {
    t->mx4_scale_bytes = mx4_scale_bytes;
    t->mx4_quantize = mx4_quantize;
    t->mx4_dequantize = mx4_dequantize;
    t->mx4_matmul = mx4_matmul;
    t->block_norm = block_norm;
}

}  // namespace luxcuda
