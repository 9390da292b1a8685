// The 8-bit products' translation unit of libw4a8_b200.so.
#include "common.cuh"
#include "gemm_w8a8.cuh"

namespace w4a8 {

// The device-side error word of this translation unit, read and cleared (w4a8_device_status).
cudaError_t w8a8_take_device_error(unsigned int *v) {
    const unsigned int zero = 0;
    cudaError_t e = cudaMemcpyFromSymbol(v, g_dev_error, sizeof(*v));
    if (e == cudaSuccess && *v != 0) e = cudaMemcpyToSymbol(g_dev_error, &zero, sizeof(zero));
    return e;
}

}  // namespace w4a8

using namespace w4a8;

// What a product's arguments have to be; *empty: there is nothing to do.
static int check_product(const char *who, const int8_t *xq, const float *xs, const int8_t *wq, const float *ws, const float *bias, const void *Y, int64_t ldy, int M, int N, int K,
                         int dtype, bool *empty) {
    const size_t size = row_size(dtype);
    if (!size) return fail(W4A8_ERR_ARG, "%s: dtype=%d (0 fp32, 1 fp16, 2 bf16)", who, dtype);
    if (M < 0 || N < 0 || K < 0 || K % QBLK != 0) return fail(W4A8_ERR_ARG, "%s: M=%d N=%d K=%d (K must be a multiple of %d)", who, M, N, K, QBLK);
    if (K > w8a8::MAX_K) return fail(W4A8_ERR_UNSUPPORTED, "%s: K=%d (at most %d: sums have to fit 32 bits)", who, K, w8a8::MAX_K);
    if (M > w8a8::MAX_ROWS || N > w8a8::MAX_ROWS) return fail(W4A8_ERR_UNSUPPORTED, "%s: M=%d N=%d (at most %d: places in the last tiles are counted in 31 bits)", who, M, N, w8a8::MAX_ROWS);
    *empty = M == 0 || N == 0;
    if (*empty) return W4A8_OK;
    if (K == 0) return fail(W4A8_ERR_ARG, "%s: K=0", who);
    if (!xq || !xs || !wq || !ws || !Y) return fail(W4A8_ERR_ARG, "%s: null pointer argument", who);
    if (ldy < N) return fail(W4A8_ERR_ARG, "%s: Y has rows of %d elements, a pitch of %lld", who, N, (long long)ldy);
    if (!aligned(xq, 16) || !aligned(wq, 16)) return fail(W4A8_ERR_ALIGN, "%s: xq and wq must be 16-byte aligned", who);
    if (!aligned(xs, 4) || !aligned(ws, 4) || (bias && !aligned(bias, 4)) || !aligned(Y, size)) return fail(W4A8_ERR_ALIGN, "%s: pointers must be aligned to their elements", who);
    const Rows y = {Y, ldy, N, M, size}, in[] = {{xq, K, K, M, 1}, {xs, M, M, 1, 4}, {wq, K, K, N, 1}, {ws, N, N, 1, 4}, {bias, N, N, 1, 4}};
    static const char *const names[] = {"xq", "xs", "wq", "ws", "bias"};
    for (int i = 0; i < 5; i++)
        if (rows_overlap(y, in[i])) return fail(W4A8_ERR_ARG, "%s: Y overlaps %s", who, names[i]);
    return W4A8_OK;
}

W4A8_API int w4a8_gemm_w8a8(const int8_t *xq, const float *xs, const int8_t *wq, const float *ws, const float *bias, void *Y, int64_t ldy, int M, int N, int K,
                            int dtype, void *stream) {
    bool empty;
    int rc = check_product("gemm_w8a8", xq, xs, wq, ws, bias, Y, ldy, M, N, K, dtype, &empty);
    if (rc != W4A8_OK || empty || (rc = require_sm100()) != W4A8_OK) return rc;
    w8a8::Args a = {xs, ws, bias, Y, ldy, M, N, K};
    w8a8::Plan plan;
    if ((rc = w8a8::plan_cached(M, N, K, &plan)) != W4A8_OK) return rc;
    return w8a8::launch(xq, wq, a, plan, dtype, (cudaStream_t)stream);
}

W4A8_API int w4a8_linear_w8a8(const void *x, int64_t ldx, int8_t *xq, float *xs, const int8_t *wq, const float *ws, const float *bias, void *Y, int64_t ldy,
                              int S, int N, int K, int x_dtype, int y_dtype, int skip_quantize, void *stream) {
    if (S > 0 && N > 0 && !skip_quantize && !x) return fail(W4A8_ERR_ARG, "linear_w8a8: null pointer argument");
    bool empty;
    int rc = check_product("linear_w8a8", xq, xs, wq, ws, bias, Y, ldy, S, N, K, y_dtype, &empty);      // before the first of the two launches
    if (rc != W4A8_OK || empty) return rc;
    if (!skip_quantize) {
        const size_t size = row_size(x_dtype);
        w8a8::Plan plan;
        const Rows in = {size && ldx >= K ? x : nullptr, ldx, K, S, size}, codes = {xq, K, K, S, 1}, scales = {xs, S, S, 1, 4}, y = {Y, ldy, N, S, row_size(y_dtype)};
        // codes and scales are written while CTAs still read weights (one launch) or before they do (two)
        const Rows read[] = {in, {wq, K, K, N, 1}, {ws, N, N, 1, 4}, {bias, N, N, 1, 4}, codes};
        static const char *const names[] = {"x", "wq", "ws", "bias", "xq"};
        for (int i = 0; i < 5; i++) {
            if (i < 4 && rows_overlap(codes, read[i])) return fail(W4A8_ERR_ARG, "linear_w8a8: xq overlaps %s", names[i]);
            if (rows_overlap(scales, read[i])) return fail(W4A8_ERR_ARG, "linear_w8a8: xs overlaps %s", names[i]);
        }
        // a row or two by the product itself (what is not right with x is the quantizer's to say; an output in x's place needs x read first)
        if (S <= w8a8::ROWS_MAX && in.p && K <= 32768 && aligned(x, 16) && ldx * size % 16 == 0 && !rows_overlap(y, in) && (rc = require_sm100()) == W4A8_OK && (rc = w8a8::plan_cached(S, N, K, &plan)) == W4A8_OK &&
            w8a8::row_plan(plan, S, K)) {
            w8a8::Args a = {xs, ws, bias, Y, ldy, S, N, K};
            a.x = x; a.ldx = ldx; a.x_dtype = x_dtype; a.xq_out = xq; a.xs_out = xs;
            return w8a8::launch(xq, wq, a, plan, y_dtype, (cudaStream_t)stream);
        }
        if (rc != W4A8_OK || (rc = w4a8_quantize_rows_q8(x, ldx, S, K, x_dtype, xq, xs, stream)) != W4A8_OK) return rc;
    }
    return w4a8_gemm_w8a8(xq, xs, wq, ws, bias, Y, ldy, S, N, K, y_dtype, stream);
}
