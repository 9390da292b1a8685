// The layer operators' translation unit of libw4a8_b200.so: residual add and norms, rotary positions, the choice of experts.
#include "common.cuh"
#include "rows.cuh"
#include "add_norm.cuh"
#include "rope.cuh"
#include "moe_route.cuh"

using namespace w4a8;

static int check_rows(const void *p, int64_t ld, int64_t columns, size_t size, const char *name, const char *who) {
    if (ld < columns) return fail(W4A8_ERR_ARG, "%s: %s has rows of %lld elements, a pitch of %lld", who, name, (long long)columns, (long long)ld);
    if (!aligned(p, 16) || ((uint64_t)ld * size) % 16 != 0) return fail(W4A8_ERR_ALIGN, "%s: %s and its rows must be 16-byte aligned", who, name);
    return W4A8_OK;
}
// Every output against every input and every other output; `in_place` pairs may be the same memory.
static int check_apart(const char *who, const Rows *r, const char *const *names, int count, int first_out, bool (*in_place)(int out, int in)) {
    for (int o = first_out; o < count; o++)
        for (int i = 0; i < o; i++)
            if (rows_overlap(r[o], r[i]) && !(i < first_out && in_place(o, i) && r[o].same(r[i])))
                return fail(W4A8_ERR_ARG, "%s: %s overlaps %s", who, names[o], names[i]);
    return W4A8_OK;
}
static bool variant_ok(int v) { return v >= W4A8_NORM_NONE && v <= W4A8_NORM_NO_SCALE; }

W4A8_API int w4a8_add_norm(const w4a8_norm *norm, const void *h, int64_t ldh, const void *y, int64_t ldy, void *h_out, int64_t ldo, void *n_out, int64_t ldn,
                           int8_t *xq, float *xs, int32_t *xsum, int group, int S, void *stream) {
    const char *who = "add_norm";
    if (!norm) return fail(W4A8_ERR_ARG, "%s: null norm", who);
    const int K = norm->K;
    const size_t size = row_size(norm->dtype), ysize = row_size(norm->y_dtype);
    if (S < 0 || K < 0 || K % QBLK != 0) return fail(W4A8_ERR_ARG, "%s: K=%d S=%d (K must be a multiple of %d)", who, K, S, QBLK);
    if (!size || (y && !ysize)) return fail(W4A8_ERR_ARG, "%s: dtype=%d y_dtype=%d (0 fp32, 1 fp16, 2 bf16)", who, norm->dtype, norm->y_dtype);
    if (y && norm->y_dtype != norm->dtype && norm->y_dtype != W4A8_F32) return fail(W4A8_ERR_ARG, "%s: y_dtype=%d (h's type or fp32)", who, norm->y_dtype);
    if (!variant_ok(norm->variant) || !variant_ok(norm->post_variant)) return fail(W4A8_ERR_ARG, "%s: variant=%d post_variant=%d (-1 none, 0 scale, 1 one-plus-scale, 2 no scale)", who, norm->variant, norm->post_variant);
    if (!(norm->eps >= 0.0)) return fail(W4A8_ERR_ARG, "%s: eps=%g", who, norm->eps);
    if (K > addnorm::MAX_K) return fail(W4A8_ERR_UNSUPPORTED, "%s: rows of %d elements (at most %d)", who, K, addnorm::MAX_K);
    if (group != 0 && group != 32) return fail(W4A8_ERR_ARG, "%s: group=%d (32, or 0: one scale for a row)", who, group);
    if (S == 0 || K == 0) return W4A8_OK;
    const bool takes_w = norm->variant == W4A8_NORM_SCALE || norm->variant == W4A8_NORM_ONE_PLUS;
    const bool takes_pw = y && (norm->post_variant == W4A8_NORM_SCALE || norm->post_variant == W4A8_NORM_ONE_PLUS);
    if (!h || (takes_w && !norm->weight) || (takes_pw && !norm->post_weight) || (xq && !xs)) return fail(W4A8_ERR_ARG, "%s: null pointer argument", who);
    if (!h_out && !n_out && !xq) return fail(W4A8_ERR_ARG, "%s: no output", who);
    if (!xq && (xs || xsum)) return fail(W4A8_ERR_ARG, "%s: xs or xsum without xq", who);
    if (group == 0 && xsum) return fail(W4A8_ERR_ARG, "%s: rows of one scale have no xsum", who);
    int rc;
    if ((rc = check_rows(h, ldh, K, size, "h", who)) != W4A8_OK || (y && (rc = check_rows(y, ldy, K, ysize, "y", who)) != W4A8_OK) ||
        (h_out && (rc = check_rows(h_out, ldo, K, size, "h_out", who)) != W4A8_OK) || (n_out && (rc = check_rows(n_out, ldn, K, size, "n_out", who)) != W4A8_OK))
        return rc;
    const bool gate_rows = y && norm->gate && norm->gate_ld != 0;
    if (y && norm->gate && (rc = check_rows(norm->gate, gate_rows ? norm->gate_ld : K, K, 4, "gate", who)) != W4A8_OK) return rc;
    if ((takes_w && !aligned(norm->weight, 16)) || (takes_pw && !aligned(norm->post_weight, 16)) || (xq && !aligned(xq, 16)) || (xs && !aligned(xs, 4)) || (xsum && !aligned(xsum, 4)))
        return fail(W4A8_ERR_ALIGN, "%s: weights and xq must be 16-byte aligned, xs and xsum 4-byte", who);
    const int64_t scales = group ? K / 32 : 1;
    const Rows r[] = {{h, ldh, K, S, size}, {y, ldy, K, S, ysize}, {takes_w ? norm->weight : nullptr, K, K, 1, 4}, {takes_pw ? norm->post_weight : nullptr, K, K, 1, 4},
                      {y ? norm->gate : nullptr, gate_rows ? norm->gate_ld : K, K, gate_rows ? S : 1, 4},
                      {h_out, ldo, K, S, size}, {n_out, ldn, K, S, size}, {xq, K, K, S, 1}, {xs, scales, scales, S, 4}, {xsum, scales, scales, S, 4}};
    static const char *const names[] = {"h", "y", "weight", "post_weight", "gate", "h_out", "n_out", "xq", "xs", "xsum"};
    if ((rc = check_apart(who, r, names, 10, 5, [](int o, int i) { return (o == 5 && i == 0) || (o == 6 && i <= 1); })) != W4A8_OK) return rc;
    if ((rc = require_sm100()) != W4A8_OK) return rc;
    addnorm::Args a = {h, y, h_out, n_out, norm->weight, norm->post_weight, norm->gate, ldh, ldy, ldo, ldn, gate_rows ? norm->gate_ld : 0, xq, xs, xsum,
                       1.0 / K, norm->eps, norm->alpha, K, norm->variant, norm->post_variant, group};
    return addnorm::launch(a, S, norm->dtype, y ? norm->y_dtype : norm->dtype, (cudaStream_t)stream);
}

W4A8_API int w4a8_quantize_rows_q8(const void *x, int64_t ldx, int S, int K, int dtype, int8_t *xq, float *xs, void *stream) {
    const w4a8_norm plain = {nullptr, nullptr, nullptr, 0, 0.0, 1.f, K, W4A8_NORM_NONE, W4A8_NORM_NONE, dtype, dtype};
    if (S > 0 && K > 0 && (!x || !xq || !xs)) return fail(W4A8_ERR_ARG, "quantize_rows_q8: null pointer argument");
    return w4a8_add_norm(&plain, x, ldx, nullptr, 0, nullptr, 0, nullptr, 0, xq, xs, nullptr, 0, S, stream);
}

W4A8_API int w4a8_rope_table(int rotary, double base, int scaling, double factor, double original, double low, double high, const double *divisor, uint64_t *turns_host,
                             float *magnitude) {
    const char *who = "rope_table";
    if (rotary < 0 || rotary % 2 != 0 || rotary > 1024) return fail(W4A8_ERR_ARG, "%s: rotary=%d (a multiple of 2, at most 1024)", who, rotary);
    if (!(base > 0.0 && base <= 1e30)) return fail(W4A8_ERR_ARG, "%s: base=%g", who, base);
    if (scaling < W4A8_ROPE_NONE || scaling > W4A8_ROPE_DIVISORS) return fail(W4A8_ERR_ARG, "%s: scaling=%d", who, scaling);
    const bool by_factor = scaling >= W4A8_ROPE_LINEAR && scaling <= W4A8_ROPE_BANDS, by_turns = scaling == W4A8_ROPE_YARN || scaling == W4A8_ROPE_BANDS;
    if (by_factor && !(factor > 0.0 && factor <= 1e9)) return fail(W4A8_ERR_ARG, "%s: factor=%g", who, factor);
    if (by_turns && (!(original > 0.0 && original <= 1e12) || !(low >= 0.0 && high >= 0.0) || !((high > 0 ? high : scaling == W4A8_ROPE_YARN ? 32 : 4) > (low > 0 ? low : 1))))
        return fail(W4A8_ERR_ARG, "%s: original=%g low=%g high=%g", who, original, low, high);
    if (scaling == W4A8_ROPE_YARN && base == 1.0) return fail(W4A8_ERR_ARG, "%s: base=%g", who, base);
    if (!magnitude || (rotary && !turns_host) || (scaling == W4A8_ROPE_DIVISORS && rotary && !divisor)) return fail(W4A8_ERR_ARG, "%s: null pointer argument", who);
    if (scaling == W4A8_ROPE_DIVISORS)
        for (int i = 0; i < rotary / 2; i++)
            if (!(divisor[i] > 0.0)) return fail(W4A8_ERR_ARG, "%s: divisor[%d]=%g", who, i, divisor[i]);
    if (!rope::table(rotary, base, scaling, factor, original, low, high, divisor, turns_host, magnitude)) return fail(W4A8_ERR_ARG, "%s: a frequency that is not a number or too large", who);
    return W4A8_OK;
}

W4A8_API int w4a8_rope_qk(const w4a8_rope *r, const void *q, int64_t ldq, int heads_q, const void *k, int64_t ldk, int heads_k, const int32_t *position, int T,
                          void *q_out, int64_t ldqo, void *k_out, int64_t ldko, int dtype, void *stream) {
    const char *who = "rope_qk";
    if (!r) return fail(W4A8_ERR_ARG, "%s: null rope", who);
    const size_t size = row_size(dtype);
    if (!size) return fail(W4A8_ERR_ARG, "%s: dtype=%d (0 fp32, 1 fp16, 2 bf16)", who, dtype);
    if (T < 0 || heads_q < 0 || heads_k < 0 || heads_q > 65535 || heads_k > 65535) return fail(W4A8_ERR_ARG, "%s: T=%d heads_q=%d heads_k=%d", who, T, heads_q, heads_k);
    if (r->dim <= 0 || r->dim % 8 != 0 || r->dim > rope::MAX_DIM) return fail(W4A8_ERR_ARG, "%s: dim=%d (a multiple of 8, at most %d)", who, r->dim, rope::MAX_DIM);
    if (r->rotary < 0 || r->rotary % 8 != 0 || r->rotary > r->dim) return fail(W4A8_ERR_ARG, "%s: rotary=%d (a multiple of 8, at most dim=%d)", who, r->rotary, r->dim);
    if (!variant_ok(r->variant) || !(r->eps >= 0.0)) return fail(W4A8_ERR_ARG, "%s: variant=%d (-1 none, 0 scale, 1 one-plus-scale, 2 no scale) eps=%g", who, r->variant, r->eps);
    if (T == 0 || heads_q + heads_k == 0) return W4A8_OK;
    const bool takes_w = r->variant == W4A8_NORM_SCALE || r->variant == W4A8_NORM_ONE_PLUS;
    if (!position || (r->rotary && !r->turns) || (heads_q && (!q || !q_out || (takes_w && !r->q_weight))) || (heads_k && (!k || !k_out || (takes_w && !r->k_weight))))
        return fail(W4A8_ERR_ARG, "%s: null pointer argument", who);
    const int64_t nq = (int64_t)heads_q * r->dim, nk = (int64_t)heads_k * r->dim;
    int rc;
    if ((heads_q && ((rc = check_rows(q, ldq, nq, size, "q", who)) != W4A8_OK || (rc = check_rows(q_out, ldqo, nq, size, "q_out", who)) != W4A8_OK)) ||
        (heads_k && ((rc = check_rows(k, ldk, nk, size, "k", who)) != W4A8_OK || (rc = check_rows(k_out, ldko, nk, size, "k_out", who)) != W4A8_OK)))
        return rc;
    if (takes_w && ((heads_q && !aligned(r->q_weight, 16)) || (heads_k && !aligned(r->k_weight, 16)))) return fail(W4A8_ERR_ALIGN, "%s: weights must be 16-byte aligned", who);
    if (r->rotary && !aligned(r->turns, 8)) return fail(W4A8_ERR_ALIGN, "%s: turns must be 8-byte aligned", who);
    const Rows rows[] = {{heads_q ? q : nullptr, ldq, nq, T, size}, {heads_k ? k : nullptr, ldk, nk, T, size}, {position, T, T, 1, 4}, {r->turns, r->rotary / 2, r->rotary / 2, 1, 8},
                         {takes_w && heads_q ? r->q_weight : nullptr, r->dim, r->dim, 1, 4}, {takes_w && heads_k ? r->k_weight : nullptr, r->dim, r->dim, 1, 4},
                         {heads_q ? q_out : nullptr, ldqo, nq, T, size}, {heads_k ? k_out : nullptr, ldko, nk, T, size}};
    static const char *const names[] = {"q", "k", "position", "turns", "q_weight", "k_weight", "q_out", "k_out"};
    if ((rc = check_apart(who, rows, names, 8, 6, [](int o, int i) { return (o == 6 && i == 0) || (o == 7 && i == 1); })) != W4A8_OK) return rc;
    if ((rc = require_sm100()) != W4A8_OK) return rc;
    const bool bare = r->variant == W4A8_NORM_NONE;
    rope::Args a = {r->turns, r->q_weight, r->k_weight, position, q, k, q_out, k_out, ldq, ldk, ldqo, ldko, r->eps, r->magnitude, 1.f / r->dim, (float)r->eps,
                    heads_q, heads_q + heads_k, r->dim, r->rotary, r->interleaved != 0, r->variant, 0, bare && q == q_out, bare && k == k_out};
    return rope::launch(a, T, dtype, (cudaStream_t)stream);
}

W4A8_API int w4a8_moe_route(const w4a8_router *r, const void *logits, int64_t ld, int S, int dtype, int32_t *idx, float *weight, void *stream) {
    const char *who = "moe_route";
    if (!r) return fail(W4A8_ERR_ARG, "%s: null router", who);
    const size_t size = row_size(dtype);
    if (!size) return fail(W4A8_ERR_ARG, "%s: dtype=%d (0 fp32, 1 fp16, 2 bf16)", who, dtype);
    if (S < 0) return fail(W4A8_ERR_ARG, "%s: S=%d", who, S);
    if (r->experts <= 0 || r->experts > route::MAX_EXPERTS || r->topk <= 0 || r->topk > route::MAX_TOPK || r->groups <= 0 || r->groups > route::MAX_GROUPS)
        return fail(W4A8_ERR_ARG, "%s: experts=%d (1 to %d) topk=%d (1 to %d) groups=%d (1 to %d)", who, r->experts, route::MAX_EXPERTS, r->topk, route::MAX_TOPK, r->groups, route::MAX_GROUPS);
    if (r->experts % r->groups != 0 || r->topk_groups <= 0 || r->topk_groups > r->groups) return fail(W4A8_ERR_ARG, "%s: %d experts in %d groups, %d of them taken", who, r->experts, r->groups, r->topk_groups);
    if (r->topk > r->experts / r->groups * r->topk_groups) return fail(W4A8_ERR_ARG, "%s: %d of the %d experts that take part", who, r->topk, r->experts / r->groups * r->topk_groups);
    if (r->scoring < 0 || r->scoring > 1 || r->group_score < 0 || r->group_score > 1) return fail(W4A8_ERR_ARG, "%s: scoring=%d group_score=%d", who, r->scoring, r->group_score);
    if (r->group_score == 1 && r->topk_groups < r->groups && r->experts / r->groups < 2) return fail(W4A8_ERR_ARG, "%s: a group of one expert has no two to add", who);
    if (ld < r->experts) return fail(W4A8_ERR_ARG, "%s: logits have rows of %d elements, a pitch of %lld", who, r->experts, (long long)ld);
    if (S == 0) return W4A8_OK;
    if (!logits || !idx || !weight) return fail(W4A8_ERR_ARG, "%s: null pointer argument", who);
    if (!aligned(logits, size) || !aligned(idx, 4) || !aligned(weight, 4) || (r->bias && !aligned(r->bias, 4))) return fail(W4A8_ERR_ALIGN, "%s: pointers must be aligned to their elements", who);
    const Rows rows[] = {{logits, ld, r->experts, S, size}, {r->bias, r->experts, r->experts, 1, 4}, {idx, r->topk, r->topk, S, 4}, {weight, r->topk, r->topk, S, 4}};
    static const char *const names[] = {"logits", "bias", "idx", "weight"};
    int rc = check_apart(who, rows, names, 4, 2, [](int, int) { return false; });
    if (rc != W4A8_OK || (rc = require_sm100()) != W4A8_OK) return rc;
    route::Args a = {logits, r->bias, idx, weight, ld, S, r->experts, r->topk, r->scoring, r->groups, r->topk_groups, r->group_score == 1 && r->topk_groups < r->groups, r->renormalise != 0, 0, 0, 0, r->scale};
    return route::launch(a, dtype, (cudaStream_t)stream);
}
