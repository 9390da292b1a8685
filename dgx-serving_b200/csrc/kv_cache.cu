// The KV cache's translation unit of libw4a8_b200.so: block tables, rows into and out of the 8-bit blocks, attention over them.
#include <type_traits>

#include "common.cuh"
#include "kv_cache.cuh"
#include "attention_q8.cuh"
#include "attention_q8_tc.cuh"

namespace w4a8 {

// The device-side error word of this translation unit, read and cleared (w4a8_device_status).
cudaError_t kv_take_device_error(unsigned int *v) {
    const unsigned int zero = 0;
    cudaError_t e = cudaMemcpyFromSymbol(v, g_dev_error, sizeof(*v));
    if (e == cudaSuccess && *v != 0) e = cudaMemcpyToSymbol(g_dev_error, &zero, sizeof(zero));
    return e;
}
const char *kv_device_error_text(unsigned int v) {
    switch (v) {
        case kv::ERR_BLOCK_ID: return "a block table names a block that the cache does not have, for a token that was needed";
        case kv::ERR_SLOT: return "kv_append: a slot beyond the cache";
        case kv::ERR_LENGTH: return "attention: a request has more tokens than its block table's row holds, or than 2^31 - 512";
        default: return "a kernel's bounded wait ran out";
    }
}

static bool size_of(int dtype, size_t *size) {
    *size = dtype == W4A8_F32 ? 4 : 2;
    return dtype == W4A8_F32 || dtype == W4A8_F16 || dtype == W4A8_BF16;
}

static int check_cache(const w4a8_kv_cache *c, const char *who) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) return fail(W4A8_ERR_ARG, "%s: null cache pointer", who);
    if (c->dim != 64 && c->dim != 128 && c->dim != 256) return fail(W4A8_ERR_ARG, "%s: dim=%d (64, 128 or 256)", who, c->dim);
    if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128) return fail(W4A8_ERR_ARG, "%s: block=%d (16, 32, 64 or 128 tokens)", who, c->block);
    if (c->heads <= 0 || c->heads > 65535 || c->num_blocks <= 0) return fail(W4A8_ERR_ARG, "%s: heads=%d num_blocks=%d", who, c->heads, c->num_blocks);
    if ((int64_t)c->num_blocks * c->block > 0x7fffffff || (int64_t)c->num_blocks * c->heads * c->block > 0x7fffffff)
        return fail(W4A8_ERR_UNSUPPORTED, "%s: %d blocks of %d heads and %d tokens: slots, and the rows of all heads, have to fit 31 bits", who, c->num_blocks, c->heads, c->block);
    if (!aligned(c->k, 16) || !aligned(c->v, 16)) return fail(W4A8_ERR_ALIGN, "%s: k and v of the cache must be 16-byte aligned", who);
    return W4A8_OK;
}

static int check_rows(const void *p, int64_t ld, int64_t columns, size_t size, const char *name, const char *who) {
    if (!p) return fail(W4A8_ERR_ARG, "%s: null %s", who, name);
    if (ld < columns) return fail(W4A8_ERR_ARG, "%s: %s has rows of %lld elements, a pitch of %lld", who, name, (long long)columns, (long long)ld);
    if (!aligned(p, 16) || (ld * size) % 16 != 0) return fail(W4A8_ERR_ALIGN, "%s: %s and its rows must be 16-byte aligned", who, name);
    return W4A8_OK;
}

}  // namespace w4a8

using namespace w4a8;

W4A8_API int w4a8_kv_plan(const int32_t *kv_len, const int32_t *new_len, int R, int block, int32_t *block_table, int table_width,
                          const int32_t *free_blocks, int num_free, const int32_t *first_free, int32_t *seq_len, int32_t *cu_new, int32_t *slot,
                          int32_t *position, int T, int32_t *status, void *stream) {
    if (R < 0 || T < 0 || num_free < 0 || table_width < 0) return fail(W4A8_ERR_ARG, "kv_plan: negative size R=%d T=%d num_free=%d table_width=%d", R, T, num_free, table_width);
    if (block != 16 && block != 32 && block != 64 && block != 128) return fail(W4A8_ERR_ARG, "kv_plan: block=%d (16, 32, 64 or 128 tokens)", block);
    if (R > kv::PLAN_MAX_R) return fail(W4A8_ERR_UNSUPPORTED, "kv_plan: %d requests (at most %d)", R, kv::PLAN_MAX_R);
    if (!first_free || !cu_new || !status || (T && !slot) || (num_free && !free_blocks) || (R && (!kv_len || !new_len || !seq_len || (table_width && !block_table))))
        return fail(W4A8_ERR_ARG, "kv_plan: null pointer argument");
    // every CTA reads the inputs to its end, and what is written early may be one of them (seq_len and kv_len, status and first_free)
    const struct { const void *p; size_t n; const char *name; } in[] = {{kv_len, (size_t)R, "kv_len"}, {new_len, (size_t)R, "new_len"}, {free_blocks, (size_t)num_free, "free_blocks"},
                                                                        {first_free, 1, "first_free"}},
        out[] = {{seq_len, (size_t)R, "seq_len"}, {cu_new, (size_t)R + 1, "cu_new"}, {slot, (size_t)T, "slot"}, {position, (size_t)T, "position"}, {status, 4, "status"},
                 {block_table, (size_t)R * table_width, "block_table"}};
    for (const auto &i : in)
        for (const auto &o : out)
            if (i.p && o.p && i.n && o.n && (uintptr_t)i.p < (uintptr_t)o.p + o.n * 4 && (uintptr_t)o.p < (uintptr_t)i.p + i.n * 4)
                return fail(W4A8_ERR_ARG, "kv_plan: %s overlaps %s, an input that is read to the end", o.name, i.name);
    int rc = require_sm100();
    if (rc != W4A8_OK) return rc;
    kv::PlanArgs a = {kv_len, new_len, free_blocks, first_free, block_table, seq_len, cu_new, slot, position, status, R, block, table_width, num_free, T, 0x7fffffffu / (unsigned)block};
    return kv::launch_plan(a, (cudaStream_t)stream);
}

W4A8_API int w4a8_kv_append_q8(const void *K, const void *V, int64_t ld, const int32_t *slot, int T, const w4a8_kv_cache *cache, int dtype, void *stream) {
    const char *who = "kv_append_q8";
    size_t size;
    if (T < 0) return fail(W4A8_ERR_ARG, "%s: T=%d", who, T);
    if (!size_of(dtype, &size)) return fail(W4A8_ERR_ARG, "%s: dtype=%d (0 fp32, 1 fp16, 2 bf16)", who, dtype);
    int rc = check_cache(cache, who);
    if (rc != W4A8_OK || T == 0) return rc;
    const int64_t columns = (int64_t)cache->heads * cache->dim;
    if ((rc = check_rows(K, ld, columns, size, "K", who)) != W4A8_OK || (rc = check_rows(V, ld, columns, size, "V", who)) != W4A8_OK) return rc;
    if (!slot) return fail(W4A8_ERR_ARG, "%s: null slot", who);
    if ((rc = require_sm100()) != W4A8_OK) return rc;
    kv::AppendArgs a = {K, V, slot, cache->k, cache->v, cache->k_scale, cache->v_scale, ld, T, cache->heads, cache->block, 1, cache->num_blocks * cache->block};
    a.span = kv::append_span(T, cache->heads, cache->block);
    return kv::by_type(dtype, cache->dim, [&](auto t, auto d) { return kv::launch_append_t<decltype(t), decltype(d)::value>(a, (cudaStream_t)stream); });
}

W4A8_API int w4a8_kv_read_q8(const w4a8_kv_cache *cache, const int32_t *block_table, int table_width, const int32_t *begin, const int32_t *cu, int R, int T,
                             void *K, void *V, int64_t ld, int dtype, void *stream) {
    const char *who = "kv_read_q8";
    size_t size;
    if (R < 0 || T < 0 || table_width < 0) return fail(W4A8_ERR_ARG, "%s: negative size R=%d T=%d table_width=%d", who, R, T, table_width);
    if (!size_of(dtype, &size)) return fail(W4A8_ERR_ARG, "%s: dtype=%d (0 fp32, 1 fp16, 2 bf16)", who, dtype);
    int rc = check_cache(cache, who);
    if (rc != W4A8_OK || R == 0 || T == 0) return rc;
    const int64_t columns = (int64_t)cache->heads * cache->dim;
    if ((rc = check_rows(K, ld, columns, size, "K", who)) != W4A8_OK || (rc = check_rows(V, ld, columns, size, "V", who)) != W4A8_OK) return rc;
    if (!begin || !cu || !block_table) return fail(W4A8_ERR_ARG, "%s: null pointer argument", who);
    if ((rc = require_sm100()) != W4A8_OK) return rc;
    kv::ReadArgs a = {cache->k, cache->v, cache->k_scale, cache->v_scale, block_table, begin, cu, K, V, ld, R, T, table_width, cache->heads, cache->block, cache->num_blocks, 1};
    a.tokens = kv::read_tokens(T, cache->heads, cache->dim);
    return kv::by_type(dtype, cache->dim, [&](auto t, auto d) { return kv::launch_read_t<decltype(t), decltype(d)::value>(a, (cudaStream_t)stream); });
}

W4A8_API size_t w4a8_attention_q8_workspace_bytes(const w4a8_kv_cache *cache, int heads_q, int T, int max_q) {
    if (!cache || heads_q <= 0 || T < 0 || max_q < 0) return 0;
    return attn::workspace_bytes(cache->dim);
}

W4A8_API int w4a8_attention_q8(const void *Q, int64_t ldq, const w4a8_kv_cache *cache, const int32_t *block_table, int table_width, const int32_t *cu_q,
                               const int32_t *seq_len, int R, int T, int heads_q, void *O, int64_t ldo, float *lse, float scale, int causal, int window,
                               float softcap, int max_q, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
    const char *who = "attention_q8";
    size_t size;
    if (R < 0 || T < 0 || table_width < 0 || max_q < 0) return fail(W4A8_ERR_ARG, "%s: negative size R=%d T=%d table_width=%d max_q=%d", who, R, T, table_width, max_q);
    if (!size_of(dtype, &size)) return fail(W4A8_ERR_ARG, "%s: dtype=%d (0 fp32, 1 fp16, 2 bf16)", who, dtype);
    int rc = check_cache(cache, who);
    if (rc != W4A8_OK) return rc;
    if (heads_q <= 0 || heads_q % cache->heads != 0) return fail(W4A8_ERR_ARG, "%s: heads_q=%d is not a multiple of the cache's %d heads", who, heads_q, cache->heads);
    // (a cap whose quotients leave fp32 is none)
    if (window < 0 || !(softcap == 0.f || (softcap >= 1e-30f && softcap <= 1e30f)) || !(scale == scale)) return fail(W4A8_ERR_ARG, "%s: window=%d softcap=%g scale=%g", who, window, softcap, scale);
    if (R == 0 || T == 0) return W4A8_OK;
    const int64_t columns = (int64_t)heads_q * cache->dim;
    if ((rc = check_rows(Q, ldq, columns, size, "Q", who)) != W4A8_OK || (rc = check_rows(O, ldo, columns, size, "O", who)) != W4A8_OK) return rc;
    if (!cu_q || !seq_len || (table_width && !block_table)) return fail(W4A8_ERR_ARG, "%s: null pointer argument", who);
    const size_t need = attn::workspace_bytes(cache->dim);
    if (!workspace || workspace_bytes < need) return fail(W4A8_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, workspace ? workspace_bytes : (size_t)0, need);
    if (!aligned(workspace, 256)) return fail(W4A8_ERR_ALIGN, "%s: workspace must be 256-byte aligned", who);
    if ((rc = require_sm100()) != W4A8_OK) return rc;
    attn::Call c = {};
    attn::Args &a = c.a;
    a.q = Q; a.out = O; a.lse = lse; a.ks = cache->k_scale; a.vs = cache->v_scale;
    a.table = block_table; a.cu_q = cu_q; a.seq_len = seq_len; a.ldq = ldq; a.ldo = ldo;
    a.R = R; a.T = T; a.width = table_width; a.Hq = heads_q; a.Hkv = cache->heads; a.G = heads_q / cache->heads;
    a.block = cache->block; a.num_blocks = cache->num_blocks;
    a.causal = causal != 0; a.window = window; a.scale = scale; a.softcap = softcap;
    a.few = 0x7fffffff;
    attn::lay_out(a, workspace, cache->dim);
    c.k = cache->k; c.v = cache->v; c.dtype = dtype; c.dim = cache->dim;
    const int64_t rows = (int64_t)(max_q > 0 && max_q < T ? max_q : T) * a.G;
    if (rows > attn::FEW_ROWS) {
        // requests with many rows on the tensor cores' tiles of rows; the others, if there can be any, by the streaming kernel
        a.few = R == 1 ? 0 : attn::FEW_ROWS;
        for (int r0 = 0; r0 < R; r0 += attn_tc::MAX_R) {
            attn::Call part = c;
            part.a.R = R - r0 < attn_tc::MAX_R ? R - r0 : attn_tc::MAX_R;
            part.a.cu_q += r0; part.a.seq_len += r0; part.a.table += (size_t)r0 * table_width;
            if ((rc = attn_tc::launch(part, (cudaStream_t)stream)) != W4A8_OK) return rc;
        }
        if (R == 1) return W4A8_OK;
        return attn::launch(c, attn::FEW_ROWS, (cudaStream_t)stream);
    }
    return attn::launch(c, (int)rows, (cudaStream_t)stream);
}
