// What the token-step operators refuse before anything is launched (include/hipvoc_ops.h).  Pure C++: tests/native/fuzz_ops.cpp runs it on
// the CPU.  Each check returns the reason, or "" where the call is sound.
#pragma once
#include <stdarg.h>
#include <stdio.h>

#include <string>

#include "../../include/hipvoc_ops.h"
#include "ops_index.hpp"

namespace hipvoc {

static inline std::string ops_say(const char *f, ...) {
    char buf[256];
    va_list ap;
    va_start(ap, f);
    vsnprintf(buf, sizeof buf, f, ap);
    va_end(ap);
    return buf;
}

static inline bool act_type(int t) { return t == HIPVOC_T_F32 || t == HIPVOC_T_F16 || t == HIPVOC_T_BF16; }
static inline int type_bytes(int t) { return t == HIPVOC_T_F32 ? 4 : t == HIPVOC_T_F16 || t == HIPVOC_T_BF16 ? 2 : 1; }
static inline bool odd16(const void *p) { return ((uintptr_t)p & 15) != 0; }
static inline bool odd16(int64_t stride, int type) { return ((uint64_t)stride * (uint64_t)type_bytes(type) & 15) != 0; }
static const int64_t OPS_MAX_STRIDE = (int64_t)1 << 40;

static inline std::string check_cache(const hipvoc_kv_cache *k, int dtype) {
    if (!k || !k->k || !k->v) return "cache: null pointer";
    if (!act_type(dtype)) return "dtype must be F32, F16 or BF16";
    const bool coded = k->dtype == HIPVOC_T_INT8 || k->dtype == HIPVOC_T_E4M3;
    if (!coded && k->dtype != dtype) return ops_say("a cache of an act type is used in that type (cache %d, call %d)", k->dtype, dtype);
    if (coded && (!k->k_scale || !k->v_scale)) return "an 8-bit cache needs k_scale and v_scale";
    if (!coded && (k->k_scale || k->v_scale)) return "only an 8-bit cache has scales";
    if (k->head_dim != 64 && k->head_dim != 128) return ops_say("head_dim must be 64 or 128, not %d", k->head_dim);
    if (k->page < 8 || k->page > 1024 || (k->page & (k->page - 1))) return ops_say("page must be a power of two from 8 to 1024, not %d", k->page);
    if (k->n_pages < 1 || k->kv_heads < 1 || k->kv_heads > 1024) return ops_say("cache: n_pages %d, kv_heads %d (1 .. 1024)", k->n_pages, k->kv_heads);
    if (k->page_stride < (int64_t)k->kv_heads * k->page * k->head_dim) return ops_say("page_stride %lld is shorter than a page", (long long)k->page_stride);
    if (k->page_stride > OPS_MAX_STRIDE) return "page_stride too large";
    if (odd16(k->k) || odd16(k->v) || odd16(k->page_stride, k->dtype)) return "cache pages must be 16-byte aligned";
    if (odd16(k->k_scale) || odd16(k->v_scale)) return "cache scales must be 16-byte aligned";
    return "";
}

static inline std::string check_table(const int32_t *table, int64_t stride, int width, int n_seqs, int page) {
    if (n_seqs < 0 || n_seqs > 65535) return ops_say("n_seqs %d is not in 0 .. 65535", n_seqs);
    if (width < 0 || (int64_t)width * page > 0x7fffff00) return ops_say("table_width %d: a sequence may have up to 2^31 - 256 positions", width);
    if (n_seqs > 0 && width > 0 && !table) return "table: null pointer";
    if ((n_seqs > 1 && stride < width) || stride < 0 || stride > OPS_MAX_STRIDE) return "table_stride is shorter than table_width";
    if ((uintptr_t)table & 3) return "table is not aligned to its type";
    return "";
}

static inline std::string check_move(const hipvoc_kv_cache *cache, const void *k, const void *v, int64_t ks, int64_t vs, int dtype,
                                     const hipvoc_kv_rows *r, int n_rows) {
    std::string why = check_cache(cache, dtype);
    if (!why.empty()) return why;
    if (!r) return "rows: null pointer";
    why = check_table(r->table, r->table_stride, r->table_width, r->n_seqs, cache->page);
    if (!why.empty()) return why;
    if (n_rows < 0 || n_rows > 1 << 28) return ops_say("n_rows %d is not in 0 .. 2^28", n_rows);
    if (n_rows == 0 || r->n_seqs == 0) return "";
    if ((int64_t)n_rows * kv_parts(cache->kv_heads, cache->head_dim) * 64 + 256 > OPS_MAX_THREADS) return "n_rows: too many for one call with that many heads";
    if (!k || !v || !r->cu || !r->first) return "null pointer";
    if (((uintptr_t)r->cu | (uintptr_t)r->first) & 3) return "cu / first are not aligned to their type";
    const int64_t row = (int64_t)cache->kv_heads * cache->head_dim;
    if (ks < row || vs < row || ks > OPS_MAX_STRIDE || vs > OPS_MAX_STRIDE) return "k_stride / v_stride shorter than kv_heads * head_dim";
    if (odd16(k) || odd16(v) || odd16(ks, dtype) || odd16(vs, dtype)) return "rows must be 16-byte aligned";
    return "";
}

static inline std::string check_attention(const hipvoc_kv_cache *cache, const void *q, int64_t q_stride, const void *out, int64_t out_stride,
                                          const float *lse, int dtype, int n_heads, const int32_t *table, int64_t table_stride, int table_width,
                                          const int32_t *lens, int n_seqs, int max_len, int window, float scale, const void *workspace,
                                          size_t workspace_bytes) {
    std::string why = check_cache(cache, dtype);
    if (why.empty()) why = check_table(table, table_stride, table_width, n_seqs, cache->page);
    if (!why.empty()) return why;
    if (n_heads < 1 || n_heads % cache->kv_heads || n_heads > 16384) return ops_say("n_heads %d is no multiple of kv_heads %d (up to 16384)", n_heads, cache->kv_heads);
    if (max_len < 0 || max_len > (int64_t)table_width * cache->page) return ops_say("max_len %d does not fit %d pages of %d", max_len, table_width, cache->page);
    if (window < 0) return "window must not be negative";
    if (!(scale > -1e38f && scale < 1e38f)) return "scale must be finite";
    if (n_seqs == 0) return "";
    if (!q || !out || !lens) return "null pointer";
    if (((uintptr_t)lens | (uintptr_t)lse) & 3) return "lens / lse are not aligned to their type";
    const int64_t row = (int64_t)n_heads * cache->head_dim;
    if (q_stride < row || out_stride < row || q_stride > OPS_MAX_STRIDE || out_stride > OPS_MAX_STRIDE) return "q_stride / out_stride shorter than n_heads * head_dim";
    if (odd16(q) || odd16(out) || odd16(q_stride, dtype) || odd16(out_stride, dtype)) return "rows must be 16-byte aligned";
    const AttnPlan p = attention_plan(dtype, cache->dtype != dtype, cache->head_dim, cache->kv_heads, n_heads, n_seqs, max_len, window);
    if (!p.workers && (int64_t)n_seqs * p.heads * 256 > OPS_MAX_THREADS) return "n_seqs: too many for one call with that many heads";
    if (p.bytes && (!workspace || odd16(workspace) || workspace_bytes < p.bytes))
        return ops_say("workspace: %zu bytes needed, 16-byte aligned (hipvoc_attention_workspace)", p.bytes);
    return "";
}

static inline std::string check_norm(const void *x, int64_t x_stride, const void *residual, int64_t residual_stride, const void *weight, const void *sum,
                                     int64_t sum_stride, const void *y, int64_t y_stride, const float *scales, int dtype, int out_dtype, int group,
                                     float eps, int rows, int cols) {
    const bool coded = out_dtype == HIPVOC_T_INT8 || out_dtype == HIPVOC_T_E4M3;
    if (!act_type(dtype)) return "dtype must be F32, F16 or BF16";
    if (!coded && out_dtype != dtype) return "out_dtype must be dtype, INT8 or E4M3";
    if (rows < 0 || rows >= 1 << 22 || cols < 1 || cols > 1 << 20) return ops_say("rows %d (under 2^22), cols %d (1 .. 2^20)", rows, cols);
    if (coded ? group != 0 && ((group != 32 && group != 64 && group != 128) || cols % group) : group != 0)
        return ops_say("group %d must be 0, or for 8-bit rows 32, 64 or 128 and a divisor of cols %d", group, cols);
    if (!(eps >= 0.f && eps < 1e30f)) return "eps must be finite and not negative";
    if (rows == 0) return "";
    if (!x || !weight || !y || (coded && !scales)) return "null pointer";
    if (!coded && scales) return "only 8-bit rows have scales";
    if (sum && !residual) return "sum without a residual would be x itself";
    if (x_stride < cols || y_stride < cols || (residual && residual_stride < cols) || (sum && sum_stride < cols)) return "a stride is shorter than cols";
    if (x_stride > OPS_MAX_STRIDE || y_stride > OPS_MAX_STRIDE || residual_stride > OPS_MAX_STRIDE || sum_stride > OPS_MAX_STRIDE) return "a stride is too large";
    const uintptr_t align = (uintptr_t)type_bytes(dtype) - 1;
    if ((((uintptr_t)x | (uintptr_t)residual | (uintptr_t)weight | (uintptr_t)sum | (coded ? 0 : (uintptr_t)y)) & align) || ((uintptr_t)scales & 3))
        return "a pointer is not aligned to its type";
    return "";
}

static inline std::string check_q4(const void *codes, const void *scales, const void *mins, int n_out, int n_in, int group, const void *x, int64_t x_stride,
                                   int x_dtype, const float *x_scale, int x_groups, const void *y, int64_t y_stride, int y_dtype, int n_rows) {
    const bool coded = x_dtype == HIPVOC_T_INT8;
    if (!coded && !act_type(x_dtype)) return "x_dtype must be F32, F16, BF16 or INT8";
    if (!act_type(y_dtype) || (!coded && y_dtype != x_dtype)) return "y_dtype must be x_dtype, or for INT8 rows F32, F16 or BF16";
    if (group != 32 && group != 64 && group != 128) return ops_say("group must be 32, 64 or 128, not %d", group);
    if (n_out < 0 || n_out > 1 << 24 || n_in < group || n_in % group || n_in > 1 << 20) return ops_say("n_out %d (up to 2^24), n_in %d (a multiple of group, up to 2^20)", n_out, n_in);
    if (n_rows < 0 || n_rows > 65535) return ops_say("n_rows %d is not in 0 .. 65535", n_rows);
    if (coded ? (x_groups != 1 && x_groups != n_in / group) : x_groups != 0) return ops_say("x_groups %d must be 1 or n_in / group for INT8 rows, 0 otherwise", x_groups);
    if (n_rows == 0 || n_out == 0) return "";
    if (!codes || !scales || !x || !y || (coded && !x_scale)) return "null pointer";
    if (!coded && x_scale) return "only INT8 rows have scales";
    if (x_stride < n_in || x_stride > OPS_MAX_STRIDE || y_stride < n_out || y_stride > OPS_MAX_STRIDE) return "x_stride / y_stride shorter than a row";
    if (odd16(codes) || odd16(scales) || odd16(mins) || odd16(x) || odd16(x_stride, x_dtype)) return "codes, scales, mins and the rows of x must be 16-byte aligned";
    if (((uintptr_t)y & ((uintptr_t)type_bytes(y_dtype) - 1)) || ((uintptr_t)x_scale & 3)) return "a pointer is not aligned to its type";
    return "";
}

}  // namespace hipvoc
