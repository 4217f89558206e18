// C ABI of the token-step operators (include/hipvoc_ops.h), included by hipvoc.cpp: argument checks, the handle's deferred error word, the
// caller's stream.  The kernels are in kernels_kv.hip, kernels_attn.hip, kernels_norm.hip and kernels_q4.hip.
#include "ops_checks.hpp"
#include "ops_kernels.h"

namespace hipvoc {

// The operators run inside the caller's step: the calling thread's current device is put back.
struct DeviceScope {
    int before = -1;
    bool ok = true;
    explicit DeviceScope(int device) {
        if (hipGetDevice(&before) != hipSuccess) before = -1;
        if (before != device) ok = hipSetDevice(device) == hipSuccess;
        else before = -1;
    }
    ~DeviceScope() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

#define OPS(h)                                                                                                             \
    Ctx *c = (Ctx *)(h);                                                                                                   \
    if (!c) return HIPVOC_E_ARG;                                                                                           \
    if (!c->is_ops) return ops_fail(c, HIPVOC_E_ARG, "this handle is no operator handle (hipvoc_ops_open)");               \
    DeviceScope scope(c->device);                                                                                          \
    if (!scope.ok) return ops_fail(c, HIPVOC_E_HIP, "hipSetDevice failed");
#define OPS_HIP(expr)                                                                                                      \
    do {                                                                                                                   \
        const hipError_t e__ = (expr);                                                                                     \
        if (e__ != hipSuccess) return ops_fail(c, HIPVOC_E_HIP, fmt("%s failed: %s", #expr, hipGetErrorString(e__)));      \
    } while (0)

// a stream of another device would run the kernels there
static int ops_stream(Ctx *c, void *stream) {
    if (!stream) return HIPVOC_OK;
    hipDevice_t dev = c->device;
    if (hipStreamGetDevice((hipStream_t)stream, &dev) != hipSuccess) {
        (void)hipGetLastError();
        return ops_fail(c, HIPVOC_E_ARG, "no such stream");
    }
    if (dev != c->device) return ops_fail(c, HIPVOC_E_ARG, fmt("the stream is of device %d, the handle of device %d", (int)dev, c->device));
    return HIPVOC_OK;
}

static int ops_launched(Ctx *c, const char *what, hipError_t e) {
    return e == hipSuccess ? HIPVOC_OK : ops_fail(c, HIPVOC_E_HIP, fmt("%s: launch failed: %s", what, hipGetErrorString(e)));
}

static int ops_move(Ctx *c, const char *what, bool write, const hipvoc_kv_cache *cache, void *k, void *v, int64_t ks, int64_t vs, int dtype,
                    const hipvoc_kv_rows *rows, int n_rows, void *stream) {
    const std::string why = check_move(cache, k, v, ks, vs, dtype, rows, n_rows);
    if (!why.empty()) return ops_fail(c, HIPVOC_E_ARG, why);
    const int rc = ops_stream(c, stream);
    if (rc || n_rows == 0 || rows->n_seqs == 0) return rc;
    const KvMoveArgs a = {*cache, *rows, __builtin_ctz((unsigned)cache->page), k, v, ks, vs, dtype, n_rows, c->d_err};
    return ops_launched(c, what, write ? launch_kv_write(a, (hipStream_t)stream) : launch_kv_read(a, (hipStream_t)stream));
}

// Calls on one handle may come from several threads, which share its deferred error word and the words it is collected in.
// One of the latter for a collecting caller, its own until the end: callers that wait for different streams do not wait for each other
// (for one of 63 to end, if there are as many)
struct OpsWord {
    Ctx *c;
    int word;
    explicit OpsWord(Ctx *ctx) : c(ctx) {
        std::unique_lock<std::mutex> lock(c->ops_words_lock);
        c->ops_word_free.wait(lock, [this] { return ~c->ops_words != 0; });
        word = __builtin_ctzll(~c->ops_words);
        c->ops_words |= 1ull << word;
    }
    ~OpsWord() {
        {
            std::lock_guard<std::mutex> lock(c->ops_words_lock);
            c->ops_words &= ~(1ull << word);
        }
        c->ops_word_free.notify_one();
    }
};

// Takes the deferred error word on `stream` (one atomic exchange, so that nothing another stream raises meanwhile is lost) and waits for it.
static int ops_collect(Ctx *c, hipStream_t stream) {
    hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
    if (stream && hipStreamIsCapturing(stream, &cap) == hipSuccess && cap != hipStreamCaptureStatusNone)
        return ops_fail(c, HIPVOC_E_ARG, "the stream is being captured: it cannot be waited for");
    int bits = 0;
    {
        const OpsWord mine(c);
        OPS_HIP(launch_take_error(c->d_err, mine.word, stream));
        OPS_HIP(hipStreamSynchronize(stream));
        OPS_HIP(hipMemcpyWithStream(&bits, c->d_err + mine.word, sizeof bits, hipMemcpyDeviceToHost, stream));
    }
    if (!bits) return HIPVOC_OK;
    return ops_fail(c, HIPVOC_E_CODE, fmt("on the device:%s%s%s", bits & OPS_ERR_POSITION ? " a row's position outside its sequence's pages;" : "",
                                          bits & OPS_ERR_PAGE ? " a page number outside the cache;" : "",
                                          bits & OPS_ERR_LENGTH ? " a length outside 0 .. max_len;" : ""));
}

static int ops_sync_device(Ctx *c) {
    DeviceScope scope(c->device);
    if (!scope.ok) return ops_fail(c, HIPVOC_E_HIP, "hipSetDevice failed");
    OPS_HIP(hipDeviceSynchronize());
    return ops_collect(c, nullptr);
}

static void *ops_open_impl(int device_id) {
    auto fail = [](const std::string &m) -> void * {
        set_load_error(m.c_str());
        return nullptr;
    };
    const int ndev = hipvoc_device_count();
    if (ndev <= 0) return fail("no HIP device available (libhipvoc has no CPU fallback)");
    if (device_id < 0 || device_id >= ndev) return fail(fmt("device %d out of range (%d devices)", device_id, ndev));
    DeviceScope scope(device_id);
    if (!scope.ok) return fail("hipSetDevice failed");
    std::unique_ptr<Ctx> c(new Ctx);
    c->device = device_id;
    c->is_ops = true;
    void *p = nullptr;
    if (hipMalloc(&p, 64 * sizeof(int)) != hipSuccess) return fail("hipMalloc failed");
    c->dev_allocs.push_back(p);
    if (hipMemset(p, 0, 64 * sizeof(int)) != hipSuccess || hipDeviceSynchronize() != hipSuccess) return fail("device error while opening");
    c->d_err = (int *)p;
    return c.release();
}

}  // namespace hipvoc

extern "C" {

void *hipvoc_ops_open(int device_id) {
    try {
        return ops_open_impl(device_id);
    } catch (const std::bad_alloc &) {
        set_load_error("hipvoc_ops_open: out of host memory");
    } catch (const std::exception &e) {
        set_load_error(e.what());
    } catch (...) {
        set_load_error("hipvoc_ops_open: unknown C++ exception");
    }
    return nullptr;
}

int hipvoc_ops_sync(void *h, void *stream) {
    return guarded(h, [&]() -> int {
        OPS(h);
        int rc = ops_stream(c, stream);
        if (rc) return rc;
        return ops_collect(c, (hipStream_t)stream);
    });
}

int hipvoc_kv_write(void *h, const hipvoc_kv_cache *cache, const void *k, const void *v, int64_t k_stride, int64_t v_stride, int dtype,
                    const hipvoc_kv_rows *rows, int n_rows, void *stream) {
    return guarded(h, [&]() -> int {
        OPS(h);
        return ops_move(c, "hipvoc_kv_write", true, cache, const_cast<void *>(k), const_cast<void *>(v), k_stride, v_stride, dtype, rows, n_rows, stream);
    });
}

int hipvoc_kv_read(void *h, const hipvoc_kv_cache *cache, void *k, void *v, int64_t k_stride, int64_t v_stride, int dtype,
                   const hipvoc_kv_rows *rows, int n_rows, void *stream) {
    return guarded(h, [&]() -> int {
        OPS(h);
        return ops_move(c, "hipvoc_kv_read", false, cache, k, v, k_stride, v_stride, dtype, rows, n_rows, stream);
    });
}

size_t hipvoc_attention_workspace(const hipvoc_kv_cache *cache, int n_heads, int n_seqs, int max_len, int window) {
    if (!cache || cache->kv_heads < 1 || n_heads < 1 || n_heads % cache->kv_heads || n_seqs < 1 || max_len < 1 || window < 0) return 0;
    // the act type is not asked for: what either kernel needs
    const bool coded = cache->dtype == HIPVOC_T_INT8 || cache->dtype == HIPVOC_T_E4M3;
    return std::max(attention_plan(HIPVOC_T_F32, coded, cache->head_dim, cache->kv_heads, n_heads, n_seqs, max_len, window).bytes,
                    attention_plan(HIPVOC_T_BF16, coded, cache->head_dim, cache->kv_heads, n_heads, n_seqs, max_len, window).bytes);
}

int hipvoc_attention(void *h, const hipvoc_kv_cache *cache, const void *q, int64_t q_stride, void *out, int64_t out_stride, float *lse, int dtype,
                     int n_heads, const int32_t *table, int64_t table_stride, int table_width, const int32_t *lens, int n_seqs, int max_len,
                     int window, float scale, void *workspace, size_t workspace_bytes, void *stream) {
    return guarded(h, [&]() -> int {
        OPS(h);
        const std::string why = check_attention(cache, q, q_stride, out, out_stride, lse, dtype, n_heads, table, table_stride, table_width, lens,
                                                n_seqs, max_len, window, scale, workspace, workspace_bytes);
        if (!why.empty()) return ops_fail(c, HIPVOC_E_ARG, why);
        const int rc = ops_stream(c, stream);
        if (rc || n_seqs == 0) return rc;
        const AttnPlan p = attention_plan(dtype, cache->dtype != dtype, cache->head_dim, cache->kv_heads, n_heads, n_seqs, max_len, window);
        AttnArgs a = {};
        a.page_shift = __builtin_ctz((unsigned)cache->page);
        a.c = *cache;
        a.q = q;
        a.out = out;
        a.lse = lse;
        a.q_stride = q_stride;
        a.out_stride = out_stride;
        a.dtype = dtype;
        a.n_heads = n_heads;
        a.group = n_heads / cache->kv_heads;
        a.table = table;
        a.table_stride = table_stride;
        a.table_width = table_width;
        a.lens = lens;
        a.n_seqs = n_seqs;
        a.max_len = max_len;
        a.window = window;
        a.scale_log2 = scale * 1.44269504088896340736f;
        a.heads = p.heads;
        a.workers = p.workers;
        a.least = p.least;
        a.part = (float *)workspace;
        a.before = p.workers ? (int64_t *)((char *)workspace + p.bytes) - (n_seqs + 1) : nullptr;
        a.err = c->d_err;
        return ops_launched(c, "hipvoc_attention", launch_attention_decode(a, (hipStream_t)stream));
    });
}

int hipvoc_add_rmsnorm(void *h, const void *x, int64_t x_stride, const void *residual, int64_t residual_stride, const void *weight, void *sum,
                       int64_t sum_stride, void *y, int64_t y_stride, float *scales, int dtype, int out_dtype, int group, float eps, int rows,
                       int cols, void *stream) {
    return guarded(h, [&]() -> int {
        OPS(h);
        const std::string why = check_norm(x, x_stride, residual, residual_stride, weight, sum, sum_stride, y, y_stride, scales, dtype, out_dtype, group, eps, rows, cols);
        if (!why.empty()) return ops_fail(c, HIPVOC_E_ARG, why);
        const int rc = ops_stream(c, stream);
        if (rc || rows == 0) return rc;
        NormArgs a = {x, residual, weight, sum, y, scales, x_stride, residual ? residual_stride : 0, sum_stride, y_stride, dtype, out_dtype, group, eps, rows, cols};
        return ops_launched(c, "hipvoc_add_rmsnorm", launch_add_rmsnorm(a, (hipStream_t)stream));
    });
}

int hipvoc_q4_matvec(void *h, const uint8_t *codes, const void *scales, const void *mins, int n_out, int n_in, int group, const void *x,
                     int64_t x_stride, int x_dtype, const float *x_scale, int x_groups, void *y, int64_t y_stride, int y_dtype, int n_rows,
                     void *stream) {
    return guarded(h, [&]() -> int {
        OPS(h);
        const std::string why = check_q4(codes, scales, mins, n_out, n_in, group, x, x_stride, x_dtype, x_scale, x_groups, y, y_stride, y_dtype, n_rows);
        if (!why.empty()) return ops_fail(c, HIPVOC_E_ARG, why);
        const int rc = ops_stream(c, stream);
        if (rc || n_rows == 0 || n_out == 0) return rc;
        Q4Args a = {codes, scales, mins, n_out, n_in, group, x, x_stride, x_dtype, x_scale, x_groups, y, y_stride, y_dtype, n_rows};
        return ops_launched(c, "hipvoc_q4_matvec", launch_q4_matvec(a, (hipStream_t)stream));
    });
}

}  // extern "C"
