// Host-side checks of the token-step operators: the index arithmetic that the kernels run (ops_index.hpp) on lengths, offsets, windows and
// page numbers that are sound, extreme or malformed, and what the entry points refuse before a launch (ops_checks.hpp).
#include <limits.h>
#include <stdio.h>
#include <stdlib.h>

#include <algorithm>
#include <random>
#include <string>
#include <vector>

#include "../../qwen3-tts_amd/csrc/ops_checks.hpp"

using namespace hipvoc;

#define CHECK(x) do { if (!(x)) { fprintf(stderr, "failed: %s (line %d)\n", #x, __LINE__); exit(1); } } while (0)
static int refused = 0;
#define REFUSED(x) do { CHECK(!(x).empty()); refused++; } while (0)
#define FINE(x) do { std::string w = (x); if (!w.empty()) { fprintf(stderr, "refused: %s (line %d)\n", w.c_str(), __LINE__); exit(1); } } while (0)

static std::mt19937 rng(7);
static int pick(int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); }

static void spans() {
    const int odd[] = {INT_MIN, -1, 0, 1, 31, 32, 33, 127, 128, 129, 255, 256, 257, 4095, 131071, INT_MAX - 256};
    for (int it = 0; it < 20000; it++) {
        const int max_len = it % 3 ? pick(0, 200000) : odd[pick(2, 15)], len = it % 2 ? odd[pick(0, 15)] : pick(0, max_len);
        const int window = it % 5 ? 0 : odd[pick(3, 15)];
        const AttnSpan s = attn_span(len, max_len, window);
        CHECK(s.bad == (len < 0 || len > max_len));
        if (s.bad) { CHECK(s.hi == 0 && s.lo == 0 && s.tiles == 0); continue; }
        CHECK(s.hi == len && s.lo == (window > 0 && len > window ? len - window : 0));
        CHECK(s.base % 32 == 0 && s.base <= s.lo && s.lo - s.base < 32 && s.tiles == (int)(((int64_t)len - s.base + 31) / 32));
        CHECK((len == 0) == (s.tiles == 0));
    }
}

// The row of tiles, as kernel and join walk it: every tile in one piece, every piece in a slot of its own inside the workspace, and a pair in one
// piece exactly where the join thinks so.
static void cuts() {
    for (int it = 0; it < 3000; it++) {
        const int seqs = it % 4 ? pick(1, 12) : pick(1, 300), kv = pick(1, 8), group = pick(1, 20), dtype = pick(0, 2), hd = it % 2 ? 64 : 128;
        const int max_len = it % 7 ? pick(1, 40000) : pick(1, 400), window = it % 3 ? 0 : pick(1, 3000);
        const bool coded = it % 3 == 0;
        const AttnPlan p = attention_plan(dtype, coded, hd, kv, kv * group, seqs, max_len, window);
        const int most = dtype || coded ? 16 : group < 3 ? group : 4;
        CHECK(p.heads == kv * ((group + most - 1) / most) && (p.bytes > 0) == (p.workers > 0));
        if (!p.workers) continue;
        std::vector<int64_t> before(seqs + 1, 0);
        for (int b = 0; b < seqs; b++) before[b + 1] = before[b] + attn_span(pick(0, 9) ? pick(0, 5) ? pick(0, max_len) : pick(-3, 40) : max_len, max_len, window).tiles;
        const int64_t total = before[seqs] * p.heads, workers = attn_workers(total, p.least, p.workers);
        CHECK(workers <= p.workers && (workers > 0) == (total > 0));
        if (!total) continue;
        const int64_t slots = p.workers + (int64_t)seqs * p.heads, n = group < most ? group : most;
        CHECK((size_t)(slots * n * (hd + 2)) * sizeof(float) + (seqs + 1) * sizeof(int64_t) <= p.bytes);
        int64_t last_slot = -1, x = 0;
        for (int64_t w = 0; w < workers; w++) {
            CHECK(x == attn_first(w, total, workers));
            const int64_t end = attn_first(w + 1, total, workers);
            CHECK(end > x || total < workers);
            while (x < end) {
                int seq = 0;
                for (int m = seqs; m > 1;) { const int half = m / 2; if (before[seq + half] * p.heads <= x) seq += half; m -= half; }
                while (before[seq + 1] * p.heads <= x) seq++;
                CHECK(seq < seqs && before[seq] * p.heads <= x);
                const int64_t tiles = before[seq + 1] - before[seq], rest = x - before[seq] * p.heads, pair = rest / tiles, tile = rest % tiles;
                CHECK(pair < p.heads);
                const int64_t m = std::min(tiles - tile, end - x), slot = w + seq * (int64_t)p.heads + pair;
                CHECK(slot > last_slot && slot < slots);
                last_slot = slot;
                const int64_t first = before[seq] * p.heads + pair * tiles, w0 = attn_worker_of(first, total, workers), w1 = attn_worker_of(first + tiles - 1, total, workers);
                CHECK(w0 <= w && w <= w1 && (m == tiles) == (w0 == w1));
                CHECK(attn_worker_of(x, total, workers) == w && attn_worker_of(x + m - 1, total, workers) == w);
                x += m;
            }
        }
        CHECK(x == total);
    }
}

static void rows() {
    for (int it = 0; it < 20000; it++) {
        const int width = pick(0, 5000), shift = pick(3, 10), cu = it % 7 ? pick(0, 1000) : pick(INT_MIN, INT_MAX), t = pick(0, 1 << 28);
        const int first = it % 3 ? pick(0, 100000) : pick(INT_MIN, INT_MAX);
        const int64_t pos = row_position(t, cu, first, width, shift);
        CHECK(pos == -1 || (pos >= 0 && (pos >> shift) < width));
        if (pos >= 0) CHECK(pos == (int64_t)first + t - cu);
    }
    CHECK(page_ok(0, 1) && !page_ok(1, 1) && !page_ok(-1, 5) && !page_ok(INT_MIN, INT_MAX) && !page_ok(0, 0));
}

static hipvoc_kv_cache cache() {
    hipvoc_kv_cache c = {};
    c.k = (void *)0x1000; c.v = (void *)0x2000;
    c.n_pages = 4; c.kv_heads = 2; c.page = 16; c.head_dim = 64; c.dtype = HIPVOC_T_BF16;
    c.page_stride = 2 * 16 * 64;
    return c;
}

static void caches() {
    FINE(check_cache(nullptr, 2).empty() ? "a null cache passed" : "");
    hipvoc_kv_cache c = cache();
    FINE(check_cache(&c, HIPVOC_T_BF16));
    REFUSED(check_cache(&c, HIPVOC_T_F32));
    REFUSED(check_cache(&c, HIPVOC_T_INT8));
    REFUSED(check_cache(&c, 9));
    c.k = nullptr; REFUSED(check_cache(&c, 2)); c = cache();
    c.v = (void *)0x2008; REFUSED(check_cache(&c, 2)); c = cache();
    c.k_scale = (float *)0x3000; REFUSED(check_cache(&c, 2)); c = cache();
    c.dtype = HIPVOC_T_INT8; REFUSED(check_cache(&c, 2));
    c.k_scale = c.v_scale = (float *)0x3000; FINE(check_cache(&c, 2)); FINE(check_cache(&c, 0));
    c.v_scale = (float *)0x3004; REFUSED(check_cache(&c, 2)); c = cache();
    const int heads[] = {0, 32, 96, 65, 256, -64};
    for (int h : heads) { c.head_dim = h; c.page_stride = 1 << 20; REFUSED(check_cache(&c, 2)); }
    c = cache();
    const int pages[] = {0, 4, 12, 2048, -16, INT_MIN};
    for (int p : pages) { c.page = p; c.page_stride = 1 << 30; REFUSED(check_cache(&c, 2)); }
    c = cache(); c.page_stride -= 8; REFUSED(check_cache(&c, 2));
    c = cache(); c.page_stride += 4; REFUSED(check_cache(&c, 2));
    c = cache(); c.page_stride = INT64_MAX / 2; REFUSED(check_cache(&c, 2));
    c = cache(); c.n_pages = -1; REFUSED(check_cache(&c, 2));
    c = cache(); c.kv_heads = 0; REFUSED(check_cache(&c, 2));
}

static void moves() {
    hipvoc_kv_cache c = cache();
    hipvoc_kv_rows r = {(int32_t *)0x100, (int32_t *)0x200, (int32_t *)0x300, 3, 3, 2};
    const void *k = (void *)0x4000, *v = (void *)0x5000;
    FINE(check_move(&c, k, v, 128, 128, 2, &r, 5));
    FINE(check_move(&c, nullptr, nullptr, 0, 0, 2, &r, 0));
    REFUSED(check_move(&c, k, v, 128, 128, 2, nullptr, 5));
    REFUSED(check_move(&c, k, nullptr, 128, 128, 2, &r, 5));
    REFUSED(check_move(&c, k, v, 127, 128, 2, &r, 5));
    REFUSED(check_move(&c, k, v, 128, 132, 2, &r, 5));
    REFUSED(check_move(&c, (void *)0x4002, v, 128, 128, 2, &r, 5));
    REFUSED(check_move(&c, k, v, 128, 128, 2, &r, -1));
    REFUSED(check_move(&c, k, v, 128, 128, 2, &r, INT_MAX));
    REFUSED(check_move(&c, k, v, 128, INT64_MAX / 4, 2, &r, 5));
    hipvoc_kv_rows b = r;
    b.cu = nullptr; REFUSED(check_move(&c, k, v, 128, 128, 2, &b, 5)); b = r;
    b.first = nullptr; REFUSED(check_move(&c, k, v, 128, 128, 2, &b, 5)); b = r;
    b.table = nullptr; REFUSED(check_move(&c, k, v, 128, 128, 2, &b, 5)); b = r;
    b.table_stride = 2; REFUSED(check_move(&c, k, v, 128, 128, 2, &b, 5)); b = r;
    b.table_width = -1; REFUSED(check_move(&c, k, v, 128, 128, 2, &b, 5)); b = r;
    b.table_width = 1 << 28; b.table_stride = 1 << 28; REFUSED(check_move(&c, k, v, 128, 128, 2, &b, 5)); b = r;
    b.n_seqs = 70000; REFUSED(check_move(&c, k, v, 128, 128, 2, &b, 5)); b = r;
    b.n_seqs = -1; REFUSED(check_move(&c, k, v, 128, 128, 2, &b, 5));
    // a launch's threads count in 32 bits
    for (int hd = 64; hd <= 128; hd *= 2)
        for (int heads = 1; heads <= 1024; heads += heads < 40 ? 1 : 123) {
            c.head_dim = hd; c.kv_heads = heads; c.page_stride = (int64_t)heads * 16 * hd;
            const int64_t parts = kv_parts(heads, hd), row = (int64_t)heads * hd;
            CHECK(parts * KV_U * 64 * 8 >= 2 * row && (parts - 1) * KV_U * 64 * 8 < 2 * row);
            const int most = (int)std::min<int64_t>(1 << 28, ((int64_t)1 << 32) / 64 / parts - 8);
            FINE(check_move(&c, k, v, row, row, 2, &r, most));
            CHECK((most * parts + 3) / 4 * 256 < (int64_t)1 << 32);
            if (most < 1 << 28) REFUSED(check_move(&c, k, v, row, row, 2, &r, most + 16));
        }
}

struct A {
    hipvoc_kv_cache c = cache();
    const void *q = (void *)0x1000, *out = (void *)0x2000, *ws = (void *)0x3000;
    int64_t qs = 256, os = 256, ts = 64;
    const float *lse = (float *)0x5000;
    const int32_t *table = (int32_t *)0x6000, *lens = (int32_t *)0x7000;
    int dtype = 2, heads = 4, width = 64, seqs = 3, max_len = 1024, window = 0;
    float scale = 0.125f;
    size_t bytes = 1 << 24;
    std::string go() const { return check_attention(&c, q, qs, out, os, lse, dtype, heads, table, ts, width, lens, seqs, max_len, window, scale, ws, bytes); }
};

static void attentions() {
    FINE(A().go());
    A a;
    a.heads = 3; REFUSED(a.go()); a = A();
    a.heads = 0; REFUSED(a.go()); a = A();
    a.heads = 20000; a.qs = a.os = 20000 * 64; REFUSED(a.go()); a = A();
    a.max_len = 1025; REFUSED(a.go()); a = A();
    a.max_len = -1; REFUSED(a.go()); a = A();
    a.window = -1; REFUSED(a.go()); a = A();
    a.scale = 1e30f * 1e30f; REFUSED(a.go()); a = A();
    a.scale = a.scale * 0.f / 0.f; REFUSED(a.go()); a = A();
    a.scale = 3e38f; REFUSED(a.go()); a = A();
    a.q = nullptr; REFUSED(a.go()); a = A();
    a.out = (void *)0x2001; REFUSED(a.go()); a = A();
    a.lens = nullptr; REFUSED(a.go()); a = A();
    a.lens = (int32_t *)0x7002; REFUSED(a.go()); a = A();
    a.qs = 255; REFUSED(a.go()); a = A();
    a.os = 260; REFUSED(a.go()); a = A();
    a.ws = nullptr; REFUSED(a.go()); a = A();
    a.bytes = 16; REFUSED(a.go()); a = A();
    a.ts = 63; REFUSED(a.go()); a = A();
    a.seqs = 0; a.q = nullptr; FINE(a.go()); a = A();
    a.seqs = 65535; FINE(a.go());
    a.c.kv_heads = 512; a.c.page_stride = 512 * 16 * 64; a.heads = 512; a.qs = a.os = 512 * 64; REFUSED(a.go()); a = A();
    a.max_len = 0; a.ws = nullptr; a.bytes = 0; FINE(a.go());
}

static void norms() {
    auto go = [](int dtype, int out, int group, int rows, int cols, int64_t stride, float eps, uintptr_t x, uintptr_t res, uintptr_t sum, uintptr_t sc) {
        return check_norm((void *)x, stride, (void *)res, stride, (void *)0x900, (void *)sum, stride, (void *)0xa00, stride, (float *)sc, dtype, out, group, eps, rows, cols);
    };
    FINE(go(2, 2, 0, 3, 100, 100, 1e-6f, 0x100, 0x200, 0x300, 0));
    FINE(go(2, 3, 32, 3, 96, 100, 0.f, 0x102, 0, 0, 0x500));
    FINE(go(0, 4, 0, 3, 7, 7, 1e-6f, 0x104, 0x200, 0, 0x500));
    FINE(go(2, 2, 0, 0, 7, 7, 1e-6f, 0, 0, 0, 0));
    REFUSED(go(3, 3, 0, 3, 96, 96, 1e-6f, 0x100, 0, 0, 0x500));
    REFUSED(go(2, 1, 0, 3, 96, 96, 1e-6f, 0x100, 0, 0, 0));
    REFUSED(go(2, 3, 32, 3, 100, 100, 1e-6f, 0x100, 0, 0, 0x500));
    REFUSED(go(2, 3, 16, 3, 96, 96, 1e-6f, 0x100, 0, 0, 0x500));
    REFUSED(go(2, 2, 32, 3, 96, 96, 1e-6f, 0x100, 0, 0, 0));
    REFUSED(go(2, 3, 32, 3, 96, 96, 1e-6f, 0x100, 0, 0, 0));
    REFUSED(go(2, 2, 0, 3, 96, 96, 1e-6f, 0x100, 0, 0, 0x500));
    REFUSED(go(2, 2, 0, 3, 96, 95, 1e-6f, 0x100, 0, 0, 0));
    REFUSED(go(2, 2, 0, 3, 96, 96, 1e-6f, 0x100, 0, 0x300, 0));
    REFUSED(go(2, 2, 0, 3, 96, 96, -1.f, 0x100, 0, 0, 0));
    REFUSED(go(2, 2, 0, 3, 96, 96, 0.f / 0.f * 1.f, 0x100, 0, 0, 0));
    REFUSED(go(2, 2, 0, 3, 0, 96, 1e-6f, 0x100, 0, 0, 0));
    REFUSED(go(2, 2, 0, 3, (1 << 20) + 1, 1 << 21, 1e-6f, 0x100, 0, 0, 0));
    REFUSED(go(2, 2, 0, -1, 96, 96, 1e-6f, 0x100, 0, 0, 0));
    FINE(go(2, 2, 0, (1 << 22) - 1, 96, 96, 1e-6f, 0x100, 0, 0, 0));
    REFUSED(go(2, 2, 0, 1 << 22, 96, 96, 1e-6f, 0x100, 0, 0, 0));
    REFUSED(go(2, 2, 0, 3, 96, 96, 1e-6f, 0x101, 0, 0, 0));
    REFUSED(go(0, 0, 0, 3, 96, 96, 1e-6f, 0x102, 0, 0, 0));
    REFUSED(go(2, 2, 0, 3, 96, 96, 1e-6f, 0, 0, 0, 0));
}

static void products() {
    auto go = [](int n_out, int n_in, int group, int xt, int yt, int xg, int rows, int64_t xs, uintptr_t codes, uintptr_t sc, uintptr_t xsc) {
        return check_q4((void *)codes, (void *)sc, nullptr, n_out, n_in, group, (void *)0x1000, xs, xt, (float *)xsc, xg, (void *)0x2000, n_out > 0 ? n_out : 1, yt, rows);
    };
    FINE(go(5, 256, 32, 2, 2, 0, 3, 256, 0x10, 0x20, 0));
    FINE(go(5, 256, 32, 3, 0, 8, 3, 256, 0x10, 0x20, 0x40));
    FINE(go(5, 256, 128, 3, 2, 1, 3, 272, 0x10, 0x20, 0x40));
    FINE(go(0, 256, 32, 2, 2, 0, 3, 256, 0, 0, 0));
    FINE(go(5, 256, 32, 2, 2, 0, 0, 256, 0, 0, 0));
    REFUSED(go(5, 256, 32, 4, 2, 0, 3, 256, 0x10, 0x20, 0));
    REFUSED(go(5, 256, 32, 2, 1, 0, 3, 256, 0x10, 0x20, 0));
    REFUSED(go(5, 256, 16, 2, 2, 0, 3, 256, 0x10, 0x20, 0));
    REFUSED(go(5, 224, 128, 2, 2, 0, 3, 256, 0x10, 0x20, 0));
    REFUSED(go(5, 0, 32, 2, 2, 0, 3, 256, 0x10, 0x20, 0));
    REFUSED(go(-1, 256, 32, 2, 2, 0, 3, 256, 0x10, 0x20, 0));
    REFUSED(go(5, 256, 32, 3, 2, 4, 3, 256, 0x10, 0x20, 0x40));
    REFUSED(go(5, 256, 32, 3, 2, 8, 3, 256, 0x10, 0x20, 0));
    REFUSED(go(5, 256, 32, 2, 2, 0, 3, 256, 0x10, 0x20, 0x40));
    REFUSED(go(5, 256, 32, 2, 2, 8, 3, 256, 0x10, 0x20, 0));
    REFUSED(go(5, 256, 32, 2, 2, 0, -1, 256, 0x10, 0x20, 0));
    REFUSED(go(5, 256, 32, 2, 2, 0, 70000, 256, 0x10, 0x20, 0));
    REFUSED(go(5, 256, 32, 2, 2, 0, 3, 255, 0x10, 0x20, 0));
    REFUSED(go(5, 256, 32, 2, 2, 0, 3, 260, 0x10, 0x20, 0));
    REFUSED(go(5, 256, 32, 2, 2, 0, 3, 256, 0x18, 0x20, 0));
    REFUSED(go(5, 256, 32, 2, 2, 0, 3, 256, 0x10, 0, 0));
}

int main() {
    spans();
    cuts();
    rows();
    caches();
    moves();
    attentions();
    norms();
    products();
    printf("fuzz_ops OK (%d refusals)\n", refused);
    return 0;
}
