// Index arithmetic of the token-step operators, the same on host and device: how a call's keys are cut, which of them a workgroup has, and
// where a token's row is.  Pure C++, so that tests/native/fuzz_ops.cpp can check on the CPU that no length, offset or page number leads
// out of bounds.
#pragma once
#include <stddef.h>
#include <stdint.h>

#ifdef __HIPCC__
#define OPS_FN __host__ __device__ __forceinline__
#else
#define OPS_FN inline
#endif

namespace hipvoc {

// ---- attention: which keys a token sees, and which of them a workgroup has ---------------------------------------------------------------
// Keys come in tiles of 32, counted from `base`, the first seen key lo rounded down to a tile.  A length outside 0 .. max_len is bad: no
// key is read.
struct AttnSpan { int lo, hi, base, tiles; bool bad; };
OPS_FN AttnSpan attn_span(int n, int max_len, int window) {
    AttnSpan s;
    s.bad = n < 0 || n > max_len;
    s.hi = s.bad ? 0 : n;
    s.lo = window > 0 && s.hi > window ? s.hi - window : 0;
    s.base = s.lo & ~31;
    s.tiles = (int)(((int64_t)s.hi - s.base + 31) / 32);
    return s;
}

// A call is cut over all its tiles at once: they stand in a row (sequence by sequence, in it head by head), `total` of them, and worker w of
// `workers` (a wave, or a workgroup for 32-bit caches) has the tiles [first(w), first(w + 1)), whatever sequences they belong to.  So
// sequences of unequal length load the card alike.  A piece (the part of one sequence and head that a worker has) leaves its state in slot
// w + pair, pair = sequence * heads + head: along the row every piece has a larger w or a larger pair than the one before, so no two share one.
OPS_FN int64_t attn_workers(int64_t total, int least, int most) {              // a worker has `least` tiles, if there are that many
    const int64_t w = (total + least - 1) / least;
    return w < most ? w : most;
}
OPS_FN int64_t attn_first(int64_t w, int64_t total, int64_t workers) { return w * total / workers; }
OPS_FN int64_t attn_worker_of(int64_t tile, int64_t total, int64_t workers) { return ((tile + 1) * workers - 1) / total; }

// Position of row t of a call in its sequence (rows start at cu, the first stands at position `first`); -1: not in the sequence's pages
OPS_FN int64_t row_position(int t, int cu, int first, int table_width, int page_shift) {
    const int64_t pos = (int64_t)first + t - cu;
    return pos < 0 || t < cu || pos >= ((int64_t)table_width << page_shift) ? -1 : pos;
}
OPS_FN bool page_ok(int page, int n_pages) { return (unsigned)page < (unsigned)n_pages; }

// A launch's threads have to be counted in 32 bits.
static const int64_t OPS_MAX_THREADS = ((int64_t)1 << 32) - 1;
// Waves that have a token's 2 * kv_heads rows: a wave has KV_U times as many as its lanes hold at eight values each
enum { KV_U = 4 };
OPS_FN int kv_parts(int kv_heads, int head_dim) { return (2 * kv_heads * head_dim + 512 * KV_U - 1) / (512 * KV_U); }

struct AttnPlan { int heads, workers, least; size_t bytes; };
enum { ATTN_MAX_SEQS = 1024 };      // sequences whose lengths a workgroup adds up
// How a call is cut, from sizes alone.  `heads`: (key head, tile of query heads) pairs of a sequence.  A workgroup each (workers 0) if the spans are so
// short that cutting and joining would cost more than it gives, or the sequences so many that they fill the card (2 query heads in bf16, us, whole /
// cut: 16 pairs of 512 keys 10 / 12, of 768 13 / 12; 64 of 768 15 / 16, of 1024 18 / 17; 256 of 1024 22 / 29).  Else the workers that the card
// holds at a time share the tiles.
inline AttnPlan attention_plan(int dtype, bool coded, int head_dim, int kv_heads, int n_heads, int n_seqs, int max_len, int window) {
    AttnPlan p;
    const bool rows = dtype == 0 && !coded;              // 32-bit caches: a kernel of their own
    const int group = n_heads / kv_heads, most = !rows ? 16 : group < 3 ? group : 4;      // query heads of a pair
    const int64_t span = window > 0 && (int64_t)window + 31 < max_len ? (int64_t)window + 31 : max_len, tiles = (span + 31) / 32;
    p.heads = kv_heads * ((group + most - 1) / most);
    p.least = rows ? 8 : 1;
    p.workers = 0;
    p.bytes = 0;
    const int64_t pairs = (int64_t)n_seqs * p.heads;
    if (tiles > (pairs < 256 ? 24 : 32) && n_seqs <= ATTN_MAX_SEQS) {
        // what the card holds, and no more pieces of a pair than the join is quick with (2 x 32768 tokens of one key head: 512 16 us, 1536 21)
        // (32-bit caches: 3 workgroups a CU, or 2 with the 200 registers of 4 query heads -- 3 x 6920 tokens, 28 heads on 4 of 64, planned for 2 / 3:
        // 26 / 34 us; else 12 or 8 waves)
        const int64_t held = 256 * (rows ? (most == 4 ? 2 : 3) : coded && (dtype != 0 || head_dim == 64) ? 12 : 8);
        p.workers = (int)attn_workers(pairs * tiles, p.least, (int)(held < 512 * pairs ? held : 512 * pairs));
        // slots of up to `most` heads: (m, l) and the sums; then the row's length before each sequence
        p.bytes = (size_t)(p.workers + pairs) * (size_t)(group < most ? group : most) * (size_t)(head_dim + 2) * sizeof(float);
        p.bytes = (p.bytes + 15) / 16 * 16 + (size_t)(n_seqs + 1) * sizeof(int64_t);
    }
    return p;
}

}  // namespace hipvoc
