// Index arithmetic of the token-step operators, the same on host and device: how a sequence is cut into chunks, which keys a chunk has, and
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

// Keys [from, to) of chunk `c` of a sequence of n tokens, out of those its new token sees, [lo, hi); `active` chunks have any.  A length
// outside 0 .. max_len is bad: no key is read, and chunk 0 is there to say so.
struct AttnSpan { int lo, hi, from, to, active; bool bad; };
OPS_FN AttnSpan attn_span(int n, int max_len, int window, int chunk, int c) {
    AttnSpan s;
    s.bad = n < 0 || n > max_len;
    s.hi = s.bad ? 0 : n;
    s.lo = window > 0 && s.hi > window ? s.hi - window : 0;
    const int base = s.lo & ~31;                            // chunks start on a multiple of the 32-key tile
    s.active = s.bad ? 1 : (int)(((int64_t)s.hi - base + chunk - 1) / chunk);
    const int64_t from = (int64_t)base + (int64_t)c * chunk, to = from + chunk;
    s.from = (int)(from < s.hi ? from : s.hi);
    s.to = (int)(to < s.hi ? to : s.hi);
    return s;
}

// Position of row t of a call in its sequence (rows start at cu, the first stands at position `first`); -1: not in the sequence's pages
OPS_FN int64_t row_position(int t, int cu, int first, int table_width, int page_shift) {
    const int64_t pos = (int64_t)first + t - cu;
    return pos < 0 || t < cu || pos >= ((int64_t)table_width << page_shift) ? -1 : pos;
}
OPS_FN bool page_ok(int page, int n_pages) { return (unsigned)page < (unsigned)n_pages; }

struct AttnPlan { int chunk, n_chunks; size_t bytes; };
// How a call is cut, from sizes alone.  The longest sequence decides the chunk; shorter ones have fewer of the same length.
inline AttnPlan attention_plan(int head_dim, int kv_heads, int n_heads, int n_seqs, int max_len, int window) {
    AttnPlan p;
    const int64_t span = window > 0 && (int64_t)window + 31 < max_len ? (int64_t)window + 31 : max_len;
    const int64_t pairs = (int64_t)n_seqs * kv_heads;
    int64_t parts = 2048 / (pairs > 0 ? pairs : 1);
    if (parts < 1) parts = 1;
    int64_t chunk = (span + parts - 1) / parts;
    chunk = (chunk + 127) / 128 * 128;
    if (chunk < 256) chunk = 256;
    p.chunk = (int)chunk;
    p.n_chunks = (int)((span + chunk - 1) / chunk);
    if (p.n_chunks < 1) p.n_chunks = 1;
    p.bytes = p.n_chunks > 1 ? (size_t)n_seqs * n_heads * p.n_chunks * (head_dim + 2) * sizeof(float) : 0;
    return p;
}

}  // namespace hipvoc
