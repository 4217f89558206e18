// Attention of one new token per sequence over the paged cache (include/hipvoc_ops.h: hipvoc_attention).
//
// Mathematics: one pass over the keys with a running maximum m and sum l per query head (softmax in powers of two, s = q.k * scale *
// log2(e)):  m' = max(m, s), l' = l 2^(m-m') + 2^(s-m'), o' = o 2^(m-m') + 2^(s-m') v.  States (m, l, o) of disjoint key sets join by
// the same rule.
// Bound: memory.  Every key and value row is read once for all query heads of its key head (up to 16 of them; 4 on a 32-bit cache).
// Split: n_seqs * kv_heads workgroups do not fill 256 CUs, and sequences differ in length.  So all the tiles of a call stand in one row and
// every wave (32-bit caches: workgroup) has an equal share of it, wherever its ends fall (ops_index.hpp); the pieces of a sequence are
// joined by a second kernel, without atomics: the order of every sum follows from the call's lengths.  A grid of fixed
// chunks gave the chip's dies unequal ones: 32 sequences of up to 4095 tokens, 8 key heads of 128, 16 query heads in bf16 (272 MB) 72 us, so 55.5 us
// (4.9 TB/s).  131071 tokens, 32 query heads in f16 (537 MB) 96 us, 5.6 TB/s; 64 sequences of up to 8192 in 8 bits (566 MB) 110 us, 5.1 TB/s.
// 32-bit activations, 32 sequences of up to 4095: 544 MB of 32-bit cache 109 us; 8 bits as fast as 16-bit activations (below).  32-bit caches, 4 query heads
// at a time: 3 x 6920 tokens, 28 heads on 4 of 64 (read twice): 26 us, 16 heads 22.
#include <type_traits>

#include "ops_device.h"

namespace hipvoc {

// A piece of work: the keys [from, to) of one sequence for one pair (key head, up to H of its query heads), out of those seen, [lo, hi).
// slot < 0: all the keys there are, the result is written at once.
struct AttnPiece { int seq, kvh, h0, lo, from, to; int64_t slot; bool bad; };

// What is left in a slot: o [H][head_dim], (m, l) [H]
template <int HD, int H> __device__ __forceinline__ float *slot_o(const AttnArgs &a, int64_t slot, int h) {
    const int n = min(a.group, H);
    return a.part + (slot * n + h) * HD;
}
template <int HD, int H> __device__ __forceinline__ f32v2 *slot_ml(const AttnArgs &a, int64_t slot, int h) {
    const int n = min(a.group, H);
    return (f32v2 *)(a.part + ((int64_t)a.workers + (int64_t)a.n_seqs * a.heads) * n * HD) + slot * n + h;
}

// The row of a call's tiles, as every workgroup finds it by itself: the lengths, and tiles (of one pair) before each sequence, by a scan over up
// to 1024 lengths in LDS, which costs a microsecond and spares a launch.  The first workgroup leaves it for the join.
__device__ __forceinline__ int64_t attn_row(const AttnArgs &a, int64_t *before, int *lens) {
    __shared__ int64_t wave_sum[4];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    int64_t mine[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int b = 4 * t + i, n = b < a.n_seqs ? a.lens[b] : 0;
        lens[b] = n;
        sum += attn_span(n, a.max_len, a.window).tiles;
        mine[i] = sum;
    }
    int64_t upto = sum;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const int64_t v = __shfl_up(upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 63) wave_sum[wave] = upto;
    __syncthreads();
    int64_t start = upto - sum;
    for (int w = 0; w < wave; w++) start += wave_sum[w];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int b = 4 * t + i;
        if (b < a.n_seqs) before[b + 1] = start + mine[i];
    }
    if (t == 0) before[0] = 0;
    __syncthreads();
    if (blockIdx.x == 0)
        for (int b = t; b <= a.n_seqs; b += 256) a.before[b] = before[b];
    return before[a.n_seqs] * a.heads;
}
// The sequence that tile x of the row belongs to
__device__ __forceinline__ int attn_seq_of(const AttnArgs &a, const int64_t *before, int64_t x) {
    int seq = 0;
    for (int n = a.n_seqs; n > 1;) {
        const int half = n / 2;
        if (before[seq + half] * a.heads <= x) seq += half;
        n -= half;
    }
    while (before[seq + 1] * a.heads <= x) seq++;
    return seq;
}

// Runs `work` on a workgroup's pieces: its own pair, or its share of the row.
template <int H, typename Work> __device__ __forceinline__ void attn_pieces(const AttnArgs &a, Work &&work) {
    __shared__ int64_t before[ATTN_MAX_SEQS + 1];
    __shared__ int lens[ATTN_MAX_SEQS];
    const bool cut = a.workers > 0;
    int64_t x = 0, end = 1;
    int seq = blockIdx.x / a.heads;
    if (cut) {
        const int64_t total = attn_row(a, before, lens), workers = attn_workers(total, a.least, a.workers);
        if (blockIdx.x >= workers) return;                             // nothing at all: no workers
        x = attn_first(blockIdx.x, total, workers);
        end = attn_first(blockIdx.x + 1, total, workers);
        seq = attn_seq_of(a, before, x);
    }
    while (x < end) {
        AttnPiece p;
        int pair = blockIdx.x % a.heads, tile = 0;
        int64_t n = 1;
        if (cut)
            while (before[seq + 1] * a.heads <= x) seq++;
        const AttnSpan s = attn_span(cut ? lens[seq] : a.lens[seq], a.max_len, a.window);
        p.slot = -1;
        p.to = s.hi;
        if (cut) {
            const int64_t rest = x - before[seq] * a.heads;
            pair = (int)(rest / s.tiles);
            tile = (int)(rest - (int64_t)pair * s.tiles);
            n = min((int64_t)(s.tiles - tile), end - x);
            if (n < s.tiles) {
                p.slot = blockIdx.x + (int64_t)seq * a.heads + pair;
                p.to = (int)min((int64_t)s.hi, s.base + 32 * (tile + n));
            }
        }
        const int tiles = (a.group + H - 1) / H;
        p.seq = seq;
        p.kvh = pair / tiles;
        p.h0 = p.kvh * a.group + pair % tiles * H;
        p.lo = s.lo;
        p.from = s.base + 32 * tile;
        p.bad = s.bad;
        work(p);
        x += n;
    }
}

__device__ __forceinline__ float lse_of(float m, float l) { return (m + log2f(l)) * 0.69314718055994530942f; }

// Joins the states of a workgroup's NW waves and leaves the piece's state, or writes the result where the piece is all there is.
// ml(w, h) = (m, l) of wave w for the piece's head h, o(w, h, d) its sums.
template <int ACT, int HD, int NW, int H, typename ML, typename O>
__device__ __forceinline__ void attn_finish(const AttnArgs &a, const AttnPiece &p, int nh, bool nan, ML &&ml, O &&o) {
    for (int i = threadIdx.x; i < nh * HD; i += 64 * NW) {
        const int h = i / HD, d = i % HD, head = p.h0 + h;
        float top = ml(0, h)[0];
#pragma unroll
        for (int w = 1; w < NW; w++) top = fmaxf(top, ml(w, h)[0]);
        const float safe = top == -__builtin_inff() ? 0.f : top;
        float x = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const f32v2 s = ml(w, h);
            const float f = exp2f(s[0] - safe);
            sum += s[1] * f;
            x += o(w, h, d) * f;
        }
        if (nan) x = sum = top = __builtin_nanf("");
        if (p.slot >= 0) {
            slot_o<HD, H>(a, p.slot, h)[d] = x;
            if (d == 0) *slot_ml<HD, H>(a, p.slot, h) = (f32v2){top, sum};
        } else {
            store1<ACT>(a.out, p.seq * a.out_stride + (int64_t)head * HD + d, sum == 0.f ? 0.f : x / sum);
            if (d == 0 && a.lse) a.lse[(int64_t)p.seq * a.n_heads + head] = lse_of(top, sum);
        }
    }
}

// 32-bit caches: a wave reads rows of HD values with HD / 8 lanes each, U rows per lane in flight, and keeps HT query heads in registers.
template <int HD, int HT>
__global__ __launch_bounds__(256) void attn_rows_kernel(AttnArgs a) {
    constexpr int ACT = HIPVOC_T_F32;
    constexpr int LPR = HD / 8, KPS = 64 / LPR, U = 4, TILE = U * KPS, NW = 4;
    __shared__ float sh_o[NW][HT][HD], sh_m[NW][HT], sh_l[NW][HT];
    __shared__ int sh_bad[NW];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), d = (lane % LPR) * 8, kl = lane / LPR;
    attn_pieces<HT>(a, [&](const AttnPiece &sp) {
        const int seq = sp.seq, kvh = sp.kvh, h0 = sp.h0, nh = min(HT, (kvh + 1) * a.group - h0);
        if (sp.bad && threadIdx.x == 0) raise(a.err, OPS_ERR_LENGTH);
        float q[HT][8], o[HT][8], m[HT], l[HT];
#pragma unroll
        for (int h = 0; h < HT; h++) {
            m[h] = -__builtin_inff();
            l[h] = 0.f;
            load8<ACT>((const float *)a.q + seq * a.q_stride + (int64_t)min(h0 + h, h0 + nh - 1) * HD + d, q[h]);
#pragma unroll
            for (int i = 0; i < 8; i++) o[h][i] = 0.f;
        }
        const int32_t *table = a.table + seq * a.table_stride;
        bool bad = false;
        const auto tile = [&](int base, auto partial) {
            constexpr bool PART = decltype(partial)::value;
            float k[U][8], v[U][8], s[HT][U];
            bool in[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int key = base + u * KPS + kl, kc = PART ? min(max(key, sp.lo), sp.to - 1) : key;       // what is masked is read from a row that is not
                in[u] = !PART || (key >= sp.lo && key < sp.to);
                int page = table[kc >> a.page_shift];
                if (!page_ok(page, a.c.n_pages)) { bad = true; page = 0; }
                const int in_page = kc & (a.c.page - 1);
                const int64_t row = page * a.c.page_stride + ((int64_t)kvh * a.c.page + in_page) * HD + d;
                load8<ACT>((const float *)a.c.k + row, k[u]);
                load8<ACT>((const float *)a.c.v + row, v[u]);
            }
#pragma unroll
            for (int h = 0; h < HT; h++) {
                float top = m[h];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    float x = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; i++) x = fmaf(q[h][i], k[u][i], x);
                    x = sum_lanes<LPR>(x);
                    s[h][u] = in[u] ? x * a.scale_log2 : -__builtin_inff();
                    top = fmaxf(top, s[h][u]);
                }
                const float safe = top == -__builtin_inff() ? 0.f : top, old = __builtin_amdgcn_exp2f(m[h] - safe);
                m[h] = top;
                l[h] *= old;
#pragma unroll
                for (int i = 0; i < 8; i++) o[h][i] *= old;
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (PART && h == 0) {                                // that row may hold an infinity, and 0 times it is NaN
#pragma unroll
                        for (int i = 0; i < 8; i++) v[u][i] = in[u] ? v[u][i] : 0.f;
                    }
                    const float p = __builtin_amdgcn_exp2f(s[h][u] - safe);
                    l[h] += p;
#pragma unroll
                    for (int i = 0; i < 8; i++) o[h][i] = fmaf(p, v[u][i], o[h][i]);
                }
            }
        };
        for (int base = sp.from + wave * TILE; base < sp.to; base += NW * TILE) {
            if (base >= sp.lo && base + TILE <= sp.to) tile(base, std::false_type());
            else tile(base, std::true_type());
        }
        const bool wave_bad = __any(bad);
        if (lane == 0) {
            if (wave_bad) raise(a.err, OPS_ERR_PAGE);
            sh_bad[wave] = wave_bad || sp.bad;
        }
        // join the wave's KPS key groups, then the four waves
#pragma unroll
        for (int h = 0; h < HT; h++) {
#pragma unroll
            for (int off = LPR; off < 64; off *= 2) {
                const float m2 = __shfl_xor(m[h], off), l2 = __shfl_xor(l[h], off), top = fmaxf(m[h], m2), safe = top == -__builtin_inff() ? 0.f : top;
                const float f1 = exp2f(m[h] - safe), f2 = exp2f(m2 - safe);
                m[h] = top;
                l[h] = l[h] * f1 + l2 * f2;
#pragma unroll
                for (int i = 0; i < 8; i++) o[h][i] = o[h][i] * f1 + __shfl_xor(o[h][i], off) * f2;
            }
            if (kl == 0) {
#pragma unroll
                for (int i = 0; i < 8; i++) sh_o[wave][h][d + i] = o[h][i];
                if (d == 0) { sh_m[wave][h] = m[h]; sh_l[wave][h] = l[h]; }
            }
        }
        __syncthreads();
        attn_finish<ACT, HD, NW, HT>(a, sp, nh, (sh_bad[0] | sh_bad[1] | sh_bad[2] | sh_bad[3]) != 0, [&](int w, int h) { return f32v2{sh_m[w][h], sh_l[w][h]}; },
                                    [&](int w, int h, int d) { return sh_o[w][h][d]; });
        __syncthreads();                                                     // another piece may follow
    });
}

// ---------------------------------------------------------------------------------------------------------------------
// 16-bit activations, and 32-bit ones on 8-bit caches, on the matrix cores.  A wave has tiles of 32 keys for up to 16 query heads:
//   S^T = K Q^T   (rows = keys, columns = heads): a lane of (m = lane % 16, j = lane / 16) reads key rows as they lie, 16 bytes at a time.
//                 Row m of half t is key 8 (m / 4) + 4 t + m % 4, so a lane's eight results are the scores of ONE head for the keys 8j .. 8j+7,
//   O^T = V^T P^T (rows = values' columns, columns = heads): and these, rounded, are at once the right operand.  The left one needs a column
//                 of V for eight keys: the lane reads HD/16 neighbouring columns of its eight keys' rows (whole rows across 16 lanes) and
//                 turns them with one byte permutation per two values; row m of product i is column m HD/16 + i.
// So neither K, V nor P passes through LDS.  Scores, m, l and O are in 32 bits; P goes into the product with V as two values of V's own type (bf16 for
// 8-bit codes, which bf16 and f16 hold exactly, and whose scales are in the scores and in P): see weights().  A 32-bit q or weight is three bf16, exactly:
// three matrix instructions for one, which cost no time: 32 sequences of 2048 .. 4095 tokens, 8 key heads of 128 in INT8 (203 MB), 16 query heads 50 us in
// 32 bits and 52 in bf16, 64 query heads 55 and 58.
// What is masked is read from a row that is not (so that no stale value, NaN or page number behind the last token matters).

// four codes to two pairs of 16-bit values, exactly
template <int ST, bool F16> __device__ __forceinline__ u32x2 widen4(unsigned w) {
    if constexpr (ST == HIPVOC_T_E4M3) {
        if constexpr (F16)
            return (u32x2){__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false)),
                           __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true))};
        else
            return (u32x2){__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false)),
                           __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true))};
    } else {
        float f[4];
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = (float)(int8_t)(w >> (8 * i));
        if constexpr (F16) return (u32x2){pack_f16(f[0], f[1]), pack_f16(f[2], f[3])};
        else return (u32x2){pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3])};
    }
}
template <bool F16> __device__ __forceinline__ f32x4 mfma32(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
}
// two floats as the sums of three bf16 each, exactly: cut off (not rounded: nothing can overflow) after 8 significant bits
__device__ __forceinline__ void thirds(float x, float y, unsigned &a, unsigned &b, unsigned &c) {
    const float x0 = bf16_hi(__float_as_uint(x)), y0 = bf16_hi(__float_as_uint(y)), x1 = bf16_hi(__float_as_uint(x - x0)), y1 = bf16_hi(__float_as_uint(y - y0));
    a = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302);
    b = __builtin_amdgcn_perm(__float_as_uint(y1), __float_as_uint(x1), 0x07060302);
    c = __builtin_amdgcn_perm(__float_as_uint(y - y0 - y1), __float_as_uint(x - x0 - x1), 0x07060302);
}
// maximum over the four lanes of a head (lane % 16)
__device__ __forceinline__ float max_of_head(float v) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Keys and values are read once: non-temporal loads (512 MB: 6.9 TB/s against 6.1).
template <typename T> __device__ __forceinline__ T once(const T *p) { return __builtin_nontemporal_load(p); }

// Waves per SIMD that the matrix kernels' registers have to leave room for: 3 with up to 168 registers, of which attn_stream_kernel has 158 .. 165 for
// head_dim 128; three times q does not fit those.
constexpr int attn_waves(int act) { return act == HIPVOC_T_F32 ? 2 : 3; }

// The keys and values of one tile for one wave, and what they do to the state of its heads
template <int ACT, int ST, int HD> struct AttnWave {
    static constexpr bool CODED = ST != ACT, WIDE = ACT == HIPVOC_T_F32, QF16 = ACT == HIPVOC_T_F16, PF16 = QF16 && !CODED;
    static constexpr int QP = WIDE ? 3 : 1, P = WIDE ? 3 : 2;            // operands that are together q, and the weights
    static constexpr int NC = HD / 32, NV = HD / 16;                     // products of S per 16 keys, and of O
    static constexpr int KW = CODED ? HD / 64 : NC, VW = CODED ? HD / 64 : HD / 32;      // 16-byte words of a key row, dwords of a value row that a lane reads
    typedef typename Store<ACT>::type act_t;
    typedef typename Store<ST>::type st_t;

    // A tile: its first key, the keys seen, the key head, the sequence's pages
    struct Tile { int base, lo, hi, kvh; const int32_t *table; };

    u32x4 q[QP][NC], k[2][KW];
    unsigned v[8][VW];
    f32x4 ks[2], vs[2], o[NV];
    float m, l;

    // The state counts in 2^SHIFT: l and o hold 2^(s - m + SHIFT).  Without it an f16 weight under 2^-14 of the largest would lose bits (and a long
    // cache of small weights its sum); so they keep theirs down to 2^-29.
    static constexpr float SHIFT = PF16 ? 15.f : 0.f;
    __device__ __forceinline__ float base_of() const { return m - SHIFT; }          // what a state's sums are relative to

    static __device__ __forceinline__ bool whole(const Tile &t) { return t.base >= t.lo && t.base + 32 <= t.hi; }
    // group e of eight keys, or another one where all of it is masked
    static __device__ __forceinline__ int group(const Tile &t, int e) {
        const int g = t.base + 8 * e;
        return whole(t) ? g : min(max(g, t.lo & ~7), (t.hi - 1) & ~7);
    }
    static __device__ __forceinline__ int page_k(const AttnArgs &a, const Tile &t, int lane) { return t.table[group(t, (lane & 15) >> 2) >> a.page_shift]; }
    static __device__ __forceinline__ int page_v(const AttnArgs &a, const Tile &t, int lane) { return t.table[group(t, lane >> 4) >> a.page_shift]; }

    __device__ __forceinline__ void start(const AttnArgs &a, int seq, int h0, int nh, int lane) {
        const int m16 = lane & 15, j = lane >> 4;
        const act_t *row = (const act_t *)a.q + seq * a.q_stride + (int64_t)(h0 + min(m16, nh - 1)) * HD;
#pragma unroll
        for (int i = 0; i < NC; i++) {
            const act_t *at = row + (CODED ? (i >> 1) * 64 + 16 * j + 8 * (i & 1) : 32 * i + 8 * j);
            if constexpr (WIDE) {
                float f[8];
                load8<ACT>(at, f);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    unsigned a, b, c;
                    thirds(f[2 * e], f[2 * e + 1], a, b, c);
                    q[0][i][e] = a;
                    q[1][i][e] = b;
                    q[2][i][e] = c;
                }
            } else {
                q[0][i] = *(const u32x4 *)at;
            }
        }
        m = -__builtin_inff();
        l = 0.f;
#pragma unroll
        for (int i = 0; i < NV; i++) o[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }

    // Loads are always issued, so that the compiler can count them in order: where there is no tile every lane reads the same row.
    __device__ __forceinline__ void load_k(const AttnArgs &a, const Tile &t, int page, int page_v, bool real, int lane) {
        const int m16 = lane & 15, j = lane >> 4, g = group(t, m16 >> 2);
        const st_t *kp = (const st_t *)a.c.k + page * a.c.page_stride + (int64_t)t.kvh * a.c.page * HD;
        const auto rows = [&](const st_t *r0, const st_t *r1) {
#pragma unroll
            for (int i = 0; i < KW; i++) {
                k[0][i] = once((const u32x4 *)(r0 + (CODED ? 64 : 32) * i));
                k[1][i] = once((const u32x4 *)(r1 + (CODED ? 64 : 32) * i));
            }
        };
        const int in_row = (CODED ? 16 : 8) * j;
        if (whole(t)) {                                                  // eight keys of a group are eight rows of one page
            const st_t *row = kp + (real ? ((g & (a.c.page - 1)) + (m16 & 3)) * HD + in_row : 0);
            rows(row, row + 4 * HD);
        } else {
            const auto row = [&](int e) { return kp + (min(max(g + e, t.lo), t.hi - 1) & (a.c.page - 1)) * HD + in_row; };
            rows(row(m16 & 3), row(4 + (m16 & 3)));
        }
        if constexpr (CODED) {
            const float *sc = a.c.k_scale + ((int64_t)page_v * a.c.kv_heads + t.kvh) * a.c.page + (group(t, j) & (a.c.page - 1));
            ks[0] = once((const f32x4 *)sc);
            ks[1] = once((const f32x4 *)(sc + 4));
        }
    }
    __device__ __forceinline__ void load_v(const AttnArgs &a, const Tile &t, int page, bool real, int lane) {
        const int m16 = lane & 15, j = lane >> 4, g = group(t, j);
        const st_t *vp = (const st_t *)a.c.v + page * a.c.page_stride + (int64_t)t.kvh * a.c.page * HD;
        const auto row = [&](int e, const st_t *r) {
            if constexpr (VW == 4) *(u32x4 *)v[e] = once((const u32x4 *)r);
            else if constexpr (VW == 2) *(u32x2 *)v[e] = once((const u32x2 *)r);
            else v[e][0] = once((const unsigned *)r);
        };
        if (whole(t)) {
            const st_t *r = vp + (real ? (g & (a.c.page - 1)) * HD + m16 * NV : 0);
#pragma unroll
            for (int e = 0; e < 8; e++) row(e, r + e * HD);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) row(e, vp + (min(max(g + e, t.lo), t.hi - 1) & (a.c.page - 1)) * HD + m16 * NV);
        }
        if constexpr (CODED) {
            const float *sc = a.c.v_scale + ((int64_t)page * a.c.kv_heads + t.kvh) * a.c.page + (g & (a.c.page - 1));
            vs[0] = once((const f32x4 *)sc);
            vs[1] = once((const f32x4 *)(sc + 4));
        }
    }

    // scores of the keys base + 8j + 4t + r for head m16, in powers of two
    __device__ __forceinline__ void scores(const AttnArgs &a, const Tile &tl, float (&s)[8], int lane) const {
        const int j = lane >> 4;
#pragma unroll
        for (int t = 0; t < 2; t++) {
            f32x4 acc = {};
            if constexpr (CODED) {
#pragma unroll
                for (int i = 0; i < KW; i++) {
                    const u32x2 a0 = widen4<ST, QF16>(k[t][i][0]), a1 = widen4<ST, QF16>(k[t][i][1]), a2 = widen4<ST, QF16>(k[t][i][2]), a3 = widen4<ST, QF16>(k[t][i][3]);
#pragma unroll
                    for (int p = 0; p < QP; p++) {
                        acc = mfma32<QF16>((u32x4){a0[0], a0[1], a1[0], a1[1]}, q[p][2 * i], acc);
                        acc = mfma32<QF16>((u32x4){a2[0], a2[1], a3[0], a3[1]}, q[p][2 * i + 1], acc);
                    }
                }
                acc *= ks[t];
            } else {
#pragma unroll
                for (int i = 0; i < NC; i++) acc = mfma32<QF16>(k[t][i], q[0][i], acc);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) s[4 * t + r] = acc[r] * a.scale_log2;
        }
        if (!whole(tl)) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int key = tl.base + 8 * j + e;
                if (key < tl.lo || key >= tl.hi) s[e] = -__builtin_inff();
            }
        }
    }
    // The running maximum and sum, and the weights as the right operand of the product with V: two operands whose sum they are, in the second what
    // the first leaves over.  One alone (bf16: 8 bits, f16: 11) would add as much error again as the rounding of the result, or a good part of it, and
    // the second product costs a tile 8 matrix instructions of 16 cycles and 20 vector ones, under the time of its loads: no time measured.
    __device__ __forceinline__ void weights(const Tile &tl, const float (&s)[8], int lane, u32x4 (&pp)[P]) {
        const int j = lane >> 4;
        float top = m;
#pragma unroll
        for (int e = 0; e < 8; e++) top = fmaxf(top, s[e]);
        top = max_of_head(top);
        if (__any(top > m)) {                                            // else nothing to scale down
            const float f = __builtin_amdgcn_exp2f(base_of() - (top == -__builtin_inff() ? 0.f : top - SHIFT));
            m = top;
            l *= f;
#pragma unroll
            for (int i = 0; i < NV; i++) o[i] *= f;
        }
        const float safe = m == -__builtin_inff() ? 0.f : base_of();
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            p[e] = __builtin_amdgcn_exp2f(s[e] - safe);
            l += p[e];
            if constexpr (CODED) p[e] *= vs[e >> 2][e & 3];
        }
        if constexpr (CODED) {
            if (!whole(tl)) {                                            // a scale that nothing was written to may be anything
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int key = tl.base + 8 * j + e;
                    if (key < tl.lo || key >= tl.hi) p[e] = 0.f;
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if constexpr (WIDE) {
                unsigned a, b, c;
                thirds(p[2 * e], p[2 * e + 1], a, b, c);
                pp[0][e] = a;
                pp[1][e] = b;
                pp[2][e] = c;
            } else if constexpr (PF16) {
                const unsigned hi = pack_f16(p[2 * e], p[2 * e + 1]);
                const h16x2 most = __builtin_bit_cast(h16x2, hi);       // (cast from pp[0][e] itself the compiler takes pp[0][0])
                pp[0][e] = hi;
                pp[1][e] = pack_f16(p[2 * e] - (float)most[0], p[2 * e + 1] - (float)most[1]);
            } else {
                pp[0][e] = pack_bf16(p[2 * e], p[2 * e + 1]);
                pp[1][e] = pack_bf16(p[2 * e] - bf16_lo(pp[0][e]), p[2 * e + 1] - bf16_hi(pp[0][e]));
            }
        }
    }
    __device__ __forceinline__ void values(const u32x4 (&pp)[P]) {
        unsigned w[8][HD / 32];                                          // the value rows in 16 bits
#pragma unroll
        for (int e = 0; e < 8; e++) {
#pragma unroll
            for (int i = 0; i < VW; i++) {
                if constexpr (CODED) {
                    const u32x2 x = widen4<ST, false>(v[e][i]);
                    w[e][2 * i] = x[0];
                    w[e][2 * i + 1] = x[1];
                } else {
                    w[e][i] = v[e][i];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < NV; i++) {
            u32x4 col;
#pragma unroll
            for (int e = 0; e < 4; e++) col[e] = __builtin_amdgcn_perm(w[2 * e + 1][i >> 1], w[2 * e][i >> 1], i & 1 ? 0x07060302 : 0x05040100);
#pragma unroll
            for (int p = 0; p < P; p++) o[i] = mfma32<PF16>(col, pp[p], o[i]);
        }
    }
    __device__ __forceinline__ float sum_of_head() const {
        float x = l + __shfl_xor(l, 16);
        return x + __shfl_xor(x, 32);
    }
};

// A workgroup per (sequence, pair), its four waves on every fourth tile
template <int ACT, int ST, int HD>
__global__ __launch_bounds__(256, attn_waves(ACT)) void attn_whole_kernel(AttnArgs a) {
    typedef AttnWave<ACT, ST, HD> Wave;
    constexpr int NW = 4, NV = HD / 16;
    __shared__ __attribute__((aligned(16))) float sh_o[NW][16][HD + 4];
    __shared__ float sh_m[NW][16], sh_l[NW][16];
    __shared__ int sh_bad[NW];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m16 = lane & 15, j = lane >> 4;
    const int seq = blockIdx.x / a.heads, pair = blockIdx.x % a.heads, tiles = (a.group + 15) / 16, kvh = pair / tiles;
    const int h0 = kvh * a.group + pair % tiles * 16, nh = min(16, (kvh + 1) * a.group - h0);
    const AttnSpan sp = attn_span(a.lens[seq], a.max_len, a.window);
    bool bad = false;
    Wave w;
    w.start(a, seq, h0, nh, lane);
    typename Wave::Tile t = {sp.base + 32 * wave, sp.lo, sp.hi, kvh, a.table + seq * a.table_stride};
    if (t.base < sp.hi) {
        const auto sound = [&](int page) {
            if (page_ok(page, a.c.n_pages)) return page;
            bad = true;
            return 0;
        };
        const auto step = [&](typename Wave::Tile &x) { x.base += x.base + 32 * NW < sp.hi ? 32 * NW : 0; };
        int pk = sound(Wave::page_k(a, t, lane)), pv = sound(Wave::page_v(a, t, lane));
        w.load_k(a, t, pk, pv, true, lane);
        w.load_v(a, t, pv, true, lane);
        typename Wave::Tile next = t;
        step(next);
        int nk = Wave::page_k(a, next, lane), nv = Wave::page_v(a, next, lane);
        for (;;) {                                                       // the next tile is on its way while one is worked on
            const bool more = next.base > t.base;
            float s[8];
            w.scores(a, t, s, lane);
            pk = sound(nk);
            pv = sound(nv);
            w.load_k(a, next, pk, pv, more, lane);
            u32x4 pp[Wave::P];
            w.weights(t, s, lane, pp);
            w.values(pp);
            if (!more) break;
            w.load_v(a, next, pv, true, lane);
            t = next;
            step(next);
            nk = Wave::page_k(a, next, lane);
            nv = Wave::page_v(a, next, lane);
        }
    }
    const float l = w.sum_of_head();
    const bool wave_bad = __any(bad);
    if (lane == 0) {
        if (wave_bad) raise(a.err, OPS_ERR_PAGE);
        sh_bad[wave] = wave_bad || sp.bad;
    }
    if (sp.bad && threadIdx.x == 0) raise(a.err, OPS_ERR_LENGTH);
    if (m16 < nh) {
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int i = 0; i < NV; i += 4) *(f32x4 *)&sh_o[wave][m16][(4 * j + r) * NV + i] = (f32x4){w.o[i][r], w.o[i + 1][r], w.o[i + 2][r], w.o[i + 3][r]};
        if (j == 0) { sh_m[wave][m16] = w.base_of(); sh_l[wave][m16] = l; }
    }
    __syncthreads();
    AttnPiece p = {seq, kvh, h0, sp.lo, sp.base, sp.hi, -1, sp.bad};
    attn_finish<ACT, HD, NW, 16>(a, p, nh, (sh_bad[0] | sh_bad[1] | sh_bad[2] | sh_bad[3]) != 0, [&](int w, int h) { return f32v2{sh_m[w][h], sh_l[w][h]}; },
                                [&](int w, int h, int d) { return sh_o[w][h][d]; });
}

// A wave per share of the row of tiles.  Its pipeline runs on over the ends of pieces: while a tile is worked on, the next one's keys are on
// their way as soon as this one's are used up, its values likewise, and the pages of the one after that; at a piece's end only the state is
// written and the next head's q read.
template <int ACT, int ST, int HD>
__global__ __launch_bounds__(256, attn_waves(ACT)) void attn_stream_kernel(AttnArgs a) {
    typedef AttnWave<ACT, ST, HD> Wave;
    constexpr int NV = HD / 16;
    __shared__ int64_t before[ATTN_MAX_SEQS + 1];
    __shared__ int lens[ATTN_MAX_SEQS];
    const int lane = threadIdx.x & 63, m16 = lane & 15, j = lane >> 4;
    const int64_t total = attn_row(a, before, lens), workers = attn_workers(total, a.least, a.workers);
    const int64_t worker = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (worker >= workers) return;
    const int64_t x = attn_first(worker, total, workers);
    int64_t left = attn_first(worker + 1, total, workers) - x;
    const int tiles16 = (a.group + 15) / 16;

    struct Pos { int seq, pair, tile, tiles, base0; typename Wave::Tile t; };
    const auto enter = [&](Pos &p) {                                     // a sequence's span and pages
        const AttnSpan s = attn_span(__builtin_amdgcn_readfirstlane(lens[p.seq]), a.max_len, a.window);
        p.tiles = s.tiles;
        p.base0 = s.base;
        p.t.lo = s.lo;
        p.t.hi = s.hi;
        p.t.table = a.table + p.seq * a.table_stride;
    };
    const auto place = [&](Pos &p) {
        p.t.base = p.base0 + 32 * p.tile;
        p.t.kvh = tiles16 == 1 ? p.pair : p.pair / tiles16;
    };
    const auto step = [&](Pos &p) {                                      // to the next tile of the row
        if (++p.tile == p.tiles) {
            p.tile = 0;
            if (++p.pair == a.heads) {
                p.pair = 0;
                do {
                    p.seq++;
                    enter(p);
                } while (p.tiles == 0);
            }
        }
        place(p);
    };
    Pos cur, next, after;
    cur.seq = __builtin_amdgcn_readfirstlane(attn_seq_of(a, before, x));
    enter(cur);
    const int64_t rest = x - before[cur.seq] * a.heads;
    cur.pair = (int)(rest / cur.tiles);
    cur.tile = (int)(rest - (int64_t)cur.pair * cur.tiles);
    place(cur);
    int first = cur.tile;                                                // of the piece
    bool bad = false, next_bad = false;
    const auto sound = [&](int page, bool &flag) {
        if (page_ok(page, a.c.n_pages)) return page;
        flag = true;
        return 0;
    };
    Wave w;
    {
        const int pk = sound(Wave::page_k(a, cur.t, lane), bad), pv = sound(Wave::page_v(a, cur.t, lane), bad);
        w.load_k(a, cur.t, pk, pv, true, lane);
        w.load_v(a, cur.t, pv, true, lane);
    }
    next = cur;
    if (left > 1) step(next);
    int nk = Wave::page_k(a, next.t, lane), nv = Wave::page_v(a, next.t, lane);
    const auto heads_of = [&](const Pos &p, int &h0) {
        h0 = p.t.kvh * a.group + (tiles16 == 1 ? 0 : p.pair % tiles16 * 16);
        return min(16, (p.t.kvh + 1) * a.group - h0);
    };
    int h0, nh = heads_of(cur, h0);
    w.start(a, cur.seq, h0, nh, lane);
    for (;;) {
        const int sk = sound(nk, next_bad), sv = sound(nv, next_bad);
        after = next;
        if (left > 2) step(after);
        nk = Wave::page_k(a, after.t, lane);
        nv = Wave::page_v(a, after.t, lane);
        float s[8];
        w.scores(a, cur.t, s, lane);
        w.load_k(a, next.t, sk, sv, left > 1, lane);
        u32x4 pp[Wave::P];
        w.weights(cur.t, s, lane, pp);
        w.values(pp);
        w.load_v(a, next.t, sv, left > 1, lane);
        left--;
        if (left == 0 || next.tile == 0) {                               // the piece ends
            const float l = w.sum_of_head();
            const bool all = first == 0 && cur.tile + 1 == cur.tiles, nan = __any(bad);
            if (nan && lane == 0) raise(a.err, OPS_ERR_PAGE);
            if (m16 < nh) {
                const float f = nan ? __builtin_nanf("") : all ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
                const int64_t slot = worker + (int64_t)cur.seq * a.heads + cur.pair;
                float *part = slot_o<HD, 16>(a, slot, m16);
                typename Wave::act_t *out = (typename Wave::act_t *)a.out + cur.seq * a.out_stride + (int64_t)(h0 + m16) * HD;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float y[NV];
#pragma unroll
                    for (int i = 0; i < NV; i++) y[i] = w.o[i][r] * f;
                    const int d = (4 * j + r) * NV;
                    if (all) {
                        if constexpr (NV == 8) store8<ACT>(out + d, y);
                        else if constexpr (ACT == HIPVOC_T_F32) *(f32x4 *)(out + d) = (f32x4){y[0], y[1], y[2], y[3]};
                        else *(u32x2 *)(out + d) = ACT == HIPVOC_T_F16 ? (u32x2){pack_f16(y[0], y[1]), pack_f16(y[2], y[3])} : (u32x2){pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3])};
                    } else {
#pragma unroll
                        for (int i = 0; i < NV; i += 4) *(f32x4 *)(part + d + i) = (f32x4){y[i], y[i + 1], y[i + 2], y[i + 3]};
                    }
                }
                if (j == 0) {
                    const float m = nan ? __builtin_nanf("") : w.base_of(), ll = nan ? __builtin_nanf("") : l;
                    if (!all) *slot_ml<HD, 16>(a, slot, m16) = (f32v2){m, ll};
                    else if (a.lse) a.lse[(int64_t)cur.seq * a.n_heads + h0 + m16] = lse_of(m, ll);
                }
            }
            if (left == 0) break;
            bad = false;
            first = 0;
            nh = heads_of(next, h0);
            w.start(a, next.seq, h0, nh, lane);
        }
        bad = bad || next_bad;
        next_bad = false;
        cur = next;
        next = after;
    }
}

// Joins the pieces of the pairs that were cut.  A pair's result is I = heads * head_dim / 4 quads; a workgroup has `per` of them (all the pair's, or
// fewer where the pairs do not fill the card) and walks the pieces 256 / per at a time, each thread with a running state of its own; the
// threads of a quad are joined through LDS, by halves.  A sequence without a tile has no piece: its result is written here.
template <int ACT, int HD, int H>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a, int per) {
    __shared__ __attribute__((aligned(16))) f32x4 sh_o[256];
    __shared__ f32v2 sh_ml[256];
    const int seq = blockIdx.y, pair = blockIdx.x, t = threadIdx.x, tiles_h = (a.group + H - 1) / H, kvh = pair / tiles_h;
    const int h0 = kvh * a.group + pair % tiles_h * H, nh = min(H, (kvh + 1) * a.group - h0), quads = nh * (HD / 4), groups = 256 / per;
    const int64_t b0 = a.before[seq], b1 = a.before[seq + 1], total = a.before[a.n_seqs] * a.heads, tiles = b1 - b0;
    int64_t slot0 = 0;
    int n = 0;
    bool bad = false;
    if (tiles == 0) {
        bad = attn_span(a.lens[seq], a.max_len, a.window).bad;
        if (bad && t == 0) raise(a.err, OPS_ERR_LENGTH);
    } else {
        const int64_t workers = attn_workers(total, a.least, a.workers), x = b0 * a.heads + pair * tiles;
        const int64_t w0 = attn_worker_of(x, total, workers), w1 = attn_worker_of(x + tiles - 1, total, workers);
        if (w0 == w1) return;                                           // one piece: written already
        slot0 = w0 + (int64_t)seq * a.heads + pair;
        n = (int)(w1 - w0) + 1;
    }
    const int g = t / per;
    for (int first = blockIdx.z * per; first < quads; first += gridDim.z * per) {
        const int quad = first + t % per, h = min(quad / (HD / 4), nh - 1), d = quad % (HD / 4) * 4;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        float m = -__builtin_inff(), l = bad ? __builtin_nanf("") : 0.f;
        const auto join = [&](f32v2 ml, f32x4 v) {
            const float top = fmaxf(m, ml[0]), safe = top == -__builtin_inff() ? 0.f : top;
            const float f = __builtin_amdgcn_exp2f(m - safe), e = __builtin_amdgcn_exp2f(ml[0] - safe);      // a NaN is dropped by the maximum and kept by these
            m = top;
            l = l * f + ml[1] * e;
            o = o * f + v * e;
        };
#pragma unroll 4
        for (int c = g; c < n; c += groups) join(*slot_ml<HD, H>(a, slot0 + c, h), *(const f32x4 *)(slot_o<HD, H>(a, slot0 + c, h) + d));
        for (int half = groups / 2; half; half /= 2) {
            if (g >= half && g < 2 * half) {
                sh_o[t] = o;
                sh_ml[t] = (f32v2){m, l};
            }
            __syncthreads();
            if (g < half) join(sh_ml[t + half * per], sh_o[t + half * per]);
        }
        if (g == 0 && quad < quads) {
            const int64_t at = seq * a.out_stride + (int64_t)(h0 + h) * HD + d;
#pragma unroll
            for (int i = 0; i < 4; i++) store1<ACT>(a.out, at + i, l == 0.f ? 0.f : bad ? l : o[i] / l);
            if (d == 0 && a.lse) a.lse[(int64_t)seq * a.n_heads + h0 + h] = bad ? l : lse_of(m, l);
        }
        __syncthreads();
    }
}

template <int ACT, int ST, int HD, int H> static hipError_t attn_launch(const AttnArgs &a, hipStream_t s) {
    const unsigned pairs = (unsigned)a.n_seqs * (unsigned)a.heads;
    if constexpr (ST == HIPVOC_T_F32) attn_rows_kernel<HD, H><<<a.workers ? (unsigned)a.workers : pairs, 256, 0, s>>>(a);
    else if (a.workers) attn_stream_kernel<ACT, ST, HD><<<(a.workers + 3) / 4, 256, 0, s>>>(a);
    else attn_whole_kernel<ACT, ST, HD><<<pairs, 256, 0, s>>>(a);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && a.workers) {
        const int quads = (a.group < H ? a.group : H) * (HD / 4);
        int per = 8;
        while (per < 256 && per < quads && pairs * (unsigned)((quads + per - 1) / per) > 1024) per *= 2;
        attn_join_kernel<ACT, HD, H><<<dim3(a.heads, a.n_seqs, (quads + per - 1) / per), 256, 0, s>>>(a, per);
        e = hipGetLastError();
    }
    return e;
}
template <int ACT, int ST, int HD> static hipError_t attn_go(const AttnArgs &a, hipStream_t s) {
    if constexpr (ST == HIPVOC_T_F32) {
        if (a.group == 1) return attn_launch<ACT, ST, HD, 1>(a, s);
        if (a.group == 2) return attn_launch<ACT, ST, HD, 2>(a, s);
        return attn_launch<ACT, ST, HD, 4>(a, s);
    } else {
        return attn_launch<ACT, ST, HD, 16>(a, s);
    }
}
template <int ACT> static hipError_t attn_act(const AttnArgs &a, hipStream_t s) {
    const bool wide = a.c.head_dim == 128;
    if (a.c.dtype == HIPVOC_T_INT8) return wide ? attn_go<ACT, HIPVOC_T_INT8, 128>(a, s) : attn_go<ACT, HIPVOC_T_INT8, 64>(a, s);
    if (a.c.dtype == HIPVOC_T_E4M3) return wide ? attn_go<ACT, HIPVOC_T_E4M3, 128>(a, s) : attn_go<ACT, HIPVOC_T_E4M3, 64>(a, s);
    return wide ? attn_go<ACT, ACT, 128>(a, s) : attn_go<ACT, ACT, 64>(a, s);
}
hipError_t launch_attention_decode(const AttnArgs &a, hipStream_t s) {
    if (a.dtype == HIPVOC_T_F32) return attn_act<HIPVOC_T_F32>(a, s);
    if (a.dtype == HIPVOC_T_F16) return attn_act<HIPVOC_T_F16>(a, s);
    return attn_act<HIPVOC_T_BF16>(a, s);
}

}  // namespace hipvoc
