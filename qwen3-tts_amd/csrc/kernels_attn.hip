// Attention of one new token per sequence over the paged cache (include/hipvoc_ops.h: hipvoc_attention).
//
// Mathematics: one pass over the keys with a running maximum m and sum l per query head (softmax in powers of two, s = q.k * scale *
// log2(e)):  m' = max(m, s), l' = l 2^(m-m') + 2^(s-m'), o' = o 2^(m-m') + 2^(s-m') v.  States (m, l, o) of disjoint key sets join by
// the same rule, so a sequence is cut into chunks, one workgroup each; the chunks of a sequence are joined by a second small kernel
// (no atomics: the order of every sum is fixed).
// Bound: memory.  Every key and value row is read once for all query heads of its key head; the split exists because n_seqs * kv_heads
// workgroups do not fill 256 CUs.
#include "ops_device.h"

namespace hipvoc {

// where chunk c of (seq, head) leaves its state
__device__ __forceinline__ float *part_o(const AttnArgs &a, int seq, int head, int c) {
    return a.part + (((int64_t)seq * a.n_heads + head) * a.n_chunks + c) * a.c.head_dim;
}
__device__ __forceinline__ float *part_ml(const AttnArgs &a, int seq, int head, int c) {
    return a.part + (int64_t)a.n_seqs * a.n_heads * a.n_chunks * a.c.head_dim + (((int64_t)seq * a.n_heads + head) * a.n_chunks + c) * 2;
}
__device__ __forceinline__ float lse_of(float m, float l) { return (m + log2f(l)) * 0.69314718055994530942f; }

// Joins the states of a workgroup's NW waves and writes the chunk's state, or the result where there is one chunk.  ml(w, h) = (m, l) of
// wave w for the workgroup's head h, o(w, h, d) its sums.
template <int ACT, int HD, int NW, typename ML, typename O>
__device__ __forceinline__ void attn_finish(const AttnArgs &a, int seq, int c, int h0, int nh, bool nan, ML &&ml, O &&o) {
    for (int i = threadIdx.x; i < nh * HD; i += 64 * NW) {
        const int h = i / HD, d = i % HD, head = h0 + h;
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
        if (a.n_chunks > 1) {
            part_o(a, seq, head, c)[d] = x;
            if (d == 0) *(f32v2 *)part_ml(a, seq, head, c) = (f32v2){top, sum};
        } else {
            store1<ACT>(a.out, seq * a.out_stride + (int64_t)head * HD + d, sum == 0.f ? 0.f : x / sum);
            if (d == 0 && a.lse) a.lse[(int64_t)seq * a.n_heads + head] = lse_of(top, sum);
        }
    }
}

// 32-bit activations: a wave reads rows of HD values with HD / 8 lanes each, U rows per lane in flight, and keeps HT query heads in registers.
template <int ACT, int ST, int HD, int HT>
__global__ __launch_bounds__(256) void attn_rows_kernel(AttnArgs a) {
    constexpr int LPR = HD / 8, KPS = 64 / LPR, U = 4, TILE = U * KPS, NW = 4;
    typedef typename Store<ACT>::type act_t;
    typedef typename Store<ST>::type st_t;
    __shared__ float sh_o[NW][HT][HD], sh_m[NW][HT], sh_l[NW][HT];
    __shared__ int sh_bad;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, seq = blockIdx.z, c = blockIdx.x;
    const int tiles = (a.group + HT - 1) / HT, kvh = blockIdx.y / tiles, h0 = kvh * a.group + (blockIdx.y % tiles) * HT;
    const int nh = min(HT, (kvh + 1) * a.group - h0), d = (lane % LPR) * 8, kl = lane / LPR;
    const AttnSpan sp = attn_span(a.lens[seq], a.max_len, a.window, a.chunk, c);
    if (c >= sp.active && !(c == 0 && a.n_chunks == 1)) return;
    if (threadIdx.x == 0) sh_bad = sp.bad;
    if (sp.bad && threadIdx.x == 0) raise(a.err, OPS_ERR_LENGTH);
    float q[HT][8], o[HT][8], m[HT], l[HT];
#pragma unroll
    for (int h = 0; h < HT; h++) {
        m[h] = -__builtin_inff();
        l[h] = 0.f;
        load8<ACT>((const act_t *)a.q + seq * a.q_stride + (int64_t)min(h0 + h, h0 + nh - 1) * HD + d, q[h]);
#pragma unroll
        for (int i = 0; i < 8; i++) o[h][i] = 0.f;
    }
    __syncthreads();
    const int32_t *table = a.table + seq * a.table_stride;
    bool bad = false;
    for (int base = sp.from + wave * TILE; base < sp.to; base += NW * TILE) {
        float k[U][8], v[U][8], ks[U], vs[U], s[HT][U];
        bool in[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int key = base + u * KPS + kl, kc = min(max(key, sp.lo), sp.to - 1);       // what is masked is read from a row that is not
            in[u] = key >= sp.lo && key < sp.to;
            int page = table[kc >> a.page_shift];
            if (!page_ok(page, a.c.n_pages)) { bad = true; page = 0; }
            const int at = kc & (a.c.page - 1);
            const int64_t row = page * a.c.page_stride + ((int64_t)kvh * a.c.page + at) * HD + d;
            load8<ST>((const st_t *)a.c.k + row, k[u]);
            load8<ST>((const st_t *)a.c.v + row, v[u]);
            ks[u] = vs[u] = 1.f;
            if constexpr (ST != ACT) {
                const int64_t sc = ((int64_t)page * a.c.kv_heads + kvh) * a.c.page + at;
                ks[u] = a.c.k_scale[sc];
                vs[u] = a.c.v_scale[sc];
            }
        }
#pragma unroll
        for (int h = 0; h < HT; h++) {
            float top = m[h];
#pragma unroll
            for (int u = 0; u < U; u++) {
                float x = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i++) x = fmaf(q[h][i], k[u][i], x);
#pragma unroll
                for (int off = 1; off < LPR; off *= 2) x += __shfl_xor(x, off);
                if constexpr (ST != ACT) x *= ks[u];
                s[h][u] = in[u] ? x * a.scale_log2 : -__builtin_inff();
                top = fmaxf(top, s[h][u]);
            }
            const float safe = top == -__builtin_inff() ? 0.f : top, old = exp2f(m[h] - safe);
            m[h] = top;
            l[h] *= old;
#pragma unroll
            for (int i = 0; i < 8; i++) o[h][i] *= old;
#pragma unroll
            for (int u = 0; u < U; u++) {
                float p = exp2f(s[h][u] - safe);
                l[h] += p;
                if constexpr (ST != ACT) p = in[u] ? p * vs[u] : 0.f;
#pragma unroll
                for (int i = 0; i < 8; i++) o[h][i] = fmaf(p, v[u][i], o[h][i]);
            }
        }
    }
    if (bad) {
        raise(a.err, OPS_ERR_PAGE);
        sh_bad = 1;
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
    attn_finish<ACT, HD, NW>(a, seq, c, h0, nh, sh_bad != 0, [&](int w, int h) { return f32v2{sh_m[w][h], sh_l[w][h]}; }, [&](int w, int h, int d) { return sh_o[w][h][d]; });
}

// ---------------------------------------------------------------------------------------------------------------------
// 16-bit activations, on the matrix cores.  A wave has tiles of 32 keys for up to 16 query heads:
//   S^T = K Q^T   (rows = keys, columns = heads): a lane of (m = lane % 16, j = lane / 16) reads key rows as they lie, 16 bytes at a time.
//                 Row m of half t is key 8 (m / 4) + 4 t + m % 4, so a lane's eight results are the scores of ONE head for the keys 8j .. 8j+7,
//   O^T = V^T P^T (rows = values' columns, columns = heads): and these, rounded, are at once the right operand.  The left one needs a column
//                 of V for eight keys: the lane reads HD/16 neighbouring columns of its eight keys' rows (whole rows across 16 lanes) and
//                 turns them with one byte permutation per two values; row m of product i is column m HD/16 + i.
// So neither K, V nor P passes through LDS.  Scores, m, l and O are in 32 bits; P is rounded to 16 bits for the product with V (V's own type,
// bf16 for 8-bit codes, which bf16 and f16 hold exactly, and whose scales are in the scores and in P).
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
// maximum over the four lanes of a head (lane % 16)
__device__ __forceinline__ float max_of_head(float v) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

template <int ACT, int ST, int HD>
__global__ __launch_bounds__(256) void attn_tile_kernel(AttnArgs a) {
    constexpr bool CODED = ST != ACT, QF16 = ACT == HIPVOC_T_F16, PF16 = QF16 && !CODED;
    constexpr int NW = 4, NC = HD / 32, NV = HD / 16;                    // products of S per 16 keys, and of O
    constexpr int KW = CODED ? HD / 64 : NC, VW = CODED ? HD / 64 : HD / 32;      // 16-byte words of a key row, dwords of a value row that a lane reads
    typedef typename Store<ACT>::type act_t;
    typedef typename Store<ST>::type st_t;
    __shared__ __attribute__((aligned(16))) float sh_o[NW][16][HD + 4];
    __shared__ float sh_m[NW][16], sh_l[NW][16];
    __shared__ int sh_bad;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, seq = blockIdx.z, c = blockIdx.x, m16 = lane & 15, j = lane >> 4;
    const int tiles = (a.group + 15) / 16, kvh = blockIdx.y / tiles, h0 = kvh * a.group + (blockIdx.y % tiles) * 16;
    const int nh = min(16, (kvh + 1) * a.group - h0);
    const AttnSpan sp = attn_span(a.lens[seq], a.max_len, a.window, a.chunk, c);
    if (c >= sp.active && !(c == 0 && a.n_chunks == 1)) return;
    if (threadIdx.x == 0) sh_bad = sp.bad;
    if (sp.bad && threadIdx.x == 0) raise(a.err, OPS_ERR_LENGTH);
    u32x4 q[NC];
    {
        const act_t *row = (const act_t *)a.q + seq * a.q_stride + (int64_t)(h0 + min(m16, nh - 1)) * HD;
#pragma unroll
        for (int i = 0; i < NC; i++) q[i] = *(const u32x4 *)(row + (CODED ? (i >> 1) * 64 + 16 * j + 8 * (i & 1) : 32 * i + 8 * j));
    }
    __syncthreads();
    float m = -__builtin_inff(), l = 0.f;
    f32x4 o[NV] = {};
    const int32_t *table = a.table + seq * a.table_stride;
    const int64_t head_at = (int64_t)kvh * a.c.page * HD;
    bool bad = false;
    for (int base = sp.from + wave * 32; base < sp.to; base += NW * 32) {
        const bool full = base >= sp.lo && base + 32 <= sp.to;
        // the groups of eight keys that this lane reads keys / values of: if all of one is masked, another
        int gk = base + 8 * (m16 >> 2), gv = base + 8 * j;
        if (!full) {
            const int first = sp.lo & ~7, last = (sp.to - 1) & ~7;
            gk = min(max(gk, first), last);
            gv = min(max(gv, first), last);
        }
        int pk = table[gk >> a.page_shift], pv = table[gv >> a.page_shift];
        if (!page_ok(pk, a.c.n_pages) || !page_ok(pv, a.c.n_pages)) { bad = true; pk = pv = 0; }
        const st_t *kp = (const st_t *)a.c.k + pk * a.c.page_stride + head_at, *vp = (const st_t *)a.c.v + pv * a.c.page_stride + head_at;
        u32x4 k[2][KW];
        unsigned v[8][VW];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            int key = gk + 4 * t + (m16 & 3);
            if (!full) key = min(max(key, sp.lo), sp.to - 1);
            const st_t *row = kp + (int64_t)(key & (a.c.page - 1)) * HD + (CODED ? 16 : 8) * j;
#pragma unroll
            for (int i = 0; i < KW; i++) k[t][i] = *(const u32x4 *)(row + (CODED ? 64 : 32) * i);
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            int key = gv + e;
            if (!full) key = min(max(key, sp.lo), sp.to - 1);
            const st_t *row = vp + (int64_t)(key & (a.c.page - 1)) * HD + m16 * NV;
            if constexpr (VW == 4) *(u32x4 *)v[e] = *(const u32x4 *)row;
            else if constexpr (VW == 2) *(u32x2 *)v[e] = *(const u32x2 *)row;
            else v[e][0] = *(const unsigned *)row;
        }
        f32x4 ks[2], vs[2];
        if constexpr (CODED) {
            const int64_t at = ((int64_t)pv * a.c.kv_heads + kvh) * a.c.page + (gv & (a.c.page - 1));
#pragma unroll
            for (int t = 0; t < 2; t++) {
                ks[t] = *(const f32x4 *)(a.c.k_scale + at + 4 * t);
                vs[t] = *(const f32x4 *)(a.c.v_scale + at + 4 * t);
            }
        }
        // scores of the keys base + 8j + 4t + r for head m16
        float s[8], top = m;
#pragma unroll
        for (int t = 0; t < 2; t++) {
            f32x4 acc = {};
            if constexpr (CODED) {
#pragma unroll
                for (int i = 0; i < KW; i++) {
                    const u32x2 a0 = widen4<ST, QF16>(k[t][i][0]), a1 = widen4<ST, QF16>(k[t][i][1]), a2 = widen4<ST, QF16>(k[t][i][2]), a3 = widen4<ST, QF16>(k[t][i][3]);
                    acc = mfma32<QF16>((u32x4){a0[0], a0[1], a1[0], a1[1]}, q[2 * i], acc);
                    acc = mfma32<QF16>((u32x4){a2[0], a2[1], a3[0], a3[1]}, q[2 * i + 1], acc);
                }
                acc *= ks[t];
            } else {
#pragma unroll
                for (int i = 0; i < NC; i++) acc = mfma32<QF16>(k[t][i], q[i], acc);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int key = base + 8 * j + 4 * t + r;
                s[4 * t + r] = full || (key >= sp.lo && key < sp.to) ? acc[r] * a.scale_log2 : -__builtin_inff();
                top = fmaxf(top, s[4 * t + r]);
            }
        }
        top = max_of_head(top);
        if (__any(top > m)) {                                            // else nothing to scale down
            const float f = __builtin_amdgcn_exp2f(m - (top == -__builtin_inff() ? 0.f : top));
            m = top;
            l *= f;
#pragma unroll
            for (int i = 0; i < NV; i++) o[i] *= f;
        }
        const float safe = m == -__builtin_inff() ? 0.f : m;
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            p[e] = __builtin_amdgcn_exp2f(s[e] - safe);
            l += p[e];
            if constexpr (CODED) {
                const int key = base + 8 * j + e;
                p[e] = full || (key >= sp.lo && key < sp.to) ? p[e] * vs[e >> 2][e & 3] : 0.f;
            }
        }
        u32x4 pp;
#pragma unroll
        for (int e = 0; e < 4; e++) pp[e] = PF16 ? pack_f16(p[2 * e], p[2 * e + 1]) : pack_bf16(p[2 * e], p[2 * e + 1]);
        unsigned w[8][HD / 32];                                          // the value rows in 16 bits
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if constexpr (CODED) {
#pragma unroll
                for (int i = 0; i < VW; i++) {
                    const u32x2 x = widen4<ST, false>(v[e][i]);
                    w[e][2 * i] = x[0];
                    w[e][2 * i + 1] = x[1];
                }
            } else {
#pragma unroll
                for (int i = 0; i < VW; i++) w[e][i] = v[e][i];
            }
        }
#pragma unroll
        for (int i = 0; i < NV; i++) {
            u32x4 col;
#pragma unroll
            for (int e = 0; e < 4; e++) col[e] = __builtin_amdgcn_perm(w[2 * e + 1][i >> 1], w[2 * e][i >> 1], i & 1 ? 0x07060302 : 0x05040100);
            o[i] = mfma32<PF16>(col, pp, o[i]);
        }
    }
    if (bad) {
        raise(a.err, OPS_ERR_PAGE);
        sh_bad = 1;
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (m16 < nh) {
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int i = 0; i < NV; i += 4) *(f32x4 *)&sh_o[wave][m16][(4 * j + r) * NV + i] = (f32x4){o[i][r], o[i + 1][r], o[i + 2][r], o[i + 3][r]};
        if (j == 0) { sh_m[wave][m16] = m; sh_l[wave][m16] = l; }
    }
    __syncthreads();
    attn_finish<ACT, HD, NW>(a, seq, c, h0, nh, sh_bad != 0, [&](int w, int h) { return f32v2{sh_m[w][h], sh_l[w][h]}; }, [&](int w, int h, int d) { return sh_o[w][h][d]; });
}

// Joins a sequence's chunks: one workgroup per (head, sequence), HD / 4 threads across a row of o and 256 / (HD / 4) chunks at a time.
template <int ACT, int HD>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
    constexpr int W = HD / 4, G = 256 / W;
    __shared__ float sh[G][HD + 4], sh_m[4], sh_l[G];
    const int head = blockIdx.x, seq = blockIdx.y, t = threadIdx.x, d = (t % W) * 4, g = t / W;
    const AttnSpan sp = attn_span(a.lens[seq], a.max_len, a.window, a.chunk, 0);
    float top = -__builtin_inff();
    for (int c = t; c < sp.active; c += 256) {
        top = fmaxf(top, part_ml(a, seq, head, c)[0]);               // a NaN is dropped here and comes through the factor below
    }
#pragma unroll
    for (int off = 1; off < 64; off *= 2) top = fmaxf(top, __shfl_xor(top, off));
    if ((t & 63) == 0) sh_m[t >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; w++) top = fmaxf(top, sh_m[w]);
    const float safe = top == -__builtin_inff() ? 0.f : top;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
    for (int c = g; c < sp.active; c += G) {
        const float *ml = part_ml(a, seq, head, c), f = exp2f(ml[0] - safe);
        l += ml[1] * f;
        o += *(const f32x4 *)(part_o(a, seq, head, c) + d) * f;
    }
    *(f32x4 *)&sh[g][d] = o;
    if (d == 0) sh_l[g] = l;
    __syncthreads();
    if (t < HD) {
        float x = 0.f, sum = 0.f;
#pragma unroll
        for (int i = 0; i < G; i++) { x += sh[i][t]; sum += sh_l[i]; }
        store1<ACT>(a.out, seq * a.out_stride + (int64_t)head * HD + t, sum == 0.f ? 0.f : x / sum);
        if (t == 0 && a.lse) a.lse[(int64_t)seq * a.n_heads + head] = lse_of(top, sum);
    }
}

template <int ST, int HD, int HT> static void attn_rows(const AttnArgs &a, hipStream_t s) {
    const int tiles = (a.group + HT - 1) / HT;
    attn_rows_kernel<HIPVOC_T_F32, ST, HD, HT><<<dim3(a.n_chunks, a.c.kv_heads * tiles, a.n_seqs), 256, 0, s>>>(a);
}
template <int ACT, int ST, int HD> static hipError_t attn_go(const AttnArgs &a, hipStream_t s) {
    if constexpr (ACT == HIPVOC_T_F32) {
        if (a.group == 1) attn_rows<ST, HD, 1>(a, s);
        else if (a.group == 2) attn_rows<ST, HD, 2>(a, s);
        else attn_rows<ST, HD, 4>(a, s);
    } else {
        attn_tile_kernel<ACT, ST, HD><<<dim3(a.n_chunks, a.c.kv_heads * ((a.group + 15) / 16), a.n_seqs), 256, 0, s>>>(a);
    }
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && a.n_chunks > 1) {
        attn_join_kernel<ACT, HD><<<dim3(a.n_heads, a.n_seqs), 256, 0, s>>>(a);
        e = hipGetLastError();
    }
    return e;
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
