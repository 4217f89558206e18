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

// A wave reads rows of HD values with HD / 8 lanes each, U rows per lane in flight, and keeps HT query heads in registers.
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
    const bool nan = sh_bad != 0;
    for (int i = threadIdx.x; i < nh * HD; i += 256) {
        const int h = i / HD, dd = i % HD, head = h0 + h;
        float top = sh_m[0][h];
        for (int w = 1; w < NW; w++) top = fmaxf(top, sh_m[w][h]);
        const float safe = top == -__builtin_inff() ? 0.f : top;
        float x = 0.f, sum = 0.f;
        for (int w = 0; w < NW; w++) {
            const float f = exp2f(sh_m[w][h] - safe);
            sum += sh_l[w][h] * f;
            x += sh_o[w][h][dd] * f;
        }
        if (nan) x = sum = top = __builtin_nanf("");
        if (a.n_chunks > 1) {
            part_o(a, seq, head, c)[dd] = x;
            if (dd == 0) { part_ml(a, seq, head, c)[0] = top; part_ml(a, seq, head, c)[1] = sum; }
        } else {
            store1<ACT>(a.out, seq * a.out_stride + (int64_t)head * HD + dd, sum == 0.f ? 0.f : x / sum);
            if (dd == 0 && a.lse) a.lse[(int64_t)seq * a.n_heads + head] = lse_of(top, sum);
        }
    }
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

template <int ACT, int ST, int HD, int HT> static void attn_go(const AttnArgs &a, hipStream_t s) {
    const int tiles = (a.group + HT - 1) / HT;
    attn_rows_kernel<ACT, ST, HD, HT><<<dim3(a.n_chunks, a.c.kv_heads * tiles, a.n_seqs), 256, 0, s>>>(a);
}
template <int ACT, int ST, int HD> static hipError_t attn_ht(const AttnArgs &a, hipStream_t s) {
    if (a.group == 1) attn_go<ACT, ST, HD, 1>(a, s);
    else if (a.group == 2) attn_go<ACT, ST, HD, 2>(a, s);
    else attn_go<ACT, ST, HD, 4>(a, s);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && a.n_chunks > 1) {
        attn_join_kernel<ACT, HD><<<dim3(a.n_heads, a.n_seqs), 256, 0, s>>>(a);
        e = hipGetLastError();
    }
    return e;
}
template <int ACT> static hipError_t attn_act(const AttnArgs &a, hipStream_t s) {
    const bool wide = a.c.head_dim == 128;
    if (a.c.dtype == HIPVOC_T_INT8) return wide ? attn_ht<ACT, HIPVOC_T_INT8, 128>(a, s) : attn_ht<ACT, HIPVOC_T_INT8, 64>(a, s);
    if (a.c.dtype == HIPVOC_T_E4M3) return wide ? attn_ht<ACT, HIPVOC_T_E4M3, 128>(a, s) : attn_ht<ACT, HIPVOC_T_E4M3, 64>(a, s);
    return wide ? attn_ht<ACT, ACT, 128>(a, s) : attn_ht<ACT, ACT, 64>(a, s);
}
hipError_t launch_attention_decode(const AttnArgs &a, hipStream_t s) {
    if (a.dtype == HIPVOC_T_F32) return attn_act<HIPVOC_T_F32>(a, s);
    if (a.dtype == HIPVOC_T_F16) return attn_act<HIPVOC_T_F16>(a, s);
    return attn_act<HIPVOC_T_BF16>(a, s);
}

}  // namespace hipvoc
