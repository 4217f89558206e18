// Products of a few rows with 4-bit weights and group scales (include/hipvoc_ops.h: hipvoc_q4_matvec).
//
// Mathematics: y[m][n] = sum_g s[n][g] * sum_{k in g} (c - 8) x[m][k], c = 0 .. 15 (with least values: s * c + min).  A code becomes a matrix
// operand without any conversion: its four bits are put into the top of the mantissa of 16, so the operand is 16 + c exactly (bf16 has 7, f16 10
// mantissa bits), and the group's sum is put right afterwards by 16 (24 without least values) times X[m][g] = sum of x, which a matrix instruction
// with ones gives in the same registers.  No product has a rounding; all sums are in 32 bits.  32-bit rows are cut into three bf16 parts of 8
// mantissa bits each (exactly x together), three matrix instructions for one.  8-bit rows: a code's two's complement of (c - 8) is moved to the
// top of a byte, 16 (c - 8), the group's sum is an exact integer, and 1/16 is part of the scale.
// Bound: memory, half a byte per weight read once (non-temporal); next to it the vector ALU, which turns 8 codes into operands with 8 instructions
// (5 for 8-bit rows), and the cache's line rate.  16 x 4096 x 65536 in f16 with groups of 64: 39 us, 4.0 TB/s; 1 x 1024 x 65536: 14 us.
// Layout: one wave has RT tiles of 16 weight rows and slabs of 128 columns: a lane reads 16 bytes of one row, and the four lanes of a row exchange their
// dwords (permlane swaps) so that a matrix instruction's 32 columns are one group.  x rows are the other side of the matrix instruction
// (up to 16 of them; rows behind the last repeat it and are not stored), so a lane's four results belong to ONE weight row: one scale per
// lane and group.  q4_kernel: the workgroup's waves share 16 RT rows and take every NW-th slab, x read by each for itself; q4_wide_kernel: for
// many weight rows, x through LDS.
#include <atomic>
#include <type_traits>

#include "ops_device.h"

namespace hipvoc {

__device__ __forceinline__ void swap32(unsigned &a, unsigned &b) {      // upper half of a <-> lower half of b
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}
__device__ __forceinline__ void swap16(unsigned &a, unsigned &b) {      // odd rows of 16 lanes of a <-> even rows of b
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}

// Eight codes of a dword as a matrix operand, in the order 0 4 1 5 2 6 3 7 (16-bit types; bytes: 0 2 4 6 1 3 5 7).  `e`: the bits of 16, twice, in a register (with two literals the mask and the or would be two instructions)
template <int XT> struct Codes {
    static __device__ __forceinline__ unsigned sixteen() {
        unsigned e = XT == HIPVOC_T_F16 ? 0x4c004c00u : 0x41804180u;
        asm("" : "+v"(e));
        return e;
    }
    static __device__ __forceinline__ u32x4 of(unsigned w, unsigned e) {
        if constexpr (XT == HIPVOC_T_F16) {
            constexpr unsigned M = 0x03c003c0u;
            return (u32x4){((w << 6) & M) | e, ((w << 2) & M) | e, ((w >> 2) & M) | e, ((w >> 6) & M) | e};
        } else {
            constexpr unsigned M = 0x00780078u;
            return (u32x4){((w << 3) & M) | e, ((w >> 1) & M) | e, ((w >> 5) & M) | e, ((w >> 9) & M) | e};
        }
    }
};
__device__ __forceinline__ u32x4 order16(u32x4 x) {                     // 0 1 2 3 4 5 6 7 -> 0 4 1 5 2 6 3 7
    return (u32x4){__builtin_amdgcn_perm(x[2], x[0], 0x05040100), __builtin_amdgcn_perm(x[2], x[0], 0x07060302),
                   __builtin_amdgcn_perm(x[3], x[1], 0x05040100), __builtin_amdgcn_perm(x[3], x[1], 0x07060302)};
}
__device__ __forceinline__ f32x4 mfma16(bool f16, u32x4 a, u32x4 b, f32x4 c) {
    if (f16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
}

// Eight values of x as matrix operands in the codes' order: P of them (three bf16 parts for 32-bit rows)
template <int XT> struct XRow {
    static constexpr int P = XT == HIPVOC_T_F32 ? 3 : 1;
    u32x4 raw[XT == HIPVOC_T_F32 ? 2 : 1];
    __device__ __forceinline__ void load(const void *x) {
        if constexpr (XT == HIPVOC_T_INT8) {
            const u32x2 v = *(const u32x2 *)x;
            raw[0] = (u32x4){v[0], v[1], 0u, 0u};
        } else {
            raw[0] = ((const u32x4 *)x)[0];
            if constexpr (XT == HIPVOC_T_F32) raw[1] = ((const u32x4 *)x)[1];
        }
    }
    __device__ __forceinline__ void parts(long *p) const {
        const u32x2 r = {__builtin_amdgcn_perm(raw[0][1], raw[0][0], 0x06040200), __builtin_amdgcn_perm(raw[0][1], raw[0][0], 0x07050301)};
        p[0] = __builtin_bit_cast(long, r);
    }
    __device__ __forceinline__ void parts(u32x4 *p) const {
        if constexpr (XT == HIPVOC_T_F32) {
            // x = a + b + c, each cut off (not rounded: nothing can overflow) after 8 significant bits, c not below bf16's least, 2^-133
            unsigned a[8], b[8], c[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const unsigned v = raw[i >> 2][i & 3];
                a[i] = v & 0xffff0000u;
                const float r = __uint_as_float(v) - __uint_as_float(a[i]);
                b[i] = __float_as_uint(r) & 0xffff0000u;
                c[i] = __float_as_uint(r - __uint_as_float(b[i]));
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                p[0][i] = __builtin_amdgcn_perm(a[i + 4], a[i], 0x07060302);
                p[1][i] = __builtin_amdgcn_perm(b[i + 4], b[i], 0x07060302);
                p[2][i] = __builtin_amdgcn_perm(c[i + 4], c[i], 0x07060302);
            }
        } else {
            p[0] = order16(raw[0]);
        }
    }
};

static constexpr int Q4_WAVES = 8;                    // waves of a workgroup
static constexpr int Q4_GROUPS = 128;                 // groups of a row whose scales are in LDS at a time
static constexpr int Q4_AHEAD = 2;                    // slabs of codes a wave of q4_kernel has asked for

// x of a slab of 128 columns, as a wave reads it for itself: 16 rows at `row` (this lane's), eight columns from 8 (lane / 16) of every 32
template <int XT> constexpr int x_bytes() { return XT == HIPVOC_T_F32 ? 4 : XT == HIPVOC_T_INT8 ? 1 : 2; }
template <int XT> struct XSlab {
    XRow<XT> x[4];
    __device__ __forceinline__ void load(const Q4Args &a, const char *row, int s, int lane) {
        constexpr int XB = x_bytes<XT>();
        const char *at = row + ((int64_t)s * 128 + 8 * (lane >> 4)) * XB;
        const int have = (a.n_in - s * 128) / 32;                                 // a group behind the last is not used: read the slab's first instead
#pragma unroll
        for (int c = 0; c < 4; c++) x[c].load(at + (have >= 4 || c < have ? c : 0) * 32 * XB);
    }
};
// Slab s of this lane's rows of the weights
template <int RT> __device__ __forceinline__ void q4_codes(const Q4Args &a, const uint8_t *const (&rows)[RT], u32x4 (&w)[RT], int s, int lane) {
    const int j = lane >> 4, at = s * 64 + (s * 128 + 32 * j < a.n_in ? 16 * j : 0);
#pragma unroll
    for (int t = 0; t < RT; t++) w[t] = __builtin_nontemporal_load((const u32x4 *)(rows[t] + at));
}

// sc: (scale, least value), two f16, of the slab's first group for this lane's row of tile 0; tile t is t * 16 rows of `stride` further on.
// sx: the scales of x rows 4j .. 4j + 3 for the slab's first group
// x(c, part) is the operand of 32 columns c.
template <int XT, int G, bool MINS, int RT, typename X>
__device__ __forceinline__ void q4_use(const Q4Args &a, u32x4 (&w)[RT], X &&x, int k0, const h16x2 *sc, int stride, const f32x4 *sx, f32x4 (&out)[RT]) {
    constexpr int NG = 128 / G, PER = 4 / NG;                                     // matrix instructions of 32 columns per group
    {
#pragma unroll
        for (int t = 0; t < RT; t++) {
            unsigned d[4] = {w[t][0], w[t][1], w[t][2], w[t][3]};
            swap32(d[0], d[2]);
            swap32(d[1], d[3]);
            swap16(d[0], d[1]);
            swap16(d[2], d[3]);
            w[t] = (u32x4){d[0], d[1], d[2], d[3]};
        }
    }
    const auto group = [&](int g) {
        if constexpr (XT == HIPVOC_T_INT8) {
            i32x4 acc[RT] = {}, sum = {};
#pragma unroll
            for (int p = 0; p < PER; p++) {
                const int c = g * PER + p;
                long xc[1];
                x(c, xc);
                if constexpr (MINS) sum = __builtin_amdgcn_mfma_i32_16x16x32_i8(xc[0], 0x0101010101010101L, sum, 0, 0, 0);
#pragma unroll
                for (int t = 0; t < RT; t++) {
                    const unsigned v = w[t][c] ^ 0x88888888u;
                    const u32x2 wc = {(v << 4) & 0xf0f0f0f0u, v & 0xf0f0f0f0u};
                    acc[t] = __builtin_amdgcn_mfma_i32_16x16x32_i8(xc[0], __builtin_bit_cast(long, wc), acc[t], 0, 0, 0);
                }
            }
            f32x4 xs = {1.f, 1.f, 1.f, 1.f};
            if (a.x_groups > 1) xs = sx[4 * g];
#pragma unroll
            for (int t = 0; t < RT; t++) {
                const h16x2 p = sc[t * 16 * stride + g];
                const float s = (float)p[0] * 0.0625f, off = MINS ? fmaf(128.f, s, (float)p[1]) : 0.f;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float v = s * (float)acc[t][r];
                    if constexpr (MINS) v = fmaf(off, (float)sum[r], v);
                    out[t][r] = fmaf(xs[r], v, out[t][r]);
                }
            }
        } else {
            constexpr bool F16 = XT == HIPVOC_T_F16;
            constexpr unsigned ONE = F16 ? 0x3c003c00u : 0x3f803f80u;
            const u32x4 ones = {ONE, ONE, ONE, ONE};
            const unsigned e16 = Codes<XT>::sixteen();
            // What the codes have too much comes off before the scale, so that the sum over groups never holds it; for 32-bit rows, whose result shows it,
            // after every 32 columns (1536 columns in groups of 128: error 8.6e-7 -> 4.9e-7 of the result, 3 % of the time).
            constexpr float EXTRA = MINS ? -16.f : -24.f;
            constexpr bool OFTEN = XT == HIPVOC_T_F32;
            f32x4 acc[RT] = {}, sum = {};
#pragma unroll
            for (int p = 0; p < PER; p++) {
                const int c = g * PER + p;
                u32x4 xc[XRow<XT>::P];
                x(c, xc);
                f32x4 here = OFTEN ? (f32x4){0.f, 0.f, 0.f, 0.f} : sum;
#pragma unroll
                for (int i = 0; i < XRow<XT>::P; i++) here = mfma16(F16, xc[i], ones, here);
#pragma unroll
                for (int t = 0; t < RT; t++) {
                    const u32x4 wc = Codes<XT>::of(w[t][c], e16);
                    f32x4 v = OFTEN ? (f32x4){0.f, 0.f, 0.f, 0.f} : acc[t];
#pragma unroll
                    for (int i = 0; i < XRow<XT>::P; i++) v = mfma16(F16, xc[i], wc, v);
                    if constexpr (OFTEN) {
#pragma unroll
                        for (int r = 0; r < 4; r++) acc[t][r] += fmaf(EXTRA, here[r], v[r]);
                    } else {
                        acc[t] = v;
                    }
                }
                if constexpr (OFTEN) sum += here;
                else sum = here;
            }
#pragma unroll
            for (int t = 0; t < RT; t++) {
                const h16x2 p = sc[t * 16 * stride + g];
                const float s = (float)p[0], off = (float)p[1];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    out[t][r] = fmaf(s, OFTEN ? acc[t][r] : fmaf(EXTRA, sum[r], acc[t][r]), out[t][r]);
                    if constexpr (MINS) out[t][r] = fmaf(off, sum[r], out[t][r]);
                }
            }
        }
    };
    if (k0 + 128 <= a.n_in) {                                                     // no branch between the groups of a whole slab
#pragma unroll
        for (int g = 0; g < NG; g++) group(g);
    } else {
#pragma unroll
        for (int g = 0; g < NG; g++)
            if (k0 + g * G < a.n_in) group(g);
    }
}

__host__ __device__ constexpr int q4_stride(int held) { return held + 1 + (held & 1); }      // odd: 16 rows in 16 banks
static size_t q4_lds(bool int8, int rows, int groups, int kw) {
    const int held = groups < Q4_GROUPS ? groups : Q4_GROUPS;
    const size_t scales = (int8 ? (size_t)held * 64 : 0) + (size_t)rows * q4_stride(held) * 4, sums = (size_t)kw * 16 * (rows + 1) * 4;
    return scales > sums ? scales : sums;
}

// Adds the waves' sums up and stores them
template <int XT, int RT>
__device__ __forceinline__ void q4_finish(const Q4Args &a, const f32x4 (&out)[RT], float *red, int kw, int part, int row0, int wg_rows, int n0, int m0) {
    const int lane = threadIdx.x & 63, r16 = lane & 15, j = lane >> 4;
    __syncthreads();                                                              // the scales' place is free
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) red[(part * 16 + 4 * j + r) * (wg_rows + 1) + row0 + 16 * t + r16] = out[t][r];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * wg_rows; i += blockDim.x) {
        const int ml = i / wg_rows, nl = i - ml * wg_rows, n = n0 + nl, m = m0 + ml;
        if (n >= a.n_out || m >= a.n_rows) continue;
        float v = 0.f;
        for (int w = 0; w < kw; w++) v += red[(w * 16 + ml) * (wg_rows + 1) + nl];
        if constexpr (XT == HIPVOC_T_INT8) {
            if (a.x_groups == 1) v *= a.x_scale[m];
        }
        const int64_t at = m * a.y_stride + n;
        if (a.y_dtype == HIPVOC_T_F32) store1<HIPVOC_T_F32>(a.y, at, v);
        else if (a.y_dtype == HIPVOC_T_F16) store1<HIPVOC_T_F16>(a.y, at, v);
        else store1<HIPVOC_T_BF16>(a.y, at, v);
    }
}

// The scales of the workgroup's rows (and of x's, for 8-bit rows) of up to Q4_GROUPS groups, into LDS: read once in whole lines by all waves (a lane's
// own reads would touch 16 lines for 32 bytes, in every slab)
template <int XT, bool MINS>
__device__ __forceinline__ void q4_stage_scales(const Q4Args &a, h16x2 *scales, float (*x_scales)[16], int n0, int m0, int wg_rows, int groups, int g0, int stride) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6, n = min(Q4_GROUPS, groups - g0);
    if (groups % 8 == 0 && groups <= Q4_GROUPS) {                                 // the rows are one piece of memory: eight groups a load
        const int per_row = groups / 8, count = min(wg_rows, a.n_out - n0) * per_row, step = blockDim.x;
        const u32x4 *s = (const u32x4 *)((const _Float16 *)a.scales + (int64_t)n0 * groups), *l = (const u32x4 *)((const _Float16 *)a.mins + (int64_t)n0 * groups);
        for (int first = threadIdx.x; first < count; first += 4 * step) {
            u32x4 v[4], m[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int at = min(first + i * step, count - 1);
                v[i] = s[at];
                m[i] = MINS ? l[at] : (u32x4){0u, 0u, 0u, 0u};
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int at = first + i * step, row = at / per_row, g = (at - row * per_row) * 8;
                if (at < count) {
                    unsigned *to = (unsigned *)scales + row * stride + g;
#pragma unroll
                    for (int e = 0; e < 8; e++) to[e] = __builtin_amdgcn_perm(m[i][e >> 1], v[i][e >> 1], e & 1 ? 0x07060302 : 0x05040100);
                }
            }
        }
    } else {
        for (int first = wave; first < wg_rows; first += 8 * nw) {                // eight rows' loads at a time: one latency
            _Float16 v[8][2], m[8][2];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int64_t at = (int64_t)min(n0 + first + i * nw, a.n_out - 1) * groups + g0;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int g = min(lane + 64 * h, n - 1);
                    v[i][h] = ((const _Float16 *)a.scales)[at + g];
                    m[i][h] = MINS ? ((const _Float16 *)a.mins)[at + g] : (_Float16)0.f;
                }
            }
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int h = 0; h < 2; h++)
                    if (first + i * nw < wg_rows && lane + 64 * h < n) scales[(first + i * nw) * stride + lane + 64 * h] = (h16x2){v[i][h], m[i][h]};
        }
    }
    if constexpr (XT == HIPVOC_T_INT8) {
        if (a.x_groups > 1)
            for (int row = wave; row < 16; row += nw) {
                const int64_t at = (int64_t)min(m0 + row, a.n_rows - 1) * groups + g0;
                for (int g = lane; g < n; g += 64) x_scales[g][row] = a.x_scale[at + g];
            }
    }
}

template <int XT, int G, bool MINS, int RT>
__global__ __launch_bounds__(64 * Q4_WAVES) void q4_kernel(Q4Args a, int kw) {
    constexpr bool INT8 = XT == HIPVOC_T_INT8;
    // LDS: the scales of x (8-bit rows), those of the weights, and at the end, in their place, the waves' sums (q4_lds)
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6, r16 = lane & 15, j = lane >> 4;
    const int part = wave % kw, row0 = wave / kw * 16 * RT, wg_rows = nw / kw * 16 * RT;
    const int n0 = blockIdx.x * wg_rows, m0 = blockIdx.y * 16, slabs = (a.n_in + 127) / 128, groups = a.n_in / G;
    const int held = min(groups, Q4_GROUPS), stride = q4_stride(held);
    float (*x_scales)[16] = (float (*)[16])lds;
    h16x2 *scales = (h16x2 *)(lds + (INT8 ? held * 64 : 0));
    float *red = (float *)lds;                                                    // [kw][16][wg_rows + 1]
    f32x4 out[RT] = {};
    XSlab<XT> cur, next;
    u32x4 w[Q4_AHEAD][RT];                                                        // codes of the next slabs, each asked for again once used
    const uint8_t *rows[RT];
#pragma unroll
    for (int t = 0; t < RT; t++) rows[t] = a.codes + (int64_t)min(n0 + row0 + 16 * t + r16, a.n_out - 1) * (a.n_in / 2);
    const char *x = (const char *)a.x + min(m0 + r16, a.n_rows - 1) * a.x_stride * x_bytes<XT>();
#pragma unroll
    for (int u = 0; u < Q4_AHEAD; u++)
        if (part + u * kw < slabs) q4_codes<RT>(a, rows, w[u], part + u * kw, lane);
    if (part < slabs) cur.load(a, x, part, lane);
    // a share of the scales' groups is a multiple of Q4_AHEAD * kw slabs, or the row's rest
    for (int g0 = 0; g0 < groups; g0 += Q4_GROUPS) {
        if (g0) __syncthreads();
        q4_stage_scales<XT, MINS>(a, scales, x_scales, n0, m0, wg_rows, groups, g0, stride);
        __syncthreads();
        const int last = min(slabs, (g0 + Q4_GROUPS) * G / 128);
        for (int i0 = g0 * G / 128 + part; i0 < last; i0 += Q4_AHEAD * kw) {
#pragma unroll
            for (int u = 0; u < Q4_AHEAD; u++) {
                const int i = i0 + u * kw;
                if (i >= last) break;
                if (i + kw < slabs) next.load(a, x, i + kw, lane);
                const int g = i * 128 / G - g0;
                q4_use<XT, G, MINS, RT>(a, w[u], [&](int c, auto *o) { cur.x[c].parts(o); }, i * 128, &scales[(row0 + r16) * stride + g], stride, INT8 ? (const f32x4 *)&x_scales[g][4 * j] : nullptr, out);
                if (i + Q4_AHEAD * kw < slabs) q4_codes<RT>(a, rows, w[u], i + Q4_AHEAD * kw, lane);
                cur = next;
            }
        }
    }
    q4_finish<XT, RT>(a, out, red, kw, part, row0, wg_rows, n0, m0);
}

// Many rows of weights: x goes through LDS.  A matrix operand's 16 rows of x are 16 lines for one load of 1 KB, and the cache serves a line in about
// four cycles whatever is taken of it: read by every wave for itself, x costs more than the weights (see q4_rt).  Here all waves read it along its rows, a block of BS slabs ahead, and lay it down in operand order.
// KW waves share a block's slabs, so the workgroup has 16 RT Q4_WAVES / KW rows.
template <int XT, int KW> constexpr int q4_block() { return XT == HIPVOC_T_F32 ? KW : 8; }         // slabs of a block
template <int XT, int G, bool MINS, int RT, int KW>
__global__ __launch_bounds__(64 * Q4_WAVES) void q4_wide_kernel(Q4Args a) {
    constexpr int kw = KW;
    constexpr bool INT8 = XT == HIPVOC_T_INT8;
    constexpr int BS = q4_block<XT, KW>(), MINE = BS / KW, P = XRow<XT>::P, UNITS = BS * 256 / (64 * Q4_WAVES);     // of a block's slabs a wave's own; what a thread lays down of x
    typedef typename std::conditional<INT8, long, u32x4>::type op_t;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), nw = Q4_WAVES, r16 = lane & 15, j = lane >> 4;
    const int part = wave % kw, row0 = wave / kw * 16 * RT, wg_rows = nw / kw * 16 * RT;
    const int n0 = blockIdx.x * wg_rows, m0 = blockIdx.y * 16, slabs = (a.n_in + 127) / 128, groups = a.n_in / G;
    const int held = min(groups, Q4_GROUPS), stride = q4_stride(held);
    op_t *xl = (op_t *)lds;                                                       // [BS slabs][4][P][64 lanes]
    float (*x_scales)[16] = (float (*)[16])(lds + BS * 256 * P * sizeof(op_t));
    h16x2 *scales = (h16x2 *)(lds + BS * 256 * P * sizeof(op_t) + (INT8 ? held * 64 : 0));
    float *red = (float *)lds;
    XRow<XT> ahead[UNITS];
    const auto fetch = [&](int s0) {
#pragma unroll
        for (int i = 0; i < UNITS; i++) {
            const int u = tid + i * 64 * Q4_WAVES, m = u / (BS * 16), k = s0 * 128 + u % (BS * 16) * 8;
            ahead[i].load((const char *)a.x + (min(m0 + m, a.n_rows - 1) * a.x_stride + (k < a.n_in ? k : 0)) * x_bytes<XT>());
        }
    };
    // row m of eight columns q stands at m ^ q % 16: sixteen threads that write one row's columns, and sixteen that read one column's rows, hit all
    // banks once
    const auto lay = [&]() {
#pragma unroll
        for (int i = 0; i < UNITS; i++) {
            const int u = tid + i * 64 * Q4_WAVES, m = u / (BS * 16), q = u % (BS * 16);       // q: eight columns; 16 of them a slab, 4 an operand
            op_t o[P];
            ahead[i].parts(o);
#pragma unroll
            for (int p = 0; p < P; p++) xl[((q >> 2) * P + p) * 64 + (q & 3) * 16 + (m ^ (q & 15))] = o[p];
        }
    };
    f32x4 out[RT] = {};
    u32x4 w[MINE][RT];                                                            // a block's codes, each asked for again for the next block once used
    const uint8_t *rows[RT];
#pragma unroll
    for (int t = 0; t < RT; t++) rows[t] = a.codes + (int64_t)min(n0 + row0 + 16 * t + r16, a.n_out - 1) * (a.n_in / 2);
    fetch(0);
#pragma unroll
    for (int i = 0; i < MINE; i++)
        if (part + i * kw < slabs) q4_codes<RT>(a, rows, w[i], part + i * kw, lane);
    for (int s0 = 0; s0 < slabs; s0 += BS) {
        const int g0 = s0 * 128 / G;
        if (s0) __syncthreads();                                                  // the last block is used up
        lay();
        if (g0 % Q4_GROUPS == 0) q4_stage_scales<XT, MINS>(a, scales, x_scales, n0, m0, wg_rows, groups, g0, stride);
        __syncthreads();
        if (s0 + BS < slabs) fetch(s0 + BS);
#pragma unroll
        for (int i = 0; i < MINE; i++) {
            const int s = s0 + part + i * kw;
            if (s >= slabs) break;
            const int g = (s * 128 / G) % Q4_GROUPS;
            const op_t *xs = xl + (s - s0) * 4 * P * 64 + 16 * j;
            q4_use<XT, G, MINS, RT>(a, w[i], [&](int c, op_t *o) {
#pragma unroll
                for (int p = 0; p < P; p++) o[p] = xs[(c * P + p) * 64 + (r16 ^ (4 * c + j))];
            }, s * 128, &scales[(row0 + r16) * stride + g], stride, INT8 ? (const f32x4 *)&x_scales[g][4 * j] : nullptr, out);
            if (s + BS < slabs) q4_codes<RT>(a, rows, w[i], s + BS, lane);
        }
    }
    q4_finish<XT, RT>(a, out, red, kw, part, row0, wg_rows, n0, m0);
}

template <int XT, int RT, int KW> static size_t q4_wide_lds(int groups) {
    const size_t x = (size_t)q4_block<XT, KW>() * 256 * (XT == HIPVOC_T_INT8 ? 8 : 16 * XRow<XT>::P);
    return x + q4_lds(XT == HIPVOC_T_INT8, 16 * RT * Q4_WAVES / KW, groups, KW);
}
static constexpr size_t Q4_LDS = 160 * 1024;
template <int XT, int G, bool MINS, int RT, int KW> static hipError_t q4_wide(const Q4Args &a, hipStream_t s) {
    constexpr int rows = 16 * RT * Q4_WAVES / KW;
    const size_t lds = q4_wide_lds<XT, RT, KW>(a.n_in / G);
    const auto kernel = q4_wide_kernel<XT, G, MINS, RT, KW>;
    if (lds > 65536) {                                                            // over the default of a launch: said once per device
        static std::atomic<bool> said[64];
        int dev = 0;
        hipError_t e = hipGetDevice(&dev);
        if (e == hipSuccess && (dev >= 64 || !said[dev].load())) {
            e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, Q4_LDS);
            if (e == hipSuccess && dev < 64) said[dev] = true;
        }
        if (e != hipSuccess) return e;
    }
    kernel<<<dim3((a.n_out + rows - 1) / rows, (a.n_rows + 15) / 16), 64 * Q4_WAVES, lds, s>>>(a);
    return hipGetLastError();
}
// Which kernel, by the number of weight rows.  A workgroup is slow by itself (it goes through all columns: scales, codes, sums), so one workgroup per
// CU with as few tiles as that takes is best while 256 of them can have all rows; beyond, x is better shared in LDS.  us, 2 rows of x in bf16, 4096
// columns, groups of 64 / 16 rows, 1024 columns / 2 rows in f32, 2048 columns (RT for q4_kernel, RT x KW for q4_wide_kernel):
//    rows    1                  2                  4                  2 x 4              4 x 2
//    5000    8.7 / 5.7 / 10.5   8.5 / 5.2 / 7.7    12 / 6.8 / 10      14 / 6.0 / 12      31 / 13 / 26
//   12288    13 / 8.2 / 15      15 / 8.8 / 14      12 / 6.9 / 10      14 / 6.2 / 12      32 / 13 / 27
//   24576    23 / 15 / 28       22 / 13 / 21       23 / 12 / 19       21 / 8.3 / 17      33 / 14 / 27
//   65536    56 / 36 / 72       56 / 32 / 52       46 / 24 / 38       40 / 15 / 32       36 / 15 / 28
template <int XT, int G, bool MINS> static hipError_t q4_rt(const Q4Args &a, hipStream_t s) {
    const int slabs = (a.n_in + 127) / 128, kw = slabs < Q4_WAVES ? slabs : Q4_WAVES;
    const auto direct = [&](int rt, auto kernel) {
        kernel<<<dim3((a.n_out + 16 * rt - 1) / (16 * rt), (a.n_rows + 15) / 16), 64 * kw, q4_lds(XT == HIPVOC_T_INT8, 16 * rt, a.n_in / G, kw), s>>>(a, kw);
        return hipGetLastError();
    };
    const int64_t rows = (int64_t)a.n_out * ((a.n_rows + 15) / 16);              // the weights are gone through once for every 16 rows of x
    // few columns leave a workgroup few waves, which are slow to fetch many rows' scales (11954 x 128: 4.9 us, with 4 tiles 9.8; x 896: 8.9, 7.9)
    if (rows <= 4096 || (slabs <= 4 && rows <= 16384)) return direct(1, q4_kernel<XT, G, MINS, 1>);
    if (rows <= 8192) return direct(2, q4_kernel<XT, G, MINS, 2>);
    if (rows <= 16384) return direct(4, q4_kernel<XT, G, MINS, 4>);
    // 16-bit rows of over 126 groups: the scales of 256 rows and x do not fit the LDS beside each other
    if (rows >= 65536 && q4_wide_lds<XT, 4, 2>(a.n_in / G) <= Q4_LDS) return q4_wide<XT, G, MINS, 4, 2>(a, s);
    return q4_wide<XT, G, MINS, 2, 4>(a, s);
}
template <int XT, int G> static hipError_t q4_mins(const Q4Args &a, hipStream_t s) { return a.mins ? q4_rt<XT, G, true>(a, s) : q4_rt<XT, G, false>(a, s); }
template <int XT> static hipError_t q4_group(const Q4Args &a, hipStream_t s) {
    if (a.group == 32) return q4_mins<XT, 32>(a, s);
    if (a.group == 64) return q4_mins<XT, 64>(a, s);
    return q4_mins<XT, 128>(a, s);
}
hipError_t launch_q4_matvec(const Q4Args &a, hipStream_t s) {
    if (a.x_dtype == HIPVOC_T_INT8) return q4_group<HIPVOC_T_INT8>(a, s);
    if (a.x_dtype == HIPVOC_T_F32) return q4_group<HIPVOC_T_F32>(a, s);
    if (a.x_dtype == HIPVOC_T_F16) return q4_group<HIPVOC_T_F16>(a, s);
    return q4_group<HIPVOC_T_BF16>(a, s);
}

}  // namespace hipvoc
