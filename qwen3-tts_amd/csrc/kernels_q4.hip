// Products of a few rows with 4-bit weights and group scales (include/hipvoc_ops.h: hipvoc_q4_matvec).
//
// Mathematics: y[m][n] = sum_g s[n][g] * sum_{k in g} (c - 8) x[m][k], c = 0 .. 15 (with least values: s * c + min).  A code becomes a matrix
// operand without any conversion: its four bits are put into the top of the mantissa of 16, so the operand is 16 + c exactly (bf16 has 7, f16 10
// mantissa bits), and the group's sum is put right afterwards by (min - 16 s) or -24 s times X[m][g] = sum of x, which a matrix instruction with
// ones gives in the same registers.  No product has a rounding; all sums are in 32 bits.  32-bit rows are cut into three bf16 parts of 8
// mantissa bits each (exactly x together), three matrix instructions for one.  8-bit rows: a code's two's complement of (c - 8) is moved to the
// top of a byte, 16 (c - 8), the group's sum is an exact integer, and 1/16 is part of the scale.
// Bound: memory, half a byte per weight read once; next to it the vector ALU, which turns 8 codes into operands with 8 instructions (4 for
// 8-bit rows).
// Layout: one wave has RT tiles of 16 weight rows, the workgroup's waves share the rows and take every NW-th slab of 128 columns: a lane
// reads 16 bytes of one row.  x rows are the other side of the matrix instruction (up to 16 of them; rows behind the last repeat it and are
// not stored), so a lane's four results belong to ONE weight row: one scale per lane and group.  With groups shorter than a slab the four lanes of
// a row exchange their dwords (two permlane swaps) so that a matrix instruction's 32 columns are one group.
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

// Eight codes of a dword as a matrix operand, in the order 0 4 1 5 2 6 3 7 (16-bit types) or 0 2 4 6 1 3 5 7 (bytes)
template <int XT> struct Codes {
    static __device__ __forceinline__ u32x4 of(unsigned w) {
        if constexpr (XT == HIPVOC_T_F16) {
            constexpr unsigned M = 0x03c003c0u, E = 0x4c004c00u;
            return (u32x4){((w << 6) & M) | E, ((w << 2) & M) | E, ((w >> 2) & M) | E, ((w >> 6) & M) | E};
        } else {
            constexpr unsigned M = 0x00780078u, E = 0x41804180u;
            return (u32x4){((w << 3) & M) | E, ((w >> 1) & M) | E, ((w >> 5) & M) | E, ((w >> 9) & M) | E};
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
    __device__ __forceinline__ void load(const void *x, int64_t at) {
        if constexpr (XT == HIPVOC_T_F32) {
            raw[0] = *(const u32x4 *)((const float *)x + at);
            raw[1] = *(const u32x4 *)((const float *)x + at + 4);
        } else if constexpr (XT == HIPVOC_T_INT8) {
            const u32x2 v = *(const u32x2 *)((const uint8_t *)x + at);
            raw[0] = (u32x4){v[0], v[1], 0u, 0u};
        } else {
            raw[0] = *(const u32x4 *)((const uint16_t *)x + at);
        }
    }
    __device__ __forceinline__ void parts(u32x4 *p) const {
        if constexpr (XT == HIPVOC_T_F32) {
            // x = a + b + c, each cut off (not rounded: nothing can overflow) after 8 significant bits
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
    __device__ __forceinline__ long bytes() const {
        const u32x2 r = {__builtin_amdgcn_perm(raw[0][1], raw[0][0], 0x06040200), __builtin_amdgcn_perm(raw[0][1], raw[0][0], 0x07050301)};
        return __builtin_bit_cast(long, r);
    }
};

static constexpr int Q4_WAVES = 8;

// What a wave reads of one slab of 128 columns
template <int XT, int G, bool MINS, int RT> struct Slab {
    static constexpr int NG = 128 / G;
    u32x4 w[RT];
    XRow<XT> x[4];
    float s[RT][NG], least[RT][MINS ? NG : 1], sx[XT == HIPVOC_T_INT8 ? 4 : 1][NG];
};

template <int XT, int G, bool MINS, int RT>
__device__ __forceinline__ void q4_load(const Q4Args &a, Slab<XT, G, MINS, RT> &b, int k0, int n0, int m0, int lane) {
    constexpr int NG = 128 / G;
    const int r16 = lane & 15, j = lane >> 4, groups = a.n_in / G, g0 = k0 / G;
    const bool whole = k0 + 128 <= a.n_in;
    const int xm = min(m0 + r16, a.n_rows - 1);
#pragma unroll
    for (int t = 0; t < RT; t++) {
        const int n = min(n0 + 16 * t + r16, a.n_out - 1);
        const int64_t row = (int64_t)n * (a.n_in / 2);
        const int at = k0 + 32 * j < a.n_in ? k0 / 2 + 16 * j : k0 / 2;           // a column behind the last belongs to no group that is used
        b.w[t] = *(const u32x4 *)(a.codes + row + at);
        const int64_t sc = (int64_t)n * groups + g0;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            const int64_t i = sc + (whole || g0 + g < groups ? g : 0);
            b.s[t][g] = (float)((const _Float16 *)a.scales)[i];
            if constexpr (MINS) b.least[t][g] = (float)((const _Float16 *)a.mins)[i];
        }
    }
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const int k = G == 128 ? k0 + 32 * j + 8 * c : k0 + (whole || k0 + 32 * c < a.n_in ? 32 * c : 0) + 8 * j;
        b.x[c].load(a.x, xm * a.x_stride + k);
    }
    if constexpr (XT == HIPVOC_T_INT8) {
        if (a.x_groups > 1) {
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int64_t row = (int64_t)min(m0 + 4 * j + r, a.n_rows - 1) * groups + g0;
#pragma unroll
                for (int g = 0; g < NG; g++) b.sx[r][g] = a.x_scale[row + (whole || g0 + g < groups ? g : 0)];
            }
        } else {
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int g = 0; g < NG; g++) b.sx[r][g] = 1.f;                    // one scale per row: at the end
        }
    }
}

template <int XT, int G, bool MINS, int RT>
__device__ __forceinline__ void q4_use(const Q4Args &a, Slab<XT, G, MINS, RT> &b, int k0, f32x4 (&out)[RT]) {
    constexpr int NG = 128 / G, PER = 4 / NG;                                     // matrix instructions of 32 columns per group
    const bool whole = k0 + 128 <= a.n_in;
    if constexpr (G < 128) {
#pragma unroll
        for (int t = 0; t < RT; t++) {
            unsigned d[4] = {b.w[t][0], b.w[t][1], b.w[t][2], b.w[t][3]};
            swap32(d[0], d[2]);
            swap32(d[1], d[3]);
            swap16(d[0], d[1]);
            swap16(d[2], d[3]);
            b.w[t] = (u32x4){d[0], d[1], d[2], d[3]};
        }
    }
#pragma unroll
    for (int g = 0; g < NG; g++) {
        if (!whole && k0 + g * G >= a.n_in) break;
        if constexpr (XT == HIPVOC_T_INT8) {
            i32x4 acc[RT] = {}, sum = {};
#pragma unroll
            for (int p = 0; p < PER; p++) {
                const int c = g * PER + p;
                const long x = b.x[c].bytes();
                if constexpr (MINS) sum = __builtin_amdgcn_mfma_i32_16x16x32_i8(x, 0x0101010101010101L, sum, 0, 0, 0);
#pragma unroll
                for (int t = 0; t < RT; t++) {
                    const unsigned w = b.w[t][c] ^ 0x88888888u;
                    const u32x2 v = {(w << 4) & 0xf0f0f0f0u, w & 0xf0f0f0f0u};
                    acc[t] = __builtin_amdgcn_mfma_i32_16x16x32_i8(x, __builtin_bit_cast(long, v), acc[t], 0, 0, 0);
                }
            }
#pragma unroll
            for (int t = 0; t < RT; t++) {
                const float s = b.s[t][g] * 0.0625f;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float v = s * (float)acc[t][r];
                    if constexpr (MINS) v = fmaf(fmaf(8.f, b.s[t][g], b.least[t][g]), (float)sum[r], v);
                    out[t][r] = fmaf(b.sx[r][g], v, out[t][r]);
                }
            }
        } else {
            constexpr bool F16 = XT == HIPVOC_T_F16;
            constexpr unsigned ONE = F16 ? 0x3c003c00u : 0x3f803f80u;
            const u32x4 ones = {ONE, ONE, ONE, ONE};
            f32x4 acc[RT] = {}, sum = {};
#pragma unroll
            for (int p = 0; p < PER; p++) {
                const int c = g * PER + p;
                u32x4 x[XRow<XT>::P];
                b.x[c].parts(x);
#pragma unroll
                for (int i = 0; i < XRow<XT>::P; i++) sum = mfma16(F16, x[i], ones, sum);
#pragma unroll
                for (int t = 0; t < RT; t++) {
                    const u32x4 w = Codes<XT>::of(b.w[t][c]);
#pragma unroll
                    for (int i = 0; i < XRow<XT>::P; i++) acc[t] = mfma16(F16, x[i], w, acc[t]);
                }
            }
#pragma unroll
            for (int t = 0; t < RT; t++) {
                const float s = b.s[t][g], off = MINS ? fmaf(-16.f, s, b.least[t][g]) : -24.f * s;
#pragma unroll
                for (int r = 0; r < 4; r++) out[t][r] = fmaf(s, acc[t][r], fmaf(off, sum[r], out[t][r]));
            }
        }
    }
}

template <int XT, int G, bool MINS, int RT>
__global__ __launch_bounds__(64 * Q4_WAVES) void q4_kernel(Q4Args a) {
    __shared__ float red[Q4_WAVES][16][16 * RT + 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nw = blockDim.x >> 6;
    const int n0 = blockIdx.x * 16 * RT, m0 = blockIdx.y * 16, slabs = (a.n_in + 127) / 128;
    f32x4 out[RT] = {};
    Slab<XT, G, MINS, RT> cur, next;
    if (wave < slabs) q4_load(a, cur, wave * 128, n0, m0, lane);
    for (int s = wave; s < slabs; s += nw) {
        if (s + nw < slabs) q4_load(a, next, (s + nw) * 128, n0, m0, lane);
        q4_use(a, cur, s * 128, out);
        cur = next;
    }
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) red[wave][4 * (lane >> 4) + r][16 * t + (lane & 15)] = out[t][r];
    __syncthreads();
    for (int i = threadIdx.x; i < 256 * RT; i += blockDim.x) {
        const int n = n0 + i % (16 * RT), ml = i / (16 * RT), m = m0 + ml;
        if (n >= a.n_out || m >= a.n_rows) continue;
        float v = 0.f;
        for (int w = 0; w < nw; w++) v += red[w][ml][i % (16 * RT)];
        if constexpr (XT == HIPVOC_T_INT8) {
            if (a.x_groups == 1) v *= a.x_scale[m];
        }
        const int64_t at = m * a.y_stride + n;
        if (a.y_dtype == HIPVOC_T_F32) store1<HIPVOC_T_F32>(a.y, at, v);
        else if (a.y_dtype == HIPVOC_T_F16) store1<HIPVOC_T_F16>(a.y, at, v);
        else store1<HIPVOC_T_BF16>(a.y, at, v);
    }
}

template <int XT, int G, bool MINS> static void q4_rt(const Q4Args &a, hipStream_t s) {
    const int slabs = (a.n_in + 127) / 128, nw = slabs < Q4_WAVES ? slabs : Q4_WAVES, tiles = (a.n_out + 15) / 16, my = (a.n_rows + 15) / 16;
    if (tiles >= 1024) q4_kernel<XT, G, MINS, 2><<<dim3((tiles + 1) / 2, my), 64 * nw, 0, s>>>(a);
    else q4_kernel<XT, G, MINS, 1><<<dim3(tiles, my), 64 * nw, 0, s>>>(a);
}
template <int XT, int G> static void q4_mins(const Q4Args &a, hipStream_t s) {
    if (a.mins) q4_rt<XT, G, true>(a, s);
    else q4_rt<XT, G, false>(a, s);
}
template <int XT> static hipError_t q4_group(const Q4Args &a, hipStream_t s) {
    if (a.group == 32) q4_mins<XT, 32>(a, s);
    else if (a.group == 64) q4_mins<XT, 64>(a, s);
    else q4_mins<XT, 128>(a, s);
    return hipGetLastError();
}
hipError_t launch_q4_matvec(const Q4Args &a, hipStream_t s) {
    if (a.x_dtype == HIPVOC_T_INT8) return q4_group<HIPVOC_T_INT8>(a, s);
    if (a.x_dtype == HIPVOC_T_F32) return q4_group<HIPVOC_T_F32>(a, s);
    if (a.x_dtype == HIPVOC_T_F16) return q4_group<HIPVOC_T_F16>(a, s);
    return q4_group<HIPVOC_T_BF16>(a, s);
}

}  // namespace hipvoc
