// Root-mean-square norm with the residual's addition (include/hipvoc_ops.h: hipvoc_add_rmsnorm), in the act type or in 8 bits.
//
// Mathematics: s = x + r, y = s / sqrt(mean s^2 + eps) * w; 8 bits: y ~ code * (max|y| / TOP) per group of columns.  Everything in 32
// bits; s is rounded once where it is stored, y once (or to a code).
// Bound: memory (and, for a few rows, the latency of one load, one reduction and one store).  A row is read once and stays in
// registers: NV vectors of eight values per thread, TH threads per row; rows of up to 1024 values are a wave's own, four rows to a workgroup
// (no barrier); 2048 values: 256 threads and one vector each beat a wave with four (8192 rows to e4m3, when both were measured: 26.5 against 28.2 us;
// the kernel now: 19.6).
#include "ops_device.h"

namespace hipvoc {

__device__ __forceinline__ float wave_sum(float v) {
    v = sum_lanes<16>(v);
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// Eight values anywhere (ODD: a row whose length, stride or place is no multiple of 16 bytes; global memory is read and written in up to 16 bytes at any
// alignment)
template <int T, bool ODD> __device__ __forceinline__ void load_vec(const typename Store<T>::type *p, float *f) {
    if constexpr (!ODD) {
        load8<T>(p, f);
    } else {
        Raw8<T> raw;
        __builtin_memcpy(&raw, p, sizeof raw);
        load8<T>(&raw, f);
    }
}
template <int T, bool ODD> __device__ __forceinline__ void store_vec(typename Store<T>::type *p, const float *f) {
    if constexpr (!ODD) {
        store8<T>(p, f);
    } else {
        Raw8<T> raw;
        store8<T>(&raw, f);
        __builtin_memcpy(p, &raw, sizeof raw);
    }
}
template <bool ODD> __device__ __forceinline__ void store_codes(uint8_t *p, u32x2 c) {
    if constexpr (!ODD) *(u32x2 *)p = c;
    else __builtin_memcpy(p, &c, 8);
}

// OUT == ACT: y in the act type, else codes.  TH threads (64, 256 or 1024) have a row; a workgroup has max(TH, 256) threads.  ODD: the last vector of a
// row that is no multiple of 8 long ends with the row; what it has in common with the one before counts once, is read before anything is
// written, and is written twice alike (8192 x 2047 in bf16: 26 us; element by element, 45).
template <int ACT, int OUT, int TH, int NV, bool ODD>
__global__ __launch_bounds__(TH < 256 ? 256 : TH) void add_rmsnorm_kernel(NormArgs a) {
    constexpr int ROWS = TH < 256 ? 256 / TH : 1, NWAVE = TH / 64;
    typedef typename Store<ACT>::type act_t;
    __shared__ float sh[NWAVE > 1 ? NWAVE : 1];
    __shared__ unsigned sh_top[NWAVE > 1 ? NWAVE : 1];
    const int t = threadIdx.x % TH, row = blockIdx.x * ROWS + threadIdx.x / TH;
    if (ROWS > 1 && row >= a.rows) return;                      // a wave's own row: no barrier follows
    const act_t *x = (const act_t *)a.x + row * a.x_stride, *r = (const act_t *)a.residual + row * a.residual_stride, *weight = (const act_t *)a.weight;
    const auto has = [&](int v) { return (v * TH + t) * 8 < a.cols; };
    const auto at = [&](int v) { return ODD ? min((v * TH + t) * 8, a.cols - 8) : (v * TH + t) * 8; };       // where this thread's vector v stands
    float s[NV][8], w[NV][8], sq = 0.f;
#pragma unroll
    for (int v = 0; v < NV; v++) {
        if (has(v)) {
            load_vec<ACT, ODD>(x + at(v), s[v]);
            load_vec<ACT, ODD>(weight + at(v), w[v]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) s[v][e] = w[v][e] = 0.f;
        }
    }
    if (a.residual) {
#pragma unroll
        for (int v = 0; v < NV; v++) {
            if (has(v)) {
                float b[8];
                load_vec<ACT, ODD>(r + at(v), b);
#pragma unroll
                for (int e = 0; e < 8; e++) s[v][e] += b[e];
            }
        }
    }
#pragma unroll
    for (int v = 0; v < NV; v++) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float one = ODD && at(v) + e < (v * TH + t) * 8 ? 0.f : s[v][e];
            sq = fmaf(one, one, sq);
        }
    }
    sq = wave_sum(sq);
    if constexpr (NWAVE > 1) {
        if ((t & 63) == 0) sh[t >> 6] = sq;
        __syncthreads();
        sq = 0.f;
#pragma unroll
        for (int i = 0; i < NWAVE; i++) sq += sh[i];
    }
    const float rs = 1.f / sqrtf(sq / (float)a.cols + a.eps);
    unsigned top = 0;
#pragma unroll
    for (int v = 0; v < NV; v++) {
        if (a.sum && has(v)) store_vec<ACT, ODD>((act_t *)a.sum + row * a.sum_stride + at(v), s[v]);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            s[v][e] = s[v][e] * rs * w[v][e];
            if constexpr (OUT != ACT) top = amax_bits(top, s[v][e]);
        }
        if constexpr (OUT == ACT) {
            if (has(v)) store_vec<ACT, ODD>((act_t *)a.y + row * a.y_stride + at(v), s[v]);
        }
    }
    if constexpr (OUT != ACT) {
        uint8_t *y = (uint8_t *)a.y + row * a.y_stride;
        if (a.group == 0) {
            top = amax_wave(top);
            if constexpr (NWAVE > 1) {
                if ((t & 63) == 0) sh_top[t >> 6] = top;
                __syncthreads();
#pragma unroll
                for (int i = 0; i < NWAVE; i++) top = max(top, sh_top[i]);
            }
            const float scale = scale8<OUT>(__uint_as_float(top));
            const Coder<OUT> code(scale);
            if (t == 0) a.scales[row] = scale;
#pragma unroll
            for (int v = 0; v < NV; v++) {
                if (has(v)) store_codes<ODD>(y + at(v), code.eight(s[v]));
            }
        } else {
            // a group is 4, 8 or 16 neighbouring lanes of one vector index (TH is a multiple of 16), and a row whole groups
            const int lanes = a.group / 8;
#pragma unroll
            for (int v = 0; v < NV; v++) {
                const int i = v * TH + t;
                unsigned g = 0;
#pragma unroll
                for (int e = 0; e < 8; e++) g = amax_bits(g, s[v][e]);
                const float scale = scale8<OUT>(__uint_as_float(amax_lanes(g, lanes)));
                if (has(v)) {
                    store_codes<ODD>(y + i * 8, Coder<OUT>(scale).eight(s[v]));
                    if (i % lanes == 0) a.scales[(int64_t)row * (a.cols / a.group) + i / lanes] = scale;
                }
            }
        }
    }
}

// Rows under 8 or over 32768 values: a workgroup per row, one value at a time.  s is made anew in every pass, and the stored sum may be x or the residual: it is
// written last, behind a barrier where another thread may still read its place.
template <int ACT, int OUT>
__global__ __launch_bounds__(256) void add_rmsnorm_any_kernel(NormArgs a) {
    typedef typename Store<ACT>::type act_t;
    __shared__ float sh[4];
    const int t = threadIdx.x, row = blockIdx.x;
    const act_t *x = (const act_t *)a.x + row * a.x_stride, *r = (const act_t *)a.residual + row * a.residual_stride;
    auto s_of = [&](int i) { return (float)x[i] + (a.residual ? (float)r[i] : 0.f); };
    float sq = 0.f;
    for (int i = t; i < a.cols; i += 256) {
        const float s = s_of(i);
        sq = fmaf(s, s, sq);
    }
    sq = wave_sum(sq);
    if ((t & 63) == 0) sh[t >> 6] = sq;
    __syncthreads();
    const float rs = 1.f / sqrtf((sh[0] + sh[1] + sh[2] + sh[3]) / (float)a.cols + a.eps);
    auto y_of = [&](int i) { return s_of(i) * rs * (float)((const act_t *)a.weight)[i]; };
    if constexpr (OUT == ACT) {
        for (int i = t; i < a.cols; i += 256) {
            const float s = s_of(i);
            store1<ACT>(a.y, row * a.y_stride + i, s * rs * (float)((const act_t *)a.weight)[i]);
            if (a.sum) store1<ACT>(a.sum, row * a.sum_stride + i, s);
        }
    } else {
        uint8_t *y = (uint8_t *)a.y + row * a.y_stride;
        const int n = a.group ? a.group : a.cols, groups = a.cols / n, lane = t & 63;
        // a group per wave; the whole row: all four waves find the same maximum over all of it, and each codes a quarter
        const bool whole = a.group == 0;
        for (int g = whole ? 0 : t >> 6; g < groups; g += 4) {
            unsigned top = 0;
            for (int i = lane; i < n; i += 64) top = amax_bits(top, y_of(g * n + i));
            const float scale = scale8<OUT>(__uint_as_float(amax_wave(top)));
            const Coder<OUT> code(scale);
            if (lane == 0 && (!whole || t == 0)) a.scales[(int64_t)row * groups + g] = scale;
            for (int i = whole ? t : lane; i < n; i += whole ? 256 : 64) y[g * n + i] = code.one(y_of(g * n + i));
        }
        __syncthreads();
        if (a.sum)
            for (int i = t; i < a.cols; i += 256) store1<ACT>(a.sum, row * a.sum_stride + i, s_of(i));
    }
}

template <int ACT, int OUT, int TH, int NV> static void norm_go(const NormArgs &a, bool odd, hipStream_t s) {
    constexpr int ROWS = TH < 256 ? 256 / TH : 1, THREADS = TH < 256 ? 256 : TH;
    const int blocks = (a.rows + ROWS - 1) / ROWS;
    if (odd) add_rmsnorm_kernel<ACT, OUT, TH, NV, true><<<blocks, THREADS, 0, s>>>(a);
    else add_rmsnorm_kernel<ACT, OUT, TH, NV, false><<<blocks, THREADS, 0, s>>>(a);
}
template <int ACT, int OUT> static hipError_t norm_out(const NormArgs &a, hipStream_t s) {
    constexpr int A = ACT == HIPVOC_T_F32 ? 4 : 2;
    auto off = [](const void *p, int64_t stride, int size) { return (((uintptr_t)p) | (uint64_t)(stride * size)) & 15; };
    bool odd = a.cols % 8 || off(a.x, a.x_stride, A) || off(a.weight, 0, A) || (a.residual && off(a.residual, a.residual_stride, A)) ||
               (a.sum && off(a.sum, a.sum_stride, A));
    odd = odd || (OUT == ACT ? off(a.y, a.y_stride, A) != 0 : ((((uintptr_t)a.y) | (uint64_t)a.y_stride) & 7) != 0);
    const int vecs = (a.cols + 7) / 8;
    if (a.cols < 8 || vecs > 4096) add_rmsnorm_any_kernel<ACT, OUT><<<a.rows, 256, 0, s>>>(a);
    else if (vecs <= 64) norm_go<ACT, OUT, 64, 1>(a, odd, s);
    else if (vecs <= 128) norm_go<ACT, OUT, 64, 2>(a, odd, s);
    else if (vecs <= 256) norm_go<ACT, OUT, 256, 1>(a, odd, s);
    else if (vecs <= 512) norm_go<ACT, OUT, 256, 2>(a, odd, s);
    else if (vecs <= 1024) norm_go<ACT, OUT, 256, 4>(a, odd, s);
    else norm_go<ACT, OUT, 1024, 4>(a, odd, s);
    return hipGetLastError();
}
template <int ACT> static hipError_t norm_act(const NormArgs &a, hipStream_t s) {
    if (a.out_dtype == HIPVOC_T_INT8) return norm_out<ACT, HIPVOC_T_INT8>(a, s);
    if (a.out_dtype == HIPVOC_T_E4M3) return norm_out<ACT, HIPVOC_T_E4M3>(a, s);
    return norm_out<ACT, ACT>(a, s);
}
hipError_t launch_add_rmsnorm(const NormArgs &a, hipStream_t s) {
    if (a.dtype == HIPVOC_T_F32) return norm_act<HIPVOC_T_F32>(a, s);
    if (a.dtype == HIPVOC_T_F16) return norm_act<HIPVOC_T_F16>(a, s);
    return norm_act<HIPVOC_T_BF16>(a, s);
}

}  // namespace hipvoc
