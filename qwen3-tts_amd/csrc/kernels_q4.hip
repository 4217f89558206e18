// Products of a few rows with 4-bit weights and group scales (include/hipvoc_ops.h: hipvoc_q4_matvec).
//
// Mathematics: y[m][n] = sum_g s[n][g] * sum_k (c - 8) x[m][k]  (or s * sum c x + min * sum x), c = 0 .. 15.
// Bound: memory: half a byte per weight, read once.
#include "ops_device.h"

namespace hipvoc {

template <int XT> __device__ __forceinline__ float q4_x(const Q4Args &a, int m, int k) {
    const float v = load1<XT>(a.x, m * a.x_stride + k);
    if constexpr (XT == HIPVOC_T_INT8) return v * a.x_scale[(int64_t)m * a.x_groups + (a.x_groups == 1 ? 0 : k / a.group)];
    return v;
}

// One wave per weight row and row of x
template <int XT, int YT>
__global__ __launch_bounds__(256) void q4_row_kernel(Q4Args a) {
    const int n = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63, m = blockIdx.y;
    if (n >= a.n_out) return;
    float acc = 0.f;
    for (int b = lane; b < a.n_in / 2; b += 64) {
        const int c = a.codes[(int64_t)n * (a.n_in / 2) + b], g = 2 * b / a.group;
        const int64_t at = (int64_t)n * (a.n_in / a.group) + g;
        const float s = (float)((const _Float16 *)a.scales)[at], least = a.mins ? (float)((const _Float16 *)a.mins)[at] : -8.f * s;
        acc = fmaf(fmaf(s, (float)(c & 15), least), q4_x<XT>(a, m, 2 * b), acc);
        acc = fmaf(fmaf(s, (float)(c >> 4), least), q4_x<XT>(a, m, 2 * b + 1), acc);
    }
#pragma unroll
    for (int o = 1; o < 64; o *= 2) acc += __shfl_xor(acc, o);
    if (lane == 0) store1<YT>(a.y, m * a.y_stride + n, acc);
}

template <int XT, int YT> static hipError_t q4_go(const Q4Args &a, hipStream_t s) {
    q4_row_kernel<XT, YT><<<dim3((a.n_out + 3) / 4, a.n_rows), 256, 0, s>>>(a);
    return hipGetLastError();
}
hipError_t launch_q4_matvec(const Q4Args &a, hipStream_t s) {
    if (a.x_dtype == HIPVOC_T_INT8) {
        if (a.y_dtype == HIPVOC_T_F32) return q4_go<HIPVOC_T_INT8, HIPVOC_T_F32>(a, s);
        if (a.y_dtype == HIPVOC_T_F16) return q4_go<HIPVOC_T_INT8, HIPVOC_T_F16>(a, s);
        return q4_go<HIPVOC_T_INT8, HIPVOC_T_BF16>(a, s);
    }
    if (a.x_dtype == HIPVOC_T_F32) return q4_go<HIPVOC_T_F32, HIPVOC_T_F32>(a, s);
    if (a.x_dtype == HIPVOC_T_F16) return q4_go<HIPVOC_T_F16, HIPVOC_T_F16>(a, s);
    return q4_go<HIPVOC_T_BF16, HIPVOC_T_BF16>(a, s);
}

}  // namespace hipvoc
