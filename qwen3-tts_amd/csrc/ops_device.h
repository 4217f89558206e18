// Device helpers of the token-step operators: the five storage types, rows of eight values, 8-bit codes.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ops_kernels.h"

namespace hipvoc {

typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32v2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// storage types; N bytes per value
template <int T> struct Store;
template <> struct Store<HIPVOC_T_F32> { typedef float type; };
template <> struct Store<HIPVOC_T_F16> { typedef _Float16 type; };
template <> struct Store<HIPVOC_T_BF16> { typedef __bf16 type; };
template <> struct Store<HIPVOC_T_INT8> { typedef int8_t type; };
template <> struct Store<HIPVOC_T_E4M3> { typedef uint8_t type; };

__device__ __forceinline__ float bf16_lo(unsigned u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf16_hi(unsigned u) { return __uint_as_float(u & 0xffff0000u); }
__device__ __forceinline__ unsigned pack_bf16(float a, float b) {      // round to nearest even: v_cvt_pk_bf16_f32
    b16x2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(unsigned, v);
}
__device__ __forceinline__ unsigned pack_f16(float a, float b) {       // round to nearest even (v_cvt_f16_f32 twice, not the truncating pack)
    h16x2 v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(unsigned, v);
}

// eight consecutive values as floats; p is 16-byte aligned (8-bit types: 8-byte aligned)
template <int T> __device__ __forceinline__ void load8(const void *p, float *f) {
    if constexpr (T == HIPVOC_T_F32) {
        const f32x4 a = ((const f32x4 *)p)[0], b = ((const f32x4 *)p)[1];
#pragma unroll
        for (int i = 0; i < 4; i++) { f[i] = a[i]; f[4 + i] = b[i]; }
    } else if constexpr (T == HIPVOC_T_BF16) {
        const u32x4 a = *(const u32x4 *)p;
#pragma unroll
        for (int i = 0; i < 4; i++) { f[2 * i] = bf16_lo(a[i]); f[2 * i + 1] = bf16_hi(a[i]); }
    } else if constexpr (T == HIPVOC_T_F16) {
        const h16x8 a = *(const h16x8 *)p;
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = (float)a[i];
    } else if constexpr (T == HIPVOC_T_INT8) {
        const u32x2 a = *(const u32x2 *)p;
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = (float)(int8_t)(a[i >> 2] >> (8 * (i & 3)));
    } else {
        const u32x2 a = *(const u32x2 *)p;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(a[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(a[i], true);
            f[4 * i] = lo[0]; f[4 * i + 1] = lo[1]; f[4 * i + 2] = hi[0]; f[4 * i + 3] = hi[1];
        }
    }
}

// eight values as they are
template <int T> struct Raw8 { u32x4 w[T == HIPVOC_T_F32 ? 2 : 1]; };
template <int T> __device__ __forceinline__ Raw8<T> load_raw8(const void *p) {
    Raw8<T> r;
    r.w[0] = ((const u32x4 *)p)[0];
    if constexpr (T == HIPVOC_T_F32) r.w[1] = ((const u32x4 *)p)[1];
    return r;
}
template <int T> __device__ __forceinline__ void store_raw8(void *p, const Raw8<T> &r) {
    ((u32x4 *)p)[0] = r.w[0];
    if constexpr (T == HIPVOC_T_F32) ((u32x4 *)p)[1] = r.w[1];
}

// eight floats rounded once to act type T
template <int T> __device__ __forceinline__ void store8(void *p, const float *f) {
    if constexpr (T == HIPVOC_T_F32) {
        ((f32x4 *)p)[0] = (f32x4){f[0], f[1], f[2], f[3]};
        ((f32x4 *)p)[1] = (f32x4){f[4], f[5], f[6], f[7]};
    } else if constexpr (T == HIPVOC_T_BF16) {
        *(u32x4 *)p = (u32x4){pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7])};
    } else {
        *(u32x4 *)p = (u32x4){pack_f16(f[0], f[1]), pack_f16(f[2], f[3]), pack_f16(f[4], f[5]), pack_f16(f[6], f[7])};
    }
}

template <int T> __device__ __forceinline__ void store1(void *p, int64_t i, float f) { ((typename Store<T>::type *)p)[i] = (typename Store<T>::type)f; }

// The 8-bit types: scale = max|x| * (1 / TOP), both factors 32-bit numbers, code = x / scale (IEEE division, so the code is a function of
// the 32-bit quotient alone) rounded to nearest even.  The factor is the reciprocal's, by definition (include/hipvoc_ops.h): against max|x| / TOP rounded
// once, 4 % (INT8) or 59 % (E4M3) of the scales differ in the last bit and with them codes that stand on a border; what is held is as near to x either way
// (100000 bf16 rows of 128: 0.0064696 and 0.0257150 of it, to 9 digits the same).  |x / scale| <= TOP * (1 + 2^-22), which rounds to TOP in both types unless the scale
// is subnormal (it may then be off by half its value, or 0): the clamp is for that.  scale 0: code 0.
template <int T> __device__ __forceinline__ constexpr float top8() { return T == HIPVOC_T_INT8 ? 127.f : 448.f; }
template <int T> __device__ __forceinline__ float scale8(float amax) {
    constexpr float inv = 1.0f / (T == HIPVOC_T_INT8 ? 127.f : 448.f);
    return amax * inv;
}
// max|x| that keeps NaN (fmaxf would drop it): magnitudes compare like their bits, a NaN above an infinity.  A row with a NaN gets scale NaN, one with
// an infinity scale infinity, and both read back as NaN.
__device__ __forceinline__ unsigned amax_bits(unsigned m, float x) { return max(m, __float_as_uint(x) & 0x7fffffffu); }
// ... over 4, 8 or 16 neighbouring lanes (quad permutations, then mirrors of 8 and 16: what is left of a mirror is alike in all its lanes), or the wave
template <int CTRL> __device__ __forceinline__ unsigned dpp(unsigned v) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true); }
__device__ __forceinline__ unsigned amax_lanes(unsigned m, int lanes) {
    m = max(m, dpp<0xb1>(m));
    m = max(m, dpp<0x4e>(m));
    if (lanes > 4) m = max(m, dpp<0x141>(m));
    if (lanes > 8) m = max(m, dpp<0x140>(m));
    return m;
}
template <int LANES> __device__ __forceinline__ float sum_lanes(float v) {          // LANES = 8 or 16
    v += __uint_as_float(dpp<0xb1>(__float_as_uint(v)));
    v += __uint_as_float(dpp<0x4e>(__float_as_uint(v)));
    v += __uint_as_float(dpp<0x141>(__float_as_uint(v)));
    if (LANES > 8) v += __uint_as_float(dpp<0x140>(__float_as_uint(v)));
    return v;
}
__device__ __forceinline__ unsigned amax_wave(unsigned m) {
    m = amax_lanes(m, 16);
    m = max(m, (unsigned)__shfl_xor((int)m, 16));
    return max(m, (unsigned)__shfl_xor((int)m, 32));
}

// x / scale, correctly rounded, for many x: with y = 1 / scale correctly rounded, q = x y is within an ulp or two of the quotient, x - q scale is exact in
// one fused step and q + (x - q scale) y is the quotient rounded once (Markstein 1990), three instructions for a dozen.  It needs room below x
// for the remainder, so small scales take the division.  scale 0, infinite or NaN: 0, which reads back as 0 or NaN.
template <int T> struct Coder {
    float scale, inv;
    bool fast;
    __device__ __forceinline__ explicit Coder(float s) : scale(s) {
        fast = s > 0x1p-80f && s < 0x1p+80f;
        inv = 1.f / (fast ? s : 1.f);
    }
    __device__ __forceinline__ float quotient(float x) const {
        float t;
        if (fast) {
            const float q = x * inv;
            t = fmaf(fmaf(-q, scale, x), inv, q);
        } else {
            t = scale > 0.f && scale < __builtin_inff() ? x / scale : 0.f;
        }
        return fminf(fmaxf(t, -top8<T>()), top8<T>());
    }
    __device__ __forceinline__ u32x2 eight(const float *x) const {
        float t[8];
        if (fast) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float q = x[i] * inv;
                t[i] = fmaf(fmaf(-q, scale, x[i]), inv, q);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) t[i] = quotient(x[i]);
        }
        u32x2 r;
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
            for (int i = 0; i < 4; i++) t[4 * h + i] = __builtin_amdgcn_fmed3f(t[4 * h + i], -top8<T>(), top8<T>());
            if constexpr (T == HIPVOC_T_INT8) {
                unsigned u = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) u |= ((unsigned)(int)rintf(t[4 * h + i]) & 0xffu) << (8 * i);
                r[h] = u;
            } else {
                int u = __builtin_amdgcn_cvt_pk_fp8_f32(t[4 * h], t[4 * h + 1], 0, false);
                u = __builtin_amdgcn_cvt_pk_fp8_f32(t[4 * h + 2], t[4 * h + 3], u, true);
                r[h] = (unsigned)u;
            }
        }
        return r;
    }
    __device__ __forceinline__ uint8_t one(float x) const {
        const float t = quotient(x);
        if constexpr (T == HIPVOC_T_INT8) return (uint8_t)(int)rintf(t);
        else return (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(t, t, 0, false) & 0xff);
    }
};

__device__ __forceinline__ void raise(int *err, int bit) { atomicOr(err, bit); }

}  // namespace hipvoc
