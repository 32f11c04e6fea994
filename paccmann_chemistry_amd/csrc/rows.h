// Device helpers of the kernels that rank or normalise rows of logits
// (topbeam.hip, distill.hip): element types, sort keys, wave reductions.
#pragma once
#include "common.h"

// ---- element types --------------------------------------------------------------
template <int DT> struct RowType;
template <> struct RowType<PCM_DTYPE_F32> {
    typedef float T;
    static __device__ __forceinline__ float up(T v) { return v; }
    static __device__ __forceinline__ T down(float v) { return v; }
};
template <> struct RowType<PCM_DTYPE_BF16> {
    typedef __bf16 T;
    static __device__ __forceinline__ float up(T v) { return (float)v; }
    static __device__ __forceinline__ T down(float v) { return (T)v; }
};
template <> struct RowType<PCM_DTYPE_F16> {
    typedef _Float16 T;
    static __device__ __forceinline__ float up(T v) { return (float)v; }
    static __device__ __forceinline__ T down(float v) { return (T)v; }
};
static inline size_t pcm_dtype_bytes(int dtype) {
    return dtype == PCM_DTYPE_F32 ? 4 : 2;
}
static inline bool pcm_dtype_known(int dtype) {
    return dtype >= PCM_DTYPE_F32 && dtype <= PCM_DTYPE_F16;
}
// run `call` with the constant DT equal to a dtype code
#define PCM_BY_DTYPE(dtype, call)                                    \
    do {                                                             \
        if ((dtype) == PCM_DTYPE_F32) {                              \
            constexpr int DT = PCM_DTYPE_F32; call;                  \
        } else if ((dtype) == PCM_DTYPE_BF16) {                      \
            constexpr int DT = PCM_DTYPE_BF16; call;                 \
        } else {                                                     \
            constexpr int DT = PCM_DTYPE_F16; call;                  \
        }                                                            \
    } while (0)

// ---- sort keys --------------------------------------------------------------------
// (value, index) as ONE double, so that a compare-exchange is v_max_f64 /
// v_min_f64 and "largest value, lowest index on ties" is "largest key".  A
// double orders like its sign-magnitude bits: the float's bits are its high
// word (fp32 infinities are finite doubles there, exponent 0x7f8) and the low
// word breaks ties, growing with a falling index where the value is positive and
// with a rising one where it is negative.  Keys of one row are distinct; a NaN
// ranks below -inf.  KEY_NONE (the double -inf) is below every key.
#define KEY_NONE (-__builtin_inf())
static __device__ __forceinline__ double key_of(float x, int idx) {
    unsigned u = __float_as_uint(x + 0.0f);   // -0 ties with +0
    if (x != x) u = 0xFF900000u;
    const unsigned low = (int)u < 0 ? (unsigned)idx : ~(unsigned)idx;
    return __hiloint2double((int)u, (int)low);
}
static __device__ __forceinline__ int key_index(double k) {
    const int hi = __double2hiint(k), lo = __double2loint(k);
    return hi < 0 ? lo : ~lo;
}
static __device__ __forceinline__ float key_value(double k) {
    return __int_as_float(__double2hiint(k));
}

// ---- wave reductions ----------------------------------------------------------------
static __device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
    return v;
}
static __device__ __forceinline__ double wave_max(double v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = fmax(v, __shfl_xor(v, off, 64));
    return v;
}
static __device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}
static __device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}
