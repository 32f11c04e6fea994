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
#define PCM_BY_DTYPE(dtype, ...)                                     \
    do {                                                             \
        if ((dtype) == PCM_DTYPE_F32) {                              \
            constexpr int DT = PCM_DTYPE_F32; __VA_ARGS__;                  \
        } else if ((dtype) == PCM_DTYPE_BF16) {                      \
            constexpr int DT = PCM_DTYPE_BF16; __VA_ARGS__;                 \
        } else {                                                     \
            constexpr int DT = PCM_DTYPE_F16; __VA_ARGS__;                  \
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


// ---- lanes --------------------------------------------------------------------------
// Value of lane ^ M.  Within a row of 16 lanes by DPP, across rows by the
// row-swap instructions of gfx950: no LDS traffic, a few cycles each.
template <int M>
static __device__ __forceinline__ unsigned lane_xor(unsigned v) {
    static_assert(M == 1 || M == 2 || M == 4 || M == 8 || M == 16 || M == 32,
                  "one bit");
    if constexpr (M == 1)          // quad_perm 1 0 3 2
        return __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, true);
    else if constexpr (M == 2)     // quad_perm 2 3 0 1
        return __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, true);
    else if constexpr (M == 4) {   // half-row mirror (^7), then quads (^3)
        v = __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, true);
        return __builtin_amdgcn_update_dpp(0, v, 0x1B, 0xf, 0xf, true);
    } else if constexpr (M == 8)   // row rotation by 8
        return __builtin_amdgcn_update_dpp(0, v, 0x128, 0xf, 0xf, true);
    else if constexpr (M == 16) {  // [0] even rows of both, [1] odd rows
        auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return (threadIdx.x & 16) ? r[0] : r[1];
    } else {
        auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return (threadIdx.x & 32) ? r[0] : r[1];
    }
}
template <int M>
static __device__ __forceinline__ float lane_xor(float v) {
    return __uint_as_float(lane_xor<M>(__float_as_uint(v)));
}
template <int M>
static __device__ __forceinline__ int lane_xor(int v) {
    return (int)lane_xor<M>((unsigned)v);
}
template <int M>
static __device__ __forceinline__ double lane_xor(double v) {
    return __hiloint2double(lane_xor<M>(__double2hiint(v)),
                            lane_xor<M>(__double2loint(v)));
}

// ---- wave reductions ----------------------------------------------------------------
// every lane gets the result; the order of the sums is fixed
static __device__ __forceinline__ float pcm_max(float a, float b) { return fmaxf(a, b); }
static __device__ __forceinline__ double pcm_max(double a, double b) { return fmax(a, b); }
template <typename T>
static __device__ __forceinline__ T wave_max(T v) {
    v = pcm_max(v, lane_xor<1>(v));
    v = pcm_max(v, lane_xor<2>(v));
    v = pcm_max(v, lane_xor<4>(v));
    v = pcm_max(v, lane_xor<8>(v));
    v = pcm_max(v, lane_xor<16>(v));
    return pcm_max(v, lane_xor<32>(v));
}
template <typename T>
static __device__ __forceinline__ T wave_sum(T v) {
    v += lane_xor<1>(v);
    v += lane_xor<2>(v);
    v += lane_xor<4>(v);
    v += lane_xor<8>(v);
    v += lane_xor<16>(v);
    return v + lane_xor<32>(v);
}

// reductions over the LPR lanes of a row
template <int LPR, typename T>
static __device__ __forceinline__ T row_max(T v) {
    v = pcm_max(v, lane_xor<1>(v));
    v = pcm_max(v, lane_xor<2>(v));
    if constexpr (LPR == 16) {
        v = pcm_max(v, lane_xor<4>(v));
        v = pcm_max(v, lane_xor<8>(v));
    }
    return v;
}
template <int LPR, typename T>
static __device__ __forceinline__ T row_sum(T v) {
    v += lane_xor<1>(v);
    v += lane_xor<2>(v);
    if constexpr (LPR == 16) {
        v += lane_xor<4>(v);
        v += lane_xor<8>(v);
    }
    return v;
}
// block-wide maximum / sum, every thread gets it
template <int NT, typename T>
static __device__ __forceinline__ T all_max(T v, T *red, int tid) {
    v = wave_max(v);
    if constexpr (NT > 64) {
        __syncthreads();
        if ((tid & 63) == 0) red[tid >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int i = 1; i < NT / 64; ++i) v = pcm_max(v, red[i]);
    }
    return v;
}
template <int NT, typename T>
static __device__ __forceinline__ T all_sum(T v, T *red, int tid) {
    v = wave_sum(v);
    if constexpr (NT > 64) {
        __syncthreads();
        if ((tid & 63) == 0) red[tid >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int i = 1; i < NT / 64; ++i) v += red[i];
    }
    return v;
}

// ---- sorting 64 keys across a wave ------------------------------------------------------
// (one comparison and a choice: a maximum of values that a lane swap brought would
// be preceded by two that quiet NaNs, which keys never are)
template <int STRIDE>
static __device__ __forceinline__ double key_exchange(double v, bool keep_max) {
    const double o = lane_xor<STRIDE>(v);
    return (v > o) == keep_max ? v : o;
}
template <int SIZE, int STRIDE>
static __device__ __forceinline__ double key_sort_steps(double v, int lane) {
    v = key_exchange<STRIDE>(v, ((lane & STRIDE) == 0) ==
                                    ((lane & SIZE) == 0));
    if constexpr (STRIDE > 1) v = key_sort_steps<SIZE, STRIDE / 2>(v, lane);
    return v;
}
// a bitonic sequence, sorted: largest in lane 0
static __device__ __forceinline__ double key_merge(double v, int lane) {
    return key_sort_steps<64, 32>(v, lane);
}
static __device__ __forceinline__ double key_sort(double v, int lane) {
    v = key_sort_steps<2, 1>(v, lane);
    v = key_sort_steps<4, 2>(v, lane);
    v = key_sort_steps<8, 4>(v, lane);
    v = key_sort_steps<16, 8>(v, lane);
    v = key_sort_steps<32, 16>(v, lane);
    return key_merge(v, lane);
}
// value of one lane, known to all
static __device__ __forceinline__ double key_lane(double v, int lane) {
    return __hiloint2double(
        __builtin_amdgcn_readlane(__double2hiint(v), lane),
        __builtin_amdgcn_readlane(__double2loint(v), lane));
}

// ---- eight elements of a row in registers -----------------------------------------------
// Kept as they lie in memory (16-bit types packed) and widened where they are
// used.  A row starts at any element: the loads are 16 bytes wide and aligned to
// the element only, which global memory takes.
typedef unsigned row_u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned row_u32x4 __attribute__((ext_vector_type(4)));
typedef row_u32x4 row_u32x4_e2 __attribute__((aligned(2)));
typedef row_u32x4 row_u32x4_e4 __attribute__((aligned(4)));
template <int DT> struct Row8;
template <> struct Row8<PCM_DTYPE_F32> {
    row_u32x4 a, b;
    __device__ __forceinline__ void load(const float *p) {
        a = *(const row_u32x4_e4 *)p;
        b = *(const row_u32x4_e4 *)(p + 4);
    }
    __device__ __forceinline__ void lowest() { a = b = 0xFF800000u; }
    // -inf in the places of the bits
    __device__ __forceinline__ void drop(unsigned bits) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (bits >> i & 1) set(i, -INFINITY);
    }
    // What is derived from the elements is derived after this, and after what has
    // gone into `so_far` (or to memory): a pass over a row that touches each group
    // before it uses it neither keeps values widened by an earlier pass in
    // registers nor widens all groups at once.
    __device__ __forceinline__ void touch(float &so_far) {
        asm volatile("" : "+v"(a), "+v"(b), "+v"(so_far));
    }
    __device__ __forceinline__ void touch() {
        asm volatile("" : "+v"(a), "+v"(b) : : "memory");
    }
    static __device__ __forceinline__ void store(float *p, const float *v) {
        row_u32x4 x, y;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = __float_as_uint(v[i]);
            y[i] = __float_as_uint(v[4 + i]);
        }
        *(row_u32x4_e4 *)p = x;
        *(row_u32x4_e4 *)(p + 4) = y;
    }
    __device__ __forceinline__ void set(int i, float v) {
        if (i < 4) a[i] = __float_as_uint(v); else b[i - 4] = __float_as_uint(v);
    }
    __device__ __forceinline__ float get(int i) const {
        return __uint_as_float(i < 4 ? a[i] : b[i - 4]);
    }
};
template <> struct Row8<PCM_DTYPE_BF16> {
    row_u32x4 a;
    __device__ __forceinline__ void load(const __bf16 *p) {
        a = *(const row_u32x4_e2 *)p;
    }
    __device__ __forceinline__ void lowest() { a = 0xFF80FF80u; }
    __device__ __forceinline__ void drop(unsigned bits) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (bits >> i & 1) set(i, (__bf16)-INFINITY);
    }
    __device__ __forceinline__ void touch(float &so_far) {
        asm volatile("" : "+v"(a), "+v"(so_far));
    }
    __device__ __forceinline__ void touch() {
        asm volatile("" : "+v"(a) : : "memory");
    }
    static __device__ __forceinline__ void store(__bf16 *p, const float *v) {
        row_u32x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned short lo =
                __builtin_bit_cast(unsigned short, (__bf16)v[2 * i]);
            const unsigned short hi =
                __builtin_bit_cast(unsigned short, (__bf16)v[2 * i + 1]);
            x[i] = lo | (unsigned)hi << 16;
        }
        *(row_u32x4_e2 *)p = x;
    }
    __device__ __forceinline__ void set(int i, __bf16 v) {
        const unsigned u = __builtin_bit_cast(unsigned short, v);
        a[i >> 1] = i & 1 ? (a[i >> 1] & 0xffffu) | (u << 16)
                          : (a[i >> 1] & 0xffff0000u) | u;
    }
    __device__ __forceinline__ float get(int i) const {
        return __uint_as_float(i & 1 ? a[i >> 1] & 0xffff0000u : a[i >> 1] << 16);
    }
};
template <> struct Row8<PCM_DTYPE_F16> {
    row_u32x4 a;
    __device__ __forceinline__ void load(const _Float16 *p) {
        a = *(const row_u32x4_e2 *)p;
    }
    __device__ __forceinline__ void lowest() { a = 0xFC00FC00u; }
    __device__ __forceinline__ void drop(unsigned bits) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (bits >> i & 1) set(i, (_Float16)-INFINITY);
    }
    __device__ __forceinline__ void touch(float &so_far) {
        asm volatile("" : "+v"(a), "+v"(so_far));
    }
    __device__ __forceinline__ void touch() {
        asm volatile("" : "+v"(a) : : "memory");
    }
    static __device__ __forceinline__ void store(_Float16 *p, const float *v) {
        row_u32x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned short lo =
                __builtin_bit_cast(unsigned short, (_Float16)v[2 * i]);
            const unsigned short hi =
                __builtin_bit_cast(unsigned short, (_Float16)v[2 * i + 1]);
            x[i] = lo | (unsigned)hi << 16;
        }
        *(row_u32x4_e2 *)p = x;
    }
    __device__ __forceinline__ void set(int i, _Float16 v) {
        const unsigned u = __builtin_bit_cast(unsigned short, v);
        a[i >> 1] = i & 1 ? (a[i >> 1] & 0xffffu) | (u << 16)
                          : (a[i >> 1] & 0xffff0000u) | u;
    }
    __device__ __forceinline__ float get(int i) const {
        const unsigned short u =
            (unsigned short)(i & 1 ? a[i >> 1] >> 16 : a[i >> 1]);
        return (float)__builtin_bit_cast(_Float16, u);
    }
};

// Waves per SIMD that a kernel is to leave room for: two blocks of 1024 threads
// per CU where the row takes at most 32 registers of the 64 that this leaves, so
// that one block loads while the other computes.
constexpr int row_waves(int dt, int nt, int g) {
    return nt * (dt == PCM_DTYPE_F32 ? 2 * g : g) <= 8192 ? 8 : 4;
}

// n elements of a row, dealt to NT threads in groups of eight: element j of
// group g of thread tid is (g * NT + tid) * 8 + j.  What lies past n is -inf.
template <int DT, int NT, int G> struct RowRegs {
    Row8<DT> r[G];
    static __device__ __forceinline__ int at(int g, int tid) {
        return (g * NT + tid) * 8;
    }
    __device__ __forceinline__ void load(const typename RowType<DT>::T *p, int n,
                                         int tid) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int e = at(g, tid);
            if (e + 8 <= n) {
                r[g].load(p + e);
            } else {
                r[g].lowest();
                if (e < n) {
#pragma unroll
                    for (int j = 0; j < 7; ++j)
                        if (e + j < n) r[g].set(j, p[e + j]);
                }
            }
        }
    }
};

// elements e .. e + 7 of n, -inf past the end
template <int DT>
static __device__ __forceinline__ void load_group(
    Row8<DT> &q, const typename RowType<DT>::T *p, int n, int e) {
    if (e + 8 <= n) {
        q.load(p + e);
    } else {
        q.lowest();
#pragma unroll
        for (int j = 0; j < 7; ++j)
            if (e + j < n) q.set(j, p[e + j]);
    }
}

// every group of eight elements of the stretch, f(elements, group): thread tid
// has the groups at (g * NT + tid) * 8; four loads in flight
template <int DT, int NT, typename F>
static __device__ __forceinline__ void each_group(const typename RowType<DT>::T *p, int n,
                                           int tid, F f) {
    constexpr int U = 4;
    int g = 0;
    for (; (g + U) * NT * 8 <= n; g += U) {
        Row8<DT> q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) q[u].load(p + ((g + u) * NT + tid) * 8);
#pragma unroll
        for (int u = 0; u < U; ++u) f(q[u], g + u);
    }
    for (; g * NT * 8 < n; ++g) {
        Row8<DT> q;
        load_group(q, p, n, (g * NT + tid) * 8);
        f(q, g);
    }
}
