// Distillation from a teacher's top logits: the loss over every (step, row) and
// its gradient with respect to the student's logits.
//
// A row is compared over k + 1 outcomes, the listed tokens and "any other".
// With u = the teacher's values / tau, N = lse of these and the rest, x = logits / tau,
// R = lse of the x that are not listed and Z = lse of all:
//   row = sum_j p_j (u_j - N - x_j + Z) + p_rest (rest - N - R + Z)
//   d row / d x_v = q_v - p_v (listed),  q_v (1 - p_rest / q_rest) (other)
// R is summed over the other tokens themselves and Z joined from R and the
// listed ones, so q_rest keeps its digits when the list holds nearly
// everything (lse(all) minus the list would not), and the gradient of the others
// is exp(x - m_R) times ONE factor per row.
//
// Where student and teacher are near each other the terms of the first sum cancel:
// logarithms of 10 known to 1e-6 for a sum of 1e-3.  Probabilities of the outcomes
// sum to 1 on both sides, so with d = log q - log p
//   sum p (log p - log q) = sum p (e^d - 1 - d),
// terms that are not negative, in which an error of a normaliser, common to all d,
// is multiplied by sum (q - p) = 0.  d and e^d - 1 - d are taken in 64 bits, for the
// k + 1 outcomes only; the normalisers' logarithm in 32.  (An outcome without p adds
// its q; an index that appears twice has its q once.)
#include "rows.h"

namespace {

struct DistillArgs {
    const void *logits, *values;
    const int32_t *indices;
    const float *rest;
    const int64_t *targets;
    const int32_t *lengths;
    const float *weight;   // [T], or null: weight_all
    const float *factor;   // of the gradient, on the device, or null: 1
    float *rowloss;        // one sum per block, or null: the gradient only
    void *dlogits;
    int32_t *status;
    long long ld, rows;
    int B, V, k, values_dtype;
    float weight_all;
    double inv_t64;        // 1 / tau
    float scale;           // log2(e) / tau
    float soft, hard;      // (1 - hard) tau^2; hard
    float dsoft;           // (1 - hard) tau
};

constexpr float LOG2E = 1.4426950408889634f;

// weight of every step: 1 / rows that run at it
__global__ __launch_bounds__(256) void distill_weight_kernel(
    const int32_t *lengths, int T, int B, float *out) {
    const int t = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (t >= T) return;
    int c = 0;
    for (int b = lane; b < B; b += 64) c += lengths[b] > t ? 1 : 0;
    c = (int)wave_sum((float)c);   // (exact: B < 2^24 is checked)
    if (lane == 0) out[t] = c > 0 ? 1.0f / (float)c : 0.0f;
}

__device__ __forceinline__ float row_weight(const DistillArgs &a, long long row) {
    const int t = (int)row / a.B;   // (rows fit 31 bits; both loads at once)
    const int len = a.lengths ? a.lengths[row - (long long)t * a.B] : t + 1;
    const float w = a.weight ? a.weight[t] : a.weight_all;
    return t < len ? w : 0.f;
}
// weight of the row's gradient
__device__ __forceinline__ float grad_weight(const DistillArgs &a, float w) {
    return a.factor ? w * a.factor[0] : w;
}
__device__ __forceinline__ float teacher_value(const DistillArgs &a,
                                               long long at) {
    if (a.values_dtype == PCM_DTYPE_F32) return ((const float *)a.values)[at];
    if (a.values_dtype == PCM_DTYPE_BF16)
        return (float)((const __bf16 *)a.values)[at];
    return (float)((const _Float16 *)a.values)[at];
}
// index of a listed token; -1: absent
__device__ __forceinline__ int teacher_index(const DistillArgs &a, long long at) {
    const int i = a.indices[at];
    if (i >= a.V) {
        if (a.status) atomicOr(a.status, PCM_STATUS_BAD_TOKEN);
        return -1;
    }
    return i < 0 ? -1 : i;
}
__device__ __forceinline__ int target_of(const DistillArgs &a, long long row,
                                         bool report) {
    const long long t = a.targets[row];
    if (t >= 0 && t < a.V) return (int)t;
    if (report && a.status) atomicOr(a.status, PCM_STATUS_BAD_TOKEN);
    return t < 0 ? 0 : a.V - 1;
}
// exp((x - m) c) for x <= m; c carries log2(e).  m is finite.
__device__ __forceinline__ float exp_below(float x, float m, float c) {
    return __builtin_amdgcn_exp2f((x - m) * c);
}
__device__ __forceinline__ float finite_or_0(float m) {
    return m == -INFINITY ? 0.f : m;
}

// the same value in every lane, in a scalar register
__device__ __forceinline__ float uniform(float v) {
    return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v)));
}

// c (p (log p - log q) + q - p) of an outcome, d = log q - log p.  (Below 1e-30 p
// has lost digits, and what it adds to q is nothing unless q is 0.  The row's factor c
// goes in before 64 bits become 32: masks of the type's lowest value have parts
// that leave them where the loss does not.)
__device__ __forceinline__ float kl_term(float p, double d, float q, double c) {
    if (!(p <= 1e-30f)) return (float)(c * ((double)p * (expm1(d) - d)));
    return (float)(c * (p == 0.f ? (double)q : (double)q - (double)p * (1. + d)));
}

// probability of the outcome "any other token".  (Where none is left mo is not a
// maximum, and 0 times a power of it need not be 0.)
__device__ __forceinline__ float other_q(float mo, float s, float ma, float sa,
                                         float scale) {
    return s == 0.f ? 0.f : exp_below(mo, ma, scale) * s / sa;
}

// A teacher's outcomes relative to its largest listed value v0 (0 if it lists none):
// differences of values before the product with 1 / tau, so that neither a list far
// from 0 nor one of nothing but the type's lowest value loses digits or range.
// The rest, which is at the temperature already, is relative to it in 64 bits; h,
// not below 0 if anything is listed, is the largest of both.
struct Teacher {
    float v0, hl;     // hl: h log2(e)
    double rb, h;     // the rest, relative
    __device__ __forceinline__ Teacher(const DistillArgs &a, float vmax, float rest) {
        v0 = finite_or_0(vmax);
        rb = rest - (double)v0 * a.inv_t64;
        h = fmax(rb, vmax > -INFINITY ? 0. : rb);
        if (h == -INFINITY) h = 0.;
        hl = (float)(h * 1.4426950408889634);
    }
    __device__ __forceinline__ float listed(const DistillArgs &a, float v) const {
        return __builtin_amdgcn_exp2f(fmaf(v - v0, a.scale, -hl));
    }
    __device__ __forceinline__ float other() const {
        return __builtin_amdgcn_exp2f((float)((rb - h) * 1.4426950408889634));
    }
    // log of the same
    __device__ __forceinline__ double log_listed(const DistillArgs &a,
                                                 float v) const {
        return ((double)v - v0) * a.inv_t64 - h;
    }
    __device__ __forceinline__ double log_other() const { return rb - h; }
};

// What a row's factors are made of: the others' maximum m and sum(s), the listed
// tokens' xm and sums, the teacher's; w: the weight of its gradient.  (Sums relative
// to exp(max).)
struct RowStats {
    float ma;        // maximum of the row
    float sa, ha;    // sums over the row relative to it: / tau, plain
    float cq, ch;    // gradient of an other token: exp((x - mo) / tau) cq +
                     // exp(x - mo) ch
};
__device__ __forceinline__ RowStats row_stats(const DistillArgs &a, float w,
                                              float m, float s, float h,
                                              float xm, float xs, float xh,
                                              bool taught, float pr) {
    RowStats r;
    const float mo = finite_or_0(m), xo = finite_or_0(xm);
    r.ma = fmaxf(m, xm);
    // a part that is empty is 0, not 0 times a power of the other's maximum
    const float fo = s == 0.f ? 0.f : exp_below(mo, r.ma, a.scale);
    const float fx = xs == 0.f ? 0.f : exp_below(xo, r.ma, a.scale);
    r.sa = s * fo + xs * fx;
    r.cq = 0.f;
    if (taught)
        r.cq = a.dsoft * w * (fo / r.sa - (pr > 0.f && s > 0.f ? pr / s : 0.f));
    r.ha = 1.f;
    r.ch = 0.f;
    if (a.hard > 0.f) {
        const float go = h == 0.f ? 0.f : exp_below(mo, r.ma, LOG2E);
        const float gx = xh == 0.f ? 0.f : exp_below(xo, r.ma, LOG2E);
        r.ha = h * go + xh * gx;
        r.ch = a.hard * w * go / r.ha;
    }
    return r;
}

// ---- short rows -----------------------------------------------------------------
// V <= 512: LPR lanes share a row (4 for V <= 128, else 16), a wave takes
// 64 / LPR rows.  A row of 60 is 240 bytes: what counts is the number of
// instructions per row, and the reductions over it are two DPP steps here, six
// with a wave per row.  The row is in registers; a copy in LDS is where the
// listed tokens are looked up, and where the gradients meet: of the others from the
// registers, of the listed ones and the target from their entries.
// 61440 ragged x 60 fp32, k = 8, with targets: 18.9 us for 24.6 MB (1.3 TB/s), bound
// by the instructions and LDS accesses of the lists (2.5 us of it are the loss's 64
// bits); a wave per row took 201 us.  fp16, the loss alone 13.5 us, the gradient 15.
template <int DT, int LPR, int G, bool HARD>
__global__ __launch_bounds__(64) void distill_short_kernel(DistillArgs a) {
    typedef RowType<DT> R;
    typedef typename R::T T;
    constexpr int ROWS = 64 / LPR, MW = LPR * G / 4;
    extern __shared__ float sm[];
    const int lane = threadIdx.x, r = lane / LPR, sub = lane % LPR;
    const int V = a.V, k = a.k, LD = V | 1, LK = k | 1;
    float *tile = sm + r * LD;                         // a row: logits, gradients
    float *u = sm + ROWS * LD + r * LK;                // its list: values, then p
    float *lx = sm + ROWS * (LD + LK) + r * LK;        // its logits
    int *li = (int *)(sm + ROWS * (LD + 2 * LK)) + r * LK;   // its indices; -1:
                                // absent; -2 - index: an earlier entry has it
    unsigned *marks = (unsigned *)(sm + ROWS * (LD + 3 * LK)) + r * MW;
    const long long row = (long long)blockIdx.x * ROWS + r;
    const bool inside = row < a.rows;
    const float w = inside ? row_weight(a, row) : 0.f;
    const bool live = w != 0.f;
    const float wg = grad_weight(a, w);
    const T *x = (const T *)a.logits + row * a.ld;
    RowRegs<DT, LPR, G> regs;
    float rest = -INFINITY;
    int tg = 0;
    if (live) {
        regs.load(x, V, sub);
        if (a.rest) rest = a.rest[row];
        if (HARD) tg = target_of(a, row, sub == 0);
        for (int j = sub; j < k; j += LPR) {
            const int idx = teacher_index(a, row * k + j);
            li[j] = idx;
            u[j] = idx < 0 ? -INFINITY : teacher_value(a, row * k + j);
        }
        for (int i = sub; i < MW; i += LPR) marks[i] = 0;
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int e = regs.at(g, sub) + j;
                if (e < V) tile[e] = regs.r[g].get(j);
            }
    }
    __syncthreads();
    float xt = 0.f, um = -INFINITY;
    int flags = rest != rest ? 1 : 0;   // 1: a NaN; 2: an index twice
    if (live) {
        if (HARD) xt = tile[tg];
        for (int j = sub; j < k; j += LPR) {
            const int idx = li[j];
            um = fmaxf(um, u[j]);
            if (u[j] != u[j]) flags |= 1;
            lx[j] = idx < 0 ? -INFINITY : tile[idx];
            if (idx >= 0) {
                const unsigned bit = 1u << (idx & 31);
                if (atomicOr(&marks[idx >> 5], bit) & bit) flags |= 2;
            }
        }
    }
    __syncthreads();
    um = row_max<LPR>(um);
    flags |= lane_xor<1>(flags);
    flags |= lane_xor<2>(flags);
    if constexpr (LPR == 16) {
        flags |= lane_xor<4>(flags);
        flags |= lane_xor<8>(flags);
    }
    const bool twice = flags & 2;
    if (live && twice && sub == 0)   // rare: only the first entry stands for it
        for (int j = 1; j < k; ++j)
            for (int i = 0; i < j; ++i)
                if (li[j] >= 0 && li[i] == li[j]) {
                    li[j] = -2 - li[j];
                    break;
                }
    __syncthreads();
    // teacher, and the listed tokens' part of the student
    const bool taught =
        a.soft > 0.f && (um > -INFINITY || rest > -INFINITY || (flags & 1));
    const Teacher said(a, um, rest);
    float us = 0.f, xm = -INFINITY;
    if (live)
        for (int j = sub; j < k; j += LPR) {
            us += said.listed(a, u[j]);
            if (li[j] >= 0) xm = fmaxf(xm, lx[j]);
        }
    us = row_sum<LPR>(us);
    xm = row_max<LPR>(xm);
    const float ro = said.other();
    us += ro;
    const float ius = 1.f / us, pr = taught ? ro * ius : 0.f;
    const float xo = finite_or_0(xm);
    float xs = 0.f, xh = 0.f, m = -INFINITY;
    if (live) {
        for (int j = sub; j < k; j += LPR)
            if (li[j] >= 0) {
                xs += exp_below(lx[j], xo, a.scale);
                if (HARD) xh += exp_below(lx[j], xo, LOG2E);
            }
        // the others
        const unsigned char *mark8 = (const unsigned char *)marks;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const unsigned bits = mark8[g * LPR + sub];
            if (bits) regs.r[g].drop(bits);
#pragma unroll
            for (int j = 0; j < 8; ++j) m = fmaxf(m, regs.r[g].get(j));
        }
    }
    m = row_max<LPR>(m);
    xs = row_sum<LPR>(xs);
    if (HARD) xh = row_sum<LPR>(xh);
    const float mo = finite_or_0(m);
    float s = 0.f, h = 0.f, e[G * 8], eh[HARD ? G * 8 : 1];
    if (live) {   // (kept: an exponential costs four other instructions)
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float v = regs.r[g].get(j);
                e[g * 8 + j] = exp_below(v, mo, a.scale);
                s += e[g * 8 + j];
                if (HARD) {
                    eh[g * 8 + j] = exp_below(v, mo, LOG2E);
                    h += eh[g * 8 + j];
                }
            }
    }
    s = row_sum<LPR>(s);
    if (HARD) h = row_sum<LPR>(h);
    const RowStats st = row_stats(a, wg, m, s, h, xm, xs, xh, taught, pr);
    auto teacher_p = [&](int j) { return said.listed(a, u[j]) * ius; };
    // gradients: the others', the listed ones', the target's
    if (a.dlogits) {
        if (live) {
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int at = regs.at(g, sub) + j;
                    float q = e[g * 8 + j] * st.cq;
                    if (HARD) q += eh[g * 8 + j] * st.ch;
                    if (at < V) tile[at] = q;
                }
        }
        __syncthreads();
        if (live) {
            const float cs = taught ? a.dsoft * wg : 0.f;
            const float ca = cs / st.sa, ch = HARD ? a.hard * wg / st.ha : 0.f;
            for (int j = sub; j < k; j += LPR)
                if (li[j] >= 0) {
                    float q = ca * exp_below(lx[j], st.ma, a.scale);
                    if (HARD) q += ch * exp_below(lx[j], st.ma, LOG2E);
                    if (!twice && taught) q -= cs * teacher_p(j);
                    tile[li[j]] = q;
                }
        }
        __syncthreads();
        if (live && sub == 0) {
            if (twice && taught)
                for (int j = 0; j < k; ++j) {
                    const int idx = li[j] >= -1 ? li[j] : -2 - li[j];
                    if (idx >= 0) tile[idx] -= a.dsoft * wg * teacher_p(j);
                }
            if (HARD) tile[tg] -= a.hard * wg;
        }
        __syncthreads();
        if (inside) {
            T *dl = (T *)a.dlogits + row * V;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const int at = regs.at(g, sub);
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    v[j] = live && at + j < V ? tile[at + j] : 0.f;
                if (at + 8 <= V) Row8<DT>::store(dl + at, v);
                else {
#pragma unroll
                    for (int j = 0; j < 7; ++j)
                        if (at + j < V) dl[at + j] = R::down(v[j]);
                }
            }
        }
    }
    // the row's loss, when the registers are free again
    if (!a.rowloss) return;
    float loss = 0.f;
    if (live && taught) {
        const double c = logf(us / st.sa), soft = (double)a.soft * w;
        // (entry k: any other token)
        for (int j = sub; j <= k; j += LPR) {
            const bool other = j == k;
            const int idx = other ? 0 : li[j];
            const float p = other ? pr : teacher_p(j), at = other ? mo : lx[j];
            const double d = ((double)at - st.ma) * a.inv_t64 + c -
                             (other ? said.log_other() - log((double)s)
                                    : said.log_listed(a, u[j]));
            const float q = other ? other_q(mo, s, st.ma, st.sa, a.scale)
                                  : exp_below(at, st.ma, a.scale) / st.sa;
            if (idx != -1 || p != p) loss += kl_term(p, d, q, soft);
            if (idx < -1) loss -= (float)(q * soft);
        }
    }
    if (HARD && live && sub == 0)
        loss += a.hard * w * (logf(st.ha) - (xt - st.ma));
    loss = wave_sum(loss);
    if (lane == 0) a.rowloss[blockIdx.x] = loss;
}

// ---- longer rows ----------------------------------------------------------------
// One block per row.  KEEP: the row stays in registers, read once and written
// once; else it is read twice.  Wave 0 holds the list, one entry per lane; the
// listed tokens are marked in a bitmap in LDS -- a group of eight elements is one
// byte of it -- and become -inf in the registers, so the passes see the others
// only.  What bounds it is memory, as long as two blocks fit a CU and one loads
// while the other computes: 2048 x 32000 bf16 in 60 us (4.4 TB/s; a large copy
// reaches 4.7), fp16 in 47 (the loss alone, vector units 0.87) and 54 (the gradient);
// 1024 ragged x 50021 fp32 with targets in 85 us (3.6 TB/s: at most four rows per CU,
// so two turns of loads with little to hide behind); 7 x 601 fp16 in 5.2 us (latency).
// LG: up to so many more groups of a thread are kept in LDS, in the threads' order
// (each thread reads what it wrote: no barrier).
template <int DT, int NT, int G, bool HARD, bool KEEP, int LG = 0>
__global__ __launch_bounds__(NT, KEEP ? row_waves(DT, NT, G) : 8) void
distill_row_kernel(DistillArgs a) {
    static_assert(LG == 0 || (KEEP && DT == PCM_DTYPE_F32), "fp32 halves in LDS");
    typedef RowType<DT> R;
    typedef typename R::T T;
    extern __shared__ __align__(16) unsigned marks[];   // a bit per element
    __shared__ float red[NT / 64], red2[NT / 64];
    __shared__ float s_list[8];
    __shared__ double s_other;   // log of the other's p, not normalised; h
    __shared__ double s_high;
    // what wave 0 needs of its list after the passes (registers are the row's)
    __shared__ int w_idx[64];
    __shared__ float w_x[64], w_p[64], w_value[64], w_mass[64];
    const int tid = threadIdx.x, lane = tid & 63;
    const long long row = blockIdx.x;
    const int V = a.V, k = a.k;
    const float w = uniform(row_weight(a, row));
    T *dl = a.dlogits ? (T *)a.dlogits + row * V : nullptr;
    const int groups = KEEP ? G + LG : (V + NT * 8 - 1) / (NT * 8);
    if (w == 0.f) {
        if (tid == 0 && a.rowloss) a.rowloss[row] = 0.f;
        if (dl)
            for (int g = 0; g < groups; ++g) {
                const int e = (g * NT + tid) * 8;
                const float zero[8] = {};
                if (e + 8 <= V) Row8<DT>::store(dl + e, zero);
                else
                    for (int j = e; j < V; ++j) dl[j] = R::down(0.f);
            }
        return;
    }
    const T *x = (const T *)a.logits + row * a.ld;
    RowRegs<DT, NT, G> regs;
    if (KEEP) regs.load(x, V, tid);
    const int words = groups * NT / 4;   // groups * NT bytes
    // a group in LDS: the first halves of all its threads, then the second ones
    // (neighbours 16 bytes apart: no bank is asked twice)
    auto each_kept = [&](auto f) {
#pragma unroll 1
        for (int l = 0; l < LG; ++l) {
            const int e = ((G + l) * NT + tid) * 8;
            if (e >= V) break;
            const int last = (V - (G + l) * NT * 8 + 7) / 8;
            float *lo = (float *)(marks + words) + l * NT * 8 + tid * 4;
            f(e, G + l, (row_u32x4 *)lo,
              (row_u32x4 *)(lo + 4 * (last < NT ? last : NT)));
        }
    };
    if constexpr (LG > 0)
        each_kept([&](int e, int, row_u32x4 *lo, row_u32x4 *hi) {
            Row8<DT> q;
            load_group(q, x, V, e);
            *lo = q.a;
            *hi = q.b;
        });
    // the list: lane j of wave 0 holds entry j
    int idx = -1, tg = -1;
    float value = -INFINITY, lx = -INFINITY, xt = 0.f, rest = -INFINITY;
    if (tid < 64) {
        if (a.rest) rest = a.rest[row];
        if (HARD) {
            tg = __builtin_amdgcn_readfirstlane(target_of(a, row, lane == 0));
            xt = uniform(R::up(x[tg]));
        }
        if (lane < k) {
            idx = teacher_index(a, row * k + lane);
            if (idx >= 0) {
                value = teacher_value(a, row * k + lane);
                lx = R::up(x[idx]);
            }
        }
    }
    for (int i = tid; i < words; i += NT) marks[i] = 0;
    __syncthreads();
    bool first = false;
    if (tid < 64 && idx >= 0) {
        const unsigned bit = 1u << (idx & 31);
        first = !(atomicOr(&marks[idx >> 5], bit) & bit);
    }
    __syncthreads();
    // the others' maximum, beside it (wave 0) what the list gives
    float m = -INFINITY;
    const unsigned char *mark8 = (const unsigned char *)marks;
    auto unlist = [&](Row8<DT> &q, int g) {   // group g without the listed tokens
        const unsigned bits = mark8[g * NT + tid];
        if (bits) q.drop(bits);
    };
    float s = 0.f, h = 0.f;
    if (KEEP) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
            regs.r[g].touch(m);
            unlist(regs.r[g], g);
#pragma unroll
            for (int j = 0; j < 8; ++j) m = fmaxf(m, regs.r[g].get(j));
        }
        if constexpr (LG > 0)
            each_kept([&](int, int g, row_u32x4 *lo, row_u32x4 *hi) {
                Row8<DT> q;
                q.a = *lo;
                q.b = *hi;
                const unsigned bits = mark8[g * NT + tid];
                if (bits) {
                    q.drop(bits);
                    *lo = q.a;
                    *hi = q.b;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) m = fmaxf(m, q.get(j));
            });
    } else {
        // maximum and sums in one pass, relative to the thread's running maximum
        each_group<DT, NT>(x, V, tid, [&](Row8<DT> &q, int g) {
            unlist(q, g);
            float v[8], gm = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = q.get(j);
                gm = fmaxf(gm, v[j]);
            }
            if (gm > m) {
                if (m > -INFINITY) {
                    s *= __builtin_amdgcn_exp2f((m - gm) * a.scale);
                    if (HARD) h *= __builtin_amdgcn_exp2f((m - gm) * LOG2E);
                }
                m = gm;
            }
            const float mm = finite_or_0(m);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                s += __builtin_amdgcn_exp2f((v[j] - mm) * a.scale);
                if (HARD) h += __builtin_amdgcn_exp2f((v[j] - mm) * LOG2E);
            }
        });
    }
    if (tid < 64) {
        float p = 0.f, mass = 0.f;
        if (__any(idx >= 0 && !first)) {   // rare: an index that appears twice
            bool again = false;
            for (int j = 0; j < k; ++j) {
                const int ij = __builtin_amdgcn_readlane(idx, j);
                again |= j < lane && ij == idx;
            }
            first = idx >= 0 && !again;
        }
        const float um = wave_max(value);
        const bool bad = __any(value != value || rest != rest);
        const bool taught =
            a.soft > 0.f && (um > -INFINITY || rest > -INFINITY || bad);
        const Teacher said(a, um, rest);
        const float e = said.listed(a, value), ro = said.other();
        const float us = wave_sum(e) + ro;
        if (taught) p = e / us;
        mass = p;
        if (__any(idx >= 0 && !first)) {
            mass = 0.f;
            for (int j = 0; j < k; ++j) {
                const int ij = __builtin_amdgcn_readlane(idx, j);
                const float pj = __int_as_float(
                    __builtin_amdgcn_readlane(__float_as_int(p), j));
                if (ij == idx) mass += pj;
            }
        }
        const float xm = wave_max(first ? lx : -INFINITY);
        const float xo = finite_or_0(xm);
        const float xs = wave_sum(first ? exp_below(lx, xo, a.scale) : 0.f);
        const float xh =
            HARD ? wave_sum(first ? exp_below(lx, xo, LOG2E) : 0.f) : 0.f;
        w_idx[lane] = first ? idx : idx >= 0 ? -2 : -1;   // (an entry that is not
        w_x[lane] = lx;           // the first of its index: a loss, no gradient)
        w_p[lane] = p;
        w_value[lane] = value;
        w_mass[lane] = mass;
        if (lane == 0) {
            s_list[5] = us;
            s_list[6] = said.v0;
            s_list[7] = xt;
            s_other = said.log_other();
            s_high = said.h;
            s_list[0] = xm;
            s_list[1] = xs;
            s_list[2] = xh;
            s_list[3] = taught ? 1.f : 0.f;
            s_list[4] = taught ? ro / us : 0.f;
        }
    }
    const float mt = finite_or_0(m);   // (KEEP: not used)
    m = uniform(all_max<NT>(m, red, tid));
    const float mo = finite_or_0(m);
    if (KEEP) {
        auto add = [&](const Row8<DT> &q) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float d = q.get(j) - mo;
                s += __builtin_amdgcn_exp2f(d * a.scale);
                if (HARD) h += __builtin_amdgcn_exp2f(d * LOG2E);
            }
        };
#pragma unroll
        for (int g = 0; g < G; ++g) {
            regs.r[g].touch(s);
            if (HARD) regs.r[g].touch(h);
            add(regs.r[g]);
        }
        if constexpr (LG > 0)
            each_kept([&](int, int, row_u32x4 *lo, row_u32x4 *hi) {
                Row8<DT> q;
                q.a = *lo;
                q.b = *hi;
                add(q);
            });
    } else {
        // (a thread without others has the sums 0, or NaN)
        if (!(s == 0.f)) s *= __builtin_amdgcn_exp2f((mt - mo) * a.scale);
        if (HARD && !(h == 0.f)) h *= __builtin_amdgcn_exp2f((mt - mo) * LOG2E);
    }
    s = uniform(all_sum<NT>(s, red2, tid));
    if (HARD) h = uniform(all_sum<NT>(h, red, tid));
    __syncthreads();   // s_list
    const bool taught = s_list[3] != 0.f;
    const float pr = s_list[4];
    const float wg = uniform(grad_weight(a, w));
    RowStats st = row_stats(a, wg, m, s, h, s_list[0], s_list[1], s_list[2], taught,
                            pr);
    st.ma = uniform(st.ma);
    st.sa = uniform(st.sa);
    st.ha = uniform(st.ha);
    st.cq = uniform(st.cq);
    st.ch = uniform(st.ch);
    // The last wave does this after its stores (the first has the list to write): it
    // takes no registers from the row, and less than what the stores take to arrive.
    auto row_loss = [&] {
        if (!a.rowloss) return;
        float loss = 0.f;
        if (taught) {
            const double c = logf(s_list[5] / st.sa), soft = (double)a.soft * w;
            const float p = w_p[lane], at = w_x[lane];
            const float q = exp_below(at, st.ma, a.scale) / st.sa;
            const int li = w_idx[lane];
            if (li != -1 || p != p)
                loss = kl_term(p, ((double)at - st.ma) * a.inv_t64 + c -
                                      (((double)w_value[lane] - s_list[6]) *
                                           a.inv_t64 - s_high), q, soft);
            if (li < -1) loss -= (float)(q * soft);
            if (lane == 0)
                loss += kl_term(pr, ((double)mo - st.ma) * a.inv_t64 + c -
                                        (s_other - log((double)s)),
                                other_q(mo, s, st.ma, st.sa, a.scale), soft);
            loss = wave_sum(loss);
        }
        if (HARD) loss += a.hard * w * (logf(st.ha) - (s_list[7] - st.ma));
        if (lane == 0) a.rowloss[row] = loss;
    };
    if (!dl) {
        if (tid >= NT - 64) row_loss();
        return;
    }
    auto write = [&](int g, const Row8<DT> &q) {
        const int e = (g * NT + tid) * 8;
        if (e >= V) return;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float d = q.get(j) - mo;
            v[j] = __builtin_amdgcn_exp2f(d * a.scale) * st.cq;
            if (HARD) v[j] += __builtin_amdgcn_exp2f(d * LOG2E) * st.ch;
        }
        if (e + 8 <= V) Row8<DT>::store(dl + e, v);
        else {
#pragma unroll
            for (int j = 0; j < 7; ++j)
                if (e + j < V) dl[e + j] = R::down(v[j]);
        }
    };
    if (KEEP) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
            regs.r[g].touch();
            write(g, regs.r[g]);
        }
        if constexpr (LG > 0)
            each_kept([&](int, int g, row_u32x4 *lo, row_u32x4 *hi) {
                Row8<DT> q;
                q.a = *lo;
                q.b = *hi;
                write(g, q);
            });
    } else {
        each_group<DT, NT>(x, V, tid, [&](Row8<DT> &q, int g) {
            unlist(q, g);
            write(g, q);
        });
    }
    if (tid >= NT - 64) row_loss();
    __syncthreads();   // the listed tokens and the target over what is there
    if (tid < 64) {
        const int li = w_idx[lane];
        if (li >= 0) {
            const float lv = w_x[lane];
            float g = 0.f;
            if (s_list[3] != 0.f)
                g = a.dsoft * wg *
                    (exp_below(lv, st.ma, a.scale) / st.sa - w_mass[lane]);
            if (HARD) {
                g += a.hard * wg * exp_below(lv, st.ma, LOG2E) / st.ha;
                if (li == tg) g -= a.hard * wg;
            }
            dl[li] = R::down(g);
        }
        if (HARD && lane == 0 && !(marks[tg >> 5] >> (tg & 31) & 1)) {
            const float d = xt - mo;
            dl[tg] = R::down(__builtin_amdgcn_exp2f(d * a.scale) * st.cq +
                             __builtin_amdgcn_exp2f(d * LOG2E) * st.ch -
                             a.hard * wg);
        }
    }
}

// deterministic single-block sum, in 64 bits
__global__ __launch_bounds__(1024) void distill_sum_kernel(const float *x,
                                                           long long n,
                                                           float *out) {
    __shared__ double part[16];
    double s = 0.;
    for (long long i = threadIdx.x; i < n; i += 1024) s += (double)x[i];
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double total = 0.;
        for (int i = 0; i < 16; ++i) total += part[i];
        out[0] = (float)total;
    }
}

// For a gradient that was rounded before its factor was known: fp32, and bf16, which
// has fp32's exponents, so that what is rounded twice is off by half a step each
// time, however small.  (fp16 would lose here what is below 6e-8, most of a
// large vocabulary's gradient, which is what a loss scale is there to keep:
// pcm_distill_grad.)  The usual factor is 1, for which they stay as they are.
template <int DT>
__global__ __launch_bounds__(256) void scale_kernel(typename RowType<DT>::T *x,
                                                    long long n,
                                                    const float *scale) {
    typedef RowType<DT> R;
    const float f = scale[0];
    if (f == 1.0f) return;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n;
         i += (long long)gridDim.x * 256)
        x[i] = R::down(R::up(x[i]) * f);
}

// Launches the rows of a call; returns how many partial sums they leave.
// Up to 65536 a row stays in the registers of its block (read once): 1552 rows of
// 32768 in 96 us (fp32) and 51 us (bf16) against 111 and 60 when it is read
// twice, 776 of 65536 in 110 and 55 against 121 and 63.
// With 32-bit logits past 32768 the registers of a row leave one block per CU, which
// loads and computes in turn; two fit where what is past 32768 lies in LDS: 1024
// rows of 50944 in 106 us (111 with targets) against 115 (126) of 50945 in
// registers alone.
constexpr int KEPT_MAX = 50944;   // (two blocks of at most 80 KB of LDS)
template <int DT, bool HARD>
long long launch_rows(const DistillArgs &a, hipStream_t st) {
    const int V = a.V;
#define PCM_DISTILL_SHORT(LPR, G)                                              \
    do {                                                                      \
        constexpr int ROWS = 64 / (LPR);                                      \
        const size_t lds = (size_t)ROWS * ((V | 1) + 3 * (a.k | 1) +          \
                                           (LPR) * (G) / 4) * sizeof(float);  \
        const long long blocks = (a.rows + ROWS - 1) / ROWS;                  \
        hipLaunchKernelGGL((distill_short_kernel<DT, LPR, G, HARD>),          \
                           dim3((unsigned)blocks), dim3(64), lds, st, a);     \
        return blocks;                                                        \
    } while (0)
    if (V <= 64) PCM_DISTILL_SHORT(4, 2);
    if (V <= 128) PCM_DISTILL_SHORT(4, 4);
    if (V <= 512) PCM_DISTILL_SHORT(16, 4);
#undef PCM_DISTILL_SHORT
#define PCM_DISTILL_ROWS(NT, G)                                             \
    hipLaunchKernelGGL((distill_row_kernel<DT, NT, G, HARD, true>),          \
                       dim3((unsigned)a.rows), dim3(NT), (size_t)(NT) * (G), \
                       st, a)
    if (V <= 1024) PCM_DISTILL_ROWS(64, 2);
    else if (V <= 2048) PCM_DISTILL_ROWS(256, 1);
    else if (V <= 4096) PCM_DISTILL_ROWS(256, 2);
    else if (V <= 8192) PCM_DISTILL_ROWS(256, 4);
    else if (V <= 16384) PCM_DISTILL_ROWS(512, 4);
    else if (V <= 32768) PCM_DISTILL_ROWS(1024, 4);
    else if (DT == PCM_DTYPE_F32 && V <= KEPT_MAX) {
        // past 32768 in LDS, beside the bitmap
        const size_t lds = 7 * 1024 + (size_t)(V - 32768 + 7) / 8 * 32;
        hipLaunchKernelGGL((distill_row_kernel<PCM_DTYPE_F32, 1024, 4, HARD, true, 3>),
                           dim3((unsigned)a.rows), dim3(1024), lds, st, a);
    } else if (V <= 65536) PCM_DISTILL_ROWS(1024, 8);
#undef PCM_DISTILL_ROWS
    else {
        const size_t lds = (size_t)(V + 8191) / 8192 * 1024;
        hipLaunchKernelGGL((distill_row_kernel<DT, 1024, 1, HARD, false>),
                           dim3((unsigned)a.rows), dim3(1024), lds, st, a);
    }
    return a.rows;
}

}  // namespace

extern "C" {

size_t pcm_distill_scratch_floats(int32_t steps, int32_t batch) {
    if (steps < 1 || batch < 1) return 0;
    return (size_t)steps * batch + steps;
}

// loss, or the gradient times a factor
static int distill(const void *logits, int32_t dtype, int64_t ld,
                   const void *values, int32_t values_dtype,
                   const int32_t *indices, const float *rest, int32_t k,
                   const int64_t *targets, const int32_t *lengths,
                   const float *step_weight, int32_t steps, int32_t batch,
                   int32_t vocab, double temperature, double hard_weight,
                   const float *factor, float *loss, void *dlogits,
                   float *scratch, int32_t *status, void *stream) {
    PCM_REQUIRE(logits && values && indices && scratch, PCM_EINVAL,
                "distill_loss: null pointer");
    PCM_REQUIRE(pcm_dtype_known(dtype) && pcm_dtype_known(values_dtype),
                PCM_EINVAL, "distill_loss: unknown dtype %d / %d", dtype,
                values_dtype);
    PCM_REQUIRE(steps > 0 && batch > 0 && vocab > 0 && vocab <= PCM_MAX_VOCAB,
                PCM_EINVAL, "distill_loss: bad shape T=%d B=%d V=%d (V 1..%d)",
                steps, batch, vocab, PCM_MAX_VOCAB);
    PCM_REQUIRE((long long)steps * batch < (1ll << 31) && batch < (1 << 24),
                PCM_EINVAL,
                "distill_loss: too many rows");
    PCM_REQUIRE(ld >= vocab, PCM_EINVAL, "distill_loss: row stride %lld < %d",
                (long long)ld, vocab);
    PCM_REQUIRE(k >= 1 && k <= PCM_TOP_MAX, PCM_EINVAL,
                "distill_loss: k=%d outside 1..%d", k, PCM_TOP_MAX);
    // (the loss carries its square, in 32 bits)
    PCM_REQUIRE(temperature >= 1e-3 && temperature <= 1e3, PCM_EINVAL,
                "distill_loss: temperature outside 1e-3..1e3");
    PCM_REQUIRE(hard_weight >= 0. && hard_weight <= 1., PCM_EINVAL,
                "distill_loss: hard_weight=%f outside 0..1", hard_weight);
    PCM_REQUIRE(hard_weight == 0. || targets, PCM_EINVAL,
                "distill_loss: hard_weight needs targets");
    // (a launch has less than 2^32 threads)
    PCM_REQUIRE(vocab <= 2048 || (long long)steps * batch < (1ll << 22),
                PCM_EINVAL, "distill_loss: %lld rows of %d logits are too many "
                "for a launch", (long long)steps * batch, vocab);
    PCM_REQUIRE(vocab <= 512 || (long long)steps * batch < (1ll << 24),
                PCM_EINVAL, "distill_loss: %lld rows of %d logits are too many "
                "for a launch", (long long)steps * batch, vocab);
    // (16 lanes a row, in blocks of four; of up to 128 logits 4 and 16)
    PCM_REQUIRE((long long)steps * batch <= (1ll << 28) - 4, PCM_EINVAL,
                "distill_loss: %lld rows are too many for a launch",
                (long long)steps * batch);
    PCM_REQUIRE(!lengths || step_weight || steps < (1 << 26) - 4, PCM_EINVAL,
                "distill_loss: the weights of %d steps are too many for a launch",
                steps);
    hipStream_t st = (hipStream_t)stream;
    DistillArgs a;
    a.logits = logits; a.values = values; a.indices = indices; a.rest = rest;
    a.targets = targets; a.lengths = lengths; a.dlogits = dlogits;
    a.status = status;
    a.rows = (long long)steps * batch;
    a.factor = factor;
    a.rowloss = loss ? scratch : nullptr;
    a.ld = ld; a.B = batch; a.V = vocab; a.k = k;
    a.values_dtype = values_dtype;
    a.weight = step_weight;
    a.weight_all = 1.0f / (float)batch;
    a.inv_t64 = 1.0 / temperature;
    a.scale = (float)(1.4426950408889634 / temperature);
    a.soft = (float)((1.0 - hard_weight) * temperature * temperature);
    a.dsoft = (float)((1.0 - hard_weight) * temperature);
    a.hard = (float)hard_weight;
    if (lengths && !step_weight) {
        hipLaunchKernelGGL(distill_weight_kernel, dim3((steps + 3) / 4),
                           dim3(256), 0, st, lengths, steps, batch,
                           scratch + a.rows);
        a.weight = scratch + a.rows;
    }
    long long sums;
    if (hard_weight > 0.)
        PCM_BY_DTYPE(dtype, sums = launch_rows<DT, true>(a, st));
    else
        PCM_BY_DTYPE(dtype, sums = launch_rows<DT, false>(a, st));
    if (loss)
        hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, st,
                           a.rowloss, sums, loss);
    return pcm_check_launch("distill_loss");
}

int pcm_distill_loss(const void *logits, int32_t dtype, int64_t ld,
                     const void *values, int32_t values_dtype,
                     const int32_t *indices, const float *rest, int32_t k,
                     const int64_t *targets, const int32_t *lengths,
                     const float *step_weight, int32_t steps, int32_t batch,
                     int32_t vocab, double temperature, double hard_weight,
                     float *loss, void *dlogits, float *scratch,
                     int32_t *status, void *stream) {
    PCM_API_GUARD;
    PCM_REQUIRE(loss, PCM_EINVAL, "distill_loss: null pointer");
    return distill(logits, dtype, ld, values, values_dtype, indices, rest, k,
                   targets, lengths, step_weight, steps, batch, vocab,
                   temperature, hard_weight, nullptr, loss, dlogits, scratch,
                   status, stream);
}

int pcm_distill_grad(const void *logits, int32_t dtype, int64_t ld,
                     const void *values, int32_t values_dtype,
                     const int32_t *indices, const float *rest, int32_t k,
                     const int64_t *targets, const int32_t *lengths,
                     const float *step_weight, int32_t steps, int32_t batch,
                     int32_t vocab, double temperature, double hard_weight,
                     const float *factor, void *dlogits, float *scratch,
                     void *stream) {
    PCM_API_GUARD;
    PCM_REQUIRE(factor && dlogits, PCM_EINVAL, "distill_grad: null pointer");
    return distill(logits, dtype, ld, values, values_dtype, indices, rest, k,
                   targets, lengths, step_weight, steps, batch, vocab,
                   temperature, hard_weight, factor, nullptr, dlogits, scratch,
                   nullptr, stream);
}


int pcm_scale(void *x, int32_t dtype, int64_t n, const float *scale,
              void *stream) {
    PCM_API_GUARD;
    PCM_REQUIRE(x && scale && n > 0, PCM_EINVAL, "scale: bad args");
    PCM_REQUIRE(pcm_dtype_known(dtype), PCM_EINVAL, "scale: unknown dtype %d",
                dtype);
    long long blocks = (n + 2047) / 2048;
    if (blocks > 4096) blocks = 4096;
    PCM_BY_DTYPE(dtype, {
        hipLaunchKernelGGL(scale_kernel<DT>, dim3((unsigned)blocks), dim3(256), 0,
                           (hipStream_t)stream, (RowType<DT>::T *)x,
                           (long long)n, scale);
    });
    return pcm_check_launch("scale");
}

}  // extern "C"
