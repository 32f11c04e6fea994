// Distillation from a teacher's top logits: the loss over every (step, row) and
// its gradient with respect to the student's logits.
//
// A row is compared over k + 1 outcomes, the listed tokens and "any other".
// With x = logits / tau, R = lse of the x that are not listed and Z = lse of
// all:
//   row = sum_j p_j (u_j - N - x_j + Z) + p_rest (rest - N - R + Z)
//   d row / d x_v = q_v - p_v (listed),  q_v (1 - p_rest / q_rest) (other)
// R is summed over the other tokens themselves and Z joined from R and the
// listed ones, so q_rest keeps its digits when the list holds nearly
// everything (lse(all) minus the list would not), and the gradient of the others
// is exp(x - m_R) times ONE factor per row.
#include "rows.h"

namespace {

struct DistillArgs {
    const void *logits, *values;
    const int32_t *indices;
    const float *rest;
    const int64_t *targets;
    const int32_t *lengths;
    const float *weight;   // [T], or null: weight_all
    float *rowloss;        // one sum per block
    void *dlogits;
    int32_t *status;
    long long ld, rows;
    int B, V, k, values_dtype;
    float weight_all;
    float inv_t, scale;    // 1 / tau; log2(e) / tau
    float soft, hard;      // (1 - hard) tau^2; hard
    float dsoft;           // (1 - hard) tau
    float inv_v, inv_k;
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
    const int t = (int)(row / a.B);
    if (a.lengths && t >= a.lengths[row - (long long)t * a.B]) return 0.f;
    return a.weight ? a.weight[t] : a.weight_all;
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

// What a row's factors are made of: the others' maximum m and sum(s), the listed
// tokens' xm and sums, the teacher's.  (Sums relative to exp(max).)
struct RowStats {
    float ma;        // maximum of the row
    float sa, ha;    // sums over the row relative to it: / tau, plain
    float other;     // log q_rest
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
    r.other = (mo - r.ma) * a.inv_t + logf(s) - logf(r.sa);
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
// V <= 128: LPR lanes share a row, a wave takes 64 / LPR rows through LDS.  A row
// of 60 is 240 bytes: what counts is the number of instructions per row, and
// here the reductions over the row are over LPR lanes (two DPP steps) instead of
// 64.  The listed tokens are read out of the tile and replaced by -inf, so the
// passes over the row see the others only; their gradients go back into it
// and the tile leaves in one lane-linear range.
template <int DT, int LPR, bool HARD>
__global__ __launch_bounds__(64) void distill_short_kernel(DistillArgs a) {
    typedef RowType<DT> R;
    constexpr int ROWS = 64 / LPR;
    extern __shared__ float sm[];
    const int lane = threadIdx.x, r = lane / LPR, sub = lane % LPR;
    const int V = a.V, k = a.k, LD = V | 1, LK = k | 1;
    float *tile = sm;                         // [ROWS][LD]
    float *s_u = tile + ROWS * LD;            // [ROWS][LK]: u, then p
    float *s_x = s_u + ROWS * LK;             // [ROWS][LK]: listed logits
    int *s_i = (int *)(s_x + ROWS * LK);      // [ROWS][LK]: index; -1: absent; -2 - index:
                                              // an earlier entry has it
    unsigned *s_m = (unsigned *)(s_i + ROWS * LK);   // [ROWS][4] marks
    float *s_w = (float *)(s_m + ROWS * 4);   // [ROWS]
    const long long row0 = (long long)blockIdx.x * ROWS;
    const int nrows = (int)min((long long)ROWS, a.rows - row0);
    const long long row = row0 + r;
    const float w = r < nrows ? row_weight(a, row) : 0.f;
    if (sub == 0) s_w[r] = w;
    for (int i = lane; i < ROWS * 4; i += 64) s_m[i] = 0;
    __syncthreads();
    const typename R::T *x = (const typename R::T *)a.logits + row0 * a.ld;
    const int n = nrows * V;
    for (int i = lane; i < n; i += 64) {
        const int rr = pcm_fdiv(i, a.inv_v), c = i - rr * V;
        if (s_w[rr] != 0.f) tile[rr * LD + c] = R::up(x[(long long)rr * a.ld + c]);
    }
    for (int i = lane; i < nrows * k; i += 64) {
        const int rr = pcm_fdiv(i, a.inv_k), c = i - rr * k;
        if (s_w[rr] != 0.f) {
            const long long at = row0 * k + i;
            const int idx = teacher_index(a, at);
            s_i[rr * LK + c] = idx;
            s_u[rr * LK + c] =
                idx < 0 ? -INFINITY : teacher_value(a, at) * a.inv_t;
        }
    }
    __syncthreads();
    const bool live = w != 0.f;
    float *t = tile + r * LD, *u = s_u + r * LK, *lx = s_x + r * LK;
    int *li = s_i + r * LK;
    const float rest = live && a.rest ? a.rest[row] : -INFINITY;
    const int tg = live && HARD ? target_of(a, row, sub == 0) : -1;
    float xt = 0.f, um = rest;
    bool bad = rest != rest, twice = false;
    if (live) {
        if (HARD) xt = t[tg];
        for (int j = sub; j < k; j += LPR) {
            const int idx = li[j];
            um = fmaxf(um, u[j]);
            bad |= u[j] != u[j];
            lx[j] = idx < 0 ? -INFINITY : t[idx];
            if (idx >= 0) {
                const unsigned bit = 1u << (idx & 31);
                twice |= (atomicOr(&s_m[r * 4 + (idx >> 5)], bit) & bit) != 0;
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) {   // over the row's lanes
        const float ou = o == 1 ? lane_xor<1>(um) : lane_xor<2>(um);
        um = fmaxf(um, ou);
        const int f = (bad ? 1 : 0) | (twice ? 2 : 0);
        const int of = f | (o == 1 ? lane_xor<1>(f) : lane_xor<2>(f));
        bad = of & 1;
        twice = of & 2;
    }
    if (live && twice && sub == 0)   // rare: only the first entry stands for it
        for (int j = 1; j < k; ++j)
            for (int i = 0; i < j; ++i)
                if (li[j] >= 0 && li[i] == li[j]) {
                    li[j] = -2 - li[j];
                    break;
                }
    __syncthreads();
    // teacher and the listed tokens' part of the student
    const bool taught = um > -INFINITY || bad;
    const float uo = finite_or_0(um);
    float us = 0.f, xm = -INFINITY, xs = 0.f, xh = 0.f;
    if (live)
        for (int j = sub; j < k; j += LPR) {
            us += __builtin_amdgcn_exp2f((u[j] - uo) * LOG2E);
            if (li[j] >= 0) {
                xm = fmaxf(xm, lx[j]);
                t[li[j]] = -INFINITY;
            }
        }
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) {
        xm = fmaxf(xm, o == 1 ? lane_xor<1>(xm) : lane_xor<2>(xm));
        us += o == 1 ? lane_xor<1>(us) : lane_xor<2>(us);
    }
    const float ro = __builtin_amdgcn_exp2f((rest - uo) * LOG2E);
    us += ro;
    const float pr = taught ? ro / us : 0.f, lus = logf(us);
    const float xo = finite_or_0(xm);
    __syncthreads();
    float m = -INFINITY;
    if (live) {
        for (int j = sub; j < k; j += LPR)
            if (li[j] >= 0) {
                xs += exp_below(lx[j], xo, a.scale);
                if (HARD) xh += exp_below(lx[j], xo, LOG2E);
            }
        for (int v = sub; v < V; v += LPR) m = fmaxf(m, t[v]);
    }
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) {
        m = fmaxf(m, o == 1 ? lane_xor<1>(m) : lane_xor<2>(m));
        xs += o == 1 ? lane_xor<1>(xs) : lane_xor<2>(xs);
        if (HARD) xh += o == 1 ? lane_xor<1>(xh) : lane_xor<2>(xh);
    }
    const float mo = finite_or_0(m);
    float s = 0.f, h = 0.f;
    if (live)
        for (int v = sub; v < V; v += LPR) {
            s += exp_below(t[v], mo, a.scale);
            if (HARD) h += exp_below(t[v], mo, LOG2E);
        }
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) {
        s += o == 1 ? lane_xor<1>(s) : lane_xor<2>(s);
        if (HARD) h += o == 1 ? lane_xor<1>(h) : lane_xor<2>(h);
    }
    const RowStats st = row_stats(a, w, m, s, h, xm, xs, xh, taught, pr);
    const float lsa = logf(st.sa);
    // the row's loss
    float kl = 0.f;
    if (live && taught) {
        for (int j = sub; j < k; j += LPR) {
            const float p = __builtin_amdgcn_exp2f((u[j] - uo) * LOG2E) / us;
            if (!(p == 0.f))
                kl += p * ((u[j] - uo - lus) -
                           ((lx[j] - st.ma) * a.inv_t - lsa));
            if (a.dlogits) u[j] = p;
        }
        if (sub == 0 && !(pr == 0.f)) kl += pr * ((rest - uo - lus) - st.other);
    }
    float loss = a.soft * kl;
    if (HARD && live && sub == 0)
        loss += a.hard * (logf(st.ha) - (xt - st.ma));
    loss = wave_sum(live ? loss * w : 0.f);
    if (lane == 0) a.rowloss[blockIdx.x] = loss;
    if (!a.dlogits) return;
    // gradients into the tile: the others, the listed ones, their teacher's part
    if (live)
        for (int v = sub; v < V; v += LPR) {
            float g = exp_below(t[v], mo, a.scale) * st.cq;
            if (HARD) g += exp_below(t[v], mo, LOG2E) * st.ch;
            t[v] = g;
        }
    __syncthreads();
    if (live) {
        const float cs = taught ? a.dsoft * w : 0.f;
        for (int j = sub; j < k; j += LPR)
            if (li[j] >= 0) {
                float g = cs * exp_below(lx[j], st.ma, a.scale) / st.sa;
                if (HARD)
                    g += a.hard * w * exp_below(lx[j], st.ma, LOG2E) / st.ha;
                if (!twice && taught) g -= cs * u[j];
                t[li[j]] = g;
            }
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    if (live && sub == 0) {
        if (twice && taught)
            for (int j = 0; j < k; ++j) {
                const int idx = li[j] >= -1 ? li[j] : -2 - li[j];
                if (idx >= 0) t[idx] -= a.dsoft * w * u[j];
            }
        if (HARD) t[tg] -= a.hard * w;
    }
    __syncthreads();
    typename R::T *dl = (typename R::T *)a.dlogits + row0 * V;
    for (int i = lane; i < n; i += 64) {
        const int rr = pcm_fdiv(i, a.inv_v), c = i - rr * V;
        dl[i] = R::down(s_w[rr] != 0.f ? tile[rr * LD + c] : 0.f);
    }
}

// ---- longer rows ----------------------------------------------------------------
// One block per row.  KEEP: the row stays in registers, read once and written
// once; else (rows beyond 65536) it is read again for every pass.  Wave 0 holds
// the list, one entry per lane; the listed tokens are marked in a bitmap in LDS
// -- a group of eight elements is one byte of it -- and become -inf in the
// registers, so the passes see the others only.
template <int DT, int NT, int G, bool HARD, bool KEEP>
__global__ __launch_bounds__(NT, KEEP ? row_waves(DT, NT, G) : 8) void
distill_row_kernel(DistillArgs a) {
    typedef RowType<DT> R;
    typedef typename R::T T;
    extern __shared__ unsigned marks[];   // a bit per element
    __shared__ float red[NT / 64], red2[NT / 64];
    __shared__ float s_list[6];
    const int tid = threadIdx.x, lane = tid & 63;
    const long long row = blockIdx.x;
    const int V = a.V, k = a.k;
    const float w = row_weight(a, row);
    T *dl = a.dlogits ? (T *)a.dlogits + row * V : nullptr;
    const int groups = KEEP ? G : (V + NT * 8 - 1) / (NT * 8);
    if (w == 0.f) {
        if (tid == 0) a.rowloss[row] = 0.f;
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
    // the list: lane j of wave 0 holds entry j
    int idx = -1, tg = -1;
    float u = -INFINITY, lx = -INFINITY, xt = 0.f, rest = -INFINITY;
    if (tid < 64) {
        if (a.rest) rest = a.rest[row];
        if (HARD) {
            tg = target_of(a, row, lane == 0);
            xt = R::up(x[tg]);
        }
        if (lane < k) {
            idx = teacher_index(a, row * k + lane);
            if (idx >= 0) {
                u = teacher_value(a, row * k + lane) * a.inv_t;
                lx = R::up(x[idx]);
            }
        }
    }
    const int words = groups * NT / 4;   // groups * NT bytes
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
    auto group = [&](int g, Row8<DT> &q) {   // group g without the listed tokens
        if (!KEEP) {
            const int e = (g * NT + tid) * 8;
            q.lowest();
            if (e + 8 <= V) q.load(x + e);
            else {
#pragma unroll
                for (int j = 0; j < 7; ++j)
                    if (e + j < V) q.set(j, x[e + j]);
            }
        }
        const unsigned bits = mark8[g * NT + tid];
        if (bits) q.drop(bits);
    };
    if (KEEP) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
            regs.r[g].touch();
            group(g, regs.r[g]);
#pragma unroll
            for (int j = 0; j < 8; ++j) m = fmaxf(m, regs.r[g].get(j));
        }
    } else {
        for (int g = 0; g < groups; ++g) {
            Row8<DT> q;
            group(g, q);
#pragma unroll
            for (int j = 0; j < 8; ++j) m = fmaxf(m, q.get(j));
        }
    }
    float p = 0.f, mass = 0.f, logp = 0.f, logpr = 0.f;
    if (tid < 64) {
        if (__any(idx >= 0 && !first)) {   // rare: an index that appears twice
            bool again = false;
            for (int j = 0; j < k; ++j) {
                const int ij = __builtin_amdgcn_readlane(idx, j);
                again |= j < lane && ij == idx;
            }
            first = idx >= 0 && !again;
        }
        const float um = wave_max(fmaxf(u, rest));
        const bool bad = __any(u != u || rest != rest);
        const bool taught = um > -INFINITY || bad;
        const float uo = finite_or_0(um);
        const float e = __builtin_amdgcn_exp2f((u - uo) * LOG2E);
        const float ro = __builtin_amdgcn_exp2f((rest - uo) * LOG2E);
        const float us = wave_sum(e) + ro, lus = logf(us);
        if (taught) p = e / us;
        logp = u - uo - lus;
        logpr = rest - uo - lus;
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
        if (lane == 0) {
            s_list[0] = xm;
            s_list[1] = xs;
            s_list[2] = xh;
            s_list[3] = taught ? 1.f : 0.f;
            s_list[4] = taught ? ro / us : 0.f;
        }
    }
    m = all_max<NT>(m, red, tid);
    const float mo = finite_or_0(m);
    float s = 0.f, h = 0.f;
    auto add = [&](const Row8<DT> &q) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float d = q.get(j) - mo;
            s += __builtin_amdgcn_exp2f(d * a.scale);
            if (HARD) h += __builtin_amdgcn_exp2f(d * LOG2E);
        }
    };
    if (KEEP) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
            regs.r[g].touch();
            add(regs.r[g]);
        }
    } else {
        for (int g = 0; g < groups; ++g) {
            Row8<DT> q;
            group(g, q);
            add(q);
        }
    }
    s = all_sum<NT>(s, red2, tid);
    if (HARD) h = all_sum<NT>(h, red, tid);
    __syncthreads();   // s_list
    const bool taught = s_list[3] != 0.f;
    const float pr = s_list[4];
    const RowStats st = row_stats(a, w, m, s, h, s_list[0], s_list[1], s_list[2],
                                  taught, pr);
    if (tid < 64) {
        const float lsa = logf(st.sa);
        float kl = 0.f;
        if (!(p == 0.f)) kl = p * (logp - ((lx - st.ma) * a.inv_t - lsa));
        if (lane == 0 && !(pr == 0.f)) kl += pr * (logpr - st.other);
        float loss = a.soft * wave_sum(kl);
        if (HARD) loss += a.hard * (logf(st.ha) - (xt - st.ma));
        if (lane == 0) a.rowloss[row] = loss * w;
    }
    if (!dl) return;
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
    } else {
        for (int g = 0; g < groups; ++g) {
            Row8<DT> q;
            group(g, q);
            write(g, q);
        }
    }
    __syncthreads();   // the listed tokens and the target over what is there
    if (tid < 64) {
        if (first) {
            float g = 0.f;
            if (taught)
                g = a.dsoft * w * (exp_below(lx, st.ma, a.scale) / st.sa - mass);
            if (HARD) {
                g += a.hard * w * exp_below(lx, st.ma, LOG2E) / st.ha;
                if (idx == tg) g -= a.hard * w;
            }
            dl[idx] = R::down(g);
        }
        if (HARD && lane == 0 && !(marks[tg >> 5] >> (tg & 31) & 1)) {
            const float d = xt - mo;
            dl[tg] = R::down(__builtin_amdgcn_exp2f(d * a.scale) * st.cq +
                             __builtin_amdgcn_exp2f(d * LOG2E) * st.ch -
                             a.hard * w);
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
template <int DT, bool HARD>
long long launch_rows(const DistillArgs &a, hipStream_t st) {
    const int V = a.V;
    if (V <= 128) {
        constexpr int LPR = 4, ROWS = 64 / LPR;
        const long long blocks = (a.rows + ROWS - 1) / ROWS;
        const size_t lds =
            (size_t)ROWS * ((V | 1) + 3 * (a.k | 1) + 5) * sizeof(float);
        hipLaunchKernelGGL((distill_short_kernel<DT, LPR, HARD>),
                           dim3((unsigned)blocks), dim3(64), lds, st, a);
        return blocks;
    }
#define PCM_DISTILL_ROWS(NT, G)                                             \
    hipLaunchKernelGGL((distill_row_kernel<DT, NT, G, HARD, true>),          \
                       dim3((unsigned)a.rows), dim3(NT), (size_t)(NT) * (G), \
                       st, a)
    if (V <= 512) PCM_DISTILL_ROWS(64, 1);
    else if (V <= 1024) PCM_DISTILL_ROWS(64, 2);
    else if (V <= 2048) PCM_DISTILL_ROWS(256, 1);
    else if (V <= 4096) PCM_DISTILL_ROWS(256, 2);
    else if (V <= 8192) PCM_DISTILL_ROWS(256, 4);
    else if (V <= 16384) PCM_DISTILL_ROWS(512, 4);
    else if (V <= 32768) PCM_DISTILL_ROWS(1024, 4);
    else if (V <= 65536) PCM_DISTILL_ROWS(1024, 8);
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

int pcm_distill_loss(const void *logits, int32_t dtype, int64_t ld,
                     const void *values, int32_t values_dtype,
                     const int32_t *indices, const float *rest, int32_t k,
                     const int64_t *targets, const int32_t *lengths,
                     const float *step_weight, int32_t steps, int32_t batch,
                     int32_t vocab, double temperature, double hard_weight,
                     float *loss, void *dlogits, float *scratch,
                     int32_t *status, void *stream) {
    PCM_API_GUARD;
    PCM_REQUIRE(logits && values && indices && loss && scratch, PCM_EINVAL,
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
    PCM_REQUIRE(temperature > 1e-30 && temperature < 1e30, PCM_EINVAL,
                "distill_loss: temperature must be positive");
    PCM_REQUIRE(hard_weight >= 0. && hard_weight <= 1., PCM_EINVAL,
                "distill_loss: hard_weight=%f outside 0..1", hard_weight);
    PCM_REQUIRE(hard_weight == 0. || targets, PCM_EINVAL,
                "distill_loss: hard_weight needs targets");
    hipStream_t st = (hipStream_t)stream;
    DistillArgs a;
    a.logits = logits; a.values = values; a.indices = indices; a.rest = rest;
    a.targets = targets; a.lengths = lengths; a.dlogits = dlogits;
    a.status = status;
    a.rows = (long long)steps * batch;
    a.rowloss = scratch;
    a.ld = ld; a.B = batch; a.V = vocab; a.k = k;
    a.values_dtype = values_dtype;
    a.weight = step_weight;
    a.weight_all = 1.0f / (float)batch;
    a.inv_t = (float)(1.0 / temperature);
    a.scale = (float)(1.4426950408889634 / temperature);
    a.soft = (float)((1.0 - hard_weight) * temperature * temperature);
    a.dsoft = (float)((1.0 - hard_weight) * temperature);
    a.hard = (float)hard_weight;
    a.inv_v = 1.0f / (float)vocab;
    a.inv_k = 1.0f / (float)k;
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
    hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, st,
                       a.rowloss, sums, loss);
    return pcm_check_launch("distill_loss");
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
