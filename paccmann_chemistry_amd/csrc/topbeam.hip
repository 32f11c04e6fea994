// Top logits of a row, the selection of a beam search over beams and
// vocabulary, and the reordering of the beams' states.
#include "rows.h"
#include "topbeam.h"

namespace {

// ---- the largest of a stretch -------------------------------------------------------
// NT threads find the k <= 64 largest keys of n elements in one pass over memory
// and a second look at the few threads that hold them.  Only elements above
// -inf are looked at (NaN is not): where there are fewer than k of them the caller
// fills up.
//   1. in the pass every thread keeps its maximum and the group of eight where
//      it first appeared: the key (maximum, last index of that group) is not above
//      the thread's largest one.  The threads form 64 (k > 32: 128) teams, one
//      lane of every (other) wave each; the k-th largest of the teams' largest
//      keys is a bound that k elements reach at least, and not many more: with
//      random data an element in 64 ln 2 / k teams' shares does, 44 for k = 32.
//      It costs one sort of 64 keys (two), in registers.  (A single wave sorts
//      its lanes' keys, or both halves of their groups');
//   2. the threads whose own key reaches it hold all of those elements (groups
//      are disjoint stretches).  A wave reads such a thread's elements again, one
//      per lane, and appends those at or above the bound to a list in LDS (ONE:
//      a thread has a single group, still in its registers, and does so itself);
//   3. the list is sorted, 64 at a time.
// Keys are distinct, so the order in 2 does not matter, and ties take no special
// path.  A list that overflows (few teams hold most of the large elements) is
// made by k passes instead.
// (64 threads, 512 elements: fewer threads than k may hold all of them)
constexpr int top_room(int nt) { return nt == 64 ? 512 : 1024; }
template <int NT> struct TopLds {
    double list[NT / 64][64];
    double buf[top_room(NT)];
    double bound;
    int held[NT];    // threads that reach the bound
    int holders, count;
};

// element of thread `holder` that `lane` looks at when a wave reads eight of its
// groups from g0 on
template <int NT>
__device__ __forceinline__ int held_at(int g0, int holder, int lane) {
    return ((g0 + (lane >> 3)) * NT + holder) * 8 + (lane & 7);
}
// Holders that a wave reads again: of the SPAN from h0 on, those at h0 + wave,
// h0 + wave + NT / 64, ...; sixteen groups each (two elements per lane), all
// loads in flight at once.  Longer stretches are read where they are needed.
template <int DT, int NT> struct Held {
    static constexpr int N = 4096 / NT, SPAN = 64;
    float v[N][2];
    static __device__ __forceinline__ bool fits(int n) { return n <= NT * 128; }
    __device__ __forceinline__ void load(const typename RowType<DT>::T *p, int n,
                                         const TopLds<NT> &lds, int h0,
                                         int holders, int lane, int wave) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int h = h0 + wave + i * (NT / 64);
            if (h < holders) {
                const int holder = lds.held[h];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int e = held_at<NT>(t * 8, holder, lane);
                    v[i][t] = e < n ? RowType<DT>::up(p[e]) : -INFINITY;
                }
            }
        }
    }
};

// the 64 largest of the first `lists` waves' sorted lists; in wave 0 afterwards
template <int NT>
__device__ __forceinline__ double merge_waves(double v, double (*list)[64],
                                              int lists, int lane, int wave) {
    if constexpr (NT > 64) {
        for (int s = NT / 128; s > 0; s >>= 1) {
            if (s >= lists) continue;
            if (wave >= s && wave < 2 * s) list[wave][lane] = v;
            __syncthreads();
            if (wave < s)
                v = key_merge(fmax(v, list[wave + s][63 - lane]), lane);
        }
    }
    return v;
}

// sorted top 64 of n keys in memory (LDS or global; SORTED: every 64 of them are);
// in wave 0 afterwards
template <int NT, bool SORTED = false>
__device__ __forceinline__ double top_of_list(const double *keys, int n,
                                              double (*list)[64], int lane,
                                              int wave) {
    double v = KEY_NONE;
    for (int c = wave * 64; c < n; c += NT) {
        double x = c + lane < n ? keys[c + lane] : KEY_NONE;
        if (!SORTED) x = key_sort(x, lane);
        // both descending: turn one around
        const double turned = __shfl(x, 63 - lane, 64);
        v = c == wave * 64 ? x : key_merge(fmax(v, turned), lane);
    }
    if (n > 64) v = merge_waves<NT>(v, list, (n + 63) / 64, lane, wave);
    return v;
}

// the k-th largest of the teams' largest keys, known to all
template <int NT>
__device__ __forceinline__ double bound_of(double key, int k, TopLds<NT> &lds,
                                           int lane, int wave) {
    lds.list[wave][lane] = key;
    __syncthreads();
    const bool two = k > 32;
    if (wave < (two ? 2 : 1)) {
        // 64 teams: lane l of all waves; 128: of the even, of the odd waves
#pragma unroll
        for (int w = 0; w < NT / 64; ++w)
            if (!two || (w & 1) == wave) key = fmax(key, lds.list[w][lane]);
        key = key_sort(key, lane);
    }
    if (two) {
        __syncthreads();
        if (wave == 1) lds.list[1][lane] = key;
        __syncthreads();
        if (wave == 0) key = key_merge(fmax(key, lds.list[1][63 - lane]), lane);
    }
    if (wave == 0 && lane == k - 1) lds.bound = key;
    __syncthreads();   // (and lds.count; the lists are free again)
    return lds.bound;
}

// Steps 1 (from the threads' maxima on) to 3.  bv, bg: the thread's maximum and
// the group where it first appeared.  Returns in wave 0: lane j holds the j-th
// largest key (KEY_NONE past `found`).  `slot`: the thread's place among the
// holders, -1 if it holds none of the k largest.
template <int DT, int NT, bool ONE>
__device__ __forceinline__ double top_of_threads(
    const typename RowType<DT>::T *p, const Row8<DT> &q, int n, int first, int k,
    float bv, int bg, TopLds<NT> &lds, Held<DT, NT> &held, int tid, int &found,
    int &slot) {
    typedef RowType<DT> R;
    const int lane = tid & 63, wave = tid >> 6;
    if (tid == 0) lds.count = lds.holders = 0;
    double key = bv > -INFINITY ? key_of(bv, first + (bg * NT + tid) * 8 + 7)
                                : KEY_NONE;
    double bound;
    if constexpr (NT == 64) {
        // a wave has a key per lane, or (k > 32) one for each half of a group;
        // of 128 elements all are candidates
        if (n <= 128) {
            bound = KEY_NONE;
        } else if (k <= 32) {
            bound = key_lane(key_sort(key, lane), k - 1);
        } else {
            double half[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float v = -INFINITY;
#pragma unroll
                for (int j = 0; j < 4; ++j) v = fmaxf(v, q.get(4 * i + j));
                half[i] = v > -INFINITY ? key_of(v, first + tid * 8 + 4 * i + 3)
                                        : KEY_NONE;
            }
            key = fmax(half[0], half[1]);
            half[0] = key_sort(half[0], lane);
            half[1] = __shfl(key_sort(half[1], lane), 63 - lane, 64);
            bound = key_lane(key_merge(fmax(half[0], half[1]), lane), k - 1);
        }
        __syncthreads();   // lds.count
    } else {
        bound = bound_of<NT>(key, k, lds, lane, wave);
    }
    const float bound_v = bound == KEY_NONE ? -INFINITY : key_value(bound);
    slot = -1;
    if (key > KEY_NONE && key >= bound) {
        if (ONE) {
            slot = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float v = q.get(j);
                if (v >= bound_v && v > -INFINITY) {
                    const double ek = key_of(v, first + tid * 8 + j);
                    if (ek >= bound) {
                        const int at = atomicAdd(&lds.count, 1);
                        if (at < top_room(NT)) lds.buf[at] = ek;
                    }
                }
            }
        } else {
            slot = atomicAdd(&lds.holders, 1);
            lds.held[slot] = tid;
        }
    }
    __syncthreads();
    const int holders = lds.holders;   // (ONE: 0)
    auto append = [&](float v, int e) {
        if (v >= bound_v && v > -INFINITY) {
            const double ek = key_of(v, first + e);
            if (ek >= bound) {
                const int at = atomicAdd(&lds.count, 1);
                if (at < top_room(NT)) lds.buf[at] = ek;
            }
        }
    };
    typedef Held<DT, NT> H;
    if (ONE) {
    } else if (H::fits(n)) {
        for (int h0 = 0; h0 < holders; h0 += H::SPAN) {
            held.load(p, n, lds, h0, holders, lane, wave);
#pragma unroll
            for (int i = 0; i < H::N; ++i) {
                const int h = h0 + wave + i * (NT / 64);
                if (h < holders) {
                    const int holder = lds.held[h];
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        append(held.v[i][t], held_at<NT>(t * 8, holder, lane));
                }
            }
        }
    } else {
        for (int i = wave; i < holders; i += NT / 64) {
            const int holder = lds.held[i];
            for (int g0 = 0; g0 * NT * 8 < n; g0 += 8) {
                const int e = held_at<NT>(g0, holder, lane);
                append(e < n ? R::up(p[e]) : -INFINITY, e);
            }
        }
    }
    __syncthreads();
    found = lds.count;
    if (found > top_room(NT)) {
        double prev = __builtin_inf();
        for (int j = 0; j < k; ++j) {
            double best = KEY_NONE;
            for (int g = 0; g * NT * 8 < n; ++g)
                for (int i = 0; i < 8; ++i) {
                    const int e = (g * NT + tid) * 8 + i;
                    if (e >= n) break;
                    const float v = R::up(p[e]);
                    const double ek = key_of(v, first + e);
                    if (v > -INFINITY && ek < prev && ek > best) best = ek;
                }
            prev = all_max<NT>(best, &lds.list[0][0], tid);
            if (tid == 0) lds.buf[j] = prev;
        }
        __syncthreads();
        found = k;   // (there were more than that)
    }
    return top_of_list<NT>(lds.buf, found, lds.list, lane, wave);
}

// ---- the largest of a short row ---------------------------------------------------
// LPR lanes share a row; each sorts its groups of eight (19 comparators of two
// instructions, v_max_f64 and v_min_f64), merges them into a list of KT, then the
// lanes' lists are merged pairwise; every lane ends with the row's list.  A row
// of 60 costs about 40 instructions of a wave this way (16 rows in it) against
// 800 for a wave per row.  All elements are ranked, -inf and NaN too.  Top 8 of
// 61440 x 60 fp32: 11.6 us (70 for a wave per row), 18.9 MB at 1.6 TB/s: bound by
// the comparators in 64 bits and, at four waves per SIMD, by waiting for the loads;
// bf16 10.0, fp16 10.5.
template <int KT> struct ShortTop {
    double l[KT];
    static __device__ __forceinline__ void order(double &a, double &b) {
        const double hi = fmax(a, b);
        b = fmin(a, b);
        a = hi;
    }
    static __device__ __forceinline__ void sort8(double (&g)[8]) {
        constexpr int net[19][2] = {
            {0, 1}, {2, 3}, {4, 5}, {6, 7}, {0, 2}, {1, 3}, {4, 6},
            {5, 7}, {1, 2}, {5, 6}, {0, 4}, {3, 7}, {1, 5}, {2, 6},
            {1, 4}, {3, 6}, {2, 4}, {3, 5}, {3, 4}};
#pragma unroll
        for (int i = 0; i < 19; ++i) order(g[net[i][0]], g[net[i][1]]);
    }
    // l is bitonic: sort it
    __device__ __forceinline__ void settle() {
#pragma unroll
        for (int s = KT / 2; s > 0; s >>= 1)
#pragma unroll
            for (int j = 0; j < KT; ++j)
                if ((j & s) == 0) order(l[j], l[j + s]);
    }
    // the list and a sorted group: its largest meet the list's smallest
    __device__ __forceinline__ void take(const double (&g)[8]) {
        constexpr int N = KT < 8 ? KT : 8;
#pragma unroll
        for (int j = 0; j < N; ++j)
            l[KT - 1 - j] = fmax(l[KT - 1 - j], g[j]);
        settle();
    }
    template <int M> __device__ __forceinline__ void merge() {
        double o[KT];
#pragma unroll
        for (int j = 0; j < KT; ++j) o[j] = lane_xor<M>(l[j]);
#pragma unroll
        for (int j = 0; j < KT; ++j) l[j] = fmax(l[j], o[KT - 1 - j]);
        settle();
    }
    template <int DT, int LPR, int G>
    __device__ __forceinline__ void of(const RowRegs<DT, LPR, G> &x, int V,
                                       int sub) {
#pragma unroll
        for (int j = 0; j < KT; ++j) l[j] = KEY_NONE;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            double e[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int at = x.at(g, sub) + j;
                const double key = key_of(x.r[g].get(j), at);
                e[j] = at < V ? key : KEY_NONE;
            }
            sort8(e);
            if (g == 0) {
#pragma unroll
                for (int j = 0; j < (KT < 8 ? KT : 8); ++j) l[j] = e[j];
            } else {
                take(e);
            }
        }
        merge<1>();
        merge<2>();
        if constexpr (LPR == 16) {
            merge<4>();
            merge<8>();
        }
    }
};
// run the call with the constants LPR (lanes per row), G (groups of eight per
// lane) and KT (list) for short rows.  Four lanes share a row of at most 128 where
// there are enough rows to fill the chip with a wave for 16 of them, else sixteen.
#define PCM_BY_SHORT_LIST(k, ...)                                     \
    do {                                                              \
        if ((k) <= 4) { constexpr int KT = 4; __VA_ARGS__; }          \
        else if ((k) <= 8) { constexpr int KT = 8; __VA_ARGS__; }     \
        else { constexpr int KT = 16; __VA_ARGS__; }                  \
    } while (0)
#define PCM_BY_SHORT(rows, V, k, ...)                                         \
    do {                                                                      \
        if ((V) <= 128 && (rows) < 8192) {                                    \
            constexpr int LPR = 16, G = 1; PCM_BY_SHORT_LIST(k, __VA_ARGS__); \
        } else if ((V) <= 64) {                                               \
            constexpr int LPR = 4, G = 2; PCM_BY_SHORT_LIST(k, __VA_ARGS__);  \
        } else if ((V) <= 128) {                                              \
            constexpr int LPR = 4, G = 4; PCM_BY_SHORT_LIST(k, __VA_ARGS__);  \
        } else if ((V) <= 512) {                                              \
            constexpr int LPR = 16, G = 4; PCM_BY_SHORT_LIST(k, __VA_ARGS__); \
        } else {                                                              \
            constexpr int LPR = 16, G = 8; PCM_BY_SHORT_LIST(k, __VA_ARGS__); \
        }                                                                     \
    } while (0)
// Rows of more than 128 only where there are many: sixteen lanes that share a row
// take 14 x 804 logits in 46 us, a block for each (and the join) in 13.
inline bool short_rows(long long rows, int V, int k) {
    return k <= 16 && (V <= 128 || (V <= 1024 && rows >= 8192));
}

// ---- top logits -------------------------------------------------------------------
struct TopArgs {
    const void *logits;
    void *values;
    int32_t *indices;
    float *rest;
    double *keys;        // split rows: [rows][parts][64]
    float *part;         // ... [rows][parts][2]: maximum and sum of the others
    long long ld;
    int V, k, parts, len;   // len: elements of one part
    float scale, inv_t;     // log2(e) / temperature; 1 / temperature
};

// A listed element as it is in its row x.  Its key holds a value; the sign of a zero
// and a NaN's payload are not in it, and these are read again.
template <int DT>
__device__ __forceinline__ typename RowType<DT>::T listed_value(
    const typename RowType<DT>::T *x, double key) {
    const float v = key_value(key);
    return fabsf(v) > 0.f ? RowType<DT>::down(v) : x[key_index(key)];
}

// Entries past the `found` numbers above -inf: the -inf ones by index, then the
// NaN by index.  One wave; rare.
template <int DT>
__device__ void top_fill(const typename RowType<DT>::T *x, int V, int have, int k,
                         typename RowType<DT>::T *values, int32_t *indices,
                         int lane) {
    typedef RowType<DT> R;
    for (int nan = 0; nan < 2 && have < k; ++nan)
        for (int c = 0; c < V && have < k; c += 64) {
            const int v = c + lane;
            const float xv = v < V ? R::up(x[v]) : 0.f;
            const bool hit = v < V && (nan ? xv != xv : xv == -INFINITY);
            const unsigned long long m = __ballot(hit);
            const int at = have + __popcll(m & ((1ull << lane) - 1));
            if (hit && at < k) {
                values[at] = x[v];
                indices[at] = v;
            }
            have += __popcll(m);
        }
}

__device__ __forceinline__ float top_rest(float m, float s, float inv_t) {
    if (s != s) return s;
    return isinf(m) ? m : m * inv_t + logf(s);
}

// Rows of at most 1024, lists of at most 16.
template <int DT, int LPR, int G, int KT>
__global__ __launch_bounds__(256) void top_short_kernel(TopArgs a, long long rows) {
    typedef RowType<DT> R;
    typedef typename R::T T;
    const int sub = threadIdx.x % LPR;
    const long long row =
        (long long)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
    if (row >= rows) return;   // (all lanes of a row)
    const T *logits = (const T *)a.logits + row * a.ld;
    RowRegs<DT, LPR, G> x;
    x.load(logits, a.V, sub);
    ShortTop<KT> top;
    top.template of<DT, LPR, G>(x, a.V, sub);
    T *values = (T *)a.values + row * a.k;
    int32_t *indices = a.indices + row * a.k;
    double last = top.l[0];
#pragma unroll
    for (int j = 0; j < KT; ++j)
        if (j < a.k) {
            last = top.l[j];
            if (j % LPR == sub) {
                values[j] = listed_value<DT>(logits, last);
                indices[j] = key_index(last);
            }
        }
    const float last_v = key_value(last);
    const int last_i = key_index(last);
    float m = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float v = x.r[g].get(j);
            nan |= v != v;
            if (v < last_v || (v == last_v && x.at(g, sub) + j > last_i))
                m = fmaxf(m, v);
        }
    m = row_max<LPR>(nan ? INFINITY : m);
    const float mm = isinf(m) ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float v = x.r[g].get(j);
            if (!(v > last_v || (v == last_v && x.at(g, sub) + j <= last_i)))
                s += __builtin_amdgcn_exp2f((v - mm) * a.scale);
        }
    s = row_sum<LPR>(s);
    if (sub == 0) a.rest[row] = top_rest(m, s, a.inv_t);
}

// One block per row, or per part of a row.  The sum of the others is taken in the
// same pass, by thread and over everything, relative to the thread's running
// maximum; a wave takes the sums of the threads that hold listed elements again,
// without those.  (The whole row's sum minus the listed ones' would lose what
// the others are when the list holds nearly all of it.)
// Top 32 of 1024 x 50021 bf16: 34 us (102.6 MB, 3.0 TB/s; 22 at the rate of a large
// copy), bound by the issue of vector instructions, which have 0.81 of the slots:
// 1526 per wave, about 700 of them in the pass (7 per element), the rest in the
// selection and the second look; k passes took 8.4 ms.  (The holders' sums without
// wave reductions, 250 instructions fewer, were level; why is not known.)  The same
// in fp32: 50 us (4.1 TB/s), memory.  Top 64 of three rows of 131071 fp16: 8.4 to 9.6 us in
// 31 blocks a row, and 4.9 to join them: latency.
template <int DT, int NT, bool ONE>
__global__ __launch_bounds__(NT, 8) void top_kernel(TopArgs a) {
    typedef RowType<DT> R;
    typedef typename R::T T;
    __shared__ TopLds<NT> lds;
    __shared__ float red[NT / 64], red2[NT / 64];
    __shared__ float s_m[ONE ? 1 : NT], s_s[ONE ? 1 : NT];   // by holder
    __shared__ double s_last;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const long long row = blockIdx.x / a.parts;
    const int part = (int)(blockIdx.x - row * a.parts), first = part * a.len;
    const int n = min(a.len, a.V - first);
    const T *x = (const T *)a.logits + row * a.ld, *p = x + first;
    auto exp_from = [&](float v, float shift) {
        return __builtin_amdgcn_exp2f((v - shift) * a.scale);
    };
    // (v - m first: a mask of the type's lowest value times scale need not be
    // finite, nor its rounding small)
    float m = -INFINITY, s = 0.f;
    int bg = 0;
    Row8<DT> own;
    auto pass = [&](const Row8<DT> &q, int g) {
        float v[8], gm = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = q.get(j);
            gm = fmaxf(gm, v[j]);
        }
        if (gm > m) {
            if (m > -INFINITY) s *= exp_from(m, gm);
            m = gm;
            bg = g;
        }
        const float mm = isinf(m) ? 0.f : m;
#pragma unroll
        for (int j = 0; j < 8; ++j) s += exp_from(v[j], mm);
    };
    if (ONE) {
        load_group(own, p, n, tid * 8);
        pass(own, 0);
    } else {
        each_group<DT, NT>(p, n, tid, pass);
    }
    int found, slot;
    Held<DT, NT> held;   // (afterwards: the last SPAN of them)
    const double key = top_of_threads<DT, NT, ONE>(
        p, own, n, first, a.k, m, bg, lds, held, tid, found, slot);
    if (tid < 64) {
        if (a.parts > 1) {
            a.keys[(row * a.parts + part) * 64 + lane] =
                lane < a.k ? key : KEY_NONE;
        } else {
            T *values = (T *)a.values + row * a.k;
            int32_t *indices = a.indices + row * a.k;
            if (lane < min(found, a.k)) {
                values[lane] = listed_value<DT>(x, key);
                indices[lane] = key_index(key);
            }
            if (found < a.k) top_fill<DT>(x, a.V, found, a.k, values, indices, lane);
        }
        if (lane == a.k - 1) s_last = key;
    }
    __syncthreads();
    // the holders' others: below the list's last (none if it is not full)
    const double last = s_last;
    const float last_v = last == KEY_NONE ? -INFINITY : key_value(last);
    const int last_i = last == KEY_NONE ? 0x7fffffff : key_index(last) - first;
    const int holders = lds.holders;   // (ONE: 0)
    auto is_other = [&](float v, int e) {
        return v < last_v || (v == last_v && e > last_i);
    };
    typedef Held<DT, NT> H;
    if (ONE) {
    } else if (H::fits(n)) {
        for (int h0 = 0; h0 < holders; h0 += H::SPAN) {
            if (holders > H::SPAN) held.load(p, n, lds, h0, holders, lane, wave);
#pragma unroll
            for (int i = 0; i < H::N; ++i) {
                const int h = h0 + wave + i * (NT / 64);
                if (h < holders) {
                    const int holder = lds.held[h];
                    float ov[2];
                    bool nan = false;
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const float v = held.v[i][t];
                        nan |= v != v;
                        ov[t] = is_other(v, held_at<NT>(t * 8, holder, lane))
                                    ? v : -INFINITY;
                    }
                    const float om = wave_max(fmaxf(ov[0], ov[1]));
                    const float mm = isinf(om) ? 0.f : om;
                    const float os =
                        wave_sum(exp_from(ov[0], mm) + exp_from(ov[1], mm));
                    nan = __any(nan);
                    if (lane == 0) {
                        s_m[h] = om;
                        s_s[h] = nan ? NAN : os;
                    }
                }
            }
        }
    } else {
        for (int i = wave; i < holders; i += NT / 64) {
            const int holder = lds.held[i];
            float om = -INFINITY, os = 0.f;
            bool nan = false;
            for (int g0 = 0; g0 * NT * 8 < n; g0 += 8) {
                const int e = held_at<NT>(g0, holder, lane);
                const float v = e < n ? R::up(p[e]) : -INFINITY;
                nan |= v != v;
                if (is_other(v, e)) om = fmaxf(om, v);
            }
            om = wave_max(om);
            const float mm = isinf(om) ? 0.f : om;
            for (int g0 = 0; g0 * NT * 8 < n; g0 += 8) {
                const int e = held_at<NT>(g0, holder, lane);
                const float v = e < n ? R::up(p[e]) : -INFINITY;
                if (is_other(v, e)) os += exp_from(v, mm);
            }
            os = wave_sum(os);
            nan = __any(nan);
            if (lane == 0) {
                s_m[i] = om;
                s_s[i] = nan ? NAN : os;
            }
        }
    }
    if (ONE) {
        if (slot >= 0) {
            m = -INFINITY;
            bool take[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float v = own.get(j);
                take[j] = v != v || is_other(v, tid * 8 + j);
                if (take[j]) m = fmaxf(m, v);
            }
            const float mm = isinf(m) ? 0.f : m;
            s = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (take[j]) s += exp_from(own.get(j), mm);
        }
    } else {
        __syncthreads();
        if (slot >= 0) {
            m = s_m[slot];
            s = s_s[slot];
        }
    }
    const float mx = all_max<NT>(m, red, tid);
    // (a thread without others has the sum 0, or NaN)
    s = all_sum<NT>(s == 0.f ? 0.f
                             : s * exp_from(isinf(m) ? 0.f : m,
                                            isinf(mx) ? 0.f : mx),
                    red2, tid);
    if (tid == 0) {
        if (a.parts > 1) {
            float *q = a.part + (row * a.parts + part) * 2;
            q[0] = mx;
            q[1] = s;
        } else {
            a.rest[row] = top_rest(mx, s, a.inv_t);
        }
    }
}

// Joins the parts of a row: their lists into one, what did not get into it and
// the parts' others into the row's.
template <int DT>
__global__ __launch_bounds__(1024) void top_join_kernel(TopArgs a) {
    typedef RowType<DT> R;
    typedef typename R::T T;
    __shared__ double list[16][64];
    __shared__ float red[16];
    __shared__ double s_last;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const long long row = blockIdx.x;
    const int n = a.parts * 64;
    const double *keys = a.keys + row * n;
    const double key = top_of_list<1024, true>(keys, n, list, lane, wave);
    if (wave == 0) {
        T *values = (T *)a.values + row * a.k;
        int32_t *indices = a.indices + row * a.k;
        const int found = __popcll(__ballot(key > KEY_NONE && lane < a.k));
        if (lane < found) {
            values[lane] = listed_value<DT>((const T *)a.logits + row * a.ld, key);
            indices[lane] = key_index(key);
        }
        if (found < a.k)
            top_fill<DT>((const T *)a.logits + row * a.ld, a.V, found, a.k,
                         values, indices, lane);
        if (lane == a.k - 1) s_last = key;
    }
    __syncthreads();
    const double last = s_last;
    float m = -INFINITY;
    for (int i = tid; i < n; i += 1024)
        if (keys[i] < last && keys[i] > KEY_NONE) m = fmaxf(m, key_value(keys[i]));
    if (tid < a.parts) m = fmaxf(m, a.part[(row * a.parts + tid) * 2]);
    m = all_max<1024>(m, red, tid);
    const float mm = isinf(m) ? 0.f : m;
    float s = 0.f;
    for (int i = tid; i < n; i += 1024)
        if (keys[i] < last && keys[i] > KEY_NONE)
            s += __builtin_amdgcn_exp2f((key_value(keys[i]) - mm) * a.scale);
    if (tid < a.parts) {
        const float *p = a.part + (row * a.parts + tid) * 2;
        const float pm = isinf(p[0]) ? 0.f : p[0];
        // (a part without others has the sum 0)
        if (p[1] != 0.f)
            s += p[1] * __builtin_amdgcn_exp2f((pm - mm) * a.scale);
    }
    s = all_sum<1024>(s, red, tid);
    if (tid == 0) a.rest[row] = top_rest(m, s, a.inv_t);
}

// ---- beam selection ---------------------------------------------------------------
struct BeamArgs {
    const void *logits;
    const double *scores;
    const uint8_t *finished;
    double *keys;       // [beams][batch][parts][width]
    double *part;       // [beams][batch][parts][2]: maximum, sum (64 bits)
    int64_t *tokens;
    int32_t *parents;
    double *scores_out;
    uint8_t *finished_out;
    long long ld;
    int beams, batch, V, width, parts, len, end;
    const int32_t *end_at;   // the end token on the device, or null: end
    double inv_t;         // 1 / temperature
    double scale, least;  // log2(e) / temperature; the difference 2^-1000 is of
};

// exp of logits relative to a maximum m (finite) in 64 bits, to a step of theirs:
// beams compete by the difference of two log-sum-exps, for which 32 bits are too
// few.  d = v - m first (of a product less a rounded product 3e38 times
// temperature leaves 1e22, of either sign); what is below 2^-1000 counts as that.
// d scale, rounded to the nearest integer n (by adding 1.5 * 2^52: n is then the
// low word too), leaves at most 1/2, where the polynomial of degree 10 with the
// least largest relative error (found by a Remez exchange) is off by 2.1e-16; n
// goes into the exponent's bits.  Additions and fused multiplications only.  (Of
// degree 8 it is off by 7.7e-13 and 1.1 us faster over 8 x 64 x 32000 logits.)
struct Exp64 {
    double scale, least, m;
    __device__ __forceinline__ Exp64(const BeamArgs &a, float m_)
        : scale(a.scale), least(a.least), m((double)m_) {}
    __device__ __forceinline__ double operator()(float v) const {
        const double big = 6755399441055744.0;
        const double d = fmax((double)v - m, least);
        const double r = fma(d, scale, big), f = fma(d, scale, -(r - big));
        double p = 7.0372783532743875056e-9;
        p = fma(p, f, 1.0208537941213722185e-7);
        p = fma(p, f, 1.3215662838955003129e-6);
        p = fma(p, f, 0.000015252658116348336923);
        p = fma(p, f, 0.00015403529961120784315);
        p = fma(p, f, 0.0013333558228561871466);
        p = fma(p, f, 0.0096181291080346023214);
        p = fma(p, f, 0.055504108664458830714);
        p = fma(p, f, 0.24022650695908767754);
        p = fma(p, f, 0.69314718055994977511);
        p = fma(p, f, 1.0);
        return __hiloint2double(__double2hiint(p) + (__double2loint(r) << 20),
                                __double2loint(p));
    }
};
// score of a candidate: the differences first here too (a row whose tokens all
// hold the type's lowest value is uniform)
__device__ __forceinline__ double beam_score(const BeamArgs &a, double score,
                                             float v, double m, double log_s) {
    return score + (((double)v - m) * a.inv_t - log_s);
}

__device__ __forceinline__ int end_token_of(const BeamArgs &a) {
    return a.end_at ? *a.end_at : a.end;
}

// The j-th candidate of a beam that has ended: end_token, then the others, which are
// -inf, in order; of one that holds no score all are, so all are in order.
__device__ __forceinline__ int ended_token(int end, int j, double score) {
    if (!(score > -INFINITY)) return j;
    return j == 0 ? end : j - 1 + (j - 1 >= end ? 1 : 0);
}

// Per beam row (or part of one): the `width` largest logits -- the row's
// normaliser does not change their order -- and its maximum and sum, in one
// pass.  8 x 64 rows of 32000 bf16: 24 us (26 MB; 19 operations in 64 bits per
// element are 11 us of it, the first loads and the selection most of the rest);
// four rows of 131071 in 31 blocks each: 7.5 us, latency.  5 x 256 rows of 129: 6.7 us,
// of 700: 7.9 (latency), of 5003: 22, of 8192 bf16: 24.
// (Long rows: 4 waves per SIMD, not 8, so that the eight exponentials in flight
// stay in registers; it is bound by 64-bit arithmetic, not by latency.)
template <int DT, int NT, bool ONE>
__global__ __launch_bounds__(NT, ONE ? 8 : 4) void beam_rows_kernel(BeamArgs a) {
    typedef typename RowType<DT>::T T;
    __shared__ TopLds<NT> lds;
    __shared__ float redf[NT / 64];
    __shared__ double red[NT / 64];
    const int tid = threadIdx.x, lane = tid & 63;
    const long long row = blockIdx.x / a.parts;
    const int part = (int)(blockIdx.x - row * a.parts), first = part * a.len;
    // (the join does not look at the rows of these)
    if (!(a.scores[row] > -INFINITY) || (a.finished && a.finished[row])) return;
    const int n = min(a.len, a.V - first);
    const T *p = (const T *)a.logits + row * a.ld + first;
    float m = -INFINITY;
    int bg = 0;
    bool nan = false;
    double s = 0.;
    Row8<DT> own;
    auto pass = [&](const Row8<DT> &q, int g) {
        float v[8], gm = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = q.get(j);
            gm = fmaxf(gm, v[j]);
            nan |= v[j] != v[j];
        }
        if (gm > m) {
            if (m > -INFINITY) s *= Exp64(a, gm)(m);
            m = gm;
            bg = g;
        }
        // (without any element above -inf yet, or with a +inf: not used)
        const Exp64 e(a, isinf(m) ? 0.f : m);
        double sum = 0.;
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += e(v[j]);
        if (m > -INFINITY) s += sum;
    };
    if (ONE) {
        load_group(own, p, n, tid * 8);
        pass(own, 0);
    } else {
        each_group<DT, NT>(p, n, tid, pass);
    }
    int found, slot;
    Held<DT, NT> held;   // (afterwards: the last SPAN of them)
    const double key = top_of_threads<DT, NT, ONE>(
        p, own, n, first, a.width, m, bg, lds, held, tid, found, slot);
    if (tid < a.width) a.keys[(row * a.parts + part) * a.width + lane] = key;
    const float mx = all_max<NT>(nan ? INFINITY : m, redf, tid);
    if (!isinf(mx))
        s = all_sum<NT>(m == -INFINITY ? 0. : s * Exp64(a, mx)(m), red, tid);
    if (tid == 0) {
        double *q = a.part + (row * a.parts + part) * 2;
        q[0] = mx;   // +inf: a NaN or +inf in this part, no distribution
        q[1] = isinf(mx) ? 0. : s;
    }
}

// Places of the candidates of `rows` batch rows from b0 on, [row][beam][width],
// every beam's own sorted: a candidate's place is the number of better ones,
// counted list by list from the top until one is not better (or `width` of them
// are): width + beams steps at most.  Lanes next to each other are of one batch
// row and mostly read the same entry.  An entry's flat place is 2 (beam V + token),
// plus 1 if the beam had ended (a load of `finished` here would be 0.3 us more).
__device__ __forceinline__ void beam_rank(const double *all_c, const int *all_f,
                                          const BeamArgs &a, int end, int rows,
                                          int b0) {
    const int W = a.width, n = a.beams * W;
    for (int at = threadIdx.x; at < rows * n; at += blockDim.x) {
        const int r = at / n, i = at - r * n, own = i / W;
        const double *c = all_c + r * n;
        const int *f = all_f + r * n;
        const double mine = c[i];
        const int flat = f[i];
        int place = i - own * W;
        for (int k = 0; k < a.beams && place < W; ++k) {
            if (k == own) continue;
            for (int j = k * W; j < (k + 1) * W && place < W; ++j) {
                if (!(c[j] > mine || (c[j] == mine && f[j] < flat))) break;
                ++place;
            }
        }
        if (place < W) {
            const int id = flat >> 1, from = id / a.V, t = id - from * a.V;
            const int b = b0 + r;
            const long long o = (long long)place * a.batch + b;
            a.tokens[o] = t;
            a.parents[o] = from;
            a.scores_out[o] = mine;
            if (a.finished_out)
                a.finished_out[o] = (flat & 1) || t == end;
        }
    }
}

// One block per batch row, one wave per beam: the beam's parts become `width`
// candidates with their scores, all of which are ranked by score, then beam and
// token.  A chain of latencies (the rows' results out of memory, a logarithm, two
// barriers): 6.0 us for one batch row of four beams in 31 parts, 8.0 for 64 of eight
// beams.
__global__ __launch_bounds__(1024) void beam_join_kernel(BeamArgs a) {
    __shared__ double s_c[PCM_BEAM_MAX * PCM_BEAM_MAX];
    __shared__ int s_f[PCM_BEAM_MAX * PCM_BEAM_MAX];
    const int lane = threadIdx.x & 63;
    const int k = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = blockIdx.x, W = a.width, end = end_token_of(a);
    const long long row = (long long)k * a.batch + b;
    // everything a beam needs is asked for at once (rows that are not looked at
    // hold whatever the workspace held)
    const double score = a.scores[row];
    const bool done = a.finished && a.finished[row];
    const double *keys = a.keys + row * a.parts * W;
    const double *part = a.part + row * a.parts * 2;
    const int n = a.parts * W;
    double key = lane < n ? keys[lane] : KEY_NONE;
    const double pm = lane < a.parts ? part[2 * lane] : -INFINITY;
    const double ps = lane < a.parts ? part[2 * lane + 1] : 0.;
    int tok = -1;
    double c = -INFINITY;
    if (done) {
        tok = ended_token(end, lane, score);
        if (lane == 0 && score > -INFINITY) c = score;
    } else {
        const double m = score > -INFINITY ? wave_max(pm) : -INFINITY;
        tok = lane;   // a row without a distribution: the tokens in order
        if (!isinf(m)) {
            const double s = wave_sum(
                ps > 0. ? ps * Exp64(a, (float)m)((float)pm) : 0.);
            const double log_s = log(s);
            if (a.parts > 1) key = key_sort(key, lane);
            for (int at = 64; at < n; at += 64) {
                const double x =
                    key_sort(at + lane < n ? keys[at + lane] : KEY_NONE, lane);
                key = key_merge(fmax(key, __shfl(x, 63 - lane, 64)), lane);
            }
            const bool real = key > KEY_NONE && lane < W;
            const int found = __popcll(__ballot(real));
            if (real) {
                tok = key_index(key);
                c = beam_score(a, score, key_value(key), m, log_s);
            } else if (lane < W) {
                // fewer tokens above -inf: the lowest ones that are not listed
                int want = lane - found, t = 0;
                for (;; ++t) {
                    bool listed = false;
                    for (int j = 0; j < found; ++j)
                        listed |= key_index(key_lane(key, j)) == t;
                    if (!listed && want-- == 0) break;
                    if (t >= 2 * PCM_BEAM_MAX) break;
                }
                tok = t;
            }
        }
    }
    if (lane < W) {
        s_c[k * W + lane] = c;
        s_f[k * W + lane] =
            tok < a.V ? 2 * (k * a.V + tok) + (done ? 1 : 0) : 0x7fffffff;
    }
    __syncthreads();
    beam_rank(s_c, s_f, a, end, 1, b);
}

// Short rows, everything in one launch: a block takes 64 / LPR batch rows, one
// wave per beam.  3 x 4096 x 60 fp32: 6.7 us (2.9 MB; one turn of 768 waves, bound by
// its latency).
template <int DT, int LPR, int G, int KT>
__global__ __launch_bounds__(1024) void beam_short_kernel(BeamArgs a) {
    typedef typename RowType<DT>::T T;
    constexpr int RB = 64 / LPR;
    extern __shared__ double beam_c[];        // [RB][beams * width] scores
    const int per = a.beams * a.width;
    int *beam_f = (int *)(beam_c + RB * per); // ... beam * V + token
    const int lane = threadIdx.x & 63, sub = lane % LPR, rb = lane / LPR;
    const int k = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = blockIdx.x * RB + rb, end = end_token_of(a);
    if (b < a.batch) {
        const long long row = (long long)k * a.batch + b;
        const double score = a.scores[row];
        const bool done = a.finished && a.finished[row];
        double log_s = 0.;
        float m = 0.f;
        bool live = !done && score > -INFINITY;
        ShortTop<KT> top;
        if (live) {
            RowRegs<DT, LPR, G> x;
            x.load((const T *)a.logits + row * a.ld, a.V, sub);
            top.template of<DT, LPR, G>(x, a.V, sub);
            bool nan = false;
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float v = x.r[g].get(j);
                    nan |= v != v;
                }
            // (the list's first is the maximum; a NaN anywhere ends the row)
            m = row_max<LPR>(nan ? INFINITY : key_value(top.l[0]));
            live = !isinf(m);
            if (live) {
                const Exp64 e(a, m);
                double s = 0.;
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int j = 0; j < 8; ++j) s += e(x.r[g].get(j));
                s = row_sum<LPR>(s);
                log_s = log(s);
            }
        }
#pragma unroll
        for (int j = 0; j < KT; ++j)
            if (j < a.width && j % LPR == sub) {
                int tok = j;   // a row without a distribution: tokens in order
                double c = -INFINITY;
                if (done) {
                    tok = ended_token(end, j, score);
                    if (j == 0 && score > -INFINITY) c = score;
                } else if (live) {
                    tok = top.l[j] > KEY_NONE ? key_index(top.l[j]) : a.V;
                    // (a masked token is -inf beside a score of +inf too)
                    const float v = key_value(top.l[j]);
                    if (v > -INFINITY) c = beam_score(a, score, v, m, log_s);
                }
                const int at = rb * per + k * a.width + j;
                beam_c[at] = tok < a.V ? c : -INFINITY;
                beam_f[at] = tok < a.V ? 2 * (k * a.V + tok) + (done ? 1 : 0)
                                       : 0x7fffffff;
            }
    }
    __syncthreads();
    beam_rank(beam_c, beam_f, a, end,
              min(RB, a.batch - (int)blockIdx.x * RB), blockIdx.x * RB);
}

// How a row of V logits is dealt out: `parts` blocks of `len` elements each.
// Few rows leave most of the 256 CUs idle, so rows of at least `least` are split
// until there are about 512 blocks or a part is down to 4096 elements.  Joining
// top logits is a launch more: it pays beyond 131072 (top 12 of one row of 131071:
// 18 us in two launches, 14.6 in one; of 262144: 18 and 22), for long lists beyond
// 65536 (top 64 of one of 65536: 18 and 15; of 131071: 18 and 21).  Beams are joined
// anyway.
constexpr int top_split(int k) { return k > 32 ? 65537 : 131073; }
constexpr int BEAM_SPLIT = 8193;
struct RowPlan {
    int parts, len;
};
RowPlan row_plan(long long rows, int V, int least) {
    RowPlan p;
    long long parts = 1;
    if (rows < 256 && V >= least) {
        long long want = 512 / rows, most = V / 4096;
        if (want > most) want = most;
        if (want > 64) want = 64;
        if (want > parts) parts = want;
    }
    p.len = (int)((V + parts - 1) / parts);
    p.len = (p.len + 7) / 8 * 8;
    p.parts = (V + p.len - 1) / p.len;
    return p;
}
// A launch has less than 2^32 threads: may these rows be one?
bool rows_fit(long long rows, int V, int k, const RowPlan &p) {
    // (at most 16 lanes a row, and blocks of at most 64 rows that need not be full;
    // beams: 4 batch rows of 16)
    if (short_rows(rows, V, k)) return rows <= (1ll << 28) - 64;
    const int threads = p.len <= 512 ? 64 : p.len <= 2048 ? 256 : 1024;
    return rows * p.parts * threads < (1ll << 32);
}
// run the call with the constants NT (threads) and ONE (a group of eight per
// thread) for `blocks` stretches of `len` elements.  Long ones: 1024 threads while
// that fills the chip (top 64 of one row of 32767: 13.5 us against 18 with 512),
// 512 when there are enough blocks that one computes while another loads (top 32
// of 1024 x 50021: 34 us against 43 with 1024 and 63 with 256).
#define PCM_BY_LENGTH(blocks, len, ...)                                        \
    do {                                                                       \
        if ((len) <= 512) {                                                    \
            constexpr int NT = 64; constexpr bool ONE = true; __VA_ARGS__;     \
        } else if ((len) <= 2048) {                                            \
            constexpr int NT = 256; constexpr bool ONE = true; __VA_ARGS__;    \
        } else if ((len) <= 4096) {                                            \
            constexpr int NT = 512; constexpr bool ONE = true; __VA_ARGS__;    \
        } else if ((len) <= 8192) {                                            \
            constexpr int NT = 1024; constexpr bool ONE = true; __VA_ARGS__;   \
        } else if ((blocks) < 256) {                                           \
            constexpr int NT = 1024; constexpr bool ONE = false; __VA_ARGS__;  \
        } else {                                                               \
            constexpr int NT = 512; constexpr bool ONE = false; __VA_ARGS__;   \
        }                                                                      \
    } while (0)

// ---- states follow their beams ------------------------------------------------------
struct ReorderState {
    char *data;
    long long outer_stride, row_stride;
    unsigned units, per_row;   // of 16 .. 1 bytes: of all outer indices; of one
    unsigned magic, shift;     // o = unit / per_row
    int bytes;                 // of a unit
};
struct ReorderArgs {
    const int32_t *parents;
    int32_t *status;
    int beams, batch, count;
    int split;                 // blocks per batch row
    ReorderState s[PCM_MAX_STATES];
};

// The bytes of a state: pieces of `piece` bytes from lo on, at multiples of `step`
// from each other (0: one piece), all before hi.
struct StateBytes {
    uintptr_t lo, hi;
    unsigned long long piece, step;
    // rows (or outer indices) that lie end to end are one piece
    StateBytes(const pcm_state &s, long long rows) {
        lo = (uintptr_t)s.data;
        hi = lo + (s.outer - 1) * s.outer_stride + (rows - 1) * s.row_stride +
             s.row_bytes;
        long long at[2] = {s.row_stride, s.outer_stride}, n[2] = {rows, s.outer};
        if (n[1] > 1 && (n[0] == 1 || at[1] < at[0])) {   // the inner ones first
            const long long t = at[0], m = n[0];
            at[0] = at[1]; n[0] = n[1];
            at[1] = t; n[1] = m;
        }
        piece = s.row_bytes;
        step = 0;
        for (int i = 0; i < 2; ++i) {
            if (n[i] == 1) continue;
            if (step == 0 && (unsigned long long)at[i] == piece) piece *= n[i];
            else step = common(step, at[i]);
        }
    }
    StateBytes(const void *data, long long bytes)
        : lo((uintptr_t)data), hi(lo + bytes), piece(bytes), step(0) {}
    static unsigned long long common(unsigned long long a, unsigned long long b) {
        while (b) {
            const unsigned long long c = a % b;
            a = b;
            b = c;
        }
        return a;
    }
    // Whether they share no byte: one lies before the other, or between the
    // other's pieces, as seen modulo a number that divides all steps.
    bool apart(const StateBytes &o) const {
        if (hi <= o.lo || o.hi <= lo) return true;
        const unsigned long long m = common(step, o.step);
        if (m == 0) return false;
        const unsigned long long d = o.lo >= lo ? (o.lo - lo) % m
                                                : (m - (lo - o.lo) % m) % m;
        return d >= piece && d + o.piece <= m;
    }
};

// A thread owns the same units of one batch row in ALL beams: it loads what
// every beam will hold before it stores any of it, so the move is in place
// whatever the parents are.  K bounds the beams (the arrays stay in registers),
// N units are in flight at once; the parents are the same for the whole block,
// so a beam that keeps its row costs a scalar branch.
// 3 x 4096 beams of 14 KB (two hidden layers and a 50 x 50 stack): 51 us for the
// 211 MB that random parents move, 4.1 of the 4.7 TB/s of a large copy (into a second
// tensor it would be all rows, moved or not); one molecule: 4.1 us, latency.
template <typename U, int K, int N>
__device__ __forceinline__ void reorder_units(const ReorderState &s, int b,
                                              long long beam_stride,
                                              const int (&par)[K], unsigned first,
                                              unsigned step) {
    for (unsigned c0 = first; c0 < s.units; c0 += N * step) {
        U v[N][K];
        char *at[N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const unsigned c = c0 + n * step;
            const unsigned o = s.per_row == s.units ? 0u
                               : s.per_row == 1 ? c
                               : __umulhi(c, s.magic) >> s.shift;
            at[n] = s.data + (long long)o * s.outer_stride +
                    (long long)b * s.row_stride +
                    (long long)(c - o * s.per_row) * sizeof(U);
            if (c < s.units) {
#pragma unroll
                for (int k = 0; k < K; ++k)
                    if (par[k] != k) v[n][k] = *(const U *)(at[n] + par[k] * beam_stride);
            }
        }
#pragma unroll
        for (int n = 0; n < N; ++n)
            if (c0 + n * step < s.units) {
#pragma unroll
                for (int k = 0; k < K; ++k)
                    if (par[k] != k) *(U *)(at[n] + k * beam_stride) = v[n][k];
            }
    }
}

template <int K>
__global__ __launch_bounds__(256) void reorder_kernel(ReorderArgs a) {
    constexpr int N = K <= 4 ? 4 : K <= 8 ? 2 : 1;
    const int b = blockIdx.x / a.split, part = blockIdx.x - b * a.split;
    int par[K];
    bool moves = false;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        par[k] = k;
        if (k < a.beams) {
            const int p = __builtin_amdgcn_readfirstlane(
                a.parents[(long long)k * a.batch + b]);
            if (p >= 0 && p < a.beams) par[k] = p;
            else if (a.status && threadIdx.x == 0 && part == 0)
                atomicOr(a.status, PCM_STATUS_BAD_PARENT);
            moves |= par[k] != k;
        }
    }
    if (!moves) return;
    const unsigned first = part * 256 + threadIdx.x, step = a.split * 256;
    for (int i = 0; i < a.count; ++i) {
        const ReorderState &s = a.s[i];
        const long long stride = s.row_stride * a.batch;
        switch (s.bytes) {
        case 16: reorder_units<row_u32x4, K, N>(s, b, stride, par, first, step); break;
        case 8: reorder_units<row_u32x2, K, N>(s, b, stride, par, first, step); break;
        case 4: reorder_units<unsigned, K, N>(s, b, stride, par, first, step); break;
        case 2: reorder_units<unsigned short, K, N>(s, b, stride, par, first, step); break;
        default: reorder_units<unsigned char, K, N>(s, b, stride, par, first, step); break;
        }
    }
}

// ---- joint beam search: first scores, final sequences -----------------------------
__global__ __launch_bounds__(256) void beam_start_kernel(double *scores,
                                                         uint8_t *finished,
                                                         int beams, int batch,
                                                         const int64_t *end_in,
                                                         int vocab,
                                                         int32_t *end_at,
                                                         int32_t *status) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= beams * batch) return;
    if (end_in && i == 0) {
        const int64_t end = *end_in;
        *end_at = end >= 0 && end < vocab ? (int32_t)end : -1;
        if (end >= vocab && status) atomicOr(status, PCM_STATUS_BAD_TOKEN);
    }
    scores[i] = i < batch ? 0. : -INFINITY;   // one beam to begin with
    finished[i] = 0;
}

__global__ __launch_bounds__(256) void beam_trace_kernel(
    const int64_t *tokens, const int32_t *parents, const double *scores,
    int beams, int batch, int G, int64_t *best_out, int64_t *beams_out,
    double *scores_out) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= beams * batch) return;
    const int b = i / beams, j = i - b * beams;
    if (scores_out) scores_out[i] = scores[(long long)j * batch + b];
    int slot = j;
    for (int t = G - 1; t >= 0; --t) {
        const long long at = ((long long)t * beams + slot) * batch + b;
        const int64_t tok = tokens[at];
        slot = parents[at];
        if (beams_out) beams_out[(long long)i * G + t] = tok;
        if (j == 0) best_out[(long long)b * G + t] = tok;
    }
}

}  // namespace

void pcm_launch_beam_start(double *scores, uint8_t *finished, int beams,
                           int batch, const int64_t *end_in, int vocab,
                           int32_t *end_at, int32_t *status, hipStream_t st) {
    hipLaunchKernelGGL(beam_start_kernel, dim3((beams * batch + 255) / 256),
                       dim3(256), 0, st, scores, finished, beams, batch, end_in,
                       vocab, end_at, status);
}

void pcm_launch_beam_trace(const int64_t *tokens, const int32_t *parents,
                           const double *scores, int beams, int batch, int G,
                           int64_t *best_out, int64_t *beams_out,
                           double *scores_out, hipStream_t st) {
    hipLaunchKernelGGL(beam_trace_kernel, dim3((beams * batch + 255) / 256),
                       dim3(256), 0, st, tokens, parents, scores, beams, batch,
                       G, best_out, beams_out, scores_out);
}

extern "C" {

size_t pcm_top_logits_workspace_bytes(int64_t rows, int32_t vocab, int32_t k) {
    if (rows < 1 || vocab < 1 || vocab > PCM_MAX_VOCAB || k < 1) return 0;
    const RowPlan p = row_plan(rows, vocab, top_split(k));
    if (p.parts == 1) return 0;
    return (size_t)rows * p.parts * (64 * sizeof(double) + 2 * sizeof(float));
}

int pcm_top_logits(const void *logits, int32_t dtype, int64_t rows, int64_t ld,
                   int32_t vocab, int32_t k, double temperature, void *values,
                   int32_t *indices, float *rest, void *workspace,
                   size_t workspace_bytes, void *stream) {
    PCM_API_GUARD;
    PCM_REQUIRE(logits && values && indices && rest, PCM_EINVAL,
                "top_logits: null pointer");
    PCM_REQUIRE(pcm_dtype_known(dtype), PCM_EINVAL,
                "top_logits: unknown dtype %d", dtype);
    PCM_REQUIRE(rows > 0 && rows < (1ll << 31) && vocab > 0 &&
                    vocab <= PCM_MAX_VOCAB, PCM_EINVAL,
                "top_logits: %lld rows of %d logits (1..2^31-1 rows, 1..%d "
                "logits)", (long long)rows, vocab, PCM_MAX_VOCAB);
    PCM_REQUIRE(ld >= vocab, PCM_EINVAL, "top_logits: row stride %lld < %d",
                (long long)ld, vocab);
    PCM_REQUIRE(k >= 1 && k <= PCM_TOP_MAX && k <= vocab, PCM_EINVAL,
                "top_logits: k=%d outside 1..min(%d, vocab %d)", k, PCM_TOP_MAX,
                vocab);
    // (1 / temperature has to be a 32-bit number)
    PCM_REQUIRE(temperature > 1e-30 && temperature < 1e30, PCM_EINVAL,
                "top_logits: temperature outside 1e-30..1e30");
    const size_t need = pcm_top_logits_workspace_bytes(rows, vocab, k);
    PCM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), PCM_ENOMEM,
                "top_logits: workspace %zu < %zu bytes", workspace_bytes, need);
    PCM_REQUIRE(((uintptr_t)workspace & 7) == 0, PCM_EINVAL,
                "top_logits: workspace must be 8-byte aligned");
    hipStream_t st = (hipStream_t)stream;
    const RowPlan plan = row_plan(rows, vocab, top_split(k));
    TopArgs a;
    a.logits = logits; a.values = values; a.indices = indices; a.rest = rest;
    a.keys = (double *)workspace;
    a.part = plan.parts > 1
                 ? (float *)(a.keys + (size_t)rows * plan.parts * 64) : nullptr;
    a.ld = ld; a.V = vocab; a.k = k; a.parts = plan.parts; a.len = plan.len;
    a.scale = (float)(1.4426950408889634 / temperature);
    a.inv_t = (float)(1.0 / temperature);
    PCM_REQUIRE(rows_fit(rows, vocab, k, plan), PCM_EINVAL,
                "top_logits: %lld rows of %d logits are too many for a launch",
                (long long)rows, vocab);
    if (short_rows(rows, vocab, k)) {
        PCM_BY_DTYPE(dtype, PCM_BY_SHORT(rows, vocab, k, {
            constexpr int per_block = 256 / LPR;
            hipLaunchKernelGGL((top_short_kernel<DT, LPR, G, KT>),
                               dim3((unsigned)((rows + per_block - 1) / per_block)),
                               dim3(256), 0, st, a, (long long)rows);
        }));
        return pcm_check_launch("top_logits");
    }
    PCM_BY_DTYPE(dtype, PCM_BY_LENGTH(rows * plan.parts, plan.len, {
        hipLaunchKernelGGL((top_kernel<DT, NT, ONE>),
                           dim3((unsigned)(rows * plan.parts)), dim3(NT), 0, st,
                           a);
    }));
    if (plan.parts > 1)
        PCM_BY_DTYPE(dtype, {
            hipLaunchKernelGGL(top_join_kernel<DT>, dim3((unsigned)rows),
                               dim3(1024), 0, st, a);
        });
    return pcm_check_launch("top_logits");
}

size_t pcm_beam_select_workspace_bytes(int32_t beams, int32_t batch,
                                       int32_t vocab, int32_t width) {
    if (beams < 1 || batch < 1 || width < 1 || vocab < 1 ||
        vocab > PCM_MAX_VOCAB)
        return 0;
    const size_t rows = (size_t)beams * batch;
    if (short_rows(rows, vocab, width)) return 0;
    return rows * row_plan(rows, vocab, BEAM_SPLIT).parts * (width + 2) * sizeof(double);
}

}  // extern "C"

int pcm_launch_beam_select(const void *logits, int32_t dtype, int64_t ld,
                           const double *scores, const uint8_t *finished,
                           int32_t beams, int32_t batch, int32_t vocab,
                           int32_t width, double temperature, int32_t end_token,
                           const int32_t *end_at, int64_t *tokens,
                           int32_t *parents, double *scores_out,
                           uint8_t *finished_out, void *workspace,
                           size_t workspace_bytes, hipStream_t st) {
    PCM_REQUIRE(logits && scores && tokens && parents && scores_out, PCM_EINVAL,
                "beam_select: null pointer");
    PCM_REQUIRE(pcm_dtype_known(dtype), PCM_EINVAL,
                "beam_select: unknown dtype %d", dtype);
    PCM_REQUIRE(beams >= 1 && beams <= PCM_BEAM_MAX && width >= 1 &&
                    width <= PCM_BEAM_MAX, PCM_EINVAL,
                "beam_select: beams=%d width=%d outside 1..%d", beams, width,
                PCM_BEAM_MAX);
    PCM_REQUIRE(batch >= 1 && batch < (1 << 24) && vocab >= 1 &&
                    vocab <= PCM_MAX_VOCAB, PCM_EINVAL,
                "beam_select: batch=%d vocab=%d (vocab 1..%d)", batch, vocab,
                PCM_MAX_VOCAB);
    PCM_REQUIRE(width <= (long long)beams * vocab, PCM_EINVAL,
                "beam_select: width=%d exceeds the %d x %d candidates", width,
                beams, vocab);
    PCM_REQUIRE(ld >= vocab, PCM_EINVAL, "beam_select: row stride %lld < %d",
                (long long)ld, vocab);
    PCM_REQUIRE(temperature > 1e-30 && temperature < 1e30, PCM_EINVAL,
                "beam_select: temperature must be positive");
    PCM_REQUIRE(!finished || (finished_out &&
                              (end_at || (end_token >= 0 && end_token < vocab))),
                PCM_EINVAL,
                "beam_select: finished beams need finished_out and an end_token "
                "in [0, %d), got %d", vocab, end_token);
    const size_t need =
        pcm_beam_select_workspace_bytes(beams, batch, vocab, width);
    PCM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), PCM_ENOMEM,
                "beam_select: workspace %zu < %zu bytes", workspace_bytes, need);
    PCM_REQUIRE(((uintptr_t)workspace & 7) == 0, PCM_EINVAL,
                "beam_select: workspace must be 8-byte aligned");
    const long long rows = (long long)beams * batch;
    const RowPlan plan = row_plan(rows, vocab, BEAM_SPLIT);
    PCM_REQUIRE(rows_fit(rows, vocab, width, plan), PCM_EINVAL,
                "beam_select: %lld rows of %d logits are too many for a launch",
                rows, vocab);
    BeamArgs a;
    a.logits = logits; a.scores = scores; a.finished = finished;
    a.keys = (double *)workspace;
    a.part = a.keys + (size_t)rows * plan.parts * width;
    a.tokens = tokens; a.parents = parents; a.scores_out = scores_out;
    a.finished_out = finished_out;
    a.ld = ld; a.beams = beams; a.batch = batch; a.V = vocab; a.width = width;
    a.parts = plan.parts; a.len = plan.len; a.end = end_token; a.end_at = end_at;
    a.inv_t = 1.0 / temperature;
    a.scale = 1.4426950408889634 / temperature;
    a.least = -1000. / a.scale;
    if (short_rows(rows, vocab, width)) {
        PCM_BY_DTYPE(dtype, PCM_BY_SHORT(rows, vocab, width, {
            constexpr int per_block = 64 / LPR;
            const size_t lds = (size_t)per_block * beams * width *
                               (sizeof(double) + sizeof(int));
            hipLaunchKernelGGL((beam_short_kernel<DT, LPR, G, KT>),
                               dim3((unsigned)((batch + per_block - 1) / per_block)),
                               dim3(64 * beams), lds, st, a);
        }));
        return pcm_check_launch("beam_select");
    }
    PCM_BY_DTYPE(dtype, PCM_BY_LENGTH(rows * plan.parts, plan.len, {
        hipLaunchKernelGGL((beam_rows_kernel<DT, NT, ONE>),
                           dim3((unsigned)(rows * plan.parts)), dim3(NT), 0, st,
                           a);
    }));
    hipLaunchKernelGGL(beam_join_kernel, dim3((unsigned)batch), dim3(64 * beams),
                       0, st, a);
    return pcm_check_launch("beam_select");
}

extern "C" {

int pcm_beam_select(const void *logits, int32_t dtype, int64_t ld,
                    const double *scores, const uint8_t *finished,
                    int32_t beams, int32_t batch, int32_t vocab, int32_t width,
                    double temperature, int32_t end_token, int64_t *tokens,
                    int32_t *parents, double *scores_out,
                    uint8_t *finished_out, void *workspace,
                    size_t workspace_bytes, void *stream) {
    PCM_API_GUARD;
    return pcm_launch_beam_select(
        logits, dtype, ld, scores, finished, beams, batch, vocab, width,
        temperature, end_token, nullptr, tokens, parents, scores_out,
        finished_out, workspace, workspace_bytes, (hipStream_t)stream);
}

int pcm_reorder_states(const int32_t *parents, int32_t beams, int32_t batch,
                       const pcm_state *states, int32_t count, int32_t *status,
                       void *stream) {
    PCM_API_GUARD;
    PCM_REQUIRE(parents && states, PCM_EINVAL, "reorder_states: null pointer");
    PCM_REQUIRE(beams >= 1 && beams <= PCM_BEAM_MAX && batch >= 1 &&
                    batch < (1 << 24), PCM_EINVAL,
                "reorder_states: beams=%d (1..%d) batch=%d (1..2^24-1)", beams,
                PCM_BEAM_MAX, batch);
    PCM_REQUIRE(count >= 1 && count <= PCM_MAX_STATES, PCM_EINVAL,
                "reorder_states: %d states (1..%d)", count, PCM_MAX_STATES);
    ReorderArgs a;
    a.parents = parents; a.status = status;
    a.beams = beams; a.batch = batch; a.count = 0;
    const long long rows = (long long)beams * batch;
    int known[PCM_MAX_STATES];   // states that are not empty
    long long most = 0;
    for (int i = 0; i < count; ++i) {
        pcm_state s = states[i];
        PCM_REQUIRE(s.outer >= 0 && s.row_bytes >= 0, PCM_EINVAL,
                    "reorder_states: state %d has a negative size", i);
        if (s.outer == 0 || s.row_bytes == 0) continue;
        PCM_REQUIRE(s.data, PCM_EINVAL, "reorder_states: state %d is null", i);
        // rows within an outer index, or outer indices within a row
        const bool rows_inside =
            s.row_stride >= s.row_bytes &&
            (s.outer == 1 || s.outer_stride >= s.row_stride * (rows - 1) +
                                                   s.row_bytes);
        const bool outer_inside =
            s.outer > 1 && s.outer_stride >= s.row_bytes &&
            (rows == 1 || s.row_stride >= s.outer_stride * (s.outer - 1) +
                                              s.row_bytes);
        PCM_REQUIRE(rows_inside || outer_inside || (rows == 1 && s.outer == 1),
                    PCM_EINVAL,
                    "reorder_states: rows of state %d share memory", i);
        const int n = a.count;
        const StateBytes bytes(s, rows);
        known[n] = i;
        for (int j = 0; j < n; ++j)
            PCM_REQUIRE(bytes.apart(StateBytes(states[known[j]], rows)),
                        PCM_EINVAL,
                        "reorder_states: state %d shares memory with another",
                        i);
        int unit = 16;
        const unsigned long long bits =
            (unsigned long long)bytes.lo | (unsigned long long)s.row_bytes |
            (unsigned long long)s.row_stride |
            (s.outer > 1 ? (unsigned long long)s.outer_stride : 0ull);
        while (bits & (unit - 1)) unit >>= 1;
        const long long per_row = s.row_bytes / unit;
        const long long units = per_row * s.outer;
        PCM_REQUIRE(units < (1ll << 30), PCM_EINVAL,
                    "reorder_states: state %d has rows of %lld pieces of %d "
                    "bytes (2^30 at most)", i, units, unit);
        ReorderState &q = a.s[n];
        q.data = (char *)s.data;
        q.outer_stride = s.outer > 1 ? s.outer_stride : 0;
        q.row_stride = s.row_stride;
        q.units = (unsigned)units;
        q.per_row = (unsigned)per_row;
        q.bytes = unit;
        // c / per_row for c < 2^31: a multiplication by ceil(2^(32 + l) / per_row),
        // 2^l < per_row <= 2^(l + 1)
        int l = 0;
        while ((2ll << l) < per_row) ++l;
        q.shift = l;
        q.magic = per_row > 1
                      ? (unsigned)(((1ull << (32 + l)) + per_row - 1) / per_row)
                      : 0;
        most = units > most ? units : most;
        a.count = n + 1;
    }
    const StateBytes from(parents, 4 * rows);
    for (int n = 0; n < a.count; ++n)
        PCM_REQUIRE(StateBytes(states[known[n]], rows).apart(from), PCM_EINVAL,
                    "reorder_states: state %d shares memory with the parents",
                    known[n]);
    // enough blocks per batch row to spread a small batch over the chip
    long long split = (most + 255) / 256;
    const long long want = (2048 + batch - 1) / batch;
    if (split > want) split = want;
    if (split < 1) split = 1;
    a.split = (int)split;
    const dim3 grid((unsigned)(split * batch));
#define PCM_REORDER(K) \
    hipLaunchKernelGGL(reorder_kernel<K>, grid, dim3(256), 0, (hipStream_t)stream, a)
    if (beams <= 2) PCM_REORDER(2);
    else if (beams <= 3) PCM_REORDER(3);
    else if (beams <= 4) PCM_REORDER(4);
    else if (beams <= 6) PCM_REORDER(6);
    else if (beams <= 8) PCM_REORDER(8);
    else PCM_REORDER(16);
#undef PCM_REORDER
    return pcm_check_launch("reorder_states");
}

}  // extern "C"
