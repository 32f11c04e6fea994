// Top logits of a row, the selection of a beam search over beams and
// vocabulary, and the reordering of the beams' states.
#include "rows.h"
#include "topbeam.h"

namespace {

// ---- top logits -------------------------------------------------------------------
// One wave per row; the j-th largest key is the largest one below the (j-1)-th,
// so nothing has to be marked.
template <int DT>
__global__ __launch_bounds__(256) void top_logits_kernel(
    const typename RowType<DT>::T *logits, long long rows, long long ld, int V,
    int k, float scale, typename RowType<DT>::T *values, int32_t *indices,
    float *rest) {
    typedef RowType<DT> R;
    const int lane = threadIdx.x & 63;
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    const typename R::T *x = logits + row * ld;
    double prev = __builtin_inf();
    for (int j = 0; j < k; ++j) {
        double best = KEY_NONE;
        for (int v = lane; v < V; v += 64) {
            const double key = key_of(R::up(x[v]), v);
            if (key < prev && key > best) best = key;
        }
        prev = wave_max(best);
        if (lane == 0) {
            values[row * k + j] = R::down(key_value(prev));
            indices[row * k + j] = key_index(prev);
        }
    }
    float m = -INFINITY;
    for (int v = lane; v < V; v += 64) {
        const float xv = R::up(x[v]);
        if (key_of(xv, v) < prev) m = fmaxf(m, xv);
    }
    m = wave_max(m);
    float s = 0.f;
    bool nan = false;
    for (int v = lane; v < V; v += 64) {
        const float xv = R::up(x[v]);
        nan |= xv != xv;
        if (key_of(xv, v) < prev) s += exp2f((xv - m) * scale);
    }
    s = wave_sum(s);
    if (lane == 0)
        rest[row] = __any(nan) ? NAN
                    : isinf(m) ? m
                               : m * (scale * 0.6931471805599453f) + logf(s);
    else
        (void)__any(nan);
}

// ---- beam selection ---------------------------------------------------------------
// First kernel: the `width` best tokens of every beam row by logit (the row's
// normaliser does not change their order) with their scores in 64 bits.
template <int DT>
__global__ __launch_bounds__(256) void beam_rows_kernel(
    const typename RowType<DT>::T *logits, long long ld, const double *scores,
    const uint8_t *finished, int rows, int V, int width, double inv_t, int end,
    double *cand, int32_t *ctok) {
    typedef RowType<DT> R;
    const int lane = threadIdx.x & 63;
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    const double score = scores[row];
    double *co = cand + (long long)row * width;
    int32_t *to = ctok + (long long)row * width;
    if (finished && finished[row]) {
        // end_token, then the others in order
        for (int j = lane; j < width; j += 64) {
            int tok = j == 0 ? end : j - 1 + (j - 1 >= end ? 1 : 0);
            co[j] = j == 0 && score == score ? score : -INFINITY;
            to[j] = tok < V ? tok : -1;
        }
        return;
    }
    const typename R::T *x = logits + (long long)row * ld;
    float m = -INFINITY;
    bool bad = !(score > -INFINITY);
    if (!bad) {
        for (int v = lane; v < V; v += 64) {
            const float xv = R::up(x[v]);
            m = fmaxf(m, xv);
            bad |= xv != xv;
        }
        m = wave_max(m);
        bad = __any(bad) || isinf(m);
    }
    if (bad) {   // no beam here, or no distribution: every candidate is -inf
        for (int j = lane; j < width; j += 64) {
            co[j] = -INFINITY;
            to[j] = j < V ? j : -1;
        }
        return;
    }
    double s = 0.;
    for (int v = lane; v < V; v += 64)
        s += exp(((double)R::up(x[v]) - (double)m) * inv_t);
    s = wave_sum(s);
    const double lse = (double)m * inv_t + log(s);
    double prev = __builtin_inf();
    for (int j = 0; j < width; ++j) {
        double best = KEY_NONE;
        for (int v = lane; v < V; v += 64) {
            const double key = key_of(R::up(x[v]), v);
            if (key < prev && key > best) best = key;
        }
        prev = wave_max(best);
        if (lane == 0) {
            const bool none = j >= V;
            co[j] = none ? -INFINITY
                         : score + ((double)key_value(prev) * inv_t - lse);
            to[j] = none ? -1 : key_index(prev);
        }
    }
}

// Second kernel: one wave per batch row ranks the beams * width survivors (at
// most 256: four per lane).
__global__ __launch_bounds__(256) void beam_join_kernel(
    const double *cand, const int32_t *ctok, const uint8_t *finished, int beams,
    int batch, int V, int width, int end, int64_t *tokens, int32_t *parents,
    double *scores_out, uint8_t *finished_out) {
    const int lane = threadIdx.x & 63;
    const int b = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (b >= batch) return;
    double c[4];
    int f[4];   // k * V + token, 0x7fffffff where there is no candidate
    const int n = beams * width;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int at = lane + 64 * i;
        c[i] = KEY_NONE;
        f[i] = 0x7fffffff;
        if (at < n) {
            const int k = at / width, j = at - k * width;
            const long long o = ((long long)k * batch + b) * width + j;
            const int tok = ctok[o];
            if (tok >= 0) {
                c[i] = cand[o];
                f[i] = k * V + tok;
            }
        }
    }
    for (int j = 0; j < width; ++j) {
        double bc = c[0];
        int bf = f[0];
#pragma unroll
        for (int i = 1; i < 4; ++i)
            if (c[i] > bc || (c[i] == bc && f[i] < bf)) { bc = c[i]; bf = f[i]; }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            const double oc = __shfl_xor(bc, off, 64);
            const int of = __shfl_xor(bf, off, 64);
            if (oc > bc || (oc == bc && of < bf)) { bc = oc; bf = of; }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (f[i] == bf) { c[i] = KEY_NONE; f[i] = 0x7fffffff; }
        if (lane == 0) {
            const int k = bf / V, tok = bf - k * V;
            const long long o = (long long)j * batch + b;
            tokens[o] = tok;
            parents[o] = k;
            scores_out[o] = bc;
            if (finished_out)
                finished_out[o] =
                    (finished && finished[(long long)k * batch + b]) ||
                    tok == end;
        }
    }
}

// ---- states follow their beams ------------------------------------------------------
struct ReorderArgs {
    const int32_t *parents;
    int32_t *status;
    int beams, batch, count;
    int split;                        // blocks per batch row
    int unit[PCM_MAX_STATES];         // bytes a thread moves at once
    long long chunks[PCM_MAX_STATES]; // units of all outer indices of one row
    long long per_row[PCM_MAX_STATES];
    pcm_state s[PCM_MAX_STATES];
};

// A thread owns one unit of one batch row in ALL beams: it loads what every
// beam will hold before it stores any of it, so the move is in place whatever
// the parents are.
template <typename U>
__device__ void reorder_unit(char *at, long long beam_stride, const int *par,
                             int beams) {
    U v[PCM_BEAM_MAX];
#pragma unroll
    for (int k = 0; k < PCM_BEAM_MAX; ++k)
        if (k < beams && par[k] != k)
            v[k] = *(const U *)(at + par[k] * beam_stride);
#pragma unroll
    for (int k = 0; k < PCM_BEAM_MAX; ++k)
        if (k < beams && par[k] != k) *(U *)(at + k * beam_stride) = v[k];
}

__global__ __launch_bounds__(256) void reorder_kernel(ReorderArgs a) {
    const int b = blockIdx.x / a.split, part = blockIdx.x - b * a.split;
    int par[PCM_BEAM_MAX];
    bool moves = false;
#pragma unroll
    for (int k = 0; k < PCM_BEAM_MAX; ++k) {
        par[k] = k;
        if (k < a.beams) {
            const int p = a.parents[(long long)k * a.batch + b];
            if (p >= 0 && p < a.beams) par[k] = p;
            else if (a.status && threadIdx.x == 0 && part == 0)
                atomicOr(a.status, PCM_STATUS_BAD_PARENT);
            moves |= par[k] != k;
        }
    }
    if (!moves) return;
    for (int i = 0; i < a.count; ++i) {
        const pcm_state &s = a.s[i];
        const long long stride = s.row_stride * a.batch;
        for (long long c = (long long)part * 256 + threadIdx.x;
             c < a.chunks[i]; c += (long long)a.split * 256) {
            const long long o = c / a.per_row[i], e = c - o * a.per_row[i];
            char *at = (char *)s.data + o * s.outer_stride +
                       b * s.row_stride + e * a.unit[i];
            switch (a.unit[i]) {
            case 16: reorder_unit<uint4>(at, stride, par, a.beams); break;
            case 8: reorder_unit<uint2>(at, stride, par, a.beams); break;
            case 4: reorder_unit<unsigned>(at, stride, par, a.beams); break;
            case 2: reorder_unit<unsigned short>(at, stride, par, a.beams); break;
            default: reorder_unit<unsigned char>(at, stride, par, a.beams); break;
            }
        }
    }
}

// ---- joint beam search: first scores, final sequences -----------------------------
__global__ __launch_bounds__(256) void beam_start_kernel(double *scores,
                                                         uint8_t *finished,
                                                         int beams, int batch) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= beams * batch) return;
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
                           int batch, hipStream_t st) {
    hipLaunchKernelGGL(beam_start_kernel, dim3((beams * batch + 255) / 256),
                       dim3(256), 0, st, scores, finished, beams, batch);
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
    (void)rows; (void)vocab; (void)k;
    return 0;
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
    PCM_REQUIRE(temperature > 0. && temperature < 1e30, PCM_EINVAL,
                "top_logits: temperature must be positive");
    const size_t need = pcm_top_logits_workspace_bytes(rows, vocab, k);
    PCM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), PCM_ENOMEM,
                "top_logits: workspace %zu < %zu bytes", workspace_bytes, need);
    hipStream_t st = (hipStream_t)stream;
    const float scale = (float)(1.4426950408889634 / temperature);
    PCM_BY_DTYPE(dtype, {
        typedef RowType<DT>::T T;
        hipLaunchKernelGGL(top_logits_kernel<DT>,
                           dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st,
                           (const T *)logits, (long long)rows, (long long)ld,
                           vocab, k, scale, (T *)values, indices, rest);
    });
    return pcm_check_launch("top_logits");
}

size_t pcm_beam_select_workspace_bytes(int32_t beams, int32_t batch,
                                       int32_t vocab, int32_t width) {
    (void)vocab;
    if (beams < 1 || batch < 1 || width < 1) return 0;
    return (size_t)beams * batch * width * (sizeof(double) + sizeof(int32_t));
}

int pcm_beam_select(const void *logits, int32_t dtype, int64_t ld,
                    const double *scores, const uint8_t *finished,
                    int32_t beams, int32_t batch, int32_t vocab, int32_t width,
                    double temperature, int32_t end_token, int64_t *tokens,
                    int32_t *parents, double *scores_out,
                    uint8_t *finished_out, void *workspace,
                    size_t workspace_bytes, void *stream) {
    PCM_API_GUARD;
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
    PCM_REQUIRE(!finished || (finished_out && end_token >= 0 &&
                              end_token < vocab), PCM_EINVAL,
                "beam_select: finished beams need finished_out and an end_token "
                "in [0, %d), got %d", vocab, end_token);
    const size_t need =
        pcm_beam_select_workspace_bytes(beams, batch, vocab, width);
    PCM_REQUIRE(workspace && workspace_bytes >= need, PCM_ENOMEM,
                "beam_select: workspace %zu < %zu bytes", workspace_bytes, need);
    PCM_REQUIRE(((uintptr_t)workspace & 7) == 0, PCM_EINVAL,
                "beam_select: workspace must be 8-byte aligned");
    hipStream_t st = (hipStream_t)stream;
    const int rows = beams * batch;
    double *cand = (double *)workspace;
    int32_t *ctok = (int32_t *)(cand + (size_t)rows * width);
    PCM_BY_DTYPE(dtype, {
        typedef RowType<DT>::T T;
        hipLaunchKernelGGL(beam_rows_kernel<DT>, dim3((rows + 3) / 4), dim3(256),
                           0, st, (const T *)logits, (long long)ld, scores,
                           finished, rows, vocab, width, 1.0 / temperature,
                           end_token, cand, ctok);
    });
    hipLaunchKernelGGL(beam_join_kernel, dim3((batch + 3) / 4), dim3(256), 0, st,
                       cand, ctok, finished, beams, batch, vocab, width,
                       end_token, tokens, parents, scores_out, finished_out);
    return pcm_check_launch("beam_select");
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
    uintptr_t lo[PCM_MAX_STATES], hi[PCM_MAX_STATES];
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
        lo[n] = (uintptr_t)s.data;
        hi[n] = lo[n] + (s.outer - 1) * s.outer_stride +
                (rows - 1) * s.row_stride + s.row_bytes;
        for (int j = 0; j < n; ++j)
            PCM_REQUIRE(hi[n] <= lo[j] || hi[j] <= lo[n], PCM_EINVAL,
                        "reorder_states: state %d shares memory with another",
                        i);
        int unit = 16;
        const unsigned long long bits =
            (unsigned long long)lo[n] | (unsigned long long)s.row_bytes |
            (unsigned long long)s.row_stride |
            (s.outer > 1 ? (unsigned long long)s.outer_stride : 0ull);
        while (bits & (unit - 1)) unit >>= 1;
        a.s[n] = s;
        a.unit[n] = unit;
        a.per_row[n] = s.row_bytes / unit;
        a.chunks[n] = a.per_row[n] * s.outer;
        most = a.chunks[n] > most ? a.chunks[n] : most;
        a.count = n + 1;
    }
    // enough blocks per batch row to spread a small batch over the chip
    long long split = (most + 255) / 256;
    const long long want = (2048 + batch - 1) / batch;
    if (split > want) split = want;
    if (split < 1) split = 1;
    a.split = (int)split;
    hipLaunchKernelGGL(reorder_kernel, dim3((unsigned)(split * batch)),
                       dim3(256), 0, (hipStream_t)stream, a);
    return pcm_check_launch("reorder_states");
}

}  // extern "C"
