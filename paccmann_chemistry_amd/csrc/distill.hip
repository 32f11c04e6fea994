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
    const float *weight;   // [T]
    float *rowloss;        // [T*B]
    void *dlogits;
    int32_t *status;
    long long ld, rows;
    int B, V, k;
    float inv_t, scale;    // 1 / tau; log2(e) / tau
    float soft, hard;      // (1 - hard) tau^2; hard
    float dsoft;           // (1 - hard) tau
};

// weight of every step: the caller's, or 1 / rows that run at it
__global__ __launch_bounds__(256) void distill_weight_kernel(
    const int32_t *lengths, const float *step_weight, int T, int B, float *out) {
    const int t = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (t >= T) return;
    if (step_weight) {
        if (lane == 0) out[t] = step_weight[t];
        return;
    }
    int c = 0;
    for (int b = lane; b < B; b += 64)
        c += !lengths || lengths[b] > t ? 1 : 0;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) c += __shfl_xor(c, off, 64);
    if (lane == 0) out[t] = c > 0 ? 1.0f / (float)c : 0.0f;
}

// Block reductions over 256 threads (4 waves), every thread gets the result.
struct BlockRed {
    float v[4];
};
__device__ __forceinline__ float block_max(float v, BlockRed &r) {
    v = wave_max(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) r.v[threadIdx.x >> 6] = v;
    __syncthreads();
    return fmaxf(fmaxf(r.v[0], r.v[1]), fmaxf(r.v[2], r.v[3]));
}
__device__ __forceinline__ float block_sum(float v, BlockRed &r) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) r.v[threadIdx.x >> 6] = v;
    __syncthreads();
    return (r.v[0] + r.v[1]) + (r.v[2] + r.v[3]);
}

// One block per row; the row is read three times.  Listed tokens are marked in
// a bitmap in LDS.
template <int DT, int DTV>
__global__ __launch_bounds__(256) void distill_kernel(DistillArgs a) {
    typedef RowType<DT> R;
    typedef RowType<DTV> RV;
    extern __shared__ unsigned marks[];   // ceil(V / 32) words
    __shared__ int s_idx[PCM_TOP_MAX];    // -1: absent
    __shared__ float s_u[PCM_TOP_MAX], s_p[PCM_TOP_MAX], s_x[PCM_TOP_MAX];
    __shared__ float s_mass[PCM_TOP_MAX];
    __shared__ int s_first[PCM_TOP_MAX];
    __shared__ BlockRed red;
    const int tid = threadIdx.x;
    const long long row = blockIdx.x;
    const int t = (int)(row / a.B), b = (int)(row - (long long)t * a.B);
    const float w = a.weight[t];
    const int V = a.V, k = a.k;
    typename R::T *dl = a.dlogits ? (typename R::T *)a.dlogits + row * V : nullptr;
    if ((a.lengths && t >= a.lengths[b]) || w == 0.f) {
        if (tid == 0) a.rowloss[row] = 0.f;
        if (dl)
            for (int v = tid; v < V; v += 256) dl[v] = R::down(0.f);
        return;
    }
    const typename R::T *x = (const typename R::T *)a.logits + row * a.ld;
    const float rest = a.rest ? a.rest[row] : -INFINITY;
    for (int i = tid; i < (V + 31) / 32; i += 256) marks[i] = 0;
    if (tid < k) {
        int idx = a.indices[row * k + tid];
        if (idx >= V) {
            if (a.status) atomicOr(a.status, PCM_STATUS_BAD_TOKEN);
            idx = -1;
        }
        s_idx[tid] = idx < 0 ? -1 : idx;
        s_u[tid] = idx < 0 ? -INFINITY
                           : RV::up(((const typename RV::T *)a.values)[row * k + tid]) *
                                 a.inv_t;
        s_x[tid] = idx < 0 ? -INFINITY : R::up(x[idx]);
    }
    __syncthreads();
    // an index that appears twice: the first entry stands for it
    if (tid < k) {
        int first = s_idx[tid] >= 0 ? 1 : 0;
        for (int j = 0; j < tid; ++j)
            if (s_idx[j] == s_idx[tid]) first = 0;
        s_first[tid] = first;
        if (first) atomicOr(&marks[s_idx[tid] >> 5], 1u << (s_idx[tid] & 31));
    }
    // teacher
    float nm = rest;
    for (int j = 0; j < k; ++j) nm = fmaxf(nm, s_u[j]);
    const bool taught = nm > -INFINITY || nm != nm;
    float ns = expf(rest - nm);
    for (int j = 0; j < k; ++j) ns += expf(s_u[j] - nm);
    const float N = nm + logf(ns);
    const float pr = taught ? expf(rest - N) : 0.f;
    if (tid < k) s_p[tid] = taught ? expf(s_u[tid] - N) : 0.f;
    __syncthreads();
    if (tid < k) {
        float mass = 0.f;
        for (int j = 0; j < k; ++j)
            if (s_idx[j] == s_idx[tid]) mass += s_p[j];
        s_mass[tid] = mass;
    }
    // student: the others' maximum and sums, then the listed ones
    float m = -INFINITY;
    for (int v = tid; v < V; v += 256)
        if (!((marks[v >> 5] >> (v & 31)) & 1)) m = fmaxf(m, R::up(x[v]));
    m = block_max(m, red);
    const float mo = m == -INFINITY ? 0.f : m;   // nothing left: every term is 0
    float s = 0.f, h = 0.f;
    for (int v = tid; v < V; v += 256)
        if (!((marks[v >> 5] >> (v & 31)) & 1)) {
            const float d = R::up(x[v]) - mo;
            s += expf(d * a.inv_t);
            if (a.hard > 0.f) h += expf(d);
        }
    s = block_sum(s, red);
    if (a.hard > 0.f) h = block_sum(h, red);
    float ma = m;
    for (int j = 0; j < k; ++j)
        if (s_first[j]) ma = fmaxf(ma, s_x[j]);
    // (no others: their share is 0, not 0 times a power of -ma)
    float sa = s > 0.f ? s * expf((mo - ma) * a.inv_t) : s;
    float ha = h > 0.f ? h * expf(mo - ma) : h;
    for (int j = 0; j < k; ++j)
        if (s_first[j]) {
            sa += expf((s_x[j] - ma) * a.inv_t);
            ha += expf(s_x[j] - ma);
        }
    const float Z = ma * a.inv_t + logf(sa);    // lse(x / tau)
    const float ZH = ma + logf(ha);             // lse(x)
    // the row's loss
    long long tg = 0;
    if (a.hard > 0.f) {
        tg = a.targets[row];
        if (tg < 0 || tg >= V) {
            tg = tg < 0 ? 0 : V - 1;
            if (tid == 0 && a.status) atomicOr(a.status, PCM_STATUS_BAD_TOKEN);
        }
    }
    if (tid == 0) {
        float kl = 0.f;
        for (int j = 0; j < k; ++j)
            if (s_p[j] > 0.f || s_p[j] != s_p[j])
                kl += s_p[j] * ((s_u[j] - N) - (s_x[j] * a.inv_t - Z));
        if (pr > 0.f || pr != pr)
            kl += pr * ((rest - N) - (mo * a.inv_t + logf(s) - Z));
        float loss = a.soft * kl;
        if (a.hard > 0.f) loss += a.hard * (ZH - R::up(x[tg]));
        a.rowloss[row] = loss * w;
    }
    if (!dl) return;
    // gradient: the others first, then the listed ones and the target
    const float cq = taught ? a.dsoft * w * (expf(mo * a.inv_t - Z) -
                                             (pr > 0.f && s > 0.f ? pr / s : 0.f))
                            : 0.f;
    const float ch = a.hard * w;
    for (int v = tid; v < V; v += 256)
        if (!((marks[v >> 5] >> (v & 31)) & 1)) {
            const float xv = R::up(x[v]);
            float g = expf((xv - mo) * a.inv_t) * cq;
            if (a.hard > 0.f)
                g += ch * (expf(xv - ZH) - (v == (int)tg ? 1.f : 0.f));
            dl[v] = R::down(g);
        }
    if (tid < k && s_first[tid]) {
        const float xv = s_x[tid];
        float g = 0.f;
        if (taught)
            g = a.dsoft * w * (expf(xv * a.inv_t - Z) - s_mass[tid]);
        if (a.hard > 0.f)
            g += ch * (expf(xv - ZH) - (s_idx[tid] == (int)tg ? 1.f : 0.f));
        dl[s_idx[tid]] = R::down(g);
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
    PCM_REQUIRE((long long)steps * batch < (1ll << 31), PCM_EINVAL,
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
    a.rowloss = scratch; a.weight = scratch + a.rows;
    a.ld = ld; a.B = batch; a.V = vocab; a.k = k;
    a.inv_t = (float)(1.0 / temperature);
    a.scale = (float)(1.4426950408889634 / temperature);
    a.soft = (float)((1.0 - hard_weight) * temperature * temperature);
    a.dsoft = (float)((1.0 - hard_weight) * temperature);
    a.hard = (float)hard_weight;
    hipLaunchKernelGGL(distill_weight_kernel, dim3((steps + 3) / 4), dim3(256),
                       0, st, lengths, step_weight, steps, batch,
                       scratch + a.rows);
    const size_t lds = (size_t)(vocab + 31) / 32 * 4;
    PCM_BY_DTYPE(dtype, {
        constexpr int DX = DT;
        PCM_BY_DTYPE(values_dtype, {
            hipLaunchKernelGGL((distill_kernel<DX, DT>), dim3((unsigned)a.rows),
                               dim3(256), lds, st, a);
        });
    });
    hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, st,
                       a.rowloss, a.rows, loss);
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
