// Draws from and probabilities of the paths of a candidate trellis (snk_sample_paths, snk_path_posterior).
//
// A path takes one candidate a_t of every row t of an utterance; with the target costs d and
//     C[t,a,b] = J[t,a,b] + B[class_t, bucket(cand[t+1,b] - cand[t,a])]        (join cost + bias by relative position)
//     p(path)  ~ exp(-(sum_t d[t,a_t] + sum_t C[t,a_t,a_t+1]) / tau)
// a candidate takes part if its unit can join (1 <= id < N - 1, as in the Viterbi search) and its target cost is finite.
//     alpha_0[b]   = -d[0,b] / tau          alpha_t+1[b] = -d[t+1,b] / tau + log sum_a exp(alpha_t[a] - C[t,a,b] / tau)
//     beta_T-1[a]  = 0                      beta_t[a]    = log sum_b exp(-C[t,a,b] / tau - d[t+1,b] / tau + beta_t+1[b])
//     log Z        = log sum_a exp(alpha_T-1[a])
//     draw: a_T-1 from alpha_T-1, then a_t from alpha_t[.] - C[t,.,a_t+1] / tau, every row of scores truncated like those of
//           sample_kernels.hip; temperature 0 keeps the largest term of every sum instead (tau = 1), and the draws follow it
#include "sample_device.h"

namespace snk {

__device__ __forceinline__ bool trellis_usable(int64_t id, int64_t n_units) { return id >= 1 && id < n_units - 1; }

// -d / tau of a candidate that takes part
__device__ __forceinline__ double trellis_local(int64_t id, double d, int64_t n_units, double inv_tau)
{
    return trellis_usable(id, n_units) && d - d == 0.0 ? -d * inv_tau : -__builtin_inf();
}

// ---- position bias, in place on the join costs: a workgroup per pair of rows ----------------------------------------------------
__global__ void __launch_bounds__(256)
position_bias_kernel(const int64_t *__restrict__ cand, const int32_t *__restrict__ join_class, const double *__restrict__ bias,
                     const int64_t *__restrict__ edges, int n_classes, int n_buckets, int K, double *__restrict__ C)
{
    __shared__ int64_t e[64];
    __shared__ double b[64];
    const int64_t t = blockIdx.x;
    const int c = join_class ? join_class[t] : 0;
    if (c < 0 || c >= n_classes) return;                        // a join without a class carries no bias
    const int tid = threadIdx.x;
    if (tid < n_buckets - 1) e[tid] = edges[tid];
    if (tid < n_buckets) b[tid] = bias[(int64_t)c * n_buckets + tid];
    __syncthreads();
    for (int i = blockIdx.y * 256 + tid; i < K * K; i += gridDim.y * 256) {
        const int64_t apart = cand[(t + 1) * K + i % K] - cand[t * K + i / K];
        int k = 0;
        for (int j = 0; j < n_buckets - 1; ++j) k += apart >= e[j] ? 1 : 0;
        C[t * K * K + i] += b[k];
    }
}

// ---- forward: a workgroup per utterance -------------------------------------------------------------------------------------------
template <bool SUM>
__global__ void __launch_bounds__(1024)
trellis_forward_kernel(const int64_t *__restrict__ cand, const double *__restrict__ tdist, const double *__restrict__ C,
                       const int64_t *__restrict__ off, int first, int64_t c0, int K, int64_t n_units, double inv_tau,
                       double *__restrict__ alpha, double *__restrict__ logz)
{
    __shared__ double cur[256], part_max[1024], part_sum[1024];
    const int tid = threadIdx.x;
    const int KB = (K + 63) & ~63, P = 1024 / KB;
    const int b = tid % KB, part = tid / KB;
    const int64_t r0 = off[first + blockIdx.x], T = off[first + blockIdx.x + 1] - r0;
    const double ninf = -__builtin_inf();
    const bool mine = b < K && part < P;
    if (tid < K) {
        const double v = trellis_local(cand[r0 * K + tid], tdist[r0 * K + tid], n_units, inv_tau);
        cur[tid] = v;
        alpha[r0 * K + tid] = v;
    }
    __syncthreads();
    for (int64_t t = 0; t + 1 < T; ++t) {
        const double *__restrict__ c = C + (r0 + t - c0) * K * K + b;
        double top = ninf, sum = 0.0;
        if (mine) {
            for (int a = part; a < K; a += P) top = fmax(top, cur[a] - c[(int64_t)a * K] * inv_tau);
            if (SUM && top > ninf)
                for (int a = part; a < K; a += P) sum += exp(cur[a] - c[(int64_t)a * K] * inv_tau - top);
        }
        part_max[tid] = top;
        part_sum[tid] = sum;
        __syncthreads();
        if (tid < K) {
            double all = ninf;
            for (int q = 0; q < P; ++q) all = fmax(all, part_max[q * KB + tid]);
            double v = all;
            if (SUM && all > ninf) {
                double s = 0.0;
                for (int q = 0; q < P; ++q)
                    if (part_max[q * KB + tid] > ninf) s += part_sum[q * KB + tid] * exp(part_max[q * KB + tid] - all);
                v = all + log(s);
            }
            const int64_t at = (r0 + t + 1) * K + tid;
            v += trellis_local(cand[at], tdist[at], n_units, inv_tau);
            cur[tid] = v;
            alpha[at] = v;
        }
        __syncthreads();
    }
    if (logz && tid == 0) {
        double all = ninf;
        for (int a = 0; a < K; ++a) all = fmax(all, cur[a]);
        double s = 0.0;
        if (all > ninf)
            for (int a = 0; a < K; ++a) s += exp(cur[a] - all);
        logz[first + blockIdx.x] = all > ninf ? all + log(s) : ninf;
    }
}

// ---- backward: a workgroup per utterance, a wavefront per predecessor ----------------------------------------------------------
__global__ void __launch_bounds__(1024)
trellis_backward_kernel(const int64_t *__restrict__ cand, const double *__restrict__ tdist, const double *__restrict__ C,
                        const int64_t *__restrict__ off, int first, int64_t c0, int K, int64_t n_units, double inv_tau, double *__restrict__ beta)
{
    __shared__ double into[2][256];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t r0 = off[first + blockIdx.x], T = off[first + blockIdx.x + 1] - r0;
    const double ninf = -__builtin_inf();
    if (tid < K) {
        const int64_t at = (r0 + T - 1) * K + tid;
        beta[at] = 0.0;
        into[(T - 1) & 1][tid] = trellis_local(cand[at], tdist[at], n_units, inv_tau);
    }
    __syncthreads();
    for (int64_t t = T - 2; t >= 0; --t) {
        const double *next = into[(t + 1) & 1];
        for (int a = wave; a < K; a += 16) {
            const double *__restrict__ c = C + (r0 + t - c0) * K * K + (int64_t)a * K;
            double x[4], top = ninf;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int b = lane + 64 * j;
                x[j] = b < K ? next[b] - c[b] * inv_tau : ninf;
                top = fmax(top, x[j]);
            }
            top = wave_max(top);
            double s = 0.0;
            if (top > ninf) {
#pragma unroll
                for (int j = 0; j < 4; ++j) s += exp(x[j] - top);
#pragma unroll
                for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o, 64);
            }
            if (lane == 0) {
                const double v = top > ninf ? top + log(s) : ninf;
                const int64_t at = (r0 + t) * K + a;
                beta[at] = v;
                into[t & 1][a] = v + trellis_local(cand[at], tdist[at], n_units, inv_tau);
            }
        }
        __syncthreads();
    }
}

// ---- posteriors: a workgroup per row; the row's bucket uses as integers in units of 2^-50 (sums in any order are the same) --------
__global__ void __launch_bounds__(256)
trellis_posterior_kernel(const int64_t *__restrict__ cand, const double *__restrict__ tdist, const double *__restrict__ C,
                         const double *__restrict__ alpha, const double *__restrict__ beta, const double *__restrict__ logz,
                         const int64_t *__restrict__ off, int first, int n_utts, int64_t c0, int K, int64_t n_units, double inv_tau,
                         const int64_t *__restrict__ edges, int n_buckets, double *__restrict__ posterior, double *__restrict__ row_uses)
{
    __shared__ double in[256];
    __shared__ double out[256];
    __shared__ int64_t e[64], id0[256], id1[256];
    __shared__ u64 uses[64];
    const int64_t t = c0 + blockIdx.x;
    const int tid = threadIdx.x;
    int u = first, hi = first + n_utts;                         // off[u] <= t < off[u + 1]
    while (hi - u > 1) { const int mid = (u + hi) >> 1; if (off[mid] <= t) u = mid; else hi = mid; }
    const double z = logz[u];
    const bool dead = !(z > -__builtin_inf());
    const bool last = t + 1 == off[u + 1];
    if (tid < K) {
        const double a = alpha[t * K + tid];
        posterior[t * K + tid] = dead ? 0.0 : exp(a + beta[t * K + tid] - z);
        in[tid] = a - z;
        id0[tid] = cand[t * K + tid];
        if (!last) {
            const int64_t at = (t + 1) * K + tid;
            id1[tid] = cand[at];
            out[tid] = trellis_local(cand[at], tdist[at], n_units, inv_tau) + beta[at];
        }
    }
    if (!row_uses) return;
    if (tid < 64) uses[tid] = 0;
    if (tid < n_buckets - 1) e[tid] = edges[tid];
    __syncthreads();
    if (!last && !dead) {
        for (int i = tid; i < K * K; i += 256) {
            const int a = i / K, b = i - a * K;
            const double x = in[a] - C[(t - c0) * K * K + i] * inv_tau + out[b];
            const u64 w = x < -36.0 ? 0ull : (u64)__double2ll_rn(exp(x) * 1125899906842624.0);
            if (!w) continue;
            const int64_t apart = id1[b] - id0[a];
            int k = 0;
            for (int j = 0; j < n_buckets - 1; ++j) k += apart >= e[j] ? 1 : 0;
            atomicAdd(&uses[k], w);
        }
    }
    __syncthreads();
    if (tid < n_buckets) row_uses[t * n_buckets + tid] = (double)uses[tid] * (1.0 / 1125899906842624.0);
}

// uses[class, bucket] = sum over the rows of the class: a workgroup per class, the rows in a fixed order
__global__ void __launch_bounds__(256)
trellis_uses_kernel(const double *__restrict__ row_uses, const int32_t *__restrict__ join_class, int64_t rows, int n_buckets,
                    double *__restrict__ uses)
{
    __shared__ double part[256];
    const int tid = threadIdx.x, k = blockIdx.y;
    double s = 0.0;
    for (int64_t t = tid; t < rows; t += 256)
        if ((join_class ? join_class[t] : 0) == (int)blockIdx.x) s += row_uses[t * n_buckets + k];
    part[tid] = s;
    __syncthreads();
    for (int o = 128; o; o >>= 1) {
        if (tid < o) part[tid] += part[tid + o];
        __syncthreads();
    }
    if (tid == 0) uses[(int64_t)blockIdx.x * n_buckets + k] = part[0];
}

// ---- draws: a wavefront per (utterance, draw) walks the trellis from its end ------------------------------------------------------
template <int E>
__global__ void __launch_bounds__(64)
trellis_draw_kernel(const int64_t *__restrict__ cand, const double *__restrict__ tdist, const double *__restrict__ C,
                    const double *__restrict__ alpha, const int64_t *__restrict__ off, int first, int64_t c0, int K, int64_t n_units, double inv_tau,
                    SampleRule rule, bool greedy, const double *__restrict__ u, int64_t rows, int n_utts, int64_t *__restrict__ path,
                    double *__restrict__ cost, double *__restrict__ logp)
{
    const int v = first + blockIdx.x, s = blockIdx.y, lane = threadIdx.x;
    const int64_t r0 = off[v], T = off[v + 1] - r0;
    const double ninf = -__builtin_inf();
    double spent = 0.0, lp = 0.0;
    int after = 0;
    for (int64_t t = T - 1; t >= 0; --t) {
        double x[E], c[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int a = lane * E + e;
            c[e] = (t + 1 < T && a < K) ? C[(r0 + t - c0) * K * K + (int64_t)a * K + after] : 0.0;
            x[e] = a < K ? alpha[(r0 + t) * K + a] - c[e] * inv_tau : ninf;
        }
        WaveRow<E> row;
        wave_row_weights<E>(x, rule, 2251799813685248.0, row);
        if (!(row.m > ninf)) {                                  // no complete path (only the last row can be empty)
            for (int64_t i = lane; i < T; i += 64) path[s * rows + r0 + i] = -1;
            if (lane == 0) { cost[(int64_t)s * n_utts + v] = -ninf; if (logp) logp[(int64_t)s * n_utts + v] = ninf; }
            return;
        }
        int l, slot;
        const int k = wave_row_pick<E>(row, greedy ? 0.0 : u[(int64_t)s * rows + r0 + t], l, slot);
        lp += sample_exponent(wave_row_value<E>(x, l, slot), row.m, rule.inv_tau) - row.log_total;
        spent += wave_row_value<E>(c, l, slot) + tdist[(r0 + t) * K + k];
        after = k;
        if (lane == 0) path[s * rows + r0 + t] = cand[(r0 + t) * K + k];
    }
    if (lane == 0) { cost[(int64_t)s * n_utts + v] = spent; if (logp) logp[(int64_t)s * n_utts + v] = lp; }
}

void launch_position_bias(const int64_t *cand, const int32_t *join_class, const double *bias, const int64_t *edges, int n_classes,
                          int n_buckets, int64_t rows, int K, double *C, hipStream_t s)
{
    if (rows < 2) return;
    hipLaunchKernelGGL(position_bias_kernel, dim3((unsigned)(rows - 1), (unsigned)((K * K + 4095) / 4096)), dim3(256), 0, s, cand, join_class, bias, edges,
                       n_classes, n_buckets, K, C);
}

void launch_trellis_forward(const TrellisView &v, bool sum, double *alpha, double *logz, hipStream_t s)
{
    if (sum) hipLaunchKernelGGL((trellis_forward_kernel<true>), dim3(v.n_utts), dim3(1024), 0, s, v.cand, v.tdist, v.C, v.off, v.first, v.c0, v.K, v.n_units, v.inv_tau, alpha, logz);
    else hipLaunchKernelGGL((trellis_forward_kernel<false>), dim3(v.n_utts), dim3(1024), 0, s, v.cand, v.tdist, v.C, v.off, v.first, v.c0, v.K, v.n_units, v.inv_tau, alpha, logz);
}

void launch_trellis_backward(const TrellisView &v, double *beta, hipStream_t s)
{
    hipLaunchKernelGGL(trellis_backward_kernel, dim3(v.n_utts), dim3(1024), 0, s, v.cand, v.tdist, v.C, v.off, v.first, v.c0, v.K, v.n_units, v.inv_tau, beta);
}

void launch_trellis_posterior(const TrellisView &v, const double *alpha, const double *beta, const double *logz, const int64_t *edges,
                              int n_buckets, double *posterior, double *row_uses, hipStream_t s)
{
    hipLaunchKernelGGL(trellis_posterior_kernel, dim3((unsigned)v.rows), dim3(256), 0, s, v.cand, v.tdist, v.C, alpha, beta, logz, v.off, v.first,
                       v.n_utts, v.c0, v.K, v.n_units, v.inv_tau, edges, n_buckets, posterior, row_uses);
}

void launch_trellis_uses(const double *row_uses, const int32_t *join_class, int64_t rows, int n_classes, int n_buckets, double *uses, hipStream_t s)
{
    hipLaunchKernelGGL(trellis_uses_kernel, dim3(n_classes, n_buckets), dim3(256), 0, s, row_uses, join_class, rows, n_buckets, uses);
}

void launch_trellis_draw(const TrellisView &v, const SampleRuleHost &rule, const double *alpha, const double *u, int n_draws, int64_t all_rows,
                         int all_utts, int64_t *path, double *cost, double *logp, hipStream_t s)
{
    // the scores of a row carry the temperature already
    SampleRule k;
    const bool greedy = !(rule.temperature > 0.0);
    k.inv_tau = 1.0; k.top_k = greedy ? 1 : rule.top_k; k.top_p = rule.top_p; k.min_p = rule.min_p;
#define SNK_DRAW(E_) hipLaunchKernelGGL((trellis_draw_kernel<E_>), dim3(v.n_utts, n_draws), dim3(64), 0, s, v.cand, v.tdist, v.C, alpha, v.off, v.first, v.c0, \
                                        v.K, v.n_units, v.inv_tau, k, greedy, u, all_rows, all_utts, path, cost, logp)
    if (v.K <= 64) SNK_DRAW(1);
    else if (v.K <= 128) SNK_DRAW(2);
    else SNK_DRAW(4);
#undef SNK_DRAW
}

}  // namespace snk
