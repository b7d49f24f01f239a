// Draws from rows of scores with temperature, top-k, top-p and min-p (snk_sample_rows; the mathematics: sample_device.h).
#include "sample_device.h"
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace snk {

template <typename T> __device__ __forceinline__ double score_value(T v);
template <> __device__ __forceinline__ double score_value<double>(double v) { return v; }
template <> __device__ __forceinline__ double score_value<float>(float v) { return (double)v; }
template <> __device__ __forceinline__ double score_value<__half>(__half v) { return (double)__half2float(v); }
template <> __device__ __forceinline__ double score_value<__hip_bfloat16>(__hip_bfloat16 v) { return (double)__bfloat162float(v); }

// -0 and +0 are equal scores; NaN takes no part
template <typename T>
__device__ __forceinline__ double score_load(const T *p)
{
    const double v = score_value<T>(*p) + 0.0;
    return v != v ? -__builtin_inf() : v;
}

// keys in the order of the scores
template <typename T> struct ScoreKey { typedef unsigned int type; static constexpr int bits = 32; };
template <> struct ScoreKey<double> { typedef u64 type; static constexpr int bits = 64; };
template <typename T>
__device__ __forceinline__ typename ScoreKey<T>::type score_key(double x)
{
    if constexpr (ScoreKey<T>::bits == 64) {
        const u64 b = (u64)__double_as_longlong(x);
        return (b >> 63) ? ~b : b | 0x8000000000000000ull;
    } else {
        const unsigned int b = __float_as_uint((float)x);
        return (b >> 31) ? ~b : b | 0x80000000u;
    }
}

// ---- rows of up to 64 E scores: a wavefront each ------------------------------------------------------------------------------
template <typename T, int E>
__global__ void __launch_bounds__(256)
sample_rows_wave_kernel(const T *__restrict__ scores, int64_t stride, int64_t R, int V, const double *__restrict__ u, int n_draws,
                        SampleRule call, const double *__restrict__ rules, double unit, int64_t *__restrict__ index,
                        double *__restrict__ logp)
{
    const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= R) return;
    const int lane = threadIdx.x & 63;
    const SampleRule rule = sample_rule(call, rules, r);
    const T *__restrict__ p = scores + r * stride;
    double x[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int i = lane * E + e;
        x[e] = i < V ? score_load(p + i) : -__builtin_inf();
    }
    const double ninf = -__builtin_inf();
    double m = ninf;
#pragma unroll
    for (int e = 0; e < E; ++e) m = fmax(m, x[e]);
    m = wave_max(m);
    if (m == ninf) {
        for (int d = lane; d < n_draws; d += 64) {
            index[r * n_draws + d] = -1;
            if (logp) logp[r * n_draws + d] = ninf;
        }
        return;
    }
    WaveRow<E> row;
#pragma unroll
    for (int e = 0; e < E; ++e) row.w[e] = x[e] == ninf ? 0 : sample_weight(sample_exponent(x[e], m, rule.inv_tau), unit);
    wave_row_keep<E>(x, rule, unit, row);
    const double log_total = log((double)row.total / unit);
    for (int d = 0; d < n_draws; ++d) {
        int l, s;
        const int pick = wave_row_pick<E>(row, u[r * n_draws + d], l, s);
        const double lp = sample_exponent(wave_row_value<E>(x, l, s), m, rule.inv_tau) - log_total;
        if (lane == 0) {
            index[r * n_draws + d] = pick;
            if (logp) logp[r * n_draws + d] = lp;
        }
    }
}

// ---- longer rows: a workgroup each, the row read once per pass ---------------------------------------------------------------------
#define SNK_SAMPLE_TILES 4096
#define SNK_SAMPLE_VEC 4

template <int NT> struct BlockScratch {
    u64 mass[NT / 64];
    u64 count[NT / 64];
    double top[NT / 64];
};

template <int NT>
__device__ __forceinline__ double block_max(double v, BlockScratch<NT> &s)
{
    v = wave_max(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.top[threadIdx.x >> 6] = v;
    __syncthreads();
    double m = s.top[0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) m = fmax(m, s.top[i]);
    return m;
}
// inclusive sums over the threads of both counts; totals to every thread
template <int NT>
__device__ __forceinline__ void block_scan2(u64 &a, u64 &b, u64 &ta, u64 &tb, BlockScratch<NT> &s)
{
    a = wave_scan_add(a);
    b = wave_scan_add(b);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) { s.mass[threadIdx.x >> 6] = a; s.count[threadIdx.x >> 6] = b; }
    __syncthreads();
    u64 xa = 0, xb = 0;
    ta = 0; tb = 0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) {
        if (i < (int)(threadIdx.x >> 6)) { xa += s.mass[i]; xb += s.count[i]; }
        ta += s.mass[i]; tb += s.count[i];
    }
    a += xa; b += xb;
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT)
sample_rows_block_kernel(const T *__restrict__ scores, int64_t stride, int64_t V, const double *__restrict__ u, int n_draws,
                         SampleRule call, const double *__restrict__ rules, double unit, int64_t *__restrict__ index,
                         double *__restrict__ logp)
{
    typedef typename ScoreKey<T>::type Key;
    constexpr int BITS = ScoreKey<T>::bits;
    constexpr int64_t TILE = (int64_t)NT * SNK_SAMPLE_VEC;
    __shared__ BlockScratch<NT> scratch;
    __shared__ u64 hist_mass[256];
    __shared__ unsigned int hist_count[256];
    __shared__ u64 tile_mass[SNK_SAMPLE_TILES];
    __shared__ unsigned int tile_ties[SNK_SAMPLE_TILES];
    __shared__ u64 sh_a, sh_b;
    __shared__ unsigned int sh_digit;

    const int tid = threadIdx.x;
    const int64_t r = blockIdx.x;
    const SampleRule rule = sample_rule(call, rules, r);
    const T *__restrict__ p = scores + r * stride;
    const double ninf = -__builtin_inf();

    double m = ninf;
    for (int64_t i = tid; i < V; i += NT) m = fmax(m, score_load(p + i));
    m = block_max<NT>(m, scratch);
    if (m == ninf) {
        for (int d = tid; d < n_draws; d += NT) {
            index[r * n_draws + d] = -1;
            if (logp) logp[r * n_draws + d] = ninf;
        }
        return;
    }

    // the order's prefix by radix: eight bits of the key a pass, from the top; what lies above the digit is known, the elements that
    // share it go on.  Counts and masses are integers: the order of the atomics does not show.
    Key cut = 0;
    bool all = true;
    u64 n_tie = 0;
    auto search = [&](bool by_mass, u64 want) -> bool {          // false: fewer than `want`: the prefix is the whole row
        Key prefix = 0;
        u64 above = 0;
        for (int shift = BITS - 8; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += NT) { hist_count[i] = 0; hist_mass[i] = 0; }
            __syncthreads();
            for (int64_t i = tid; i < V; i += NT) {
                const double x = score_load(p + i);
                if (x == ninf) continue;
                const Key k = score_key<T>(x);
                if (shift + 8 < BITS && (k >> (shift + 8)) != (prefix >> (shift + 8))) continue;
                const int digit = (int)((k >> shift) & 255);
                if (by_mass) {
                    const u64 w = sample_weight(sample_exponent(x, m, rule.inv_tau), unit);
                    if (w) atomicAdd(&hist_mass[digit], w);
                }
                atomicAdd(&hist_count[digit], 1u);
            }
            __syncthreads();
            if (tid < 64) {
                // lane l: digits 255 - 4 l .. 252 - 4 l, from the top
                u64 v[4], sum = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) { const int d = 255 - (4 * tid + j); v[j] = by_mass ? hist_mass[d] : (u64)hist_count[d]; sum += v[j]; }
                const u64 upto = wave_scan_add(sum);
                const u64 hit = __ballot(above + upto >= want);
                if (!hit) { if (tid == 0) sh_digit = 256; }
                else if (tid == __ffsll((long long)hit) - 1) {
                    u64 a = above + upto - sum;
                    for (int j = 0; j < 4; ++j) {
                        if (a + v[j] >= want) { sh_digit = 255 - (4 * tid + j); sh_a = a; break; }
                        a += v[j];
                    }
                }
            }
            __syncthreads();
            const unsigned int digit = sh_digit;
            if (digit == 256) { __syncthreads(); return false; }
            above = sh_a;
            prefix |= (Key)digit << shift;
            if (shift == 0) {
                const u64 c = hist_count[digit];
                if (by_mass) {
                    const u64 each = hist_mass[digit] / c;
                    n_tie = (want - above + each - 1) / each;
                } else n_tie = want - above;
            }
            __syncthreads();
        }
        cut = prefix;
        all = false;
        return true;
    };
    // mass and equal elements of what is kept, per tile
    auto element = [&](double x, bool use_min, u64 &w, unsigned int &tie) {
        w = 0; tie = 0;
        if (x == ninf) return;
        const Key k = score_key<T>(x);
        if (!all && k < cut) return;
        const double e = sample_exponent(x, m, rule.inv_tau);
        if (e < SNK_SAMPLE_FLOOR) return;
        const double v = exp(e);
        if (use_min && v < rule.min_p) return;
        if (!all && k == cut) { tie = 1; return; }
        w = sample_fix(v, unit);
    };
    const int64_t n_tiles = (V + TILE - 1) / TILE;
    u64 w_tie = 0;
    auto totals = [&](bool use_min) -> u64 {
        if (tid == 0) { sh_a = 0; sh_b = 0; }
        for (int i = tid; i < n_tiles; i += NT) { tile_mass[i] = 0; tile_ties[i] = 0; }
        __syncthreads();
        u64 tw = 0;
        for (int64_t t = 0; t < n_tiles; ++t) {
            u64 mass = 0;
            unsigned int ties = 0;
            for (int j = 0; j < SNK_SAMPLE_VEC; ++j) {
                const int64_t i = t * TILE + (int64_t)j * NT + tid;
                if (i >= V) break;
                const double x = score_load(p + i);
                u64 w; unsigned int q;
                element(x, use_min, w, q);
                mass += w; ties += q;
                if (q) tw = sample_weight(sample_exponent(x, m, rule.inv_tau), unit);
            }
            mass = wave_add(mass);
            const u64 all_ties = wave_add((u64)ties);
            if ((tid & 63) == 0) {
                if (mass) atomicAdd(&tile_mass[t], mass);
                if (all_ties) atomicAdd(&tile_ties[t], (unsigned int)all_ties);
            }
        }
        if (tw) sh_b = tw;                                      // (every holder writes the same value)
        __syncthreads();
        w_tie = sh_b;
        u64 mass = 0, ties = 0, tm, tt;
        for (int i = tid; i < n_tiles; i += NT) { mass += tile_mass[i]; ties += tile_ties[i]; }
        block_scan2<NT>(mass, ties, tm, tt, scratch);
        return tm + w_tie * (tt < n_tie ? tt : n_tie);
    };
    if (rule.top_k > 0 && rule.top_k < V) search(false, (u64)rule.top_k);
    if (rule.top_p < 1.0) {
        const u64 total = totals(false);
        search(true, sample_reach(rule.top_p, total));
    }
    const u64 total = totals(rule.min_p > 0.0);
    const double log_total = log((double)total / unit);

    for (int d = 0; d < n_draws; ++d) {
        const u64 t = sample_exceed(u[r * n_draws + d], total);
        // the tile: the first wavefront walks the tiles' sums
        if (tid < 64) {
            u64 mass0 = 0, ties0 = 0;
            for (int64_t b = 0; b < n_tiles; b += 64) {
                const u64 mass = b + tid < n_tiles ? tile_mass[b + tid] : 0, ties = b + tid < n_tiles ? tile_ties[b + tid] : 0;
                const u64 cm = mass0 + wave_scan_add(mass), ct = ties0 + wave_scan_add(ties);
                const u64 hit = __ballot(cm + w_tie * (ct < n_tie ? ct : n_tie) > t);
                if (hit) {
                    const int l = __ffsll((long long)hit) - 1;
                    if (tid == l) { sh_digit = (unsigned int)(b + l); sh_a = cm - mass; sh_b = ct - ties; }
                    break;
                }
                mass0 = __shfl(cm, 63, 64); ties0 = __shfl(ct, 63, 64);
            }
        }
        __syncthreads();
        const int64_t base = (int64_t)sh_digit * TILE + (int64_t)tid * SNK_SAMPLE_VEC;
        const u64 mass0 = sh_a, ties0 = sh_b;
        u64 w[SNK_SAMPLE_VEC]; unsigned int q[SNK_SAMPLE_VEC];
        double x[SNK_SAMPLE_VEC];
        u64 mass = 0, ties = 0;
#pragma unroll
        for (int j = 0; j < SNK_SAMPLE_VEC; ++j) {
            x[j] = base + j < V ? score_load(p + base + j) : ninf;
            element(x[j], rule.min_p > 0.0, w[j], q[j]);
            mass += w[j]; ties += q[j];
        }
        u64 cm = mass, ct = ties, ignore_a, ignore_b;
        block_scan2<NT>(cm, ct, ignore_a, ignore_b, scratch);
        u64 am = mass0 + cm - mass, at = ties0 + ct - ties;
#pragma unroll
        for (int j = 0; j < SNK_SAMPLE_VEC; ++j) {
            const u64 lo = am + w_tie * (at < n_tie ? at : n_tie);
            am += w[j]; at += q[j];
            const u64 hi = am + w_tie * (at < n_tie ? at : n_tie);
            if (lo <= t && t < hi) {
                index[r * n_draws + d] = base + j;
                if (logp) logp[r * n_draws + d] = sample_exponent(x[j], m, rule.inv_tau) - log_total;
            }
        }
        __syncthreads();
    }
}

template <typename T>
static void launch_sample_t(const T *scores, int64_t stride, int64_t R, int64_t V, const double *u, int n_draws, const SampleRule &rule,
                            const double *rules, int64_t *index, double *logp, hipStream_t s)
{
    int s_bits = 62;
    for (int64_t v = 1; v < V; v <<= 1) --s_bits;
    if (s_bits > 51) s_bits = 51;
    const double unit = (double)(1ull << s_bits);
#define SNK_WAVE(E_) hipLaunchKernelGGL((sample_rows_wave_kernel<T, E_>), dim3((unsigned)((R + 3) / 4)), dim3(256), 0, s, scores, stride, R, (int)V, u, n_draws, rule, rules, unit, index, logp)
    if (V <= 64) SNK_WAVE(1);
    else if (V <= 128) SNK_WAVE(2);
    else if (V <= 256) SNK_WAVE(4);
    else if (V <= 512) SNK_WAVE(8);
    else if (V <= 1024) SNK_WAVE(16);
    else
        hipLaunchKernelGGL((sample_rows_block_kernel<T, 1024>), dim3((unsigned)R), dim3(1024), 0, s, scores, stride, V, u, n_draws, rule, rules, unit,
                           index, logp);
#undef SNK_WAVE
}

int64_t sample_rows_max() { return (int64_t)SNK_SAMPLE_TILES * 1024 * SNK_SAMPLE_VEC; }

void launch_sample_rows(const void *scores, int dtype, int64_t stride, int64_t R, int64_t V, const double *u, int n_draws,
                        const SampleRuleHost &rule, const double *rules, int64_t *index, double *logp, hipStream_t s)
{
    SampleRule k;
    k.inv_tau = rule.temperature > 0.0 ? 1.0 / rule.temperature : __builtin_inf();
    k.top_k = rule.temperature > 0.0 ? rule.top_k : 1;
    k.top_p = rule.top_p;
    k.min_p = rule.min_p;
    if (dtype == 0) launch_sample_t((const double *)scores, stride, R, V, u, n_draws, k, rules, index, logp, s);
    else if (dtype == 1) launch_sample_t((const float *)scores, stride, R, V, u, n_draws, k, rules, index, logp, s);
    else if (dtype == 2) launch_sample_t((const __half *)scores, stride, R, V, u, n_draws, k, rules, index, logp, s);
    else launch_sample_t((const __hip_bfloat16 *)scores, stride, R, V, u, n_draws, k, rules, index, logp, s);
}

}  // namespace snk
