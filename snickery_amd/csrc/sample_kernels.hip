// Draws from rows of scores with temperature, top-k, top-p and min-p (snk_sample_rows; the mathematics: sample_device.h).
#include "sample_device.h"
#include <algorithm>
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
// A row is read once, its sums are data-parallel moves within the wavefront, and a lane has a draw.  One row of 30: 2.9 us, a launch;
// 600 rows of 100, top_p 0.9: 9 us; 19200 rows of 100, top_k 40, top_p 0.95, min_p 0.02, 8 draws: 50 us, 0.4 TB/s: bound by the search
// for the cuts (wave_row_keep).  8.4 million float32 scores, top_p 0.9: 130 us in rows of 128, 89 of 256, 85 of 512, 96 of 1024.
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
    for (int d0 = 0; d0 < n_draws; d0 += 64) {                  // a lane has a draw
        const int n = n_draws - d0 < 64 ? n_draws - d0 : 64;
        const int64_t at = r * n_draws + d0 + lane;
        const int pick = wave_row_picks<E>(row, lane < n ? u[at] : 0.0, n);
        if (lane < n) {
            index[at] = pick;
            if (logp) logp[at] = sample_exponent(score_load(p + pick), m, rule.inv_tau) - log_total;
        }
    }
}

// ---- longer rows without a workspace: a workgroup each, the row read once per pass ------------------------------------------------------
// For rows that the passes below leave over and for captured calls without a workspace.  Bound by what one compute unit reads: a row of
// 1048576 float32 3.2 ms, 37 rows of 50003 178 us.
#define SNK_SAMPLE_TILES 2048
#define SNK_SAMPLE_VEC 8

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
                         SampleRule call, const double *__restrict__ rules, double unit, const int *__restrict__ only, int64_t *__restrict__ index,
                         double *__restrict__ logp)
{
    if (only && !only[blockIdx.x]) return;                      // (rows that the kernels below left over)
    typedef typename ScoreKey<T>::type Key;
    constexpr int BITS = ScoreKey<T>::bits;
    constexpr int64_t TILE = (int64_t)NT * SNK_SAMPLE_VEC;
    __shared__ BlockScratch<NT> scratch;
    __shared__ u64 hist_mass[256], hist_more[256];
    __shared__ u64 tile_mass[SNK_SAMPLE_TILES], tile_more[SNK_SAMPLE_TILES];      // the count: scores equal to the cut
    __shared__ u128 sh_above;
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
    auto search = [&](bool by_mass, u128 want) -> bool {         // false: fewer than `want`: the prefix is the whole row
        Key prefix = 0;
        u128 above = 0;
        auto amount = [&](u64 mass, u64 more) -> u128 { return by_mass ? sample_sum(mass, more) : (u128)sample_count(more); };
        for (int shift = BITS - 8; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += NT) { hist_more[i] = 0; hist_mass[i] = 0; }
            __syncthreads();
            for (int64_t i = tid; i < V; i += NT) {
                const double x = score_load(p + i);
                if (x == ninf) continue;
                const Key k = score_key<T>(x);
                if (shift + 8 < BITS && (k >> (shift + 8)) != (prefix >> (shift + 8))) continue;
                const int digit = (int)((k >> shift) & 255);
                u64 w = 0;
                if (by_mass) {
                    w = sample_weight(sample_exponent(x, m, rule.inv_tau), unit);
                    if (w) atomicAdd(&hist_mass[digit], w);
                }
                atomicAdd(&hist_more[digit], SNK_MORE_ONE + sample_more(w));
            }
            __syncthreads();
            if (tid < 64) {
                // lane l: digits 255 - 4 l .. 252 - 4 l, from the top
                u64 mass = 0, more = 0;
                for (int j = 0; j < 4; ++j) { const int d = 255 - (4 * tid + j); mass += hist_mass[d]; more += hist_more[d]; }
                const u64 upto_mass = wave_scan_add(mass), upto_more = wave_scan_add(more);
                const u64 hit = __ballot(above + amount(upto_mass, upto_more) >= want);
                if (!hit) { if (tid == 0) sh_digit = 256; }
                else if (tid == __ffsll((long long)hit) - 1) {
                    u128 a = above + amount(upto_mass - mass, upto_more - more);
                    for (int j = 0; j < 4; ++j) {
                        const int d = 255 - (4 * tid + j);
                        const u128 v = amount(hist_mass[d], hist_more[d]);
                        if (a + v >= want) { sh_digit = d; sh_above = a; break; }
                        a += v;
                    }
                }
            }
            __syncthreads();
            const unsigned int digit = sh_digit;
            if (digit == 256) { __syncthreads(); return false; }
            above = sh_above;
            prefix |= (Key)digit << shift;
            if (shift == 0) {                                   // (equal scores, equal weights)
                const u64 more = hist_more[digit], c = sample_count(more), upper = (more & (SNK_MORE_ONE - 1)) / c;
                const u64 each = (upper << 40) + (hist_mass[digit] - ((upper * c) << 40)) / c;
                n_tie = by_mass ? sample_ties(want - above, each) : (u64)(want - above);
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
        if (!(e >= SNK_SAMPLE_FLOOR)) return;
        const double v = sample_exp(e);
        if (use_min && (double)sample_fix(v, unit) < rule.min_p * unit) return;
        if (!all && k == cut) { tie = 1; return; }
        w = sample_fix(v, unit);
    };
    const int64_t n_tiles = (V + TILE - 1) / TILE;
    u64 w_tie = 0;
    auto totals = [&](bool use_min) -> u128 {
        if (tid == 0) sh_b = 0;
        for (int i = tid; i < n_tiles; i += NT) { tile_mass[i] = 0; tile_more[i] = 0; }
        __syncthreads();
        u64 tw = 0;
        for (int64_t t = 0; t < n_tiles; ++t) {
            u64 mass = 0, more = 0;
            for (int j = 0; j < SNK_SAMPLE_VEC; ++j) {
                const int64_t i = t * TILE + (int64_t)j * NT + tid;
                if (i >= V) break;
                const double x = score_load(p + i);
                u64 w; unsigned int q;
                element(x, use_min, w, q);
                mass += w; more += sample_more(w) + (q ? SNK_MORE_ONE : 0);
                if (q) tw = sample_weight(sample_exponent(x, m, rule.inv_tau), unit);
            }
            mass = wave_add(mass);
            more = wave_add(more);
            if ((tid & 63) == 0) {
                if (mass) atomicAdd(&tile_mass[t], mass);
                if (more) atomicAdd(&tile_more[t], more);
            }
        }
        if (tw) sh_b = tw;                                      // (every holder writes the same value)
        __syncthreads();
        w_tie = sh_b;
        u64 mass = 0, more = 0, tm, tt;
        for (int i = tid; i < n_tiles; i += NT) { mass += tile_mass[i]; more += tile_more[i]; }
        block_scan2<NT>(mass, more, tm, tt, scratch);
        return sample_sum(tm, tt) + (u128)w_tie * min(sample_count(tt), n_tie);
    };
    if (rule.top_k > 0 && rule.top_k < V) search(false, (u128)rule.top_k);
    if (rule.top_p < 1.0) {
        const u128 total = totals(false);
        search(true, sample_reach(rule.top_p, total));
    }
    const u128 total = totals(rule.min_p > 0.0);
    const double log_total = log(sample_double(total) / unit);

    for (int d = 0; d < n_draws; ++d) {
        const u128 t = sample_exceed(u[r * n_draws + d], total);
        // the tile: the first wavefront walks the tiles' sums
        if (tid == 0) {
            sh_digit = 0xffffffffu;
            index[r * n_draws + d] = -1;
            if (logp) logp[r * n_draws + d] = ninf;
        }
        if (tid < 64) {
            u64 mass0 = 0, more0 = 0;
            for (int64_t b = 0; b < n_tiles; b += 64) {
                const u64 mass = b + tid < n_tiles ? tile_mass[b + tid] : 0, more = b + tid < n_tiles ? tile_more[b + tid] : 0;
                const u64 cm = mass0 + wave_scan_add(mass), ct = more0 + wave_scan_add(more);
                const u64 hit = __ballot(sample_sum(cm, ct) + (u128)w_tie * min(sample_count(ct), n_tie) > t);
                if (hit) {
                    const int l = __ffsll((long long)hit) - 1;
                    if (tid == l) {                             // what is left of t in the tile, and the equal scores before it
                        const u64 before = sample_count(ct - more);
                        sh_digit = (unsigned int)(b + l);
                        sh_a = (u64)(t - (sample_sum(cm - mass, ct - more) + (u128)w_tie * min(before, n_tie)));
                        sh_b = before;
                    }
                    break;
                }
                mass0 = wave_lane(cm, 63); more0 = wave_lane(ct, 63);
            }
        }
        __syncthreads();
        if (sh_digit == 0xffffffffu) { __syncthreads(); continue; }      // (only where the scores changed under the call)
        const int64_t base = (int64_t)sh_digit * TILE + (int64_t)tid * SNK_SAMPLE_VEC;
        const u64 goal = sh_a, ties0 = sh_b, kept0 = min(ties0, n_tie);
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
        u64 am = cm - mass, at = ties0 + ct - ties;
#pragma unroll
        for (int j = 0; j < SNK_SAMPLE_VEC; ++j) {
            const u64 lo = am + w_tie * (min(at, n_tie) - kept0);
            am += w[j]; at += q[j];
            const u64 hi = am + w_tie * (min(at, n_tie) - kept0);
            if (lo <= goal && goal < hi) {
                index[r * n_draws + d] = base + j;
                if (logp) logp[r * n_draws + d] = sample_exponent(x[j], m, rule.inv_tau) - log_total;
            }
        }
        __syncthreads();
    }
}

__device__ __forceinline__ int score_bin(double e, double scale, int bins)
{
    const double b = -e * scale;
    return b < (double)(bins - 1) ? (int)b : bins - 1;
}

// ---- rows of up to 8 NT scores: a workgroup each, the row in registers ---------------------------------------------------------------
// One read of the row and one launch.  A prefix of the order is found as below for longer rows -- the bin of the exponent in which the
// count or the mass reaches its goal, then the place among that bin's scores by radix on their keys -- but bins and digits are in LDS
// and the scores never leave the registers: no list, nothing left over, no workspace that a captured graph would share.  A thread's
// scores are neighbours, so that the ranks of equal ones and the kept mass are scans over the threads.  128 registers at most, some
// spilled: with 190 and none the rows of 2048 and 4096 scores took 86 and 115 us instead of 74 and 78.  Bound by the scans' and the
// radix's barriers, some 30 of them.  float32, top_p 0.9, 8.4 million scores in all:
//     scores a row     1025   2000   4096   8192 us, one row 8192
//     this              128     71     74    113              27
//     passes below      677    370    214    147              50
// Sixteen scores a thread, rows of 16384: 169 us, the passes below 110.
#define SNK_HELD_MOST 8192
template <typename T, int NT, int EACH>
__global__ void __launch_bounds__(NT, 4)
sample_rows_held_kernel(const T *__restrict__ scores, int64_t stride, int V, const double *__restrict__ u, int n_draws, SampleRule call,
                        const double *__restrict__ rules, double unit, int64_t *__restrict__ index, double *__restrict__ logp)
{
    constexpr int BINS = 1024, PER = BINS / NT, NW = NT / 64;
    __shared__ BlockScratch<NT> scratch;
    __shared__ u64 bin_mass[BINS], digit_mass[256], sh_above;
    __shared__ unsigned int bin_count[BINS], digit_count[256];
    __shared__ double ends[2 * NW];
    __shared__ int sh_bin, sh_digit;
    const int tid = threadIdx.x, at = tid * EACH;
    const int64_t r = blockIdx.x;
    const SampleRule rule = sample_rule(call, rules, r);
    const T *__restrict__ p = scores + r * stride;
    const double inf = __builtin_inf();
    double x[EACH];
    if ((((uintptr_t)p) & 15) == 0 && at + EACH <= V) {
        union { uint4 w[EACH * sizeof(T) / 16]; T v[EACH]; } raw;
#pragma unroll
        for (int j = 0; j < (int)(EACH * sizeof(T) / 16); ++j) raw.w[j] = reinterpret_cast<const uint4 *>(p + at)[j];
#pragma unroll
        for (int j = 0; j < EACH; ++j) x[j] = score_load(raw.v + j);
    } else {
#pragma unroll
        for (int j = 0; j < EACH; ++j) x[j] = at + j < V ? score_load(p + at + j) : -inf;
    }
    // largest and smallest of the scores that `in` marks
    auto extremes = [&](unsigned int in, double &most, double &least) {
        most = -inf; least = inf;
#pragma unroll
        for (int j = 0; j < EACH; ++j)
            if ((in >> j) & 1) { most = fmax(most, x[j]); least = fmin(least, x[j]); }
        most = wave_max(most);
        least = -wave_max(-least);
        __syncthreads();
        if ((tid & 63) == 0) { ends[tid >> 6] = most; ends[NW + (tid >> 6)] = least; }
        __syncthreads();
        for (int i = 0; i < NW; ++i) { most = fmax(most, ends[i]); least = fmin(least, ends[NW + i]); }
    };
    unsigned int in = 0;
#pragma unroll
    for (int j = 0; j < EACH; ++j) in |= x[j] > -inf ? 1u << j : 0;
    double m, least;
    extremes(in, m, least);
    if (m == -inf) {
        for (int d = tid; d < n_draws; d += NT) {
            index[r * n_draws + d] = -1;
            if (logp) logp[r * n_draws + d] = m;
        }
        return;
    }
    u64 q[EACH];                                                // weights; 0: not kept
    unsigned int bins[EACH / 2];                                // two scores' bins a word
    const bool counted = rule.top_k > 0 && rule.top_k < V, shared = rule.top_p < 1.0;
    const double range = fmin(-sample_exponent(least, m, rule.inv_tau), -SNK_SAMPLE_FLOOR);
    const double scale = range > 0.0 ? fmin((double)BINS / range, 1e300) : 0.0;
    for (int i = tid; i < BINS; i += NT) { bin_mass[i] = 0; bin_count[i] = 0; }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        const double e = sample_exponent(x[j], m, rule.inv_tau);
        q[j] = x[j] == -inf ? 0 : sample_weight(e, unit);
        const unsigned int b = q[j] ? score_bin(e, scale, BINS) : 0;
        if (q[j] && (counted || shared)) {
            atomicAdd(&bin_mass[b], q[j]);
            atomicAdd(&bin_count[b], 1u);
        }
        bins[j / 2] = j & 1 ? bins[j / 2] | b << 16 : b;
    }
    __syncthreads();
    u64 total = 0;                                              // mass that top_k keeps
#pragma unroll 1
    for (int by_mass = 0; by_mass < 2; ++by_mass) {
        if (by_mass ? !shared : !counted) continue;
        // the bin
        u64 vm[PER], vc[PER], sm = 0, sc = 0, total_m, total_c;
#pragma unroll
        for (int i = 0; i < PER; ++i) { vm[i] = bin_mass[tid * PER + i]; vc[i] = bin_count[tid * PER + i]; sm += vm[i]; sc += vc[i]; }
        if (tid == 0) sh_bin = -1;
        u64 um = sm, uc = sc;
        block_scan2<NT>(um, uc, total_m, total_c, scratch);
        const u64 want = by_mass ? sample_reach(rule.top_p, total ? total : total_m) : (u64)rule.top_k;
        const u64 upto = by_mass ? um : uc;
        u64 a = upto - (by_mass ? sm : sc);
        if (a < want && upto >= want) {
            bool found = false;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const u64 n = by_mass ? vm[i] : vc[i];
                if (!found && a + n >= want) { found = true; sh_bin = tid * PER + i; sh_above = a; }
                a += n;
            }
        }
        __syncthreads();
        const int bin = sh_bin;
        u64 above = sh_above;
        __syncthreads();
        if (bin < 0) continue;                                  // fewer scores than the goal
        // its scores, and the one among them at which the order reaches the goal
        in = 0;
#pragma unroll
        for (int j = 0; j < EACH; ++j)
            in |= q[j] && (int)((bins[j / 2] >> (j & 1 ? 16 : 0)) & 0xffff) == bin ? 1u << j : 0;
        double high, low;
        extremes(in, high, low);
        const u64 key_min = score_key<double>(low), key_max = score_key<double>(high);
        u64 key = key_min;
        if (key_min != key_max) {
            // (keys that differ share their leading bits: start at the first digit in which they do)
            int shift = ((63 - __clzll((long long)(key_min ^ key_max))) >> 3) << 3;
            u64 prefix = shift + 8 < 64 ? (key_min >> (shift + 8)) << (shift + 8) : 0;
            for (; shift >= 0; shift -= 8) {
                for (int i = tid; i < 256; i += NT) { digit_mass[i] = 0; digit_count[i] = 0; }
                if (tid == 0) { sh_digit = 0; sh_above = above; }
                __syncthreads();
#pragma unroll
                for (int j = 0; j < EACH; ++j)
                    if ((in >> j) & 1) {
                        double v = x[j];
                        asm volatile("" : "+v"(v));             // (or all the keys are made before the loop and kept beside the scores)
                        const u64 k = score_key<double>(v);
                        if (shift + 8 < 64 && (k >> (shift + 8)) != (prefix >> (shift + 8))) continue;
                        const int digit = (int)((k >> shift) & 255);
                        if (by_mass) atomicAdd(&digit_mass[digit], q[j]);
                        else atomicAdd(&digit_count[digit], 1u);
                    }
                __syncthreads();
                if (tid < 64) {
                    // lane l: digits 255 - 4 l .. 252 - 4 l, from the top
                    u64 v[4], sum = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) { const int d = 255 - (4 * tid + j); v[j] = by_mass ? digit_mass[d] : (u64)digit_count[d]; sum += v[j]; }
                    const u64 reach = wave_scan_add(sum), hit = __ballot(above + reach >= want);
                    if (hit && tid == __ffsll((long long)hit) - 1) {
                        u64 b = above + reach - sum;
                        for (int j = 0; j < 4; ++j) {
                            if (b + v[j] >= want) { sh_digit = 255 - (4 * tid + j); sh_above = b; break; }
                            b += v[j];
                        }
                    }
                }
                __syncthreads();
                above = sh_above;
                prefix |= (u64)sh_digit << shift;
                __syncthreads();
            }
            key = prefix;
        }
        const double cut = __longlong_as_double((long long)((key >> 63) ? key & 0x7fffffffffffffffull : ~key));
        const u64 each = sample_weight(sample_exponent(cut, m, rule.inv_tau), unit);
        u64 n_tie = by_mass ? (each ? (want - above + each - 1) / each : 0) : want - above;
        u64 ties = 0, mass = 0, all_ties, all_mass;
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            if (q[j] && x[j] == cut) ++ties;
            if (x[j] > cut) mass += q[j];
        }
        u64 rank = ties;
        block_scan2<NT>(rank, mass, all_ties, all_mass, scratch);
        rank -= ties;                                           // equal ones before this thread's
        if (n_tie > all_ties) n_tie = all_ties;
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            const bool tie = q[j] && x[j] == cut;
            if (x[j] < cut || (tie && rank >= n_tie)) q[j] = 0;
            rank += tie ? 1 : 0;
        }
        total = all_mass + each * n_tie;
    }
    u64 mass = 0, none = 0, kept, unused;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        if (rule.min_p > 0.0 && (double)q[j] < rule.min_p * unit) q[j] = 0;
        mass += q[j];
    }
    u64 upto = mass;
    block_scan2<NT>(upto, none, kept, unused, scratch);
    const double log_kept = logp ? log((double)kept / unit) : 0.0;
    for (int d = 0; d < n_draws; ++d) {
        const u64 t = sample_exceed(u[r * n_draws + d], kept);
        if (t >= upto || t < upto - mass) continue;
        u64 c = upto - mass;
        int pick = at;                                          // weights that do not reach t are passed over
#pragma unroll
        for (int j = 0; j < EACH - 1; ++j) {
            c += q[j];
            pick += c <= t ? 1 : 0;
        }
        index[r * n_draws + d] = pick;
        if (logp) logp[r * n_draws + d] = sample_exponent(score_load(p + pick), m, rule.inv_tau) - log_kept;
    }
}

// ---- longer rows, every pass over all of the chip ----------------------------------------------------------------------------------
// A row is cut into chunks of SNK_CHUNK scores, a workgroup each:
//   extremes   the chunks' largest and smallest score
//   histogram  count and mass by bins of the exponent (m - x) / tau, as many bins as the row's own range needs
//   boundary   the bin in which the order reaches its goal (a count, or a share of the mass); the bin's scores go to a list
//   select     the goal's place in the list, by radix on the scores' keys: the cut, and how many equal to it are kept
//   masses     what every chunk keeps
//   draw       the chunk, then the score that a random number falls on
// top_k and top_p take a boundary / select pair each.  Counts and masses are integers: neither the order of the atomics nor the cutting
// shows in a result.  A boundary bin of equal scores needs no list; one of more than SNK_LIST different ones (or a workspace that a
// captured graph would have to share) leaves the row to the kernel above.  us a pass, for 1 row of 1048576 float32, 37 of 50003 float32
// (top_p 0.95: 7.4 MB, 1.5 us at a copy's rate) and 128 of 131071 bfloat16 (top_k 50 and top_p 0.9: 34 MB, 6.6 us):
//     extremes 4, 5, 12    histogram 17, 11, 38    boundary 12, 11, 2 x 21    select 12, 12, 2 x 6    masses 8, 11, 18    draw 13, 13, 10
// The first two are launches and the latency of a few dependent reads each; the third is bound by the float64 work on every score (weight
// and bin, tested again for the boundary).
#define SNK_CHUNK 8192
#define SNK_LIST 16383                          // (weights of 2^50 that 64 bits can add)
#define SNK_BINS_MOST 4096

struct RowState {
    double m, bin_scale;        // largest score, bins per unit of exponent
    double cut;                 // kept: above the cut, and the first n_tie equal to it
    u64 n_tie;
    u128 total;                 // mass of what the goals so far keep
    u128 above, want;
    unsigned int listed, want_bin;
    int all, pad;
};

struct RowsWork {
    RowState *state;
    double *chunk_max, *chunk_min;          // [rows][spans]
    u64 *hist_mass, *hist_more;             // [rows][bins]
    double *list_x;                         // [rows][list]
    u64 *chunk_mass, *chunk_more;           // the count: scores equal to the cut
    int *left;                              // rows for the kernel above
    int64_t span;                           // scores that a workgroup of the first passes takes: chunks, as many as leave workgroups enough
    int bins, chunks, spans;
    unsigned int list;                      // entries of a row's list: SNK_LIST, or the row's length
};

template <typename T> __device__ __forceinline__ double score_bits(const T *v, int j) { return score_load(v + j); }

// every score of [lo, hi) once: 16-byte loads from the first aligned one on
template <typename T, int NT, typename F>
__device__ __forceinline__ void chunk_scores(const T *__restrict__ p, int64_t lo, int64_t hi, F f)
{
    constexpr int VEC = 16 / (int)sizeof(T);
    const int tid = threadIdx.x;
    const int skip = (int)(((16 - ((uintptr_t)(p + lo) & 15)) & 15) / sizeof(T));
    const int64_t a = lo + skip < hi ? lo + skip : hi, n = (hi - a) / VEC, b = a + n * VEC;
    if (lo + tid < a) f(score_load(p + lo + tid), lo + tid);
    // four loads in flight: what f does with a score can keep the next load from being moved ahead of it
    for (int64_t i = tid; i < n; i += 4 * NT) {
        union { uint4 q; T v[VEC]; } u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k * NT < n) u[k].q = *reinterpret_cast<const uint4 *>(p + a + (i + k * NT) * VEC);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k * NT < n) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) f(score_bits(u[k].v, j), a + (i + k * NT) * VEC + j);
            }
    }
    if (b + tid < hi) f(score_load(p + b + tid), b + tid);
}

template <typename T>
__global__ void __launch_bounds__(512)
rows_extremes_kernel(const T *__restrict__ scores, int64_t stride, int64_t V, const RowsWork w)
{
    __shared__ double hi[8], lo[8];
    const int64_t r = blockIdx.y, c = blockIdx.x;
    const int tid = threadIdx.x;
    const double inf = __builtin_inf();
    if (c == 0) {
        for (int i = tid; i < w.bins; i += 512) { w.hist_mass[r * w.bins + i] = 0; w.hist_more[r * w.bins + i] = 0; }
        if (tid == 0) {
            RowState s;
            s.m = -inf; s.bin_scale = 0.0; s.cut = -inf; s.n_tie = 0; s.total = 0; s.above = 0;
            s.listed = 0; s.want_bin = 0; s.all = 1; s.pad = 0; s.want = 0;
            w.state[r] = s;
            w.left[r] = 0;
        }
    }
    double m = -inf, n = inf;
    chunk_scores<T, 512>(scores + r * stride, c * w.span, min((c + 1) * w.span, V), [&](double x, int64_t) {
        m = fmax(m, x);
        n = x > -inf ? fmin(n, x) : n;
    });
    m = wave_max(m);
    n = -wave_max(-n);
    if ((tid & 63) == 0) { hi[tid >> 6] = m; lo[tid >> 6] = n; }
    __syncthreads();
    if (tid == 0) {
        for (int i = 1; i < 8; ++i) { hi[0] = fmax(hi[0], hi[i]); lo[0] = fmin(lo[0], lo[i]); }
        w.chunk_max[r * w.spans + c] = hi[0];
        w.chunk_min[r * w.spans + c] = lo[0];
    }
}

template <typename T>
__global__ void __launch_bounds__(512)
rows_histogram_kernel(const T *__restrict__ scores, int64_t stride, int64_t V, SampleRule call, const double *__restrict__ rules, double unit, const RowsWork w)
{
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ double hi[8], lo[8];
    u64 *mass = reinterpret_cast<u64 *>(smem), *more = mass + w.bins;
    const int64_t r = blockIdx.y, c = blockIdx.x;
    const int tid = threadIdx.x;
    const double inf = __builtin_inf();
    const SampleRule rule = sample_rule(call, rules, r);
    double m = -inf, n = inf;
    for (int i = tid; i < w.spans; i += 512) { m = fmax(m, w.chunk_max[r * w.spans + i]); n = fmin(n, w.chunk_min[r * w.spans + i]); }
    m = wave_max(m);
    n = -wave_max(-n);
    if ((tid & 63) == 0) { hi[tid >> 6] = m; lo[tid >> 6] = n; }
    for (int i = tid; i < w.bins; i += 512) { mass[i] = 0; more[i] = 0; }
    __syncthreads();
    for (int i = 0; i < 8; ++i) { m = fmax(m, hi[i]); n = fmin(n, lo[i]); }
    if (m == -inf) return;                                      // an empty row
    const double range = fmin(-sample_exponent(n, m, rule.inv_tau), -SNK_SAMPLE_FLOOR);
    const double scale = range > 0.0 ? fmin((double)w.bins / range, 1e300) : 0.0;
    if (c == 0 && tid == 0) { w.state[r].m = m; w.state[r].bin_scale = scale; }
    chunk_scores<T, 512>(scores + r * stride, c * w.span, min((c + 1) * w.span, V), [&](double x, int64_t) {
        if (x == -inf) return;
        const double e = sample_exponent(x, m, rule.inv_tau);
        const u64 q = sample_weight(e, unit);
        if (!q) return;
        const int b = score_bin(e, scale, w.bins);
        atomicAdd(&mass[b], q);
        atomicAdd(&more[b], SNK_MORE_ONE + sample_more(q));
    });
    __syncthreads();
    for (int i = tid; i < w.bins; i += 512)
        if (more[i]) { atomicAdd(&w.hist_mass[r * w.bins + i], mass[i]); atomicAdd(&w.hist_more[r * w.bins + i], more[i]); }
}

// by_mass 0: the top_k-th score; 1: where top_p of the mass kept so far is reached
template <typename T>
__global__ void __launch_bounds__(512)
rows_boundary_kernel(const T *__restrict__ scores, int64_t stride, int64_t V, SampleRule call, const double *__restrict__ rules, double unit, int by_mass,
                     const RowsWork w)
{
    constexpr int PER = SNK_BINS_MOST / 512;
    constexpr unsigned int HITS = 2048;
    __shared__ BlockScratch<512> scratch;
    __shared__ int bin_s;
    __shared__ double hit[HITS], ends[16];
    __shared__ unsigned int n_hit, place;
    const int64_t r = blockIdx.y, c = blockIdx.x;
    const int tid = threadIdx.x;
    const SampleRule rule = sample_rule(call, rules, r);
    RowState *st = w.state + r;
    const double m = st->m, scale = st->bin_scale, ninf = -__builtin_inf();
    if (m == ninf || w.left[r]) return;
    if (by_mass ? !(rule.top_p < 1.0) : !(rule.top_k > 0 && rule.top_k < V)) return;
    const u64 *__restrict__ mass = w.hist_mass + r * w.bins;
    const u64 *__restrict__ more = w.hist_more + r * w.bins;
    // every workgroup finds the bin for itself: a thread sums its neighbouring bins, the sums are scanned, the bin is in one thread's
    const int per = w.bins >> 9;
    u64 vm[PER], vc[PER], sm = 0, sc = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        vm[i] = i < per ? mass[tid * per + i] : 0;
        vc[i] = i < per ? more[tid * per + i] : 0;
        sm += vm[i]; sc += vc[i];
    }
    if (tid == 0) bin_s = -1;
    u64 um = sm, uc = sc, total_m, total_c;
    block_scan2<512>(um, uc, total_m, total_c, scratch);
    auto amount = [&](u64 sum, u64 also) -> u128 { return by_mass ? sample_sum(sum, also) : (u128)sample_count(also); };
    const u128 want = by_mass ? sample_reach(rule.top_p, st->all ? sample_sum(total_m, total_c) : st->total) : (u128)rule.top_k;
    u128 a = amount(um - sm, uc - sc);
    if (a < want && amount(um, uc) >= want) {
        bool found = false;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const u128 n = amount(vm[i], vc[i]);
            if (!found && a + n >= want) {
                found = true;
                bin_s = tid * per + i;
                if (c == 0) { st->want = want; st->above = a; st->want_bin = (unsigned int)(tid * per + i); }
            }
            a += n;
        }
    }
    __syncthreads();
    const int bin = bin_s;
    if (bin < 0) {                                              // fewer scores than the goal: all are kept
        if (c == 0 && tid == 0) { st->want_bin = (unsigned int)-1; st->total = sample_sum(total_m, total_c); }
        return;
    }
    // the bin's scores by way of LDS: one place in the row's list is asked for by a workgroup, not one a score (atomics on one address
    // from all XCDs take tens of nanoseconds each)
    if (tid == 0) n_hit = 0;
    __syncthreads();
    const int64_t lo = c * w.span, hi = min((c + 1) * w.span, V);
    auto of_bin = [&](double x) -> bool {
        if (x == ninf) return false;
        const double e = sample_exponent(x, m, rule.inv_tau);
        return e >= SNK_SAMPLE_FLOOR && score_bin(e, scale, w.bins) == bin && sample_weight(e, unit) != 0;
    };
    double most = ninf, least = -ninf;
    chunk_scores<T, 512>(scores + r * stride, lo, hi, [&](double x, int64_t) {
        if (!of_bin(x)) return;
        most = fmax(most, x);
        least = fmin(least, x);
        const unsigned int at = atomicAdd(&n_hit, 1u);
        if (at < HITS) hit[at] = x;
    });
    most = wave_max(most);
    least = -wave_max(-least);
    if ((tid & 63) == 0) { ends[tid >> 6] = most; ends[8 + (tid >> 6)] = least; }
    __syncthreads();
    const unsigned int n = n_hit;
    if (tid == 0) {
        for (int i = 1; i < 8; ++i) { most = fmax(most, ends[i]); least = fmin(least, ends[8 + i]); }
        w.chunk_max[r * w.spans + c] = most;
        w.chunk_min[r * w.spans + c] = least;
        place = n ? atomicAdd(&st->listed, n) : 0;
        n_hit = 0;
    }
    __syncthreads();
    const unsigned int base = place;
    if (n <= HITS) {
        for (unsigned int i = tid; i < n; i += 512)
            if (base + i < w.list) w.list_x[r * w.list + base + i] = hit[i];
    } else
        chunk_scores<T, 512>(scores + r * stride, lo, hi, [&](double x, int64_t) {
            if (!of_bin(x)) return;
            const unsigned int at = base + atomicAdd(&n_hit, 1u);
            if (at < w.list) w.list_x[r * w.list + at] = x;
        });
}

__global__ void __launch_bounds__(1024)
rows_select_kernel(int64_t V, SampleRule call, const double *__restrict__ rules, double unit, int by_mass, const RowsWork w)
{
    __shared__ u64 hist_mass[256], hist_count[256];
    __shared__ u64 sh_above;
    __shared__ unsigned int sh_digit;
    __shared__ u64 red[32];
    __shared__ double ends[32];
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x;
    const SampleRule rule = sample_rule(call, rules, r);
    RowState *st = w.state + r;
    const double m = st->m;
    if (m == -__builtin_inf() || w.left[r]) return;
    if (by_mass ? !(rule.top_p < 1.0) : !(rule.top_k > 0 && rule.top_k < V)) return;
    if ((int)st->want_bin < 0) return;
    const unsigned int n = st->listed;
    u128 need = st->want - st->above;                           // of the bin
    double most = -__builtin_inf(), least = __builtin_inf();    // of the bin's scores
    for (int i = tid; i < w.spans; i += 1024) { most = fmax(most, w.chunk_max[r * w.spans + i]); least = fmin(least, w.chunk_min[r * w.spans + i]); }
    most = wave_max(most);
    least = -wave_max(-least);
    if ((tid & 63) == 0) { ends[tid >> 6] = most; ends[16 + (tid >> 6)] = least; }
    __syncthreads();
    for (int i = 0; i < 16; ++i) { most = fmax(most, ends[i]); least = fmin(least, ends[16 + i]); }
    const u64 key_min = score_key<double>(least), key_max = score_key<double>(most);
    u64 key = key_min;
    u64 ties = n, each = 0;                                     // of the cut's own scores
    if (key_min != key_max) {
        if (n > w.list) { if (tid == 0) w.left[r] = 1; return; }
        u64 prefix = 0, above = 0;
        const u64 want = (u64)need;                             // (the list's sums fit 64 bits)
        // (keys that differ share their leading bits: start at the first digit in which they do)
        int top = 63 - __clzll((long long)(key_min ^ key_max));
        top = (top >> 3) << 3;
        prefix = top + 8 < 64 ? (key >> (top + 8)) << (top + 8) : 0;
        for (int shift = top; shift >= 0; shift -= 8) {
            if (tid < 256) { hist_mass[tid] = 0; hist_count[tid] = 0; }
            if (tid == 0) { sh_digit = 0; sh_above = above; }
            __syncthreads();
            for (unsigned int i = tid; i < n; i += 1024) {
                const double x = w.list_x[r * w.list + i];
                const u64 k = score_key<double>(x);
                if (shift + 8 < 64 && (k >> (shift + 8)) != (prefix >> (shift + 8))) continue;
                const int d = (int)((k >> shift) & 255);
                atomicAdd(&hist_mass[d], sample_weight(sample_exponent(x, m, rule.inv_tau), unit));
                atomicAdd(&hist_count[d], 1ull);
            }
            __syncthreads();
            if (tid < 64) {
                u64 v[4], sum = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) { const int d = 255 - (4 * tid + j); v[j] = by_mass ? hist_mass[d] : hist_count[d]; sum += v[j]; }
                const u64 upto = wave_scan_add(sum), hit = __ballot(above + upto >= want);
                if (hit && tid == __ffsll((long long)hit) - 1) {
                    u64 a = above + upto - sum;
                    for (int j = 0; j < 4; ++j) {
                        if (a + v[j] >= want) { sh_digit = 255 - (4 * tid + j); sh_above = a; break; }
                        a += v[j];
                    }
                }
            }
            __syncthreads();
            above = sh_above;
            prefix |= (u64)sh_digit << shift;
            ties = hist_count[sh_digit];
            __syncthreads();
        }
        key = prefix;
        need = want - above;
    }
    // the cut's value back from its key
    const double cut = __longlong_as_double((long long)((key >> 63) ? key & 0x7fffffffffffffffull : ~key));
    each = sample_weight(sample_exponent(cut, m, rule.inv_tau), unit);
    const u64 n_tie = by_mass ? sample_ties(need, each) : (u64)need;
    // the mass above the cut: whole bins, and the list's scores above it
    u64 mass = 0, more = 0;
    const int bin = (int)st->want_bin;
    for (int i = tid; i < bin; i += 1024) { mass += w.hist_mass[r * w.bins + i]; more += w.hist_more[r * w.bins + i]; }
    if (key_min != key_max)
        for (unsigned int i = tid; i < n; i += 1024) {
            const double x = w.list_x[r * w.list + i];
            const u64 q = x > cut ? sample_weight(sample_exponent(x, m, rule.inv_tau), unit) : 0;
            mass += q; more += sample_more(q);
        }
    mass = wave_add(mass);
    more = wave_add(more);
    if ((tid & 63) == 0) { red[tid >> 6] = mass; red[16 + (tid >> 6)] = more; }
    __syncthreads();
    if (tid == 0) {
        u64 t = 0, also = 0;
        for (int i = 0; i < 16; ++i) { t += red[i]; also += red[16 + i]; }
        st->cut = cut; st->n_tie = n_tie < ties ? n_tie : ties; st->all = 0;
        st->total = sample_sum(t, also) + (u128)each * st->n_tie;
        st->listed = 0;
    }
}

// weight of a score that is kept for certain, or whether it is one of the cut's
__device__ __forceinline__ void row_element(double x, const RowState &st, const SampleRule &rule, double unit, u64 &q, unsigned int &tie)
{
    q = 0; tie = 0;
    if (x == -__builtin_inf() || (!st.all && x < st.cut)) return;
    const u64 weight = sample_weight(sample_exponent(x, st.m, rule.inv_tau), unit);
    if ((double)weight < rule.min_p * unit) return;
    if (!st.all && x == st.cut) tie = weight ? 1 : 0;
    else q = weight;
}

template <typename T>
__global__ void __launch_bounds__(512)
rows_masses_kernel(const T *__restrict__ scores, int64_t stride, int64_t V, SampleRule call, const double *__restrict__ rules, double unit, const RowsWork w)
{
    __shared__ u64 sm[8], sc[8];
    const int64_t r = blockIdx.y, c = blockIdx.x;
    const int tid = threadIdx.x;
    const RowState st = w.state[r];
    if (st.m == -__builtin_inf() || w.left[r]) return;
    const SampleRule rule = sample_rule(call, rules, r);
    u64 mass = 0, more = 0;
    chunk_scores<T, 512>(scores + r * stride, c * SNK_CHUNK, min((c + 1) * SNK_CHUNK, V), [&](double x, int64_t) {
        u64 q; unsigned int t;
        row_element(x, st, rule, unit, q, t);
        mass += q; more += sample_more(q) + (t ? SNK_MORE_ONE : 0);
    });
    mass = wave_add(mass);
    more = wave_add(more);
    if ((tid & 63) == 0) { sm[tid >> 6] = mass; sc[tid >> 6] = more; }
    __syncthreads();
    if (tid == 0) {
        u64 a = 0, b = 0;
        for (int i = 0; i < 8; ++i) { a += sm[i]; b += sc[i]; }
        w.chunk_mass[r * w.chunks + c] = a;
        w.chunk_more[r * w.chunks + c] = b;
    }
}

template <typename T>
__global__ void __launch_bounds__(1024)
rows_draw_kernel(const T *__restrict__ scores, int64_t stride, int64_t V, const double *__restrict__ u, int n_draws, int draw0, SampleRule call,
                 const double *__restrict__ rules, double unit, const RowsWork w, int64_t *__restrict__ index, double *__restrict__ logp)
{
    constexpr int EACH = SNK_CHUNK / 1024;
    __shared__ BlockScratch<1024> scratch;
    __shared__ u64 sh_goal, sh_ties;
    __shared__ int sh_chunk;
    const int64_t r = blockIdx.x, at = r * n_draws + draw0 + blockIdx.y;
    const int tid = threadIdx.x;
    const RowState st = w.state[r];
    if (w.left[r]) return;
    if (st.m == -__builtin_inf()) {
        if (tid == 0) { index[at] = -1; if (logp) logp[at] = st.m; }
        return;
    }
    const SampleRule rule = sample_rule(call, rules, r);
    const u64 each = st.all ? 0 : sample_weight(sample_exponent(st.cut, st.m, rule.inv_tau), unit);
    const u64 n_tie = st.all || (double)each < rule.min_p * unit ? 0 : st.n_tie;
    // chunks: a thread takes `per` neighbours
    const int per = (w.chunks + 1023) / 1024;
    u64 mass = 0, more = 0, total_m, total_t;
    for (int i = 0; i < per; ++i) {
        const int c = tid * per + i;
        if (c < w.chunks) { mass += w.chunk_mass[r * w.chunks + c]; more += w.chunk_more[r * w.chunks + c]; }
    }
    u64 cm = mass, ct = more;
    block_scan2<1024>(cm, ct, total_m, total_t, scratch);
    auto kept = [&](u64 sum, u64 also) -> u128 { return sample_sum(sum, also) + (u128)each * min(sample_count(also), n_tie); };
    const u128 total = kept(total_m, total_t), t = sample_exceed(u[at], total);
    u64 am = cm - mass, an = ct - more;
    if (tid == 0) { sh_chunk = -1; index[at] = -1; if (logp) logp[at] = -__builtin_inf(); }
    __syncthreads();
    for (int i = 0; i < per; ++i) {
        const int c = tid * per + i;
        if (c >= w.chunks) break;
        const u128 lo = kept(am, an);
        const u64 t0 = sample_count(an);
        am += w.chunk_mass[r * w.chunks + c]; an += w.chunk_more[r * w.chunks + c];
        if (lo <= t && t < kept(am, an)) { sh_chunk = c; sh_goal = (u64)(t - lo); sh_ties = t0; }
    }
    __syncthreads();
    if (sh_chunk < 0) return;                                   // (only where the scores changed under the call: nothing is read beyond them)
    const T *__restrict__ p = scores + r * stride;
    const int64_t base = (int64_t)sh_chunk * SNK_CHUNK + tid * EACH;
    const u64 goal = sh_goal, ties0 = sh_ties, kept0 = min(ties0, n_tie);      // what is left of t in the chunk; equal scores before it
    double x[EACH];
    u64 q[EACH], ties = 0; unsigned int k[EACH];
    mass = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        x[i] = base + i < V ? score_load(p + base + i) : -__builtin_inf();
        row_element(x[i], st, rule, unit, q[i], k[i]);
        mass += q[i]; ties += k[i];
    }
    cm = mass; ct = ties;
    block_scan2<1024>(cm, ct, total_m, total_t, scratch);
    am = cm - mass; an = ties0 + ct - ties;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const u64 lo = am + each * (min(an, n_tie) - kept0);
        am += q[i]; an += k[i];
        const u64 hi = am + each * (min(an, n_tie) - kept0);
        if (lo <= goal && goal < hi) {
            index[at] = base + i;
            if (logp) logp[at] = sample_exponent(x[i], st.m, rule.inv_tau) - log(sample_double(total) / unit);
        }
    }
}

static int rows_bins(int64_t V) { int b = 1024; while (b < SNK_BINS_MOST && b * 256 < V) b <<= 1; return b; }
static int64_t rows_chunks(int64_t V) { return (V + SNK_CHUNK - 1) / SNK_CHUNK; }
// What every workgroup of the first three passes does besides its scores -- the row's largest, the histogram, the boundary's bin -- is as
// much work as a chunk or two.  So a workgroup takes several chunks where 512 workgroups are left, half of what runs at once (boundary of
// 128 rows of 131071 bfloat16: 33 us with a chunk each, 24 with two, 20 with four).
static int64_t rows_span(int64_t R, int64_t V)
{
    int64_t span = SNK_CHUNK;
    while (span < 8 * SNK_CHUNK && R * ((V + 2 * span - 1) / (2 * span)) >= 512) span *= 2;
    return span;
}
static unsigned int rows_list(int64_t V) { return V < SNK_LIST ? (unsigned int)V : SNK_LIST; }
#define SNK_ALIGNED(bytes_) (((size_t)(bytes_) + 255) & ~(size_t)255)

// rows that no workgroup holds: bytes of workspace a row takes, and how many rows go together at most (2 GB)
size_t sample_rows_work_bytes(int64_t V)
{
    if (V <= SNK_HELD_MOST) return 0;
    const size_t c = (size_t)rows_chunks(V), b = (size_t)rows_bins(V);
    return sizeof(RowState) + c * (2 * sizeof(double) + 2 * sizeof(u64)) + b * 2 * sizeof(u64) + rows_list(V) * sizeof(double) + sizeof(int);
}
int64_t sample_rows_together(int64_t R, int64_t V)
{
    const size_t each = sample_rows_work_bytes(V);
    if (!each) return R;
    const int64_t most = (int64_t)(((size_t)2 << 30) / each);
    return std::min<int64_t>(R, std::max<int64_t>(1, std::min<int64_t>(most, 32768)));
}
size_t sample_rows_work(int64_t rows, int64_t V) { return V <= SNK_HELD_MOST ? 0 : rows * sample_rows_work_bytes(V) + 16 * 256; }

template <typename T>
static void launch_rows_split(const T *scores, int64_t stride, int64_t R, int64_t V, const double *u, int n_draws, const SampleRule &rule,
                              const double *rules, double unit, char *work, int64_t *index, double *logp, hipStream_t s)
{
    RowsWork w;
    w.bins = rows_bins(V);
    w.chunks = (int)rows_chunks(V);
    w.span = rows_span(R, V);
    w.spans = (int)((V + w.span - 1) / w.span);
    size_t at = 0;
    auto take = [&](size_t bytes) { char *p = work + at; at += SNK_ALIGNED(bytes); return p; };
    const size_t n = (size_t)R * w.chunks;
    w.state = (RowState *)take(R * sizeof(RowState));
    w.chunk_max = (double *)take(n * 8); w.chunk_min = (double *)take(n * 8);
    w.chunk_mass = (u64 *)take(n * 8); w.chunk_more = (u64 *)take(n * 8);
    w.hist_mass = (u64 *)take((size_t)R * w.bins * 8); w.hist_more = (u64 *)take((size_t)R * w.bins * 8);
    w.list = rows_list(V);
    w.list_x = (double *)take((size_t)R * w.list * 8);
    w.left = (int *)take(R * 4);
    const dim3 grid((unsigned)w.chunks, (unsigned)R), spans((unsigned)w.spans, (unsigned)R);
    hipLaunchKernelGGL((rows_extremes_kernel<T>), spans, dim3(512), 0, s, scores, stride, V, w);
    const size_t bins_lds = (size_t)w.bins * 16;
    static size_t attr_set[32] = {0};
    if (w.bins == SNK_BINS_MOST)                                // 64 KB, and the workgroup's own few words
        lds_attr_ensure(attr_set, bins_lds, [&] {
            (void)hipFuncSetAttribute(reinterpret_cast<const void *>(&rows_histogram_kernel<T>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bins_lds); });
    hipLaunchKernelGGL((rows_histogram_kernel<T>), spans, dim3(512), bins_lds, s, scores, stride, V, rule, rules, unit, w);
    for (int by_mass = 0; by_mass < 2; ++by_mass) {
        if (!rules && (by_mass ? !(rule.top_p < 1.0) : !(rule.top_k > 0 && rule.top_k < V))) continue;
        hipLaunchKernelGGL((rows_boundary_kernel<T>), spans, dim3(512), 0, s, scores, stride, V, rule, rules, unit, by_mass, w);
        hipLaunchKernelGGL(rows_select_kernel, dim3((unsigned)R), dim3(1024), 0, s, V, rule, rules, unit, by_mass, w);
    }
    hipLaunchKernelGGL((rows_masses_kernel<T>), grid, dim3(512), 0, s, scores, stride, V, rule, rules, unit, w);
    for (int d = 0; d < n_draws; d += 32768)
        hipLaunchKernelGGL((rows_draw_kernel<T>), dim3((unsigned)R, std::min(n_draws - d, 32768)), dim3(1024), 0, s, scores, stride, V, u, n_draws, d, rule,
                           rules, unit, w, index, logp);
    hipLaunchKernelGGL((sample_rows_block_kernel<T, 1024>), dim3((unsigned)R), dim3(1024), 0, s, scores, stride, V, u, n_draws, rule, rules, unit, w.left,
                       index, logp);
}

template <typename T>
static void launch_sample_t(const T *scores, int64_t stride, int64_t R, int64_t V, const double *u, int n_draws, const SampleRule &rule,
                            const double *rules, char *work, int64_t *index, double *logp, hipStream_t s)
{
    const double unit = V <= 4096 ? SNK_SAMPLE_UNIT : 0.5 * SNK_SAMPLE_UNIT;      // (sample_device.h: what the sums hold)
#define SNK_WAVE(E_) hipLaunchKernelGGL((sample_rows_wave_kernel<T, E_>), dim3((unsigned)((R + 3) / 4)), dim3(256), 0, s, scores, stride, R, (int)V, u, n_draws, rule, rules, unit, index, logp)
#define SNK_HELD(NT_, EACH_) hipLaunchKernelGGL((sample_rows_held_kernel<T, NT_, EACH_>), dim3((unsigned)R), dim3(NT_), 0, s, scores, stride, (int)V, u, n_draws, rule, rules, unit, index, logp)
    if (V <= 64) SNK_WAVE(1);
    else if (V <= 128) SNK_WAVE(2);
    else if (V <= 256) SNK_WAVE(4);
    else if (V <= 512) SNK_WAVE(8);
    else if (V <= 1024) SNK_WAVE(16);
    else if (V <= SNK_HELD_MOST) {
        if (V <= 2048) SNK_HELD(256, 8);
        else if (V <= 4096) SNK_HELD(512, 8);
        else SNK_HELD(1024, 8);
    } else if (work) launch_rows_split(scores, stride, R, V, u, n_draws, rule, rules, unit, work, index, logp, s);
    else
        hipLaunchKernelGGL((sample_rows_block_kernel<T, 1024>), dim3((unsigned)R), dim3(1024), 0, s, scores, stride, V, u, n_draws, rule, rules, unit,
                           (const int *)nullptr, index, logp);
#undef SNK_WAVE
#undef SNK_HELD
}

int64_t sample_rows_max() { return (int64_t)SNK_SAMPLE_TILES * 1024 * SNK_SAMPLE_VEC; }

void launch_sample_rows(const void *scores, int dtype, int64_t stride, int64_t R, int64_t V, const double *u, int n_draws,
                        const SampleRuleHost &rule, const double *rules, char *work, int64_t *index, double *logp, hipStream_t s)
{
    SampleRule k;
    k.inv_tau = rule.temperature > 0.0 ? 1.0 / rule.temperature : __builtin_inf();
    k.top_k = rule.temperature > 0.0 ? rule.top_k : 1;
    k.top_p = rule.top_p;
    k.min_p = rule.min_p;
    // a launch holds fewer than 2^32 threads, 64 a row or 1024
    const int64_t most = V <= 1024 ? (int64_t)1 << 25 : (int64_t)1 << 21;
    const int64_t step = std::min(work ? sample_rows_together(R, V) : R, most);
    const size_t width = dtype == 0 ? 8 : dtype == 1 ? 4 : 2;
    for (int64_t r = 0; r < R; r += step) {
        const int64_t n = R - r < step ? R - r : step;
        const void *p = (const char *)scores + (size_t)r * stride * width;
        const double *ru = u + r * n_draws, *rr = rules ? rules + 4 * r : nullptr;
        int64_t *ri = index + r * n_draws;
        double *rl = logp ? logp + r * n_draws : nullptr;
        if (dtype == 0) launch_sample_t((const double *)p, stride, n, V, ru, n_draws, k, rr, work, ri, rl, s);
        else if (dtype == 1) launch_sample_t((const float *)p, stride, n, V, ru, n_draws, k, rr, work, ri, rl, s);
        else if (dtype == 2) launch_sample_t((const __half *)p, stride, n, V, ru, n_draws, k, rr, work, ri, rl, s);
        else launch_sample_t((const __hip_bfloat16 *)p, stride, n, V, ru, n_draws, k, rr, work, ri, rl, s);
    }
}

}  // namespace snk
