// Device helpers of the sampling operators (sample_kernels.hip: rows of scores; trellis_kernels.hip: the rows of a trellis).
//
// A row of scores x_i, temperature tau, one random number u in [0, 1):
//     m    = max x_i                       (NaN and -inf take no part; a row without any other score is empty)
//     w_i  = exp((x_i - m) / tau)          (exactly 1 where x_i = m, so +inf shares the row among its holders)
//     order: x descending, equal scores by ascending index
//     kept = the first top_k of the order; of those the shortest prefix that holds top_p of their mass; of those w_i >= min_p
//     draw = the smallest kept i with  sum_{j <= i, kept} w_j  >  u * sum_{kept} w_j
//
// A draw is a whole number: it has to come out the same however the row is split over lanes and workgroups.  So masses are
// 64-bit integers, w_i rounded to nearest in units of 2^-s: integer sums are exact in any order, and every comparison above is
// one between integers.  s <= 51 leaves the rounding of one weight at half a unit of float64's last place next to 1 (the weights
// themselves are computed in float64); rows of more than 2^11 scores take s = 62 - ceil(log2 V), so that a sum never overflows.
#pragma once
#include "snk_internal.h"

namespace snk {

typedef unsigned long long u64;

struct SampleRule {             // what a row is truncated by, in the form the kernels use
    double inv_tau;             // +inf: temperature 0 (with top_k 1: the lowest index of the maximum)
    double top_p;               // >= 1: off
    double min_p;               // <= 0: off
    long long top_k;            // <= 0: off
};

// rule of a row: the call's, or its own four numbers (temperature, top_k, top_p, min_p); a number without meaning is "off"
__device__ __forceinline__ SampleRule sample_rule(const SampleRule &call, const double *__restrict__ rows, int64_t r)
{
    if (!rows) return call;
    const double tau = rows[4 * r], k = rows[4 * r + 1], p = rows[4 * r + 2], q = rows[4 * r + 3];
    SampleRule out;
    out.top_k = (k >= 1.0) ? (k < 9.0e15 ? (long long)k : 0) : 0;
    out.inv_tau = 1.0 / tau;
    if (!(tau > 0.0)) { out.inv_tau = __builtin_inf(); out.top_k = 1; }
    out.top_p = (p > 0.0 && p < 1.0) ? p : 1.0;
    out.min_p = (q > 0.0) ? (q < 1.0 ? q : 1.0) : 0.0;
    return out;
}

__device__ __forceinline__ double sample_exponent(double x, double m, double inv_tau)
{
    return x == m ? 0.0 : (x - m) * inv_tau;
}

// w in units of 2^-s; unit = 2^s, s <= 51.  2^52 + w 2^s < 2^53: the sum's last place is 1, its mantissa is the rounded weight
__device__ __forceinline__ u64 sample_fix(double w, double unit)
{
    const double t = __fma_rn(w, unit, 4503599627370496.0);
    return (u64)__double_as_longlong(t) - 0x4330000000000000ull;
}

// exponents below this round to nothing in the finest unit (2^-52)
#define SNK_SAMPLE_FLOOR (-36.1)

__device__ __forceinline__ u64 sample_weight(double e, double unit)
{
    return e < SNK_SAMPLE_FLOOR ? 0ull : sample_fix(exp(e), unit);
}

// thresholds: the mass a prefix has to reach (top_p) / to exceed (a draw)
__device__ __forceinline__ u64 sample_reach(double top_p, u64 total)
{
    const double t = ceil(top_p * (double)total);
    const u64 v = t >= (double)total ? total : (u64)t;
    return v < 1 ? 1 : v;
}
__device__ __forceinline__ u64 sample_exceed(double u, u64 total)
{
    const double t = floor(u * (double)total);
    if (!(t > 0.0)) return 0;
    return t >= (double)total ? total - 1 : (u64)t;
}

// ---- one wavefront, one row of up to 64 E scores: lane l holds the elements l E .. l E + E - 1 --------------------------------
__device__ __forceinline__ double wave_max(double v)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) v = fmax(v, __shfl_xor(v, o, 64));
    return v;
}
__device__ __forceinline__ u64 wave_add(u64 v)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ __forceinline__ u64 wave_scan_add(u64 v)        // inclusive
{
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const u64 b = __shfl_up(v, o, 64);
        if (lane >= o) v += b;
    }
    return v;
}

template <int E>
struct WaveRow {
    double m;                   // the row's maximum; -inf: empty
    double log_total;           // log of the kept mass
    u64 total;                  // the kept mass
    u64 before;                 // kept mass in the lanes below
    u64 w[E];                   // kept weights (0: not kept)
};

// n-th set bit of a mask that has more than n of them (uniform)
__device__ __forceinline__ int nth_bit(u64 mask, int n)
{
    for (; n; --n) mask &= mask - 1;
    return __ffsll((long long)mask) - 1;
}

template <int E>
__device__ __forceinline__ void wave_row_weights(const double (&x)[E], const SampleRule &rule, double unit, WaveRow<E> &row)
{
    const double ninf = -__builtin_inf();
    double m = ninf;
#pragma unroll
    for (int e = 0; e < E; ++e) m = fmax(m, x[e]);
    m = wave_max(m);
    row.m = m;
    if (m == ninf) { row.total = 0; return; }
    u64 mass = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        row.w[e] = x[e] == ninf ? 0 : sample_weight(sample_exponent(x[e], m, rule.inv_tau), unit);
        mass += row.w[e];
    }

    // The order's prefix: found by bisection on the scores themselves.  `live` are the elements whose side is not known yet; a
    // pivot among them splits them, one ballot per element slot counts a side.  The middle live element is the pivot: a sorted
    // list is halved, an unsorted one takes ~ 2 ln V rounds.
    double cut = ninf;          // kept: x > cut, and the first n_tie of the elements equal to it
    int n_tie = 64 * E;
    auto search = [&](bool by_mass, u64 want) {
        u64 above = 0;                                          // count / mass of everything above the live elements
        unsigned live = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) live |= (by_mass ? row.w[e] != 0 : x[e] > ninf) ? 1u << e : 0u;
        for (;;) {
            u64 b[E];
            int n = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) { b[e] = __ballot((live >> e) & 1u); n += __popcll(b[e]); }
            if (n == 0) return;                                 // (the prefix is the whole row)
            // the middle one
            int left = n >> 1;
            double pivot = 0.0;
            bool found = false;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int c = __popcll(b[e]);
                if (!found && left < c) { pivot = __shfl(x[e], nth_bit(b[e], left), 64); found = true; }
                if (!found) left -= c;
            }
            u64 gt = 0, eq = 0;
            unsigned mgt = 0, meq = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const bool l = (live >> e) & 1u, g = l && x[e] > pivot, q = l && x[e] == pivot;
                mgt |= g ? 1u << e : 0u;
                meq |= q ? 1u << e : 0u;
                if (by_mass) { gt += g ? row.w[e] : 0; eq += q ? row.w[e] : 0; }
                else { gt += __popcll(__ballot(g)); eq += __popcll(__ballot(q)); }
            }
            if (by_mass) { gt = wave_add(gt); eq = wave_add(eq); }
            if (above + gt >= want) { live = mgt; continue; }
            if (above + gt + eq >= want) {
                cut = pivot;
                if (by_mass) {
                    int c = 0;
#pragma unroll
                    for (int e = 0; e < E; ++e) c += __popcll(__ballot((meq >> e) & 1u));
                    const u64 each = eq / (u64)c;               // (equal scores: equal weights)
                    n_tie = (int)((want - above - gt + each - 1) / each);
                } else n_tie = (int)(want - above - gt);
                return;
            }
            above += gt + eq;
            live &= ~(mgt | meq);
        }
    };
    auto apply = [&]() {        // weights outside the prefix -> 0
        int ties = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) ties += (x[e] == cut) ? 1 : 0;
        int rank = (int)(wave_scan_add((u64)ties)) - ties;       // equal elements in the lanes below
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const bool tie = x[e] == cut;
            if (!(x[e] > cut || (tie && rank < n_tie))) row.w[e] = 0;
            rank += tie ? 1 : 0;
        }
    };
    if (rule.top_k > 0 && rule.top_k < 64 * E) {
        search(false, (u64)rule.top_k);
        if (cut > ninf) {
            apply();
            mass = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) mass += row.w[e];
        }
    }
    if (rule.top_p < 1.0) {
        const u64 total = wave_add(mass);
        cut = ninf; n_tie = 64 * E;
        search(true, sample_reach(rule.top_p, total));
        if (cut > ninf) apply();
    }
    if (rule.min_p > 0.0) {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (row.w[e] && exp(sample_exponent(x[e], m, rule.inv_tau)) < rule.min_p) row.w[e] = 0;
    }
    mass = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) mass += row.w[e];
    const u64 upto = wave_scan_add(mass);
    row.before = upto - mass;
    row.total = __shfl(upto, 63, 64);
    row.log_total = log((double)row.total / unit);
}

// element that u picks (uniform), the lane that holds it and its slot
template <int E>
__device__ __forceinline__ int wave_row_pick(const WaveRow<E> &row, double u, int &lane_out, int &slot_out)
{
    const u64 t = sample_exceed(u, row.total);
    u64 cum = row.before;
    int slot = -1;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        cum += row.w[e];
        if (slot < 0 && cum > t) slot = e;
    }
    const int lane = __ffsll((long long)__ballot(slot >= 0)) - 1;
    lane_out = lane;
    slot_out = __shfl(slot, lane, 64);
    return lane * E + slot_out;
}

template <int E>
__device__ __forceinline__ double wave_row_value(const double (&x)[E], int lane, int slot)
{
    double v = x[0];
#pragma unroll
    for (int e = 1; e < E; ++e) v = slot == e ? x[e] : v;
    return __shfl(v, lane, 64);
}

}  // namespace snk
