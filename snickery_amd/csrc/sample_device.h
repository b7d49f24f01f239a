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
// integers, w_i rounded to nearest in units of 2^-s: integer sums are exact in any order, and every comparison above is one between
// integers.  s = 51 leaves the rounding of one weight at a unit of float64's last place next to 1 (the weights themselves are computed in
// float64), and the sums of up to 4096 of them in 64 bits; rows of more scores take s = 50, whose sums of up to 8192 fit, and
// longer sums a second word (sample_sum below).  A row's largest weight is 1, so that V 2^-(s+1) is also the share of the mass that
// rounding can move: 2e-13 of 208 scores, 5e-10 of 2^20, 7e-9 of 2^24.
#pragma once
#include "snk_internal.h"

namespace snk {

typedef unsigned long long u64;
typedef unsigned __int128 u128;

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
#define SNK_SAMPLE_UNIT 2251799813685248.0       // 2^51
__device__ __forceinline__ u64 sample_fix(double w, double unit)
{
    const double t = __fma_rn(w, unit, 4503599627370496.0);
    return (u64)__double_as_longlong(t) - 0x4330000000000000ull;
}

// exp(e) for -37 < e <= 0: e = n ln 2 + r, |r| <= ln 2 / 2 (ln 2 in two parts, Cody and Waite), the Taylor series of exp(r) to the twelfth
// power (the next term is below 2^-52), times 2^n.  exp(0) is exactly 1.  17 instructions where the general function checks and handles
// every range.
__device__ __forceinline__ double sample_exp(double e)
{
    const double n = rint(e * 1.44269504088896340736);
    double r = __fma_rn(n, -6.93147180369123816490e-01, e);
    r = __fma_rn(n, -1.90821492927058770002e-10, r);
    double p = 2.08767569878680989792e-09;                      // 1 / 12!
    p = __fma_rn(p, r, 2.50521083854417187751e-08);
    p = __fma_rn(p, r, 2.75573192239858906526e-07);
    p = __fma_rn(p, r, 2.75573192239858906526e-06);
    p = __fma_rn(p, r, 2.48015873015873015873e-05);
    p = __fma_rn(p, r, 1.98412698412698412698e-04);
    p = __fma_rn(p, r, 1.38888888888888888889e-03);
    p = __fma_rn(p, r, 8.33333333333333333333e-03);
    p = __fma_rn(p, r, 4.16666666666666666667e-02);
    p = __fma_rn(p, r, 1.66666666666666666667e-01);
    p = __fma_rn(p, r, 0.5);
    p = __fma_rn(p, r, 1.0);
    p = __fma_rn(p, r, 1.0);
    return __longlong_as_double(__double_as_longlong(p) + ((long long)(int)n << 52));
}

// exponents below this round to nothing in the finest unit (2^-52)
#define SNK_SAMPLE_FLOOR (-36.1)

__device__ __forceinline__ u64 sample_weight(double e, double unit)
{
    return e >= SNK_SAMPLE_FLOOR ? sample_fix(sample_exp(e), unit) : 0ull;     // (an exponent that is not a number weighs nothing)
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

// ---- sums of up to 2^24 weights of up to 2^50, in two words that any order of additions leaves the same: `mass`, the sum modulo 2^64, and
// `more`, the sum of the weights' upper parts (w >> 40, 34 bits) below a count (24 bits).  What the lower parts add up to is less than 2^64
// and therefore known from both.  (A word for the carry alone would need atomics that return what they found.)
#define SNK_MORE_ONE (1ull << 36)
__device__ __forceinline__ u64 sample_more(u64 w) { return w >> 40; }
__device__ __forceinline__ u64 sample_count(u64 more) { return more >> 36; }
__device__ __forceinline__ u128 sample_sum(u64 mass, u64 more)
{
    const u64 upper = more & (SNK_MORE_ONE - 1);
    return ((u128)upper << 40) + (mass - (upper << 40));
}
__device__ __forceinline__ double sample_double(u128 v) { return __fma_rn((double)(u64)(v >> 64), 18446744073709551616.0, (double)(u64)v); }
__device__ __forceinline__ u128 sample_whole(double t)          // of a whole number, 0 <= t < 2^96
{
    const double upper = floor(t * 0x1p-32);
    return ((u128)(u64)upper << 32) + (u64)__fma_rn(-upper, 4294967296.0, t);
}
__device__ __forceinline__ u128 sample_reach(double top_p, u128 total)
{
    const double all = sample_double(total), t = ceil(top_p * all);
    const u128 v = t >= all ? total : sample_whole(t);
    return v < 1 ? 1 : v;
}
__device__ __forceinline__ u128 sample_exceed(double u, u128 total)
{
    const double all = sample_double(total), t = floor(u * all);
    if (!(t > 0.0)) return 0;
    return t >= all ? total - 1 : sample_whole(t);
}
// how many weights of `each` reach `need`: the quotient in float64, then put right (it is below 2^25)
__device__ __forceinline__ u64 sample_ties(u128 need, u64 each)
{
    if (!each) return 0;
    u64 n = (u64)(sample_double(need) / (double)each);
    while ((u128)n * each < need) ++n;
    while (n && (u128)(n - 1) * each >= need) --n;
    return n;
}

// ---- wavefront sums and maxima on the data-parallel moves: a step costs two moves and one operation, where a shuffle through
// the LDS pipe waits ~ 100 cycles -- the six steps of a reduction are most of what a short row costs -------------------------------
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp_move(u64 old, u64 v)
{
    const int lo = __builtin_amdgcn_update_dpp((int)(unsigned int)old, (int)(unsigned int)v, CTRL, ROWS, 0xf, false);
    const int hi = __builtin_amdgcn_update_dpp((int)(unsigned int)(old >> 32), (int)(unsigned int)(v >> 32), CTRL, ROWS, 0xf, false);
    return ((u64)(unsigned int)hi << 32) | (unsigned int)lo;
}
// (every lane of the wavefront has to be active in these)
__device__ __forceinline__ u64 wave_scan_add(u64 v)        // inclusive: within rows of 16 lanes, then the rows below
{
    v += dpp_move<0x111, 0xf>(0, v);
    v += dpp_move<0x112, 0xf>(0, v);
    v += dpp_move<0x114, 0xf>(0, v);
    v += dpp_move<0x118, 0xf>(0, v);
    v += dpp_move<0x142, 0xa>(0, v);
    v += dpp_move<0x143, 0xc>(0, v);
    return v;
}
__device__ __forceinline__ u64 wave_lane(u64 v, int lane)    // uniform lane
{
    const unsigned int lo = (unsigned int)__builtin_amdgcn_readlane((int)(unsigned int)v, lane);
    const unsigned int hi = (unsigned int)__builtin_amdgcn_readlane((int)(unsigned int)(v >> 32), lane);
    return ((u64)hi << 32) | lo;
}
__device__ __forceinline__ double wave_lane(double v, int lane)
{
    return __longlong_as_double((long long)wave_lane((u64)__double_as_longlong(v), lane));
}
__device__ __forceinline__ u64 wave_add(u64 v) { return wave_lane(wave_scan_add(v), 63); }
__device__ __forceinline__ double dpp_max(double v, u64 moved) { return fmax(v, __longlong_as_double((long long)moved)); }
__device__ __forceinline__ double wave_max(double v)
{
#define SNK_BITS(x_) ((u64)__double_as_longlong(x_))
    v = dpp_max(v, dpp_move<0x111, 0xf>(SNK_BITS(v), SNK_BITS(v)));
    v = dpp_max(v, dpp_move<0x112, 0xf>(SNK_BITS(v), SNK_BITS(v)));
    v = dpp_max(v, dpp_move<0x114, 0xf>(SNK_BITS(v), SNK_BITS(v)));
    v = dpp_max(v, dpp_move<0x118, 0xf>(SNK_BITS(v), SNK_BITS(v)));
    v = dpp_max(v, dpp_move<0x142, 0xa>(SNK_BITS(v), SNK_BITS(v)));
    v = dpp_max(v, dpp_move<0x143, 0xc>(SNK_BITS(v), SNK_BITS(v)));
    return wave_lane(v, 63);
}
__device__ __forceinline__ double row16_max(double v)      // of each row of 16 lanes, in its last lane
{
    v = dpp_max(v, dpp_move<0x111, 0xf>(SNK_BITS(v), SNK_BITS(v)));
    v = dpp_max(v, dpp_move<0x112, 0xf>(SNK_BITS(v), SNK_BITS(v)));
    v = dpp_max(v, dpp_move<0x114, 0xf>(SNK_BITS(v), SNK_BITS(v)));
    v = dpp_max(v, dpp_move<0x118, 0xf>(SNK_BITS(v), SNK_BITS(v)));
    return v;
}
__device__ __forceinline__ double row16_sum(double v)      // of each row of 16 lanes, in all of them: mirrored, so that they agree to the last bit
{
    v += __longlong_as_double((long long)dpp_move<0xb1, 0xf>(0, SNK_BITS(v)));
    v += __longlong_as_double((long long)dpp_move<0x4e, 0xf>(0, SNK_BITS(v)));
    v += __longlong_as_double((long long)dpp_move<0x141, 0xf>(0, SNK_BITS(v)));
    v += __longlong_as_double((long long)dpp_move<0x140, 0xf>(0, SNK_BITS(v)));
    return v;
}
__device__ __forceinline__ double quad_sum(double v)       // of each four lanes, in all of them
{
    v += __longlong_as_double((long long)dpp_move<0xb1, 0xf>(0, SNK_BITS(v)));
    v += __longlong_as_double((long long)dpp_move<0x4e, 0xf>(0, SNK_BITS(v)));
    return v;
}
__device__ __forceinline__ double eight_sum(double v)      // of two neighbouring fours that hold a sum each, in all eight lanes
{
    return v + __longlong_as_double((long long)dpp_move<0x141, 0xf>(0, SNK_BITS(v)));
}
__device__ __forceinline__ double rows4_sum(double v)      // of the same lane of the four rows of 16, in all of them
{
    v += __shfl_xor(v, 16, 64);
    v += __shfl_xor(v, 32, 64);
    return v;
}
__device__ __forceinline__ double wave_sum(double v)
{
    v += __longlong_as_double((long long)dpp_move<0x111, 0xf>(0, SNK_BITS(v)));
    v += __longlong_as_double((long long)dpp_move<0x112, 0xf>(0, SNK_BITS(v)));
    v += __longlong_as_double((long long)dpp_move<0x114, 0xf>(0, SNK_BITS(v)));
    v += __longlong_as_double((long long)dpp_move<0x118, 0xf>(0, SNK_BITS(v)));
    v += __longlong_as_double((long long)dpp_move<0x142, 0xa>(0, SNK_BITS(v)));
    v += __longlong_as_double((long long)dpp_move<0x143, 0xc>(0, SNK_BITS(v)));
#undef SNK_BITS
    return wave_lane(v, 63);
}

// ---- one wavefront, one row of up to 64 E scores: lane l holds the elements l E .. l E + E - 1 --------------------------------
template <int E>
struct WaveRow {
    u64 total;                  // the kept mass
    u64 before;                 // kept mass in the lanes below
    u64 w[E];                   // kept weights (0: not kept)
};

// The truncations.  x: the order's values (-inf: takes no part), row.w: their weights in units of 1 / unit (equal values, equal
// weights; the largest weighs `unit`).  On return row.w is what is kept, row.before / row.total its sums.
template <int E>
__device__ __forceinline__ void wave_row_keep(const double (&x)[E], const SampleRule &rule, double unit, WaveRow<E> &row)
{
    const double ninf = -__builtin_inf();
    // The order's prefix, by bisection on the values.  `live`: the lanes, per element slot, whose side is not known yet; one of them is
    // the pivot, taken a third of the wavefront further on every round (about 2 ln V rounds, sorted rows or not).  A comparison with
    // the pivot is a mask of lanes: masks, counts and the pivot's choice are scalar work beside the other wavefronts' vector work.
    // A round is a dependent chain of some 70 instructions, as many of them scalar: neither halving the interval of values, which needs
    // no pivot, nor masses of 32 bits with the rest looked at where those leave it open made it faster (1.66 and 1.46 ms for the
    // pointers of 9600 rows of 100 candidates, top_k 20, top_p 0.9, four draws; 1.31 like this).
    double cut = ninf;          // kept: x > cut, and the first n_tie of the elements equal to it
    int n_tie = 0, ties = 0;
    auto search = [&](bool by_mass, u64 want) {
        u64 live[E];
#pragma unroll
        for (int e = 0; e < E; ++e) live[e] = __ballot(row.w[e] != 0);
        for (int turn = 21;; turn += 21) {
            double pivot = 0.0;
            u64 each = 0;
            bool found = false;
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (!found && live[e]) {
                    const u64 later = live[e] & (~0ull << (turn & 63));
                    const int l = __ffsll((long long)(later ? later : live[e])) - 1;
                    pivot = wave_lane(x[e], l);
                    if (by_mass) each = wave_lane(row.w[e], l);      // (equal values: equal weights)
                    found = true;
                }
            if (!found) return;                                 // (the prefix is the whole row)
            u64 g[E], q[E], gt = 0, part = 0;                   // gt: count / mass of everything above the pivot
            unsigned int eq = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const bool more = x[e] > pivot;
                g[e] = __ballot(more);
                q[e] = __ballot(x[e] == pivot) & live[e];
                eq += __popcll(q[e]);
                if (by_mass) part += more ? row.w[e] : 0;
                else gt += __popcll(g[e]);
            }
            if (by_mass) gt = wave_add(part);
            else each = 1;
            const bool over = gt >= want;
            if (!over && gt + each * (u64)eq >= want) {
                cut = pivot;
                ties = (int)eq;
                u64 need = want - gt;
                n_tie = 0;
                if (each == 1) n_tie = (int)need;
                else while (need) { ++n_tie; need = need > each ? need - each : 0; }
                return;
            }
#pragma unroll
            for (int e = 0; e < E; ++e) live[e] = over ? live[e] & g[e] : live[e] & ~(g[e] | q[e]);
        }
    };
    auto apply = [&]() {        // weights outside the prefix -> 0
        if (ties == n_tie) {
#pragma unroll
            for (int e = 0; e < E; ++e) row.w[e] = x[e] >= cut ? row.w[e] : 0;
            return;
        }
        int mine = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) mine += (x[e] == cut) ? 1 : 0;
        int rank = (int)wave_scan_add((u64)mine) - mine;         // equal elements in the lanes below
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const bool tie = x[e] == cut;
            if (!(x[e] > cut || (tie && rank < n_tie))) row.w[e] = 0;
            rank += tie ? 1 : 0;
        }
    };
    auto sum = [&]() {
        u64 mass = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) mass += row.w[e];
        return mass;
    };
    if (rule.top_k > 0 && rule.top_k < 64 * E) {
        search(false, (u64)rule.top_k);
        if (cut > ninf) apply();
    }
    if (rule.top_p < 1.0) {
        const u64 total = wave_add(sum());
        cut = ninf;
        search(true, sample_reach(rule.top_p, total));
        if (cut > ninf) apply();
    }
    if (rule.min_p > 0.0) {
        const double least = rule.min_p * unit;
#pragma unroll
        for (int e = 0; e < E; ++e) row.w[e] = (double)row.w[e] < least ? 0 : row.w[e];
    }
    const u64 mass = sum(), upto = wave_scan_add(mass);
    row.before = upto - mass;
    row.total = wave_lane(upto, 63);
}

// Elements that up to 64 random numbers pick: u is lane d's of draw d < n, so is the result.
template <int E>
__device__ __forceinline__ int wave_row_picks(const WaveRow<E> &row, double u, int n)
{
    const u64 t = sample_exceed(u, row.total);
    u64 upto[E];
#pragma unroll
    for (int e = 0; e < E; ++e) upto[e] = (e ? upto[e > 0 ? e - 1 : 0] : row.before) + row.w[e];
    int mine = 0;
    for (int d = 0; d < n; ++d) {
        const u64 goal = wave_lane(t, d);
        int below = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) below += upto[e] <= goal ? 1 : 0;
        const int lane = __ffsll((long long)__ballot(below < E)) - 1;
        const int pick = lane * E + __builtin_amdgcn_readlane(below, lane);
        mine = (int)(threadIdx.x & 63) == d ? pick : mine;
    }
    return mine;
}

template <int E, typename V>
__device__ __forceinline__ V wave_row_value(const V (&x)[E], int lane, int slot)
{
    V v = x[0];
#pragma unroll
    for (int e = 1; e < E; ++e) v = slot == e ? x[e] : v;
    return wave_lane(v, lane);
}

}  // namespace snk
