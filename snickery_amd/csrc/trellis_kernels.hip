// Draws from and probabilities of the paths of a candidate trellis (snk_sample_paths, snk_path_posterior).
//
// A path takes one candidate a_t of every row t of an utterance; with the target costs d and
//     C[t,a,b] = J[t,a,b] + B[class_t, bucket(cand[t+1,b] - cand[t,a])]        (join cost + bias by relative position)
//     p(path)  ~ exp(-(sum_t d[t,a_t] + sum_t C[t,a_t,a_t+1]) / tau)
// a candidate takes part if its unit can join (1 <= id < N - 1, as in the Viterbi search) and its target cost is finite.
// With  l[t,a] = exp((min d[t,.] - d[t,a]) / tau)  and  E[t,a,b] = exp((min B - C[t,a,b]) / tau), both at most 1,
//     v_0 = l_0              v_t+1[b] = l_t+1[b] * sum_a v_t[a] E[t,a,b]        up to a factor per row: p(a_t | rows <= t)
//     x_T-1 = l_T-1          w_t[a]   = sum_b E[t,a,b] x_t+1[b],  x_t = l_t w_t                      p(rows > t | a_t)
//     log Z = log sum v_T-1 + what was scaled out
//     draw: a_T-1 from v_T-1, then a_t from v_t[.] E[t,.,a_t+1]: rows of weights, truncated like those of sample_kernels.hip
//
// The exponentials are taken once per cell, where the costs are made; the recursions are products and sums.  Every row is scaled by
// a power of two, and an utterance whose weights span more than float64's exponents carry -- a tau far below the costs, or a
// candidate that only a forbidden join leaves -- is recognised (a cost beyond SNK_COST_RANGE tau, a target cost beyond
// SNK_LOCAL_RANGE tau, a weight below SNK_WEIGHT_LEAST) and done again in logarithms: the launches named _log work on the flagged
// utterances only.  Within those limits no product underflows: weight, cell and local weight 2^-490 e^-230 e^-100 > 2^-967, the
// weights of the two directions 2^-490 2^-490.
#include "sample_device.h"

#define SNK_COST_RANGE 230.0
#define SNK_LOCAL_RANGE 100.0
#define SNK_WEIGHT_LEAST 0x1p-490
#define SNK_USES_UNIT 1125899906842624.0      // 2^50

namespace snk {

typedef double f64x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ bool trellis_usable(int64_t id, int64_t n_units) { return id >= 1 && id < n_units - 1; }
__device__ __forceinline__ bool trellis_takes_part(int64_t id, double d, int64_t n_units) { return trellis_usable(id, n_units) && d - d == 0.0; }

// -d / tau of a candidate that takes part, kept finite (a sum over 2^23 rows stays so)
__device__ __forceinline__ double trellis_local(int64_t id, double d, int64_t n_units, double inv_tau)
{
    return trellis_takes_part(id, d, n_units) ? fmin(fmax(-d * inv_tau, -1e300), 1e300) : -__builtin_inf();
}

// utterance of a row (first .. first + n - 1): off[u] <= t < off[u + 1]
__device__ __forceinline__ int trellis_utterance(const int64_t *__restrict__ off, int first, int n, int64_t t)
{
    int u = first, hi = first + n;
    while (hi - u > 1) { const int mid = (u + hi) >> 1; if (off[mid] <= t) u = mid; else hi = mid; }
    return u;
}

// Bucket of a distance: the number of edges up to it.  63 edges at most, in LDS behind INT_MAX padding: which sixteen of them it falls
// among, which four of those, which of those: nine comparisons and two LDS latencies, where two steps of eight take fifteen and one
// and a search by halves waits for LDS five times.
#define SNK_EDGE_WORDS 80                                       // the edges, then every fourth one
struct TrellisEdges { int head[3]; const int *all; };
__device__ __forceinline__ TrellisEdges trellis_edges(const int *lds)
{
    TrellisEdges e;
    e.all = lds;
#pragma unroll
    for (int i = 0; i < 3; ++i) e.head[i] = lds[16 * i + 15];
    return e;
}
__device__ __forceinline__ int trellis_bucket(int apart, const TrellisEdges &e)
{
    int k = 4 * ((apart >= e.head[0]) + (apart >= e.head[1]) + (apart >= e.head[2]));
    const int4 x = *reinterpret_cast<const int4 *>(e.all + 64 + k);
    k = 4 * (k + (apart >= x.x) + (apart >= x.y) + (apart >= x.z));
    const int4 y = *reinterpret_cast<const int4 *>(e.all + k);
    return k + (apart >= y.x) + (apart >= y.y) + (apart >= y.z);
}
__device__ __forceinline__ void trellis_load_edges(int *lds, const int *__restrict__ edges, int n_buckets)
{
    const int i = threadIdx.x;
    if (i >= 64) return;
    const int e = i < n_buckets - 1 ? edges[i] : 0x7fffffff;
    lds[i] = e;
    if ((i & 3) == 3) lds[64 + (i >> 2)] = e;
}

__device__ __forceinline__ double trellis_pow2(int e)           // 2^e, -1022 <= e <= 1023
{
    return __longlong_as_double((long long)(e + 1023) << 52);
}
// exponent of the power of two that scales a row whose largest weight is m to [1, 2): 0 for an empty row
__device__ __forceinline__ int trellis_exponent(double m)
{
    return m > 0.0 ? (int)(((u64)__double_as_longlong(m) >> 52) & 0x7ff) - 1023 : 0;
}

// ---- an utterance's first row and flag.  The offsets travel as arguments: a copy would need a page-locked place that lives on -----------
struct TrellisOffsets { int64_t v[256]; };
__global__ void __launch_bounds__(256)
trellis_offsets_kernel(const TrellisOffsets part, int first, int n_utts, int flag_value, int64_t *__restrict__ off, int *__restrict__ flag)
{
    const int i = first + threadIdx.x;
    if (i <= n_utts) off[i] = part.v[threadIdx.x];
    if (i < n_utts) flag[i] = flag_value;
}

// ---- local weights: a wavefront per row; 9600 rows of 100: 9 us, 2.5 TB/s ---------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256)
trellis_local_kernel(const TrellisView v, double *__restrict__ local, double *__restrict__ least, int *__restrict__ flag)
{
    const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= v.rows) return;
    const int64_t t = v.c0 + i;
    const int lane = threadIdx.x & 63;
    const double inf = __builtin_inf();
    double d[4], lo = inf, hi = -inf;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int a = lane + 64 * j;
        d[j] = inf;
        if (a < v.K) {
            const double c = v.tdist[t * v.K + a];
            if (trellis_takes_part(v.cand[t * v.K + a], c, v.n_units)) { d[j] = c; hi = fmax(hi, c); }
        }
        lo = fmin(lo, d[j]);
    }
    lo = -wave_max(-lo);
    hi = wave_max(hi);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int a = lane + 64 * j;
        if (a < v.Kp) local[t * v.Kp + a] = d[j] < inf ? exp((lo - d[j]) * v.inv_tau) : 0.0;
    }
    if (lane == 0) {
        least[t] = lo < inf ? lo : 0.0;
        if ((hi - lo) * v.inv_tau > SNK_LOCAL_RANGE) flag[trellis_utterance(v.off, v.first, v.n_utts, t)] = 1;
    }
}

// ---- costs: a workgroup per pair of rows and tile of 16 RT x 16 RT cells ------------------------------------------------------------
// |e - s|^2 = |e|^2 + |s|^2 - 2 e.s on the float64 matrix pipe: half the instructions of the difference form (one fused multiply-add
// a column instead of a subtraction and one), which ran at two thirds of the vector pipe's rate.  Both sides are taken relative to
// one unit of the second row, so that the norms are those of the candidates' spread and not of their distance from the origin.  Where
// the difference is small against the norms -- neighbouring frames -- the product form cancels: a cell below SNK_COST_NEAR of them is taken
// again in differences.  A unit and its natural successor join at exactly 0.  The others carry a relative error of at most Dj 2^-53 / SNK_COST_NEAR,
// an absolute one of 2^5 Dj 2^-53 of the norms' root.  (2^-8 took 4 % longer for 9600 rows of 100 and halved the error of the posteriors, which
// with 2^-10 is 9e-15 at most over 335 rows of 50, a log Z of 455, against 80-bit arithmetic.)
// Frames that are not finite: a distance that is infinite or no number joins nothing.  The product form says so only while the unit that both
// sides are taken relative to is finite; where it is not, or a frame brings an infinity of its own into a product, a cell's value is no
// number, and every such cell of units that can join counts as near: the differences, which know its own two frames alone, decide.
// A wavefront owns RM x CM tiles of 16 x 16; DC columns of the two sets of rows go through LDS at a time, weighted and widened on
// the way, the next ones are in flight meanwhile: 32, a cache line of a row (197 us for 600 rows of 100 candidates and 302 columns, 206
// with 16, before what follows), or 16 in the larger tiles, whose registers hold no more (2.55 ms for 9600 rows, 2.73 with 32 and
// spills; what the rest of this kernel took before later steps).  9600 rows of 100 candidates, 302 columns: 2.0 ms, 29 TFLOP/s of a large
// product's 62 (36 with the cells that pad K to 112); bound by the float64 units, which the products hold 48 % of the time and weighing
// the cells, staging and padding the most of the rest: neither overlaps with products of another wavefront.  1200 rows of 200, 151
// columns: 0.64 ms.
#define SNK_COST_NEAR 0x1p-10
typedef double f64x4 __attribute__((ext_vector_type(4)));

// weight of a column; 0 behind the last.  (Loads from a clamped place, here and of the rows: a load that is left out behind a condition
// goes through the stack's address space.)
__device__ __forceinline__ double trellis_weight(const TrellisCosts &c, int j)
{
    const double w = c.wj[min(j, c.Dj - 1)];
    return j < c.Dj ? w : 0.0;
}

// sum of squared differences of a pair of join rows by a row of sixteen lanes; in every one of them
__device__ __forceinline__ double trellis_difference(const TrellisCosts &c, int end, int start)
{
    const float *__restrict__ pe = c.JC + (int64_t)(end + 1) * c.Jp, *__restrict__ ps = c.JC + (int64_t)start * c.Jp;
    double d2 = 0.0;
    for (int j0 = 0; j0 < c.Dj; j0 += 128) {                    // (rows are padded to multiples of four columns; a lane beyond them reads their last four)
        float4 e[2], s[2];
        double w[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int j = j0 + 64 * h + 4 * (threadIdx.x & 15), at = min(j, c.Jp - 4);
            e[h] = *reinterpret_cast<const float4 *>(pe + at);
            s[h] = *reinterpret_cast<const float4 *>(ps + at);
#pragma unroll
            for (int k = 0; k < 4; ++k) w[h][k] = trellis_weight(c, j + k);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float e4[4] = {e[h].x, e[h].y, e[h].z, e[h].w}, s4[4] = {s[h].x, s[h].y, s[h].z, s[h].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const double d = (double)e4[k] * w[h][k] - (double)s4[k] * w[h][k];
                d2 = __fma_rn(d, d, d2);
            }
        }
    }
    return row16_sum(d2);
}

// A constant that the compiler keeps in scalar registers: written as a number it is moved into a pair of vector registers for every
// multiply-add that adds it, two of three instructions of the polynomial below.
#define SNK_SCALAR(name_, value_) double name_ = value_; asm("" : "+s"(name_))

// exp(x), -SNK_COST_RANGE <= x <= 0, to about a unit in the last place: 2^(n / 32) from a table in LDS times a series of degree 6 in
// what is left, |r| <= ln 2 / 64 (the next term is below 2^-58)
__device__ const double trellis_powers[32] = {                  // 2^(j / 32)
    0x1.0000000000000p+0, 0x1.059b0d3158574p+0, 0x1.0b5586cf9890fp+0, 0x1.11301d0125b51p+0, 0x1.172b83c7d517bp+0, 0x1.1d4873168b9aap+0,
    0x1.2387a6e756238p+0, 0x1.29e9df51fdee1p+0, 0x1.306fe0a31b715p+0, 0x1.371a7373aa9cbp+0, 0x1.3dea64c123422p+0, 0x1.44e086061892dp+0,
    0x1.4bfdad5362a27p+0, 0x1.5342b569d4f82p+0, 0x1.5ab07dd485429p+0, 0x1.6247eb03a5585p+0, 0x1.6a09e667f3bcdp+0, 0x1.71f75e8ec5f74p+0,
    0x1.7a11473eb0187p+0, 0x1.82589994cce13p+0, 0x1.8ace5422aa0dbp+0, 0x1.93737b0cdc5e5p+0, 0x1.9c49182a3f090p+0, 0x1.a5503b23e255dp+0,
    0x1.ae89f995ad3adp+0, 0x1.b7f76f2fb5e47p+0, 0x1.c199bdd85529cp+0, 0x1.cb720dcef9069p+0, 0x1.d5818dcfba487p+0, 0x1.dfc97337b9b5fp+0,
    0x1.ea4afa2a490dap+0, 0x1.f50765b6e4540p+0};
__device__ __forceinline__ double trellis_exp(double x, const double *powers)
{
    SNK_SCALAR(per, 46.16624130844682903552);                   // 32 / ln 2
    SNK_SCALAR(whole, 6755399441055744.0);                      // 1.5 2^52: a sum with it has its integer in the low bits
    SNK_SCALAR(hi, -6.93147180369123816490e-01 / 32);
    SNK_SCALAR(lo, -1.90821492927058770002e-10 / 32);
    SNK_SCALAR(c6, 1.38888888888888888889e-03);
    SNK_SCALAR(c5, 8.33333333333333333333e-03);
    SNK_SCALAR(c4, 4.16666666666666666667e-02);
    SNK_SCALAR(c3, 1.66666666666666666667e-01);
    const double t = __fma_rn(x, per, whole), n = t - whole;
    const int i = (int)__double_as_longlong(t);
    const double r = __fma_rn(n, lo, __fma_rn(n, hi, x)), power = powers[i & 31];
    double p = __fma_rn(r, c6, c5);
    p = __fma_rn(p, r, c4);
    p = __fma_rn(p, r, c3);
    p = __fma_rn(p, r, 0.5);
    p = __fma_rn(p, r, 1.0);
    p = __fma_rn(power, p * r, power);
    return __longlong_as_double(__double_as_longlong(p) + ((long long)(i >> 5) << 52));
}

// sqrt(x), x >= 0, to a unit in the last place, infinite for neither: the reciprocal root refined by Goldschmidt's step and a
// correction by the remainder.  Below 2^-1000 it is 2^-500.
__device__ __forceinline__ double trellis_root(double x)
{
    x = fmax(x, 0x1p-1000);
    const double y = __builtin_amdgcn_rsq(x);
    double g = x * y, h = 0.5 * y;
    const double r = __fma_rn(-h, g, 0.5);
    g = __fma_rn(g, r, g);
    h = __fma_rn(h, r, h);
    return __fma_rn(__fma_rn(-g, g, x), h, g);
}

template <int RT, int RM, int CM, int NTH, int OCC, int DC, bool LOG>
__global__ void __launch_bounds__(NTH, OCC)
trellis_cost_kernel(const TrellisView v, const TrellisCosts c, int *__restrict__ flag, double *__restrict__ X)
{
    constexpr int N = 16 * RT, QL = DC / 4, LD = DC + 2, NW = NTH / 64, NR = NTH / QL, PASS = (N + NR - 1) / NR;
    constexpr int HALF = 32 / DC;                               // sums of a norm that a thread keeps: see below
    static_assert(HALF * DC == 32 && HALF <= 2, "a norm has eight sums");
    constexpr int WC = RT / CM;                                 // wavefronts side by side
    static_assert(RT % RM == 0 && RT % CM == 0 && (RT / RM) * WC <= NW, "every tile has its wavefront");
    __shared__ __align__(16) double Es[2 * N * LD];             // of the first row's candidates, then of the second's
    __shared__ double powers[32];
    __shared__ double nE[N], nS[N];
    __shared__ int idE[N], idS[N];                              // unit id, -1: cannot join
    __shared__ __align__(16) int edges[SNK_EDGE_WORDS];
    __shared__ double bias[64];
    __shared__ unsigned int n_near;
    double *const Ss = Es + N * LD;
    unsigned short *const near_cell = reinterpret_cast<unsigned short *>(Es);           // cells to take again, when the products are done
    static_assert(N * N * sizeof(short) <= sizeof Es, "a list of every cell");
    const int64_t t = v.c0 + blockIdx.x;
    const int u = trellis_utterance(v.off, v.first, v.n_utts, t);
    if (t + 1 == v.off[u + 1]) return;
    if (LOG && !flag[u]) return;
    const int tid = threadIdx.x, lane = tid & 63, c16 = lane & 15, g = lane >> 4;
    const int wave = ((tid >> 6) + blockIdx.x) % NW;            // (one of eight has no tiles: not always on the same SIMD)
    const int row0 = (wave / WC) * RM, col0 = (wave % WC) * CM;
    const bool busy = row0 < RT;
    const int a0 = blockIdx.y * N, b0 = blockIdx.z * N;
    for (int i = tid; i < 2 * N; i += NTH) {
        const bool second = i >= N;
        const int k = second ? b0 + i - N : a0 + i;
        const int64_t id = k < v.K ? v.cand[(t + (second ? 1 : 0)) * v.K + k] : -1;
        (second ? idS[i - N] : idE[i]) = trellis_usable(id, v.n_units) ? (int)id : -1;
    }
    int cls = -1;
    if (c.n_classes) {
        cls = c.join_class ? c.join_class[t] : 0;
        if (cls >= c.n_classes) cls = -1;
        trellis_load_edges(edges, c.edges, c.n_buckets);
        if (cls >= 0 && tid < c.n_buckets) bias[tid] = c.bias[(int64_t)cls * c.n_buckets + tid];
    }
    if (tid == 0) n_near = 0;
    if (!LOG && tid < 32) powers[tid] = trellis_powers[tid];
    __syncthreads();
    // the unit that both sides are taken relative to: the second row's first one that can join (of the whole row: a cell's value does
    // not depend on the tiles)
    int about = 0;
    bool found = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t id = lane + 64 * i < v.K ? v.cand[(t + 1) * v.K + lane + 64 * i] : -1;
        const u64 can = __ballot(trellis_usable(id, v.n_units));
        if (can && !found) { about = __builtin_amdgcn_readlane((int)id, __ffsll((long long)can) - 1); found = true; }
    }

    const int q = tid & (QL - 1), r0 = tid / QL;            // a thread takes four columns of the rows r0, r0 + NR, ..
    const float *pe[PASS], *ps[PASS], *pc = c.JC + (int64_t)about * c.Jp + 4 * q;
    float4 fe[PASS], fs[PASS], fc;
    // A norm is the sum of eight, of the columns 4 i .. 4 i + 3 of every 32, whatever the tile: with 32 columns at a time a thread has one
    // of them, with 16 two, which take turns.  So a cell is the same to the last bit in every tile, and an utterance's results do not
    // depend on how many rows stand beside it.
    double w[4], ne[HALF][PASS], ns[HALF][PASS];
#pragma unroll
    for (int p = 0; p < PASS; ++p) {
        const int r = r0 + NR * p < N ? r0 + NR * p : 0;
        pe[p] = c.JC + (int64_t)(idE[r] >= 0 ? idE[r] + 1 : about) * c.Jp + 4 * q;
        ps[p] = c.JC + (int64_t)(idS[r] >= 0 ? idS[r] : about) * c.Jp + 4 * q;
#pragma unroll
        for (int h = 0; h < HALF; ++h) ne[h][p] = ns[h][p] = 0.0;
    }
    auto turn = [&]() {                                         // the other half of 32 columns is next
        if (HALF == 2)
#pragma unroll
            for (int p = 0; p < PASS; ++p) {
                const double e = ne[0][p], s = ns[0][p];
                ne[0][p] = ne[HALF - 1][p]; ns[0][p] = ns[HALF - 1][p];
                ne[HALF - 1][p] = e; ns[HALF - 1][p] = s;
            }
    };
    auto fetch = [&](int col) {
        const int at = min(col, c.Jp - 4 - 4 * q);              // (rows are padded to multiples of four columns)
        fc = *reinterpret_cast<const float4 *>(pc + at);
#pragma unroll
        for (int p = 0; p < PASS; ++p) {
            fe[p] = *reinterpret_cast<const float4 *>(pe[p] + at);
            fs[p] = *reinterpret_cast<const float4 *>(ps[p] + at);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = trellis_weight(c, col + 4 * q + e);
    };
    f64x4 acc[RM][CM];
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < CM; ++j) acc[i][j] = f64x4{0.0, 0.0, 0.0, 0.0};
    fetch(0);
    for (int col = 0; col < c.Dj; col += DC) {
        const float c4[4] = {fc.x, fc.y, fc.z, fc.w};
#pragma unroll
        for (int p = 0; p < PASS; ++p) {
            const int r = r0 + NR * p;
            if (r < N) {
                const float e4[4] = {fe[p].x, fe[p].y, fe[p].z, fe[p].w}, s4[4] = {fs[p].x, fs[p].y, fs[p].z, fs[p].w};
                double de[4], ds[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const double m = (double)c4[e] * w[e];
                    de[e] = __fma_rn((double)e4[e], w[e], -m);
                    ds[e] = __fma_rn((double)s4[e], w[e], -m);
                    ne[0][p] = __fma_rn(de[e], de[e], ne[0][p]);
                    ns[0][p] = __fma_rn(ds[e], ds[e], ns[0][p]);
                }
                f64x2 *te = reinterpret_cast<f64x2 *>(&Es[r * LD + 4 * q]), *ts = reinterpret_cast<f64x2 *>(&Ss[r * LD + 4 * q]);
                te[0] = f64x2{de[0], de[1]}; te[1] = f64x2{de[2], de[3]};
                ts[0] = f64x2{ds[0], ds[1]}; ts[1] = f64x2{ds[2], ds[3]};
            }
        }
        turn();
        __syncthreads();
        if (col + DC < c.Dj) fetch(col + DC);
        if (busy) {
#pragma unroll
            for (int ks = 0; ks < DC / 4; ++ks) {
                if (col + 4 * ks >= c.Dj) break;
                double fa[RM], fb[CM];
#pragma unroll
                for (int i = 0; i < RM; ++i) fa[i] = Es[((row0 + i) * 16 + c16) * LD + 4 * ks + g];
#pragma unroll
                for (int j = 0; j < CM; ++j) fb[j] = Ss[((col0 + j) * 16 + c16) * LD + 4 * ks + g];
#pragma unroll
                for (int j = 0; j < CM; ++j)
#pragma unroll
                    for (int i = 0; i < RM; ++i) acc[i][j] = __builtin_amdgcn_mfma_f64_16x16x4f64(fa[i], fb[j], acc[i][j], 0, 0, 0);
            }
        }
        __syncthreads();
    }
    if (((c.Dj + DC - 1) / DC) & 1) turn();
#pragma unroll
    for (int p = 0; p < PASS; ++p) {
        const int r = r0 + NR * p;
        double e = quad_sum(ne[0][p]), s = quad_sum(ns[0][p]);
        if (HALF == 2) { e += quad_sum(ne[HALF - 1][p]); s += quad_sum(ns[HALF - 1][p]); }
        if (QL == 8) { e = eight_sum(e); s = eight_sum(s); }
        if (r < N && q == 0) {                                  // what cannot join is infinitely far
            nE[r] = idE[r] >= 0 ? e : __builtin_inf();
            nS[r] = idS[r] >= 0 ? s : __builtin_inf();
        }
    }
    __syncthreads();
    bool wide = false;
    double *__restrict__ out = X + (t - v.c0) * v.K * v.Kp;
    const TrellisEdges look = trellis_edges(edges);
    auto value = [&](double d2, int ie, int is) -> double {     // a cell from the squared distance, infinite: cannot join
        double cost = LOG ? sqrt(d2) : trellis_root(d2);
        if (cls >= 0) cost += bias[trellis_bucket(is - ie, look)];
        if (LOG) return cost < __builtin_inf() ? fmin(fmax(-cost * v.inv_tau, -1e300), 1e300) : -__builtin_inf();      // (as trellis_local)
        const bool ok = cost < __builtin_inf();                 // (the root of an infinite square is not a number)
        const double x = (c.bias_min - cost) * v.inv_tau;
        wide |= ok && x < -SNK_COST_RANGE;
        return ok ? trellis_exp(fmax(x, -SNK_COST_RANGE), powers) : 0.0;
    };
    // (a loop over the tiles, not RM CM copies of its body; a wavefront's k-th tile is picked by uniform branches)
#pragma unroll 1
    for (int k = 0; k < (busy ? RM * CM : 0); ++k) {
        f64x4 p = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
            for (int j = 0; j < CM; ++j)
                if (i * CM + j == k) p = acc[i][j];
        const int ti = row0 + k / CM, tj = col0 + k % CM;
        const int bl = tj * 16 + c16, is = idS[bl], b = b0 + bl;
        const double sn = nS[bl];
        bool again[4];
        int any = 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int al = ti * 16 + g + 4 * r, ie = idE[al], a = a0 + al;
            const double both = nE[al] + sn, apart = __fma_rn(-2.0, p[r], both);
            const bool natural = is == ie + 1;                  // (the same frame)
            again[r] = (ie | is) >= 0 && (natural ? !(both < __builtin_inf()) : !(apart >= SNK_COST_NEAR * both));      // (true of what is no number)
            any += again[r] ? 1 : 0;
            const double x = value(natural ? 0.0 : fmax(apart, 0.0), ie, is);
            if (a < v.K && b < v.Kp) out[(int64_t)a * v.Kp + b] = x;
        }
        if (__ballot(any)) {
            const unsigned int upto = (unsigned int)wave_scan_add((u64)any);
            unsigned int at = 0;
            if (lane == 63) at = atomicAdd(&n_near, upto);
            at = (unsigned int)__builtin_amdgcn_readlane((int)at, 63) + upto - any;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (again[r]) {
                    near_cell[at] = (unsigned short)((ti * 16 + g + 4 * r) * N + bl);
                    ++at;
                }
        }
    }
    __syncthreads();
    // the near cells in differences, sixteen lanes each: up to sixteen one after the other, then each lane has one of its own to weigh
    for (int base = 0, left = (int)n_near; left > 0; base += 64 * NW, left -= 64 * NW) {
        const int each = (min(left, 64 * NW) + 4 * NW - 1) / (4 * NW), first = base + (tid >> 4) * each, n = min(each, (int)n_near - first);
        double d2 = 0.0;
        for (int i = 0; i < n; ++i) {
            const int cell = near_cell[first + i];
            const double d = trellis_difference(c, idE[cell / N], idS[cell % N]);
            if (c16 == i) d2 = d;
        }
        if (c16 < n) {
            const int cell = near_cell[first + c16], al = cell / N, bl = cell % N, a = a0 + al, b = b0 + bl;
            const double x = value(d2 < __builtin_inf() ? d2 : __builtin_inf(), idE[al], idS[bl]);
            if (a < v.K && b < v.Kp) out[(int64_t)a * v.Kp + b] = x;
        }
    }
    if (!LOG && wide) flag[u] = 1;
}

// ---- the recursions, cut into pieces ---------------------------------------------------------------------------------------------------
// A step of a recursion is one K x K slab of cells through one compute unit: a chain of T of them takes T times 1 - 5 us and keeps
// one unit of 256 busy.  So an utterance's T - 1 slabs are cut into pieces of L, and
//     1. every piece's product  M = prod E[t] diag(l_t+1)  is formed, sixteen of its rows a workgroup, on the float64 matrix pipe
//     2. the weights at the pieces' ends follow from the products, one vector-matrix product a piece (both directions)
//     3. every piece runs its own recursion from there, all pieces side by side
// Pieces of L take  L (product + step) + T / L ends  where the chain takes T steps, and a product, a step and an end cost about the
// same on their own: L = sqrt(T).  Below 24 slabs the chain is as fast, the third launch alone.  Only an utterance's own length decides:
// its results are the same in any batch.  A piece is found without a table: no piece has less than 8 slabs, so those of utterance u
// begin at  floor((off[u] - c0) / 8) + u - first.
#define SNK_PIECE_LEAST 8
__host__ __device__ __forceinline__ int64_t trellis_piece_length(int64_t slabs)
{
    if (slabs < 24) return slabs > 0 ? slabs : 1;
    const int64_t L = (int64_t)ceil(sqrt((double)slabs));
    return L < SNK_PIECE_LEAST ? SNK_PIECE_LEAST : L;
}

struct TrellisPiece { int64_t r0, T, L; int u, k, n, P; int64_t at; };   // rows of the utterance; piece k of P, n of L slabs, its place in the tables

__device__ __forceinline__ TrellisPiece trellis_piece(const TrellisView &v, int utt, int k)
{
    TrellisPiece p;
    p.u = v.first + utt;
    p.r0 = v.off[p.u];
    p.T = v.off[p.u + 1] - p.r0;
    const int64_t S = p.T - 1;
    p.L = trellis_piece_length(S);
    p.P = S > p.L ? (int)((S + p.L - 1) / p.L) : 1;
    p.k = k;
    const int64_t left = S - (int64_t)k * p.L;
    p.n = k < p.P ? (int)(left < p.L ? left : p.L) : 0;
    p.at = (p.r0 - v.c0) / SNK_PIECE_LEAST + utt + k;
    return p;
}

// 1. products: workgroup = sixteen start candidates of one piece, wavefront = CT tiles of sixteen end candidates; v_mfma_f64_16x16x4
// over KH CH steps of four.  The weights X alternate between two LDS buffers; the slab's fragments live in registers and each is
// reloaded with the next slab's (or the next half's) right after its use.  The row blocks of a piece are dealt to one XCD, so that a
// slab comes from memory once and from that XCD's L2 for the others: a step re-reads the slab for sixteen rows, 50 bytes a cycle and
// compute unit.  Thirty-two rows halve that but leave two workgroups a compute unit where sixteen leave three: 0.72 against 0.63 ms for
// 9600 rows of 100 (30 TFLOP/s, 36 with the padding); 1200 rows of 200: 0.62 ms; 600 of 100: 71 us, 24 steps of 3 us.  Sizes of their own
// for 80 and 160 candidates: 350 instead of 445 us and 2.3 instead of 3.1 ms for 9600 rows.  CT 1 where the registers of CT 2 leave one
// wavefront a SIMD (2.3 against 2.5 ms), not below (0.74 against 0.63 ms).
template <int CT, int KH, int CH, int NTH>
__global__ void __launch_bounds__(NTH, NTH == 256 && KH <= 26 ? 3 : 2)
trellis_product_kernel(const TrellisView v, const double *__restrict__ local, int max_pieces, int row_blocks, bool skip_last, int *__restrict__ flag,
                       double *__restrict__ M, int *__restrict__ exps)
{
    constexpr int W = NTH / 64, COLS = 4 * KH * CH, LDX = COLS + 2;      // (sixteen rows 4 odd banks apart)
    __shared__ double X[2][16 * LDX];
    __shared__ double top[2][W][16];
    __shared__ int bad, done;                                   // done: another piece's workgroup may flag the utterance at any time, so one
    const int j = blockIdx.x >> 3;                              // thread looks for all
    const int i0 = (j % row_blocks) * 16, flat = (j / row_blocks) * 8 + (blockIdx.x & 7);
    if (flat >= max_pieces * v.n_utts) return;
    const TrellisPiece p = trellis_piece(v, flat / max_pieces, flat % max_pieces);
    if (p.k >= p.P || p.P == 1 || (skip_last && p.k == p.P - 1)) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c16 = lane & 15, g = lane >> 4;
    const int K = v.K, Kp = v.Kp, slab_bytes = K * Kp * 8;
    const int64_t first_row = p.r0 + (int64_t)p.k * p.L;
    const double *__restrict__ slab0 = v.C + (first_row - v.c0) * ((int64_t)K * Kp);
    int col[CT], voff[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        col[c] = (wave * CT + c) * 16 + c16;
        voff[c] = col[c] < Kp ? (g * Kp + col[c]) * 8 : 0x7ff00000;
    }
    double frag[KH][CT];
    auto load = [&](int slab, int half, int ks, int c) {        // (rows beyond K lie beyond the slab: they read as 0)
        slab = slab < p.n ? slab : p.n - 1;
        const __amdgpu_buffer_rsrc_t res = __builtin_amdgcn_make_buffer_rsrc(const_cast<double *>(slab0 + slab * ((int64_t)K * Kp)), 0, slab_bytes, 0x00020000);
        const int row = min((half * KH + ks) * 4 * Kp * 8, slab_bytes);
        frag[ks][c] = __builtin_bit_cast(double, __builtin_amdgcn_raw_buffer_load_b64(res, voff[c], row, 0));
    };
    if (p.n > 1) {
#pragma unroll
        for (int ks = 0; ks < KH; ++ks)
#pragma unroll
            for (int c = 0; c < CT; ++c) load(1, 0, ks, c);
    }
    for (int i = tid; i < 2 * 16 * LDX; i += NTH) (&X[0][0])[i] = 0.0;
    if (tid == 0) { bad = 0; done = flag[p.u]; }
    __syncthreads();
    if (done) return;
    // the first slab: the start candidate's own cells
    bool small = false;
    double most[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) most[r] = 0.0;
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        if (col[c] >= Kp) continue;
        const double l = local[(first_row + 1) * Kp + col[c]];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = g + 4 * r;
            const double x = i0 + row < K ? slab0[(int64_t)(i0 + row) * Kp + col[c]] * l : 0.0;
            X[0][row * LDX + col[c]] = x;
            most[r] = fmax(most[r], x);
            small |= x > 0.0 && x < SNK_WEIGHT_LEAST;
        }
    }
    auto row_max = [&](int at) {                                // largest weight of every row, per wavefront (lane 15 of each row of lanes has it)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const double m = row16_max(most[r]);
            if (c16 == 15) top[at][wave][g + 4 * r] = m;
        }
    };
    auto row_exponent = [&](int at, int row) -> int {
        double m = top[at][0][row];
#pragma unroll
        for (int w = 1; w < W; ++w) m = fmax(m, top[at][w][row]);
        return trellis_exponent(m);
    };
    row_max(0);
    __syncthreads();
    auto read = [&](int at, int step) { return X[at][c16 * LDX + step * 4 + g]; };
    int e4[4] = {};
    for (int s = 1; s < p.n; ++s) {
        const int from = (s - 1) & 1, to = s & 1;
        f64x4 acc[CT];
#pragma unroll
        for (int c = 0; c < CT; ++c) acc[c] = f64x4{0.0, 0.0, 0.0, 0.0};
        double lw[CT];
#pragma unroll
        for (int c = 0; c < CT; ++c) lw[c] = col[c] < Kp ? local[(first_row + s + 1) * Kp + col[c]] : 0.0;
        double x[3] = {read(from, 0), read(from, 1), 0.0};
#pragma unroll
        for (int half = 0; half < CH; ++half) {
            const int nslab = half + 1 < CH ? s : s + 1, nhalf = half + 1 < CH ? half + 1 : 0;
#pragma unroll
            for (int ks = 0; ks < KH; ++ks) {
                // weights two steps ahead, products, reloads: in this order (left to itself the compiler moves the reloads behind the
                // last product, where the next slab waits for them)
                if (half * KH + ks + 2 < KH * CH) x[(half * KH + ks + 2) % 3] = read(from, half * KH + ks + 2);
#pragma unroll
                for (int c = 0; c < CT; ++c) acc[c] = __builtin_amdgcn_mfma_f64_16x16x4f64(x[(half * KH + ks) % 3], frag[ks][c], acc[c], 0, 0, 0);
#pragma unroll
                for (int c = 0; c < CT; ++c) load(nslab, nhalf, ks, c);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = g + 4 * r, e = row_exponent(from, row);
            const double f = trellis_pow2(-e);
            e4[r] += e;
            most[r] = 0.0;
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                const double x = (acc[c][r] * f) * lw[c];
                if (col[c] < Kp) X[to][row * LDX + col[c]] = x;
                most[r] = fmax(most[r], x);
                small |= x > 0.0 && x < SNK_WEIGHT_LEAST;
            }
        }
        row_max(to);
        __syncthreads();
    }
    if (small) bad = 1;
    __syncthreads();
    if (bad) { if (tid == 0) flag[p.u] = 1; return; }
    // out: rows scaled to [1, 2), their exponents beside them
    const int at = (p.n - 1) & 1;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int row = g + 4 * r, i = i0 + row, e = row_exponent(at, row);
        const double f = trellis_pow2(-e);
        if (i < K) {
#pragma unroll
            for (int c = 0; c < CT; ++c)
                if (col[c] < Kp) M[(p.at * K + i) * Kp + col[c]] = X[at][row * LDX + col[c]] * f;
            if (wave == 0 && c16 == 0) exps[p.at * K + i] = e4[r] + e;
        }
    }
}

// 2. the weights at the pieces' ends: a workgroup per utterance; what a step waits for is what it costs (two barriers, no sum in a row).
// Forward: a wavefront owns 32 columns, CW of them side by side, RG such groups and the four rows of lanes in each split the rows.
// Backward: Q threads a row.  A thread's cells come in H parts of R; each is reloaded with the next part's right after its use.  Every
// wavefront keeps the weights of all candidates, S a lane, and scales them itself.  Bound by a step's latency: 25 pieces of 100
// candidates 47 us, both directions of 18 pieces of 50 20 us each.
template <int R, int H, int CW, int RG, int Q, int S, int NTH>
__global__ void __launch_bounds__(NTH)
trellis_ends_kernel(const TrellisView v, const double *__restrict__ local, const double *__restrict__ M, const int *__restrict__ exps,
                    int *__restrict__ flag, double *__restrict__ ends_out, int64_t *__restrict__ scaled_out)
{
    constexpr bool BACK = Q > 0;
    constexpr int PARTS = BACK ? 1 : RG, STEP = BACK ? 2 * Q : 4 * RG;   // columns / rows between a thread's cells
    __shared__ __align__(16) double vec[256], part[PARTS][256];
    __shared__ int bad;
    const TrellisPiece p = trellis_piece(v, blockIdx.x, 0);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, K = v.K, Kp = v.Kp;
    if (flag[p.u]) return;
    const int bytes = K * Kp * 8;
    const double *__restrict__ m0 = M + p.at * K * Kp;
    const int *__restrict__ e0 = exps + p.at * K;
    double *__restrict__ ends = ends_out + p.at * Kp;
    if (tid == 0) bad = 0;
    const int group = BACK ? 0 : wave / (CW ? CW : 1);
    const int b = BACK ? 2 * (tid % (BACK ? Q : 1)) : (wave % (CW ? CW : 1)) * 32 + 2 * (lane & 15), a = BACK ? tid / (BACK ? Q : 1) : group * 4 + (lane >> 4);
    const bool on = BACK ? a < K : b < Kp && group < RG;
    const int off = on ? (a * Kp + b) * 8 : 0x7ff00000;
    const int steps = p.P - 1, pieces = steps * H;
    f64x2 m[R];
    auto load = [&](int piece, int i) {                         // (rows beyond K and columns beyond Kp read as 0 or meet a weight of 0)
        piece = piece < pieces ? piece : pieces - 1;
        const int k = BACK ? p.P - 1 - piece / H : piece / H, n = (piece % H) * R + i;
        const __amdgpu_buffer_rsrc_t res = __builtin_amdgcn_make_buffer_rsrc(const_cast<double *>(m0 + (int64_t)k * K * Kp), 0, bytes, 0x00020000);
        const int more = min(BACK ? n * STEP * 8 : n * STEP * Kp * 8, bytes);
        m[i] = __builtin_bit_cast(f64x2, __builtin_amdgcn_raw_buffer_load_b128(res, off, more, 0));
    };
    double x[S];                                                // weights of candidates lane, lane + 64 ..
    int e_next[S];
    auto store = [&](int64_t k) {
        if (wave == 0)
#pragma unroll
            for (int i = 0; i < S; ++i)
                if (lane + 64 * i < Kp) ends[k * Kp + lane + 64 * i] = x[i];
    };
    auto exponents = [&](int s) {                               // (a step ahead, like the cells)
        s = s < steps ? s : steps - 1;
#pragma unroll
        for (int i = 0; i < S; ++i) e_next[i] = s >= 0 && lane + 64 * i < K ? e0[(int64_t)(BACK ? p.P - 1 - s : s) * K + lane + 64 * i] : 0;
    };
#pragma unroll
    for (int i = 0; i < S; ++i) {
        const int c = lane + 64 * i;
        x[i] = BACK ? (c < K ? 1.0 : 0.0) : c < Kp ? local[p.r0 * Kp + c] : 0.0;
    }
    store(BACK ? p.P - 1 : 0);
    if (tid < 256)
        for (int i = 0; i < PARTS; ++i) part[i][tid] = 0.0;
    if (tid < 256) vec[tid] = 0.0;
    if (pieces > 0) {
#pragma unroll
        for (int i = 0; i < R; ++i) load(0, i);
    }
    exponents(0);
    __syncthreads();
    int64_t scaled = 0;
    bool small = false;
    // scales the weights x 2^e to at most 2: forward the exponents belong to what goes into a product, backward to what comes out
    auto scale = [&](const int (&e)[S]) {
        int t[S];
        double most = -1e30;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            t[i] = e[i] + trellis_exponent(x[i]);
            if (x[i] > 0.0) most = fmax(most, (double)t[i]);
        }
        most = wave_max(most);
        if (!(most > -1e29)) return;                            // (nothing left: all are 0)
        scaled += (int64_t)most;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const int d = t[i] - (int)most;
            const bool lost = x[i] > 0.0 && d < -489;
            small |= lost;
            x[i] = x[i] > 0.0 && !lost ? x[i] * trellis_pow2(-trellis_exponent(x[i])) * trellis_pow2(d) : 0.0;      // (to [1, 2), then down)
        }
    };
    for (int s = 0; s < steps; ++s) {
        const int k = BACK ? p.P - 1 - s : s;
        int e[S];
#pragma unroll
        for (int i = 0; i < S; ++i) e[i] = e_next[i];
        exponents(s + 1);
        if (!BACK) scale(e);
        if (wave == 0)
#pragma unroll
            for (int i = 0; i < S; ++i)
                if (lane + 64 * i < Kp) vec[lane + 64 * i] = x[i];
        __syncthreads();
        f64x2 sum = {0.0, 0.0};
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int n = h * R + i;
                if (BACK) {
                    const f64x2 w = *reinterpret_cast<const f64x2 *>(&vec[min(b + n * STEP, 254)]);
                    sum[0] = __fma_rn(w[0], m[i][0], sum[0]);
                    sum[1] = __fma_rn(w[1], m[i][1], sum[1]);
                } else {
                    const double w = vec[min(a + n * STEP, 255)];
                    sum[0] = __fma_rn(w, m[i][0], sum[0]);
                    sum[1] = __fma_rn(w, m[i][1], sum[1]);
                }
                load(s * H + h + 1, i);
                if (H == 1 && (i & 1)) __builtin_amdgcn_sched_barrier(0);      // (the reloads stay beside the products)
            }
        if (BACK) {
            double y = quad_sum(sum[0] + sum[1]);
            if (Q == 8) y = eight_sum(y);
            if (on && b == 0) part[0][a] = y;
        } else {
            sum[0] = rows4_sum(sum[0]);
            sum[1] = rows4_sum(sum[1]);
            if (on && lane < 16) *reinterpret_cast<f64x2 *>(&part[group][b]) = sum;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < S; ++i) {
            x[i] = part[0][lane + 64 * i];
#pragma unroll
            for (int g = 1; g < PARTS; ++g) x[i] += part[g][lane + 64 * i];
        }
        if (BACK) scale(e);
        store(BACK ? k - 1 : k + 1);
    }
    if (small) bad = 1;
    __syncthreads();
    if (tid == 0) {
        if (bad) flag[p.u] = 1;
        if (!BACK) scaled_out[p.u] = scaled;
    }
}

// 3. forward.  A wavefront owns 32 columns (two a lane); its four rows of 16 lanes split the predecessors, so a step's sums end inside
// the wavefront and a step costs one barrier.  A thread's KPM CH predecessors come in CH parts; every cell's register is reloaded
// with a later slab's right after its use (NB parts ahead).  9600 rows of 100: 172 us, 4.5 TB/s of a copy's 5.1: bound by memory;
// 600 rows: 38 us, 24 steps.
template <int KPM, int CH, int NB, int NTH>
__global__ void __launch_bounds__(NTH)
trellis_forward_kernel(const TrellisView v, const double *__restrict__ local, const double *__restrict__ least, double bias_min,
                       const double *__restrict__ ends, const int64_t *__restrict__ ends_scaled, int *__restrict__ flag, double *__restrict__ V,
                       double *__restrict__ logz)
{
    constexpr int W = NTH / 64, R = KPM * CH;
    static_assert(NB % CH == 0 || CH % NB == 0, "a step's parts go round the buffers");
    __shared__ __align__(16) double cur[2][4 * R];
    __shared__ double top[2][W];
    __shared__ double part[NTH];
    __shared__ int bad, done;
    const TrellisPiece p = trellis_piece(v, blockIdx.y, blockIdx.x);
    if (p.k >= p.P) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int b = wave * 32 + (lane & 15) * 2, rows = lane >> 4;
    const int K = v.K, Kp = v.Kp, n = p.n;
    const bool lead = rows == 0 && b < Kp;
    const int slab_bytes = K * Kp * 8;
    const int voff = b < Kp ? (rows * R * Kp + b) * 8 : 0x7ff00000;
    const int64_t first_row = p.r0 + (int64_t)p.k * p.L;
    for (int i = tid; i < 8 * R; i += NTH) (&cur[0][0])[i] = 0.0;
    if (tid == 0) { bad = 0; done = flag[p.u]; }
    __syncthreads();
    if (done) return;

    f64x2 cell[NB][KPM];
    const int pieces = n * CH;
    const double *__restrict__ slab0 = v.C + (first_row - v.c0) * ((int64_t)K * Kp);
    auto load = [&](int piece, int i, f64x2 &dst) {             // (rows beyond K lie beyond the slab: they read as 0)
        piece = piece < pieces ? piece : pieces - 1;
        const __amdgpu_buffer_rsrc_t res = __builtin_amdgcn_make_buffer_rsrc(const_cast<double *>(slab0 + (piece / CH) * ((int64_t)K * Kp)), 0, slab_bytes, 0x00020000);
        const int row = min(((piece % CH) * KPM + i) * Kp * 8, slab_bytes);
        dst = __builtin_bit_cast(f64x2, __builtin_amdgcn_raw_buffer_load_b128(res, voff, row, 0));
    };
    auto load_local = [&](int t) -> f64x2 {
        f64x2 x = {0.0, 0.0};
        if (lead) x = *reinterpret_cast<const f64x2 *>(local + (first_row + (t < n ? t : n)) * Kp + b);
        return x;
    };
    // new weights of the lead lanes: LDS, memory, their maximum; small ones are remembered
    bool small = false;
    auto publish = [&](int t, f64x2 x, int at, bool store) {
        double m = 0.0;
        if (lead) {
            *reinterpret_cast<f64x2 *>(&cur[at][b]) = x;
            if (store) *reinterpret_cast<f64x2 *>(V + (first_row + t) * Kp + b) = x;
            m = fmax(x[0], x[1]);
            small |= (x[0] > 0.0 && x[0] < SNK_WEIGHT_LEAST) || (x[1] > 0.0 && x[1] < SNK_WEIGHT_LEAST);
        }
        m = row16_max(m);
        if (lane == 15) top[at][wave] = m;
    };
    if (pieces > 0) {
#pragma unroll
        for (int s = 0; s < NB; ++s)
#pragma unroll
            for (int i = 0; i < KPM; ++i) load(s, i, cell[s][i]);
    }
    f64x2 l1 = load_local(1), l2 = load_local(2);
    {
        f64x2 x = {0.0, 0.0};
        if (lead) x = p.k == 0 ? load_local(0) : *reinterpret_cast<const f64x2 *>(ends + p.at * Kp + b);
        publish(0, x, 0, p.k == 0);
    }
    __syncthreads();
    int64_t scaled = 0;                                         // sum of the exponents taken out
    constexpr int TRIP = NB / CH > 0 ? NB / CH : 1;             // steps a trip, so that buffer indexes are constants
    for (int t = 1; t <= n; t += TRIP) {
#pragma unroll
        for (int s = 0; s < TRIP; ++s) {
            const int now = t + s, from = (now - 1) & 1;
            const bool valid = now <= n;
            f64x2 sum = {0.0, 0.0};
#pragma unroll
            for (int ch = 0; ch < CH; ++ch) {
                f64x2(&c)[KPM] = cell[(s * CH + ch) % NB];
                const double *w = &cur[from][rows * R + ch * KPM];
                double x[KPM];
#pragma unroll
                for (int i = 0; i < KPM; ++i) x[i] = w[i];
                f64x2 more = {0.0, 0.0};
#pragma unroll
                for (int i = 0; i < KPM; i += 2) {              // (the reloads stay beside the products: see trellis_product_kernel)
                    sum[0] = __fma_rn(x[i], c[i][0], sum[0]);
                    sum[1] = __fma_rn(x[i], c[i][1], sum[1]);
                    more[0] = __fma_rn(x[i + 1], c[i + 1][0], more[0]);
                    more[1] = __fma_rn(x[i + 1], c[i + 1][1], more[1]);
                    load((now - 1) * CH + ch + NB, i, c[i]);
                    load((now - 1) * CH + ch + NB, i + 1, c[i + 1]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                sum[0] += more[0];
                sum[1] += more[1];
            }
            sum[0] = rows4_sum(sum[0]);
            sum[1] = rows4_sum(sum[1]);
            double m = top[from][0];
#pragma unroll
            for (int i = 1; i < W; ++i) m = fmax(m, top[from][i]);
            const int e = trellis_exponent(m);
            const double f = trellis_pow2(-e);
            if (valid) {
                scaled += e;
                const f64x2 x = {l1[0] * (sum[0] * f), l1[1] * (sum[1] * f)};
                publish(now, x, 1 - from, true);
            }
            l1 = l2;
            l2 = load_local(now + 2);
            __syncthreads();
        }
    }
    if (small) bad = 1;
    __syncthreads();
    if (bad) { if (tid == 0) flag[p.u] = 1; return; }
    if (!logz || p.k != p.P - 1) return;
    double s = 0.0;
    for (int64_t t = tid; t < p.T; t += NTH) s += least[p.r0 + t];
    part[tid] = s;
    __syncthreads();
    if (tid == 0) {
        s = 0.0;
        for (int i = 0; i < NTH; ++i) s += part[i];
        double z = 0.0;
        for (int a = 0; a < K; ++a) z += cur[n & 1][a];
        if (p.P > 1) scaled += ends_scaled[p.u];
        logz[p.u] = z > 0.0 ? log(z) + (double)scaled * 0.69314718055994530942 - (s + (double)(p.T - 1) * bias_min) * v.inv_tau : -__builtin_inf();
    }
}

// 3. backward: a wavefront owns CH x 16 predecessors, four lanes share each one's successors.  9600 rows of 100: 188 us, 4.1 TB/s
template <int KC, int CH, int NB, int NTH>
__global__ void __launch_bounds__(NTH)
trellis_backward_kernel(const TrellisView v, const double *__restrict__ local, const double *__restrict__ ends, int *__restrict__ flag,
                        double *__restrict__ Wt)
{
    constexpr int W = NTH / 64;
    static_assert(NB % CH == 0 || CH % NB == 0, "a step's parts go round the buffers");
    __shared__ __align__(16) double cur[2][8 * KC];
    __shared__ double top[2][W];
    __shared__ int bad, done;
    const TrellisPiece p = trellis_piece(v, blockIdx.y, blockIdx.x);
    if (p.k >= p.P) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int q = lane & 3, K = v.K, Kp = v.Kp, n = p.n;
    const int slab_bytes = K * Kp * 8;
    const int64_t first_row = p.r0 + (int64_t)p.k * p.L;
    int a[CH], voff[CH];
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
        a[ch] = (ch * W + wave) * 16 + (lane >> 2);
        voff[ch] = a[ch] < K ? (a[ch] * Kp + 2 * q) * 8 : 0x7ff00000;
    }
    for (int i = tid; i < 16 * KC; i += NTH) (&cur[0][0])[i] = 0.0;
    if (tid == 0) { bad = 0; done = flag[p.u]; }
    __syncthreads();
    if (done) return;
    f64x2 cell[NB][KC];
    const int pieces = n * CH;                                  // from the last slab down
    const double *__restrict__ slab0 = v.C + (first_row - v.c0) * ((int64_t)K * Kp);
    auto load = [&](int piece, int i, f64x2 &dst, int off) {    // (columns beyond Kp are the next row's or nothing: their weights are 0)
        piece = piece < pieces ? piece : pieces - 1;
        const __amdgpu_buffer_rsrc_t res = __builtin_amdgcn_make_buffer_rsrc(const_cast<double *>(slab0 + (n - 1 - piece / CH) * ((int64_t)K * Kp)), 0, slab_bytes, 0x00020000);
        dst = __builtin_bit_cast(f64x2, __builtin_amdgcn_raw_buffer_load_b128(res, off + i * 64, 0, 0));
    };
    auto load_local = [&](int t, int ch) -> double {
        return a[ch] < K && q == 0 ? local[(first_row + (t > 0 ? t : 0)) * Kp + a[ch]] : 0.0;
    };
    if (pieces > 0) {
#pragma unroll
        for (int s = 0; s < NB; ++s)
#pragma unroll
            for (int i = 0; i < KC; ++i) load(s, i, cell[s][i], voff[s % CH]);
    }
    double l1[CH], l2[CH];
    double m0 = 0.0;
    bool small = false;
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
        if (a[ch] < K && q == 0) {
            const double w = p.k == p.P - 1 ? 1.0 : ends[p.at * Kp + a[ch]], x = load_local(n, ch) * w;
            cur[n & 1][a[ch]] = x;
            if (p.k == p.P - 1) Wt[(first_row + n) * Kp + a[ch]] = w;
            small |= x > 0.0 && x < SNK_WEIGHT_LEAST;
            m0 = fmax(m0, x);
        }
        l1[ch] = load_local(n - 1, ch);
        l2[ch] = load_local(n - 2, ch);
    }
    m0 = wave_max(m0);
    if (lane == 0) top[n & 1][wave] = m0;
    __syncthreads();
    constexpr int TRIP = NB / CH > 0 ? NB / CH : 1;
    for (int k = 0; k < n; k += TRIP) {
#pragma unroll
        for (int s = 0; s < TRIP; ++s) {
            const int t = n - 1 - (k + s);                      // the row of this step; < 0: beyond the piece
            const bool valid = t >= 0;
            const int from = (t + 1) & 1, to = 1 - from;
            double m = top[from][0];
#pragma unroll
            for (int i = 1; i < W; ++i) m = fmax(m, top[from][i]);
            const double f = trellis_pow2(-trellis_exponent(m));
            m = 0.0;
#pragma unroll
            for (int ch = 0; ch < CH; ++ch) {
                f64x2(&c)[KC] = cell[(s * CH + ch) % NB];
                f64x2 sum = {0.0, 0.0};
#pragma unroll
                for (int i = 0; i < KC; ++i) {
                    const f64x2 x = *reinterpret_cast<const f64x2 *>(&cur[from][8 * i + 2 * q]);
                    sum[0] = __fma_rn(x[0], c[i][0], sum[0]);
                    sum[1] = __fma_rn(x[1], c[i][1], sum[1]);
                    load((k + s) * CH + ch + NB, i, c[i], voff[(ch + NB) % CH]);
                    if (i & 1) __builtin_amdgcn_sched_barrier(0);      // (the reloads stay beside the products)
                }
                double y = sum[0] + sum[1];
                y = quad_sum(y) * f;
                if (valid && a[ch] < K && q == 0) {
                    const double x = l1[ch] * y;
                    cur[to][a[ch]] = x;
                    Wt[(first_row + t) * Kp + a[ch]] = y;
                    small |= x > 0.0 && x < SNK_WEIGHT_LEAST;
                    m = fmax(m, x);
                }
                l1[ch] = l2[ch];
                l2[ch] = load_local(t - 2, ch);
            }
            m = wave_max(m);
            if (valid && lane == 0) top[to][wave] = m;
            __syncthreads();
        }
    }
    if (small) bad = 1;
    __syncthreads();
    if (bad && tid == 0) flag[p.u] = 1;
}

// ---- the flagged utterances in logarithms (SUM false: temperature 0, the largest term of every sum) ----------------------------------
// Every row of the sums is taken relative to the largest weight of the row before (after) it: a row's differences stay the size of a step's
// costs over tau, where the whole path's would round to more than the differences themselves once tau is 2^-50 of them.
// A workgroup has an utterance: chains of T steps of one compute unit.  600 rows of 100 candidates: a draw 6.2 ms (2.8 at temperature 0),
// a posterior 15.4; sixteen such utterances side by side 11.9, 6.8 and 21.5.
template <bool SUM>
__global__ void __launch_bounds__(1024)
trellis_forward_log_kernel(const TrellisView v, const int *__restrict__ flag, double *__restrict__ alpha, double *__restrict__ logz)
{
    __shared__ double cur[256], part_max[1024], part_sum[1024], row_top[2][4];
    const int u = v.first + blockIdx.x;
    if (!flag[u]) return;
    const int K = v.K, Kp = v.Kp, tid = threadIdx.x;
    const int KB = (K + 63) & ~63, P = 1024 / KB;
    const int b = tid % KB, part = tid / KB;
    const int64_t r0 = v.off[u], T = v.off[u + 1] - r0;
    const double ninf = -__builtin_inf();
    const bool mine = b < K && part < P;
    double scaled = 0.0;                                        // what the rows were taken relative to
    auto publish = [&](int64_t t, double x) {                   // by the first 256 threads; x -inf beyond K
        if (tid < K) {
            cur[tid] = x;
            alpha[(r0 + t) * Kp + tid] = x;
        }
        if (SUM) {
            x = wave_max(x);
            if ((tid & 63) == 0) row_top[t & 1][tid >> 6] = x;
        }
    };
    if (tid < 256) publish(0, tid < K ? trellis_local(v.cand[r0 * K + tid], v.tdist[r0 * K + tid], v.n_units, v.inv_tau) : ninf);
    __syncthreads();
    for (int64_t t = 0; t + 1 < T; ++t) {
        double base = 0.0;
        if (SUM) {
            const double *m = row_top[t & 1];
            base = fmax(fmax(m[0], m[1]), fmax(m[2], m[3]));
            if (base == ninf) base = 0.0;
            scaled += base;
        }
        const double *__restrict__ c = v.C + (r0 + t - v.c0) * K * Kp + b;
        double top = ninf, sum = 0.0;
        if (mine) {
            for (int a = part; a < K; a += P) top = fmax(top, cur[a] + c[(int64_t)a * Kp]);
            if (SUM && top > ninf)
                for (int a = part; a < K; a += P) sum += exp(cur[a] + c[(int64_t)a * Kp] - top);
        }
        part_max[tid] = top;
        part_sum[tid] = sum;
        __syncthreads();
        if (tid < 256) {
            double x = ninf;
            if (tid < K) {
                for (int q = 0; q < P; ++q) x = fmax(x, part_max[q * KB + tid]);
                if (SUM && x > ninf) {
                    double s = 0.0;
                    for (int q = 0; q < P; ++q)
                        if (part_max[q * KB + tid] > ninf) s += part_sum[q * KB + tid] * exp(part_max[q * KB + tid] - x);
                    x = (x - base) + log(s);
                }
                const int64_t at = (r0 + t + 1) * K + tid;
                x += trellis_local(v.cand[at], v.tdist[at], v.n_units, v.inv_tau);
            }
            publish(t + 1, x);
        }
        __syncthreads();
    }
    if (logz && tid == 0) {
        double all = ninf;
        for (int a = 0; a < K; ++a) all = fmax(all, cur[a]);
        double s = 0.0;
        if (all > ninf)
            for (int a = 0; a < K; ++a) s += exp(cur[a] - all);
        logz[u] = all > ninf ? scaled + (all + log(s)) : ninf;
    }
}

__global__ void __launch_bounds__(1024)
trellis_backward_log_kernel(const TrellisView v, const int *__restrict__ flag, double *__restrict__ beta)
{
    __shared__ double into[2][256], row_top[2][16];
    const int u = v.first + blockIdx.x;
    if (!flag[u]) return;
    const int K = v.K, Kp = v.Kp, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t r0 = v.off[u], T = v.off[u + 1] - r0;
    const double ninf = -__builtin_inf();
    double top_into = ninf;
    if (tid < K) {
        const int64_t at = (r0 + T - 1) * K + tid;
        beta[(r0 + T - 1) * Kp + tid] = 0.0;
        top_into = trellis_local(v.cand[at], v.tdist[at], v.n_units, v.inv_tau);
        into[(T - 1) & 1][tid] = top_into;
    }
    top_into = wave_max(top_into);
    if (lane == 0) row_top[(T - 1) & 1][wave] = top_into;
    __syncthreads();
    for (int64_t t = T - 2; t >= 0; --t) {
        const double *next = into[(t + 1) & 1];
        double base = ninf;
        for (int i = 0; i < 16; ++i) base = fmax(base, row_top[(t + 1) & 1][i]);
        if (base == ninf) base = 0.0;
        top_into = ninf;
        for (int a = wave; a < K; a += 16) {
            const double *__restrict__ c = v.C + (r0 + t - v.c0) * K * Kp + (int64_t)a * Kp;
            double x[4], top = ninf;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int b = lane + 64 * j;
                x[j] = b < K ? next[b] + c[b] : ninf;
                top = fmax(top, x[j]);
            }
            top = wave_max(top);
            double s = 0.0;
            if (top > ninf) {
#pragma unroll
                for (int j = 0; j < 4; ++j) s += exp(x[j] - top);
                s = wave_sum(s);
            }
            if (lane == 0) {
                const double y = top > ninf ? (top - base) + log(s) : ninf;
                const int64_t at = (r0 + t) * K + a;
                beta[(r0 + t) * Kp + a] = y;
                const double x = y + trellis_local(v.cand[at], v.tdist[at], v.n_units, v.inv_tau);
                into[t & 1][a] = x;
                top_into = fmax(top_into, x);
            }
        }
        if (lane == 0) row_top[t & 1][wave] = top_into;
        __syncthreads();
    }
}

// ---- posteriors: a workgroup per row ---------------------------------------------------------------------------------------------------
// The row's bucket uses are integers in units of 2^-50: their sums are the same in any order.  The two outermost buckets take most
// cells and are summed in registers; the others go to LDS.  9600 rows of 100: 0.31 ms, 2.5 TB/s: bound by the cells' vector work (bucket,
// integer sums), 174 us for 1200 rows of 200.
__global__ void __launch_bounds__(256)
trellis_posterior_kernel(const TrellisView v, const int *__restrict__ flag, const double *__restrict__ V, const double *__restrict__ Wt,
                         const double *__restrict__ ends, const double *__restrict__ local, const double *__restrict__ logz, const int *__restrict__ bucket_edges, int n_buckets,
                         double *__restrict__ posterior, double *__restrict__ row_uses)
{
    __shared__ double in[256], out[256], red[8];
    __shared__ __align__(16) int edges[SNK_EDGE_WORDS];
    __shared__ int id0[256], id1[256];
    __shared__ u64 uses[64];
    const int64_t t = v.c0 + blockIdx.x;
    const int K = v.K, Kp = v.Kp, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int u = trellis_utterance(v.off, v.first, v.n_utts, t);
    const bool logs = flag[u] != 0, last = t + 1 == v.off[u + 1];
    const double ninf = -__builtin_inf(), z = logz[u];
    const bool dead = !(z > ninf);
    if (logs) {
        // of the row's own sum, and a candidate's share among what follows it (below) of that candidate's: both sum to 1, however large the
        // exponents and what they round away
        const double x = tid < K ? V[t * Kp + tid] + Wt[t * Kp + tid] : ninf, m = wave_max(x);
        if (lane == 0) red[wave] = m;
        __syncthreads();
        const double most = fmax(fmax(red[0], red[1]), fmax(red[2], red[3]));
        const double e = x > ninf ? exp(x - most) : 0.0, s = wave_sum(e);
        if (lane == 0) red[4 + wave] = s;
        __syncthreads();
        if (tid < K) {
            const double p = dead ? 0.0 : e / ((red[4] + red[5]) + (red[6] + red[7]));
            posterior[t * K + tid] = p;
            in[tid] = p;
        }
    } else {
        // sum_a v w of the row, and the power of two that the backward step into this row took out
        const double a = tid < K ? V[t * Kp + tid] : 0.0, w = tid < K ? Wt[t * Kp + tid] : 0.0;
        const double p = a * w, s = wave_sum(p);
        // (behind a piece's last row stand the weights that its recursion began with)
        const int64_t L = trellis_piece_length(v.off[u + 1] - v.off[u] - 1);
        const TrellisPiece piece = trellis_piece(v, u - v.first, (int)((t - v.off[u]) / L));
        const bool edge = piece.k + 1 < piece.P && (t + 1 - piece.r0) % L == 0;
        const double *__restrict__ next = edge ? ends + piece.at * Kp : Wt + (t + 1) * Kp;
        const double x = !last && tid < K ? local[(t + 1) * Kp + tid] * next[tid] : 0.0;
        const double m = wave_max(x);
        if (lane == 0) { red[wave] = s; red[4 + wave] = m; }
        __syncthreads();
        const double total = (red[0] + red[1]) + (red[2] + red[3]);
        const double most = fmax(fmax(red[4], red[5]), fmax(red[6], red[7]));
        if (tid < K) {
            posterior[t * K + tid] = dead ? 0.0 : p / total;
            // (a / total <= 1 / w <= 2^490; a candidate that leads nowhere has no share)
            in[tid] = w > 0.0 ? a / total * trellis_pow2(-trellis_exponent(most)) : 0.0;
            out[tid] = x;
        }
    }
    if (!row_uses) return;
    if (tid < K) {
        id0[tid] = (int)v.cand[t * K + tid];
        if (!last) {
            const int64_t at = (t + 1) * K + tid;
            id1[tid] = (int)v.cand[at];
            if (logs) out[tid] = trellis_local(v.cand[at], v.tdist[at], v.n_units, v.inv_tau) + Wt[(t + 1) * Kp + tid];
        }
    }
    if (tid < 64) uses[tid] = 0;
    trellis_load_edges(edges, bucket_edges, n_buckets);
    __syncthreads();
    const TrellisEdges look = trellis_edges(edges);
    if (!last && !dead) {
        const double *__restrict__ c = v.C + (t - v.c0) * K * Kp;
        u64 first = 0, far = 0;
        auto add = [&](double p, int a, int b) {
            const u64 w = sample_fix(p, SNK_USES_UNIT);
            if (!w) return;
            const int k = trellis_bucket(id1[b] - id0[a], look);
            if (k == 0) first += w;
            else if (k == n_buckets - 1) far += w;
            else atomicAdd(&uses[k], w);
        };
        for (int a = wave; a < K; a += 4) {
            const double va = in[a];
            if (logs) {
                double x[4], m = ninf, s = 0.0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int b = lane + 64 * j;
                    x[j] = b < K ? c[a * Kp + b] + out[b] : ninf;
                    m = fmax(m, x[j]);
                }
                m = wave_max(m);
                if (!(va > 0.0 && m > ninf)) continue;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    x[j] = x[j] > ninf ? exp(x[j] - m) : 0.0;
                    s += x[j];
                }
                s = va / wave_sum(s);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (x[j] > 0.0) add(x[j] * s, a, lane + 64 * j);
            } else
                for (int b = lane; b < K; b += 64) add(va * c[a * Kp + b] * out[b], a, b);
        }
        if (first) atomicAdd(&uses[0], first);
        if (far) atomicAdd(&uses[n_buckets - 1], far);
    }
    __syncthreads();
    if (tid < n_buckets) row_uses[t * n_buckets + tid] = (double)uses[tid] * (1.0 / SNK_USES_UNIT);
}

// uses[class, bucket] = sum over the rows of the class: a workgroup per class and bucket, the rows in a fixed order (9600 rows of 32
// buckets, 3 classes: 30 us, each workgroup reads its column alone)
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

// ---- draws -----------------------------------------------------------------------------------------------------------------------------
// The random number of a row does not depend on the candidate behind it, so the predecessor of EVERY candidate is drawn at once,
// all rows side by side (the weights and their truncation once per candidate, whatever the number of draws); what is left of the
// chain is following those pointers.  9600 rows of 100 candidates, four draws: 1.30 ms for the 960 000 weighted rows, 1.36 ns each as in
// sample_rows (51 us for 19200): bound by the search's dependent chain (sample_device.h), 0.6 TB/s of cells.
//
// Weights of the row of scores V[t,.] (E[t,.,after]) / alpha + X: x in the order of the scores, -inf: takes no part.
template <int E>
__device__ __forceinline__ bool trellis_row(const double (&p)[E], bool logs, const SampleRule &rule, double (&x)[E], WaveRow<E> &row, double &m)
{
    const double ninf = -__builtin_inf();
    m = ninf;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        x[e] = p[e] > (logs ? ninf : 0.0) ? p[e] : ninf;        // (neither NaN)
        m = fmax(m, x[e]);
    }
    m = wave_max(m);
    if (m == ninf) return false;
    const double inv = logs ? 0.0 : 1.0 / m;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (logs) row.w[e] = x[e] == ninf ? 0 : sample_weight(sample_exponent(x[e], m, 1.0), SNK_SAMPLE_UNIT);
        else row.w[e] = x[e] == m ? (u64)SNK_SAMPLE_UNIT : x[e] == ninf ? 0 : sample_fix(x[e] * inv, SNK_SAMPLE_UNIT);
    }
    wave_row_keep<E>(x, rule, SNK_SAMPLE_UNIT, row);
    return true;
}

// A workgroup takes 32 of a row's columns, or 8 where that leaves workgroups too few: one utterance of 120 rows of 30 candidates 4.7 us
// instead of 9.6, 600 rows of 100 79 instead of 92; 9600 rows of 100 1.35 ms with 8, 1.30 with 32.
template <int E>
__global__ void __launch_bounds__(256)
trellis_pointer_kernel(const TrellisView v, int shift, const int *__restrict__ flag, const double *__restrict__ V, SampleRule rule, bool greedy,
                       const double *__restrict__ u, int n_draws, int64_t all_rows, int all_utts, unsigned char *__restrict__ pointer,
                       int *__restrict__ root)
{
    extern __shared__ double cells[];                           // [1 << shift][LDA], LDA = K | 1
    const int64_t t = v.c0 + blockIdx.x;
    const int K = v.K, Kp = v.Kp, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int utt = trellis_utterance(v.off, v.first, v.n_utts, t);
    const bool logs = flag[utt] != 0, last = t + 1 == v.off[utt + 1];
    double vt[E];
#pragma unroll
    for (int e = 0; e < E; ++e) vt[e] = lane * E + e < K ? V[t * Kp + lane * E + e] : (logs ? -__builtin_inf() : 0.0);
    double x[E], m;
    WaveRow<E> row;
    if (last) {                                                 // the path's end
        if (blockIdx.y || wave) return;
        const bool any = trellis_row<E>(vt, logs, rule, x, row, m);
        for (int s = lane; s - lane < n_draws; s += 64) {       // a lane has a draw
            const double r = greedy || s >= n_draws ? 0.0 : u[(int64_t)s * all_rows + t];
            const int k = any ? wave_row_picks<E>(row, r, min(n_draws - (s - lane), 64)) : -1;
            if (s < n_draws) root[(int64_t)s * all_utts + utt] = k;
        }
        return;
    }
    const int LDA = K | 1, columns = 1 << shift, b0 = blockIdx.y * columns;
    const double *__restrict__ c = v.C + (t - v.c0) * K * Kp;
    for (int i = tid; i < K << shift; i += 256) {
        const int a = i >> shift, b = i & (columns - 1);
        cells[b * LDA + a] = b0 + b < K ? c[a * Kp + b0 + b] : 0.0;
    }
    const double first = greedy || lane >= n_draws ? 0.0 : u[(int64_t)lane * all_rows + t];
    __syncthreads();
    for (int b = wave; b < columns && b0 + b < K; b += 4) {
        double p[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int a = lane * E + e;
            const double cell = a < K ? cells[b * LDA + a] : 0.0;
            p[e] = logs ? vt[e] + cell : vt[e] * cell;
        }
        const bool any = trellis_row<E>(p, logs, rule, x, row, m);
        for (int s = lane; s - lane < n_draws; s += 64) {
            const double r = s < 64 ? first : greedy || s >= n_draws ? 0.0 : u[(int64_t)s * all_rows + t];
            const int k = any ? wave_row_picks<E>(row, r, min(n_draws - (s - lane), 64)) : 0;        // (a candidate nothing leads to is on no path)
            if (s < n_draws) pointer[((int64_t)s * all_rows + t) * K + b0 + b] = (unsigned char)k;
        }
    }
}

// Follows the pointers of an utterance and draw: a workgroup each, as many rows at a time as LDS holds.  The rows are cut into
// pieces of 32: all K ways through every piece side by side, then the pieces' ends one after the other, then the pieces side by side.
// 600 rows of 100: 14 us, a chain of 600 loads from LDS would take 40.
#define SNK_CHASE_BYTES (128 * 1024)
#define SNK_CHASE_PIECE 32
__global__ void __launch_bounds__(512)
trellis_chase_kernel(const TrellisView v, const unsigned char *__restrict__ pointer, const int *__restrict__ root, int64_t all_rows, int all_utts,
                     unsigned char *__restrict__ slots)
{
    extern __shared__ unsigned char lds[];
    const int utt = v.first + blockIdx.x, s = blockIdx.y, tid = threadIdx.x;
    const int K = v.K;
    const int64_t r0 = v.off[utt], T = v.off[utt + 1] - r0;
    const int at_end = root[(int64_t)s * all_utts + utt];
    if (at_end < 0) return;
    const int64_t fit = SNK_CHASE_BYTES / (K + (K + SNK_CHASE_PIECE - 1) / SNK_CHASE_PIECE + 1) - SNK_CHASE_PIECE;
    unsigned char *__restrict__ out = slots + (int64_t)s * all_rows + r0;
    int after = at_end;                                         // slot of row `hi`
    if (tid == 0) out[T - 1] = (unsigned char)at_end;
    for (int64_t hi = T - 1; hi > 0;) {
        const int n = (int)(hi < fit ? hi : fit);               // rows hi - n .. hi - 1
        const int64_t lo = hi - n;
        const int pieces = (n + SNK_CHASE_PIECE - 1) / SNK_CHASE_PIECE;
        unsigned char *ptr = lds, *way = lds + (size_t)n * K, *start = way + (size_t)pieces * K;
        const unsigned char *__restrict__ src = pointer + ((int64_t)s * all_rows + r0 + lo) * K;
        __syncthreads();
        for (int i = tid; i < n * K; i += 512) ptr[i] = src[i];
        __syncthreads();
        for (int i = tid; i < pieces * K; i += 512) {           // piece p: rows p 32 .. from its end to its first row
            const int p = i / K, from = p * SNK_CHASE_PIECE, to = from + SNK_CHASE_PIECE < n ? from + SNK_CHASE_PIECE : n;
            int k = i - p * K;
            for (int r = to - 1; r >= from; --r) k = ptr[r * K + k];
            way[i] = (unsigned char)k;
        }
        __syncthreads();
        if (tid == 0) {
            int k = after;
            for (int p = pieces - 1; p >= 0; --p) { start[p] = (unsigned char)k; k = way[p * K + k]; }
        }
        __syncthreads();
        for (int p = tid; p < pieces; p += 512) {
            const int from = p * SNK_CHASE_PIECE, to = from + SNK_CHASE_PIECE < n ? from + SNK_CHASE_PIECE : n;
            int k = start[p];
            for (int r = to - 1; r >= from; --r) { k = ptr[r * K + k]; out[lo + r] = (unsigned char)k; }
        }
        if (pieces) after = way[start[0]];
        hi = lo;
    }
}

// Unit, cost and log probability of every row of a path: a wavefront per row and draw.  The join cost is taken from the units
// themselves, in differences: the cells only hold its exponential.  9600 rows, four draws: 106 us, most of it the row's truncation again.
template <int E>
__global__ void __launch_bounds__(256)
trellis_path_kernel(const TrellisView v, const TrellisCosts c, const int *__restrict__ flag, const double *__restrict__ V, SampleRule rule,
                    const int *__restrict__ root, const unsigned char *__restrict__ slots, int64_t all_rows, int all_utts,
                    int64_t *__restrict__ path, double *__restrict__ row_cost, double *__restrict__ row_logp)
{
    const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= v.rows) return;
    const int64_t t = v.c0 + i;
    const int s = blockIdx.y, lane = threadIdx.x & 63, K = v.K, Kp = v.Kp;
    const int utt = trellis_utterance(v.off, v.first, v.n_utts, t);
    const int64_t at = (int64_t)s * all_rows + t;
    if (root[(int64_t)s * all_utts + utt] < 0) {
        if (lane == 0) path[at] = -1;
        return;
    }
    const bool logs = flag[utt] != 0, last = t + 1 == v.off[utt + 1];
    const int k = slots[at], after = last ? 0 : slots[at + 1];
    double p[E], x[E], m;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int a = lane * E + e;
        p[e] = a < K ? V[t * Kp + a] : (logs ? -__builtin_inf() : 0.0);
        if (!last && a < K) {
            const double cell = v.C[((t - v.c0) * K + a) * Kp + after];
            p[e] = logs ? p[e] + cell : p[e] * cell;
        }
    }
    WaveRow<E> row;
    trellis_row<E>(p, logs, rule, x, row, m);
    const double mine = wave_row_value<E>(x, k / E, k % E);
    const double lp = (logs ? sample_exponent(mine, m, 1.0) : mine == m ? 0.0 : log(mine * (1.0 / m))) - log((double)row.total / SNK_SAMPLE_UNIT);
    double cost = v.tdist[t * K + k];
    const int64_t id = v.cand[t * K + k];
    const int64_t next = last ? -1 : v.cand[(t + 1) * K + after];
    if (!last && (!trellis_usable(id, v.n_units) || !trellis_usable(next, v.n_units))) cost = __builtin_inf();    // (not one of these was drawn:
    else if (!last) {                                                                                             // the candidates changed under the call)
        const float *__restrict__ pe = c.JC + (id + 1) * c.Jp, *__restrict__ ps = c.JC + next * c.Jp;
        double d2 = 0.0;
        for (int j = lane; j < c.Dj; j += 64) {
            const double d = (double)pe[j] * c.wj[j] - (double)ps[j] * c.wj[j];
            d2 = __fma_rn(d, d, d2);
        }
        cost += sqrt(wave_sum(d2));
        int cls = c.n_classes ? (c.join_class ? c.join_class[t] : 0) : -1;
        if (cls >= 0 && cls < c.n_classes) {
            const bool below = lane < c.n_buckets - 1 && (int)(next - id) >= c.edges[lane];
            cost += c.bias[(int64_t)cls * c.n_buckets + __popcll(__ballot(below))];
        }
    }
    if (lane == 0) { path[at] = id; row_cost[at] = cost; row_logp[at] = lp; }
}

// sums over an utterance's rows, in a fixed order
__global__ void __launch_bounds__(256)
trellis_total_kernel(const TrellisView v, const int *__restrict__ root, const double *__restrict__ row_cost, const double *__restrict__ row_logp,
                     int64_t all_rows, int all_utts, double *__restrict__ cost, double *__restrict__ logp)
{
    __shared__ double pc[256], pl[256];
    const int utt = v.first + blockIdx.x, s = blockIdx.y, tid = threadIdx.x;
    const int64_t r0 = v.off[utt], T = v.off[utt + 1] - r0, at = (int64_t)s * all_utts + utt;
    const bool dead = root[at] < 0;
    double c = 0.0, l = 0.0;
    if (!dead)
        for (int64_t t = tid; t < T; t += 256) { c += row_cost[(int64_t)s * all_rows + r0 + t]; l += row_logp[(int64_t)s * all_rows + r0 + t]; }
    pc[tid] = c; pl[tid] = l;
    __syncthreads();
    for (int o = 128; o; o >>= 1) {
        if (tid < o) { pc[tid] += pc[tid + o]; pl[tid] += pl[tid + o]; }
        __syncthreads();
    }
    if (tid == 0) {
        cost[at] = dead ? __builtin_inf() : pc[0];
        if (logp) logp[at] = dead ? -__builtin_inf() : pl[0];
    }
}

// ---- launches ---------------------------------------------------------------------------------------------------------------------------
void launch_trellis_offsets(const int64_t *off_host, int n_utts, int flag_value, int64_t *off, int *flag, hipStream_t s)
{
    for (int v = 0; v <= n_utts; v += 256) {
        TrellisOffsets part;
        for (int i = 0; i < 256; ++i) part.v[i] = v + i <= n_utts ? off_host[v + i] : 0;
        hipLaunchKernelGGL(trellis_offsets_kernel, dim3(1), dim3(256), 0, s, part, v, n_utts, flag_value, off, flag);
    }
}

void launch_trellis_local(const TrellisView &v, double *local, double *least, int *flag, hipStream_t s)
{
    hipLaunchKernelGGL(trellis_local_kernel, dim3((unsigned)((v.rows + 3) / 4)), dim3(256), 0, s, v, local, least, flag);
}

// A wavefront's registers hold 7 tiles of 16 x 16 (two workgroups of eight wavefronts a compute unit): K is cut into as few equal
// tiles of at most 112 -- of at most 64 where that would leave less than three quarters of the workgroups that run at once (posteriors
// of 100 candidates, 302 columns, with tiles of 64 and of 112: 100 rows 233 and 258 us, 300 rows 349 and 363, 450 rows 430 and 409).
void launch_trellis_costs(const TrellisView &v, const TrellisCosts &c, bool logs, int *flag, double *X, hipStream_t s)
{
    if (v.rows < 2) return;
    int n = (v.K + 111) / 112;
    if (v.K > 64 && (v.rows - 1) * n * n < 384) n = (v.K + 63) / 64;
    const int rt = ((v.K + n - 1) / n + 15) / 16;
    const dim3 grid((unsigned)(v.rows - 1), n, n);
#define SNK_COST(RT_, RM_, CM_, NTH_, OCC_, DC_)                                                                                            \
    do {                                                                                                                     \
        if (logs) hipLaunchKernelGGL((trellis_cost_kernel<RT_, RM_, CM_, NTH_, OCC_, DC_, true>), grid, dim3(NTH_), 0, s, v, c, flag, X);      \
        else hipLaunchKernelGGL((trellis_cost_kernel<RT_, RM_, CM_, NTH_, OCC_, DC_, false>), grid, dim3(NTH_), 0, s, v, c, flag, X);          \
    } while (0)
    if (rt <= 2) SNK_COST(2, 1, 1, 256, 4, 32);
    else if (rt <= 4) SNK_COST(4, 2, 2, 256, 4, 32);
    else if (rt <= 6) SNK_COST(6, 3, 3, 256, 3, 16);
    else SNK_COST(7, 7, 1, 512, 4, 16);
#undef SNK_COST
}

int trellis_most_pieces(const int64_t *off, int n_utts)
{
    int64_t most = 1;
    for (int i = 0; i < n_utts; ++i) {
        const int64_t S = off[i + 1] - off[i] - 1, L = trellis_piece_length(S);
        if (S > L && (S + L - 1) / L > most) most = (S + L - 1) / L;
    }
    return (int)most;
}
size_t trellis_piece_places(const TrellisView &v) { return (size_t)(v.rows / SNK_PIECE_LEAST + v.n_utts); }

void launch_trellis_ends(const TrellisView &v, const double *local, bool both, int *flag, double *M, int *exps, double *ends_v, double *ends_w,
                         int64_t *scaled, hipStream_t s)
{
    const int n = v.pieces;
    if (n == 1) return;
    const int64_t all = (((int64_t)n * v.n_utts + 7) / 8) * 8;
    const int row_blocks = (v.K + 15) / 16;
    const dim3 grid((unsigned)(all * row_blocks));
#define SNK_PROD(CT_, KH_, CH_, NTH_)                                                                                                             \
    hipLaunchKernelGGL((trellis_product_kernel<CT_, KH_, CH_, NTH_>), grid, dim3(NTH_), 0, s, v, local, n, row_blocks, !both, flag, M, exps)
    if (v.K <= 32) SNK_PROD(1, 8, 1, 128);
    else if (v.K <= 64) SNK_PROD(1, 16, 1, 256);
    else if (v.K <= 80) SNK_PROD(2, 20, 1, 192);
    else if (v.K <= 104) SNK_PROD(2, 26, 1, 256);
    else if (v.K <= 128) SNK_PROD(2, 32, 1, 256);
    else if (v.K <= 160) SNK_PROD(1, 20, 2, 640);
    else SNK_PROD(2, 26, 2, 448);
#undef SNK_PROD
#define SNK_ENDS(R_, H_, CW_, RG_, RB_, HB_, Q_, S_, NTH_)                                                                                           \
    do {                                                                                                                                              \
        hipLaunchKernelGGL((trellis_ends_kernel<R_, H_, CW_, RG_, 0, S_, NTH_>), dim3(v.n_utts), dim3(NTH_), 0, s, v, local, M, exps, flag, ends_v, scaled);  \
        if (both)                                                                                                                                     \
            hipLaunchKernelGGL((trellis_ends_kernel<RB_, HB_, 0, 0, Q_, S_, 32 * ((Q_ == 8 ? 4 : 8) * Q_)>), dim3(v.n_utts), dim3(32 * ((Q_ == 8 ? 4 : 8) * Q_)), 0, s, v, local, M, \
                               exps, flag, ends_w, scaled);                                                                                           \
    } while (0)
    if (v.K <= 32) SNK_ENDS(2, 1, 1, 4, 2, 1, 8, 1, 256);
    else if (v.K <= 64) SNK_ENDS(4, 1, 2, 4, 4, 1, 8, 1, 512);
    else if (v.K <= 104) SNK_ENDS(7, 1, 4, 4, 7, 1, 8, 2, 1024);
    else if (v.K <= 128) SNK_ENDS(8, 1, 4, 4, 8, 1, 8, 2, 1024);
    else SNK_ENDS(13, 2, 7, 2, 13, 2, 4, 4, 896);
#undef SNK_ENDS
}

void launch_trellis_forward(const TrellisView &v, const double *local, const double *least, double bias_min, const double *ends,
                            const int64_t *ends_scaled, int *flag, double *V, double *logz, hipStream_t s)
{
    const dim3 grid(v.pieces, v.n_utts);
#define SNK_FWD(KPM_, CH_, NB_, NTH_) hipLaunchKernelGGL((trellis_forward_kernel<KPM_, CH_, NB_, NTH_>), grid, dim3(NTH_), 0, s, v, local, least, bias_min, ends, ends_scaled, flag, V, logz)
    if (v.K <= 32) SNK_FWD(8, 1, 4, 64);
    else if (v.K <= 64) SNK_FWD(16, 1, 1, 128);
    else if (v.K <= 104) SNK_FWD(26, 1, 1, 256);
    else if (v.K <= 128) SNK_FWD(32, 1, 1, 256);
    else SNK_FWD(26, 2, 1, 448);
#undef SNK_FWD
}

void launch_trellis_backward(const TrellisView &v, const double *local, const double *ends, int *flag, double *Wt, hipStream_t s)
{
    const dim3 grid(v.pieces, v.n_utts);
#define SNK_BWD(KC_, CH_, NB_, NTH_) hipLaunchKernelGGL((trellis_backward_kernel<KC_, CH_, NB_, NTH_>), grid, dim3(NTH_), 0, s, v, local, ends, flag, Wt)
    if (v.K <= 32) SNK_BWD(4, 1, 4, 128);
    else if (v.K <= 64) SNK_BWD(8, 1, 2, 256);
    else if (v.K <= 112) SNK_BWD(14, 1, 2, 448);
    else SNK_BWD(26, 2, 1, 448);
#undef SNK_BWD
}

void launch_trellis_forward_log(const TrellisView &v, bool sum, const int *flag, double *alpha, double *logz, hipStream_t s)
{
    if (sum) hipLaunchKernelGGL((trellis_forward_log_kernel<true>), dim3(v.n_utts), dim3(1024), 0, s, v, flag, alpha, logz);
    else hipLaunchKernelGGL((trellis_forward_log_kernel<false>), dim3(v.n_utts), dim3(1024), 0, s, v, flag, alpha, logz);
}

void launch_trellis_backward_log(const TrellisView &v, const int *flag, double *beta, hipStream_t s)
{
    hipLaunchKernelGGL(trellis_backward_log_kernel, dim3(v.n_utts), dim3(1024), 0, s, v, flag, beta);
}

void launch_trellis_posterior(const TrellisView &v, const int *flag, const double *V, const double *Wt, const double *ends, const double *local, const double *logz,
                              const int *edges, int n_buckets, double *posterior, double *row_uses, hipStream_t s)
{
    hipLaunchKernelGGL(trellis_posterior_kernel, dim3((unsigned)v.rows), dim3(256), 0, s, v, flag, V, Wt, ends, local, logz, edges, n_buckets, posterior, row_uses);
}

void launch_trellis_uses(const double *row_uses, const int32_t *join_class, int64_t rows, int n_classes, int n_buckets, double *uses, hipStream_t s)
{
    hipLaunchKernelGGL(trellis_uses_kernel, dim3(n_classes, n_buckets), dim3(256), 0, s, row_uses, join_class, rows, n_buckets, uses);
}

size_t trellis_draw_bytes(int64_t rows, int n_utts, int K, int n_draws, size_t (&at)[5])
{
    // pointers | slots | roots | row costs | row log probabilities
    const size_t n = (size_t)n_draws * rows;
    const size_t part[5] = {n * K, n, (size_t)n_draws * n_utts * sizeof(int), n * sizeof(double), n * sizeof(double)};
    size_t total = 0;
    for (int i = 0; i < 5; ++i) { at[i] = total; total += (part[i] + 255) & ~(size_t)255; }
    return total;
}

void launch_trellis_draw(const TrellisView &v, const TrellisCosts &c, const SampleRuleHost &rule, const int *flag, const double *V, const double *u,
                         int n_draws, int64_t all_rows, int all_utts, char *work, int64_t *path, double *cost, double *logp, hipStream_t s)
{
    // the weights carry the temperature already
    SampleRule k;
    const bool greedy = !(rule.temperature > 0.0);
    k.inv_tau = 1.0; k.top_k = greedy ? 1 : rule.top_k; k.top_p = rule.top_p; k.min_p = rule.min_p;
    size_t at[5];
    trellis_draw_bytes(all_rows, all_utts, v.K, n_draws, at);
    unsigned char *pointer = (unsigned char *)work + at[0], *slots = (unsigned char *)work + at[1];
    int *root = (int *)(work + at[2]);
    double *row_cost = (double *)(work + at[3]), *row_logp = (double *)(work + at[4]);
    const int shift = v.rows * ((v.K + 31) / 32) < 8192 ? 3 : 5;
    const dim3 grid((unsigned)v.rows, ((v.K - 1) >> shift) + 1);
    const size_t lds = ((size_t)(v.K | 1) << shift) * sizeof(double);
#define SNK_DRAW(E_) hipLaunchKernelGGL((trellis_pointer_kernel<E_>), grid, dim3(256), lds, s, v, shift, flag, V, k, greedy, u, n_draws, all_rows, all_utts, pointer, root)
    if (v.K <= 64) SNK_DRAW(1);
    else if (v.K <= 128) SNK_DRAW(2);
    else SNK_DRAW(4);
#undef SNK_DRAW
    static size_t attr_set[32] = {0};
    lds_attr_ensure(attr_set, SNK_CHASE_BYTES, [] {
        (void)hipFuncSetAttribute(reinterpret_cast<const void *>(&trellis_chase_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, SNK_CHASE_BYTES); });
    hipLaunchKernelGGL(trellis_chase_kernel, dim3(v.n_utts, n_draws), dim3(512), SNK_CHASE_BYTES, s, v, pointer, root, all_rows, all_utts, slots);
    const dim3 rows((unsigned)((v.rows + 3) / 4), n_draws);
#define SNK_PATH(E_) hipLaunchKernelGGL((trellis_path_kernel<E_>), rows, dim3(256), 0, s, v, c, flag, V, k, root, slots, all_rows, all_utts, path, row_cost, row_logp)
    if (v.K <= 64) SNK_PATH(1);
    else if (v.K <= 128) SNK_PATH(2);
    else SNK_PATH(4);
#undef SNK_PATH
    hipLaunchKernelGGL(trellis_total_kernel, dim3(v.n_utts, n_draws), dim3(256), 0, s, v, root, row_cost, row_logp, all_rows, all_utts, cost, logp);
}

}  // namespace snk
