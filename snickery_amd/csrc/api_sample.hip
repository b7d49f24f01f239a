// C ABI of libsnkhip.so, part 6: draws and probabilities over the candidates of a preselection (include/snk.h snk_sample_rows,
// snk_set_position_bias, snk_sample_paths, snk_path_posterior).
//
// Streams.  snk_sample_rows_dev puts its kernels straight on the caller's stream; rows of more than 8192 scores use the caller's
// workspace or the engine's, which a later call on another stream waits for.  The _dev trellis calls too run on the caller's stream: an
// event behind each makes the next one, on whatever stream, and every call that changes what they read (join frames, weights, bias)
// wait for its use of the workspaces.  (On the engine's stream, with an event either way, a call took 30 us more of the host's time.)
#include "snk_engine.h"

// the caller's device again when a _dev call returns
struct DeviceGuard {
    int before = -1;
    ~DeviceGuard() { if (before >= 0) (void)hipSetDevice(before); }
    int enter(int device)
    {
        int now = 0;
        HIPCHK(hipGetDevice(&now));
        if (now != device) { HIPCHK(hipSetDevice(device)); before = now; }
        return 0;
    }
};

static const size_t kScoreBytes[4] = {8, 4, 2, 2};

static int check_rule(const char *who, double temperature, int64_t top_k, double top_p, double min_p)
{
    if (!(temperature >= 0.0) || !(temperature - temperature == 0.0)) return fail("%s: temperature %g is not a finite number >= 0", who, temperature);
    if (top_k < 0) return fail("%s: top_k %lld < 0 (0: off)", who, (long long)top_k);
    if (!(top_p > 0.0 && top_p <= 1.0)) return fail("%s: top_p %g outside (0, 1]", who, top_p);
    if (!(min_p >= 0.0 && min_p <= 1.0)) return fail("%s: min_p %g outside [0, 1]", who, min_p);
    return 0;
}

static int check_randoms(const char *who, const double *u, int64_t n)
{
    for (int64_t i = 0; i < n; ++i)
        if (!(u[i] >= 0.0 && u[i] < 1.0)) return fail("%s: random number %lld is %g, outside [0, 1)", who, (long long)i, u[i]);
    return 0;
}

static int check_rows(const char *who, int dtype, int64_t R, int64_t V, int64_t stride, int n_draws)
{
    if (dtype < 0 || dtype > 3) return fail("%s: unknown score type %d", who, dtype);
    if (R < 0 || R > 0x7fffffff) return fail("%s: %lld rows", who, (long long)R);
    if (V < 1 || V > sample_rows_max()) return fail("%s: rows of %lld scores (1 .. %lld)", who, (long long)V, (long long)sample_rows_max());
    if (stride < V && R > 1) return fail("%s: row stride %lld < %lld scores", who, (long long)stride, (long long)V);
    if (n_draws < 1) return fail("%s: %d draws per row", who, n_draws);
    return 0;
}

// the row workspace for a call on stream `s`, behind the stream that used it last; nullptr: none needed, or `s` is being captured (a
// graph would share it with every later call)
static int rows_workspace(snk_engine *h, const char *who, int64_t R, int64_t V, hipStream_t s, char **work)
{
    *work = nullptr;
    const size_t bytes = sample_rows_work(sample_rows_together(R, V), V);
    if (!bytes) return 0;
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(s, &st) != hipSuccess) { (void)hipGetLastError(); return fail("%s: another stream's capture forbids work on this one", who); }
    if (st != hipStreamCaptureStatusNone) return 0;
    CHK(h->sr_work.ensure(bytes));
    if (!h->sr_done) HIPCHK(hipEventCreateWithFlags(&h->sr_done, hipEventDisableTiming));
    if (h->sr_used) HIPCHK(hipStreamWaitEvent(s, h->sr_done, 0));
    *work = h->sr_work.as<char>();
    return 0;
}
static int rows_workspace_used(snk_engine *h, hipStream_t s)
{
    HIPCHK(hipEventRecord(h->sr_done, s));
    h->sr_used = true;
    return 0;
}

int snk_sample_rows(snk_handle h, const void *scores, int dtype, int64_t R, int64_t V, int64_t row_stride, const double *u, int n_draws,
                    double temperature, int64_t top_k, double top_p, double min_p, const double *row_rules, int64_t *index_out,
                    double *logp_out)
{
    const char *who = "snk_sample_rows";
    if (!h) return fail("null handle");
    CHK(no_batch_in_flight(h, who));
    CHK(check_rows(who, dtype, R, V, row_stride, n_draws));
    if (R == 0) return 0;
    if (!scores || !u || !index_out) return fail("%s: null argument", who);
    if (row_rules) {
        for (int64_t r = 0; r < R; ++r) {
            const double *q = row_rules + 4 * r;
            if (!(q[1] >= 0.0 && q[1] < 9.0e15) || q[1] != floor(q[1])) return fail("%s: top_k %g of row %lld is not a whole number >= 0", who, q[1], (long long)r);
            CHK(check_rule(who, q[0], (int64_t)q[1], q[2], q[3]));
        }
    } else CHK(check_rule(who, temperature, top_k, top_p, min_p));
    CHK(check_randoms(who, u, R * n_draws));
    HIPCHK(hipSetDevice(h->device));
    const size_t width = kScoreBytes[dtype], n = (size_t)R * n_draws;
    CHK(h->sr_scores.ensure((size_t)R * V * width));
    CHK(h->sr_u.ensure(n * sizeof(double)));
    CHK(h->sr_index.ensure(n * sizeof(int64_t)));
    CHK(h->sr_logp.ensure(n * sizeof(double)));
    CHK(h2d_rows(h, h->sr_scores.p, (size_t)V * width, scores, (size_t)(R > 1 ? row_stride : V) * width, (size_t)V * width, (size_t)R, h->stream));
    CHK(h2d(h, h->sr_u.p, u, n * sizeof(double), h->stream));
    if (row_rules) {
        CHK(h->sr_rules.ensure((size_t)R * 4 * sizeof(double)));
        CHK(h2d(h, h->sr_rules.p, row_rules, (size_t)R * 4 * sizeof(double), h->stream));
    }
    char *work;
    CHK(rows_workspace(h, who, R, V, h->stream, &work));
    {
        StageTimer t(h, h->stream, TM_SAMPLE_ROWS);
        const SampleRuleHost rule = {temperature, top_k, top_p, min_p};
        launch_sample_rows(h->sr_scores.p, dtype, V, R, V, h->sr_u.as<double>(), n_draws, rule, row_rules ? h->sr_rules.as<double>() : nullptr, work,
                           h->sr_index.as<int64_t>(), logp_out ? h->sr_logp.as<double>() : nullptr, h->stream);
    }
    HIPCHK(hipGetLastError());
    if (work) CHK(rows_workspace_used(h, h->stream));
    D2HPart parts[2] = {{index_out, h->sr_index.p, n * sizeof(int64_t)}, {logp_out, h->sr_logp.p, logp_out ? n * sizeof(double) : 0}};
    CHK(staged_d2h(h, h->stream, parts, 2));
    collect_timers(h);
    return 0;
}

int snk_sample_rows_dev(snk_handle h, const void *scores_dev, int dtype, int64_t R, int64_t V, int64_t row_stride, const double *u_dev,
                        int n_draws, double temperature, int64_t top_k, double top_p, double min_p, const double *row_rules_dev,
                        int64_t *index_dev_out, double *logp_dev_out, void *workspace, size_t workspace_bytes, void *stream)
{
    const char *who = "snk_sample_rows_dev";
    if (!h) return fail("null handle");
    CHK(check_rows(who, dtype, R, V, row_stride, n_draws));
    if (R == 0) return 0;
    if (!scores_dev || !u_dev || !index_dev_out) return fail("%s: null argument", who);
    if (!row_rules_dev) CHK(check_rule(who, temperature, top_k, top_p, min_p));
    const size_t need = snk_sample_rows_workspace(R, V);
    if (workspace && ((uintptr_t)workspace & 15)) return fail("%s: the workspace is not aligned to 16 bytes", who);
    if (workspace && workspace_bytes < need) return fail("%s: a workspace of %zu bytes, %zu needed", who, workspace_bytes, need);
    DeviceGuard device;
    CHK(device.enter(h->device));
    const SampleRuleHost rule = {temperature, top_k, top_p, min_p};
    char *work = need ? (char *)workspace : nullptr;
    const bool own = !work;
    if (own) CHK(rows_workspace(h, who, R, V, (hipStream_t)stream, &work));
    launch_sample_rows(scores_dev, dtype, row_stride, R, V, u_dev, n_draws, rule, row_rules_dev, work, index_dev_out, logp_dev_out, (hipStream_t)stream);
    HIPCHK(hipGetLastError());
    if (own && work) CHK(rows_workspace_used(h, (hipStream_t)stream));
    return 0;
}

size_t snk_sample_rows_workspace(int64_t R, int64_t V)
{
    if (R < 1 || V < 1 || V > sample_rows_max()) return 0;
    return sample_rows_work(sample_rows_together(R, V), V);
}

int snk_set_position_bias(snk_handle h, const double *bias, int n_classes, int n_buckets, const int64_t *edges)
{
    const char *who = "snk_set_position_bias";
    if (!h) return fail("null handle");
    CHK(no_batch_in_flight(h, who));
    if (n_classes == 0) { h->pb_classes = 0; h->pb_buckets = 0; return 0; }
    if (n_classes < 0 || n_classes > 65535) return fail("%s: %d classes (0 .. 65535)", who, n_classes);
    if (n_buckets < 1 || n_buckets > 64) return fail("%s: %d buckets (1 .. 64)", who, n_buckets);
    if (!bias || (n_buckets > 1 && !edges)) return fail("%s: null argument", who);
    for (int i = 1; i < n_buckets - 1; ++i)
        if (edges[i] <= edges[i - 1]) return fail("%s: edges have to ascend (edge %d is %lld after %lld)", who, i, (long long)edges[i], (long long)edges[i - 1]);
    const int64_t n = (int64_t)n_classes * n_buckets;
    for (int64_t i = 0; i < n; ++i)
        if (!(bias[i] > -INFINITY)) return fail("%s: bias %lld is %g (finite, or +inf to forbid)", who, (long long)i, bias[i]);
    HIPCHK(hipSetDevice(h->device));
    CHK(trellis_settled(h));
    h->pb_classes = 0;
    CHK(h->pb_bias.ensure((size_t)n * sizeof(double)));
    CHK(h->pb_edges.ensure(64 * sizeof(int)));
    CHK(h2d_sync(h, h->pb_bias.p, bias, (size_t)n * sizeof(double)));
    // unit ids have 31 bits: distances and edges fit 32, edges beyond them are never / always reached
    int e32[64] = {0};
    for (int i = 0; i < n_buckets - 1; ++i) e32[i] = (int)std::min<int64_t>(std::max<int64_t>(edges[i], -0x7fffffff - 1LL), 0x7fffffff);
    CHK(h2d_sync(h, h->pb_edges.p, e32, sizeof(e32)));
    h->pb_min = 0.0;
    for (int64_t i = 0; i < n; ++i) h->pb_min = std::min(h->pb_min, bias[i]);
    h->pb_classes = n_classes;
    h->pb_buckets = n_buckets;
    return 0;
}

// ---- the trellis ------------------------------------------------------------------------------------------------------------------
// a launch holds fewer than 2^32 threads, 256 a row; a group of utterances holds as many rows at most
static const int64_t kTrellisMostRows = (int64_t)1 << 23;

static int check_trellis(const char *who, snk_engine *h, const void *cand, const void *tdist, const int64_t *row_offsets, int n_utts, int K)
{
    CHK(check_ready(h, false, true));
    CHK(no_batch_in_flight(h, who));
    if (!cand || !tdist || !row_offsets || n_utts < 1) return fail("%s: null/empty argument", who);
    if (K < 1 || K > 208) return fail("%s: n_candidates=%d outside 1..208", who, K);
    if (row_offsets[0] != 0) return fail("%s: row_offsets[0] must be 0 (got %lld)", who, (long long)row_offsets[0]);
    for (int v = 0; v < n_utts; ++v)
        if (row_offsets[v + 1] <= row_offsets[v]) return fail("%s: utterance %d has no rows", who, v);
        else if (row_offsets[v + 1] - row_offsets[v] > kTrellisMostRows)
            return fail("%s: utterance %d has %lld rows (at most %lld)", who, v, (long long)(row_offsets[v + 1] - row_offsets[v]), (long long)kTrellisMostRows);
    if (row_offsets[n_utts] > 0x7fffffff) return fail("%s: %lld rows", who, (long long)row_offsets[n_utts]);
    return 0;
}

// Costs of the rows of as many utterances as fit the workspace, then `use` on them; group after group on the engine's stream.
// 4 GB hold 53 000 rows of 100 candidates: larger groups would not fill the chip better, smaller ones would (a sentence alone
// keeps a handful of compute units busy in the recursions).  An utterance that is longer than that is a group by itself.
// (Launches over utterances times the pieces of the longest one: their product is bounded for the sake of short utterances beside a
// very long one, which would otherwise meet mostly empty workgroups, and more of them than a launch holds.)
static const size_t kTrellisGroupBytes = (size_t)4 << 30;
static const int64_t kTrellisGroupUtts = 32768, kTrellisGroupPieces = 262144;

static int trellis_group_end(const int64_t *off, int n_utts, int v0, size_t row_bytes)
{
    int64_t pieces = trellis_most_pieces(off + v0, 1);
    int v1 = v0 + 1;
    for (; v1 < n_utts && v1 - v0 < kTrellisGroupUtts; ++v1) {
        const int64_t rows = off[v1 + 1] - off[v0];
        if ((size_t)rows * row_bytes > kTrellisGroupBytes || rows > kTrellisMostRows) break;
        pieces = std::max<int64_t>(pieces, trellis_most_pieces(off + v1, 1));
        if (pieces * (v1 + 1 - v0) > kTrellisGroupPieces) break;
    }
    return v1;
}

struct TrellisCall {
    const char *who; bool timed;                    // stage timers (calls that wait for their results)
    const int64_t *cand; const double *tdist; const int64_t *row_offsets; const int32_t *join_class;
    int n_utts, K;
    double temperature;
    hipStream_t stream;
};

// `use` gets the group's view (cells not made yet), the costs' parts
template <typename Use>
static int trellis_groups(snk_engine *h, const TrellisCall &q, Use use)
{
    const int64_t rows = q.row_offsets[q.n_utts];
    const int Kp = roundup(q.K, 8);
    const size_t row_bytes = (size_t)q.K * Kp * sizeof(double);
    CHK(h->tr_off.ensure((size_t)(q.n_utts + 1) * sizeof(int64_t)));
    CHK(h->tr_V.ensure((size_t)rows * Kp * sizeof(double)));
    CHK(h->tr_local.ensure((size_t)rows * Kp * sizeof(double)));
    CHK(h->tr_least.ensure((size_t)rows * sizeof(double)));
    CHK(h->tr_flag.ensure((size_t)q.n_utts * sizeof(int)));
    // temperature 0: every utterance goes through the launches that keep the largest term
    launch_trellis_offsets(q.row_offsets, q.n_utts, q.temperature > 0.0 ? 0 : 1, h->tr_off.as<int64_t>(), h->tr_flag.as<int>(), q.stream);
    TrellisCosts c;
    c.JC = h->JC_unw.as<float>(); c.Jp = h->Jp; c.Dj = h->Dj; c.wj = h->wj.as<double>();
    c.join_class = q.join_class; c.bias = h->pb_bias.as<double>(); c.edges = h->pb_edges.as<int>();
    c.n_classes = h->pb_classes; c.n_buckets = h->pb_buckets;
    c.bias_min = h->pb_classes > 0 ? h->pb_min : 0.0;
    for (int v0 = 0; v0 < q.n_utts;) {
        const int v1 = trellis_group_end(q.row_offsets, q.n_utts, v0, row_bytes);
        TrellisView v;
        v.cand = q.cand; v.tdist = q.tdist; v.off = h->tr_off.as<int64_t>();
        v.first = v0; v.n_utts = v1 - v0; v.K = q.K; v.Kp = Kp;
        v.c0 = q.row_offsets[v0]; v.rows = q.row_offsets[v1] - q.row_offsets[v0];
        v.n_units = h->Njc - 1;
        v.inv_tau = q.temperature > 0.0 ? std::min(1.0 / q.temperature, 1e250) : 1.0;      // (0 times it is 0, costs times it keep their order)
        v.pieces = trellis_most_pieces(q.row_offsets + v0, v.n_utts);
        if (v.pieces > 1) {
            const size_t n = trellis_piece_places(v);
            CHK(h->tr_M.ensure(n * row_bytes));
            CHK(h->tr_exps.ensure(n * q.K * sizeof(int)));
            CHK(h->tr_ends_v.ensure(n * Kp * sizeof(double)));
            CHK(h->tr_ends_w.ensure(n * Kp * sizeof(double)));
            CHK(h->tr_scaled.ensure((size_t)q.n_utts * sizeof(int64_t)));
        }
        CHK(h->tr_C.ensure((size_t)v.rows * row_bytes));
        v.C = h->tr_C.as<double>();
        CHK(use(v, c));
        v0 = v1;
    }
    HIPCHK(hipGetLastError());
    return 0;
}

static int sample_paths_device(snk_engine *h, const TrellisCall &q, const double *u, int n_draws, const SampleRuleHost &rule, int64_t *path,
                               double *cost, double *logp)
{
    const int64_t rows = q.row_offsets[q.n_utts];
    size_t at[5];
    CHK(h->tr_draw.ensure(trellis_draw_bytes(rows, q.n_utts, q.K, n_draws, at)));
    return trellis_groups(h, q, [&](const TrellisView &v, const TrellisCosts &c) -> int {
        const bool sum = q.temperature > 0.0;
        int *flag = h->tr_flag.as<int>();
        double *V = h->tr_V.as<double>(), *X = h->tr_C.as<double>();
        if (sum) {
            {
                StageTimer t(h, q.stream, q.timed ? TM_JOIN : -1);
                launch_trellis_local(v, h->tr_local.as<double>(), h->tr_least.as<double>(), flag, q.stream);
                launch_trellis_costs(v, c, false, flag, X, q.stream);
            }
            StageTimer t(h, q.stream, q.timed ? TM_TRELLIS_SUM : -1);
            launch_trellis_ends(v, h->tr_local.as<double>(), false, flag, h->tr_M.as<double>(), h->tr_exps.as<int>(), h->tr_ends_v.as<double>(),
                                h->tr_ends_w.as<double>(), h->tr_scaled.as<int64_t>(), q.stream);
            launch_trellis_forward(v, h->tr_local.as<double>(), h->tr_least.as<double>(), c.bias_min, h->tr_ends_v.as<double>(), h->tr_scaled.as<int64_t>(),
                                   flag, V, nullptr, q.stream);
        }
        {
            StageTimer t(h, q.stream, q.timed ? TM_TRELLIS_SUM : -1);
            launch_trellis_costs(v, c, true, flag, X, q.stream);
            launch_trellis_forward_log(v, sum, flag, V, nullptr, q.stream);
        }
        StageTimer t(h, q.stream, q.timed ? TM_TRELLIS_DRAW : -1);
        launch_trellis_draw(v, c, rule, flag, V, u, n_draws, rows, q.n_utts, h->tr_draw.as<char>(), path, cost, logp, q.stream);
        return 0;
    });
}

static int path_posterior_device(snk_engine *h, const TrellisCall &q, double *logz, double *posterior, double *uses)
{
    const int64_t rows = q.row_offsets[q.n_utts];
    CHK(h->tr_W.ensure((size_t)rows * roundup(q.K, 8) * sizeof(double)));
    if (uses) CHK(h->tr_row_uses.ensure((size_t)rows * h->pb_buckets * sizeof(double)));
    CHK(trellis_groups(h, q, [&](const TrellisView &v, const TrellisCosts &c) -> int {
        int *flag = h->tr_flag.as<int>();
        double *V = h->tr_V.as<double>(), *W = h->tr_W.as<double>(), *X = h->tr_C.as<double>(), *local = h->tr_local.as<double>();
        {
            StageTimer t(h, q.stream, q.timed ? TM_JOIN : -1);
            launch_trellis_local(v, local, h->tr_least.as<double>(), flag, q.stream);
            launch_trellis_costs(v, c, false, flag, X, q.stream);
        }
        {
            StageTimer t(h, q.stream, q.timed ? TM_TRELLIS_SUM : -1);
            launch_trellis_ends(v, local, true, flag, h->tr_M.as<double>(), h->tr_exps.as<int>(), h->tr_ends_v.as<double>(), h->tr_ends_w.as<double>(),
                                h->tr_scaled.as<int64_t>(), q.stream);
            launch_trellis_forward(v, local, h->tr_least.as<double>(), c.bias_min, h->tr_ends_v.as<double>(), h->tr_scaled.as<int64_t>(), flag, V, logz,
                                   q.stream);
            launch_trellis_backward(v, local, h->tr_ends_w.as<double>(), flag, W, q.stream);
            launch_trellis_costs(v, c, true, flag, X, q.stream);
            launch_trellis_forward_log(v, true, flag, V, logz, q.stream);
            launch_trellis_backward_log(v, flag, W, q.stream);
        }
        StageTimer t(h, q.stream, q.timed ? TM_TRELLIS_POST : -1);
        launch_trellis_posterior(v, flag, V, W, h->tr_ends_w.as<double>(), local, logz, h->pb_edges.as<int>(), h->pb_buckets, posterior,
                                 uses ? h->tr_row_uses.as<double>() : nullptr, q.stream);
        return 0;
    }));
    if (uses) launch_trellis_uses(h->tr_row_uses.as<double>(), q.join_class, rows, h->pb_classes, h->pb_buckets, uses, q.stream);
    HIPCHK(hipGetLastError());
    return 0;
}

// host arrays of a trellis call -> the engine's workspaces
static int upload_trellis(snk_engine *h, const int64_t *cand, const double *tdist, int64_t rows, int K, const int32_t *join_class)
{
    StageTimer t(h, h->stream, TM_H2D);
    const size_t n = (size_t)rows * K;
    CHK(h->tr_cand.ensure(n * sizeof(int64_t)));
    CHK(h->tr_tdist.ensure(n * sizeof(double)));
    CHK(h2d(h, h->tr_cand.p, cand, n * sizeof(int64_t), h->stream));
    CHK(h2d(h, h->tr_tdist.p, tdist, n * sizeof(double), h->stream));
    if (join_class) {
        CHK(h->tr_class.ensure((size_t)rows * sizeof(int32_t)));
        CHK(h2d(h, h->tr_class.p, join_class, (size_t)rows * sizeof(int32_t), h->stream));
    }
    return 0;
}

// before a trellis call's work on stream s: behind the workspaces' last use and behind what the engine's stream holds.  Refused while s
// is being captured: a captured call would share the engine's workspaces with every later one
static int trellis_enter(snk_engine *h, const char *who, hipStream_t s)
{
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(s, &st) != hipSuccess || st != hipStreamCaptureStatusNone) {
        (void)hipGetLastError();
        return fail("%s: the stream is being captured (this call uses the engine's workspaces)", who);
    }
    if (!h->tr_in) HIPCHK(hipEventCreateWithFlags(&h->tr_in, hipEventDisableTiming));
    if (!h->tr_done) HIPCHK(hipEventCreateWithFlags(&h->tr_done, hipEventDisableTiming));
    if (h->tr_used) HIPCHK(hipStreamWaitEvent(s, h->tr_done, 0));
    if (s == h->stream) return 0;
    const hipError_t idle = hipStreamQuery(h->stream);
    if (idle == hipSuccess) return 0;
    if (idle != hipErrorNotReady) HIPCHK(idle);
    (void)hipGetLastError();
    HIPCHK(hipEventRecord(h->tr_in, h->stream));
    HIPCHK(hipStreamWaitEvent(s, h->tr_in, 0));
    return 0;
}
// behind it, whether or not all of it was queued
static int trellis_leave(snk_engine *h, hipStream_t s, int result)
{
    const hipError_t e = hipEventRecord(h->tr_done, s);
    if (e == hipSuccess) h->tr_used = true;
    else (void)hipStreamSynchronize(s);
    if (result) return result;
    HIPCHK(e);
    return 0;
}
int trellis_settled(snk_engine *h)
{
    if (h->tr_used) HIPCHK(hipEventSynchronize(h->tr_done));
    h->tr_used = false;
    return 0;
}

// (a temperature whose inverse the costs cannot be multiplied by is that of the cheapest path, ties and all)
static int check_draws(const char *who, const void *u, int n_draws, SampleRuleHost &rule, const void *path, const void *cost)
{
    if (!u || !path || !cost) return fail("%s: null argument", who);
    if (n_draws < 1 || n_draws > 65535) return fail("%s: %d draws (1 .. 65535)", who, n_draws);
    CHK(check_rule(who, rule.temperature, rule.top_k, rule.top_p, rule.min_p));
    if (rule.temperature < 1e-250) rule.temperature = 0.0;
    return 0;
}

int snk_sample_paths(snk_handle h, const int64_t *cand, const double *tdist, const int64_t *row_offsets, int n_utts, int K,
                     const int32_t *join_class, const double *u, int n_draws, double temperature, int64_t top_k, double top_p, double min_p,
                     int64_t *path_out, double *cost_out, double *logp_out)
{
    const char *who = "snk_sample_paths";
    SampleRuleHost rule = {temperature, top_k, top_p, min_p};
    CHK(check_trellis(who, h, cand, tdist, row_offsets, n_utts, K));
    CHK(check_draws(who, u, n_draws, rule, path_out, cost_out));
    const int64_t rows = row_offsets[n_utts];
    CHK(check_randoms(who, u, rows * n_draws));
    HIPCHK(hipSetDevice(h->device));
    const size_t np = (size_t)n_draws * rows * 8, nc = (size_t)n_draws * n_utts * 8;
    CHK(trellis_enter(h, who, h->stream));
    CHK(h->tr_u.ensure(np));
    CHK(h->tr_out.ensure(np + 2 * nc));
    CHK(upload_trellis(h, cand, tdist, rows, K, join_class));
    CHK(h2d(h, h->tr_u.p, u, np, h->stream));
    char *out = h->tr_out.as<char>();
    const TrellisCall q = {who, true, h->tr_cand.as<int64_t>(), h->tr_tdist.as<double>(), row_offsets, join_class ? h->tr_class.as<int32_t>() : nullptr,
                           n_utts, K, rule.temperature, h->stream};
    CHK(sample_paths_device(h, q, h->tr_u.as<double>(), n_draws, rule, (int64_t *)out, (double *)(out + np),
                            logp_out ? (double *)(out + np + nc) : nullptr));
    D2HPart parts[3] = {{path_out, out, np}, {cost_out, out + np, nc}, {logp_out, out + np + nc, logp_out ? nc : 0}};
    CHK(staged_d2h(h, h->stream, parts, 3));
    collect_timers(h);
    return 0;
}

int snk_sample_paths_dev(snk_handle h, const int64_t *cand_dev, const double *tdist_dev, const int64_t *row_offsets, int n_utts, int K,
                         const int32_t *join_class_dev, const double *u_dev, int n_draws, double temperature, int64_t top_k, double top_p,
                         double min_p, int64_t *path_dev_out, double *cost_dev_out, double *logp_dev_out, void *stream)
{
    const char *who = "snk_sample_paths_dev";
    SampleRuleHost rule = {temperature, top_k, top_p, min_p};
    CHK(check_trellis(who, h, cand_dev, tdist_dev, row_offsets, n_utts, K));
    CHK(check_draws(who, u_dev, n_draws, rule, path_dev_out, cost_dev_out));
    DeviceGuard device;
    CHK(device.enter(h->device));
    CHK(trellis_enter(h, who, (hipStream_t)stream));
    const TrellisCall q = {who, false, cand_dev, tdist_dev, row_offsets, join_class_dev, n_utts, K, rule.temperature, (hipStream_t)stream};
    return trellis_leave(h, (hipStream_t)stream, sample_paths_device(h, q, u_dev, n_draws, rule, path_dev_out, cost_dev_out, logp_dev_out));
}

static int check_posterior(const char *who, snk_engine *h, double temperature, const void *logz, const void *posterior, const void *uses)
{
    if (!logz || !posterior) return fail("%s: null argument", who);
    if (!(temperature > 0.0) || !(temperature - temperature == 0.0)) return fail("%s: temperature %g is not a finite number > 0", who, temperature);
    if (uses && h->pb_classes == 0) return fail("%s: no position bias set (snk_set_position_bias)", who);
    return 0;
}

int snk_path_posterior(snk_handle h, const int64_t *cand, const double *tdist, const int64_t *row_offsets, int n_utts, int K,
                       const int32_t *join_class, double temperature, double *logz_out, double *posterior_out, double *uses_out)
{
    const char *who = "snk_path_posterior";
    CHK(check_trellis(who, h, cand, tdist, row_offsets, n_utts, K));
    CHK(check_posterior(who, h, temperature, logz_out, posterior_out, uses_out));
    HIPCHK(hipSetDevice(h->device));
    const int64_t rows = row_offsets[n_utts];
    const size_t nz = (size_t)n_utts * 8, np = (size_t)rows * K * 8, nu = uses_out ? (size_t)h->pb_classes * h->pb_buckets * 8 : 0;
    CHK(trellis_enter(h, who, h->stream));
    CHK(h->tr_out.ensure(nz + np + nu));
    CHK(upload_trellis(h, cand, tdist, rows, K, join_class));
    char *out = h->tr_out.as<char>();
    const TrellisCall q = {who, true, h->tr_cand.as<int64_t>(), h->tr_tdist.as<double>(), row_offsets, join_class ? h->tr_class.as<int32_t>() : nullptr,
                           n_utts, K, temperature, h->stream};
    CHK(path_posterior_device(h, q, (double *)out, (double *)(out + nz), uses_out ? (double *)(out + nz + np) : nullptr));
    D2HPart parts[3] = {{logz_out, out, nz}, {posterior_out, out + nz, np}, {uses_out, out + nz + np, nu}};
    CHK(staged_d2h(h, h->stream, parts, 3));
    collect_timers(h);
    return 0;
}

int snk_path_posterior_dev(snk_handle h, const int64_t *cand_dev, const double *tdist_dev, const int64_t *row_offsets, int n_utts, int K,
                           const int32_t *join_class_dev, double temperature, double *logz_dev_out, double *posterior_dev_out,
                           double *uses_dev_out, void *stream)
{
    const char *who = "snk_path_posterior_dev";
    CHK(check_trellis(who, h, cand_dev, tdist_dev, row_offsets, n_utts, K));
    CHK(check_posterior(who, h, temperature, logz_dev_out, posterior_dev_out, uses_dev_out));
    DeviceGuard device;
    CHK(device.enter(h->device));
    CHK(trellis_enter(h, who, (hipStream_t)stream));
    const TrellisCall q = {who, false, cand_dev, tdist_dev, row_offsets, join_class_dev, n_utts, K, temperature, (hipStream_t)stream};
    return trellis_leave(h, (hipStream_t)stream, path_posterior_device(h, q, logz_dev_out, posterior_dev_out, uses_dev_out));
}
