"""Sampling operators at the ends of their ranges: frames that are not finite, batches of every size, long rows under one peak, tiny
temperatures, ties, autograd and captured calls.  Against oracle/sampling_oracle.py (64 bits)."""
import numpy as np
import pytest

import sampling_oracle as o
from test_gpu_sampling import Voice, check_paths, check_posterior, engine, on_gpu, sum_tolerance      # noqa: F401 (engine: the fixture)

pytestmark = pytest.mark.gpu


# ---- join frames that are not finite ------------------------------------------------------------------------------------------------
@pytest.fixture
def frames_oracle(monkeypatch):
    """The oracle with a join of no finite distance forbidden, whether the distance is infinite or (inf - inf, NaN) no number."""
    plain = o.trellis

    def trellis(*args, **kwargs):
        with np.errstate(invalid='ignore'):
            local, C, B = plain(*args, **kwargs)
        return local, np.where(np.isnan(C), np.inf, C), B
    monkeypatch.setattr(o, 'trellis', trellis)


@pytest.mark.parametrize('K', [20, 100])
@pytest.mark.parametrize('bad', [np.inf, -np.inf, np.nan])
def test_frames_that_are_not_finite_join_nothing(engine, frames_oracle, bad, K):
    """The frame of a row's first usable candidate (what the distances of the row before are taken relative to), of one in the middle, of
    a natural successor, and of an end alone: only joins over these frames are forbidden."""
    v = Voice(engine, Dj=37, n=900)
    v.set_bias(1, 8)
    rng = np.random.RandomState(K)
    cand, dist, offs = v.candidates([9, 4], K, pad=False)
    cand[:] = np.clip(cand, 20, 880)
    cand[2, 0], cand[4, 5], cand[5, 3] = 3, 6, 7                # 7 follows 6: both ends of a natural join are not finite
    cand[7, 2], cand[11, 0] = 11, 14
    v.JC[[3, 7, 12, 14], [0, 5, 36, 8]] = bad                   # starts of 3, 7 and 14, ends of 2, 6, 11 and 13
    engine.upload_join_only(v.JC)
    engine.set_weights(None, v.wj)
    u = rng.rand(2, 13)
    for rule in (dict(), dict(temperature=0.3, top_p=0.9), dict(temperature=0.0), dict(temperature=1e-3)):
        check_paths(v, cand, dist, offs, u, **rule)
    for tau in (1.0, 1e-3):
        check_posterior(v, cand, dist, offs, temperature=tau)
    cand[2, :] = 3                                              # a row whose frames are all bad: no path leads through
    path, cost, logp = check_paths(v, cand, dist, offs, u)
    assert np.all(path[:, :9] == -1) and np.all(path[:, 9:] > 0)
    check_posterior(v, cand, dist, offs)


# ---- a batch's size -------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('Dj', [17, 33, 151, 302])
@pytest.mark.parametrize('K', [90, 100, 130, 200])
def test_results_do_not_depend_on_the_batch_at_any_width(engine, K, Dj):
    """A sentence by itself (tiles of up to 64 candidates, 32 columns at a time) and among others (tiles of up to 112, 16 columns)."""
    v = Voice(engine, Dj=Dj, n=2000)
    v.wj = v.wj / np.sqrt(Dj)
    engine.set_weights(None, v.wj)
    v.set_bias(2, 8)
    cand, dist, offs = v.candidates([30, 26, 1, 150, 180, 2], K)
    rng = np.random.RandomState(0)
    u, cls = rng.rand(2, cand.shape[0]), rng.randint(0, 2, cand.shape[0]).astype(np.int32)
    path, cost, logp = engine.sample_paths(cand, dist, u, row_offsets=offs, join_class=cls, temperature=0.5, top_p=0.9)
    logz, post, _ = engine.path_posterior(cand, dist, row_offsets=offs, join_class=cls, temperature=0.5)
    for i in (0, 1, 2, 5):
        a, b = int(offs[i]), int(offs[i + 1])
        p, c, l = engine.sample_paths(cand[a:b], dist[a:b], u[:, a:b], join_class=cls[a:b], temperature=0.5, top_p=0.9)
        assert np.array_equal(p, path[:, a:b]) and np.array_equal(c[:, 0], cost[:, i]) and np.array_equal(l[:, 0], logp[:, i])
        z, q, _ = engine.path_posterior(cand[a:b], dist[a:b], join_class=cls[a:b], temperature=0.5)
        assert z[0] == logz[i] and np.array_equal(q, post[a:b])


@pytest.mark.parametrize('Dj', [33, 151, 302])
@pytest.mark.parametrize('K', [90, 100, 200])
def test_large_tiles_of_many_columns(engine, K, Dj):
    """Rows enough for the tiles of 96 and 112 candidates, columns enough for several turns of their loop.  The error of a join cost as
    in include/snk.h: (Dj + 4) 2^-43 of it and (Dj + 4) 2^-47 of the largest, once a row and for each sum that it enters."""
    v = Voice(engine, Dj=Dj, n=3000)
    v.wj = v.wj / np.sqrt(Dj)
    engine.set_weights(None, v.wj)
    v.set_bias(1, 8)
    lengths = [7, 200, 5, 190, 9]                               # the short ones are compared, the long ones fill the launch
    cand, dist, offs = v.candidates(lengths, K)
    logz, post, _ = engine.path_posterior(cand, dist, row_offsets=offs, temperature=0.7)
    furthest = np.sqrt((v.wj ** 2 * (v.JC.max(axis=0) - v.JC.min(axis=0)).astype(np.float64) ** 2).sum())
    u = np.random.RandomState(Dj).rand(1, cand.shape[0])
    path, cost, _ = engine.sample_paths(cand, dist, u, row_offsets=offs, temperature=0.7, top_k=30, top_p=0.9)
    for i in (0, 2, 4):
        a, b = int(offs[i]), int(offs[i + 1])
        z, p, _ = o.posterior(cand[a:b], dist[a:b], 0.7, **v.model())
        T = b - a
        tol = sum_tolerance(T, K, abs(z) + 2.0 * T / 0.7) + T * furthest * (Dj + 4.0) * (2.0 ** -43 + 2.0 ** -47) / 0.7
        assert abs(logz[i] - z) <= tol
        assert np.all(np.abs(post[a:b] - p) <= 4.0 * tol)
        want, c, _ = o.sample_path(cand[a:b], dist[a:b], u[0, a:b], 0.7, top_k=30, top_p=0.9, **v.model())
        assert np.array_equal(path[0, a:b], want) and abs(cost[0, i] - c) <= 2.0 ** -52 * 4.0 * T * max(abs(c), 1.0)


# ---- rows under one peak -----------------------------------------------------------------------------------------------------------------
def peak_and_tail(V, depth, dtype='float32'):
    """One score `depth` above V - 1 equal ones, and the tail's weight each: depths in eighths are exact in every type."""
    x = np.full((1, V), -depth, dtype=dtype)
    x[0, 0] = 0.0
    return x, float(np.exp(-np.float64(depth)))


@pytest.mark.parametrize('V,depth,dtype', [(4096, 26.5, 'float64'), (8192, 26.5, 'float32'), (8193, 27.0, 'float64'), (100003, 27.0, 'float32'),
                                           (1 << 20, 30.0, 'float32'), (1 << 20, 30.0, 'float16'), (1 << 24, 27.5, 'float32'), (1 << 24, 33.0, 'float32')])
def test_a_long_tail_under_one_peak_keeps_its_mass(engine, V, depth, dtype):
    """Weights are rounded to multiples of 2^-50 at the coarsest: the mass up to a score is off by at most V 2^-51, its index by that
    over the tail's weight, a log probability by twice that (the drawn score's own, and the mass')."""
    x, w = peak_and_tail(V, depth, dtype)
    mass = 1.0 + (V - 1) * w
    slack = V * 2.0 ** -51
    for part in (0.25, 0.5, 0.9):
        goal = part * (V - 1)                                   # scores of the tail below the drawn one
        u = np.array([[(1.0 + (goal + 0.5) * w) / mass]])
        for got in (engine.sample_rows(x, u), [a.cpu().numpy() for a in engine.sample_rows(on_gpu(x), on_gpu(u))]):
            index, logp = int(got[0][0, 0]), float(got[1][0, 0])
            assert abs(index - 1 - goal) <= 1.0 + (slack + 4.0 * 2.0 ** -53 * mass) / w, (index, goal)
            assert abs(logp - (-depth - np.log(mass))) <= 2.0 * slack + 64.0 * 2.0 ** -53 * (1.0 + depth)
        # a share of the mass that ends inside the tail: nothing behind it is drawn, something next to it is
        share = float(u[0, 0])
        last = 1.0 - 2.0 ** -53
        got = engine.sample_rows(on_gpu(x), on_gpu(np.array([[last]])), top_p=share)
        assert abs(int(got[0][0, 0]) - 1 - goal) <= 2.0 + 2.0 * (slack + 4.0 * 2.0 ** -53 * mass) / w
        assert abs(float(got[1][0, 0]) - (-depth - np.log(1.0 + goal * w))) <= 4.0 * slack + w + 64.0 * 2.0 ** -53 * (1.0 + depth)


def test_a_long_tail_in_a_captured_call_without_a_workspace(engine):
    import torch
    V, depth = 1 << 22, 29.0
    x, w = peak_and_tail(V, depth)
    mass, slack = 1.0 + (V - 1) * w, V * 2.0 ** -51
    goal = 0.7 * (V - 1)
    share = (1.0 + (goal + 0.5) * w) / mass
    gx, gu = on_gpu(x), on_gpu(np.array([[share, 1.0 - 2.0 ** -53, 0.0]]))
    index = torch.full((2, 3), -7, dtype=torch.int64, device='cuda')
    logp = torch.zeros((2, 3), dtype=torch.float64, device='cuda')
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        stream = torch.cuda.current_stream().cuda_stream
        for n, top_p in enumerate((1.0, share)):
            assert engine._lib.snk_sample_rows_dev(engine._h, gx.data_ptr(), 1, 1, V, V, gu.data_ptr(), 3, 1.0, 0, top_p, 0.0, None, index[n].data_ptr(),
                                                   logp[n].data_ptr(), None, 0, stream) == 0
    for _ in range(3):
        index.fill_(-7)
        graph.replay()
        torch.cuda.synchronize()
        got = index.cpu().numpy()
        near = 2.0 + 2.0 * (slack + 4.0 * 2.0 ** -53 * mass) / w
        assert abs(got[0, 0] - 1 - goal) <= near and abs(got[0, 1] - (V - 1)) <= near and got[0, 2] == 0
        assert abs(got[1, 1] - 1 - goal) <= near and got[1, 2] == 0
    # the same calls with a workspace: the same draws
    for n, top_p in enumerate((1.0, share)):
        i, lp = engine.sample_rows(gx, gu, top_p=top_p)
        assert torch.equal(i[0], index[n]) and torch.equal(lp[0], logp[n])


@pytest.mark.parametrize('V', [2048, 4096, 8191, 8192, 8193, 65536, 1 << 20, 1 << 24])
@pytest.mark.parametrize('dtype', ['float32', 'bfloat16'])
def test_rows_of_equal_scores(engine, V, dtype):
    """Every weight is 1, the largest mass that a row can have: a draw is floor(u V), exactly (V and u are whole multiples of powers of
    two whose product float64 holds)."""
    import torch
    x = torch.full((2, V), 0.25, dtype=getattr(torch, dtype), device='cuda')
    u = np.array([[0.0, 0.125, 0.5, 1.0 - 2.0 ** -26], [0.75, 0.875, 1.0 - 2.0 ** -25, 2.0 ** -26]])
    exact = (np.floor(u * V)).astype(np.int64)
    i, lp = engine.sample_rows(x, on_gpu(u))
    assert np.array_equal(i.cpu().numpy(), exact)
    assert np.all(np.abs(lp.cpu().numpy() + np.log(V)) <= 8.0 * 2.0 ** -53 * (1.0 + np.log(V)))
    for rule, n in ((dict(top_k=V // 2), V // 2), (dict(top_p=0.5), (V + 1) // 2), (dict(top_k=V // 2, top_p=0.5), (V // 2 + 1) // 2),
                    (dict(top_k=V - 1, min_p=1.0), V - 1)):
        i, lp = engine.sample_rows(x, on_gpu(u), **rule)
        assert np.array_equal(i.cpu().numpy(), np.floor(u * n).astype(np.int64)), rule
        assert np.all(np.abs(lp.cpu().numpy() + np.log(n)) <= 8.0 * 2.0 ** -53 * (1.0 + np.log(n)))


@pytest.mark.parametrize('V', [8192, 20000, 300000])
def test_rows_of_scores_within_a_hair(engine, V):
    """Weights of almost 1 that all differ, the largest masses of a list and of a bin; equal to the rows cut shorter by top_k."""
    rng = np.random.RandomState(V)
    x = -(rng.permutation(V) + 1.0)[None, :] * 2.0 ** -40
    order = np.argsort(-x[0], kind='stable')
    u = rng.rand(1, 5)
    for k in (1, 1000, V // 2, V - 1):
        kept = np.sort(order[:k])
        w = np.exp(x[0, kept] - x[0].max())
        c = np.cumsum(w.astype(np.longdouble))
        want = kept[np.searchsorted(c, (u[0] * c[-1]).astype(np.longdouble), side='right')]
        i, _ = engine.sample_rows(on_gpu(x), on_gpu(u), top_k=k)
        assert np.array_equal(i.cpu().numpy()[0], want)
        # the same prefix by its mass: between the k-th score's and the one's before
        mass = np.cumsum(np.exp(x[0, order] - x[0].max()).astype(np.longdouble))
        share = float((mass[k - 1] - 0.5) / mass[-1])
        i, _ = engine.sample_rows(on_gpu(x), on_gpu(u), top_p=share)
        assert np.array_equal(i.cpu().numpy()[0], want)


def test_a_row_of_the_most_bins_in_a_graph(engine):
    """Histograms of more than 64 KB, recorded with the graph's own workspace."""
    import torch
    g = torch.Generator(device='cuda').manual_seed(3)
    x = torch.randn((2, 600001), device='cuda', generator=g)
    u = torch.rand((2, 3), device='cuda', dtype=torch.float64, generator=g)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = engine.sample_rows(x, u, top_p=0.97)
    for n in range(3):
        x.copy_(torch.randn((2, 600001), device='cuda', generator=g))
        graph.replay()
        want = engine.sample_rows(x, u, top_p=0.97)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---- temperature zero ------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('tau', [9.9e-251, 1e-300, 5e-324])
def test_a_temperature_that_counts_as_zero_breaks_ties_like_it(engine, tau):
    v = Voice(engine)
    cand, dist, offs = v.candidates([12, 5], 9, pad=False)
    cand[:, 5], dist[:, 5] = cand[:, 2], dist[:, 2]             # the same unit twice in every row, as cheap
    cand[:, 7], dist[:, 7] = cand[:, 2], dist[:, 2]
    dist[:, 2] -= 3.0
    dist[:, 5], dist[:, 7] = dist[:, 2], dist[:, 2]
    u = np.random.RandomState(0).rand(4, 17)
    want = engine.sample_paths(cand, dist, u, row_offsets=offs, temperature=0.0)
    for got in (engine.sample_paths(cand, dist, u, row_offsets=offs, temperature=tau),
                [a.cpu().numpy() for a in engine.sample_paths(on_gpu(cand), on_gpu(dist), on_gpu(u), row_offsets=offs, temperature=tau)]):
        assert all(np.array_equal(a, b) for a, b in zip(got, want)) and not got[2].any()


# ---- tiny temperatures ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('tau', [1e-6, 1e-10, 1e-13, 1e-16, 1e-30])
def test_posteriors_of_tiny_temperatures_are_probabilities(engine, tau):
    """Path costs of up to 1e32 temperatures: what the exponents round away is more than 1, but a row's probabilities sum to 1, and where
    the cheapest path is alone by more than all roundings they are its."""
    v = Voice(engine)
    v.set_bias(1, 8)
    cand, dist, offs = v.candidates([30, 1, 12], 20)
    cand[:, 10:] = np.where(cand[:, 10:] > 0, cand[:, 10:], 5)
    path, cost, _ = engine.sample_paths(cand, dist, np.zeros((1, 43)), row_offsets=offs, temperature=0.0)
    logz, post, uses = engine.path_posterior(cand, dist, row_offsets=offs, temperature=tau)
    # a row's sum: K quotients and their sum, rounded K + 2 times
    assert np.all(np.abs(post.sum(axis=1) - 1.0) <= 32.0 * 2.0 ** -53 * 20)
    want = (cand == path[0][:, None]) & (post > 0.0)
    assert np.array_equal(cand[np.arange(43), post.argmax(axis=1)], path[0])
    assert np.all(np.abs((post * want).sum(axis=1) - 1.0) <= 1e-12)
    steps = np.zeros(uses.shape)
    for a, b in zip(offs[:-1], offs[1:]):
        for t in range(a, b - 1):
            steps[0, int(np.searchsorted(v.edges, path[0, t + 1] - path[0, t], side='right'))] += 1.0
    assert np.all(np.abs(uses - steps) <= 1e-9)
    # six roundings a row, of values of up to the whole sum: 1 / tau, the target cost and the join cost times it, their sum, the row's relative
    # weight and what it is relative to
    assert np.all(np.abs(logz + cost[0] / tau) <= 6.0 * np.diff(offs) * 2.0 ** -53 * cost[0] / tau + 5.0)


@pytest.mark.parametrize('scale,tau,bias', [(1e300, 1e-10, 0.0), (-1e300, 1e-10, 0.0), (-1e308, 1e-300, 0.0), (1.0, 0.5, -1e308), (1.0, 1e-10, 1e308), (1.0, 1e-10, -1e308)])
def test_posteriors_of_costs_that_overflow_are_probabilities(engine, scale, tau, bias):
    v = Voice(engine)
    cand, dist, offs = v.candidates([30, 5], 20, pad=False)
    cand = np.clip(cand, 1, v.n - 2)
    rng = np.random.RandomState(1)
    d = dist * (scale * np.where(rng.rand(35, 20) < 0.3, -0.4, 0.4))
    engine.set_position_bias(np.array([[0.0, bias]]), [1])
    logz, post, uses = engine.path_posterior(cand, d, row_offsets=offs, temperature=tau)
    assert np.all(np.abs(post.sum(axis=1) - 1.0) <= 32.0 * 2.0 ** -53 * 20) and not np.isnan(logz).any()
    assert abs(uses.sum() - 33.0) <= 33.0 * 20 * 20 * 2.0 ** -51 + 1e-13      # a join between each two rows; K K cells a row, rounded to 2^-50


# ---- autograd -----------------------------------------------------------------------------------------------------------------------------
def test_tensors_that_ask_for_a_gradient_are_refused(engine):
    import torch
    from snickery_amd import SnkError
    v = Voice(engine)
    cand, dist, offs = v.candidates([5], 6, pad=False)
    rng = np.random.RandomState(0)
    c, d, u, x = on_gpu(cand), on_gpu(dist).requires_grad_(), on_gpu(rng.rand(2, 5)), on_gpu(rng.randn(5, 6)).requires_grad_()
    for call in (lambda d, x: engine.path_posterior(c, d), lambda d, x: engine.sample_paths(c, d, u), lambda d, x: engine.sample_rows(x, u.t().contiguous())):
        with pytest.raises(SnkError, match='gradient'):
            call(d, x)
        with pytest.raises(SnkError, match='gradient'):
            call(2.0 * d, 2.0 * x)
        want = call(d.detach(), x.detach())
        with torch.no_grad():
            got = call(d, x)
        assert all(b is None or torch.equal(a, b) for a, b in zip(got, want))
    # the gradient that a program puts together itself
    logz, post, _ = engine.path_posterior(c, d.detach(), temperature=0.5)
    h = 2.0 ** -14
    e = torch.zeros_like(post)
    e[2, 3] = h
    slope = (engine.path_posterior(c, d.detach() + e, temperature=0.5)[0] - engine.path_posterior(c, d.detach() - e, temperature=0.5)[0]) / (2.0 * h)
    assert abs(float(slope) + float(post[2, 3]) / 0.5) <= h * h / 6.0 / 0.5 ** 3 + 2.0 ** -40 / h


# ---- rules of rows --------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('V', [100, 3000, 20000])
def test_a_rule_per_row_in_a_graph(engine, V):
    """Some rules a tensor, the others numbers, recorded once and replayed with other rules."""
    import torch
    rng = np.random.RandomState(V)
    R = 6
    x, u = rng.randn(R, V).astype(np.float32), rng.rand(R, 2)
    gx, gu = on_gpu(x), on_gpu(u)
    tau, k = on_gpu(np.full(R, 1.0)), on_gpu(np.full(R, 3))
    one = torch.full((), 0.9, dtype=torch.float64, device='cuda')             # a single number on the GPU: for every row
    engine.sample_rows(gx, gu, temperature=tau, top_k=k, top_p=0.9)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = engine.sample_rows(gx, gu, temperature=tau, top_k=0, top_p=0.9, min_p=1e-3)
        b = engine.sample_rows(gx, gu, temperature=0.7, top_k=k, top_p=one)
    for n in range(3):
        t, m = 0.2 + rng.rand(R), rng.randint(1, 50, R)
        tau.copy_(on_gpu(t)); k.copy_(on_gpu(m))
        graph.replay()
        torch.cuda.synchronize()
        for got, rule in ((a, dict(temperature=t, top_p=0.9, min_p=1e-3)), (b, dict(temperature=0.7, top_k=m, top_p=0.9))):
            want, lp = o.sample_rows(x, u, **rule)
            assert np.array_equal(got[0].cpu().numpy(), want)
            eager = engine.sample_rows(gx, gu, **rule)                        # numpy rules, copied
            assert torch.equal(eager[0], got[0]) and torch.equal(eager[1], got[1])


def test_rules_of_rows_refused(engine):
    import torch
    from snickery_amd import SnkError
    x, u = torch.zeros((4, 10), device='cuda'), torch.zeros((4,), dtype=torch.float64, device='cuda')
    for bad in (torch.ones(3, device='cuda'), torch.ones((4, 1), device='cuda'), np.ones(5), np.ones((1, 4)), [1.0, 2.0]):
        with pytest.raises(SnkError, match='entries'):
            engine.sample_rows(x, u, temperature=bad)
    with pytest.raises(SnkError, match='gradient'):
        engine.sample_rows(x, u, temperature=torch.ones(4, device='cuda', requires_grad=True))
    assert engine.sample_rows(x, u, temperature=[1.0, 0.5, 2.0, 0.0])[0].tolist() == [0, 0, 0, 0]


# ---- 80 bits ---------------------------------------------------------------------------------------------------------------------------------
def posterior_in_80_bits(v, cand, dist, tau):
    """log Z and posteriors of one utterance in numpy's long double, in logarithms."""
    L = np.longdouble
    W, low = v.JC.astype(L) * v.wj.astype(L), np.clip(cand, 1, v.n - 2)
    usable = (cand >= 1) & (cand < v.n - 1)
    local = np.where(usable, -dist.astype(L) / L(tau), -np.inf)
    C = []
    for t in range(len(cand) - 1):
        c = np.sqrt(((W[low[t] + 1][:, None, :] - W[low[t + 1]][None, :, :]) ** 2).sum(axis=2))
        c = c + v.bias[0][o.buckets(cand[t], cand[t + 1], v.edges)].astype(L)
        c[~usable[t]], c[:, ~usable[t + 1]] = np.inf, np.inf
        C.append(-c / L(tau))

    def lse(x, axis):
        m = x.max(axis=axis, keepdims=True)
        m = np.where(np.isfinite(m), m, L(0))
        with np.errstate(divide='ignore'):
            return (m + np.log(np.exp(x - m).sum(axis=axis, keepdims=True))).squeeze(axis)
    alpha, beta = [local[0]], [np.zeros(cand.shape[1], L)]
    for t in range(len(C)):
        alpha.append(local[t + 1] + lse(alpha[-1][:, None] + C[t], 0))
    for t in range(len(C) - 1, -1, -1):
        beta.append(lse(C[t] + (local[t + 1] + beta[-1])[None, :], 1))
    z = lse(alpha[-1], 0)
    return z, np.exp(np.array(alpha) + np.array(beta[::-1]) - z)


@pytest.mark.parametrize('T,K,Dj', [(335, 50, 302), (60, 100, 151)])
def test_posteriors_against_80_bits(engine, T, K, Dj):
    """The error that is left when the comparison has none of its own (pytest -s prints it)."""
    v = Voice(engine, Dj=Dj, n=3000)
    v.wj = v.wj / np.sqrt(Dj)
    engine.set_weights(None, v.wj)
    v.set_bias(1, 8)
    cand, dist, _ = v.candidates([T], K)
    z, p = posterior_in_80_bits(v, cand, dist, 0.5)
    logz, post, _ = engine.path_posterior(cand, dist, temperature=0.5)
    furthest = np.sqrt((v.wj ** 2 * (v.JC.max(axis=0) - v.JC.min(axis=0)).astype(np.float64) ** 2).sum())
    # the join costs as in include/snk.h, once a row; a row's products, sums and scalings: K + 16 roundings
    tol = T * (furthest * (Dj + 4.0) * (2.0 ** -43 + 2.0 ** -47) / 0.5 + (K + 16.0) * 2.0 ** -53)
    err = np.abs(post - p).max()
    print('\n%d rows of %d, %d columns: posteriors within %.1e of 80 bits (bound %.1e), log Z %.1f within %.1e' % (T, K, Dj, err, 4.0 * tol, z, abs(logz[0] - z)))
    assert err <= 4.0 * tol and abs(logz[0] - z) <= tol + 2.0 ** -52 * abs(float(z))
