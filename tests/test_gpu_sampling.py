"""Draws from rows of scores and from candidate trellises, path posteriors and the position bias on the GPU, against
oracle/sampling_oracle.py (64 bits)."""
import itertools

import numpy as np
import pytest

import sampling_oracle as o

pytestmark = pytest.mark.gpu

RULES = [dict(), dict(temperature=0.3), dict(top_k=1), dict(top_k=7), dict(top_p=0.3), dict(top_p=0.95), dict(min_p=0.1),
         dict(temperature=1.7, top_k=40, top_p=0.9, min_p=0.02), dict(temperature=0.0), dict(temperature=0.0, top_k=5, top_p=0.5)]


@pytest.fixture(scope='module')
def engine():
    import snickery_amd
    e = snickery_amd.HipSearchEngine(0)
    yield e
    e.close()


def logp_tolerance(V, e=0.0):
    """Of a log probability.  The kept mass is V weights rounded to multiples of 2^-s, s = min(51, 62 - ceil(log2 V)): V 2^-(s+1)
    over a mass of 1 at least, doubled for the drawn weight's own sum.  Exponent and logarithms: a few units of 2^-53 relative to the
    values, the oracle's sum V 2^-53 relative."""
    s = min(51, 62 - int(np.ceil(np.log2(max(V, 1)))))
    return V * 2.0 ** -s + (V + 16.0) * 2.0 ** -53 + 16.0 * 2.0 ** -53 * (40.0 + e)


def scores_of(rng, R, V, dtype):
    x = 2.0 * rng.randn(R, V)
    if dtype == 'bfloat16':                      # exactly representable in 8 bits
        import torch
        return torch.from_numpy(x).to(torch.bfloat16)
    return x.astype(dtype)


def as_f64(x):
    return x.double().numpy() if hasattr(x, 'double') else np.asarray(x, dtype=np.float64)


def on_gpu(x):
    import torch
    return (x if torch.is_tensor(x) else torch.from_numpy(np.ascontiguousarray(x))).cuda()


def check_rows(engine, x, u, **rule):
    V = x.shape[1]
    want, want_lp = o.sample_rows(as_f64(x), u.reshape(u.shape[0], -1), **rule)
    results = []
    if isinstance(x, np.ndarray):
        results.append(engine.sample_rows(x, u, **rule))
    i, lp = engine.sample_rows(on_gpu(x), on_gpu(u), **rule)
    results.append((i.cpu().numpy(), lp.cpu().numpy()))
    for i, lp in results:
        assert i.shape == u.shape and lp.shape == u.shape and i.dtype == np.int64 and lp.dtype == np.float64
        assert np.array_equal(i.reshape(want.shape), want)
        lp = lp.reshape(want.shape)
        alive = want >= 0
        assert np.all(lp[~alive] == -np.inf)
        assert np.all(np.abs(lp - want_lp)[alive] <= logp_tolerance(V, np.abs(want_lp[alive]).max() if alive.any() else 0.0))


@pytest.mark.parametrize('V', [1, 2, 30, 63, 64, 65, 100, 128, 129, 208, 256, 257, 512, 600, 1000, 1024, 1025, 1500, 4096, 4097])
@pytest.mark.parametrize('dtype', ['float64', 'float32', 'float16', 'bfloat16'])
def test_rows_sizes_and_rules(engine, V, dtype):
    rng = np.random.RandomState(V)
    x = scores_of(rng, 5, V, dtype)
    for n, rule in enumerate(RULES):
        check_rows(engine, x, rng.rand(5, 1 + n % 3), **rule)


@pytest.mark.parametrize('V,dtype', [(20000, 'float32'), (40001, 'bfloat16'), (33333, 'float64'), (70001, 'float32'), (131072, 'float16')])
def test_rows_long(engine, V, dtype):
    rng = np.random.RandomState(V)
    x = scores_of(rng, 2, V, dtype)
    for rule in (dict(), dict(top_k=50), dict(top_p=0.9), dict(temperature=0.8, top_k=3000 + V % 7, top_p=0.7, min_p=1e-3)):
        check_rows(engine, x, rng.rand(2, 2), **rule)


@pytest.mark.parametrize('V', [1100, 9000, 20000, 70000])
def test_rows_whose_scores_crowd(engine, V):
    """Rows that leave a boundary bin full: equal scores by the thousand, different ones within a hair of each other, a few far ones."""
    rng = np.random.RandomState(V)
    crowd = 1.0 + 1e-9 * rng.rand(V)
    spike = np.where(np.arange(V) % 1000 == 7, 3.0, crowd)
    x = np.stack([np.full(V, -2.5), crowd, spike, np.where(rng.rand(V) < 0.5, 0.0, np.log(0.5)), -1e6 * rng.rand(V), np.round(rng.randn(V), 1)])
    u = rng.rand(6, 2)
    for rule in (dict(), dict(top_k=V // 2), dict(top_k=20), dict(top_p=0.5), dict(top_p=0.999), dict(top_k=V - 1, top_p=0.3), dict(temperature=1e-3, top_p=0.9),
                 dict(temperature=50.0, top_k=700, top_p=0.9, min_p=0.5)):
        check_rows(engine, x, u, **rule)


def test_rows_share_a_workspace_in_turn(engine):
    """Calls on two streams at once, of sizes that make the workspace grow in between: each finds its own results."""
    import torch
    rng = np.random.RandomState(9)
    work, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for n, V in enumerate((3000, 40000, 2000, 90000, 5000, 60000)):
        x, u = rng.randn(5, V).astype(np.float32), rng.rand(5, 2)
        with torch.cuda.stream(streams[n % 2]):
            work.append((engine.sample_rows(on_gpu(x), on_gpu(u), top_k=300, top_p=0.9)[0], o.sample_rows(x, u, top_k=300, top_p=0.9)[0]))
    torch.cuda.synchronize()
    for got, want in work:
        assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize('R', [1, 3, 4, 5, 257, 1000])
def test_rows_counts(engine, R):
    rng = np.random.RandomState(R)
    check_rows(engine, rng.randn(R, 20), rng.rand(R), top_k=6, top_p=0.8)


@pytest.mark.parametrize('V', [7, 64, 100, 1000, 2000, 9000])
def test_rows_ties_take_the_lowest_index(engine, V):
    rng = np.random.RandomState(V)
    u = np.concatenate([np.array([[0.0, 1.0 - 2.0 ** -53, 0.5]]), rng.rand(3, 3)])
    # powers of two as weights: every mass is exact, borders are hit exactly
    flat = np.zeros((4, V))
    steps = np.log(2.0) * np.floor(np.arange(V) % 4)[None, :].repeat(4, 0)
    for x in (flat, flat - 3.0e38, np.where(np.arange(V) % 3 == 1, 1.0, 0.0)[None, :].repeat(4, 0)):
        for rule in (dict(), dict(top_k=3), dict(top_k=V), dict(top_k=V + 5), dict(top_p=0.5), dict(top_p=0.25), dict(top_k=5, top_p=0.5), dict(min_p=1.0)):
            check_rows(engine, x, u, **rule)
            check_rows(engine, x.astype(np.float32), u, **rule)
    check_rows(engine, steps, rng.rand(4, 3), top_k=V // 3 + 1, top_p=0.77)
    signed = np.where(np.arange(V) % 2 == 0, 0.0, -0.0)[None, :].repeat(4, 0)
    check_rows(engine, signed, u, top_k=2)


@pytest.mark.parametrize('V', [5, 100, 700, 3001])
@pytest.mark.parametrize('dtype', ['float64', 'float32', 'float16'])
def test_rows_masks_infinities_and_nan(engine, V, dtype):
    rng = np.random.RandomState(V)
    low = float(np.finfo(dtype).min)
    x = rng.randn(12, V)
    x[0, :] = -np.inf
    x[1, :] = np.nan
    x[2, ::2] = -np.inf
    x[3, 1::2] = np.nan
    x[4, :] = low                                 # nothing but the type's lowest value: all alike
    x[5, : V // 2] = low
    x[6, V // 3] = np.inf
    x[7, [0, V - 1]] = np.inf
    x[8, :] = -np.inf
    x[8, V - 1] = low
    x[9, :] = np.where(np.arange(V) % 2, np.nan, -np.inf)
    x[10, :] = np.inf
    x[11, V // 2] = float(np.finfo(dtype).max)
    x = x.astype(dtype)
    u = rng.rand(12, 2)
    for rule in RULES:
        check_rows(engine, x, u, **rule)
    assert np.all(engine.sample_rows(x, u)[0][[0, 1, 9]] == -1)


def test_rows_rule_per_row(engine):
    import torch
    rng = np.random.RandomState(3)
    for V in (90, 1800):
        x, u = rng.randn(9, V), rng.rand(9, 2)
        rules = dict(temperature=np.array([0.0, 0.2, 1.0, 2.0, 0.5, 1.0, 1.0, 0.7, 3.0]), top_k=np.array([0, 3, 0, 50, 1, 0, 2, 0, 400]),
                     top_p=np.array([1.0, 0.9, 0.3, 1.0, 0.5, 0.99, 0.01, 1.0, 0.6]), min_p=np.array([0, 0, 0.1, 0, 0, 1.0, 0, 0.05, 0]))
        check_rows(engine, x, u, **rules)
        check_rows(engine, x, u, temperature=0.6, top_p=rules['top_p'])
        i, _ = engine.sample_rows(on_gpu(x), on_gpu(u), temperature=torch.from_numpy(rules['temperature']).cuda())
        assert np.array_equal(i.cpu().numpy(), o.sample_rows(x, u, temperature=rules['temperature'])[0])


def test_rows_device_rules_and_randoms_without_meaning_stay_in_bounds(engine):
    """Device memory is not looked at first: such numbers draw a kept index all the same."""
    rng = np.random.RandomState(4)
    for V in (50, 5000):
        x = rng.randn(6, V)
        u = np.array([[-1.0], [np.nan], [1.0], [7.0], [np.inf], [-np.inf]])
        i, _ = engine.sample_rows(on_gpu(x), on_gpu(u))
        i = i.cpu().numpy()[:, 0]
        assert np.array_equal(i, [0, 0, V - 1, V - 1, V - 1, 0])
        bad = np.array([np.nan, -1.0, np.inf, 0.0, 1e300, -np.inf])
        i, _ = engine.sample_rows(on_gpu(x), on_gpu(rng.rand(6, 1)), temperature=on_gpu(np.ones(6)), top_k=on_gpu(bad), top_p=on_gpu(bad), min_p=on_gpu(bad))
        i = i.cpu().numpy()
        assert np.all((i >= 0) & (i < V))
        i, _ = engine.sample_rows(on_gpu(x), on_gpu(rng.rand(6, 1)), temperature=on_gpu(np.array([np.nan, -1.0, 0.0, -np.inf, -0.0, np.nan])))
        assert np.array_equal(i.cpu().numpy()[:, 0], x.argmax(axis=1))


@pytest.mark.parametrize('dtype', ['float64', 'float32', 'float16', 'bfloat16'])
@pytest.mark.parametrize('V', [33, 100, 1900])
def test_rows_strides_and_alignment(engine, V, dtype):
    rng = np.random.RandomState(5)
    wide = scores_of(rng, 7, V + 13, dtype)
    u = rng.rand(7, 2)
    for lo in (0, 1, 3):
        x = wide[:, lo:lo + V]
        want, _ = o.sample_rows(as_f64(x), u, top_k=20, top_p=0.9)
        g = on_gpu(wide)[:, lo:lo + V]
        assert np.array_equal(engine.sample_rows(g, on_gpu(u), top_k=20, top_p=0.9)[0].cpu().numpy(), want)
        assert np.array_equal(engine.sample_rows(g[::2], on_gpu(u[::2]), top_k=20, top_p=0.9)[0].cpu().numpy(), want[::2])
        assert np.array_equal(engine.sample_rows(on_gpu(as_f64(wide).T)[lo:lo + V].T, on_gpu(u), top_k=20, top_p=0.9)[0].cpu().numpy(), want)
        if isinstance(x, np.ndarray):
            assert np.array_equal(engine.sample_rows(x, u, top_k=20, top_p=0.9)[0], want)
            assert np.array_equal(engine.sample_rows(x[::-1], u[::-1], top_k=20, top_p=0.9)[0], want[::-1])


def test_rows_of_no_rows(engine):
    i, lp = engine.sample_rows(np.zeros((0, 5)), np.zeros((0, 2)))
    assert i.shape == (0, 2) and lp.shape == (0, 2)
    i, lp = engine.sample_rows(on_gpu(np.zeros((0, 5))), on_gpu(np.zeros((0,))))
    assert tuple(i.shape) == (0,)


def test_rows_on_another_stream_and_in_a_graph(engine):
    import torch
    rng = np.random.RandomState(6)
    side = torch.cuda.Stream()
    for V in (100, 5000):
        x = [rng.randn(40, V).astype(np.float32) for _ in range(4)]
        u = [rng.rand(40, 2) for _ in range(4)]
        want = [o.sample_rows(a, b, top_k=30, top_p=0.9)[0] for a, b in zip(x, u)]
        with torch.cuda.stream(side):
            gx, gu = on_gpu(x[0]), on_gpu(u[0])
            i, _ = engine.sample_rows(gx, gu, top_k=30, top_p=0.9)
        side.synchronize()
        assert np.array_equal(i.cpu().numpy(), want[0])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            i, lp = engine.sample_rows(gx, gu, top_k=30, top_p=0.9)
        for n in range(4):                                  # replayed with other inputs, the program's own work in between
            gx.copy_(on_gpu(x[n])); gu.copy_(on_gpu(u[n]))
            graph.replay()
            torch.cuda.synchronize()
            assert np.array_equal(i.cpu().numpy(), want[n])
            eager, _ = engine.sample_rows(gx, gu, top_k=30, top_p=0.9)
            assert torch.equal(eager, i)


def test_long_rows_in_a_graph(engine):
    """Rows whose workspace a graph would share with later calls: captured, replayed between eager calls of other sizes."""
    import torch
    rng = np.random.RandomState(8)
    side = torch.cuda.Stream()
    x, u = [rng.randn(6, 20000).astype(np.float32) for _ in range(3)], [rng.rand(6, 2) for _ in range(3)]
    want = [o.sample_rows(a, b, top_k=300, top_p=0.9)[0] for a, b in zip(x, u)]
    with torch.cuda.stream(side):
        gx, gu = on_gpu(x[0]), on_gpu(u[0])
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        i, _ = engine.sample_rows(gx, gu, top_k=300, top_p=0.9)
    for n in range(3):
        gx.copy_(on_gpu(x[n])); gu.copy_(on_gpu(u[n]))
        graph.replay()
        eager, _ = engine.sample_rows(on_gpu(x[n]), on_gpu(u[n]), top_k=300, top_p=0.9)
        engine.sample_rows(on_gpu(rng.randn(2, 70000)), on_gpu(rng.rand(2, 1)), top_p=0.5)
        torch.cuda.synchronize()
        assert np.array_equal(i.cpu().numpy(), want[n]) and torch.equal(eager, i)


def test_long_rows_captured_without_a_workspace(engine):
    """The C call without a workspace under capture: the form that needs none."""
    import torch
    rng = np.random.RandomState(4)
    x, u = rng.randn(4, 9001), rng.rand(4, 2)
    want = o.sample_rows(x, u, top_k=100, top_p=0.8, min_p=0.01)[0]
    gx, gu = on_gpu(x), on_gpu(u)
    index = torch.full((4, 2), -7, dtype=torch.int64, device='cuda')
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        stream = torch.cuda.current_stream().cuda_stream
        assert engine._lib.snk_sample_rows_dev(engine._h, gx.data_ptr(), 0, 4, 9001, 9001, gu.data_ptr(), 2, 1.0, 100, 0.8, 0.01, None, index.data_ptr(), None,
                                               None, 0, stream) == 0
    for _ in range(3):
        index.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(index.cpu().numpy(), want)


@pytest.mark.parametrize('R,V', [(600, 9000), (300, 40000), (520, 70001)])
def test_rows_of_many_long_rows(engine, R, V):
    """A workgroup takes more of a row where rows are many: the same results as a few rows at a time."""
    import torch
    g = torch.Generator(device='cuda').manual_seed(V)
    x = torch.randn((R, V), device='cuda', generator=g)
    x[1::7] *= 1e-6                                         # one bin holds all of them
    x[2::7, : V - 5] = 0.25
    x[3::7] = torch.floor(x[3::7] * 3.0)
    x[4::7, 100:] = float('-inf')
    x[5] = float('nan')
    u = torch.rand((R, 2), device='cuda', dtype=torch.float64, generator=g)
    for rule in (dict(top_p=0.9), dict(top_k=V // 3, top_p=0.5), dict(top_k=40, min_p=0.01)):
        i, lp = engine.sample_rows(x, u, **rule)
        for a in range(0, R, 97):
            j, lq = engine.sample_rows(x[a:a + 4], u[a:a + 4], **rule)
            assert torch.equal(i[a:a + 4], j) and torch.equal(lp[a:a + 4], lq)
        few = [1, 2, 3, 4, 5, R - 1]
        want, _ = o.sample_rows(x[few].double().cpu().numpy(), u[few].cpu().numpy(), **rule)
        assert np.array_equal(i[few].cpu().numpy(), want)


@pytest.mark.parametrize('V', [100, 1000, 5000, 20000])
def test_rows_past_offsets_of_32_bits(engine, V):
    import torch
    g = torch.Generator(device='cuda').manual_seed(1)
    stride = (1 << 31) + 4096 + 8
    memory = torch.zeros(2 * stride + V, dtype=torch.float16, device='cuda')
    rows = memory.as_strided((3, V), (stride, 1))
    x = torch.randn((3, V), device='cuda', generator=g).half()
    rows.copy_(x)
    u = torch.rand((3, 2), device='cuda', dtype=torch.float64, generator=g)
    i, lp = engine.sample_rows(rows, u, top_p=0.8)
    j, lq = engine.sample_rows(x, u, top_p=0.8)
    assert torch.equal(i, j) and torch.equal(lp, lq)


@pytest.mark.parametrize('R,V', [((1 << 25) + 7, 2), ((1 << 21) + 3, 1025)])
def test_more_rows_than_a_launch_holds(engine, R, V):
    """Equal scores: every weight is 2^s, the draw is the quotient by it of the mass below u."""
    import torch
    x = torch.zeros((R, V), dtype=torch.float16, device='cuda')
    u = torch.rand(R, device='cuda', dtype=torch.float64, generator=torch.Generator(device='cuda').manual_seed(0))
    i, lp = engine.sample_rows(x, u)
    s = min(51, 62 - int(np.ceil(np.log2(V))))
    want = torch.div(torch.floor(u * float(V << s)).to(torch.int64), 1 << s, rounding_mode='floor')
    assert torch.equal(i, want)
    assert (lp + np.log(V)).abs().max().item() <= logp_tolerance(V, np.log(V))


def test_rows_of_many_draws(engine):
    """More draws than a launch's second dimension holds."""
    rng = np.random.RandomState(9)
    for V, draws in ((9000, 70000), (1500, 70000), (40, 70000)):
        x, u = rng.randn(2, V).astype(np.float32), rng.rand(2, draws)
        i, lp = [a.cpu().numpy() for a in engine.sample_rows(on_gpu(x), on_gpu(u), top_p=0.9)]
        some = np.r_[0:50, 32760:32780, 65530:65540, draws - 50:draws]
        want, want_lp = o.sample_rows(as_f64(x), u[:, some], top_p=0.9)
        assert np.array_equal(i[:, some], want)
        assert np.all(np.abs(lp[:, some] - want_lp) <= logp_tolerance(V, np.abs(want_lp).max()))
        assert i.min() >= 0


def test_rows_whose_exponents_are_no_numbers(engine):
    """A temperature of infinity (a rule in device memory) and a row that +inf shares: 0 times infinity weighs nothing."""
    import torch
    rng = np.random.RandomState(5)
    for V in (50, 1000, 5000, 20000):
        x = rng.randn(4, V)
        x[0, [V // 2, V - 1]] = np.inf
        x[1, :3] = np.inf
        x[2, 7] = -np.inf
        gx, gu = on_gpu(x), on_gpu(rng.rand(4, 40))
        tau = on_gpu(np.full(4, np.inf))
        for rule in (dict(), dict(top_k=5), dict(top_p=0.5), dict(top_k=5, top_p=0.5, min_p=0.1)):
            graph = torch.cuda.CUDAGraph()
            i, _ = engine.sample_rows(gx, gu, temperature=tau, **{k: on_gpu(np.full(4, float(w))) for k, w in rule.items()})
            rules = on_gpu(np.array([[np.inf, rule.get('top_k', 0), rule.get('top_p', 1.0), rule.get('min_p', 0.0)]] * 4))
            j = torch.empty_like(i)
            with torch.cuda.graph(graph):                       # (without a workspace)
                assert engine._lib.snk_sample_rows_dev(engine._h, gx.data_ptr(), 0, 4, V, V, gu.data_ptr(), 40, 1.0, 0, 1.0, 0.0, rules.data_ptr(), j.data_ptr(),
                                                       None, None, 0, torch.cuda.current_stream().cuda_stream) == 0
            graph.replay()
            torch.cuda.synchronize()
            i, j = i.cpu().numpy(), j.cpu().numpy()
            assert np.array_equal(i, j) and np.all((i >= 0) & (i < V))
            assert set(i[0]) <= {V // 2, V - 1} and set(i[1]) <= {0, 1, 2} and 7 not in i[2]


@pytest.mark.parametrize('dtype', ['float32', 'float64', 'float16', 'bfloat16'])
@pytest.mark.parametrize('V', [1025, 2047, 2048, 2049, 4095, 4097, 8191, 8192, 8193])
def test_rows_at_the_borders_of_the_workgroups_sizes(engine, V, dtype):
    rng = np.random.RandomState(V)
    x, u = scores_of(rng, 5, V, dtype), rng.rand(5, 2)
    x[1, :] = -np.inf
    x[2, :] = -np.inf
    x[2, V - 1] = 3.0
    x[3, :V // 2] = x[3, 0]                                  # equal ones
    for rule in RULES:
        check_rows(engine, x, u, **rule)


@pytest.mark.parametrize('V', [1500, 5000, 8000])
def test_rows_in_a_workgroup_whose_scores_crowd(engine, V):
    """Every score in one bin but for one that stretches the range; equal in all but the last bits; few different ones."""
    rng = np.random.RandomState(V)
    x = np.zeros((5, V))
    x[0] = rng.permutation(V) * 2.0 ** -52 + 1.0
    x[1] = rng.permutation(V) / 2.0 ** 30
    x[1, V // 3] = -30.0
    x[2] = rng.randint(0, 3, V) * 2.0 ** -40
    x[3] = 7.0
    x[4] = -rng.rand(V) * 40.0
    u = rng.rand(5, 70)                                     # more draws than a wavefront has lanes
    for rule in (dict(top_k=V // 2), dict(top_k=1), dict(top_p=0.37), dict(top_p=1e-9), dict(top_k=V - 1, top_p=0.999), dict(top_k=100, top_p=0.5, min_p=0.9)):
        check_rows(engine, x, u, **rule)


@pytest.mark.parametrize('V', [30, 900])
def test_rows_of_a_hundred_draws(engine, V):
    rng = np.random.RandomState(V)
    check_rows(engine, rng.randn(7, V), rng.rand(7, 100), top_p=0.8)


@pytest.mark.parametrize('dtype', ['float32', 'float64', 'bfloat16'])
@pytest.mark.parametrize('V', [20000, 70001])
def test_rows_whose_boundary_is_one_chunks(engine, V, dtype):
    """The scores among which the order reaches its goal: all in one chunk, one in each, more of them than a workgroup holds at once,
    more than the list holds."""
    rng = np.random.RandomState(V)
    x = np.full((4, V), -30.0)
    x[0, 8192:8192 + 3000] = rng.permutation(3000) / 4096.0          # side by side
    x[1, ::8192] = rng.permutation(x[1, ::8192].size) / 64.0
    x[2, :12000] = rng.permutation(12000) / 2.0 ** 20
    x[3, :V - 1] = rng.permutation(V - 1) / 2.0 ** 24
    if dtype == 'bfloat16':
        import torch
        x = torch.from_numpy(x).to(torch.bfloat16)
    else:
        x = x.astype(dtype)
    u = rng.rand(4, 3)
    for rule in (dict(top_k=2), dict(top_k=1999), dict(top_p=0.5), dict(top_k=9000, top_p=0.4), dict(temperature=0.01, top_p=0.7)):
        check_rows(engine, x, u, **rule)


# ---------------------------------------------------------------------------------------------------------------- trellis
class Voice(object):
    def __init__(self, engine, Dj=9, n=400, seed=0):
        rng = np.random.RandomState(seed)
        walk = np.cumsum(rng.randn(n + 1, Dj), axis=0)
        self.JC = (walk / walk.std()).astype(np.float32)
        self.wj = 0.3 + rng.rand(Dj)
        self.n = n
        self.engine = engine
        engine.upload_join_only(self.JC)
        engine.set_weights(None, self.wj)
        engine.set_position_bias(None)
        self.bias, self.edges = None, ()

    def set_bias(self, classes, n_buckets, seed=1, forbid=False):
        rng = np.random.RandomState(seed)
        self.edges = np.array(sorted([1, 2, 0, -3, 9, -20, 40][:n_buckets - 1]), dtype=np.int64)
        self.bias = 0.7 * rng.randn(classes, n_buckets)
        if forbid:
            self.bias[0, int(np.searchsorted(self.edges, 0, side='right'))] = np.inf
        self.engine.set_position_bias(self.bias, self.edges)

    def candidates(self, lengths, K, seed=2, pad=True):
        rng = np.random.RandomState(seed)
        rows = int(sum(lengths))
        cand = rng.randint(0, self.n, (rows, K)).astype(np.int64)
        for t in range(1, rows):                            # natural successors and repetitions of the row before
            k = rng.randint(0, K, max(1, K // 3))
            cand[t, k] = np.minimum(cand[t - 1, rng.randint(0, K, k.size)] + rng.randint(0, 2, k.size), self.n - 1)
        dist = rng.rand(rows, K) * 2.0
        if pad and K > 2:
            short = rng.rand(rows) < 0.2
            cand[short, K - K // 3:] = -1
            dist[short, K - K // 3:] = 1e15
        return cand, dist, np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)

    def model(self):
        return dict(JC=self.JC, wj=self.wj, bias=self.bias, edges=self.edges)


def sum_tolerance(T, K, size):
    """Of a log-sum over paths (size: its largest term): every step rounds its sum of K terms, its logarithm and its values of up to
    `size`; 8 roundings a step in either program."""
    return 2.0 ** -53 * T * (K + 16.0) + 2.0 ** -53 * 16.0 * T * max(size, 1.0)


def check_paths(v, cand, dist, offs, u, join_class=None, **rule):
    e = v.engine
    got = [e.sample_paths(cand, dist, u, row_offsets=offs, join_class=join_class, **rule)]
    dev = e.sample_paths(on_gpu(cand), on_gpu(dist), on_gpu(u), row_offsets=offs, join_class=None if join_class is None else on_gpu(join_class), **rule)
    got.append([a.cpu().numpy() for a in dev])
    for a, b in zip(*got):
        assert np.array_equal(a, b)
    path, cost, logp = got[0]
    rule = dict(rule)
    tau = rule.pop('temperature', 1.0)
    for i in range(len(offs) - 1):
        a, b = int(offs[i]), int(offs[i + 1])
        for s in range(u.shape[0]):
            want, c, lp = o.sample_path(cand[a:b], dist[a:b], u[s, a:b], tau, join_class=None if join_class is None else join_class[a:b], **dict(v.model(), **rule))
            assert np.array_equal(path[s, a:b], want), (i, s)
            if np.isinf(c):
                assert cost[s, i] == np.inf and logp[s, i] == -np.inf
            else:
                size = np.abs(c) / (tau or 1.0) + 40.0
                assert abs(cost[s, i] - c) <= 2.0 ** -52 * 4.0 * (b - a) * max(abs(c), 1.0)
                assert abs(logp[s, i] - lp) <= 2.0 * (b - a) * logp_tolerance(cand.shape[1]) + 2.0 * sum_tolerance(b - a, cand.shape[1], size)
    return got[0]


def check_posterior(v, cand, dist, offs, join_class=None, temperature=1.0):
    e = v.engine
    got = [e.path_posterior(cand, dist, row_offsets=offs, join_class=join_class, temperature=temperature)]
    dev = e.path_posterior(on_gpu(cand), on_gpu(dist), row_offsets=offs, join_class=None if join_class is None else on_gpu(join_class), temperature=temperature)
    got.append([None if a is None else a.cpu().numpy() for a in dev])
    for a, b in zip(*got):
        assert (a is None and b is None) or np.array_equal(a, b)
    logz, post, uses = got[0]
    K, total, slack = cand.shape[1], None, 0.0
    for i in range(len(offs) - 1):
        a, b = int(offs[i]), int(offs[i + 1])
        z, p, n = o.posterior(cand[a:b], dist[a:b], temperature, join_class=None if join_class is None else join_class[a:b], **v.model())
        if z == -np.inf:
            assert logz[i] == -np.inf and not post[a:b].any()
        else:
            tol = sum_tolerance(b - a, K, abs(z) + 2.0 * (b - a) / temperature)
            assert abs(logz[i] - z) <= tol
            assert np.all(np.abs(post[a:b] - p) <= 4.0 * tol)      # a probability's error: that of its exponent, three sums in it
            # a count: the sum of its row's probabilities, each with that error, K K cells rounded to 2^-50
            slack += (b - a) * (4.0 * tol + K * K * 2.0 ** -51)
        total = n if total is None else total + n
    if v.bias is None:
        assert uses is None
    else:
        assert np.all(np.abs(uses - total) <= slack)
    return logz, post, uses


@pytest.mark.parametrize('lengths,K,Dj', [([1], 1, 3), ([1], 7, 9), ([2], 1, 9), ([5], 3, 9), ([1, 2, 1, 3], 5, 9), ([40], 30, 9), ([13, 64, 1, 30], 64, 20),
                                          ([21, 17], 65, 9), ([30], 100, 33), ([12, 9], 128, 9), ([9], 129, 9), ([7, 8], 208, 9), ([250], 12, 9)])
@pytest.mark.parametrize('bias', [None, (1, 1), (3, 8)])
def test_trellis_draws_and_posteriors(engine, lengths, K, Dj, bias):
    v = Voice(engine, Dj=Dj, n=300 + 5 * K)
    cand, dist, offs = v.candidates(lengths, K)
    rng = np.random.RandomState(K)
    cls = None
    if bias:
        v.set_bias(*bias, forbid=bias[1] > 4)
        cls = rng.randint(-1, bias[0] + 1, cand.shape[0]).astype(np.int32)      # some joins without a class
        if bias[0] == 1:
            cls = None
    u = rng.rand(2, cand.shape[0])
    for rule in (dict(), dict(temperature=0.2, top_p=0.9), dict(temperature=2.0, top_k=5, top_p=0.8, min_p=0.05), dict(temperature=0.0)):
        check_paths(v, cand, dist, offs, u, cls, **rule)
    for tau in (0.1, 1.0, 5.0):
        check_posterior(v, cand, dist, offs, cls, tau)


def test_trellis_of_extreme_temperatures(engine):
    """Path costs of thousands of temperatures apart: every sum is dominated by its largest term, none of them vanishes."""
    v = Voice(engine)
    v.set_bias(1, 8)
    cand, dist, offs = v.candidates([30, 5], 20)
    u = np.random.RandomState(0).rand(2, 35)
    for tau in (1e-4, 1e-2, 1e3):
        check_paths(v, cand, dist, offs, u, temperature=tau)
        check_posterior(v, cand, dist, offs, temperature=tau)
    # a far cheaper join into a far dearer candidate, and the other way round: the step's cheapest cell is on no path
    dist[3, :] = 1e6
    dist[3, 4] = 5e5
    for tau in (1e-2, 1.0):
        check_paths(v, cand, dist, offs, u, temperature=tau)
        check_posterior(v, cand, dist, offs, temperature=tau)


def test_trellis_of_costs_that_overflow(engine):
    """Costs over a temperature that float64 does not hold, either sign, and a bias of that size: units of the candidates, or none."""
    v = Voice(engine)
    cand, dist, offs = v.candidates([30, 5], 20)
    rng = np.random.RandomState(1)
    u = rng.rand(3, 35)
    for scale, tau, bias in ((1e300, 1e-10, 0.0), (-1e300, 1e-10, 0.0), (-1e308, 1e-300, 0.0), (1.0, 1e-300, 0.0), (1.0, 0.5, -1e308), (1.0, 1e-10, 1e308),
                             (-1e300, 1e-300, -1e300)):
        d = dist * scale
        d[rng.rand(*d.shape) < 0.3] *= -1.0
        engine.set_position_bias(np.array([[0.0, bias]]), [1])
        for t in (tau, 0.0):
            path, cost, logp = engine.sample_paths(cand, d, u, row_offsets=offs, temperature=t, top_p=0.9)
            drawn = (path[:, :, None] == cand[None]).any(axis=2)
            assert np.all(drawn | (path == -1))
        logz, post, uses = engine.path_posterior(cand, d, row_offsets=offs, temperature=tau)
        assert post.shape == cand.shape and uses.shape == (1, 2)


@pytest.mark.parametrize('tau', [1e-300, 1e-310, 5e-324])
def test_trellis_of_a_temperature_whose_inverse_overflows(engine, tau):
    """The cheapest path, as at temperature 0; all of the probability is its."""
    v = Voice(engine)
    cand, dist, offs = v.candidates([30, 1, 7], 20)
    rng = np.random.RandomState(1)
    cheapest, cost, _ = engine.sample_paths(cand, dist, rng.rand(1, 38), row_offsets=offs, temperature=0.0)
    path, c, logp = engine.sample_paths(cand, dist, rng.rand(3, 38), row_offsets=offs, temperature=tau)
    assert np.array_equal(path, np.repeat(cheapest, 3, axis=0)) and np.array_equal(c, np.repeat(cost, 3, axis=0)) and not logp.any()
    # float32 and float64 rows in the same limit
    x = rng.randn(5, 30)
    assert np.array_equal(engine.sample_rows(x, rng.rand(5), temperature=tau)[0], x.argmax(axis=1))


def test_trellis_without_a_complete_path(engine):
    v = Voice(engine)
    cand, dist, offs = v.candidates([6, 4, 1, 5], 5, pad=False)
    cand[2] = -1                                  # the first utterance breaks
    dist[6:10][1] = np.inf                        # the second one as well
    cand[10] = 0                                  # the third one's only row cannot join
    dist[13, 2] = np.nan
    dist[14, 1] = -np.inf
    u = np.random.RandomState(0).rand(3, 16)
    for rule in (dict(), dict(temperature=0.0), dict(top_k=2, top_p=0.5)):
        path, cost, logp = check_paths(v, cand, dist, offs, u, **rule)
        assert np.all(path[:, :11] == -1) and np.all(path[:, 11:] >= 1)
    check_posterior(v, cand, dist, offs)
    v.set_bias(1, 8)
    v.engine.set_position_bias(np.full((1, 1), np.inf), [])      # every join forbidden: single rows are left
    v.bias, v.edges = np.full((1, 1), np.inf), ()
    cand[10] = 7
    path, cost, logp = check_paths(v, cand, dist, offs, u)
    assert np.all(path[:, 10] == 7) and np.all(path[:, 11:] == -1)
    check_posterior(v, cand, dist, offs)


def test_trellis_with_the_same_unit_twice(engine):
    v = Voice(engine)
    v.set_bias(2, 8)
    cand, dist, offs = v.candidates([12], 6, pad=False)
    cand[:, 3] = cand[:, 0]
    dist[:, 3] = dist[:, 0]
    cand[5, :] = 11
    dist[5, :] = 0.5
    u = np.random.RandomState(0).rand(4, 12)
    for rule in (dict(), dict(top_k=1), dict(top_k=2), dict(temperature=0.0)):
        check_paths(v, cand, dist, offs, u, **rule)
    check_posterior(v, cand, dist, offs)


def test_cheapest_path_is_that_of_the_viterbi_search(engine):
    v = Voice(engine, Dj=20, n=1500)
    cand, dist, offs = v.candidates([50, 80], 40)
    path, cost, _ = v.engine.sample_paths(cand, dist, np.zeros((1, 130)), row_offsets=offs, temperature=0.0)
    for i, (a, b) in enumerate(((0, 50), (50, 130))):
        want, c = v.engine.viterbi(cand[a:b], dist[a:b])
        assert path[0, a:b].tolist() == want
        assert abs(cost[0, i] - c) <= 2.0 ** -52 * 2.0 * (b - a) * c


@pytest.mark.parametrize('bias', [None, (1, 4)])
def test_probabilities_against_all_paths(engine, bias):
    """Every path of a small trellis: logZ, posteriors and uses are sums over them; so is the probability of a draw."""
    v = Voice(engine)
    if bias:
        v.set_bias(*bias)
    T, K, tau = 5, 4, 0.6
    cand, dist, offs = v.candidates([T], K, pad=False)
    cand = np.clip(cand, 1, v.n - 2)
    local, C, B = o.trellis(cand, dist, temperature=tau, **v.model())
    paths = list(itertools.product(range(K), repeat=T))
    score = np.array([sum(local[t][p[t]] for t in range(T)) - sum(C[t][p[t], p[t + 1]] for t in range(T - 1)) / tau for p in paths])
    z = o.lse(score)
    w = np.exp(score - z)
    logz, post, uses = v.engine.path_posterior(cand, dist, temperature=tau)
    tol = sum_tolerance(T, K, abs(z)) + K ** T * 2.0 ** -53
    assert abs(logz[0] - z) <= tol
    for t in range(T):
        for k in range(K):
            assert abs(post[t, k] - sum(x for x, p in zip(w, paths) if p[t] == k)) <= 4.0 * tol
    if bias:
        n = np.zeros(v.bias.shape)
        for x, p in zip(w, paths):
            for t in range(T - 1):
                n[0, B[t][p[t], p[t + 1]]] += x
        assert np.all(np.abs(uses - n) <= T * (4.0 * tol + K * K * 2.0 ** -51))
    u = np.random.RandomState(1).rand(50, T)
    path, cost, logp = v.engine.sample_paths(cand, dist, u, temperature=tau)
    for s in range(50):
        assert abs(logp[s, 0] - (-cost[s, 0] / tau - z)) <= 4.0 * tol + 2.0 * T * logp_tolerance(K)


def test_gradients_against_differences(engine):
    """Central differences of logZ.  h^2 / 6 times a third derivative (at most 4 / tau^3 per unit) and logZ's rounding over h."""
    v = Voice(engine)
    v.set_bias(2, 6)
    tau, h = 0.8, 2.0 ** -14
    cand, dist, offs = v.candidates([15, 9], 6)
    cls = np.random.RandomState(0).randint(0, 2, 24).astype(np.int32)
    logz, post, uses = v.engine.path_posterior(cand, dist, row_offsets=offs, join_class=cls, temperature=tau)
    tol = h * h / 6.0 * 4.0 / tau ** 3 + 4.0 * sum_tolerance(15, 6, np.abs(logz).max() + 40.0) / h

    def z(d):
        return v.engine.path_posterior(cand, d, row_offsets=offs, join_class=cls, temperature=tau)[0].sum()
    for t, k in ((0, 0), (7, 3), (14, 1), (15, 2), (23, 0)):
        if cand[t, k] < 1:
            continue
        up, down = dist.copy(), dist.copy()
        up[t, k] += h
        down[t, k] -= h
        assert abs((z(up) - z(down)) / (2.0 * h) + post[t, k] / tau) <= tol
    for c in range(2):
        for b in range(6):
            values = []
            for sign in (1.0, -1.0):
                moved = v.bias.copy()
                moved[c, b] += sign * h
                v.engine.set_position_bias(moved, v.edges)
                values.append(z(dist))
            # up to 22 joins move at once: the third cumulant of a count of n is at most n^3
            assert abs((values[0] - values[1]) / (2.0 * h) + uses[c, b] / tau) <= tol + h * h / 6.0 * 22.0 ** 3 / tau ** 3


@pytest.mark.parametrize('lengths,K', [([100], 5), ([64, 1, 9, 2, 150], 30), ([200, 33], 50), ([24, 25, 26, 65, 66], 20), ([120], 100), ([90, 91, 2], 104),
                                       ([60], 120), ([70, 8, 40], 200), ([300], 64)])
def test_recursions_in_pieces(engine, lengths, K):
    """Utterances of 25 rows and more run their recursions in pieces, side by side."""
    v = Voice(engine, Dj=9, n=300 + 5 * K)
    v.set_bias(2, 8, forbid=True)
    cand, dist, offs = v.candidates(lengths, K)
    rng = np.random.RandomState(1)
    cls, u = rng.randint(0, 2, cand.shape[0]).astype(np.int32), rng.rand(1, cand.shape[0])
    for tau in (0.3, 2.0):
        check_posterior(v, cand, dist, offs, cls, tau)
        check_paths(v, cand, dist, offs, u, cls, temperature=tau, top_p=0.9)


def test_trellis_of_more_than_four_gigabytes(engine):
    """Cells of one utterance past offsets of 32 bits: the cheapest path against the search's own, probabilities that sum to 1."""
    T, K = 13000, 208
    v = Voice(engine, n=5000)
    cand, dist, offs = v.candidates([T], K, pad=False)
    assert T * K * K * 8 > 1 << 32
    u = np.random.RandomState(0).rand(1, T)
    path, cost, _ = engine.sample_paths(cand, dist, u, temperature=0.0)
    _, want_cost = engine.viterbi(cand, dist)
    product = (v.JC.shape[1] + 4.0) * 2.0 ** -45             # of a join cost by products, relative: the choice between paths that near
    assert abs(cost[0, 0] - want_cost) <= (2.0 ** -52 * 4.0 * T + 2.0 * product) * want_cost
    logz, post, _ = engine.path_posterior(cand, dist, temperature=0.8)
    size = abs(logz[0]) + 2.0 * T / 0.8
    assert np.abs(post.sum(axis=1) - 1.0).max() <= 8.0 * sum_tolerance(T, K, size) and post.min() >= 0.0
    path, cost, logp = engine.sample_paths(cand, dist, u, temperature=0.8)
    assert (path[0][:, None] == cand).any(axis=1).all() and cost[0, 0] > want_cost and logp[0, 0] < 0.0
    # without a truncation the log probability is the path's own
    assert abs(logp[0, 0] - (-cost[0, 0] / 0.8 - logz[0])) <= 2.0 * T * logp_tolerance(K) + 4.0 * sum_tolerance(T, K, size) + 4.0 * product * cost[0, 0] / 0.8


@pytest.mark.parametrize('T,K', [(30000, 3), (5000, 33)])
def test_trellis_of_a_long_utterance(engine, T, K):
    v = Voice(engine, n=2000)
    v.set_bias(1, 8)
    cand, dist, offs = v.candidates([T], K)
    u = np.random.RandomState(3).rand(1, T)
    check_posterior(v, cand, dist, offs, temperature=0.7)
    check_paths(v, cand, dist, offs, u, temperature=0.7, top_p=0.95)


def test_trellis_results_do_not_depend_on_the_batch(engine):
    v = Voice(engine)
    v.set_bias(2, 8)
    cand, dist, offs = v.candidates([11, 40, 3], 25)
    rng = np.random.RandomState(0)
    u, cls = rng.rand(3, 54), rng.randint(0, 2, 54).astype(np.int32)
    path, cost, logp = v.engine.sample_paths(cand, dist, u, row_offsets=offs, join_class=cls, temperature=0.5, top_p=0.9)
    logz, post, uses = v.engine.path_posterior(cand, dist, row_offsets=offs, join_class=cls, temperature=0.5)
    for i in range(3):
        a, b = int(offs[i]), int(offs[i + 1])
        p, c, l = v.engine.sample_paths(cand[a:b], dist[a:b], u[:, a:b], join_class=cls[a:b], temperature=0.5, top_p=0.9)
        assert np.array_equal(p, path[:, a:b]) and np.array_equal(c[:, 0], cost[:, i]) and np.array_equal(l[:, 0], logp[:, i])
        z, q, n = v.engine.path_posterior(cand[a:b], dist[a:b], join_class=cls[a:b], temperature=0.5)
        assert z[0] == logz[i] and np.array_equal(q, post[a:b])
    again = v.engine.path_posterior(cand, dist, row_offsets=offs, join_class=cls, temperature=0.5)
    assert all(np.array_equal(a, b) for a, b in zip(again, (logz, post, uses)))


@pytest.mark.parametrize('K', [64, 100, 130])
def test_trellis_tiles_do_not_depend_on_the_batch(engine, K):
    """A sentence by itself (small tiles, few workgroups) and among many others."""
    v = Voice(engine, n=2000)
    v.set_bias(2, 8)
    lengths = [60, 26, 1, 150, 200, 90, 2, 170]
    cand, dist, offs = v.candidates(lengths, K)
    rng = np.random.RandomState(0)
    u, cls = rng.rand(2, cand.shape[0]), rng.randint(0, 2, cand.shape[0]).astype(np.int32)
    path, cost, logp = v.engine.sample_paths(cand, dist, u, row_offsets=offs, join_class=cls, temperature=0.5, top_p=0.9)
    logz, post, _ = v.engine.path_posterior(cand, dist, row_offsets=offs, join_class=cls, temperature=0.5)
    for i in (0, 1, 2, 6):
        a, b = int(offs[i]), int(offs[i + 1])
        p, c, l = v.engine.sample_paths(cand[a:b], dist[a:b], u[:, a:b], join_class=cls[a:b], temperature=0.5, top_p=0.9)
        assert np.array_equal(p, path[:, a:b]) and np.array_equal(c[:, 0], cost[:, i]) and np.array_equal(l[:, 0], logp[:, i])
        z, q, _ = v.engine.path_posterior(cand[a:b], dist[a:b], join_class=cls[a:b], temperature=0.5)
        assert z[0] == logz[i] and np.array_equal(q, post[a:b])


def test_trellis_of_many_utterances(engine):
    """More utterances than a launch's second dimension holds, short ones beside a long one."""
    v = Voice(engine)
    rng = np.random.RandomState(0)
    lengths = rng.randint(1, 4, 70001)
    lengths[[5, 69000]] = 700, 900
    cand, dist, offs = v.candidates(lengths, 2)
    u = rng.rand(1, cand.shape[0])
    path, cost, logp = v.engine.sample_paths(cand, dist, u, row_offsets=offs)
    logz, post, _ = v.engine.path_posterior(cand, dist, row_offsets=offs)
    usable = ((cand >= 1) & (cand < v.n - 1)).any(axis=1)        # rows of two units that cannot be joined leave a few utterances empty
    alive = np.logical_and.reduceat(usable, offs[:-1])
    rows_alive = np.repeat(alive, lengths)
    assert 0 < (~alive).sum() < 20
    assert np.array_equal(path[0] >= 0, rows_alive) and np.array_equal(np.isfinite(cost[0]), alive) and np.array_equal(np.isfinite(logz), alive)
    assert not post[~rows_alive].any()
    # a row's probabilities sum to 1: two of them, each with the error of the recursions (sum_tolerance, and 4 roundings more)
    size = np.abs(logz[alive]).max() + 2.0 * 900
    assert np.abs(post[rows_alive].sum(axis=1) - 1.0).max() <= 8.0 * sum_tolerance(900, 2, size)
    for i in (0, 4, 5, 6, 32767, 32768, 32769, 65535, 65536, 68999, 69000, 69001, 70000):
        a, b = int(offs[i]), int(offs[i + 1])
        p, c, l = v.engine.sample_paths(cand[a:b], dist[a:b], u[:, a:b])
        assert np.array_equal(p, path[:, a:b]) and c[0, 0] == cost[0, i] and l[0, 0] == logp[0, i]
        z, q, _ = v.engine.path_posterior(cand[a:b], dist[a:b])
        assert z[0] == logz[i] and np.array_equal(q, post[a:b])


@pytest.mark.parametrize('Dj', [1, 33, 151, 302])
def test_join_costs_of_far_and_near_units(engine, Dj):
    """Frames that lie far from the origin, next to each other, and equal.  The engine may take a squared distance from products,
    |e|^2 + |s|^2 - 2 e s, where that is above 2^-10 of n = |e|^2 + |s|^2.  Its Dj + 4 roundings of 2^-53 are (Dj + 4) 2^-52 n of the
    square, (Dj + 4) 2^-53 n / c of a distance c >= 2^-5 sqrt(n): at most (Dj + 4) 2^-48 sqrt(n), n at most twice the square of the
    largest distance about the unit that both are taken relative to.  Below 2^-45 (Dj + 4) of the largest join cost, four times that:
    once a row and for each sum that it enters."""
    v = Voice(engine, Dj=Dj, n=300)
    rng = np.random.RandomState(Dj)
    JC = 3000.0 + rng.randn(301, Dj)
    JC[100:200] = JC[100] + 1e-3 * rng.randn(100, Dj)
    JC[200:250] = JC[200]
    JC[250:260] = 0.0
    v.JC = JC.astype(np.float32)
    v.wj = v.wj / np.sqrt(Dj)
    engine.upload_join_only(v.JC)
    engine.set_weights(None, v.wj)
    T, K = 30, 20
    cand = rng.randint(0, 300, (T, K)).astype(np.int64)
    cand[10:20] = rng.randint(100, 200, (10, K))
    cand[20:25] = rng.randint(200, 250, (5, K))
    dist = rng.rand(T, K)
    furthest = np.sqrt((v.wj ** 2 * (v.JC.max(axis=0) - v.JC.min(axis=0)).astype(np.float64) ** 2).sum())
    for near in (True, False):                              # without and with the frames at the origin
        if not near:
            cand[0, 0] = 255
        z, p, _ = o.posterior(cand, dist, 1.0, **v.model())
        logz, post, _ = engine.path_posterior(cand, dist)
        tol = sum_tolerance(T, K, abs(z) + 2.0 * T) + T * furthest * (Dj + 4.0) * 2.0 ** -45
        assert abs(logz[0] - z) <= tol
        assert np.all(np.abs(post - p) <= 4.0 * tol)


def test_trellis_on_another_stream(engine):
    import torch
    v = Voice(engine)
    v.set_bias(1, 8)
    cand, dist, offs = v.candidates([30, 20], 15)
    u = np.random.RandomState(0).rand(2, 50)
    want = v.engine.sample_paths(cand, dist, u, row_offsets=offs)
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            gd = torch.zeros((50, 15), dtype=torch.float64, device='cuda')
            big = torch.rand((2048, 2048), device='cuda')
            for _ in range(4):
                big = big @ big * 1e-3                      # keeps the stream busy while the call is queued
            gd += torch.from_numpy(dist).cuda()
            path, cost, logp = v.engine.sample_paths(on_gpu(cand), gd, on_gpu(u), row_offsets=offs)
            gd.fill_(-1.0)                                  # the stream's next work waits for the call
            both = torch.cat([cost.view(-1), logp.view(-1)])
        side.synchronize()
        assert np.array_equal(path.cpu().numpy(), want[0])
        assert np.array_equal(both.cpu().numpy(), np.concatenate([want[1].ravel(), want[2].ravel()]))


def test_trellis_calls_on_streams_at_once_and_changes_behind_them(engine):
    """Calls on two streams in turn share the workspaces, and so does one that waits; a bias, weights and frames that change right
    behind a queued call are not seen by it."""
    import torch
    v = Voice(engine)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    rng = np.random.RandomState(2)
    work = []
    for n, (T, K) in enumerate(((200, 40), (30, 90), (400, 20), (25, 25), (300, 40), (60, 64))):
        v.set_bias(1, 4 + n % 3, seed=n)
        v.wj = 0.3 + rng.rand(v.wj.size)
        engine.set_weights(None, v.wj)
        if n == 3:
            v.JC = v.JC[::-1].copy()
            engine.upload_join_only(v.JC)
            engine.set_weights(None, v.wj)
        cand, dist, offs = v.candidates([T, 3], K, seed=n)
        u = rng.rand(1, T + 3)
        with torch.cuda.stream(streams[n % 2]):
            args = on_gpu(cand), on_gpu(dist), on_gpu(u)
            big = torch.rand((1024, 1024), device='cuda')
            for _ in range(6):
                big = big @ big * 1e-3                      # the call is still waiting when the next one is made
            got = engine.sample_paths(*args, row_offsets=offs)
            post = engine.path_posterior(*args[:2], row_offsets=offs)
        work.append((got, post, cand, dist, offs, u, v.model()))
        if n == 4:                                          # one that waits, between the two
            host = engine.path_posterior(cand, dist, row_offsets=offs)
            torch.cuda.synchronize()
            assert all(np.array_equal(a, b.cpu().numpy()) for a, b in zip(host, post))
    torch.cuda.synchronize()
    for got, post, cand, dist, offs, u, model in work:
        for i in range(2):
            a, b = int(offs[i]), int(offs[i + 1])
            want, c, lp = o.sample_path(cand[a:b], dist[a:b], u[0, a:b], 1.0, **model)
            assert np.array_equal(got[0].cpu().numpy()[0, a:b], want)
            z, p, _ = o.posterior(cand[a:b], dist[a:b], 1.0, **model)
            tol = sum_tolerance(b - a, cand.shape[1], abs(z) + 2.0 * (b - a))
            assert abs(post[0].cpu().numpy()[i] - z) <= tol and np.all(np.abs(post[1].cpu().numpy()[a:b] - p) <= 4.0 * tol)


def test_trellis_refuses_a_stream_under_capture(engine):
    import torch
    import snickery_amd
    v = Voice(engine)
    cand, dist, offs = v.candidates([10], 5)
    g = [on_gpu(a) for a in (cand, dist, np.random.RandomState(0).rand(1, 10))]
    v.engine.sample_paths(*g)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    refused = []
    with torch.cuda.graph(graph):
        for call in (lambda: v.engine.sample_paths(*g), lambda: v.engine.path_posterior(g[0], g[1])):
            try:
                call()
            except snickery_amd.SnkError as e:
                refused.append(str(e))
        y = g[1] + 1.0
    assert len(refused) == 2 and all('captured' in r for r in refused)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, g[1] + 1.0)
