"""oracle/sampling_oracle.py against sums over every path, on the CPU."""
import itertools

import numpy as np

import sampling_oracle as o


def _small(seed=0, T=4, K=3, n=60, Dj=5):
    rng = np.random.RandomState(seed)
    JC, wj = rng.randn(n + 1, Dj).astype(np.float32), rng.rand(Dj)
    cand, dist = rng.randint(1, n - 1, (T, K)), rng.rand(T, K)
    bias, edges = rng.randn(2, 4), np.array([-3, 0, 5])
    cls = rng.randint(0, 2, T)
    return cand, dist, dict(JC=JC, wj=wj, bias=bias, edges=edges, join_class=cls)


def test_posterior_is_the_sum_over_paths():
    cand, dist, m = _small()
    T, K, tau = 4, 3, 0.7
    local, C, B = o.trellis(cand, dist, temperature=tau, **m)
    paths = list(itertools.product(range(K), repeat=T))
    w = np.exp([sum(local[t][p[t]] for t in range(T)) - sum(C[t][p[t], p[t + 1]] for t in range(T - 1)) / tau for p in paths])
    z, post, uses = o.posterior(cand, dist, tau, **m)
    assert abs(z - np.log(w.sum())) < 1e-12
    want = np.zeros((2, 4))
    for p, x in zip(paths, w / w.sum()):
        for t in range(T - 1):
            want[m['join_class'][t], B[t][p[t], p[t + 1]]] += x
    assert np.abs(uses - want).max() < 1e-12 and np.abs(post.sum(axis=1) - 1.0).max() < 1e-12


def test_draws_have_the_paths_probabilities():
    cand, dist, m = _small(1)
    tau = 0.5
    z = o.posterior(cand, dist, tau, **m)[0]
    u = np.random.RandomState(2).rand(40, 4)
    for row in u:
        _, cost, logp = o.sample_path(cand, dist, row, tau, **m)
        assert abs(logp - (-cost / tau - z)) < 1e-12
    # the draw of a row inverts its cumulative distribution: equally spaced numbers draw every index as often as its weight says
    x = np.array([0.0, np.log(3.0), -np.inf, np.log(4.0)])
    grid = (np.arange(800) + 0.5) / 800.0
    assert np.bincount([o.sample_row(x, v)[0] for v in grid], minlength=4).tolist() == [100, 300, 0, 400]


def test_truncations():
    x = np.log(np.array([4.0, 1.0, 8.0, 4.0, 2.0, 1.0]))          # of 20
    kept = lambda **k: np.flatnonzero(o.kept_weights(x, **k)).tolist()
    assert kept(top_k=2) == [0, 2] and kept(top_k=3) == [0, 2, 3] and kept(top_k=9) == [0, 1, 2, 3, 4, 5]
    assert kept(top_p=0.39) == [2] and kept(top_p=0.41) == [0, 2] and kept(top_p=0.79) == [0, 2, 3]
    assert kept(top_k=2, top_p=0.66) == [2] and kept(min_p=0.26) == [0, 2, 3] and kept(min_p=0.2) == [0, 2, 3, 4]
    assert kept(temperature=0.0) == [2] and o.sample_row(np.full(3, -np.inf), 0.5) == (-1, -np.inf)
