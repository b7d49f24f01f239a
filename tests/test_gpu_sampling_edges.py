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
