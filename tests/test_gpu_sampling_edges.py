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
