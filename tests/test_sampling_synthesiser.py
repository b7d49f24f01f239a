"""Draws through the Synthesiser on the CPU, with oracle/sampling_oracle.py in the engine's place."""
import numpy as np
import pytest

import sampling_oracle as o


class OracleEngine(object):
    def __init__(self, JC, wj):
        self.JC, self.wj = JC, wj

    def sample_rows(self, scores, u, **rule):
        return o.sample_rows(scores, u, **rule)

    def sample_paths(self, cand, dist, u, row_offsets, join_class, **rule):
        draws = [[o.sample_path(cand[a:b], dist[a:b], s[a:b], JC=self.JC, wj=self.wj, **rule) for a, b in zip(row_offsets[:-1], row_offsets[1:])] for s in u]
        return (np.array([np.concatenate([p for p, _, _ in d]) for d in draws]), np.array([[c for _, c, _ in d] for d in draws]),
                np.array([[l for _, _, l in d] for d in draws]))


@pytest.fixture
def synth():
    from snickery_amd.synthesiser import Synthesiser
    rng = np.random.RandomState(0)
    s = Synthesiser.__new__(Synthesiser)
    s.join_contexts_unweighted = rng.randn(61, 4).astype(np.float32)
    s.engine = OracleEngine(s.join_contexts_unweighted, 0.3 * np.ones(4))
    s.config = {'unit_sampling': {'temperature': 0.5, 'seed': 2}}
    s.verbose = False
    s.start_clock, s.stop_clock = (lambda comment: 0.0), (lambda start: None)
    return s


def test_the_cost_of_a_path_is_the_last_ones(synth):
    """Draws without joins have none: the cost of an earlier path does not stay."""
    rng = np.random.RandomState(1)
    cand, dist = rng.randint(1, 58, (7, 5)), rng.rand(7, 5)
    path = synth.draw_paths(['a'], [cand], [dist], [None])[0]
    slots = [int(np.flatnonzero(cand[t] == path[t])[0]) for t in range(7)]
    assert len(path) == 7 and synth.last_path_cost > dist[np.arange(7), slots].sum()
    synth.config['unit_sampling']['joins'] = False
    path = synth.draw_paths(['a'], [cand], [dist], [None])[0]
    assert len(path) == 7 and synth.last_path_cost is None


def test_candidates_without_a_finite_target_cost_are_not_drawn(synth):
    """With joins or without: the same candidates take part."""
    cand = np.array([[3, 4, 5], [6, 7, 8], [0, 9, 59]])
    dist = np.array([[0.1, -np.inf, np.nan], [np.inf, np.nan, -np.inf], [0.0, 0.2, 0.0]])
    u = np.random.RandomState(0).rand(4, 3)
    units = synth.sample_units(cand, dist, u)
    assert np.array_equal(units, np.repeat([[3, -1, 9]], 4, axis=0))
    assert np.all(synth.sample_search(cand, dist, u, row_offsets=[0, 1, 2, 3])[0] == units)
