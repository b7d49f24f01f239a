"""The position bias' training loop on the CPU, with the path model of oracle/sampling_oracle.py in the engine's place."""
import numpy as np
import pytest

import sampling_oracle as o
from snickery_amd.train_position_bias import bias_step, train_position_bias


class OracleEngine(object):
    def __init__(self, JC, wj):
        self.JC, self.wj, self.bias, self.edges = JC, wj, None, ()

    def path_posterior(self, cand, dist, row_offsets, join_class, temperature):
        logz, uses = [], np.zeros(self.bias.shape)
        for a, b in zip(row_offsets[:-1], row_offsets[1:]):
            z, _, n = o.posterior(cand[a:b], dist[a:b], temperature, self.JC, self.wj, self.bias, self.edges, None if join_class is None else join_class[a:b])
            logz.append(z)
            uses += n
        return np.array(logz), None, uses


class StubSynthesiser(object):
    def __init__(self, temperature=0.7, n_utts=3):
        rng = np.random.RandomState(0)
        self.config = {'unit_sampling': {'temperature': temperature}}
        self.engine = OracleEngine(rng.randn(101, 4).astype(np.float32), 0.3 * np.ones(4))
        self.utts = {}
        for i in range(n_utts):
            cand = rng.randint(1, 99, (8 + i, 5))
            for t in range(1, len(cand)):
                cand[t, :2] = np.minimum(cand[t - 1, 2:4] + [0, 1], 98)
            self.utts['u%d' % i] = (cand, rng.rand(8 + i, 5))
        self.classes = None

    def get_sentence_set(self, which):
        assert which == 'tune'
        return sorted(self.utts)

    def prepare_targets(self, name, synth_type, return_names):
        return name, ['/'.join(['x'] * 2 + ['ab'[t % 2]] + ['x'] * 2) for t in range(len(self.utts[name][0]))]

    def preselect_units(self, features, names):
        return self.utts[features]

    def set_position_bias(self, bias, edges, classes=None):
        self.engine.bias, self.engine.edges, self.classes = np.array(bias), np.array(edges), classes

    def join_classes(self, names, rows):
        return None if self.classes is None else np.array([self.classes.get(n.split('/')[2], -1) for n in names], dtype=np.int32)


@pytest.mark.parametrize('classes', [None, {'a': 0, 'b': 1}])
def test_training_runs(classes):
    s, lines = StubSynthesiser(), []
    res = train_position_bias(s, [0.2, 0.0, 0.6, 0.2], [0, 1, 2], classes, max_epochs=6, report=lines.append)
    n = 2 if classes else 1
    assert res['bias'].shape == (n, 4) and len(res['losses']) == 6 and np.all(np.isfinite(res['losses']))
    assert np.all(np.isinf(res['bias'][:, 1])) and np.all(np.isfinite(np.delete(res['bias'], 1, axis=1)))
    assert np.all(np.delete(res['bias'], 1, axis=1).min(axis=1) == 0.0)
    assert np.array_equal(s.engine.bias, res['bias']) and 'position_bias = ' in lines[-1]
    assert np.all(res['uses'][:, 1] == 0.0)              # the forbidden step is on no path


def test_gradient_against_differences():
    """Of F = sum of temperature logZ + n goal bias, by central differences: their error is h^2 / 6 times a third derivative
    (at most the third power of the number of joins over temperature^2) plus F's rounding over h."""
    s, tau, h = StubSynthesiser(), 0.7, 2.0 ** -12
    cand, dist = s.utts['u0']
    offs, goals = np.array([0, len(cand)]), np.array([[0.1, 0.2, 0.5, 0.2]])
    bias = np.array([[0.3, -0.2, 0.1, 0.0]])
    joins = len(cand) - 1

    def F(b):
        s.set_position_bias(b, [0, 1, 2])
        return tau * s.engine.path_posterior(cand, dist, offs, None, tau)[0].sum() + joins * (goals * b).sum()
    s.set_position_bias(bias, [0, 1, 2])
    uses = s.engine.path_posterior(cand, dist, offs, None, tau)[2]
    moved, gradient = bias_step(bias, uses, goals, tau, 0.5)
    for k in range(4):
        e = np.zeros((1, 4))
        e[0, k] = h
        assert abs((F(bias + e) - F(bias - e)) / (2.0 * h) - gradient[0, k]) <= h * h / 6.0 * joins ** 3 / tau ** 2 + 2.0 ** -45 / h
    # the step goes down the gradient: a bucket that is used more than its goal becomes dearer
    assert np.all((moved - bias) * gradient <= 0.0)
    assert np.array_equal(bias_step(bias, np.zeros((1, 4)), goals, tau, 0.5)[0], bias)


def test_refusals():
    s = StubSynthesiser()
    for goals in ([0.5, 0.5], [[0.2] * 4] * 3, [-0.1, 0.5, 0.3, 0.3], [0.0] * 4):
        with pytest.raises(ValueError):
            train_position_bias(s, goals, [0, 1, 2])
    with pytest.raises(ValueError):
        train_position_bias(StubSynthesiser(temperature=0.0), [0.25] * 4, [0, 1, 2])
    with pytest.raises(ValueError):
        train_position_bias(StubSynthesiser(n_utts=0), [0.25] * 4, [0, 1, 2])


def test_bucket_edges():
    from snickery_amd import hostprep as hp
    assert hp.position_bucket_edges(4, 10) == [0, 1, 2]
    for n, far in ((5, 10), (8, 100), (16, 1000), (64, 10 ** 6), (12, 3)):
        e = hp.position_bucket_edges(n, far)
        assert len(e) == n - 1 and all(a < b for a, b in zip(e, e[1:])) and set([0, 1, 2]) <= set(e)
    with pytest.raises(ValueError):
        hp.position_bucket_edges(3, 10)


@pytest.mark.parametrize('classes', [None, {'a': 0, 'b': 1, 'never': 2}])
def test_a_bucket_that_no_candidate_offers_stays_where_it_is(classes):
    """Units lie up to 97 apart here: steps beyond 500 are in no path."""
    s, lines = StubSynthesiser(), []
    goals = [0.2, 0.1, 0.3, 0.15, 0.25]
    res = train_position_bias(s, goals, [0, 1, 2, 500], classes, max_epochs=40, rate=0.8, thresh=1e-2, report=lines.append)
    n = 3 if classes else 1
    assert res['bias'].shape == (n, 5) and np.all(res['bias'][:, 4] == 0.0) and np.all(np.isfinite(res['bias'])) and np.abs(res['bias']).max() < 20.0
    assert np.all(res['bias'][:2, :4].min(axis=1) == 0.0)
    assert sum('no candidates offer bucket 4' in l for l in lines) == n
    if classes:                                          # a class on no join: nothing learned
        assert not res['bias'][2].any()
    wanted = np.array(goals[:4]) / sum(goals[:4])
    shares = res['uses'][0] / res['uses'][0].sum()
    assert np.abs(shares[:4] - wanted).max() <= res['losses'][-1] + 1e-12 and shares[4] == 0.0


def test_edges_of_a_setting():
    from snickery_amd import hostprep as hp
    from snickery_amd.train_position_bias import goals_and_edges
    assert goals_and_edges({'goals': [0.5, 0.5], 'edges': [1]}) == ([0.5, 0.5], [1])
    for goals in ([0.125] * 8, [[0.125] * 8] * 2):
        g, edges = goals_and_edges({'goals': goals, 'max_distance': 90})
        assert g == goals and edges == hp.position_bucket_edges(8, 90) and len(edges) == 7
    s = StubSynthesiser()
    res = train_position_bias(s, *goals_and_edges({'goals': [0.1, 0.1, 0.2, 0.3, 0.2, 0.1], 'max_distance': 40}), max_epochs=3, report=lambda line: None)
    assert res['bias'].shape == (1, 6) and res['edges'] == hp.position_bucket_edges(6, 40)
    for bad in ({'goals': [0.5, 0.5]}, {'goals': [0.5, 0.5], 'edges': [1], 'max_distance': 9}, {'goals': [0.5] * 3, 'max_distance': 9}):
        with pytest.raises(ValueError):
            goals_and_edges(bad)
