"""Draws, the position bias and its training through the Synthesiser, as a user's configuration runs them."""
import numpy as np
import pytest

import sampling_oracle as o
from voice_fixture import build_halfphone_voice, build_voice

pytestmark = pytest.mark.gpu

SAMPLING = "\nunit_sampling = {'temperature': 0.4, 'top_k': 8, 'top_p': 0.9, 'min_p': 0.01, 'seed': 3}\n"
BIAS = "\nposition_bias = {'bias': [[0.3, float('inf'), -0.2, 0.1]], 'edges': [0, 1, 2]}\n"


def _voice(tmp_path, golden, extra):
    from snickery_amd.synthesiser import Synthesiser
    cfgfile, _ = build_voice(tmp_path, golden, greedy=False, multiepoch=1, n_candidates=12, extra_config=extra)
    return Synthesiser(cfgfile, verbose=False)


def _expected(synth, mini_voice, name, rule, bias=None, edges=()):
    U = synth.prepare_targets(name)
    cand, dist = synth.preselect_units_acoustic(U)
    u = synth._random_numbers(name, (1, len(cand)))[0]
    return o.sample_path(cand, dist, u, JC=mini_voice['JC_unw'], wj=mini_voice['wj'], bias=bias, edges=edges, **rule)


@pytest.mark.parametrize('extra', [SAMPLING, BIAS, SAMPLING + BIAS])
def test_synth_utt_draws_its_path(tmp_path, golden, mini_voice, extra):
    synth = _voice(tmp_path, golden, extra)
    rule = dict(temperature=0.4, top_k=8, top_p=0.9, min_p=0.01) if 'unit_sampling' in extra else dict(temperature=0.0)
    bias, edges = (np.array([[0.3, np.inf, -0.2, 0.1]]), [0, 1, 2]) if 'position_bias' in extra else (None, ())
    want, cost, _ = _expected(synth, mini_voice, 'arctic_b0001', rule, bias, edges)
    path = synth.synth_utt('arctic_b0001', synth_type='test')
    assert path == want.tolist() and all(isinstance(k, int) for k in path)
    assert abs(synth.last_path_cost - cost) <= 2.0 ** -50 * len(path) * abs(cost)
    assert synth.synth_utt('arctic_b0001', synth_type='test') == path             # the same seed, the same draw
    assert synth.synth_utts_bulk(['arctic_b0001', 'arctic_b0001'], synth_type='test') == [path, path]
    assert synth.synth_from_config()['arctic_b0001'] == path
    if bias is not None:
        assert all(b != a for a, b in zip(path, path[1:]))                         # repetition is forbidden
    synth.mode_of_operation = 'stream_weight_balancing'
    t, j = synth.synth_utt('arctic_b0001', synth_type='test')
    assert t.shape == (len(path), 2) and j.shape == (len(path) - 1, 4)
    synth.mode_of_operation = 'normal'
    if 'unit_sampling' in extra:
        drawn = set()
        for seed in range(6):
            synth.config['unit_sampling']['seed'] = seed
            drawn.add(tuple(synth.synth_utt('arctic_b0001', synth_type='test')))
        assert len(drawn) > 1
        synth.config['unit_sampling']['tempreature'] = 1.0
        with pytest.raises(ValueError):
            synth.synth_utt('arctic_b0001', synth_type='test')
    synth.close()


def test_rows_without_joins(tmp_path, golden, mini_voice):
    synth = _voice(tmp_path, golden, SAMPLING.replace("'seed': 3", "'seed': 3, 'joins': False"))
    U = synth.prepare_targets('arctic_b0001')
    cand, dist = synth.preselect_units_acoustic(U)
    u = synth._random_numbers('arctic_b0001', (1, len(cand)))[0]
    usable = (cand >= 1) & (cand < mini_voice['JC_unw'].shape[0] - 2)
    index, _ = o.sample_rows(np.where(usable, -dist, -np.inf), u[:, None], temperature=0.4, top_k=8, top_p=0.9, min_p=0.01)
    assert synth.synth_utt('arctic_b0001', synth_type='test') == np.take_along_axis(cand, index, axis=1)[:, 0].tolist()
    synth.close()


def test_settings_unset_keep_the_viterbi_search(tmp_path, golden, mini_voice):
    synth = _voice(tmp_path, golden, '')
    plain = synth.synth_utt('arctic_b0001', synth_type='test')
    cand, dist = synth.preselect_units_acoustic(synth.prepare_targets('arctic_b0001'))
    assert plain == synth.viterbi_search(cand, dist)
    synth.set_position_bias([[0.0, 0.0]], [1])               # a bias of nothing: the same cheapest path, through the draws
    assert synth.draws_paths() and synth.synth_utt('arctic_b0001', synth_type='test') == plain
    synth.set_position_bias(None)
    assert not synth.draws_paths() and synth.synth_utt('arctic_b0001', synth_type='test') == plain
    synth.close()


def test_training_then_drawing_with_classes(tmp_path, golden):
    from snickery_amd.synthesiser import Synthesiser
    from snickery_amd.train_position_bias import train_position_bias
    cfgfile, config, db = build_halfphone_voice(tmp_path, golden, 'monophone_then_acoustic')
    synth = Synthesiser(cfgfile, verbose=False)
    names = synth.get_sentence_set('test')
    synth.get_sentence_set = lambda which: names
    prepare = synth.prepare_targets
    synth.prepare_targets = lambda base, synth_type='test', **k: prepare(base, 'test', **k)
    synth.config['unit_sampling'] = {'temperature': 0.8, 'seed': 1}
    phones = sorted(set(n.split('/')[2] for n in synth.prepare_targets(names[0], return_names=True)[1]))
    classes = dict((p, i % 2) for i, p in enumerate(phones[:-1]))                   # one phone without a class
    res = train_position_bias(synth, [[0.2, 0.1, 0.5, 0.2], [0.3, 0.0, 0.4, 0.3]], [0, 1, 2], classes, max_epochs=8, report=lambda line: None)
    assert np.all(np.isfinite(res['losses'])) and np.isinf(res['bias'][1, 1]) and np.isfinite(res['bias'][0]).all()
    U, w = synth.prepare_targets(names[0], return_names=True)
    cand, dist = synth.preselect_units(U, w)
    cls = synth.join_classes(w, len(cand))
    assert set(cls.tolist()) >= set([-1, 0])
    u = synth._random_numbers(names[0], (1, len(cand)))
    path, cost, logp = synth.sample_search(cand, dist, u, join_class=cls)
    want, c, lp = o.sample_path(cand, dist, u[0], 0.8, synth.join_contexts_unweighted, synth._device_wj, res['bias'], [0, 1, 2], cls)
    assert np.array_equal(path[0], want)
    assert synth.synth_utt(names[0], synth_type='test') == (want.tolist() if (want >= 0).all() else [])
    # the whole voice's state travels to a replica
    other = Synthesiser(cfgfile, verbose=False)
    other._restore_runtime_state(synth._runtime_state())
    assert other.synth_utt(names[0], synth_type='test') == synth.synth_utt(names[0], synth_type='test')
    other.close()
    synth.close()
