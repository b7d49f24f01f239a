#!/usr/bin/env python3
"""Learns the position bias of a voice (Synthesiser.set_position_bias): how dear it is to follow a unit by itself, by its natural
successor, by a unit further on or further back in the corpus.

The reference reads forbid_repetition / forbid_regression (script/synth_halfphone.py:3215-3216) without an effect; here the shares
of the joins that are to fall into every bucket are given (``position_goals``) and the bias is fitted to them over the tune set.
With Z the partition function of the path model exp(-cost / temperature) and n the joins of a class,

    F(bias) = sum over the utterances of temperature * log Z  +  sum over classes and buckets of n * goal * bias

is convex, and its gradient is n * goal - uses, `uses` being the expected uses of a bucket that engine.path_posterior returns.
Every iteration moves a bias by rate * temperature * log(uses / (n * goal)), a scaled step down that gradient; a bucket whose goal is
0 is forbidden (+inf).  A bucket that no two candidates of the tune set offer stays at 0, and its goal goes to the others of its class in
proportion: nothing is to be learned of it, and F would have its bias fall without end.

    position_goals = {'edges': [0, 1, 2], 'goals': [0.1, 0.0, 0.7, 0.2], 'classes': {...}}       # goals: a list, or one per class
    position_goals = {'max_distance': 1000, 'goals': [0.02, 0.03, 0.05, 0.0, 0.6, 0.15, 0.1, 0.05]}   # edges by hostprep.position_bucket_edges
    unit_sampling = {'temperature': 0.5}

    python -m snickery_amd.train_position_bias -c voice.cfg
"""
from argparse import ArgumentParser

import numpy as np

from . import hostprep as hp


def goals_and_edges(settings):
    """Goals and edges of a position_goals setting: its own edges, or as many buckets as it has goals up to its max_distance."""
    goals, edges = settings['goals'], settings.get('edges')
    if (edges is None) == ('max_distance' not in settings):
        raise ValueError('position_goals: either edges or max_distance')
    return goals, hp.position_bucket_edges(np.shape(goals)[-1], settings['max_distance']) if edges is None else edges


def bias_step(bias, uses, goals, temperature, rate, floor=1e-6):
    """One iteration: the moved bias and the gradient n goal - uses of F at the old one.  A share below `floor` counts as that, which
    bounds the step of a bucket that is hardly used; a class without joins stays as it is."""
    n = uses.sum(axis=1, keepdims=True)
    gradient = n * goals - uses
    share = np.where(n > 0.0, uses / np.where(n > 0.0, n, 1.0), goals)
    with np.errstate(divide='ignore'):
        step = rate * temperature * (np.log(np.maximum(share, floor)) - np.log(np.maximum(goals, floor)))
    return np.where(goals > 0.0, bias + step, np.inf), gradient


def train_position_bias(synth, goals, edges, classes=None, n_tune=10, max_epochs=50, rate=0.5, thresh=1e-3, report=print):
    """Fits the bias of `synth` (a Synthesiser that preselects candidates) to `goals` (buckets,) or (classes, buckets) over the
    first n_tune sentences of the tune set, and leaves it set.  Returns a dict: bias, edges, classes, losses (largest distance
    of a share from its goal, per iteration), uses."""
    goals = np.atleast_2d(np.asarray(goals, dtype=np.float64))
    n_classes = 1 if not classes else max(classes.values()) + 1
    if goals.shape[0] == 1:
        goals = np.repeat(goals, n_classes, axis=0)
    if goals.shape != (n_classes, len(edges) + 1) or (goals < 0.0).any() or (goals.sum(axis=1) <= 0.0).any():
        raise ValueError('position goals: %d classes of %d shares expected' % (n_classes, len(edges) + 1))
    goals = goals / goals.sum(axis=1, keepdims=True)
    temperature = (synth.config.get('unit_sampling') or {}).get('temperature', 1.0)
    if not temperature > 0.0:
        raise ValueError('the path model needs a temperature above 0')
    cands, dists, names = [], [], []
    for f in synth.get_sentence_set('tune')[:n_tune]:
        U, w = synth.prepare_targets(f, 'tune', return_names=True)
        c, d = synth.preselect_units(U, w)
        cands.append(c); dists.append(d); names.append(w)
    if not cands:
        raise ValueError('the tune set is empty')
    offs = np.concatenate([[0], np.cumsum([len(c) for c in cands])]).astype(np.int64)
    cand, dist = np.vstack(cands), np.vstack(dists)

    bias = np.where(goals > 0.0, 0.0, np.inf)
    synth.set_position_bias(bias, edges, classes)
    per_utt = [synth.join_classes(w, len(c)) for w, c in zip(names, cands)]
    join_class = None if per_utt[0] is None else np.concatenate(per_utt)
    # At a temperature far above every cost all paths weigh the same: what is used there is what the candidates offer.
    offered = synth.engine.path_posterior(cand, dist, row_offsets=offs, join_class=join_class, temperature=1e100)[2] > 0.0
    wanted, goals = goals > 0.0, np.where(offered, goals, 0.0)
    for c, k in zip(*np.nonzero(wanted & ~offered)):
        report('## class %d: no candidates offer bucket %d' % (c, k))
    left = goals.sum(axis=1, keepdims=True)
    goals = goals / np.where(left > 0.0, left, 1.0)
    losses, uses = [], None
    for epoch in range(max_epochs):
        logz, _, uses = synth.engine.path_posterior(cand, dist, row_offsets=offs, join_class=join_class, temperature=temperature)
        if not np.isfinite(logz).any():
            raise ValueError('no utterance has a path under these goals')
        n = uses.sum(axis=1, keepdims=True)
        loss = float(np.abs(np.where(n > 0.0, uses / np.where(n > 0.0, n, 1.0) - goals, 0.0)).max())
        losses.append(loss)
        report('=== iteration %s | loss %s ===' % (epoch + 1, loss))
        if loss < thresh:
            break
        bias, _ = bias_step(bias, uses, goals, temperature, rate)
        # a constant over a class's buckets changes no probability: the smallest stays at 0
        least = np.where(np.isfinite(bias), bias, np.inf).min(axis=1, keepdims=True)
        bias = np.where(wanted & ~offered, 0.0, bias - np.where(np.isfinite(least), least, 0.0))
        synth.set_position_bias(bias, edges, classes)
    report('## Position bias found -- you can copy it to config.')
    report('position_bias = %s' % ({'bias': bias.tolist(), 'edges': [int(e) for e in edges], 'classes': classes},))
    return {'bias': bias, 'edges': list(edges), 'classes': classes, 'losses': losses, 'uses': uses}


def main(argv=None):
    a = ArgumentParser()
    a.add_argument('-c', dest='config_fname', required=True)
    a.add_argument('--device', type=int, default=0)
    opts = a.parse_args(argv)
    from .synthesiser import Synthesiser
    synth = Synthesiser(opts.config_fname, device=opts.device)
    try:
        how = synth.config['position_goals']
        goals, edges = goals_and_edges(how)
        train_position_bias(synth, goals, edges, how.get('classes'))
    finally:
        synth.close()


if __name__ == '__main__':
    main()
