"""What the sampling and posterior operators of the engine are measured on.

Three operators over the candidates of a preselection (snickery_amd.engine.HipSearchEngine):

``sample_rows``      one draw per row of scores with temperature, top-k, top-p and min-p, from given random numbers;
``sample_paths``     draws of whole unit paths from exp(-cost / temperature) over the candidate trellis, the cost of a path
                     being its target costs, its join costs and a learned bias by buckets of the relative position of
                     consecutive units, every backward step truncated like a row of ``sample_rows``;
``path_posterior``   the log partition function of the same model with what its gradients need: the posterior of every
                     candidate and the expected uses of every bucket of the position bias.

``run`` computes them in their plain form (torch operations in 64 bits: a draw next to a border of its interval must fall
on the same side) or, where ``own`` is set, calls the engine.
"""
import math

import numpy as np
import torch

own = False

_SCORE_TYPES = {'float64': torch.float64, 'float32': torch.float32, 'float16': torch.float16, 'bfloat16': torch.bfloat16}
_NEVER = -1                       # padding of a candidate list
_VERY_BIG = 1000000000000000.0    # target cost of the padding

# sample_rows: `batch` rows of `size` scores, `draws` draws from each
# sample_paths / path_posterior: `batch` utterances of about `frames` rows, `size` candidates a row


def listed():
    return [
        # the candidates of a single frame: latency
        dict(name='rows_frame', op='rows', batch=1, size=30, draws=1, dtype='float64', temperature=0.7, top_k=0, top_p=1.0, min_p=0.0, padded=False),
        # one utterance, independently per frame
        dict(name='rows_utterance', op='rows', batch=600, size=100, draws=1, dtype='float64', temperature=0.5, top_k=0, top_p=0.9, min_p=0.0, padded=True),
        # a tune set of 32 utterances, eight renditions of each, every truncation at once
        dict(name='rows_tune_set', op='rows', batch=19200, size=100, draws=8, dtype='float64', temperature=0.8, top_k=40, top_p=0.95, min_p=0.02, padded=True),
        # scores over every unit of a small voice
        dict(name='rows_small_voice', op='rows', batch=37, size=50003, draws=1, dtype='float32', temperature=1.0, top_k=0, top_p=0.95, min_p=0.0, padded=False),
        # a batch of long rows in 16 bits
        dict(name='rows_16bit', op='rows', batch=128, size=131071, draws=1, dtype='bfloat16', temperature=0.9, top_k=50, top_p=0.9, min_p=0.0, padded=False),
        # one row over a voice of a million units
        dict(name='rows_large_voice', op='rows', batch=1, size=1048576, draws=4, dtype='float32', temperature=1.0, top_k=0, top_p=0.98, min_p=1e-4, padded=False),
        # a short phrase
        dict(name='paths_phrase', op='paths', batch=1, frames=120, size=30, columns=151, draws=1, temperature=0.5, top_k=0, top_p=1.0, min_p=0.0, classes=1, buckets=16),
        # a sentence at the headline configuration's width
        dict(name='paths_sentence', op='paths', batch=1, frames=600, size=100, columns=302, draws=1, temperature=0.3, top_k=0, top_p=0.95, min_p=0.0, classes=3, buckets=16),
        # renditions of a tune set
        dict(name='paths_tune_set', op='paths', batch=16, frames=600, size=100, columns=302, draws=4, temperature=0.5, top_k=20, top_p=0.9, min_p=0.01, classes=3, buckets=32),
        # one utterance of a training step
        dict(name='posterior_sentence', op='posterior', batch=1, frames=335, size=50, columns=302, temperature=0.5, classes=3, buckets=16),
        # a training step over a tune set
        dict(name='posterior_tune_set', op='posterior', batch=16, frames=600, size=100, columns=302, temperature=0.5, classes=3, buckets=32),
        # wide candidate lists
        dict(name='posterior_wide', op='posterior', batch=4, frames=300, size=200, columns=151, temperature=1.0, classes=1, buckets=16),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_truncation(rng, size):
    top_k = rng.choice([0, 0, 1, _log_uniform(rng, 1, max(size, 2))])
    top_p = rng.choice([1.0, 1.0, rng.uniform(0.05, 0.99), rng.uniform(0.8, 0.99)])
    min_p = rng.choice([0.0, 0.0, 10.0 ** rng.uniform(-4.0, -0.3)])
    return dict(temperature=math.exp(rng.uniform(math.log(0.2), math.log(2.0))), top_k=top_k, top_p=top_p, min_p=min_p)


def draw(rng):
    op = rng.choice(['rows', 'rows', 'paths', 'posterior'])
    if op == 'rows':
        size = _log_uniform(rng, 2, 1 << 20)
        batch = min(_log_uniform(rng, 1 if size > 4000 else 48, 19200), max(1, (1 << 23) // size))
        dtype = rng.choice(['float64', 'float32', 'float16', 'bfloat16'])
        return dict(op=op, batch=batch, size=size, draws=rng.choice([1, 1, 3, 8]), dtype=dtype, padded=rng.random() < 0.5, **_draw_truncation(rng, size))
    size = rng.choice([_log_uniform(rng, 1, 208), rng.randint(20, 120)])
    frames = _log_uniform(rng, 1, 1200)
    batch = max(1, min(_log_uniform(rng, 1, 16), 9600 * 100 * 100 // (frames * size * size)))
    case = dict(op=op, batch=batch, frames=frames, size=size, columns=rng.choice([9, 61, 151, 302]), classes=rng.choice([1, 3, 40]),
                buckets=rng.choice([1, 3, 16, 32, 64]))
    truncation = _draw_truncation(rng, size)
    if op == 'paths':
        case.update(draws=rng.choice([1, 1, 2, 4]), **truncation)
    else:
        case['temperature'] = truncation['temperature']
    return case


# ---------------------------------------------------------------------------------------------------------------- inputs
def _bucket_edges(buckets):
    """Steps of -1, 0 and +1 unit in buckets of their own as far as they go, the rest at growing distances either way."""
    order = [1, 2, 0, -1]
    far = 3
    while len(order) < buckets - 1:
        order += [far, -far]
        far = far * 2
    return np.array(sorted(order[:buckets - 1]), dtype=np.int64)


def _lengths(case):
    """Rows of each utterance: 0.6 to 1.4 times `frames` in turn, the last one takes what is left."""
    U, T = case['batch'], case['frames']
    lengths = np.maximum(1, (T * (0.6 + 0.8 * ((np.arange(U) * 0.618034) % 1.0))).astype(np.int64))
    lengths[-1] = max(1, U * T - int(lengths[:-1].sum()))
    return lengths


def _host_inputs(case, seed):
    """The inputs as numpy arrays, from the seed alone."""
    g = np.random.default_rng([seed, 71])
    if case['op'] == 'rows':
        R, V = case['batch'], case['size']
        if case['padded']:
            # scores of a candidate list in the order of its labels: minus its distances, short lists padded
            x = -(2.0 + 3.0 * g.random((R, V)) + 0.3 * g.random((R, 1)))
            short = g.random(R) < 0.1
            x[short, max(1, V // 2):] = -np.inf
        else:
            x = 2.5 * g.standard_normal((R, V), dtype=np.float32)
        return dict(scores=x, u=g.random((R, case['draws'])))
    U, K = case['batch'], case['size']
    lengths = _lengths(case)
    offsets = np.zeros(U + 1, dtype=np.int64)
    offsets[1:] = np.cumsum(lengths)
    rows = int(offsets[-1])
    n_units = 60000
    # the runs of natural speech in the candidate lists: a slot follows the unit after its last one or starts anew
    start = g.integers(0, n_units - 2000, (rows, K))
    fresh = g.random((rows, K)) < 0.35
    fresh[offsets[:-1]] = True
    t = np.arange(rows)[:, None]
    since = np.maximum.accumulate(np.where(fresh, t, -1), axis=0)
    cand = np.take_along_axis(start, since, axis=0) + (t - since)
    cand = np.take_along_axis(cand, np.argsort(g.random((rows, K)), axis=1), axis=1)
    dist = np.sort(1.0 + 2.0 * g.random((rows, K)), axis=1)
    short = np.flatnonzero(g.random(rows) < 0.05)
    cand[short, max(1, K - K // 4):] = _NEVER
    dist[short, max(1, K - K // 4):] = _VERY_BIG
    steps = g.standard_normal((n_units + 1, case['columns']), dtype=np.float32)
    walk = np.cumsum(steps, axis=0, dtype=np.float32)
    walk -= walk.mean(axis=0)
    walk /= walk.std()
    bias = 0.4 * g.standard_normal((case['classes'], case['buckets']))
    edges = _bucket_edges(case['buckets'])
    repeat = int(np.searchsorted(edges, 0, side='right'))
    if case['buckets'] >= 16:
        bias[0, repeat] = np.inf              # class 0 never joins a unit to itself
    out = dict(cand=cand.astype(np.int64), dist=dist, offsets=offsets, join=walk, wj=0.05 + 0.1 * g.random(case['columns']),
               bias=bias, edges=edges, classes=g.integers(0, case['classes'], rows).astype(np.int32))
    if case['op'] == 'paths':
        out['u'] = g.random((case['draws'], rows))
    return out


def prepare(case, seed):
    host = _host_inputs(case, seed)
    state = dict(case=case)
    if own:
        from snickery_amd.engine import HipSearchEngine
        state['engine'] = HipSearchEngine(torch.cuda.current_device())
    if case['op'] == 'rows':
        state['scores'] = torch.from_numpy(host['scores']).to('cuda').to(_SCORE_TYPES[case['dtype']])
        state['u'] = torch.from_numpy(host['u']).to('cuda')
        return state
    for name in ('cand', 'dist', 'classes'):
        state[name] = torch.from_numpy(host[name]).to('cuda')
    if case['op'] == 'paths':
        state['u'] = torch.from_numpy(host['u']).to('cuda')
    state['offsets'] = host['offsets']
    if own:
        state['engine'].upload_join_only(host['join'])
        state['engine'].set_weights(None, host['wj'])
        state['engine'].set_position_bias(host['bias'], host['edges'])
    else:
        state['join'] = torch.from_numpy(host['join']).to('cuda')
        for name in ('wj', 'bias', 'edges'):
            state[name] = torch.from_numpy(host[name]).to('cuda')
    return state


# ------------------------------------------------------------------------------------------------------------ plain forms
def _plain_draw(x, u, temperature, top_k, top_p, min_p):
    """One draw per entry of u (R, S) from each row of scores x (R, V), 64 bits: (index, log probability)."""
    x = torch.where(torch.isnan(x), -math.inf, x.double())
    V = x.shape[1]
    top = x.max(dim=1, keepdim=True).values
    empty = top == -math.inf
    w = torch.where(x == top, 1.0, torch.exp((x - top) / temperature))
    w = torch.where(x == -math.inf, 0.0, w)
    if top_k > 0 or top_p < 1.0:
        order = torch.sort(x, dim=1, descending=True, stable=True).indices
        ws = torch.gather(w, 1, order)
        if 0 < top_k < V:
            ws[:, top_k:] = 0.0
        if top_p < 1.0:
            mass = torch.cumsum(ws, 1)
            before = torch.cat([torch.zeros_like(mass[:, :1]), mass[:, :-1]], 1)
            ws = torch.where(before < top_p * mass[:, -1:], ws, 0.0)
        w = torch.zeros_like(w).scatter(1, order, ws)
    if min_p > 0.0:
        w = torch.where(w >= min_p, w, 0.0)
    mass = torch.cumsum(w, 1)
    total = mass[:, -1:]
    index = torch.searchsorted(mass, u * total, right=True)
    index = torch.minimum(index, torch.searchsorted(mass, total.expand_as(u).contiguous()))
    index = torch.where(empty, 0, index)
    logp = torch.log(torch.gather(w, 1, index)) - torch.log(total)
    return torch.where(empty, -1, index), torch.where(empty, -math.inf, logp)


def _plain_costs(s):
    """(rows, K, K) join cost + position bias between rows r and r + 1, in 64 bits; +inf where a unit cannot join."""
    cand, join, wj, edges, bias = s['cand'], s['join'], s['wj'], s['edges'], s['bias']
    rows, K = cand.shape
    n = join.shape[0] - 1
    usable = (cand >= 1) & (cand < n - 1)
    safe = torch.where(usable, cand, 0)
    cost = torch.full((rows, K, K), math.inf, dtype=torch.float64, device=cand.device)
    step = max(1, (1 << 27) // (K * K * join.shape[1]))
    for r in range(0, rows - 1, step):
        e = min(r + step, rows - 1)
        ends = join[safe[r:e] + 1].double() * wj
        starts = join[safe[r + 1:e + 1]].double() * wj
        c = torch.sqrt(torch.square(ends[:, :, None, :] - starts[:, None, :, :]).sum(-1))
        apart = cand[r + 1:e + 1][:, None, :] - cand[r:e][:, :, None]
        bucket = torch.zeros_like(apart)
        for edge in edges:
            bucket += apart >= edge
        c = c + torch.gather(bias[s['classes'][r:e].long()], 1, bucket.view(e - r, K * K)).view(e - r, K, K)
        ok = usable[r:e][:, :, None] & usable[r + 1:e + 1][:, None, :]
        cost[r:e] = torch.where(ok, c, math.inf)
    return cost, usable


def _lse(x, dim):
    top = x.max(dim=dim, keepdim=True).values
    base = torch.where(top == -math.inf, 0.0, top)
    return (base + torch.log(torch.exp(x - base).sum(dim, keepdim=True))).squeeze(dim)


def _pad(x, offsets, fill):
    """(rows, ...) -> (utterances, longest, ...)"""
    lengths = np.diff(offsets)
    out = torch.full((len(lengths), int(lengths.max())) + tuple(x.shape[1:]), fill, dtype=x.dtype, device=x.device)
    for i in range(len(lengths)):
        out[i, :int(lengths[i])] = x[int(offsets[i]):int(offsets[i + 1])]
    return out


def _plain_forward(s, temperature):
    cost, usable = _plain_costs(s)
    offsets = s['offsets']
    local = torch.where(usable, -s['dist'] / temperature, -math.inf)
    local, step = _pad(local, offsets, -math.inf), _pad(-cost / temperature, offsets, -math.inf)
    longest = local.shape[1]
    alpha = torch.empty_like(local)
    alpha[:, 0] = local[:, 0]
    for t in range(1, longest):
        alpha[:, t] = local[:, t] + _lse(alpha[:, t - 1][:, :, None] + step[:, t - 1], 1)
    return cost, local, step, alpha


def _plain_paths(s):
    case, offsets, u = s['case'], s['offsets'], s['u']
    temperature = case['temperature']
    cost, local, step, alpha = _plain_forward(s, temperature)
    device = u.device
    lengths = torch.from_numpy(np.diff(offsets)).to(device)
    first = torch.from_numpy(offsets[:-1].copy()).to(device)
    U, longest, K = local.shape
    S = u.shape[0]
    each = torch.arange(U, device=device)
    slot = torch.zeros((S, U), dtype=torch.int64, device=device)
    slots = torch.zeros((longest, S, U), dtype=torch.int64, device=device)
    logp = torch.zeros((S, U), dtype=torch.float64, device=device)
    rows = s['cand'].shape[0]
    for t in range(longest - 1, -1, -1):
        here = lengths > t
        last = lengths == t + 1
        x = alpha[:, t].expand(S, U, K)
        if t + 1 < longest:
            x = torch.where(last[None, :, None], x, x + step[each[None, :].expand(S, U), t, :, slot])
        row = torch.clamp(first + t, max=rows - 1)
        i, lp = _plain_draw(x.reshape(S * U, K), u[:, row].reshape(S * U, 1), temperature=1.0, top_k=case['top_k'], top_p=case['top_p'], min_p=case['min_p'])
        slot = torch.where(here, torch.clamp(i.view(S, U), min=0), slot)
        logp = torch.where(here, logp + lp.view(S, U), logp)
        slots[t] = slot
    dead = torch.isinf(alpha[each, lengths - 1].max(dim=1).values)
    path = torch.empty((S, rows), dtype=torch.int64, device=device)
    total = torch.empty((S, U), dtype=torch.float64, device=device)
    for v in range(U):
        a, b = int(offsets[v]), int(offsets[v + 1])
        k = slots[:b - a, :, v].T                                       # (S, T)
        r = torch.arange(a, b, device=device)
        path[:, a:b] = torch.where(dead[v], -1, s['cand'][r, k])
        total[:, v] = s['dist'][r, k].sum(1) + cost[r[:-1], k[:, :-1], k[:, 1:]].sum(1)
    return path, torch.where(dead, math.inf, total), torch.where(dead, -math.inf, logp)


def _plain_posterior(s):
    case, offsets = s['case'], s['offsets']
    temperature = case['temperature']
    cost, local, step, alpha = _plain_forward(s, temperature)
    device = cost.device
    lengths = torch.from_numpy(np.diff(offsets)).to(device)
    U, longest, K = local.shape
    each = torch.arange(U, device=device)
    beta = torch.zeros_like(local)
    for t in range(longest - 2, -1, -1):
        into = local[:, t + 1] + beta[:, t + 1]
        beta[:, t] = torch.where((lengths > t + 1)[:, None], _lse(step[:, t] + into[:, None, :], 2), 0.0)
    logz = _lse(alpha[each, lengths - 1], 1)
    base = torch.where(logz == -math.inf, math.inf, logz)
    unit = torch.exp(alpha + beta - base[:, None, None])
    rows = s['cand'].shape[0]
    posterior = torch.empty((rows, K), dtype=torch.float64, device=device)
    C, B = s['bias'].shape
    uses = torch.zeros((C, B), dtype=torch.float64, device=device)
    chunk = max(1, (1 << 24) // (K * K))
    for v in range(U):
        a, b = int(offsets[v]), int(offsets[v + 1])
        posterior[a:b] = unit[v, :b - a]
        for t in range(0, b - a - 1, chunk):
            e = min(t + chunk, b - a - 1)
            into = local[v, t + 1:e + 1] + beta[v, t + 1:e + 1]
            pair = torch.exp(alpha[v, t:e, :, None] + step[v, t:e] + into[:, None, :] - base[v])
            apart = s['cand'][a + t + 1:a + e + 1][:, None, :] - s['cand'][a + t:a + e][:, :, None]
            bucket = torch.zeros_like(apart)
            for edge in s['edges']:
                bucket += apart >= edge
            per_row = torch.stack([torch.where(bucket == i, pair, 0.0).sum((1, 2)) for i in range(B)], 1)
            member = s['classes'][a + t:a + e].long()[None, :] == torch.arange(C, device=device)[:, None]
            uses += member.double() @ per_row
    return logz, posterior, uses


def run(state):
    case = state['case']
    if case['op'] == 'rows':
        how = dict(temperature=case['temperature'], top_k=case['top_k'], top_p=case['top_p'], min_p=case['min_p'])
        if own:
            return state['engine'].sample_rows(state['scores'], state['u'], **how)
        return _plain_draw(state['scores'], state['u'], **how)
    if case['op'] == 'paths':
        if own:
            return state['engine'].sample_paths(state['cand'], state['dist'], state['u'], row_offsets=state['offsets'],
                                                join_class=state['classes'], temperature=case['temperature'],
                                                top_k=case['top_k'], top_p=case['top_p'], min_p=case['min_p'])
        return _plain_paths(state)
    if own:
        return state['engine'].path_posterior(state['cand'], state['dist'], row_offsets=state['offsets'],
                                              join_class=state['classes'], temperature=case['temperature'])
    return _plain_posterior(state)


def work(case):
    if case['op'] == 'rows':
        n = case['batch'] * case['size']
        width = torch.empty((), dtype=_SCORE_TYPES[case['dtype']]).element_size()
        # a subtraction, a scaling, an exponential and a sum per score, a comparison per draw
        return dict(bytes=n * width + case['batch'] * case['draws'] * 24, flops=4 * n + n * case['draws'])
    rows, K, D = int(_lengths(case).sum()), case['size'], case['columns']
    cells = max(rows - case['batch'], 0) * K * K
    units = min(2 * rows * K, 60001)                        # join rows touched: each once
    out = dict(bytes=rows * K * 16 + rows * 4 + units * D * 4, flops=cells * (3 * D + 6))
    if case['op'] == 'paths':
        out['bytes'] += case['draws'] * rows * 16
        out['flops'] += 5 * case['draws'] * rows * K
    else:
        out['bytes'] += rows * K * 8
        out['flops'] += 8 * cells
    return out


# ------------------------------------------------------------------------------------------------------- in 64 bits, apart
def _exact_keep(x, temperature, top_k, top_p, min_p):
    """Weights of the scores x that the truncations leave, relative to the largest; None for a row without any."""
    x = np.asarray(x, dtype=np.float64)
    alive = np.flatnonzero(~np.isnan(x) & (x != -np.inf))
    if alive.size == 0:
        return None
    best = x[alive].max()
    with np.errstate(invalid='ignore', over='ignore'):
        w = np.exp((x[alive] - best) / temperature)
    w[x[alive] == best] = 1.0
    ranked = np.argsort(-x[alive], kind='stable')
    if top_k > 0:
        ranked = ranked[:top_k]
    if top_p < 1.0:
        cum = np.cumsum(w[ranked])
        ranked = ranked[:int(np.searchsorted(cum, top_p * cum[-1], side='left')) + 1]
    keep = np.zeros(x.size)
    keep[alive[ranked]] = w[ranked]
    keep[keep < min_p] = 0.0
    return keep


def _exact_pick(keep, u):
    cum = np.cumsum(keep)
    i = int(np.searchsorted(cum, u * cum[-1], side='right'))
    while i >= keep.size or keep[i] == 0.0:
        i -= 1
    return i, math.log(keep[i]) - math.log(cum[-1])


def _exact_trellis(case, host):
    """Costs between consecutive rows and the usable candidates, by differences of the weighted join rows."""
    cand, offsets = host['cand'], host['offsets']
    n = host['join'].shape[0] - 1
    usable = (cand >= 1) & (cand < n - 1)
    table = torch.from_numpy(host['join'].astype(np.float64) * host['wj'])
    lowest = torch.from_numpy(np.where(usable, cand, 0))
    cost = []
    for r in range(cand.shape[0] - 1):
        d = torch.cdist(table[lowest[r] + 1], table[lowest[r + 1]], compute_mode='donot_use_mm_for_euclid_dist').numpy()
        bucket = np.searchsorted(host['edges'], cand[r + 1][None, :] - cand[r][:, None], side='right')
        d = d + host['bias'][host['classes'][r]][bucket]
        d[~usable[r]] = np.inf
        d[:, ~usable[r + 1]] = np.inf
        cost.append((d, bucket))
    return cost, usable


def _np_lse(x, axis):
    top = np.max(x, axis=axis, keepdims=True)
    top[np.isinf(top)] = 0.0
    with np.errstate(divide='ignore'):
        return np.squeeze(top, axis) + np.log(np.exp(x - top).sum(axis))


def exact(case, seed):
    if case['op'] == 'rows':
        n = case['batch'] * case['size']
        if n > 1 << 25:
            return None
        host = _host_inputs(case, seed)
        x = torch.from_numpy(host['scores']).to(_SCORE_TYPES[case['dtype']]).double().numpy()
        index = np.full(host['u'].shape, -1, dtype=np.int64)
        logp = np.full(host['u'].shape, -np.inf)
        for r in range(case['batch']):
            keep = _exact_keep(x[r], case['temperature'], case['top_k'], case['top_p'], case['min_p'])
            if keep is not None:
                for j in range(case['draws']):
                    index[r, j], logp[r, j] = _exact_pick(keep, host['u'][r, j])
        return index, logp
    rows, K = int(_lengths(case).sum()), case['size']
    if rows * K * K * case['columns'] > 6e9 or rows * K * K > 4e7:
        return None
    host = _host_inputs(case, seed)
    cost, usable = _exact_trellis(case, host)
    cand, dist, offsets, tau = host['cand'], host['dist'], host['offsets'], case['temperature']
    U = len(offsets) - 1
    if case['op'] == 'paths':
        S = case['draws']
        paths = np.full((S, cand.shape[0]), -1, dtype=np.int64)
        total, logq = np.full((S, U), np.inf), np.full((S, U), -np.inf)
    else:
        logz, posterior = np.full(U, -np.inf), np.zeros(cand.shape)
        uses = np.zeros(host['bias'].shape)
    for v in range(U):
        a, b = int(offsets[v]), int(offsets[v + 1])
        local = np.where(usable[a:b], -dist[a:b] / tau, -np.inf)
        alpha = [local[0]]
        for t in range(1, b - a):
            alpha.append(local[t] + _np_lse(alpha[-1][:, None] - cost[a + t - 1][0] / tau, 0))
        z = float(_np_lse(alpha[-1][None, :], 1)[0])
        if z == -np.inf:
            continue
        if case['op'] == 'posterior':
            logz[v] = z
            beta = np.zeros(K)
            posterior[b - 1] = np.exp(alpha[-1] - z)
            for t in range(b - a - 2, -1, -1):
                c, bucket = cost[a + t]
                x = -c / tau + (local[t + 1] + beta)[None, :]
                pair = np.exp(alpha[t][:, None] + x - z)
                uses[host['classes'][a + t]] += np.bincount(bucket.ravel(), pair.ravel(), minlength=uses.shape[1])
                beta = _np_lse(x, 1)
                posterior[a + t] = np.exp(alpha[t] + beta - z)
            continue
        for j in range(S):
            x, spent, lq, after = alpha[-1], 0.0, 0.0, None
            for t in range(b - a - 1, -1, -1):
                if after is not None:
                    x = alpha[t] - cost[a + t][0][:, after] / tau
                keep = _exact_keep(x, 1.0, case['top_k'], case['top_p'], case['min_p'])
                k, lp = _exact_pick(keep, host['u'][j, a + t])
                lq += lp
                spent += dist[a + t, k] + (cost[a + t][0][k, after] if after is not None else 0.0)
                paths[j, a + t] = cand[a + t, k]
                after = k
            total[j, v], logq[j, v] = spent, lq
    return (paths, total, logq) if case['op'] == 'paths' else (logz, posterior, uses)
