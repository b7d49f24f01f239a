"""Refusals and sizes of the sampling entry points through the sanitizer build of `make asan-host` (no device, kernels never run: a
launch is a no-op, results read as zero).  Run by tests/test_sampling_refusals.py in a child process; prints SAMPLING-ASAN-OK."""
import ctypes
import os
import sys

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
assert os.environ.get('SNK_LIBRARY', '').endswith('libsnkhip_host_asan.so'), 'run through tests/test_sampling_refusals.py'
import snickery_amd                                   # noqa: E402
from snickery_amd import SnkError                     # noqa: E402
from snickery_amd.engine import load_library          # noqa: E402

lib = load_library()
rng = np.random.RandomState(0)


def refused(part, fn, *a, **k):
    """The call raises SnkError with `part` in its message."""
    try:
        fn(*a, **k)
    except SnkError as e:
        assert part in str(e), (part, str(e))
        return True
    return False


e = snickery_amd.HipSearchEngine(0)

# ---- rows of scores: no voice needed ----
x, u = rng.randn(5, 40), rng.rand(5, 3)
for dtype in ('float64', 'float32', 'float16'):
    i, lp = e.sample_rows(x.astype(dtype), u)
    assert i.shape == (5, 3) and lp.shape == (5, 3) and i.dtype == np.int64
assert e.sample_rows(x, u[:, 0])[0].shape == (5,)
e.sample_rows(x[:, 3:29], u)                          # a strided view
e.sample_rows(x[::2], u[::2])
e.sample_rows(x[::-1], u)                             # a negative stride is copied
e.sample_rows(x.T.copy().T, u)                        # columns apart
e.sample_rows(np.broadcast_to(x[0], (5, 40)), u)      # stride 0 is copied
e.sample_rows(x[:1], u[:1])
assert e.sample_rows(np.zeros((0, 4)), np.zeros((0, 2)))[0].shape == (0, 2)
big = rng.randn(300, 5000)                            # 12 MB through the staging
e.sample_rows(big[:, :4999], rng.rand(300), top_k=5)
for bad in (dict(temperature=-1.0), dict(temperature=np.nan), dict(temperature=np.inf), dict(top_k=-1), dict(top_p=0.0), dict(top_p=1.5),
            dict(top_p=np.nan), dict(min_p=-0.1), dict(min_p=1.1), dict(min_p=np.nan)):
    name = list(bad)[0]
    assert refused(name, e.sample_rows, x, u, **bad)
    rows = {name: np.full(5, 1.0)}
    rows[name][3] = bad[name]
    assert refused(name, e.sample_rows, x, u, **rows)
assert refused('whole number', e.sample_rows, x, u, top_k=2.5)
assert refused('whole number', e.sample_rows, x, u, top_k=np.array([1, 2, 2.5, 1, 1]))
assert refused('5 entries', e.sample_rows, x, u, top_p=np.ones(4))
assert refused('scores (R, V)', e.sample_rows, x[0], u)
assert refused('scores (R, V)', e.sample_rows, x, u[:4])
assert refused('scores (R, V)', e.sample_rows, x, u[:, :, None])
assert refused('scores of type', e.sample_rows, x.astype(np.int32), u)
assert refused('0 scores', e.sample_rows, np.zeros((5, 0)), u)
assert refused('0 draws', e.sample_rows, x, np.zeros((5, 0)))
for bad in (1.0, -1e-9, np.nan, np.inf):
    w = u.copy()
    w[2, 1] = bad
    assert refused('random number 7', e.sample_rows, x, w)


def p(a):
    return ctypes.c_void_p(a.ctypes.data)


index, logp = np.zeros((5, 3), np.int64), np.zeros((5, 3))
for fn in (lambda *a: lib.snk_sample_rows(*a), lambda *a: lib.snk_sample_rows_dev(*a, None, 0, None)):
    def call(scores=p(x), dtype=0, R=5, V=40, stride=40, u_=p(u), n=3, t=1.0, k=0, tp=1.0, mp=0.0, out=p(index), h=e._h):
        return fn(h, scores, dtype, R, V, stride, u_, n, t, k, tp, mp, None, out, p(logp))
    assert call() == 0
    assert call(R=0) == 0
    for bad in (dict(scores=None), dict(u_=None), dict(out=None), dict(dtype=4), dict(dtype=-1), dict(R=-1), dict(V=0), dict(V=(1 << 24) + 1), dict(stride=39),
                dict(n=0), dict(t=-1.0), dict(k=-1), dict(tp=0.0), dict(mp=2.0), dict(h=None)):
        assert call(**bad) != 0, bad
        assert lib.snk_last_error()

# ---- position bias ----
edges = [-5, 0, 1, 9]
e.set_position_bias(np.zeros((3, 5)), edges)
e.set_position_bias(np.zeros((1, 1)))
e.set_position_bias(np.full((2, 64), np.inf), np.arange(63))
assert refused('ascend', e.set_position_bias, np.zeros((3, 5)), [-5, 0, 0, 9])
assert refused('ascend', e.set_position_bias, np.zeros((3, 5)), [0, -5, 1, 9])
assert refused('buckets', e.set_position_bias, np.zeros((1, 65)), np.arange(64))
assert refused('expected', e.set_position_bias, np.zeros((3, 5)), edges[:3])
assert refused('expected', e.set_position_bias, np.zeros(5), edges)
assert refused('expected', e.set_position_bias, np.zeros((0, 5)), edges)
assert refused('bias 7', e.set_position_bias, np.where(np.arange(15).reshape(3, 5) == 7, np.nan, 0.0), edges)
assert refused('bias 7', e.set_position_bias, np.where(np.arange(15).reshape(3, 5) == 7, -np.inf, 0.0), edges)
assert refused('classes', e.set_position_bias, np.zeros((65536, 1)))
e.set_position_bias(None)

# ---- a caller's workspace for long rows ----
long_rows, lu, li = np.zeros((3, 20000)), np.full((3, 1), 0.5), np.zeros((3, 1), np.int64)
need = lib.snk_sample_rows_workspace(3, 20000)
assert need > 0 and lib.snk_sample_rows_workspace(3, 8192) == 0 and lib.snk_sample_rows_workspace(0, 20000) == 0
assert lib.snk_sample_rows_workspace(3, (1 << 24) + 1) == 0 and lib.snk_sample_rows_workspace(100000, 20000) < 3 << 30
room = np.zeros(need // 8 + 4)
first = room.ctypes.data + (-room.ctypes.data) % 16


def long_call(ws, n):
    return lib.snk_sample_rows_dev(e._h, p(long_rows), 0, 3, 20000, 20000, p(lu), 1, 1.0, 5, 0.9, 0.0, None, p(li), None, ws, n, None)


assert long_call(first, need) == 0 and long_call(None, 0) == 0
assert long_call(first + 8, need) != 0 and b'aligned' in lib.snk_last_error()
assert long_call(first, need - 1) != 0 and b'needed' in lib.snk_last_error()

# ---- trellis ----
T, K, N, Dj = 30, 12, 500, 21
cand, dist = rng.randint(0, N, (T, K)), rng.rand(T, K)
w = rng.rand(2, T)
assert refused('join_contexts', e.sample_paths, cand, dist, w)
e.upload_join_only(rng.randn(N + 1, Dj).astype(np.float32))
assert refused('weights', e.sample_paths, cand, dist, w)
assert refused('weights', e.path_posterior, cand, dist)
e.set_weights(None, np.full(Dj, 0.1))
offs = [0, 1, 11, 30]
for bias in (False, True):
    if bias:
        e.set_position_bias(np.zeros((2, 5)), edges)
    for o in (None, offs):
        n = 1 if o is None else 3
        path, cost, lp = e.sample_paths(cand, dist, w, row_offsets=o, join_class=np.zeros(T, np.int32))
        assert path.shape == (2, T) and cost.shape == (2, n) and lp.shape == (2, n)
        e.sample_paths(cand, dist, w, row_offsets=o, temperature=0.0)
        logz, post, uses = e.path_posterior(cand, dist, row_offsets=o)
        assert logz.shape == (n,) and post.shape == (T, K) and (uses.shape == (2, 5) if bias else uses is None)
for call in (lambda c, d, **k: e.sample_paths(c, d, k.pop('u', w), **k), lambda c, d, u=None, **k: e.path_posterior(c, d, **k)):
    assert refused('has no rows', call, cand, dist, row_offsets=[0, 5, 5, 30])
    assert refused('has no rows', call, cand, dist, row_offsets=[0, 9, 5, 30])
    assert refused('row_offsets[0]', call, cand, dist, row_offsets=[1, 30])
    assert refused('row_offsets', call, cand, dist, row_offsets=[0, 29])
    assert refused('row_offsets', call, cand, dist, row_offsets=[30])
    assert refused('8388609 rows', call, np.zeros((8388610, 1), np.int64), np.zeros((8388610, 1)), u=np.zeros((1, 8388610)), row_offsets=[0, 1, 8388610])
    assert refused('expected', call, cand[0], dist[0])
    assert refused('fit', call, cand, dist[:, :5])
    assert refused('fit', call, cand, dist, join_class=np.zeros(T - 1, np.int32))
    assert refused('outside 1..208', call, np.zeros((T, 209), np.int64), np.zeros((T, 209)))
    assert refused('outside 1..208', call, np.zeros((T, 0), np.int64), np.zeros((T, 0)))
    assert refused('temperature', call, cand, dist, temperature=-1.0)
    assert refused('temperature', call, cand, dist, temperature=np.nan)
    assert refused('temperature', call, cand, dist, temperature=np.inf)
assert refused('has no rows', e.path_posterior, cand[:0], dist[:0])
assert refused('temperature', e.path_posterior, cand, dist, temperature=0.0)
assert refused('expected', e.sample_paths, cand, dist, w[:, :-1])
assert refused('expected', e.sample_paths, cand, dist, w[0])
assert refused('0 draws', e.sample_paths, cand, dist, w[:0])
for bad in (dict(top_k=-1), dict(top_p=0.0), dict(min_p=2.0)):
    assert refused(list(bad)[0], e.sample_paths, cand, dist, w, **bad)
assert refused('random number', e.sample_paths, cand, dist, w + 1.0)
o64 = np.array([0, T], dtype=np.int64)
out, z, q, n = np.zeros((2, T), np.int64), np.zeros(2), np.zeros((T, K)), np.zeros((2, 5))
i64p = ctypes.POINTER(ctypes.c_int64)
cc, dd = cand.astype(np.int64), dist.astype(np.float64)
for tail in ((), (None,)):                             # host and device forms
    paths, posterior = (lib.snk_sample_paths_dev, lib.snk_path_posterior_dev) if tail else (lib.snk_sample_paths, lib.snk_path_posterior)

    def draw(c=p(cc), d=p(dd), o=o64.ctypes.data_as(i64p), u_=p(w), S=2, path=p(out), cost=p(z), h=e._h):
        return paths(h, c, d, o, 1, K, None, u_, S, 1.0, 0, 1.0, 0.0, path, cost, None, *tail)

    def prob(c=p(cc), d=p(dd), o=o64.ctypes.data_as(i64p), z_=p(z), q_=p(q), n_=p(n), h=e._h):
        return posterior(h, c, d, o, 1, K, None, 1.0, z_, q_, n_, *tail)
    assert draw() == 0 and prob() == 0 and prob(n_=None) == 0
    for bad in ('c', 'd', 'o', 'u_', 'path', 'cost', 'h'):
        assert draw(**{bad: None}) != 0, bad
    assert draw(S=0) != 0 and draw(S=65536) != 0
    for bad in ('c', 'd', 'o', 'z_', 'q_', 'h'):
        assert prob(**{bad: None}) != 0, bad
    e.set_position_bias(None)
    assert prob() != 0 and b'no position bias' in lib.snk_last_error()
    e.set_position_bias(np.zeros((2, 5)), edges)
# not under a batch in flight
F = rng.randn(N, 7).astype(np.float32)
e.upload_db(F, rng.randn(N + 1, Dj).astype(np.float32))
e.set_weights(np.ones(7), np.full(Dj, 0.1))
ticket = e.knn_viterbi_batch_submit([rng.randn(20, 7)], 10)
assert refused('in flight', e.sample_rows, x, u)
assert refused('in flight', e.sample_paths, cand, dist, w)
assert refused('in flight', e.path_posterior, cand, dist)
assert refused('in flight', e.set_position_bias, np.zeros((1, 1)))
e.knn_viterbi_batch_collect(ticket)
e.sample_paths(cand, dist, w)
# groups of utterances: 4 GB of costs at most, an utterance at least
many = 1 << 13
e.path_posterior(np.zeros((many, 200), np.int64), np.zeros((many, 200)), row_offsets=np.arange(0, many + 1, 64))
e.close()
print('SAMPLING-ASAN-OK')
