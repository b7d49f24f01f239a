"""The host side of the sampling entry points after refused and failed calls, through the sanitizer build of `make asan-host` (no device,
kernels never run).  Run by tests/test_sampling_host.py in a child process; prints SAMPLING-HOST-OK."""
import os
import sys

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
assert os.environ.get('SNK_LIBRARY', '').endswith('libsnkhip_host_asan.so'), 'run through tests/test_sampling_host.py'
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
N, Dj, T, K = 500, 21, 30, 12
e.upload_join_only(rng.randn(N + 1, Dj).astype(np.float32))
e.set_weights(None, np.full(Dj, 0.1))
cand, dist, u = rng.randint(0, N, (T, K)), rng.rand(T, K), rng.rand(2, T)
x = rng.randn(5, 40)

# ---- a call that asks for more memory than there is: its error is its own, not that of the calls behind it ----
rows = 20000                                          # one utterance: rows x 208 x 208 costs of 8 bytes
wide = np.ones((rows, 208), np.int64)
index = np.zeros((5, 1), np.int64)


def rows_on_the_device():                             # ("device" memory is the host's here)
    return lib.snk_sample_rows_dev(e._h, x.ctypes.data, 0, 5, 40, 40, u.ctypes.data, 1, 1.0, 0, 1.0, 0.0, None, index.ctypes.data, None, None, 0, None)


assert rows_on_the_device() == 0
for call in (lambda: e.path_posterior(wide, np.zeros((rows, 208))), lambda: e.sample_paths(wide, np.zeros((rows, 208)), np.zeros((1, rows)))):
    assert refused('hipMalloc', call)
    assert rows_on_the_device() == 0, lib.snk_last_error()
    assert refused('hipMalloc', call)
    e.sample_rows(x, rng.rand(5))
    assert refused('hipMalloc', call)
    e.sample_paths(cand, dist, u)
    assert refused('hipMalloc', call)
    e.path_posterior(cand, dist)

# ---- a position bias that is refused leaves the one before, and its gradient ----
e.set_position_bias(np.zeros((2, 3)), [0, 1])
for bad in ((np.full((4, 2), np.nan), [0]), (np.zeros((1, 4)), [0, 2, 1]), (np.zeros((1, 65)), np.arange(64)), (np.zeros(3), [0])):
    assert refused('', e.set_position_bias, *bad)
    assert e.path_posterior(cand, dist)[2].shape == (2, 3)
e.set_position_bias(None)
assert e.path_posterior(cand, dist)[2] is None

# ---- query rows moved to page-locked memory: what is written afterwards is what is searched ----
utts = [rng.randn(n, 5) for n in (4, 1, 7)]
batch = snickery_amd.QueryBatch(utts)
before, early = batch.Q, batch.subset(1, 3)
assert np.array_equal(early.Q, np.vstack(utts[1:])) and np.shares_memory(early.Q, before)
batch.pin()
assert not np.shares_memory(batch.Q, before) and np.array_equal(batch.Q, np.vstack(utts))
try:
    before[0, 0] = 1.0                                # the rows are elsewhere: not a silent search of the old ones
    raise AssertionError('the array from before the move can be written')
except ValueError:
    pass
batch.Q[:] = 2.0
late = batch.subset(0, 2).subset(1, 2)
assert np.all(early.Q == 2.0) and early.Q.shape == (8, 5) and np.all(late.Q == 2.0) and late.Q.shape == (1, 5) and late.offsets.tolist() == [0, 1]
assert np.shares_memory(early.Q, batch.Q) and np.shares_memory(late.Q, batch.Q)
other = snickery_amd.QueryBatch(utts)
part = other.subset(0, 1).pin()                       # a subset takes its batch along
assert np.shares_memory(part.Q, other.Q) and other._pinned and other.pin().Q is other.Q
assert snickery_amd.QueryBatch([np.zeros((0, 5))]).pin().Q.shape == (0, 5)
part.Q = np.full((4, 5), 3.0)                         # rows of its own
assert np.all(part.Q == 3.0) and not np.any(other.Q == 3.0) and not np.shares_memory(part.pin().Q, other.Q) and np.all(part.Q == 3.0)

e.close()
print('SAMPLING-HOST-OK')
