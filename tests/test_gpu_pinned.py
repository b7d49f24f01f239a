"""Query rows in page-locked memory: results as from ordinary memory, and the memory lives as long as a subset of the batch does."""
import ctypes
import gc

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_pinned_batch_and_its_subset():
    import snickery_amd
    rng = np.random.RandomState(0)
    e = snickery_amd.HipSearchEngine(0)
    e.upload_db(rng.randn(3000, 20).astype(np.float32), rng.randn(3001, 15).astype(np.float32))
    e.set_weights(np.ones(20), np.full(15, 0.2))
    utts = [rng.randn(T, 20) for T in (40, 7, 90)]
    want = e.knn_viterbi_batch(utts, 10)
    batch = snickery_amd.QueryBatch(utts).pin()
    rows = batch.Q
    assert batch.pin().Q is rows                            # once
    for got in (e.knn_viterbi_batch(batch, 10), e.knn_viterbi_batch_collect(e.knn_viterbi_batch_submit(batch, 10))):
        assert all(np.array_equal(a, b) for a, b in zip(got[0], want[0])) and np.array_equal(got[1], want[1])
    part = batch.subset(1, 3)
    del batch, rows
    gc.collect()
    snickery_amd.QueryBatch([rng.randn(200, 20)]).pin()     # memory of its own, given back at once
    got = e.knn_viterbi_batch(part, 10)
    assert all(np.array_equal(a, b) for a, b in zip(got[0], want[0][1:])) and np.array_equal(got[1], want[1][1:])
    e.close()


def test_refusals():
    from snickery_amd.engine import load_library
    lib = load_library()
    p = ctypes.c_void_p()
    assert lib.snk_host_alloc(0, ctypes.byref(p)) != 0 and lib.snk_host_alloc(8, None) != 0 and lib.snk_host_free(None) != 0
