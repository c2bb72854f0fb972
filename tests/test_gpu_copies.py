"""Copies of no positions (mlq_hip_kv_copy_pages): they read and write nothing, so they stand in no other copy's way."""

import numpy as np
import pytest

from test_gpu_tree import Filled

pytestmark = pytest.mark.gpu


def test_copies_of_no_positions(hip):
    f = Filled(hip, "q8_0", 8, 32, 1, 64, 2)
    # page 5 twice, page 0 read and written, page 2 onto itself: each but for one copy of none
    f.cache.copy_pages([0, 1, 7, 2, 3], [5, 5, 0, 2, 6], [32, 0, 0, 0, 32])
    want = f.held.copy()
    want[:, :, 5] = f.held[:, :, 0]
    want[:, :, 6] = f.held[:, :, 3]
    assert np.array_equal(f.read(), want)
    f.cache.copy_pages([1, 1], [1, 1], [0, 0])
    assert np.array_equal(f.read(), want)
    # pages that are not there are refused all the same
    for src, dst in (([8], [1]), ([1], [-1])):
        with pytest.raises(hip.MlqError, match="the cache has 8"):
            f.cache.copy_pages(src, dst, [0])
    for src, dst, what in (([0, 1], [5, 5], "written twice"), ([0, 5], [5, 6], "read and written")):
        with pytest.raises(hip.MlqError, match=what):
            f.cache.copy_pages(src, dst, [1, 32])
    assert np.array_equal(f.read(), want)
