"""Decoding with several candidates without a GPU: the trees' work lists (a C++ program built with
the host sanitizers), what the entry points refuse before any device work, and the plain forms
that the device tests compare with."""

import ctypes
import os
import subprocess

import numpy as np
import pytest

import mlq_hip
from tree_reference import attention, beam, chain, checked, depths, path_to, ragged, seen, wide

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "host", "test_kv_tree")


def test_work_lists():
    assert os.path.exists(BIN), "build with __graft_entry__.build() (make -C tests/host)"
    env = dict(os.environ, ASAN_OPTIONS="verify_asan_link_order=0")
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0 and "PASS kv_tree" in r.stdout, r.stdout + r.stderr


def refused(call, code, what):
    assert call == code, mlq_hip.last_error()
    assert what in mlq_hip.last_error()


def test_null_handles():
    lib = mlq_hip.load()
    h = ctypes.c_void_p(1)
    out = ctypes.byref(h)
    refused(lib.mlq_hip_kv_tree_plan_create(None, 8, 0, 0, 0.0, 1, 1, 1, 1, out), 1, "hip_kv_tree_plan_create: null cache")
    assert h.value is None
    refused(lib.mlq_hip_kv_tree_plan_create(None, 8, 0, 0, 0.0, 1, 1, 1, 1, None), 1, "null output handle")
    for nodes in (0, -1, 1025):
        refused(lib.mlq_hip_kv_tree_plan_create(None, 8, 0, 0, 0.0, 1, 1, 1, nodes, out), 6, f"trees of {nodes} nodes")
    refused(lib.mlq_hip_kv_plan_set_tree(None, 0, None, None, None, None, None), 1, "null plan")
    refused(lib.mlq_hip_kv_tree_pick(None, None, 1, None, None, None, None, None, None), 1, "null plan")
    refused(lib.mlq_hip_kv_keep(None, None, None, None), 1, "null plan")
    refused(lib.mlq_hip_kv_copy_pages(None, 0, None, None, None, None), 1, "null cache")
    refused(lib.mlq_hip_beam_select(None, None, None, None, 0, 1, 1, 1, 1, None, None, None, None), 1, "null handle")
    assert lib.mlq_hip_beam_destroy(None) == 0


def test_beam_create_refusals():
    lib = mlq_hip.load()
    h = ctypes.c_void_p(1)
    for a in ((0, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1, 0), (-1, 1, 1, 1)):
        refused(lib.mlq_hip_beam_create(0, *a, ctypes.byref(h)), 2, "empty searches")
        assert h.value is None
    for a in ((1, 65, 1, 1), (1, 1, 1, 65)):
        refused(lib.mlq_hip_beam_create(0, *a, ctypes.byref(h)), 6, "more than 64")
    refused(lib.mlq_hip_beam_create(0, 2 ** 31 - 1, 64, 2 ** 30, 64, ctypes.byref(h)), 6, "2^28")
    refused(lib.mlq_hip_beam_create(0, 1, 1, 2 ** 30 + 1, 1, ctypes.byref(h)), 6, "2^30")
    refused(lib.mlq_hip_beam_create(0, 1, 1, 1, 1, None), 1, "null output handle")


def test_lists_hold_32_bit_integers():
    mlq_hip.load()
    plan = mlq_hip.KvPlan.__new__(mlq_hip.KvPlan)
    plan.h, plan._page_size, plan._n_seqs = None, 64, 1
    cache = mlq_hip.KvCache.__new__(mlq_hip.KvCache)
    cache.h = None
    for bad in ([1.0], [2 ** 31], np.array([2 ** 32 + 1]), [-2 ** 40], [True], ["1"]):
        for call in (lambda: plan.set([1], [1], [0], parents=bad), lambda: plan.keep(bad, [0]), lambda: plan.keep([1], bad),
                     lambda: cache.copy_pages(bad, [0]), lambda: cache.copy_pages([0], bad), lambda: cache.copy_pages([0], [1], bad)):
            with pytest.raises(ValueError):
                call()
    with pytest.raises(ValueError, match="one parent per new token"):
        plan.set([1], [1], [0], parents=[-1, 0])
    with pytest.raises(ValueError, match="one count per sequence"):
        plan.keep([1, 1], [0, 0])
    with pytest.raises(ValueError, match="2 kept nodes, the counts need 1"):
        plan.keep([1], [0, 0])
    with pytest.raises(ValueError, match="one destination"):
        cache.copy_pages([0], [1, 2])


def test_plain_forms():
    """The references by hand: a tree's mask, a chain's attention against the paged one, a path, a search's steps."""
    parents = [-1, 0, 0, 1, 2]
    assert depths(parents).tolist() == [0, 1, 1, 2, 2] and path_to(parents, 4) == [0, 2, 4]
    want = np.array([[1, 1, 0, 0, 0, 0], [1, 1, 1, 0, 0, 0], [1, 1, 0, 1, 0, 0], [1, 1, 1, 0, 1, 0], [1, 1, 0, 1, 0, 1]], bool)
    assert np.array_equal(seen(parents, 1), want)
    want[:, 0] = False
    want[3:, 1] = False
    want[0, 0] = True  # the window of two still has it
    assert np.array_equal(seen(parents, 1, window=2), want)
    want[:, 0] = True
    assert np.array_equal(seen(parents, 1, window=2, sinks=1), want)
    assert wide(6, 2) == [-1, 0, 0, 1, 1, 2] and chain(3) == [-1, 0, 1]

    from kv_reference import attention as plain
    rng = np.random.default_rng(0)
    q, k, v = rng.standard_normal((5, 4, 16)), rng.standard_normal((12, 2, 16)), rng.standard_normal((12, 2, 16))
    assert np.allclose(attention(q, k, v, seen(chain(5), 7))[0], plain(q, k, v)[0], rtol=1e-13)
    assert np.allclose(attention(q, k, v, seen(chain(5), 7, 3, 2))[0], plain(q, k, v, 3, 2)[0], rtol=1e-13)

    logits = np.zeros((5, 9))
    logits[[0, 1, 2, 3, 4], [5, 1, 7, 3, 8]] = 1
    assert checked(logits, [0, 4, 5, 1, 7], parents) == ([5, 1, 7, 3, 8], [0, 2, 4], 8)
    assert ragged(rng, 4, back=1) == chain(4)

    p, t, s = beam(np.log([[0.5, 0.3, 0.2], [0.1, 0.1, 0.8]]), [np.log(0.25), np.log(0.75)], 3)
    # (0.25 x 0.3 and 0.75 x 0.1 are equal but for their roundings)
    assert p[:2] == [1, 0] and t[:2] == [2, 0] and np.allclose(np.exp(s), [0.6, 0.125, 0.075])
    p, t, s = beam([[0.0, 0.0], [0.0, 0.0]], [-1.0, -0.5], 4, ended=[0, 1], end=1)
    assert p == [1, 0, 0, -1] and t == [1, 0, 1, -1] and s[3] == -np.inf
