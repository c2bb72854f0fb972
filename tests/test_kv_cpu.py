"""The paged key/value cache without a GPU: its work lists (a C++ program built with the
host sanitizers) and what its entry points refuse before any device work."""

import ctypes
import os
import subprocess

import mlq_hip

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "host", "test_kv_plan")


def test_work_lists():
    assert os.path.exists(BIN), "build with __graft_entry__.build() (make -C tests/host)"
    env = dict(os.environ, ASAN_OPTIONS="verify_asan_link_order=0")
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0 and "PASS kv_plan" in r.stdout, r.stdout + r.stderr


def refused(call, code, what):
    assert call == code, mlq_hip.last_error()
    assert what in mlq_hip.last_error()


def test_create_refusals():
    lib = mlq_hip.load()
    h = ctypes.c_void_p(1)

    def create(*a):
        return lib.mlq_hip_kv_cache_create(0, *a, ctypes.byref(h))

    refused(create(4, 1, 1, 32, 1, 64), 1, "hip_kv_cache_create: unsupported type 4")
    assert h.value is None
    refused(create(-1, 1, 1, 32, 1, 64), 1, "unsupported type -1")
    for a in ((0, 1, 32, 1, 64), (1, 0, 32, 1, 64), (1, 1, 32, 0, 64), (1, 1, 32, 1, 0), (1, -5, 32, 1, 64)):
        refused(create(1, *a), 2, "empty caches")
    for page in (0, 1, 16, 31, 33, 48, 100, 131072, -32):
        refused(create(1, 1, 1, page, 1, 64), 2, "page size")
    for hd in (4, 12, 33, 257, 264, 512):
        refused(create(1, 1, 1, 32, 1, hd), 2, "head_dim")
    refused(create(1, 1, 1, 32, 1 << 20, 64), 6, "KV heads")
    refused(create(0, 1 << 20, 1 << 30, 65536, 65536, 256), 6, "too large")
    assert lib.mlq_hip_kv_cache_create(0, 1, 1, 1, 32, 1, 64, None) == 1


def test_null_handles():
    lib = mlq_hip.load()
    h = ctypes.c_void_p()
    refused(lib.mlq_hip_kv_cache_info(None, *[None] * 7), 1, "null cache")
    refused(lib.mlq_hip_kv_plan_create(None, 8, 0, 0, 0.0, 1, 1, 1, ctypes.byref(h)), 1, "null cache")
    refused(lib.mlq_hip_kv_plan_create(None, 8, 0, 0, 0.0, 1, 1, 1, None), 1, "null output handle")
    refused(lib.mlq_hip_kv_plan_set(None, 0, None, None, None, None), 1, "null plan")
    refused(lib.mlq_hip_kv_write(None, 0, None, None, None, None, 0.0, 0, None), 1, "null plan")
    refused(lib.mlq_hip_kv_read(None, 0, 0, None, None, None), 1, "null plan")
    refused(lib.mlq_hip_kv_attention(None, 0, None, None, None), 1, "null plan")
    assert lib.mlq_hip_kv_cache_destroy(None) == 0 and lib.mlq_hip_kv_plan_destroy(None) == 0


def test_batches_hold_32_bit_integers():
    """Lists that would be wrapped or cut off on their way into int arrays are refused."""
    import numpy as np
    import pytest

    mlq_hip.load()
    plan = mlq_hip.KvPlan.__new__(mlq_hip.KvPlan)
    plan.h, plan._page_size = None, 64
    for bad in ([1.0], [2 ** 31], np.array([2 ** 32 + 1]), [-2 ** 40], [True], ["1"]):
        for args in ((bad, [1], [0]), ([1], bad, [0]), ([1], [1], bad)):
            with pytest.raises(ValueError):
                plan.set(*args)
    with pytest.raises(ValueError, match="one length per sequence"):
        plan.set([1, 1], [1], [0])
    with pytest.raises(ValueError, match="2 page ids, the lengths need 1"):
        plan.set([1], [64], [0, 1])
    for good in ((np.array([1], np.uint8), np.array([65], np.int64), (0, 1)), ([], [], [])):
        with pytest.raises(mlq_hip.MlqError, match="null plan"):  # past the lists' checks
            plan.set(*good)


def test_reference_quantizes_as_its_formulas(orc):
    """The values the device tests compare with, against the formats' formulas in 64 bits: a
    value is at most half a step (plus the scale's own rounding) from what is held for it."""
    import numpy as np

    from kv_reference import held

    x = np.random.default_rng(5).standard_normal((50, 3, 80)).astype(np.float32)
    for kind, steps in (("q8_0", 254), ("q4_0", 14), ("q4_1", 15)):
        got = held(orc, kind, x)
        for b in range(0, 80, 32):
            xb, gb = x[..., b:b + 32].astype(np.float64), got[..., b:b + 32].astype(np.float64)
            span = xb.max(-1) - xb.min(-1) if kind == "q4_1" else 2 * np.abs(xb).max(-1)
            # a binary16 scale is off by half a step, 2^-11, of itself, times up to 127 codes
            # (15 of them, and the minimum's own rounding, for q4_1)
            off = np.abs(xb).max(-1) * 2.0 ** -10
            assert (np.abs(xb - gb).max(-1) <= span / steps * (0.5 + 2.0 ** -10) + off).all(), kind
