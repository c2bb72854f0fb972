"""Which kernel batches of drafted trees run, without a GPU: the rule (a C++ program built with the host
sanitizers), and that the device tests' batches run the kernel that they are there for."""

import os
import subprocess

import numpy as np
import pytest

import test_gpu_tree
import test_gpu_tree_rows
from kv_reference import QT
from tree_reference import ragged

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "host", "test_kv_choice")


def run(*args, text=None):
    assert os.path.exists(BIN), "build with __graft_entry__.build() (make -C tests/host)"
    env = dict(os.environ, ASAN_OPTIONS="verify_asan_link_order=0")
    r = subprocess.run([BIN, *args], input=text, capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0, r.stdout + r.stderr
    return r.stdout


def kind(qtype, hd, heads, kv, window, sinks, forest):
    text = f"{QT[qtype]} {hd} {heads} {kv} {window} {sinks} {len(forest)}\n"
    text += "\n".join(" ".join(map(str, (len(t), c, *t))) for t, c in forest)
    return run("kind", text=text).strip()


def test_rule():
    assert "PASS kv_choice" in run()


# Of the large batches of test_gpu_tree.py those whose windows leave so little that the kernel for few rows is faster.
SMALL_WINDOWS = {("f32", 256, 64), ("q4_0", 128, 700), ("q4_1", 96, 90)}


@pytest.mark.parametrize("case", range(len(test_gpu_tree.LARGE)))
def test_large_batches(case):
    qtype, hd, heads, kv, seqs, nodes, before, window, sinks = test_gpu_tree.LARGE[case]
    rng = np.random.default_rng(50 + case)
    forest = [(ragged(rng, nodes - i, roots=1 + i % 2), before + 7 * i) for i in range(seqs)]
    assert kind(qtype, hd, heads, kv, window, sinks, forest) == ("few" if (qtype, hd, window) in SMALL_WINDOWS else "many")


@pytest.mark.parametrize("qtype", list(QT))
def test_batches_of_uneven_blocks(qtype):
    parents = [-1] + [0] * 60 + list(range(60, 255))
    for window, sinks in ((0, 0), (8, 2)):
        assert kind(qtype, 64, 8, 8, window, sinks, [(parents, 33 * (i % 2)) for i in range(70)]) == "many"


@pytest.mark.parametrize("qtype", ["f32", "q8_0", "q4_1"])
def test_recorded_batches(qtype):
    rng = np.random.default_rng(21)
    forest = [(ragged(rng, 256 - i), 900 + 9 * i) for i in range(16)]
    assert kind(qtype, 64, 8, 8, 0, 0, forest) == "many"
    assert kind(qtype, 64, 8, 8, 0, 0, forest[3:4]) == "few"


@pytest.mark.parametrize("case", range(len(test_gpu_tree_rows.WINDOWED)))
def test_windowed_batches(case):
    qtype, hd, heads, kv, _, _, _, window, sinks = test_gpu_tree_rows.WINDOWED[case]
    assert kind(qtype, hd, heads, kv, window, sinks, test_gpu_tree_rows.windowed(case)) == "many"


@pytest.mark.parametrize("qtype", list(QT))
def test_batches_with_values_that_are_not_finite(qtype):
    t = test_gpu_tree_rows
    for window, sinks in t.WINDOWS:
        assert kind(qtype, t.HD, t.HEADS, t.KV, window, sinks, t.apart()) == "many"
