"""Batches of drafted trees that run the attention's kernel for many rows (test_tree_choice_cpu.py holds
that they do): windows, and nodes, positions and slots that a node does not see and that are not finite."""

import numpy as np
import pytest

from kv_reference import QT
from test_gpu_tree import THETA, Step, dev, say
from tree_reference import attention, ragged, seen, wide

pytestmark = pytest.mark.gpu

WINDOWED = [  # kind, hd, heads, kv, sequences, nodes, before, window, sinks
    ("f32", 64, 8, 4, 12, 200, 900, 500, 40), ("f32", 128, 8, 8, 6, 200, 700, 600, 0), ("f32", 256, 8, 4, 8, 240, 900, 700, 33),
    ("q8_0", 64, 16, 8, 16, 220, 1200, 900, 1), ("q8_0", 128, 16, 8, 12, 140, 1000, 900, 4), ("q8_0", 192, 8, 4, 30, 200, 700, 90, 7),
    ("q4_0", 32, 16, 8, 24, 256, 900, 700, 70), ("q4_0", 128, 32, 8, 16, 100, 1500, 700, 1), ("q4_0", 256, 8, 4, 24, 200, 800, 64, 0),
    ("q4_1", 40, 16, 8, 16, 256, 900, 800, 2), ("q4_1", 96, 16, 8, 16, 150, 1100, 700, 7), ("q4_1", 256, 8, 2, 24, 250, 1000, 120, 5),
]


def windowed(case):
    kind, hd, heads, kv, seqs, nodes, before, window, sinks = WINDOWED[case]
    rng = np.random.default_rng(70 + case)
    return [(ragged(rng, nodes - i, back=9, roots=1 + i % 2), before + 7 * i) for i in range(seqs)]


@pytest.mark.parametrize("case", range(len(WINDOWED)))
def test_windows(hip, orc, case):
    kind, hd, heads, kv, _, _, _, window, sinks = WINDOWED[case]
    say("windowed", WINDOWED[case])
    s = Step(hip, orc, kind, windowed(case), heads, kv, hd, 64, window, sinks, seed=case)
    got = s.write().check()
    assert np.array_equal(s.run(), got), "the same call gives the same bits"


HEADS, KV, HD = 16, 8, 64
WINDOWS = ((0, 0), (400, 3))


def apart():
    return [(wide(256, 4), 600 + 13 * i) for i in range(10)]


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("kind", list(QT))
def test_what_a_node_does_not_see_has_no_part(hip, orc, kind, window, sinks):
    """A node, a position before the window or a stale slot behind the tree that is not finite: rows that do not see it stay
    within the bound of what they are without it, other KV heads as they are bit for bit, and rows that see it are NaN,
    of a value in its block's dimensions alone."""
    forest = apart()
    clean = Step(hip, orc, kind, forest, HEADS, KV, HD, 64, window, sinks).write()
    alone = clean.check()
    first = np.cumsum([0] + [len(t) + c for t, c in forest])
    row = np.cumsum([0] + [len(t) for t, _ in forest])
    sees, want, bound = [], [], []
    for i, (t, c) in enumerate(forest):
        k, v = (x[first[i]:first[i + 1]] for x in clean.held)
        sees.append(seen(t, c, window, sinks))
        w, b = attention(clean.turned[row[i]:row[i + 1]], k, v, sees[-1])
        want.append(w)
        bound.append(np.broadcast_to(b, w.shape))
    # sequence, slot, KV head: a node with children, a leaf, two of the first tile of nodes, and positions before the tree
    places = [(0, forest[0][1] + 6, 1), (1, forest[1][1] + 250, 2), (2, forest[2][1] + 1, 3), (3, forest[3][1], 4),
              (4, 5, 5), (5, forest[5][1] - 1, 6)]
    for what in (np.inf, np.nan) if kind == "f32" else (np.inf,):
        for where in "kv":
            say("apart", kind, window, what, where)
            k, v = clean.k.copy(), clean.v.copy()
            for seq, slot, head in places:
                (k if where == "k" else v)[first[seq] + slot, head, 37] = what
            x = Step(hip, orc, kind, forest, HEADS, KV, HD, 64, window, sinks, k=k, v=v)
            x.plan.write(0, x.dk, x.dv, q=x.dq, q_out=x.dq, theta=THETA, neox=True)
            got = x.run()
            of_head = {head: (seq, slot) for seq, slot, head in places}
            for head in range(HEADS):
                if head * KV // HEADS not in of_head:
                    assert np.array_equal(got[:, head], alone[:, head]), head
                    continue
                at, slot = of_head[head * KV // HEADS]
                for seq in range(len(forest)):
                    here = slice(row[seq], row[seq + 1])
                    mine = sees[seq][:, slot] if seq == at else np.zeros(len(sees[seq]), bool)
                    y, w, b = got[here, head], want[seq][:, head], bound[seq][:, head]
                    assert (np.abs(y - w) <= b)[~mine].all(), (head, seq)
                    if where == "k":
                        assert np.isnan(y[mine]).all()
                    else:
                        assert np.isnan(y[mine][:, 32:]).all() and (np.abs(y - w) <= b)[mine][:, :32].all()


@pytest.mark.parametrize("kind", list(QT))
def test_stale_slots_behind_a_tree(hip, orc, kind):
    forest = apart()
    s = Step(hip, orc, kind, forest, HEADS, KV, HD, 64)
    for i, (t, c) in enumerate(forest):
        entry = sum(-(-(len(u) + d) // 64) for u, d in forest[:i])
        n = len(t) + c
        room = min(-n % 64, 5)
        if room == 0:
            continue
        fill = hip.KvPlan(s.cache, HEADS, max_seqs=1, max_tokens=room, max_pages=-(-n // 64))
        fill.set([room], [n + room], s.batch.pages[entry:entry + -(-n // 64)])
        junk = dev(hip, np.full((room, KV, HD), np.inf))
        fill.write(0, junk, junk)
        hip.synchronize(hip.stream(0))
    s.write().check()
