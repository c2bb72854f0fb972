"""Drafted trees over the paged cache on the device: write and attention (mlq_hip_kv_plan_set_tree),
checked drafts (mlq_hip_kv_tree_pick), kept paths (mlq_hip_kv_keep) and copied pages
(mlq_hip_kv_copy_pages) against plain numpy in 64 bits (tree_reference.py, kv_reference.py)."""

import sys

import numpy as np
import pytest

from kv_reference import QT, Batch, held, rotated
from tree_reference import attention, chain, checked, depths, path_to, ragged, seen, wide

pytestmark = pytest.mark.gpu
TYPES = list(QT)
THETA = 10000.0


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def dev(hip, a):
    a = np.ascontiguousarray(a)
    return hip.DeviceBuffer.from_array(a if a.dtype == np.int32 else a.astype(np.float32))


def back(hip, buf, shape, dtype=np.float32, stream=None):
    hip.synchronize(hip.stream(0) if stream is None else stream)
    return buf.download(dtype, int(np.prod(shape))).reshape(shape)


class Step:
    """A cache whose sequences hold random keys and values, and a step of trees: forest is [(parents, positions
    before the tree)].  The nodes are written by the plan, rotated, as a layer does."""

    def __init__(self, hip, orc, kind, forest, heads=4, kv=2, hd=64, page=32, window=0, sinks=0, scale=0.0, seed=0, neox=True,
                 layers=1, layer=0, room=0, stream=None, k=None, v=None):
        self.hip, self.orc, self.kind, self.heads, self.kv, self.hd, self.layer = hip, orc, kind, heads, kv, hd, layer
        self.forest, self.window, self.sinks, self.scale, self.stream = forest, window, sinks, scale, stream
        self.rng = rng = np.random.default_rng(seed)
        self.batch = b = Batch(rng, [(len(t), len(t) + c) for t, c in forest], page)
        rand = rng.standard_normal
        drawn = [rand((b.positions, kv, hd)).astype(np.float32) for _ in range(2)]
        self.k, self.v = drawn[0] if k is None else k, drawn[1] if v is None else v
        self.q = (1.5 * rand((b.tokens, heads, hd))).astype(np.float32)
        self.pos = np.concatenate([c + depths(t) for t, c in forest] + [np.zeros(0, int)]).astype(int)
        self.cache = hip.KvCache(QT[kind], layers, b.n_pages, page, kv, hd)
        before = np.setdiff1d(np.arange(b.positions), b.rows())
        size = dict(max_seqs=max(1, len(forest)), max_pages=max(1, b.entries))
        fill = hip.KvPlan(self.cache, heads, max_tokens=max(1, len(before)), **size)
        lens, pages, at = [c for _, c in forest], [], 0
        for t, c in zip(b.kv_len, lens):
            pages += b.pages[at:at + -(-c // page)]
            at += -(-t // page)
        fill.set(lens, lens, pages, stream=stream)
        if len(before):
            self.filled = dev(hip, self.k[before]), dev(hip, self.v[before])
            fill.write(layer, *self.filled, stream=stream)
        hip.synchronize(hip.stream(0) if stream is None else stream)
        self.plan = hip.KvPlan(self.cache, heads, max_tokens=max(1, b.tokens + room), window=window, sinks=sinks, scale=scale,
                               max_nodes=max([1] + b.new), **size)
        self.plan.set(b.new, b.kv_len, b.pages, parents=sum((list(t) for t, _ in forest), []), stream=stream)
        self.dk, self.dv, self.dq = (dev(hip, x) for x in (self.k[b.rows()], self.v[b.rows()], self.q))
        self.neox = neox
        # what the cache holds after the write
        kk = self.k.copy()
        kk[b.rows()] = rotated(self.k[b.rows()], self.pos, THETA, neox)
        self.held = held(orc, kind, kk), held(orc, kind, self.v)
        self.turned = rotated(self.q, self.pos, THETA, neox)

    def write(self):
        n = self.batch.tokens
        q = dev(self.hip, np.full((n + 2, self.heads, self.hd), 7.25))
        self.plan.write(self.layer, self.dk, self.dv, q=self.dq, q_out=q, theta=THETA, neox=self.neox, stream=self.stream)
        got = back(self.hip, q, (n + 2, self.heads, self.hd), stream=self.stream)
        assert (got[n:] == 7.25).all(), "rows behind the last node"
        # Both are rounded once from 64 bits, so they are equal or neighbours, a step, 2^-23 of the value at the most, apart,
        # as far as the 64-bit results are equal: a frequency and its product with the position are off by 2^-53 of
        # themselves each, on either side, an angle (a frequency is at most 1) by 2^-51 of the position, and the result by
        # that much of its two terms.
        apart = 2.0 ** -51 * (1 + self.pos.max(initial=0)) * 2

        def near(x, want, terms):
            return (np.abs(x - want) <= 2.0 ** -23 * np.abs(want) + apart * np.abs(terms).max(initial=0)).all()

        assert near(got[:n], self.turned, self.q)
        r = [dev(self.hip, np.full((n + 1, self.kv, self.hd), 9.5)) for _ in range(2)]
        self.plan.read(self.layer, *r, new_only=True, stream=self.stream)
        rows = self.batch.rows()
        for x, want, rotated_f32 in zip(r, self.held, (self.kind == "f32", False)):
            got = back(self.hip, x, (n + 1, self.kv, self.hd), stream=self.stream)
            assert (near(got[:n], want[rows], self.k) if rotated_f32 else np.array_equal(got[:n], want[rows])) and (got[n:] == 9.5).all()
            want[rows] = got[:n]  # what the attention reads
        return self

    def run(self, plan=None, q=None):
        n = self.batch.tokens
        shape = (n + 2, self.heads, self.hd)
        q = self.turned if q is None else q
        out = dev(self.hip, np.full(shape, 7.25))
        dq = dev(self.hip, np.concatenate([q, np.full((2,) + q.shape[1:], np.nan, np.float32)]))
        (plan or self.plan).attention(self.layer, dq, out, stream=self.stream)
        got = back(self.hip, out, shape, stream=self.stream)
        assert (got[n:] == 7.25).all(), "rows behind the last node"
        return got[:n]

    def check(self, got=None, q=None):
        got = self.run(q=q) if got is None else got
        q = self.turned if q is None else q
        at = qat = 0
        for t, c in self.forest:
            n = len(t)
            if n:
                k, v = (x[at:at + n + c] for x in self.held)
                want, bound = attention(q[qat:qat + n], k, v, seen(t, c, self.window, self.sinks), self.scale)
                err = np.abs(got[qat:qat + n] - want)
                assert (err <= bound).all(), (n, c, float((err / bound).max()))
            at, qat = at + n + c, qat + n
        return got


def forest_of(rng, spec):
    """[(shape, nodes, before)]: shape 1 a chain, b children of every node, 0 ragged, -1 ragged with several roots."""
    return [(chain(n) if s == 1 else wide(n, s) if s > 1 else ragged(rng, n, roots=min(n, 3) if s else 1), c) for s, n, c in spec]


SHAPES = [  # [(shape, nodes, before)], heads, kv, hd, page, window, sinks
    ([(2, 1, 0)], 1, 1, 8, 32, 0, 0),
    ([(2, 1, 31)], 4, 2, 64, 32, 0, 0),
    ([(2, 7, 32), (0, 16, 33), (1, 5, 100), (0, 0, 50), (3, 0, 0), (0, 33, 0)], 4, 2, 64, 32, 0, 0),
    ([(0, 40, 300)], 8, 1, 64, 64, 0, 0),
    ([(4, 64, 701)], 7, 1, 80, 64, 0, 0),
    ([(-1, 30, 95), (2, 31, 64)], 2, 2, 40, 128, 0, 0),
    ([(0, 130, 500)], 8, 2, 128, 64, 0, 0),
    ([(3, 20, 700), (0, 65, 31)], 3, 3, 160, 32, 0, 0),
    ([(0, 34, 3), (2, 10, 258)], 4, 1, 256, 256, 0, 0),
    ([(0, 12, 1500)], 4, 4, 112, 32, 0, 0),
    ([(0, 50, 200), (1, 40, 10), (2, 9, 1000)], 4, 2, 64, 32, 16, 0),
    ([(1, 100, 0), (0, 60, 20)], 4, 2, 64, 32, 5, 4),
    ([(0, 70, 300), (-1, 20, 1)], 4, 1, 128, 64, 64, 40),
    ([(0, 25, 90)], 2, 1, 96, 32, 1, 1),
    ([(0, 512, 40)], 2, 1, 32, 64, 0, 0),
    ([(0, 17, 9000)], 4, 2, 64, 128, 0, 0),
]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_step(hip, orc, kind, shape):
    spec, heads, kv, hd, page, window, sinks = SHAPES[shape]
    say("step", kind, shape)
    forest = forest_of(np.random.default_rng(100 + shape), spec)
    s = Step(hip, orc, kind, forest, heads, kv, hd, page, window, sinks, seed=shape, neox=shape % 2 == 0, layers=2, layer=1)
    got = s.write().check()
    assert np.array_equal(s.run(), got), "the same call gives the same bits"


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("hd", [16, 64, 96, 128, 192, 256])
def test_row_counts(hip, orc, kind, hd):
    """Row counts around a workgroup's groups of sixteen and thirty-two, several sequences together."""
    forest = forest_of(np.random.default_rng(3), [(0, n, 10 * n) for n in (1, 15, 16, 17, 31, 32, 33, 48, 49)])
    say("rows", kind, hd)
    Step(hip, orc, kind, forest, 1, 1, hd, 32).write().check()
    forest = forest_of(np.random.default_rng(4), [(2, n, 37) for n in (2, 3, 4, 5, 8, 9)])
    Step(hip, orc, kind, forest, 8, 2, hd, 64).write().check()


@pytest.mark.parametrize("kind", ["q8_0", "f32"])
def test_many_sequences_and_long_contexts(hip, orc, kind):
    rng = np.random.default_rng(5)
    say("many", kind)
    Step(hip, orc, kind, forest_of(rng, [(0, int(rng.integers(1, 30)), int(rng.integers(0, 400))) for _ in range(70)]), 4, 1, 64).write().check()
    say("long", kind)
    Step(hip, orc, kind, forest_of(rng, [(0, 40, 30000)]), 4, 1, 64, 1024).write().check()


# Batches large enough for the kernel that converts a tile once a workgroup: by the rule in kv_plan.cpp, ns of all
# tiles by the one kernel (16 rows at a time) above those of the other (128, from five blocks on 64) and its start.
LARGE = [  # kind, hd, heads, kv, sequences, nodes, before, window, sinks
    ("f32", 64, 8, 8, 6, 256, 1000, 0, 0), ("f32", 128, 16, 4, 6, 100, 1100, 0, 0), ("f32", 80, 8, 2, 16, 130, 700, 300, 4),
    ("f32", 192, 8, 8, 8, 190, 600, 0, 0), ("f32", 256, 8, 4, 8, 150, 900, 64, 0),
    ("q8_0", 64, 8, 8, 14, 256, 1000, 0, 0), ("q8_0", 128, 16, 4, 16, 100, 1100, 0, 0), ("q8_0", 256, 8, 4, 40, 128, 900, 400, 40),
    ("q4_0", 16, 16, 16, 8, 512, 500, 0, 0), ("q4_0", 128, 32, 8, 9, 64, 1500, 700, 1), ("q4_0", 192, 8, 8, 20, 250, 700, 0, 0),
    ("q4_1", 64, 8, 8, 14, 256, 1000, 0, 0), ("q4_1", 96, 16, 4, 16, 100, 1100, 90, 7), ("q4_1", 256, 8, 2, 24, 250, 1000, 0, 0),
]


@pytest.mark.parametrize("case", range(len(LARGE)))
def test_large_batches(hip, orc, case):
    kind, hd, heads, kv, seqs, nodes, before, window, sinks = LARGE[case]
    say("large", LARGE[case])
    rng = np.random.default_rng(50 + case)
    forest = [(ragged(rng, nodes - i, roots=1 + i % 2), before + 7 * i) for i in range(seqs)]
    s = Step(hip, orc, kind, forest, heads, kv, hd, 64, window, sinks, seed=case)
    got = s.write().check()
    assert np.array_equal(s.run(), got), "the same call gives the same bits"


@pytest.mark.parametrize("kind", TYPES)
def test_large_batches_of_uneven_blocks(hip, orc, kind):
    """Rows that have to be done again, for positions before the tree, ancestors, and first positions: a node of depth 1
    whose slot lies far below the window of the last rows, but which they see as one of the first two."""
    rng = np.random.default_rng(60)
    parents = [-1] + [0] * 60 + list(range(60, 255))  # node 60 has depth 1, the last one depth 196
    forest = [(parents, 33 * (i % 2)) for i in range(70)]
    n = sum(len(t) + c for t, c in forest)
    k, v = (rng.standard_normal((n, 8, 64)).astype(np.float32) for _ in range(2))
    at = 0
    for i, (t, c) in enumerate(forest):
        for node in (60, 100, 250):
            v[at + c + node, i % 8, 32:] *= np.float32(3e-4 if node != 250 else 3000)
            k[at + c + node, (i + 1) % 8, :32] *= np.float32(1e-6)
        if c:
            v[at + 5, (i + 2) % 8, :32] *= np.float32(1e-3)
        at += len(t) + c
    for window, sinks in ((0, 0), (8, 2)):
        say("uneven", kind, window)
        Step(hip, orc, kind, forest, 8, 8, 64, 64, window, sinks, k=k, v=v).write().check()


def test_scales_and_large_queries(hip, orc):
    for scale, factor in ((0.5, 1.0), (-0.125, 1.0), (0.0, 40.0), (1e-20, 1e18)):
        s = Step(hip, orc, "q8_0", forest_of(np.random.default_rng(6), [(0, 20, 120)]), scale=scale)
        s.write().check(q=(s.turned * np.float32(factor)).astype(np.float32))


def test_chains_are_what_plain_plans_compute(hip, orc):
    """A chain sees what plain new tokens see: both forms are within their bounds of the same result, and a tree's plan
    takes batches without parents."""
    s = Step(hip, orc, "q4_0", [(chain(9), 200), (chain(40), 0)], 8, 2, 64).write()
    got = s.check()
    b = s.batch
    plan = hip.KvPlan(s.cache, 8, max_seqs=2, max_tokens=b.tokens, max_pages=b.entries)
    plan.set(b.new, b.kv_len, b.pages)
    s.check(s.run(plan))
    s.plan.set(b.new, b.kv_len, b.pages)
    assert np.array_equal(s.run(), got)


@pytest.mark.parametrize("kind", TYPES)
def test_what_a_node_does_not_see_has_no_part(hip, orc, kind):
    """Nodes of other branches that are not finite, slots after the tree and positions outside the window too; a node that
    sees one is NaN there and nowhere else."""
    rng = np.random.default_rng(7)
    parents = wide(21, 4)
    for window, sinks, bad, before in ((0, 0, 6, 70), (0, 0, 1, 33), (12, 2, 3, 70)):
        s = Step(hip, orc, kind, [(parents, before)], 4, 2, 64, 32, window, sinks)
        clean = s.write().check()
        for what, where in ((np.nan, "k"), (np.inf, "v"), (np.nan, "v")):
            if kind != "f32" and np.isnan(what):
                continue  # what a quantized block holds of NaN is up to the format
            k, v = s.k.copy(), s.v.copy()
            (k if where == "k" else v)[before + bad, 1, 5] = what
            x = Step(hip, orc, kind, [(parents, before)], 4, 2, 64, 32, window, sinks, k=k, v=v)
            x.plan.write(0, x.dk, x.dv, q=x.dq, q_out=x.dq, theta=THETA, neox=True)
            got = x.run()
            sees = seen(parents, before, window, sinks)[:, before + bad]
            assert sees.any() and not sees.all()
            assert np.array_equal(got[~sees], clean[~sees]), (what, where)
            assert np.array_equal(got[:, :2], clean[:, :2]), "the other KV head"
            if where == "k":
                assert np.isnan(got[sees][:, 2:]).all()
            else:
                assert np.isnan(got[sees][:, 2:, :32]).all() and np.array_equal(got[sees][:, 2:, 32:], clean[sees][:, 2:, 32:])
    # stale slots after the tree, in its last tile
    s = Step(hip, orc, kind, [(parents, 70)], 4, 2, 64, 32)
    fill = hip.KvPlan(s.cache, 4, max_seqs=1, max_tokens=96, max_pages=3)
    fill.set([5], [96], s.batch.pages)
    junk = dev(hip, np.full((5, 2, 64), np.inf))
    fill.write(0, junk, junk)
    s.write().check()


def test_far_pages(hip, orc):
    """Pages beyond 4 GiB of a layer: offsets pass 32 bits, in attention, copies and moves."""
    rng = np.random.default_rng(17)
    kv, hd, page = 8, 128, 1024
    cache = hip.KvCache(QT["f32"], 2, 600, page, kv, hd)
    parents, before = wide(40, 3), 1000
    n = before + 40
    k, v = (rng.standard_normal((n, kv, hd)).astype(np.float32) for _ in range(2))
    plan = hip.KvPlan(cache, kv, max_seqs=1, max_tokens=40, max_pages=2, max_nodes=40)
    fill = hip.KvPlan(cache, kv, max_seqs=1, max_tokens=n, max_pages=2)
    fill.set([n], [n], [599, 540])
    fill.write(1, dev(hip, k), dev(hip, v))
    q = rng.standard_normal((40, kv, hd)).astype(np.float32)
    want, bound = attention(q, k, v, seen(parents, before))
    out = hip.DeviceBuffer(q.nbytes)
    plan.set([40], [n], [599, 540], parents=parents)
    plan.attention(1, dev(hip, q), out)
    assert (np.abs(back(hip, out, q.shape) - want) <= bound).all()
    cache.copy_pages([599, 540], [598, 7])
    plan.set([40], [n], [598, 7], parents=parents)
    plan.attention(1, dev(hip, q), out)
    assert (np.abs(back(hip, out, q.shape) - want) <= bound).all()
    path = path_to(parents, 38)
    plan.keep([len(path)], path)
    fill.set([0], [before + len(path)], [598])
    rk, rv = (hip.DeviceBuffer(4 * n * kv * hd) for _ in range(2))
    fill.read(1, rk, rv)
    rows = list(range(before)) + [before + i for i in path]
    for r, x in ((rk, k), (rv, v)):
        assert np.array_equal(back(hip, r, (len(rows), kv, hd)), x[rows])


# ---------------------------------------------------------------- kept paths and copied pages

def layers_of(hip, cache, layers, pages, lens, page, kv, hd):
    """What the cache holds: [layer] -> (k, v) of the sequences' positions."""
    plan = hip.KvPlan(cache, kv, max_seqs=len(lens), max_tokens=1, max_pages=len(pages))
    plan.set([0] * len(lens), lens, pages)
    out = []
    for layer in range(layers):
        r = [hip.DeviceBuffer(4 * sum(lens) * kv * hd) for _ in range(2)]
        plan.read(layer, *r)
        out.append([back(hip, x, (sum(lens), kv, hd)) for x in r])
    return out


class Filled:
    """A cache of several layers whose pages are all full of random keys and values."""

    def __init__(self, hip, kind, n_pages, page, kv=2, hd=64, layers=3, seed=0):
        self.hip, self.n_pages, self.page, self.kv, self.hd, self.layers = hip, n_pages, page, kv, hd, layers
        self.rng = np.random.default_rng(seed)
        self.cache = hip.KvCache(QT[kind], layers, n_pages, page, kv, hd)
        n = n_pages * page
        fill = hip.KvPlan(self.cache, kv, max_seqs=1, max_tokens=n, max_pages=n_pages)
        fill.set([n], [n], list(range(n_pages)))
        for layer in range(layers):
            fill.write(layer, *(dev(hip, self.rng.standard_normal((n, kv, hd))) for _ in range(2)))
            hip.synchronize(hip.stream(0))
        self.held = self.read()

    def read(self):
        """[layer, k or v, page, slot, kv, hd]"""
        got = layers_of(self.hip, self.cache, self.layers, list(range(self.n_pages)), [self.n_pages * self.page], self.page, self.kv, self.hd)
        return np.array(got).reshape(self.layers, 2, self.n_pages, self.page, self.kv, self.hd)


KEEPS = [  # [(parents' shape, nodes, before, node whose path is kept or -1)], kv, hd, page, layers
    ([(2, 7, 30, 6)], 2, 64, 32, 2),
    ([(0, 40, 20, 39), (1, 10, 5, 9), (3, 30, 61, 29), (0, 25, 0, -1), (0, 0, 40, -1)], 2, 64, 32, 3),
    ([(0, 200, 50, 199)], 1, 80, 64, 2),
    ([(0, 300, 7, 299), (0, 64, 64, 60)], 3, 128, 32, 1),
    ([(5, 60, 90, 59)], 1, 256, 64, 2),
    ([(0, 33, 95, 31)], 2, 40, 32, 2),
]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("case", range(len(KEEPS)))
def test_keep(hip, kind, case):
    """Every slot of the cache, in every layer: kept ones where they belong, others of the sequences as they were."""
    spec, kv, hd, page, layers = KEEPS[case]
    rng = np.random.default_rng(case)
    forest = forest_of(rng, [x[:3] for x in spec])
    b = Batch(rng, [(len(t), len(t) + c) for t, c in forest], page)
    f = Filled(hip, kind, b.n_pages, page, kv, hd, layers, seed=case)
    plan = hip.KvPlan(f.cache, kv, max_seqs=len(forest), max_tokens=max(1, b.tokens), max_pages=b.entries, max_nodes=max(b.new))
    plan.set(b.new, b.kv_len, b.pages, parents=sum((list(t) for t, _ in forest), []))
    paths = [path_to(t, x[3]) for (t, _), x in zip(forest, spec)]
    say("keep", kind, case, [len(p) for p in paths])
    plan.keep([len(p) for p in paths], sum(paths, []))
    want, at, free = f.held.copy(), 0, np.zeros(f.held.shape[2:4], bool)
    for (t, c), path in zip(forest, paths):
        where = [(b.pages[at + p // page], p % page) for p in range(c + len(t))]
        for d, i in enumerate(path):
            want[:, :, where[c + d][0], where[c + d][1]] = f.held[:, :, where[c + i][0], where[c + i][1]]
        for p in range(c + len(path), c + len(t)):
            free[where[p]] = True  # undefined
        at += -(-(c + len(t)) // page)
    got = f.read()
    assert np.array_equal(got[:, :, ~free], want[:, :, ~free])


def test_keep_twice(hip):
    """A path that lies apart from where it moves may be moved again; a node that another one has been moved over is
    refused until the next set."""
    rng = np.random.default_rng(3)
    parents = [-1, 0, 0, 2, 3, 4, 4]
    b = Batch(rng, [(7, 40)], 32)
    f = Filled(hip, "q8_0", b.n_pages, 32, 1, 64, 2)
    plan = hip.KvPlan(f.cache, 1, max_seqs=1, max_tokens=7, max_pages=b.entries, max_nodes=7)
    plan.set(b.new, b.kv_len, b.pages, parents=parents)
    plan.keep([2], [0, 2])
    once = f.read()
    plan.keep([2], [0, 2])
    assert np.array_equal(f.read(), once)
    with pytest.raises(hip.MlqError, match="kept node 1 has been moved over by node 2"):
        plan.keep([2], [0, 1])
    plan.keep([4], [0, 2, 3, 4])
    moved = f.read()
    with pytest.raises(hip.MlqError, match="kept node 2 has been moved over by node 3"):
        plan.keep([4], [0, 2, 3, 4])
    assert np.array_equal(f.read(), moved)
    plan.set(b.new, b.kv_len, b.pages, parents=parents)
    plan.keep([2], [0, 1])
    assert np.array_equal(f.read(), moved)


@pytest.mark.parametrize("kind", TYPES)
def test_keep_many_paths(hip, kind):
    """More moves than a launch's arguments hold, paths cut between launches."""
    rng = np.random.default_rng(9)
    forest = [([-1, -1] + list(range(1, n - 1)), 3 * i) for i, n in enumerate([40] * 9 + [300] + [8] * 30)]
    b = Batch(rng, [(len(t), len(t) + c) for t, c in forest], 32)
    f = Filled(hip, kind, b.n_pages, 32, 1, 32, 1)
    plan = hip.KvPlan(f.cache, 1, max_seqs=len(forest), max_tokens=b.tokens, max_pages=b.entries, max_nodes=300)
    plan.set(b.new, b.kv_len, b.pages, parents=sum((t for t, _ in forest), []))
    paths = [path_to(t, len(t) - 1) for t, _ in forest]  # every node moves down by one
    plan.keep([len(p) for p in paths], sum(paths, []))
    got, at = f.read(), 0
    for (t, c), path in zip(forest, paths):
        for d, i in enumerate(path):
            to, src = ((b.pages[at + p // 32], p % 32) for p in (c + d, c + i))
            assert np.array_equal(got[:, :, to[0], to[1]], f.held[:, :, src[0], src[1]])
        at += -(-(c + len(t)) // 32)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("page,hd", [(32, 64), (128, 80), (64, 256)])
def test_copy_pages(hip, kind, page, hd):
    f = Filled(hip, kind, 20, page, 2, hd, 3)
    order = f.rng.permutation(20)
    src, dst = order[[0, 1, 2, 0, 3]], order[5:10]  # a page may be read twice
    for positions in ([1, page, page - 1, min(33, page), 0], None):
        f.cache.copy_pages(src, dst, positions)
        used = positions or [page] * 5
        got, want = f.read(), f.held.copy()
        known = np.ones(f.held.shape[2:4], bool)
        for a, b, n in zip(src, dst, used):
            want[:, :, b, :n] = f.held[:, :, a, :n]
            known[b, n:-(-n // 32) * 32] = False
        assert np.array_equal(got[:, :, known], want[:, :, known])
        f.held = got


def test_copy_many_pages(hip):
    """More copies than a launch's arguments hold."""
    f = Filled(hip, "q4_1", 600, 32, 1, 32, 2)
    order = f.rng.permutation(600)
    f.cache.copy_pages(order[:290], order[300:590])
    want = f.held.copy()
    want[:, :, order[300:590]] = f.held[:, :, order[:290]]
    assert np.array_equal(f.read(), want)


def test_recorded_copies(hip):
    f = Filled(hip, "q8_0", 6, 32)
    s = hip.stream_create()
    g = hip.Graph.record(lambda: f.cache.copy_pages([0, 1], [4, 5], stream=s), stream=s)
    for _ in range(3):
        f.cache.copy_pages([2, 3], [0, 1], stream=s)
        g.launch(s)
        hip.synchronize(s)
        want = f.held.copy()
        want[:, :, [0, 1, 4, 5]] = f.held[:, :, [2, 3, 2, 3]]
        assert np.array_equal(f.read(), want)
        f.cache.copy_pages([4], [2], stream=s)
        hip.synchronize(s)
    g.destroy()
    hip.stream_destroy(s)


# ---------------------------------------------------------------- checked drafts

class Drafts:
    def __init__(self, hip, trees, vocab, seed=0, stream=None, room=0, logits=None):
        self.hip, self.trees, self.vocab, self.stream = hip, trees, vocab, stream
        rng = np.random.default_rng(seed)
        self.rows = rows = sum(map(len, trees))
        self.logits = rng.standard_normal((rows, vocab)).astype(np.float32) if logits is None else logits
        self.tokens = np.zeros(rows, np.int32)
        at = 0
        for t in trees:
            for i, p in enumerate(t):
                r = self.logits[at + p]
                self.tokens[at + i] = np.argmax(r) if p >= 0 and rng.random() < 0.7 else rng.integers(vocab)
            at += len(t)
        pages = [-(-len(t) // 32) for t in trees]
        cache = hip.KvCache(QT["q8_0"], 1, max(1, sum(pages)), 32, 1, 32)
        self.plan = hip.KvPlan(cache, 1, max_seqs=len(trees) + room, max_tokens=max(1, rows) + room, max_pages=max(1, sum(pages)),
                               max_nodes=max([1] + [len(t) for t in trees]))
        n = [len(t) for t in trees]
        self.plan.set(n, n, list(range(sum(pages))), parents=sum((list(t) for t in trees), []), stream=stream)

    def buffers(self):
        return [self.hip.DeviceBuffer.from_array(np.full(n + 1, -9, np.int32)) for n in (self.rows, len(self.trees), self.rows, len(self.trees))]

    def check(self, out=None, logits=None):
        hip = self.hip
        if out is None:
            out = self.buffers()
            x = hip.DeviceBuffer.from_array(self.logits) if logits is None else logits
            self.plan.pick(x, self.vocab, hip.DeviceBuffer.from_array(self.tokens) if self.rows else None, *out, stream=self.stream)
        picks, n_kept, kept, nexts = (back(hip, b, (n + 1,), np.int32, self.stream)
                                      for b, n in zip(out, (self.rows, len(self.trees)) * 2))
        assert picks[-1] == n_kept[-1] == kept[-1] == nexts[-1] == -9
        at = 0
        for s, t in enumerate(self.trees):
            n = len(t)
            p, path, following = checked(self.logits[at:at + n], self.tokens[at:at + n], list(t))
            assert picks[at:at + n].tolist() == p
            assert n_kept[s] == len(path) and kept[at:at + n].tolist() == path + [-1] * (n - len(path)), (s, path)
            assert nexts[s] == following
            at += n
        return [picks, n_kept, kept, nexts]


@pytest.mark.parametrize("vocab", [1, 2, 63, 257, 2048, 4097, 32000, 128011])
def test_pick(hip, vocab):
    rng = np.random.default_rng(vocab)
    say("pick", vocab)
    Drafts(hip, [chain(1)], vocab).check()
    Drafts(hip, [wide(8, 2), [], chain(5), ragged(rng, 20), ragged(rng, 9, roots=3)], vocab, seed=1).check()


def test_pick_deep_and_many(hip):
    rng = np.random.default_rng(2)
    Drafts(hip, [chain(1024)], 40, seed=3).check()
    Drafts(hip, [ragged(rng, int(rng.integers(0, 70)), back=80) for _ in range(60)], 333, seed=4).check()
    # sure chains are kept whole
    d = Drafts(hip, [chain(200), chain(64), chain(65)], 500, seed=5)
    at = 0
    for t in d.trees:
        d.tokens[at + 1:at + len(t)] = d.logits[at:at + len(t) - 1].argmax(-1)
        at += len(t)
    assert d.check()[1][:3].tolist() == [200, 64, 65]


def test_pick_ties_and_values_that_are_not_finite(hip):
    rng = np.random.default_rng(8)
    vocab = 5000
    x = rng.integers(-3, 3, (24, vocab)).astype(np.float32)  # the largest many times
    x[3] = 0.0
    x[4] = -0.0
    x[4, 17] = 0.0  # equal to -0
    x[5] = -3.4e38
    x[6, 4999] = np.nan
    x[7, 0] = np.inf
    x[8, 2500] = -np.inf
    x[9, 4999] = 9.0
    x[10, 0] = 9.0
    d = Drafts(hip, [ragged(rng, 24)], vocab, logits=x)
    picks = d.check()[0]
    assert picks[3] == picks[4] == picks[5] == 0 and (picks[6:9] == -1).all() and picks[9] == 4999 and picks[10] == 0
    # the root itself: no path beyond it, even to a child whose token is -1
    x = rng.standard_normal((3, 64)).astype(np.float32)
    x[0, 5] = np.nan
    d = Drafts(hip, [chain(3)], 64, logits=x)
    d.tokens[1] = -1
    _, n_kept, kept, nexts = d.check()
    assert n_kept[0] == 1 and nexts[0] == -1
    # of two children with the right token the lower one
    x = rng.standard_normal((4, 64)).astype(np.float32)
    d = Drafts(hip, [[-1, 0, 0, 0]], 64, logits=x)
    d.tokens[1:] = [7 if x[0].argmax() != 7 else 8, x[0].argmax(), x[0].argmax()]
    assert d.check()[2][:2].tolist() == [0, 2]


def test_pick_rows_at_odd_addresses(hip):
    x = np.random.default_rng(9).standard_normal((10, 777)).astype(np.float32)
    for off in (1, 2, 3):
        buf = hip.DeviceBuffer.from_array(np.concatenate([np.full(off, 1e30, np.float32), x.ravel()]))
        Drafts(hip, [wide(10, 3)], 777, logits=x).check(logits=buf.ptr + 4 * off)
        hip.synchronize(hip.stream(0))


# ---------------------------------------------------------------- recorded, and together

def test_recorded_step(hip, orc):
    """One recorded step (write, attention, picks) serves every batch of trees that is set later, between eager work."""
    heads, kv, hd, page, most, vocab, max_seqs = 8, 2, 64, 64, 100, 300, 5
    rng = np.random.default_rng(11)
    cache = hip.KvCache(QT["q8_0"], 1, 90, page, kv, hd)
    plan = hip.KvPlan(cache, heads, max_seqs=max_seqs, max_tokens=most, max_pages=80, window=700, sinks=4, max_nodes=96)
    fill = hip.KvPlan(cache, heads, max_seqs=max_seqs, max_tokens=5000, max_pages=80)
    s = hip.stream_create()
    dk, dv = (hip.DeviceBuffer(4 * most * kv * hd) for _ in range(2))
    dq, oq, out = (hip.DeviceBuffer(4 * most * heads * hd) for _ in range(3))
    dl, dt = hip.DeviceBuffer(4 * most * vocab), hip.DeviceBuffer(4 * most)
    ints = [hip.DeviceBuffer(4 * n) for n in (most, max_seqs, most, max_seqs)]

    def step():
        plan.write(0, dk, dv, q=dq, q_out=oq, theta=THETA, neox=True, stream=s)
        plan.attention(0, oq, out, stream=s)
        plan.pick(dl, vocab, dt, *ints, stream=s)

    plan.set([1], [1], [0], parents=[-1], stream=s)
    g = hip.Graph.record(step, stream=s)
    specs = ([(2, 30, 40)], [(0, 96, 4000)], [(1, 1, 10), (0, 3, 700), (0, 0, 9), (3, 40, 1), (0, 5, 64)], [], [(0, 0, 50)],
             [(0, 33, 0), (0, 67, 900)], [(2, 1, 1)])
    for spec in specs:
        forest = forest_of(rng, spec)
        b = Batch(rng, [(len(t), len(t) + c) for t, c in forest], page, spare=0)
        k, v = (rng.standard_normal((b.positions, kv, hd)).astype(np.float32) for _ in range(2))
        q = rng.standard_normal((b.tokens, heads, hd)).astype(np.float32)
        logits = rng.standard_normal((b.tokens, vocab)).astype(np.float32)
        pos = np.concatenate([c + depths(t) for t, c in forest] + [np.zeros(0, int)]).astype(int)
        if b.positions:
            fill.set(b.kv_len, b.kv_len, b.pages, stream=s)
            fk, fv = dev(hip, k), dev(hip, v)
            fill.write(0, fk, fv, stream=s)
        plan.set(b.new, b.kv_len, b.pages, parents=sum((list(t) for t, _ in forest), []), stream=s)
        hip.synchronize(s)
        tokens, at = np.zeros(b.tokens, np.int32), 0
        for t, _ in forest:
            for i, p in enumerate(t):
                tokens[at + i] = logits[at + p].argmax() if p >= 0 and rng.random() < 0.7 else 3
            at += len(t)
        for d, x in ((dk, k[b.rows()]), (dv, v[b.rows()]), (dq, q), (dl, logits), (dt, tokens)):
            if x.size:
                d.upload(x)
        out.upload(np.full(most * heads * hd, 5.5, np.float32))
        for i in ints:
            i.upload(np.full(i.nbytes // 4, -9, np.int32))
        for _ in range(3):
            g.launch(s)
        hip.synchronize(s)
        got = out.download(np.float32, most * heads * hd).reshape(most, heads, hd)
        assert (got[b.tokens:] == 5.5).all(), spec
        picks, n_kept, kept, nexts = (i.download(np.int32, i.nbytes // 4) for i in ints)
        kk = k.copy()
        kk[b.rows()] = rotated(k[b.rows()], pos, THETA, True)
        kk, vv, qq = held(orc, "q8_0", kk), held(orc, "q8_0", v), rotated(q, pos, THETA, True)
        at = qat = 0
        for i, (t, c) in enumerate(forest):
            n = len(t)
            if n:
                want, bound = attention(qq[qat:qat + n], kk[at:at + n + c], vv[at:at + n + c], seen(t, c, 700, 4))
                assert (np.abs(got[qat:qat + n] - want) <= bound).all(), spec
            p, path, following = checked(logits[qat:qat + n], tokens[qat:qat + n], list(t))
            assert picks[qat:qat + n].tolist() == p and kept[qat:qat + n].tolist() == path + [-1] * (n - len(path))
            assert n_kept[i] == len(path) and nexts[i] == following
            at, qat = at + n + c, qat + n
        assert (picks[qat:] == -9).all() and (n_kept[len(forest):] == -9).all()
        # eager, the same bits
        step()
        hip.synchronize(s)
        assert np.array_equal(out.download(np.float32, most * heads * hd).reshape(got.shape), got), spec
    with pytest.raises(hip.MlqError, match="graph capture"):
        hip.Graph.record(lambda: plan.set([1], [1], [0], parents=[-1], stream=s), stream=s)
    with pytest.raises(hip.MlqError, match="cannot be recorded"):
        hip.Graph.record(lambda: plan.keep([1], [0], stream=s), stream=s)
    with pytest.raises(hip.MlqError, match="graph capture"):
        hip.Graph.record(lambda: hip.KvPlan(cache, heads, max_seqs=1, max_tokens=1, max_pages=1, max_nodes=1), stream=hip.stream(0))
    short = hip.DeviceBuffer(4 * (most - 1))
    with pytest.raises(hip.MlqError, match="too small"):
        hip.Graph.record(lambda: plan.pick(dl, vocab, short, *ints, stream=s), stream=s)
    g.destroy()
    hip.stream_destroy(s)


@pytest.mark.parametrize("kind", ["f32", "q8_0", "q4_1"])
def test_recorded_attention_of_large_and_small_batches(hip, orc, kind):
    """One recorded call runs whichever kernel the batch that is set takes: many rows, few, many again."""
    rng = np.random.default_rng(21)
    s = hip.stream_create()
    large = Step(hip, orc, kind, [(ragged(rng, 256 - i), 900 + 9 * i) for i in range(16)], 8, 8, 64, 64, stream=s).write()
    b, n = large.batch, large.batch.tokens
    q = dev(hip, large.turned)
    out, eager = (dev(hip, np.full(large.turned.shape, 7.25)) for _ in range(2))
    parents = [list(t) for t, _ in large.forest]
    first = [-(-t // 64) for t in b.kv_len]
    g = hip.Graph.record(lambda: large.plan.attention(0, q, out, stream=s), stream=s)
    for some in (range(16), [3], range(16), [], [0, 5], range(16)):
        pages = sum((b.pages[sum(first[:i]):sum(first[:i + 1])] for i in some), [])
        rows = sum(b.new[i] for i in some)
        large.plan.set([b.new[i] for i in some], [b.kv_len[i] for i in some], pages, parents=sum((parents[i] for i in some), []),
                       stream=s)
        for x in (out, eager):
            x.upload(np.full(large.turned.size, 7.25, np.float32))
        for _ in range(3):
            g.launch(s)
        large.plan.attention(0, q, eager, stream=s)
        got, want = (back(hip, x, large.turned.shape, stream=s) for x in (out, eager))
        assert np.array_equal(got, want) and (got[rows:] == 7.25).all()
        if rows == n:
            large.check(got)
    g.destroy()
    hip.stream_destroy(s)


@pytest.mark.parametrize("kind", TYPES)
def test_drafted_decoding_is_decoding(hip, orc, kind):
    """Two steps of drafted trees on a stream of their own: the kept path of the first is a prefix of the second, which then
    attends as a sequence does that has had those tokens one after the other."""
    rng = np.random.default_rng(21)
    heads, kv, hd, page, before = 4, 2, 64, 32, 50
    parents = ragged(rng, 25)
    path = path_to(parents, 24)
    s = hip.stream_create()
    step = Step(hip, orc, kind, [(parents, before)], heads, kv, hd, page, layers=2, layer=1, stream=s)
    step.write().check()
    step.plan.keep([len(path)], path, stream=s)
    n = before + len(path)
    # the same tokens, plainly
    rows = list(range(before)) + [before + i for i in path]
    kk, vv = step.k[rows].copy(), step.v[rows]
    kk[before:] = rotated(kk[before:], np.arange(before, n), THETA, True)
    tree2 = wide(6, 2)
    new_k, new_v = (rng.standard_normal((6, kv, hd)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((6, heads, hd)).astype(np.float32)
    plan = hip.KvPlan(step.cache, heads, max_seqs=1, max_tokens=6, max_pages=4, max_nodes=6)
    need = -(-(n + 6) // page)
    spare = [p for p in range(step.batch.n_pages) if p not in step.batch.pages]
    plan.set([6], [n + 6], (step.batch.pages + spare)[:need], parents=tree2, stream=s)
    dk, dv, dq, out = dev(hip, new_k), dev(hip, new_v), dev(hip, q), hip.DeviceBuffer(q.nbytes)
    plan.write(1, dk, dv, q=dq, q_out=dq, theta=THETA, neox=True, stream=s)
    plan.attention(1, dq, out, stream=s)
    pos = n + depths(tree2)
    k = held(orc, kind, np.concatenate([kk, rotated(new_k, pos, THETA, True)]))
    v = held(orc, kind, np.concatenate([vv, new_v]))
    want, bound = attention(rotated(q, pos, THETA, True), k, v, seen(tree2, n))
    got = back(hip, out, q.shape, stream=s)
    assert (np.abs(got - want) <= bound).all()
    hip.stream_destroy(s)


def test_forked_beams_share_a_prefix(hip, orc):
    """Beams of one sequence: full pages in common, the last page copied for each, then a token each."""
    rng = np.random.default_rng(22)
    heads, kv, hd, page, length = 4, 2, 64, 32, 75
    for kind in TYPES:
        cache = hip.KvCache(QT[kind], 2, 10, page, kv, hd)
        k, v = (rng.standard_normal((length, kv, hd)).astype(np.float32) for _ in range(2))
        fill = hip.KvPlan(cache, heads, max_seqs=1, max_tokens=length, max_pages=3)
        fill.set([length], [length], [4, 1, 7])
        for layer in range(2):
            fill.write(layer, dev(hip, k), dev(hip, v))
        cache.copy_pages([7, 7, 7], [0, 2, 9], [length % page] * 3)
        plan = hip.KvPlan(cache, heads, max_seqs=4, max_tokens=4, max_pages=12)
        plan.set([1] * 4, [length + 1] * 4, [4, 1, 7, 4, 1, 0, 4, 1, 2, 4, 1, 9])
        nk, nv = (rng.standard_normal((4, kv, hd)).astype(np.float32) for _ in range(2))
        q = rng.standard_normal((4, heads, hd)).astype(np.float32)
        out = hip.DeviceBuffer(q.nbytes)
        plan.write(1, dev(hip, nk), dev(hip, nv))
        plan.attention(1, dev(hip, q), out)
        got = back(hip, out, q.shape)
        for b in range(4):
            want, bound = attention(q[b:b + 1], held(orc, kind, np.concatenate([k, nk[b:b + 1]])),
                                    held(orc, kind, np.concatenate([v, nv[b:b + 1]])), np.ones((1, length + 1), bool))
            assert (np.abs(got[b:b + 1] - want) <= bound).all(), (kind, b)


# ---------------------------------------------------------------- refusals

def test_refusals(hip):
    cache = hip.KvCache(QT["q8_0"], 2, 6, 64, 2, 64)

    def tree(max_nodes=8, max_seqs=2, max_tokens=16, max_pages=4, heads=4, **kw):
        return hip.KvPlan(cache, heads, max_seqs=max_seqs, max_tokens=max_tokens, max_pages=max_pages, max_nodes=max_nodes, **kw)

    for bad, what in ((dict(max_nodes=-1), "trees of -1 nodes"), (dict(max_nodes=1025), "trees of 1025 nodes"),
                      (dict(heads=3), "3 heads over 2"), (dict(window=-1), "negative window"), (dict(sinks=1), "sinks need"),
                      (dict(max_tokens=0), "empty plans"), (dict(max_tokens=1 << 28, max_nodes=1024), "2\\^30")):
        with pytest.raises(hip.MlqError, match=what):
            tree(**bad)
    plain = hip.KvPlan(cache, 4, max_seqs=2, max_tokens=16, max_pages=4)
    p = tree()
    ints = [hip.DeviceBuffer(4 * 16) for _ in range(5)]
    logits = hip.DeviceBuffer(4 * 16 * 10)
    for call, what in ((lambda: plain.set([1], [1], [0], parents=[-1]), "holds no trees"),
                       (lambda: plain.keep([], []), "holds no trees"),
                       (lambda: plain.pick(logits, 10, *ints), "holds no trees"),
                       (lambda: p.pick(logits, 10, *ints), "holds no batch"), (lambda: p.keep([], []), "holds no batch"),
                       (lambda: p.set([9], [9], [0], parents=[-1] * 9), "9 nodes, the plan's trees hold 8"),
                       (lambda: p.set([9], [9], [0]), "9 nodes"),
                       (lambda: p.set([2], [2], [0], parents=[-1, 1]), "node 1 has parent 1"),
                       (lambda: p.set([2], [2], [0], parents=[0, 0]), "node 0 has parent 0"),
                       (lambda: p.set([2], [2], [0], parents=[-3, 0]), "parent -3")):
        with pytest.raises(hip.MlqError, match=what):
            call()
    with pytest.raises(ValueError):
        p.set([2], [2], [0], parents=[-1])
    p.set([3, 2], [3, 70], [0, 1, 2], parents=[-1, 0, 0, -1, 0])
    for bad in (lambda: p.keep([1], [0]), lambda: p.keep([1, 1], [0]), lambda: p.keep([1, 1], [0, 0, 0])):
        with pytest.raises(ValueError):
            bad()
    for call, what in ((lambda: p.keep([2, 0], [0, 3]), "kept node 3"), (lambda: p.keep([3, 0], [0, 1, 2]), "not a child of node 1"),
                       (lambda: p.keep([4, 0], [0, 1, 2, 2]), "4 of 3"), (lambda: p.keep([0, 1], [1]), "not a child of what came before"),
                       (lambda: p.pick(logits, 0, *ints), "vocabulary"), (lambda: p.pick(logits, 2 ** 30 + 1, *ints), "vocabulary"), (lambda: p.pick(logits, 100, *ints), "too small"),
                       (lambda: p.pick(None, 10, *ints), "null"), (lambda: p.pick(logits, 10, None, *ints[1:]), "null"),
                       (lambda: p.pick(logits, 10, *ints[:4], None), "null"),
                       (lambda: p.pick(logits.ptr + 2, 10, *ints), "aligned"),
                       (lambda: p.pick(logits, 10, ints[0], ints[0], *ints[2:]), "picks overlaps tokens"),
                       (lambda: p.pick(logits, 10, ints[0], ints[1], ints[2], ints[1], ints[4]), "kept overlaps picks"),
                       (lambda: p.pick(logits, 10, ints[0], ints[1], logits, ints[3], ints[4]), "n_kept overlaps logits")):
        with pytest.raises(hip.MlqError, match=what):
            call()
    for call, what in ((lambda: cache.copy_pages([0], [6]), "copy 0 is from page 0 to 6"), (lambda: cache.copy_pages([-1], [1]), "from page -1"),
                       (lambda: cache.copy_pages([0], [0]), "page 0 is read and written"),
                       (lambda: cache.copy_pages([0, 1], [1, 2]), "page 1 is read and written"),
                       (lambda: cache.copy_pages([0, 1], [2, 2]), "page 2 is written twice"),
                       (lambda: cache.copy_pages([0], [1], [65]), "65 positions"), (lambda: cache.copy_pages([0], [1], [-1]), "-1 positions")):
        with pytest.raises(hip.MlqError, match=what):
            call()
    with pytest.raises(ValueError):
        cache.copy_pages([0], [1, 2])
    with pytest.raises(ValueError):
        cache.copy_pages([0], [1], [1, 2])
    cache.copy_pages([], [])
    p.keep([0, 0], [])
    hip.synchronize(hip.stream(0))


def test_empty_batches(hip):
    cache = hip.KvCache(QT["q8_0"], 1, 4, 64, 2, 64)
    p = hip.KvPlan(cache, 4, max_seqs=2, max_tokens=8, max_pages=3, max_nodes=4)
    x, i = hip.DeviceBuffer(16), [hip.DeviceBuffer(16) for _ in range(4)]
    for args in (([], [], []), ([0], [0], []), ([0, 0], [0, 70], [1, 2])):
        p.set(*args, parents=[])
        p.write(0, x, x)
        p.attention(0, x, x)
        p.keep([0] * len(args[0]), [])
        i[1].upload(np.full(4, 5, np.int32))
        i[3].upload(np.full(4, 5, np.int32))
        p.pick(None, 10, None, *i)
        n = len(args[0])
        assert back(hip, i[1], (4,), np.int32).tolist() == [0] * n + [5] * (4 - n)
        assert back(hip, i[3], (4,), np.int32).tolist() == [-1] * n + [5] * (4 - n)
