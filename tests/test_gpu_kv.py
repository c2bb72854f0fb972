"""The paged key/value cache on the device (mlq_hip_kv_write / _read / _attention) against
plain numpy in 64 bits (kv_reference.py, where the attention's bound is derived)."""

import ctypes
import sys

import numpy as np
import pytest

from kv_reference import QT, Batch, attention, held, rotated, visible

pytestmark = pytest.mark.gpu
TYPES = list(QT)
THETA = 10000.0
BLOCK_BYTES = {"q8_0": 34, "q4_0": 18, "q4_1": 20}


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def dev(hip, a):
    return hip.DeviceBuffer.from_array(np.ascontiguousarray(a, np.float32))


def back(hip, buf, shape):
    hip.synchronize(hip.stream(0))
    return buf.download(np.float32, int(np.prod(shape))).reshape(shape)


class Case:
    """A cache whose sequences hold random keys and values, and a plan of its batch."""

    def __init__(self, hip, orc, kind, lens, heads=4, kv=2, hd=64, page=32, window=0, sinks=0, scale=0.0, seed=0,
                 layers=1, layer=0, keys=None, values=None, room=0):
        self.hip, self.kind, self.heads, self.kv, self.hd, self.layer = hip, kind, heads, kv, hd, layer
        self.window, self.sinks, self.scale = window, sinks, scale
        self.rng = np.random.default_rng(seed)
        self.batch = b = Batch(self.rng, lens, page)
        rand = self.rng.standard_normal
        self.k = rand((b.positions, kv, hd)).astype(np.float32) if keys is None else keys
        self.v = rand((b.positions, kv, hd)).astype(np.float32) if values is None else values
        self.q = (1.5 * rand((b.tokens, heads, hd))).astype(np.float32)
        self.cache = hip.KvCache(QT[kind], layers, b.n_pages, page, kv, hd)
        size = dict(max_seqs=max(1, len(lens)), max_pages=max(1, b.entries))
        fill = hip.KvPlan(self.cache, heads, max_tokens=max(1, b.positions), **size)
        fill.set(b.kv_len, b.kv_len, b.pages)
        if b.positions:
            fill.write(layer, dev(hip, self.k), dev(hip, self.v))
        hip.synchronize(hip.stream(0))
        self.plan = hip.KvPlan(self.cache, heads, max_tokens=max(1, b.tokens + room), window=window, sinks=sinks,
                               scale=scale, **size)
        self.plan.set(b.new, b.kv_len, b.pages)
        self.held = held(orc, kind, self.k), held(orc, kind, self.v)

    def run(self, q=None, plan=None):
        """The attention's output; two rows behind the last token have to stay as they were."""
        q = self.q if q is None else q
        n = self.batch.tokens
        mark = np.full((n + 2, self.heads, self.hd), 7.25, np.float32)
        out = dev(self.hip, mark)
        dq = dev(self.hip, np.concatenate([q, np.full((2,) + q.shape[1:], np.nan, np.float32)]))
        (plan or self.plan).attention(self.layer, dq, out)
        got = back(self.hip, out, mark.shape)
        assert (got[n:] == 7.25).all(), "rows behind the last token"
        return got[:n]

    def check(self, got=None, lens=None):
        got = self.run() if got is None else got
        at = qat = 0
        for n, t in self.batch.lens:
            if n:
                k, v = (x[at:at + t] for x in self.held)
                want, bound = attention(self.q[qat:qat + n], k, v, self.window, self.sinks, self.scale)
                err = np.abs(got[qat:qat + n] - want)
                assert (err <= bound).all(), (n, t, float((err / bound).max()))
            at, qat = at + t, qat + n
        return got


# ---------------------------------------------------------------- write and read back

SHAPES = [  # lens, heads, kv, hd, page
    ([(1, 1)], 1, 1, 8, 32),
    ([(1, 33), (1, 32), (1, 64), (1, 100)], 4, 2, 64, 32),
    ([(40, 40), (3, 95), (0, 10), (0, 0), (64, 64), (32, 96)], 2, 2, 32, 32),
    ([(70, 130), (129, 129)], 7, 1, 80, 64),
    ([(33, 65)], 2, 2, 40, 128),
    ([(35, 70), (1, 7)], 8, 2, 128, 64),
    ([(34, 50)], 3, 3, 160, 32),
    ([(33, 33), (2, 258)], 2, 1, 256, 256),
    ([(32, 32)], 1, 1, 24, 32),
    ([(5, 300)], 2, 1, 104, 1024),
]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_write_read(hip, orc, kind, shape):
    """Written in two goes (what was there, then the batch's tokens): every position reads
    back as the block formats' own bits, new tokens alone as well."""
    lens, heads, kv, hd, page = SHAPES[shape]
    rng = np.random.default_rng(shape)
    b = Batch(rng, lens, page)
    k, v = (rng.standard_normal((b.positions, kv, hd)).astype(np.float32) for _ in range(2))
    k[0, 0] = 0.0
    v[-1, -1, : hd // 2] = 3.0
    cache = hip.KvCache(QT[kind], 2, b.n_pages, page, kv, hd)
    plan = hip.KvPlan(cache, heads, max_seqs=len(lens), max_tokens=b.positions, max_pages=b.entries)
    before = [t - n for n, t in lens]
    first = Batch(rng, [(t, t) for t in before], page)
    keep = np.setdiff1d(np.arange(b.positions), b.rows())
    pages, at = [], 0
    for t, c in zip(b.kv_len, before):
        pages += b.pages[at:at + -(-c // page)]
        at += -(-t // page)
    plan.set(before, before, pages)
    if first.tokens:
        plan.write(1, dev(hip, k[keep]), dev(hip, v[keep]))
    plan.set(b.new, b.kv_len, b.pages)
    dk, dv = dev(hip, k[b.rows()]), dev(hip, v[b.rows()])
    plan.write(1, dk, dv)
    say("write_read", kind, shape)
    n = (b.positions + 1, kv, hd)
    ok, ov = (dev(hip, np.full(n, 9.5, np.float32)) for _ in range(2))
    plan.read(1, ok, ov)
    for got, x in ((back(hip, ok, n), k), (back(hip, ov, n), v)):
        assert np.array_equal(got[:-1], held(orc, kind, x))
        assert (got[-1] == 9.5).all()
    nk, nv = (dev(hip, np.full((b.tokens + 1, kv, hd), 9.5, np.float32)) for _ in range(2))
    plan.read(1, nk, nv, new_only=True)
    for got, x in ((back(hip, nk, (b.tokens + 1, kv, hd)), k), (back(hip, nv, (b.tokens + 1, kv, hd)), v)):
        assert np.array_equal(got[:-1], held(orc, kind, x)[b.rows()])
        assert (got[-1] == 9.5).all()
    # the other layer is as it was created
    plan.read(0, ok, ov)
    assert not back(hip, ok, n)[:-1].any() and not back(hip, ov, n)[:-1].any()


@pytest.mark.parametrize("kind", TYPES)
def test_write_special_values(hip, orc, kind):
    """Zeros, constants, scales that under- and overflow binary16, ties, NaN and Inf: the blocks
    of mlq_hip_quantize (a code of NaN is not defined on the host)."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((64, 1, 64)).astype(np.float32)
    x[1] = 0.0
    x[2] = 3.0
    x[3] = -0.0
    x[4] *= 1e-30
    x[5] *= 1e-7
    x[6] *= 1e6
    x[7] = np.round(x[7] * 8) / 8
    x[8, 0, 5] = 65519.996
    x[9, 0, 3] = np.nan
    x[10, 0, 40] = np.inf
    x[11, 0, 2] = -np.inf
    x[12] = np.nan
    cache = hip.KvCache(QT[kind], 1, 2, 32, 1, 64)
    plan = hip.KvPlan(cache, 1, max_seqs=1, max_tokens=64, max_pages=2)
    for n in (64, 1):  # whole tiles, and slot by slot into the same pages
        for t in range(0, 64, n):
            plan.set([n], [t + n], [1, 0][:-(-(t + n) // 32)])
            plan.write(0, dev(hip, x[t:t + n]), dev(hip, x[t:t + n]))
        ok, ov = hip.DeviceBuffer(x.nbytes), hip.DeviceBuffer(x.nbytes)
        plan.set([0], [64], [1, 0])
        plan.read(0, ok, ov)
        want = x
        if kind != "f32":
            blocks = hip.DeviceBuffer(128 * BLOCK_BYTES[kind])
            hip.quantize_device(QT[kind], dev(hip, x), 64, 64, blocks)
            blocks = back(hip, blocks, (32 * BLOCK_BYTES[kind],)).view(np.uint8).reshape(128, -1)
            with np.errstate(invalid="ignore"):
                want = orc.dequantize(QT[kind], blocks, 64, 64).reshape(x.shape)
        assert np.array_equal(back(hip, ok, x.shape), want, equal_nan=True)
        assert np.array_equal(back(hip, ov, x.shape), want, equal_nan=True)


@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("kind,heads,kv,hd", [("q8_0", 4, 2, 64), ("f32", 7, 1, 80), ("q4_0", 2, 2, 24),
                                              ("q4_1", 8, 4, 128), ("f32", 2, 1, 256), ("q8_0", 3, 3, 8)])
def test_write_rotated(hip, orc, kind, heads, kv, hd, neox):
    """RoPE in 64 bits, rounded once: queries and f32 keys are off by half a step of f32 and
    a value next to a tie may round to the other side of it (2^-24 relative, and 2^-52 of the two products)."""
    rng = np.random.default_rng(hd)
    page = 64
    lens = [(40, 40), (1, 77), (0, 5), (3, 60000), (34, 98)]
    b = Batch(rng, lens, page)
    k, v = (rng.standard_normal((b.tokens, kv, hd)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((b.tokens, heads, hd)).astype(np.float32)
    cache = hip.KvCache(QT[kind], 1, b.n_pages, page, kv, hd)
    plan = hip.KvPlan(cache, heads, max_seqs=5, max_tokens=b.tokens, max_pages=b.entries)
    plan.set(b.new, b.kv_len, b.pages)
    dq, oq = dev(hip, q), dev(hip, np.full((b.tokens + 1, heads, hd), 9.5, np.float32))
    plan.write(0, dev(hip, k), dev(hip, v), q=dq, q_out=oq, theta=THETA, neox=neox)
    got = back(hip, oq, (b.tokens + 1, heads, hd))
    assert (got[-1] == 9.5).all()
    want = rotated(q, b.pos(), THETA, neox)
    pair = np.sqrt(2) * np.abs(q).max()
    assert (np.abs(got[:-1].astype(np.float64) - want) <= np.spacing(np.abs(want)) + pair * 2.0 ** -40).all()
    assert np.mean(got[:-1] != want) < 1e-3
    nk, nv = hip.DeviceBuffer(k.nbytes), hip.DeviceBuffer(v.nbytes)
    plan.read(0, nk, nv, new_only=True)
    kr = rotated(k, b.pos(), THETA, neox)
    gk = back(hip, nk, k.shape)
    if kind == "f32":
        assert (np.abs(gk.astype(np.float64) - kr) <= np.spacing(np.abs(kr)) + pair * 2.0 ** -40).all()
    else:
        # the same codes but where a rounding moved one (a key in 10^5 or so)
        assert np.mean(gk != held(orc, kind, kr)) < 1e-3
    assert np.array_equal(back(hip, nv, v.shape), held(orc, kind, v))
    # in place
    plan.write(0, dev(hip, k), dev(hip, v), q=dq, q_out=dq, theta=THETA, neox=neox)
    assert np.array_equal(back(hip, dq, q.shape), got[:-1])


def test_write_leaves_neighbours(hip, orc):
    """Tokens of two sequences in slots of one page, and a rewritten slot: everything else stays."""
    rng = np.random.default_rng(1)
    for kind in TYPES:
        x = rng.standard_normal((32, 2, 64)).astype(np.float32)
        cache = hip.KvCache(QT[kind], 1, 1, 32, 2, 64)
        plan = hip.KvPlan(cache, 2, max_seqs=2, max_tokens=32, max_pages=2)
        plan.set([32], [32], [0])
        plan.write(0, dev(hip, x), dev(hip, -x))
        y = rng.standard_normal((9, 2, 64)).astype(np.float32)
        plan.set([2, 7], [12, 25], [0, 0])
        plan.write(0, dev(hip, y), dev(hip, 2 * y))
        want_k, want_v = x.copy(), -x
        want_k[10:12], want_k[18:25] = y[:2], y[2:]
        want_v[10:12], want_v[18:25] = 2 * y[:2], 2 * y[2:]
        plan.set([0], [32], [0])
        ok, ov = hip.DeviceBuffer(x.nbytes), hip.DeviceBuffer(x.nbytes)
        plan.read(0, ok, ov)
        assert np.array_equal(back(hip, ok, x.shape), held(orc, kind, want_k)), kind
        assert np.array_equal(back(hip, ov, x.shape), held(orc, kind, want_v)), kind


# ---------------------------------------------------------------- attention

ATTEND = [  # lens, heads, kv, hd, page, window, sinks
    ([(1, 1)], 1, 1, 8, 32, 0, 0),
    ([(1, 1), (1, 2), (1, 31), (1, 32), (1, 33), (1, 64), (1, 65), (0, 9), (0, 0), (1, 300)], 4, 2, 64, 32, 0, 0),
    ([(1, 1000), (1, 17)], 8, 1, 128, 64, 0, 0),
    ([(1, 500), (1, 130)], 3, 3, 80, 256, 0, 0),
    ([(1, 700)], 14, 2, 64, 32, 0, 0),
    ([(1, 333), (2, 64)], 16, 1, 64, 64, 0, 0),
    ([(2, 40), (5, 5), (4, 129)], 4, 2, 32, 32, 0, 0),
    ([(3, 50), (130, 130), (33, 200), (1, 70)], 4, 4, 128, 64, 0, 0),
    ([(65, 300)], 7, 1, 64, 32, 0, 0),
    ([(40, 40), (70, 133)], 2, 2, 96, 128, 0, 0),
    ([(37, 90)], 2, 1, 256, 32, 0, 0),
    ([(1, 400), (9, 60)], 4, 2, 160, 64, 0, 0),
    ([(1, 100), (1, 3), (1, 64), (20, 200)], 4, 2, 64, 32, 16, 0),
    ([(1, 500), (50, 300), (1, 20)], 4, 2, 64, 32, 40, 4),
    ([(1, 500), (100, 300)], 2, 2, 128, 64, 1, 0),
    ([(1, 700), (70, 400)], 2, 1, 64, 64, 1, 33),
    ([(1, 900), (200, 900)], 2, 1, 32, 32, 100, 70),
    ([(300, 600)], 32, 32, 32, 64, 128, 1),
]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("shape", range(len(ATTEND)))
def test_attention(hip, orc, kind, shape):
    lens, heads, kv, hd, page, window, sinks = ATTEND[shape]
    say("attention", kind, shape)
    Case(hip, orc, kind, lens, heads, kv, hd, page, window, sinks, seed=shape).check()


@pytest.mark.parametrize("kind", TYPES)
def test_attention_long(hip, orc, kind):
    """A context long enough to be split over workgroups, beside short ones; twice the same bits."""
    c = Case(hip, orc, kind, [(1, 9001), (1, 5), (2, 6000)], 8, 2, 64, 64, seed=11)
    got = c.check()
    assert np.array_equal(got, c.run())
    wide = Case(hip, orc, kind, [(40, 7000)], 4, 2, 64, 128, seed=12)
    got = wide.check()
    assert np.array_equal(got, wide.run())


HEAD_DIMS = [8, 24, 40, 72, 104, 136, 160, 192, 200, 224, 248, 256]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("hd", HEAD_DIMS)
def test_attention_head_dims(hip, orc, kind, hd):
    """Every number of blocks a head, whole and not, with one row, some and many."""
    say("head_dim", kind, hd)
    Case(hip, orc, kind, [(1, 70), (70, 101), (13, 45)], 4, 2, hd, 32, seed=hd).check()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows", [7, 8, 9, 16, 17, 63, 64, 65, 127, 128, 129, 191, 257])
def test_attention_row_counts(hip, orc, kind, rows):
    """Rows at and around what one workgroup takes, over short contexts and ones that are split."""
    say("rows", kind, rows)
    for t in (rows, rows + 31, rows + 2500):
        Case(hip, orc, kind, [(rows, t)], 1, 1, 64, 64, seed=rows).check()
    Case(hip, orc, kind, [(rows, rows + 1700), (1, 33)], 6, 2, 32, 64, window=1500, sinks=5, seed=rows).check()


def test_attention_of_many_sequences(hip, orc):
    """A batch of 300 short sequences of every kind, and one sequence listed twice (a page may be
    in several sequences as long as no two new tokens share a slot)."""
    rng = np.random.default_rng(31)
    lens = [(int(min(n, t)), int(t)) for n, t in zip(rng.choice([0, 1, 1, 1, 2, 9, 40], 300), rng.integers(0, 150, 300))]
    Case(hip, orc, "q4_0", lens, 8, 2, 64, 32, seed=32).check()
    c = Case(hip, orc, "q8_0", [(1, 90)], 4, 2, 64, 32, seed=33)
    twice = hip.KvPlan(c.cache, 4, max_seqs=2, max_tokens=2, max_pages=6)
    pages = c.batch.pages
    with pytest.raises(hip.MlqError, match="slot"):
        twice.set([1, 1], [90, 90], pages + pages)
    twice.set([1, 1], [90, 89], pages + pages)
    q = np.concatenate([c.q, c.q])
    out = hip.DeviceBuffer(q.nbytes)
    twice.attention(0, dev(hip, q), out)
    got = back(hip, out, q.shape)
    for i, t in enumerate((90, 89)):
        want, bound = attention(c.q, c.held[0][:t], c.held[1][:t])
        assert (np.abs(got[i] - want[0]) <= bound[0]).all()


def test_attention_scale_and_peaks(hip, orc):
    """A scale of one's own, scores of hundreds (one position takes all), equal scores."""
    Case(hip, orc, "q8_0", [(5, 200), (1, 90)], 4, 2, 64, scale=0.02, seed=1).check()
    Case(hip, orc, "f32", [(5, 200), (1, 90)], 4, 2, 64, scale=3.0, seed=2).check()
    Case(hip, orc, "f32", [(5, 200), (1, 90)], 4, 2, 64, scale=-0.3, seed=2).check()
    k = np.tile(np.random.default_rng(0).standard_normal((1, 2, 64)).astype(np.float32), (300, 1, 1))
    Case(hip, orc, "q4_1", [(1, 300)], 4, 2, 64, keys=k, seed=3).check()


@pytest.mark.parametrize("size", [1e-20, 1e-6, 1e5, 1e20])
def test_attention_value_range(hip, orc, size):
    """f32 values and keys far from 1: fp16 parts are taken relative to a block's largest."""
    rng = np.random.default_rng(4)
    v = (rng.standard_normal((150, 2, 64)) * size).astype(np.float32)
    Case(hip, orc, "f32", [(1, 150)], 4, 2, 64, values=v).check()
    v[::3] *= 1e-4
    v[1::5] = 0.0
    k = rng.standard_normal((150, 2, 64)).astype(np.float32)
    Case(hip, orc, "f32", [(7, 150)], 4, 2, 64, values=v, keys=k).check()
    k = (k * size).astype(np.float32)
    Case(hip, orc, "f32", [(7, 150)], 4, 2, 64, keys=k, scale=float(0.1 / size)).check()


@pytest.mark.parametrize("size", [1e-20, 1e-6, 1e5, 1e20])
@pytest.mark.parametrize("new", [3, 70])
def test_attention_range_of_all_three(hip, orc, new, size):
    """Queries of zeros and tiny ones beside ordinary ones, keys and values far from 1."""
    rng = np.random.default_rng(14)
    v = (rng.standard_normal((150, 2, 64)) * size).astype(np.float32)
    k = rng.standard_normal((150, 2, 64)).astype(np.float32)
    for keys, scale in ((k, 0.0), ((k * size).astype(np.float32), float(0.1 / size))):
        c = Case(hip, orc, "f32", [(new, 150)], 4, 2, 64, keys=keys, values=v, scale=scale)
        c.q[0] = 0.0
        c.q[1, 1] *= np.float32(1e-30)
        c.q[2, 3] *= np.float32(1e-36)
        c.q[1, 2, 1:] = 0.0
        c.check()
    # keys near the largest that count as finite, small queries
    c = Case(hip, orc, "f32", [(new, 150)], 4, 2, 64, keys=(k * 2e23).astype(np.float32), values=v)
    c.q *= np.float32(2e-23)
    c.check()


@pytest.mark.parametrize("new", [3, 70])
def test_attention_values_of_many_sizes(hip, orc, new):
    """f32 values whose sizes differ by 2^150 between positions: the sum of the weights holds those of the
    positions whose values are small, also where a tile of large ones comes behind them."""
    rng = np.random.default_rng(15)
    k, v = (rng.standard_normal((300, 2, 64)).astype(np.float32) for _ in range(2))
    any_size = (v * 10.0 ** rng.uniform(-22, 22, (300, 1, 1))).astype(np.float32)
    Case(hip, orc, "f32", [(new, 300)], 4, 2, 64, keys=k, values=any_size).check()
    for first, then in ((1e-23, 1e23), (1e23, 1e-23)):
        sizes = np.where(np.arange(300) < 150, first, then)[:, None, None]
        # scores of 0 where values are tiny, of about -14 where they are large
        keys = np.where(sizes < 1, 0.0, np.float32(-14.0 / 64)).astype(np.float32) * np.ones_like(k)
        c = Case(hip, orc, "f32", [(new, 300)], 4, 2, 64, keys=keys, values=(v * sizes).astype(np.float32), scale=1.0)
        c.q[:] = 1.0
        c.check()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, np.float32(-3.4e38)])
def test_attention_unseen_places(hip, orc, kind, bad):
    """What a token does not see has no part in its result: later tokens of its chunk, positions
    before its window, and what a page held before."""
    rng = np.random.default_rng(8)
    lens, window, sinks = [(40, 100), (1, 70)], 30, 3
    k, v = (rng.standard_normal((170, 2, 64)).astype(np.float32) for _ in range(2))
    plain = Case(hip, orc, kind, lens, 4, 2, 64, window=window, sinks=sinks, keys=k.copy(), values=v.copy(), seed=5)
    want = plain.run()
    for x in (k, v):
        x[3:31] = bad      # before every window of the first sequence (31 is the first seen)
        x[90:100] = bad    # its last ten tokens
        x[103:140] = bad   # before the second's window
    with np.errstate(all="ignore"):
        c = Case(hip, orc, kind, lens, 4, 2, 64, window=window, sinks=sinks, keys=k, values=v, seed=5)
    got = c.run()
    clean = np.r_[0:30, 40]
    assert np.array_equal(got[clean], want[clean])
    # Where the cache holds such values, what sees them shows it.  (The quantizers leave NaN out
    # of a block's scale, and Q4_1 a block of one infinity: those hold zeros.)
    hk, hv = hip.DeviceBuffer(41 * 128 * 4), hip.DeviceBuffer(41 * 128 * 4)
    c.plan.read(0, hk, hv, new_only=True)
    holds = np.isfinite(back(hip, hv, (41, 2, 64))[30:40])
    assert holds.all() if kind != "f32" and (np.isnan(bad) or (kind == "q4_1" and bad == np.inf)) else \
        not (holds.any() and bad != np.float32(-3.4e38))
    if not holds.any() or kind == "f32":
        assert not np.isfinite(got[30:40]).any()
    # a page that held such values is used again by a shorter sequence
    cache = hip.KvCache(QT[kind], 1, 1, 64, 2, 64)
    plan = hip.KvPlan(cache, 4, max_seqs=1, max_tokens=64, max_pages=1)
    plan.set([64], [64], [0])
    all_bad = np.full((64, 2, 64), bad, np.float32)
    plan.write(0, dev(hip, all_bad), dev(hip, all_bad))
    x = rng.standard_normal((37, 2, 64)).astype(np.float32)
    plan.set([37], [37], [0])
    plan.write(0, dev(hip, x), dev(hip, x))
    q = rng.standard_normal((37, 4, 64)).astype(np.float32)
    out = hip.DeviceBuffer(q.nbytes)
    plan.attention(0, dev(hip, q), out)
    h = held(orc, kind, x)
    want, bound = attention(q, h, h)
    assert (np.abs(back(hip, out, q.shape) - want) <= bound).all()


def test_attention_nonfinite_block_counts_as_nan(hip, orc):
    """A seen block that holds one element that is not finite: a value's is NaN in its 32
    dimensions, a key's makes the row NaN; other dimensions and heads stay."""
    rng = np.random.default_rng(2)
    k, v = (rng.standard_normal((60, 2, 64)).astype(np.float32) for _ in range(2))
    v[50, 0, 40] = np.inf
    c = Case(hip, orc, "f32", [(3, 60), ], 4, 2, 64, keys=k, values=v)
    got = c.run()
    assert np.isnan(got[:, :2, 32:]).all() and np.isfinite(got[:, :2, :32]).all() and np.isfinite(got[:, 2:]).all()
    v[50, 0, 40] = 0
    k[20, 1, 3] = np.nan
    got = Case(hip, orc, "f32", [(3, 60), ], 4, 2, 64, keys=k, values=v).run()
    assert np.isnan(got[:, 2:]).all() and np.isfinite(got[:, :2]).all()
    q = c.q.copy()
    q[1, 3, 5] = np.nan
    got = Case(hip, orc, "q8_0", [(3, 60), ], 4, 2, 64).run(q)
    assert np.isnan(got[1, 3]).all() and np.isfinite(got[[0, 2]]).all() and np.isfinite(got[1, :3]).all()


def test_window_moves_with_the_token(hip, orc):
    """A token alone and the same token inside a chunk see the same positions."""
    rng = np.random.default_rng(6)
    k, v = (rng.standard_normal((200, 2, 64)).astype(np.float32) for _ in range(2))
    for window, sinks in ((0, 0), (50, 0), (50, 4), (33, 40)):
        chunk = Case(hip, orc, "q8_0", [(90, 200)], 4, 2, 64, window=window, sinks=sinks, keys=k, values=v)
        got = chunk.check()
        for i in (0, 31, 89):
            t = 111 + i
            one = Case(hip, orc, "q8_0", [(1, t)], 4, 2, 64, window=window, sinks=sinks, keys=k[:t], values=v[:t])
            one.q = chunk.q[i:i + 1]
            one.check()
            see = visible(90, 200, window, sinks)[i].sum()
            assert see == (t if not window else min(t, window + min(sinks, max(0, t - window)))), (window, sinks, i)
            scale = np.abs(v).max()
            assert np.abs(one.run() - got[i]).max() < 1e-5 * scale


# ---------------------------------------------------------------- used together, streams, graphs

@pytest.mark.parametrize("kind", TYPES)
def test_serving_run(hip, orc, kind):
    """Three sequences: prompts in chunks, then token by token, two layers, a shared prefix page."""
    rng = np.random.default_rng(9)
    heads, kv, hd, page = 4, 2, 64, 32
    cache = hip.KvCache(QT[kind], 2, 20, page, kv, hd)
    plan = hip.KvPlan(cache, heads, max_seqs=3, max_tokens=128, max_pages=20)
    tables = [[4, 9, 1, 0], [4, 7, 12, 13], [2, 3, 5, 6]]  # page 4: a prefix of the first two
    shown_k = [[np.zeros((0, kv, hd), np.float32)] * 3 for _ in range(2)]
    shown_v = [[np.zeros((0, kv, hd), np.float32)] * 3 for _ in range(2)]
    length = [0, 0, 0]
    steps = [[32, 0, 40], [17, 0, 1], [1, 0, 1], [1, 20, 1], [1, 1, 0], [0, 1, 1], [1, 1, 1], [1, 1, 9]]
    for step, new in enumerate(steps):
        if step == 3:  # the second sequence starts from the first one's page
            length[1] = 32
            for layer in range(2):
                shown_k[layer][1], shown_v[layer][1] = (s[layer][0][:32] for s in (shown_k, shown_v))
        length = [t + n for t, n in zip(length, new)]
        pages = sum((tables[i][:-(-length[i] // page)] for i in range(3)), [])
        plan.set(new, length, pages)
        for layer in range(2):
            n = sum(new)
            k, v = (rng.standard_normal((n, kv, hd)).astype(np.float32) for _ in range(2))
            q = rng.standard_normal((n, heads, hd)).astype(np.float32)
            dq, out = dev(hip, q), hip.DeviceBuffer(q.nbytes)
            plan.write(layer, dev(hip, k), dev(hip, v), q=dq, q_out=dq, theta=THETA)
            plan.attention(layer, dq, out)
            got = back(hip, out, q.shape)
            pos = np.concatenate([np.arange(t - m, t) for m, t in zip(new, length)])
            kr, qr = rotated(k, pos, THETA, False), rotated(q, pos, THETA, False)
            at = 0
            for i, m in enumerate(new):
                shown_k[layer][i] = np.concatenate([shown_k[layer][i], kr[at:at + m]])
                shown_v[layer][i] = np.concatenate([shown_v[layer][i], v[at:at + m]])
                if m:
                    kk, vv = held(orc, kind, shown_k[layer][i]), held(orc, kind, shown_v[layer][i])
                    want, bound = attention(qr[at:at + m], kk, vv)
                    # a rotated element one f32 step off moves a score by 2^-23 of its size:
                    # twice the bound covers it; a code next to a tie could move (none here)
                    assert (np.abs(got[at:at + m] - want) <= 2 * bound).all(), (step, layer, i)
                at += m


def test_other_stream_and_two_plans(hip, orc):
    """Two plans (full and windowed layers) of one cache on streams of their own, calls interleaved."""
    a = Case(hip, orc, "q8_0", [(1, 3000), (40, 200)], 8, 2, 128, 64, seed=21)
    b = a.batch
    win = hip.KvPlan(a.cache, 8, max_seqs=2, max_tokens=b.tokens, max_pages=b.entries, window=64, sinks=2)
    s1, s2 = hip.stream_create(), hip.stream_create()
    win.set(b.new, b.kv_len, b.pages, stream=s2)
    dq = dev(hip, a.q)
    o1, o2 = hip.DeviceBuffer(a.q.nbytes), hip.DeviceBuffer(a.q.nbytes)
    hip.synchronize(hip.stream(0))
    for _ in range(20):
        a.plan.attention(0, dq, o1, stream=s1)
        win.attention(0, dq, o2, stream=s2)
    hip.synchronize(s1)
    hip.synchronize(s2)
    a.check(o1.download(np.float32, a.q.size).reshape(a.q.shape))
    a.window, a.sinks = 64, 2
    a.check(o2.download(np.float32, a.q.size).reshape(a.q.shape))
    for s in (s1, s2):
        hip.stream_destroy(s)


def test_graph_serves_later_batches(hip, orc):
    """A recorded write, read back and attention, replayed with batches set after the recording:
    longer, shorter, of one token and of chunks, split and not."""
    rng = np.random.default_rng(13)
    heads, kv, hd, page, most = 8, 2, 64, 32, 96
    cache = hip.KvCache(QT["q8_0"], 1, 160, page, kv, hd)
    plan = hip.KvPlan(cache, heads, max_seqs=4, max_tokens=most, max_pages=150)
    fill = hip.KvPlan(cache, heads, max_seqs=4, max_tokens=5000, max_pages=160)
    s = hip.stream_create()
    dk, dv, dq, out = (hip.DeviceBuffer(4 * most * n * hd) for n in (kv, kv, heads, heads))
    rk, rv = (hip.DeviceBuffer(4 * most * kv * hd) for _ in range(2))

    def batch(lens):
        b = Batch(rng, lens, page, spare=0)
        k, v = (rng.standard_normal((b.positions, kv, hd)).astype(np.float32) for _ in range(2))
        q = rng.standard_normal((b.tokens, heads, hd)).astype(np.float32)
        fill.set(b.kv_len, b.kv_len, b.pages)
        fill.write(0, dev(hip, k), dev(hip, v))
        hip.synchronize(hip.stream(0))
        plan.set(b.new, b.kv_len, b.pages, stream=s)
        hip.synchronize(s)
        for d, x in ((dk, k[b.rows()]), (dv, v[b.rows()]), (dq, q)):
            if x.size:
                d.upload(x)
        return b, k, v, q

    def step():
        plan.write(0, dk, dv, stream=s)
        plan.read(0, rk, rv, new_only=True, stream=s)
        plan.attention(0, dq, out, stream=s)

    batch([(1, 40)])
    g = hip.Graph.record(step, stream=s)
    for lens in ([(1, 40)], [(1, 4000)], [(90, 95), (1, 33)], [(1, 7), (1, 800), (1, 1), (1, 64)], [(40, 1500)], [],
                 [(96, 96)], [(0, 50)], [(1, 2)]):
        b, k, v, q = batch(lens)
        out.upload(np.full(most * heads * hd, 5.5, np.float32))
        for _ in range(3):
            g.launch(s)
        hip.synchronize(s)
        got = out.download(np.float32, most * heads * hd).reshape(most, heads, hd)
        assert (got[b.tokens:] == 5.5).all(), lens
        at = qat = 0
        kk, vv = held(orc, "q8_0", k), held(orc, "q8_0", v)
        if b.tokens:
            assert np.array_equal(rk.download(np.float32, b.tokens * kv * hd).reshape(-1, kv, hd), kk[b.rows()])
            assert np.array_equal(rv.download(np.float32, b.tokens * kv * hd).reshape(-1, kv, hd), vv[b.rows()])
        for n, t in lens:
            if n:
                want, bound = attention(q[qat:qat + n], kk[at:at + t], vv[at:at + t])
                assert (np.abs(got[qat:qat + n] - want) <= bound).all(), lens
            at, qat = at + t, qat + n
        # eager, the same bits where the work is split the same way
        plan.attention(0, dq, out, stream=s)
        hip.synchronize(s)
        assert np.array_equal(out.download(np.float32, most * heads * hd).reshape(got.shape), got), lens
    with pytest.raises(hip.MlqError, match="graph capture"):
        hip.Graph.record(lambda: plan.set([1], [1], [0], stream=s), stream=s)
    for create in (lambda: hip.KvCache(QT["q8_0"], 1, 4, 64, 2, 64),
                   lambda: hip.KvPlan(cache, heads, max_seqs=1, max_tokens=1, max_pages=1)):
        with pytest.raises(hip.MlqError, match="graph capture"):
            hip.Graph.record(create, stream=hip.stream(0))
    # recorded calls need room for the largest batch
    short = hip.DeviceBuffer(4 * 95 * heads * hd)
    with pytest.raises(hip.MlqError, match="too small"):
        hip.Graph.record(lambda: plan.attention(0, short, out, stream=s), stream=s)
    g.destroy()
    hip.stream_destroy(s)


@pytest.mark.parametrize("kind,hd", [(kind, 64) for kind in TYPES] + [("f32", 256), ("q4_1", 200)])
def test_recorded_write_of_whole_tiles(hip, orc, kind, hd):
    """A recorded rotation and write, replayed with whole tiles, single tokens and parts of tiles, eager calls
    between the replays."""
    rng = np.random.default_rng(19)
    heads, kv, page, most = 4, 2, 64, 200
    cache, want = (hip.KvCache(QT[kind], 1, 12, page, kv, hd) for _ in range(2))
    plan, eager = (hip.KvPlan(c, heads, max_seqs=3, max_tokens=most, max_pages=12) for c in (cache, want))
    s = hip.stream_create()
    dk, dv = (hip.DeviceBuffer(4 * most * kv * hd) for _ in range(2))
    dq, oq, eq = (hip.DeviceBuffer(4 * most * heads * hd) for _ in range(3))
    reads = [hip.DeviceBuffer(4 * 12 * page * kv * hd) for _ in range(4)]
    plan.set([1], [1], [0], stream=s)
    hip.synchronize(s)
    g = hip.Graph.record(lambda: plan.write(0, dk, dv, q=dq, q_out=oq, theta=THETA, neox=True, stream=s), stream=s)
    for new, length in (([128], [128]), ([1, 64, 3], [129, 64, 3]), ([0, 0, 1], [129, 64, 4]), ([31, 1, 100], [160, 65, 104])):
        pages = sum(([4 * i + j for j in range(-(-t // page))] for i, t in enumerate(length)), [])
        for d, n in ((dk, kv), (dv, kv), (dq, heads)):
            d.upload(rng.standard_normal(most * n * hd).astype(np.float32))
        for p in (plan, eager):
            p.set(new, length, pages, stream=s)
        oq.upload(np.full(most * heads * hd, 3.5, np.float32))
        eq.upload(np.full(most * heads * hd, 3.5, np.float32))
        for _ in range(2):
            g.launch(s)
            eager.write(0, dk, dv, q=dq, q_out=eq, theta=THETA, neox=True, stream=s)
            hip.synchronize(s)
        n = most * heads * hd
        assert np.array_equal(oq.download(np.float32, n), eq.download(np.float32, n))
        for p, (rk, rv) in ((plan, reads[:2]), (eager, reads[2:])):
            p.read(0, rk, rv, stream=s)
        hip.synchronize(s)
        n = sum(length) * kv * hd
        a, b, x, y = (r.download(np.float32, n) for r in reads)
        assert np.array_equal(a, x) and np.array_equal(b, y) and np.abs(a).max() > 0
    g.destroy()
    hip.stream_destroy(s)


def test_far_pages(hip, orc):
    """Pages beyond 4 GiB of a layer: offsets pass 32 bits."""
    rng = np.random.default_rng(17)
    kv, hd, page = 8, 128, 1024
    cache = hip.KvCache(QT["f32"], 2, 600, page, kv, hd)
    assert cache.info()["bytes"] > 2 * 4.9e9
    plan = hip.KvPlan(cache, kv, max_seqs=1, max_tokens=1100, max_pages=2)
    k, v = (rng.standard_normal((1100, kv, hd)).astype(np.float32) for _ in range(2))
    plan.set([1100], [1100], [599, 540])
    plan.write(1, dev(hip, k), dev(hip, v))
    ok, ov = hip.DeviceBuffer(k.nbytes), hip.DeviceBuffer(v.nbytes)
    plan.read(1, ok, ov)
    assert np.array_equal(back(hip, ok, k.shape), k) and np.array_equal(back(hip, ov, v.shape), v)
    plan.set([1], [1100], [599, 540])
    q = rng.standard_normal((1, kv, hd)).astype(np.float32)
    out = hip.DeviceBuffer(q.nbytes)
    plan.attention(1, dev(hip, q), out)
    want, bound = attention(q, k, v)
    assert (np.abs(back(hip, out, q.shape) - want) <= bound).all()


# ---------------------------------------------------------------- refusals

def test_refusals(hip):
    lib = hip.load()
    cache = hip.KvCache(QT["q8_0"], 2, 4, 64, 2, 64)
    info = cache.info()
    assert info == {"type": 1, "n_layers": 2, "n_pages": 4, "page_size": 64, "n_kv_heads": 2, "head_dim": 64,
                    "bytes": 2 * 4 * 64 * 2 * 2 * 2 * 34}

    def plan(*a, h=None):
        h = ctypes.c_void_p()
        return lib.mlq_hip_kv_plan_create(cache.h, *a, ctypes.byref(h))

    for a, code, what in (((3, 0, 0, 0.0, 1, 1, 1), 2, "3 heads over 2 KV heads"), ((0, 0, 0, 0.0, 1, 1, 1), 2, "0 heads"),
                          ((4, -1, 0, 0.0, 1, 1, 1), 1, "negative window"), ((4, 0, 2, 0.0, 1, 1, 1), 1, "sinks need a window"),
                          ((4, 5, -2, 0.0, 1, 1, 1), 1, "negative window or sinks"),
                          ((4, 0, 0, float("nan"), 1, 1, 1), 1, "scale"), ((4, 0, 0, 1e31, 1, 1, 1), 1, "2^100"),
                          ((4, 0, 0, float("-inf"), 1, 1, 1), 1, "scale"), ((4, 0, 0, -1e-31, 1, 1, 1), 1, "scale"),
                          ((4, 0, 0, 0.0, 0, 1, 1), 2, "empty plans"),
                          ((4, 0, 0, 0.0, 1, 0, 1), 2, "empty plans"), ((4, 0, 0, 0.0, 1, 1, -1), 2, "empty plans"),
                          ((4, 0, 0, 0.0, 1, 1 << 29, 1), 6, "2^30"), ((4, 0, 0, 0.0, 1, 1, 1 << 25), 6, "2^30")):
        assert plan(*a) == code, (a, hip.last_error())
        assert what in hip.last_error()
    p = hip.KvPlan(cache, 4, max_seqs=2, max_tokens=8, max_pages=3)
    x, y = hip.DeviceBuffer(4 * 8 * 4 * 64), hip.DeviceBuffer(4 * 8 * 4 * 64)
    with pytest.raises(hip.MlqError, match="holds no batch"):
        p.attention(0, x, y)
    p.set([2, 1], [70, 3], [0, 3, 1])
    for bad in (lambda: p.set([9], [9], [0]), lambda: p.set([1], [5], [4]), lambda: p.set([1], [200], [0, 1, 2, 3]),
                lambda: p.set([1, 1], [2, 2], [1, 1]), lambda: p.set([1, 1, 1], [2, 2, 2], [1, 2, 3])):
        with pytest.raises(hip.MlqError):
            bad()
    with pytest.raises(ValueError):
        p.set([1], [70], [0])
    # a refused set leaves the batch: three tokens
    small = hip.DeviceBuffer(4 * 3 * 4 * 64)
    p.attention(0, small, y)
    for call, what in ((lambda: p.attention(2, x, y), "layer 2 out of 2"), (lambda: p.attention(-1, x, y), "layer -1"),
                       (lambda: p.attention(0, None, y), "null"), (lambda: p.attention(0, x, None), "null"),
                       (lambda: p.attention(0, x, x), "overlaps"), (lambda: p.attention(0, x.ptr + 4, y), "aligned"),
                       (lambda: p.attention(0, hip.DeviceBuffer(4 * 3 * 4 * 64 - 4), y), "too small"),
                       (lambda: p.attention(0, np.zeros(4096, np.float32).ctypes.data // 16 * 16, y), "device pointer"),
                       (lambda: p.write(0, x, None), "null"), (lambda: p.write(2, x, y), "layer"),
                       (lambda: p.write(0, x, y, q=x), "come together"),
                       (lambda: p.write(0, x, y, q=small, q_out=small), "without a rotation"),
                       (lambda: p.write(0, x, y, theta=-1.0), "theta"), (lambda: p.write(0, x, y, theta=float("inf")), "theta"),
                       (lambda: p.write(0, x, y, q=small, q_out=x, theta=1e4), "overlaps"),
                       (lambda: p.write(0, x, y, q=small, q_out=small.ptr + 16, theta=1e4), "too small|overlaps"),
                       (lambda: p.read(0, x, x, new_only=True), "overlaps"), (lambda: p.read(0, x, y), "too small"),
                       (lambda: p.read(0, x.ptr + 8, y, new_only=True), "aligned")):
        with pytest.raises(hip.MlqError, match=what):
            call()
    hip.synchronize(hip.stream(0))


def test_a_failed_allocation_is_reported_once(hip, orc):
    """A cache that no card holds is refused with the allocation's error, and the calls after it work."""
    c = Case(hip, orc, "q8_0", [(1, 40)], 4, 2, 64)
    with pytest.raises(hip.MlqError, match="HIP error"):
        hip.KvCache(QT["f32"], 1000, 4000, 65536, 8, 128)  # 2 PB
    with pytest.raises(hip.MlqError, match="too large"):
        hip.KvCache(QT["f32"], 2 ** 31 - 1, 2 ** 31 - 1, 65536, 65536, 256)
    c.check()


def test_plan_outlives_its_cache_handle(hip, orc):
    c = Case(hip, orc, "q4_0", [(1, 50)], 4, 2, 64)
    want = c.run()
    c.cache.destroy()
    assert np.array_equal(c.run(), want)
    c.plan.destroy()


def test_empty_batches(hip, orc):
    cache = hip.KvCache(QT["q8_0"], 1, 4, 64, 2, 64)
    p = hip.KvPlan(cache, 4, max_seqs=2, max_tokens=8, max_pages=3)
    x = hip.DeviceBuffer(16)
    for args in (([], [], []), ([0], [0], []), ([0, 0], [0, 0], [])):
        p.set(*args)
        p.write(0, x, x)
        p.attention(0, x, x)
        p.read(0, x, x)
        p.read(0, x, x, new_only=True)
    p.set([0], [70], [0, 2])
    p.attention(0, x, x)
    p.write(0, x, x)
    hip.synchronize(hip.stream(0))
