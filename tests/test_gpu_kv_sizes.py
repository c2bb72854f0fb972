"""Attention over the paged cache where sizes differ inside a head: every block of 32 dimensions is
held to a bound of its own (kv_reference.attention_by_block), whatever the blocks beside it hold."""

import numpy as np
import pytest

from kv_reference import QT, attention, attention_by_block, held
from test_gpu_kv import Case, back, dev, say

pytestmark = pytest.mark.gpu


def check(c, dims=slice(None), heads=slice(None)):
    """The output against the 64-bit result, in `dims` of `heads`."""
    got = c.run()
    at = qat = 0
    for n, t in c.batch.lens:
        k, v = (x[at:at + t] for x in c.held)
        want, bound = attention_by_block(c.q[qat:qat + n], k, v, c.window, c.sinks, c.scale)
        err = np.abs(got[qat:qat + n] - want)
        ok = (err <= bound)[:, heads, dims]
        assert ok.all(), (n, t, float((err / np.maximum(bound, 1e-300))[:, heads, dims].max()))
        at, qat = at + t, qat + n
    return got


def spread(rng, positions, kv, hd, sizes):
    """Normal values whose blocks of 32 are of `sizes` in turn."""
    by = np.repeat(np.resize(np.asarray(sizes, np.float64), -(-hd // 32)), 32)[:hd]
    return (rng.standard_normal((positions, kv, hd)) * by).astype(np.float32)


FEW = [[(3, 60)], [(1, 90), (2, 40)], [(1, 5000)]]
VALUE_SIZES = [("f32", (1.0, 1e4)), ("f32", (1.0, 1e8)), ("f32", (1e20, 1e-3)), ("f32", (1e-20, 1e20)),
               ("q8_0", (1.0, 2e-4)), ("q8_0", (1e-3, 1e3)), ("q4_0", (2e-3, 1e4)), ("q4_1", (1e-3, 1e3))]


@pytest.mark.parametrize("kind,sizes", VALUE_SIZES)
@pytest.mark.parametrize("lens", FEW)
def test_few_rows_value_blocks_of_different_size(hip, orc, lens, kind, sizes):
    say("few rows, value blocks", kind, sizes, lens)
    for hd in (64, 80, 160):
        rng = np.random.default_rng(hd)
        c = Case(hip, orc, kind, lens, 4, 2, hd, values=spread(rng, sum(t for _, t in lens), 2, hd, sizes))
        check(c)


@pytest.mark.parametrize("kind,size", [("f32", 1e8), ("f32", 1e19), ("q8_0", 1e4), ("q4_0", 1e4), ("q4_1", 1e4)])
def test_few_rows_one_position_with_a_large_block(hip, orc, kind, size):
    """One position among sixty holds a block that is large; the other block of the head is as it was."""
    rng = np.random.default_rng(1)
    v = rng.standard_normal((60, 2, 64)).astype(np.float32)
    v[23, :, 32:] *= np.float32(size)
    check(Case(hip, orc, kind, [(3, 60)], 4, 2, 64, values=v))


@pytest.mark.parametrize("kind,bad", [("f32", np.inf), ("f32", np.nan), ("f32", 3e30), ("q8_0", 1e30), ("q4_0", -np.inf)])
def test_few_rows_healthy_block_beside_a_bad_one(hip, orc, kind, bad):
    """A value block that is not finite is NaN for what sees it, the head's other block what it is without it."""
    rng = np.random.default_rng(2)
    v = rng.standard_normal((60, 2, 64)).astype(np.float32)
    c = Case(hip, orc, kind, [(3, 60)], 4, 2, 64, values=v.copy())
    v[20, 0, 40] = bad
    with np.errstate(all="ignore"):
        worse = Case(hip, orc, kind, [(3, 60)], 4, 2, 64, values=v, keys=c.k)
    worse.held = c.held
    got = check(worse, dims=slice(0, 32))
    check(worse, heads=slice(2, 4))
    assert np.isnan(got[:, :2, 32:]).all()


@pytest.mark.parametrize("new", [3, 70])
@pytest.mark.parametrize("size", [1e6, -1e6])
def test_infinite_minimum_counts_as_nan(hip, orc, new, size):
    """A Q4_1 block of one large constant has a finite scale (0) and an infinite minimum: NaN for what sees it,
    whichever kernel the number of rows chooses."""
    rng = np.random.default_rng(3)
    v = rng.standard_normal((100, 2, 64)).astype(np.float32)
    c = Case(hip, orc, "q4_1", [(new, 100)], 4, 2, 64, values=v.copy())
    v[10, 1, 32:] = size
    worse = Case(hip, orc, "q4_1", [(new, 100)], 4, 2, 64, values=v, keys=c.k)
    worse.held = c.held
    got = check(worse, dims=slice(0, 32))
    check(worse, heads=slice(0, 2))
    assert np.isnan(got[:, 2:, 32:]).all()


@pytest.mark.parametrize("new", [3, 70])
@pytest.mark.parametrize("kind", list(QT))
def test_bad_block_counts_however_small_its_weight(hip, orc, kind, new):
    """A seen value block that is not finite is NaN for a token whose weight for it is below f32's range, and
    nothing to the tokens before it."""
    rng = np.random.default_rng(4)
    k, v = (rng.standard_normal((100, 2, 64)).astype(np.float32) for _ in range(2))
    k[98] = -40.0
    c = Case(hip, orc, kind, [(new, 100)], 4, 2, 64, keys=k, values=v.copy(), scale=1.0)
    c.q[:] = rng.uniform(1, 2, c.q.shape).astype(np.float32)
    v[98, 0, :32] = -1e30
    with np.errstate(all="ignore"):
        worse = Case(hip, orc, kind, [(new, 100)], 4, 2, 64, keys=k, values=v, scale=1.0)
    worse.q, worse.held = c.q, c.held
    got = check(worse, dims=slice(32, 64))
    check(worse, heads=slice(2, 4))
    assert np.isnan(got[-2:, :2, :32]).all() and np.isfinite(got[:-2]).all()


@pytest.mark.parametrize("kind,sizes", [("f32", (1.0, 1e-5)), ("f32", (1e8, 1.0)), ("f32", (1e18, 1e-18)), ("f32", (1.0, 0.0)),
                                        ("q8_0", (1e3, 1e-3)), ("q4_0", (1e4, 1e-3)), ("q4_1", (1e-3, 1e3))])
@pytest.mark.parametrize("lens", FEW)
def test_few_rows_query_blocks_of_different_size(hip, orc, lens, kind, sizes):
    """Small query blocks beside large ones, over keys whose blocks make up for it: both count in the score."""
    say("few rows, query blocks", kind, sizes, lens)
    rng = np.random.default_rng(5)
    for hd in (64, 80, 160):
        inverse = [1 / s if s else 1.0 for s in sizes]
        keys = spread(rng, sum(t for _, t in lens), 2, hd, inverse)
        c = Case(hip, orc, kind, lens, 4, 2, hd, keys=keys)
        c.q[::2] = spread(rng, len(c.q[::2]), 4, hd, sizes)
        c.q[1::2] = spread(rng, len(c.q[1::2]), 4, hd, [min(1.0, s) for s in sizes])
        check(c)


MANY = [[(70, 100)], [(200, 230), (1, 40)], [(33, 2500)]]


@pytest.mark.parametrize("kind,sizes", VALUE_SIZES)
@pytest.mark.parametrize("lens", MANY)
def test_many_rows_value_blocks_of_different_size(hip, orc, lens, kind, sizes):
    say("many rows, value blocks", kind, sizes, lens)
    for hd in (64, 80, 160):
        rng = np.random.default_rng(hd)
        check(Case(hip, orc, kind, lens, 4, 2, hd, values=spread(rng, sum(t for _, t in lens), 2, hd, sizes)))


@pytest.mark.parametrize("kind,sizes", [("f32", (1.0, 1e-5)), ("f32", (1e8, 1.0)), ("f32", (1e18, 1e-18)), ("f32", (1.0, 0.0)),
                                        ("q8_0", (1e3, 1e-3)), ("q4_0", (1e4, 1e-3)), ("q4_1", (1e-3, 1e3))])
@pytest.mark.parametrize("lens", MANY)
def test_many_rows_query_and_key_blocks_of_different_size(hip, orc, lens, kind, sizes):
    """Keys' blocks far apart in size, under queries that make up for it and under ones that read the small ones
    only; queries' blocks far apart."""
    say("many rows, key blocks", kind, sizes, lens)
    rng = np.random.default_rng(6)
    for hd in (64, 80, 160):
        inverse = [1 / s if s else 1.0 for s in sizes]
        c = Case(hip, orc, kind, lens, 4, 2, hd, keys=spread(rng, sum(t for _, t in lens), 2, hd, inverse))
        c.q[::2] = spread(rng, len(c.q[::2]), 4, hd, sizes)
        c.q[1::2] = spread(rng, len(c.q[1::2]), 4, hd, [min(1.0, s) if i < 1 else 0.0 for i, s in enumerate(sizes)])
        check(c)
        c = Case(hip, orc, kind, lens, 4, 2, hd)
        c.q[:] = spread(rng, len(c.q), 4, hd, [min(1.0, s) for s in sizes])
        check(c)


@pytest.mark.parametrize("kind", list(QT))
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 3)])
def test_many_rows_a_few_uneven_positions(hip, orc, kind, window, sinks):
    """Uneven positions that some rows see, in the middle of a long context whose parts are merged."""
    rng = np.random.default_rng(7)
    v, k = (rng.standard_normal((3000, 2, 96)).astype(np.float32) for _ in range(2))
    v[1500, :, 32:64] *= np.float32(3e4)
    v[2950, 1, :32] *= np.float32(1e-4)
    k[700, 0, 64:] *= np.float32(2e4)
    check(Case(hip, orc, kind, [(140, 3000)], 4, 2, 96, window=window, sinks=sinks, values=v, keys=k))


@pytest.mark.parametrize("kind,bad", [("f32", np.inf), ("f32", np.nan), ("f32", 3e30), ("q8_0", 1e30), ("q4_0", -np.inf)])
def test_many_rows_healthy_block_beside_a_bad_one(hip, orc, kind, bad):
    """As for few rows; the head's other blocks differ in size or not."""
    for size in (1.0, 1e-5):
        rng = np.random.default_rng(8)
        v = spread(rng, 100, 2, 96, (1.0, 1.0, size))
        c = Case(hip, orc, kind, [(70, 100)], 4, 2, 96, values=v.copy())
        v[20, 0, 40] = bad
        with np.errstate(all="ignore"):
            worse = Case(hip, orc, kind, [(70, 100)], 4, 2, 96, values=v, keys=c.k)
        worse.held = c.held
        got = check(worse, dims=np.r_[0:32, 64:96])
        check(worse, heads=slice(2, 4))
        assert np.isnan(got[:, :2, 32:64]).all()


@pytest.mark.parametrize("new", [3, 70])
def test_keys_below_the_floor_of_a_block(hip, orc, new):
    """f32 keys below 2^-80, which share one power of two, under a scale that makes their scores count."""
    rng = np.random.default_rng(9)
    k = (rng.standard_normal((150, 2, 64)) * 1e-25).astype(np.float32)
    check(Case(hip, orc, "f32", [(new, 150)], 4, 2, 64, keys=k, scale=1e24))


@pytest.mark.parametrize("kind", list(QT))
@pytest.mark.parametrize("new", [3, 70])
@pytest.mark.parametrize("size", [0.0, 1e-3, 1e-2])
def test_a_sink_with_small_values(hip, orc, kind, new, size):
    """A first position that takes nearly all the weight and whose values are zeros or small: the others' part of
    the result is what the smaller weights make it."""
    rng = np.random.default_rng(10)
    for gap in (12.0, 15.0, 20.0, 40.0):
        k, v = (rng.standard_normal((200, 2, 64)).astype(np.float32) for _ in range(2))
        k *= np.float32(0.05)
        k[0] = gap / 64
        v[0] *= np.float32(size)
        c = Case(hip, orc, kind, [(new, 200)], 4, 2, 64, keys=k, values=v, scale=1.0)
        c.q[:] = rng.uniform(0.9, 1.1, c.q.shape).astype(np.float32)
        check(c)


@pytest.mark.parametrize("kind", ["f32", "q8_0"])
@pytest.mark.parametrize("new", [3, 70])
def test_values_of_all_sizes_beside_each_other(hip, orc, kind, new):
    """Values of zero, tiny and large ones in turn, and a position that is all zeros in the middle of a tile."""
    rng = np.random.default_rng(11)
    v = rng.standard_normal((300, 2, 96)).astype(np.float32)
    v[1::5] = 0.0
    v[2::7] *= np.float32(3e-3)
    v[3::11] *= np.float32(100.0)
    check(Case(hip, orc, kind, [(new, 300)], 4, 2, 96, values=v))
    v = rng.standard_normal((300, 2, 96)).astype(np.float32)
    v[100] = 0.0
    check(Case(hip, orc, kind, [(new, 300)], 4, 2, 96, values=v))


def test_more_workgroups_than_a_launch_holds(hip, orc):
    """16400 decoding sequences of 1024 heads: 2^24 items and a few, whose workgroups would be more threads than a
    launch may have."""
    n, heads, hd, page = 16400, 1024, 8, 32
    rng = np.random.default_rng(12)
    some = rng.standard_normal((97, heads, hd)).astype(np.float32)
    k, v, q = (np.take(some, (np.arange(n) * step + 5) % 97, axis=0) for step in (1, 3, 7))
    cache = hip.KvCache(QT["q8_0"], 1, -(-n // page), page, heads, hd)
    plan = hip.KvPlan(cache, heads, max_seqs=n, max_tokens=n, max_pages=n)
    # sequence i: the first i % 32 + 1 slots of a page it shares with up to 31 others
    length, pages = np.arange(n) % page + 1, np.arange(n) // page
    plan.set(np.ones(n, int), length, pages)
    plan.write(0, dev(hip, k), dev(hip, v))
    out = dev(hip, np.full_like(q, 7.25))
    plan.attention(0, dev(hip, q), out)
    got = back(hip, out, q.shape)
    assert np.isfinite(got).all() and not (got == 7.25).all(-1).any()
    for i in (0, 1, 31, 32, 8191, 16383, 16384, 16399):
        first = i - i % page
        kk, vv = (held(orc, "q8_0", x[first:i + 1]) for x in (k, v))
        want, bound = attention(q[i:i + 1], kk, vv)
        assert (np.abs(got[i] - want[0]) <= bound[0]).all(), i


@pytest.mark.parametrize("kind", list(QT))
@pytest.mark.parametrize("first,then", [(1.0, 1e-3), (1e-3, 1.0), (1.0, 300.0), (0.0, 1.0)])
def test_values_change_size_behind_the_first_tile(hip, orc, kind, first, then):
    """The first 32 positions' values are of another size than the rest, in all blocks or in one."""
    rng = np.random.default_rng(13)
    for dims in (slice(None), slice(32, 64)):
        v = rng.standard_normal((200, 2, 96)).astype(np.float32)
        v[:32, :, dims] *= np.float32(first)
        v[32:, :, dims] *= np.float32(then)
        check(Case(hip, orc, kind, [(70, 200)], 4, 2, 96, values=v))


@pytest.mark.parametrize("new", [3, 70])
@pytest.mark.parametrize("before", [1.0, 1e-7, 1e7])
def test_values_below_the_floor_of_a_block(hip, orc, new, before):
    """f32 values below 2^-80, which share one power of two, behind ones of other sizes that nobody sees any more."""
    rng = np.random.default_rng(14)
    v = rng.standard_normal((300, 2, 64)).astype(np.float32)
    v[:64] *= np.float32(before)
    v[64:] *= np.float32(4e-25)
    check(Case(hip, orc, "f32", [(new, 300)], 4, 2, 64, values=v, window=100, seed=1))
    v[:64] = 0.0
    check(Case(hip, orc, "f32", [(new, 300)], 4, 2, 64, values=v, seed=1))


@pytest.mark.parametrize("kind", ["f32", "q4_1"])
def test_recorded_uneven_rows(hip, orc, kind):
    """A recorded attention whose workgroups take several items each, some of them with rows that are done in plain
    f32: replayed, with eager calls in between, it gives the eager call's bits and the 64-bit result."""
    rng = np.random.default_rng(15)
    lens = [(70, 90)] * 38 + [(33, 700), (70, 1300)]
    positions = sum(t for _, t in lens)
    v = rng.standard_normal((positions, 32, 64)).astype(np.float32)
    v[rng.random(positions) < 0.004, :, 32:] *= np.float32(1e-4)
    c = Case(hip, orc, kind, lens, 32, 32, 64, 64, values=v, seed=2)
    want = check(c)
    s = hip.stream_create()
    dq, out = dev(hip, c.q), dev(hip, np.zeros_like(c.q))
    g = hip.Graph.record(lambda: c.plan.attention(0, dq, out, stream=s), stream=s)
    for _ in range(3):
        out.upload(np.zeros(c.q.size, np.float32))
        g.launch(s)
        hip.synchronize(s)
        assert np.array_equal(out.download(np.float32, c.q.size).reshape(c.q.shape), want)
        assert np.array_equal(c.run(), want)
    g.destroy()
    hip.stream_destroy(s)


@pytest.mark.parametrize("kind", list(QT))
@pytest.mark.parametrize("new", [3, 70])
def test_padded_heads(hip, orc, kind, new):
    """A head's last blocks are zeros in keys, values and queries, up to some position or throughout; rows that
    see where they are not, zeros in all blocks behind, tiny ones."""
    rng = np.random.default_rng(16)
    for hd, until, behind in ((128, 300, 1.0), (96, 300, 1.0), (128, 250, 1.0), (128, 290, 1e-3), (128, 299, 300.0), (192, 40, 1.0)):
        k, v = (rng.standard_normal((300, 2, hd)).astype(np.float32) for _ in range(2))
        k[:, :, hd - 32:] = 0
        v[until:] *= np.float32(behind)
        v[:until, :, hd - 32:] = 0
        v[270:275] = 0
        c = Case(hip, orc, kind, [(new, 300)], 4, 2, hd, keys=k, values=v)
        c.q[:, :, hd - 32:] = 0
        check(c)
    v = rng.standard_normal((300, 2, 64)).astype(np.float32)
    v[:32] = 0  # nothing to go by in the first tile
    check(Case(hip, orc, kind, [(new, 300)], 4, 2, 64, values=v))
    v[:, :, 32:] *= np.float32(1e-25)
    v[100:110, :, :32] = 0
    check(Case(hip, orc, kind, [(new, 300)], 4, 2, 64, values=v), dims=slice(0, 32))


@pytest.mark.parametrize("new", [3, 70])
@pytest.mark.parametrize("size", [1.0, 300.0, 1e-3, 1e12, 1e-12, 1e-20, 1e-24])
def test_value_blocks_below_the_floor_beside_larger_ones(hip, orc, new, size):
    """f32 values below 2^-80 throughout a block, but not zeros, beside a block of another size: they are taken to
    2^-100, and no size beside them makes them overflow.  (The tolerance is the bound and that 2^-100, once: the
    weights sum to one.)"""
    rng = np.random.default_rng(17)
    for tiny, total in ((1e-25, 300), (1e-26, 1500)):
        v = rng.standard_normal((total, 2, 64)).astype(np.float32)
        v[:, :, :32] *= np.float32(size)
        v[:, :, 32:] = np.clip(v[:, :, 32:], -4, 4) * np.float32(tiny)
        v[total - 60:total - 50, :, :32] *= np.float32(1e-4)  # positions with a power of two of their own
        v[total - 40:total - 30, :, :32] *= np.float32(1e4)
        v[total - 20:total - 10, :, :32] = 0
        c = Case(hip, orc, "f32", [(new, total)], 4, 2, 64, values=v, seed=3)
        got = c.run()
        want, bound = attention_by_block(c.q, c.held[0], c.held[1])
        err = np.abs(got - want) / (bound + 2.0 ** -100)
        assert (err <= 1).all(), (tiny, float(np.max(err)), int(np.isnan(err).sum()))
