"""Beam selection on the device (mlq_hip_beam_select) against plain numpy in 64 bits
(tree_reference.beam).

How far a value may be off: it is taken in 64 bits and rounded to f32 once, half a step, 2^-24 of
itself; an exponential there is off by 2^-36 of itself, and so are the sum and, absolutely, its
logarithm.  Parents and tokens are the reference's wherever two values differ by more than that."""

import sys

import numpy as np
import pytest

from tree_reference import beam

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


class Beams:
    def __init__(self, hip, logits, scores, keep, ended=None, end=0, stream=None, handle=None):
        self.hip, self.logits, self.scores, self.keep, self.ended, self.end, self.stream = hip, logits, scores, keep, ended, end, stream
        self.groups, self.beams, self.vocab = logits.shape
        self.handle = handle or hip.BeamSelect(self.groups, self.beams, self.vocab, keep)
        self.dl, self.ds = (hip.DeviceBuffer.from_array(np.asarray(x, np.float32)) for x in (logits, scores))
        self.de = None if ended is None else hip.DeviceBuffer.from_array(np.asarray(ended, np.int32))
        n = self.groups * keep + 1
        self.out = [hip.DeviceBuffer.from_array(np.full(n, -9, t)) for t in (np.int32, np.int32, np.float32)]

    def call(self, logits=None):
        self.handle.select(self.dl if logits is None else logits, self.ds, self.groups, self.beams, self.vocab, self.keep, *self.out,
                           ended=self.de, end_token=self.end, stream=self.stream)

    def result(self):
        self.hip.synchronize(self.hip.stream(0) if self.stream is None else self.stream)
        n = self.groups * self.keep + 1
        got = [b.download(t, n) for b, t in zip(self.out, (np.int32, np.int32, np.float32))]
        assert all(x[-1] == -9 for x in got)
        return [x[:-1].reshape(self.groups, self.keep) for x in got]

    def check(self, got=None):
        if got is None:
            self.call()
            got = self.result()
        for g in range(self.groups):
            parents, tokens, values = beam(self.logits[g], self.scores[g], self.keep, None if self.ended is None else self.ended[g], self.end)
            assert got[0][g].tolist() == parents and got[1][g].tolist() == tokens, g
            values = np.array(values)
            there = np.isfinite(values)
            assert np.array_equal(got[2][g][~there], values[~there].astype(np.float32), equal_nan=True)
            assert (np.abs(got[2][g][there] - values[there]) <= np.abs(values[there]) * 2.0 ** -24 + 2.0 ** -35).all()
        return got


def random(rng, groups, beams, vocab, std=2.5):
    return (std * rng.standard_normal((groups, beams, vocab))).astype(np.float32), (-9 * rng.random((groups, beams))).astype(np.float32)


@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 255, 257, 2047, 2049, 8191, 8192, 8193, 16385, 32000, 100003])
def test_vocabularies(hip, vocab):
    rng = np.random.default_rng(vocab)
    say("vocab", vocab)
    for groups, beams, keep in ((1, 1, 1), (2, 4, 8), (3, 5, 64)):
        Beams(hip, *random(rng, groups, beams, vocab), keep).check()


@pytest.mark.parametrize("beams", [1, 2, 3, 16, 31, 64])
@pytest.mark.parametrize("keep", [1, 2, 7, 33, 64])
def test_counts(hip, beams, keep):
    rng = np.random.default_rng(100 * beams + keep)
    say("counts", beams, keep)
    Beams(hip, *random(rng, 3, beams, 9001 if beams < 20 else 1500), keep).check()


def test_wide_searches(hip):
    """Many beams whose scores lie far apart, so that a few of them hold all continuations, and many kept."""
    rng = np.random.default_rng(11)
    for groups, beams, vocab in ((5, 64, 8000), (1, 64, 33000), (3, 61, 700)):
        x, s = random(rng, groups, beams, vocab)
        Beams(hip, x, s, 64).check()
        Beams(hip, x, (s * 20).astype(np.float32), 64).check()
        s[:] = np.where(np.arange(beams) % 4 == 1, s, s - 50)
        Beams(hip, x, s, 64).check()


def test_many_groups(hip):
    Beams(hip, *random(np.random.default_rng(1), 300, 3, 777), 6).check()


def test_ties(hip):
    """Equal beams, equal logits and logits in order: the lower beam, then the lower token."""
    rng = np.random.default_rng(2)
    for vocab in (500, 20000):
        x, s = random(rng, 1, 6, vocab)
        x[:] = x[:, :1]
        s[:] = -1.5
        Beams(hip, x, s, 20).check()
        for row in (np.zeros(vocab), np.arange(vocab) / 64, -np.arange(vocab) / 64, rng.integers(0, 3, vocab), np.full(vocab, -0.0),
                    np.where(np.arange(vocab) % 2, 0.0, -0.0)):
            x[:] = row.astype(np.float32)
            for keep in (1, 20, 64):
                Beams(hip, x, s, keep).check()


def test_values_far_apart(hip):
    rng = np.random.default_rng(3)
    x, s = random(rng, 2, 4, 3000)
    Beams(hip, (x * 1e4).astype(np.float32), s, 9).check()
    Beams(hip, (x * 1e-6).astype(np.float32), s, 9).check()
    Beams(hip, x + np.float32(3e5), s, 9).check()
    Beams(hip, x, (s * 1e6).astype(np.float32), 9).check()
    x[:, :, 5] = 3e38
    x[:, :, 6] = -3e38
    Beams(hip, x, s, 64).check()


@pytest.mark.parametrize("vocab", [40, 3000, 40000])
@pytest.mark.parametrize("top", [2.0 ** 32, 2.0 ** 33, 1e10, -1e10, 1e12, -1e12, 3e38, -3e38])
def test_large_logits(hip, vocab, top):
    """Logits whose neighbours in f32 are hundreds apart and more: only the largest have a part in the sum, and a value
    keeps the logarithm of their number."""
    rng = np.random.default_rng(6)
    top = np.float32(top)
    x = np.full((1, 3, vocab), np.nextafter(top, np.float32(-np.inf)))
    x[0, 0, vocab // 2:] = -3.4e38
    x[0, 1, ::3] = -3.4e38
    x[0, 2, rng.permutation(vocab)[:vocab // 4]] = top / 2 if top > 0 else top * 1.125
    x[0, 0, [3, vocab - 1]] = top
    x[0, 1, [vocab - 2, vocab - 3, 1]] = top
    x[0, 2, vocab - 7] = top
    s = np.array([[-1.0, -0.25, -2.0]], np.float32)
    b = Beams(hip, x, s, 6)
    b.call()
    parents, tokens, values = (y[0] for y in b.result())
    want = [(s[0, 2], 2, vocab - 7)] + [(s[0, 1] - np.log(3.0), 1, t) for t in (1, vocab - 3, vocab - 2)] + \
        [(s[0, 0] - np.log(2.0), 0, t) for t in (3, vocab - 1)]
    want.sort(key=lambda w: (-w[0], w[1], w[2]))
    assert parents.tolist() == [w[1] for w in want] and tokens.tolist() == [w[2] for w in want]
    v = np.array([w[0] for w in want])
    assert (np.abs(values - v) <= np.abs(v) * 2.0 ** -24 + 2.0 ** -35).all()


def test_masked_dead_and_ended(hip):
    rng = np.random.default_rng(4)
    x, s = random(rng, 7, 8, 9000)
    x[rng.random(x.shape) < 0.3] = -np.inf
    x[1, :, 4:] = -np.inf  # four tokens a beam
    x[2] = -np.inf         # none at all
    s[3, 1:] = -np.inf     # a search starts
    s[4] = -np.inf
    x[5, 2] = -np.inf
    x[5, 3, :-1] = -np.inf
    for keep in (3, 40, 64):
        Beams(hip, x, s, keep).check()
        ended = rng.random((7, 8)) < 0.4
        ended[6] = True
        b = Beams(hip, x, s, keep, ended * 5, end=8999)
        b.check()
    # an ended beam's logits are not looked at
    x[6, 3] = np.nan
    got = Beams(hip, x, s, 5, ended, end=2).check()
    assert (got[1][6] == 2).all()


def test_values_that_are_not_finite(hip):
    rng = np.random.default_rng(5)
    x, s = random(rng, 8, 3, 8200)
    x[1, 2, 8199] = np.nan
    x[2, 0, 0] = np.inf
    s[3, 1] = np.nan
    s[4, 2] = np.inf
    s[5, 0] = -np.inf
    x[5, 0, 7] = np.nan  # of a beam that is not there
    x[6, 1, 100:200] = -np.inf
    got = Beams(hip, x, s, 4).check()
    assert np.isnan(got[2][1:5]).all() and (got[0][1:5] == -1).all() and np.isfinite(got[2][[0, 5, 6, 7]]).all()


def test_rows_at_odd_addresses(hip):
    rng = np.random.default_rng(6)
    x, s = random(rng, 2, 3, 8195)
    b = Beams(hip, x, s, 6)
    for off in (1, 2, 3):
        buf = hip.DeviceBuffer.from_array(np.concatenate([np.full(off, 1e30, np.float32), x.ravel()]))
        b.call(buf.ptr + 4 * off)
        b.check(b.result())


def test_one_handle_smaller_calls_and_the_same_bits(hip):
    rng = np.random.default_rng(7)
    h = hip.BeamSelect(4, 8, 20000, 32)
    s = hip.stream_create()
    for groups, beams, vocab, keep in ((4, 8, 20000, 32), (1, 1, 5, 1), (2, 3, 9000, 7), (4, 8, 20000, 5)):
        b = Beams(hip, *random(rng, groups, beams, vocab), keep, stream=s, handle=h)
        one = b.check()
        for _ in range(3):
            b.call()
            assert all(np.array_equal(x, y) for x, y in zip(one, b.result()))
    hip.stream_destroy(s)


def test_recorded(hip):
    """Replays with other contents of the same buffers, eager calls of the handle between them."""
    rng = np.random.default_rng(8)
    s = hip.stream_create()
    b = Beams(hip, *random(rng, 3, 4, 17000), 10, stream=s)
    other = Beams(hip, *random(rng, 2, 2, 5000), 4, stream=s, handle=b.handle)
    g = hip.Graph.record(b.call, stream=s)
    for _ in range(4):
        b.logits, b.scores = random(rng, 3, 4, 17000)
        b.dl.upload(b.logits)
        b.ds.upload(b.scores)
        g.launch(s)
        got = b.check(b.result())
        other.check()
        b.call()
        assert all(np.array_equal(x, y) for x, y in zip(got, b.result()))
    with pytest.raises(hip.MlqError, match="graph capture"):
        hip.Graph.record(lambda: hip.BeamSelect(1, 1, 10, 1), stream=hip.stream(0))
    g.destroy()
    hip.stream_destroy(s)


def test_refusals(hip):
    h = hip.BeamSelect(2, 4, 100, 8)
    x, s, e = hip.DeviceBuffer(4 * 800), hip.DeviceBuffer(32), hip.DeviceBuffer(32)
    p, t, v = (hip.DeviceBuffer(64) for _ in range(3))

    def call(logits=x, scores=s, groups=2, beams=4, vocab=100, keep=8, parents=p, tokens=t, out=v, **kw):
        h.select(logits, scores, groups, beams, vocab, keep, parents, tokens, out, **kw)

    for bad, what in ((dict(groups=3), "3 groups"), (dict(groups=-1), "-1 groups"), (dict(beams=5), "5 beams"), (dict(beams=0), "0 beams"),
                      (dict(vocab=101), "101 tokens"), (dict(vocab=0), "0 tokens"), (dict(keep=9), "9 continuations"),
                      (dict(keep=0), "0 continuations"), (dict(logits=None), "null"), (dict(scores=None), "null"),
                      (dict(parents=None), "null"), (dict(tokens=None), "null"), (dict(out=None), "null"),
                      (dict(logits=x.ptr + 2), "aligned"), (dict(logits=s), "too small"), (dict(ended=e, end_token=100), "end token 100"),
                      (dict(ended=e, end_token=-1), "end token -1"), (dict(ended=hip.DeviceBuffer(16), end_token=1), "too small"),
                      (dict(tokens=p), "tokens overlaps parents"), (dict(out=x), "out_scores overlaps logits"),
                      (dict(parents=x.ptr + 64), "parents overlaps logits"), (dict(out=t), "out_scores overlaps tokens")):
        with pytest.raises(hip.MlqError, match=what):
            call(**bad)
    call(groups=0, logits=None, scores=None, parents=None, tokens=None, out=None)
    hip.synchronize(hip.stream(0))
