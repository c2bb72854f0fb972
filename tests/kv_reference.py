"""Plain 64-bit numpy form of the paged key/value cache (mlq_hip_kv_write / _read /
_attention), for tests.  What a quantized cache holds is taken from the oracle's
block quantizers, so codes and scales have to be the same bits."""

import numpy as np

QT = {"f32": 0, "q8_0": 1, "q4_0": 2, "q4_1": 3}


def held(orc, kind, x):
    """The f32 values a cache of `kind` holds for x [..., head_dim] (f32)."""
    if kind == "f32" or not x.size:
        return x
    rows = np.ascontiguousarray(x.reshape(-1, x.shape[-1]), np.float32)
    return orc.dequantize(QT[kind], orc.quantize(QT[kind], rows), *rows.shape).reshape(x.shape)


def rotated(x, pos, theta, neox):
    """RoPE of x [tokens, heads, hd] at pos, in 64 bits, rounded to f32 once."""
    hd = x.shape[-1]
    a = np.asarray(pos, np.float64)[:, None, None] * np.float64(np.float32(theta)) ** (-2.0 * np.arange(hd // 2) / hd)
    c, s = np.cos(a), np.sin(a)
    y = np.empty(x.shape, np.float64)
    i0, i1 = (slice(0, hd // 2), slice(hd // 2, hd)) if neox else (slice(0, hd, 2), slice(1, hd, 2))
    x0, x1 = x[..., i0].astype(np.float64), x[..., i1].astype(np.float64)
    y[..., i0], y[..., i1] = x0 * c - x1 * s, x0 * s + x1 * c
    return y.astype(np.float32)


def visible(n, length, window, sinks):
    """[n, length]: which positions each of the last n tokens sees."""
    p, j = np.arange(length - n, length)[:, None], np.arange(length)[None, :]
    see = j <= p
    return see & ((j > p - window) | (j < sinks)) if window else see


def attention(q, k, v, window=0, sinks=0, scale=0.0):
    """One sequence: q [n, heads, hd], k and v [length, kv, hd].  (out, bound): the 64-bit
    result and how far f32 arithmetic may be off, per row and head.

    The bound.  The kernel's scores are sums of products of two fp16 parts: a part pair
    leaves 2^-22 of a value (half a step of fp16, 2^-11, twice), an f32 cache's keys have
    the same and lose the product of the low parts (2^-22), and a sum of hd products and
    one scaled sum per block takes an f32 rounding (2^-24) each.  So a score is off by
    at most A (3 2^-22 + (hd + 16) 2^-24) with A = scale sum |q||k|; its scaling and
    subtraction by three roundings of it and of the row's largest.  A probability is off by that much relative
    to itself, 2^-22 for the exponential, and so is the sum.  The weighted values have
    3 2^-22 for their parts and a rounding for each of 32 products a tile, for each tile
    and each of 64 parts at the most that are merged."""
    n, heads, hd = q.shape
    length, kv = k.shape[:2]
    scale = scale or 1.0 / np.sqrt(hd)
    see = visible(n, length, window, sinks)
    out, bound = np.empty(q.shape, np.float64), np.empty((n, heads, 1), np.float64)
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    for h in range(heads):
        kh, vh = k[:, h // (heads // kv)], v[:, h // (heads // kv)]
        with np.errstate(invalid="ignore", over="ignore"):
            s = np.where(see, scale * (q[:, h] @ np.where(see.any(0)[:, None], kh, 0).T), -np.inf)
            top = s.max(-1, keepdims=True)
            p = np.exp(s - top)
            p /= p.sum(-1, keepdims=True)
            for i in range(n):
                out[i, h] = p[i, see[i]] @ vh[see[i]]
            size = np.where(see, abs(scale) * (np.abs(q[:, h]) @ np.abs(kh).T), 0).max(-1)
            reach = np.where(see, np.abs(s), 0).max(-1)
            biggest = np.array([np.abs(vh[see[i]]).max() for i in range(n)])
            each = size * (3 * 2.0 ** -22 + (hd + 16) * 2.0 ** -24) + 6 * reach * 2.0 ** -24 + 2.0 ** -22
            bound[:, h, 0] = biggest * (2 * each + 3 * 2.0 ** -22 + (32 + length / 32 + 64) * 2.0 ** -24)
    return out, bound


class Batch:
    """Sequences on pages in a random order, for a KvPlan: lens is [(new, kv_len)]."""

    def __init__(self, rng, lens, page_size, spare=2):
        self.lens, self.page_size = lens, page_size
        self.new, self.kv_len = [n for n, _ in lens], [t for _, t in lens]
        need = [-(-t // page_size) for t in self.kv_len]
        ids = rng.permutation(sum(need) + spare)
        self.n_pages = len(ids)
        self.pages = [int(i) for i in ids[:sum(need)]]
        self.tokens, self.positions, self.entries = sum(self.new), sum(self.kv_len), sum(need)

    def pos(self):
        return np.concatenate([np.arange(t - n, t) for n, t in self.lens] + [np.zeros(0, int)]).astype(int)

    def rows(self):
        """Row of each new token among all positions of the batch."""
        out, at = [], 0
        for n, t in self.lens:
            out.append(np.arange(at + t - n, at + t))
            at += t
        return np.concatenate(out + [np.zeros(0, int)]).astype(int)


def attention_by_block(q, k, v, window=0, sinks=0, scale=0.0):
    """As `attention`, with a bound of its own for each of a head's blocks of 32 dimensions: (out, bound),
    both [n, heads, hd].

    A block's results are weighted sums of that block's values, so f32 arithmetic is off by what it
    loses of W = sum_j p_j max|v_j| over the block, whatever other blocks hold and however small the weights
    of the positions that hold its values.  A probability is off by the 2 `each` of `attention`, and by three
    roundings (in base 2) of the values' exponents where these go into the scores; an element and a weight by
    3 2^-22 for their parts; a sum over `length` positions by as many roundings of it (weights too small for
    fp16 beside a block's largest one are lost in there: 2^-34 of that each, 2^-24 where the positions'
    values differ by 2^10), and 96 more for parts and merges."""
    n, heads, hd = q.shape
    length, kv = k.shape[:2]
    factor = scale or 1.0 / np.sqrt(hd)
    see = visible(n, length, window, sinks)
    out, bound = np.empty(q.shape, np.float64), np.empty(q.shape, np.float64)
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    starts = np.arange(0, hd, 32)
    for h in range(heads):
        kh, vh = k[:, h // (heads // kv)], v[:, h // (heads // kv)]
        s = np.where(see, factor * (q[:, h] @ kh.T), -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        out[:, h] = p @ vh
        size = np.where(see, abs(factor) * (np.abs(q[:, h]) @ np.abs(kh).T), 0).max(-1)
        reach = np.where(see, np.abs(s), 0).max(-1)
        top = np.maximum.reduceat(np.abs(vh), starts, axis=1)  # [length, blocks]
        largest = top.max(-1)
        log = np.abs(np.log2(largest[largest > 0])).max(initial=0.0)
        each = size * (3 * 2.0 ** -22 + (hd + 16) * 2.0 ** -24) + 6 * reach * 2.0 ** -24 + 3 * log * 2.0 ** -24 + 2.0 ** -22
        rel = 2 * each + 3 * 2.0 ** -22 + (length + 96) * 2.0 ** -24
        bound[:, h] = np.repeat((p @ top) * rel[:, None], 32, axis=1)[:, :hd]
    return out, bound
