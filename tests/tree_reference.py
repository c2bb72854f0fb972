"""Plain 64-bit numpy forms of decoding with several candidates, for tests: attention of drafted
trees (mlq_hip_kv_plan_set_tree), checked drafts (mlq_hip_kv_tree_pick) and beam selection
(mlq_hip_beam_select)."""

import numpy as np


def chain(n):
    return list(range(-1, n - 1))


def wide(n, branch):
    """Every node has `branch` children, level by level."""
    return [(i - 1) // branch if i else -1 for i in range(n)]


def ragged(rng, n, back=6, roots=1):
    return [-1 if i < roots else i - 1 - int(rng.integers(min(i, back))) for i in range(n)]


def depths(parents):
    out = []
    for p in parents:
        out.append(0 if p < 0 else out[p] + 1)
    return np.array(out, int)


def path_to(parents, node):
    path = []
    while node >= 0:
        path.insert(0, node)
        node = parents[node]
    return path


def seen(parents, before, window=0, sinks=0):
    """[nodes, before + nodes]: the slots that each node sees."""
    n, depth = len(parents), depths(parents)
    see = np.zeros((n, before + n), bool)
    at = np.concatenate([np.arange(before), before + depth])  # positions of the slots
    for i in range(n):
        see[i, :before] = True
        see[i, [before + p for p in path_to(parents, i)]] = True
        if window:
            see[i] &= (at > before + depth[i] - window) | (at < sinks)
    return see


def attention(q, k, v, see, scale=0.0):
    """One sequence: q [n, heads, hd], k and v [slots, kv, hd].  (out, bound) as kv_reference.attention, whose
    derivation this follows, with who sees whom given.  Here queries, weights and f32 elements leave out the
    product of their low parts, 2^-22 of a product more, so a score is off by 4 2^-22 where it has 3, and so are the
    weighted values."""
    n, heads, hd = q.shape
    length, kv = k.shape[:2]
    scale = scale or 1.0 / np.sqrt(hd)
    out, bound = np.empty(q.shape, np.float64), np.empty((n, heads, 1), np.float64)
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    some = see.any(0)[:, None]
    for h in range(heads):
        kh, vh = np.where(some, k[:, h // (heads // kv)], 0), np.where(some, v[:, h // (heads // kv)], 0)
        s = np.where(see, scale * (q[:, h] @ kh.T), -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        out[:, h] = p @ vh
        size = np.where(see, abs(scale) * (np.abs(q[:, h]) @ np.abs(kh).T), 0).max(-1)
        reach = np.where(see, np.abs(s), 0).max(-1)
        biggest = np.where(see, np.abs(vh).max(-1)[None], 0).max(-1)
        each = size * (4 * 2.0 ** -22 + (hd + 16) * 2.0 ** -24) + 6 * reach * 2.0 ** -24 + 2.0 ** -22
        bound[:, h, 0] = biggest * (2 * each + 4 * 2.0 ** -22 + (32 + length / 32 + 64) * 2.0 ** -24)
    return out, bound


def checked(logits, tokens, parents):
    """Picks, path and next token of one sequence's tree."""
    picks = [int(np.argmax(r)) if np.isfinite(r).all() else -1 for r in logits]
    if not parents:
        return [], [], -1
    path = [0]
    while True:
        fit = [i for i in range(len(parents)) if parents[i] == path[-1] and tokens[i] == picks[path[-1]] >= 0]
        if not fit:
            return picks, path, picks[path[-1]]
        path.append(fit[0])


def beam(logits, scores, keep, ended=None, end=0):
    """One group: logits [beams, vocab], scores [beams].  (parents, tokens, values) in 64 bits."""
    found = []
    for b, (x, s) in enumerate(zip(np.asarray(logits, np.float64), np.asarray(scores, np.float64))):
        goes_on = ended is None or not ended[b]
        if np.isnan(s) or s == np.inf or (goes_on and s > -np.inf and not (x < np.inf).all()):
            return [-1] * keep, [-1] * keep, [np.nan] * keep
        if s == -np.inf:
            continue
        if not goes_on:
            found.append((-s, b, 0.0, end))
            continue
        if not (x > -np.inf).any():
            continue
        v = s + (x - (x.max() + np.log(np.exp(x - x.max()).sum())))
        at = np.lexsort((np.arange(len(x)), -x))[:keep]
        found += [(-v[t], b, -x[t], int(t)) for t in at if x[t] > -np.inf]
    found = sorted(found)[:keep]
    pad = keep - len(found)
    return [f[1] for f in found] + [-1] * pad, [f[3] for f in found] + [-1] * pad, [-f[0] for f in found] + [-np.inf] * pad
