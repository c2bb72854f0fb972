"""Decoding with several candidates over the paged key/value cache, as cases that can be timed and checked.

A step may carry a tree of drafted tokens for each sequence, or several beams of it.  A case is a dict of
plain values; ``kind`` says which operator it goes through:

  tree  a layer's pass over a step of drafted trees: the nodes' keys (rotated by their depth) and values
        written into their pages, the queries rotated, and their attention: a node sees what came before
        the tree, its ancestors and itself (``mlq_hip_kv_plan_set_tree``, ``mlq_hip_kv_write``,
        ``mlq_hip_kv_attention``)
  pick  the greedy token of every node's logits and the path of drafted tokens that they confirm
        (``mlq_hip_kv_tree_pick``)
  keep  a confirmed path's keys and values moved together behind what came before the tree, in every layer
        (``mlq_hip_kv_keep``), and read back (``mlq_hip_kv_read``)
  copy  the first positions of pages copied into other pages, in every layer, as beams that part do
        (``mlq_hip_kv_copy_pages``), and read back
  beam  the best continuations over the beams and the vocabulary (``mlq_hip_beam_select``)

``listed`` gives the cases to look at first, ``draw`` more of the same ranges.
"""

import math
import os
import sys

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
QK = 32
TYPE = {"f32": 0, "q8_0": 1, "q4_0": 2, "q4_1": 3}
#: bytes of a block of 32 elements
BLOCK = {"f32": 128, "q8_0": 34, "q4_0": 18, "q4_1": 20}
THETA = 10000.0
#: A drawn case costs no more than the largest listed one: a tree's attention flops and padded scores, the
#: elements of the sequences' keys, the logits of a call, the elements a cache operator moves.
MOST_FLOPS, MOST_SCORES, MOST_KEYS = 4 * 128 * 32 * 4 * 256 * 2000, 4 * 32 * 256 * 2256, 70 << 20
MOST_LOGITS, MOST_MOVED = 512 * 152000, 256 * 64 * 8 * 128 * 2


def listed():
    return [
        # The smallest step: eight drafted tokens for one sequence of an 896-wide model, 14 query heads over
        # 2 KV heads.  Launches and the host path count.
        {"name": "tree_8_q8_0", "kind": "tree", "type": "q8_0", "heads": 14, "kv": 2, "hd": 64, "page": 64, "seqs": 1,
         "new": 8, "ctx": 700, "ragged": False, "branch": 2, "neox": True, "window": 0, "sinks": 0},
        # One chat late in its context, a wide ragged draft, grouped heads.
        {"name": "tree_64_q8_0", "kind": "tree", "type": "q8_0", "heads": 32, "kv": 8, "hd": 128, "page": 64, "seqs": 1,
         "new": 64, "ctx": 4000, "ragged": False, "branch": 0, "neox": False, "window": 0, "sinks": 0},
        # Sixteen sequences drafting together, a sliding window with four first tokens that stay visible,
        # head_dim not a whole number of blocks.
        {"name": "tree_16x24_q4_1", "kind": "tree", "type": "q4_1", "heads": 32, "kv": 8, "hd": 80, "page": 128,
         "seqs": 16, "new": 24, "ctx": 3000, "ragged": True, "branch": 3, "neox": True, "window": 1024, "sinks": 4},
        # The largest: exhaustive drafts of four sequences over an unquantized cache, LLaMA-7B-shaped heads.
        {"name": "tree_4x256_f32", "kind": "tree", "type": "f32", "heads": 32, "kv": 32, "hd": 128, "page": 64,
         "seqs": 4, "new": 256, "ctx": 2000, "ragged": False, "branch": 4, "neox": False, "window": 0, "sinks": 0},
        # Checking one small draft.
        {"name": "pick_16", "kind": "pick", "vocab": 32000, "seqs": 1, "new": 16, "ragged": False, "branch": 2},
        # Checking the drafts of a batch over a large vocabulary.
        {"name": "pick_16x32", "kind": "pick", "vocab": 152000, "seqs": 16, "new": 32, "ragged": True, "branch": 0},
        # One sequence's confirmed path, the small model's heads.
        {"name": "keep_1_q8_0", "kind": "keep", "type": "q8_0", "heads": 14, "kv": 2, "hd": 64, "page": 64, "layers": 4,
         "seqs": 1, "new": 32, "ctx": 701, "ragged": False, "branch": 5},
        # The confirmed paths of a batch, across pages and in many layers.
        {"name": "keep_64_q4_0", "kind": "keep", "type": "q4_0", "heads": 32, "kv": 8, "hd": 128, "page": 32, "layers": 16,
         "seqs": 64, "new": 64, "ctx": 600, "ragged": True, "branch": 6},
        # Three beams leave a fourth: its last page, filled in part, in every layer.
        {"name": "copy_3_q8_0", "kind": "copy", "type": "q8_0", "heads": 14, "kv": 2, "hd": 64, "page": 64, "layers": 4,
         "pages": 3, "ragged": True},
        # A long session forked as a whole.
        {"name": "copy_256_q8_0", "kind": "copy", "type": "q8_0", "heads": 32, "kv": 8, "hd": 128, "page": 64, "layers": 4,
         "pages": 256, "ragged": False},
        # Four beams of one sequence.
        {"name": "beam_4", "kind": "beam", "vocab": 32000, "groups": 1, "beams": 4, "keep": 8, "ended": False,
         "masked": False, "first": False},
        # Eight beams each of 32 sequences over a large vocabulary whose rows start at odd places; some beams
        # have ended, some tokens are not allowed.
        {"name": "beam_32x8", "kind": "beam", "vocab": 128011, "groups": 32, "beams": 8, "keep": 16, "ended": True,
         "masked": True, "first": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["tree", "pick", "keep", "copy", "beam"], [6, 2, 2, 2, 4])[0]
    if kind == "pick":
        case = {"kind": kind, "vocab": _log(rng, 1000, 160000), "seqs": _log(rng, 1, 64), "new": _log(rng, 1, 128),
                "ragged": rng.random() < 0.7, "branch": rng.choice([0, 1, 2, 4])}
        while case["seqs"] * case["new"] * case["vocab"] > MOST_LOGITS:
            case["seqs" if case["seqs"] > 1 else "new"] //= 2
        return case
    if kind == "beam":
        case = {"kind": kind, "vocab": _log(rng, 1000, 160000), "groups": _log(rng, 1, 64), "beams": _log(rng, 1, 32),
                "keep": _log(rng, 1, 64), "ended": rng.random() < 0.4, "masked": rng.random() < 0.4,
                "first": rng.random() < 0.2}
        while case["groups"] * case["beams"] * case["vocab"] > MOST_LOGITS // 4:
            case["groups" if case["groups"] > 1 else "beams"] //= 2
        return case
    kv = rng.choice([1, 2, 4, 8, 8, 16, 32])
    heads = kv * (rng.choice([1, 2, 4, 4, 7, 8]) if kv <= 8 else rng.choice([1, 2]))
    case = {"kind": kind, "type": rng.choice(["f32", "q8_0", "q8_0", "q4_0", "q4_0", "q4_1"]), "heads": heads, "kv": kv,
            "hd": rng.choice([64, 64, 128, 128, 128, 128, 256, 80, 112, 32]), "page": rng.choice([32, 64, 64, 128, 256]),
            "ragged": rng.random() < 0.7}
    if kind == "copy":
        case |= {"layers": _log(rng, 1, 32), "pages": _log(rng, 1, 512)}
        while case["pages"] * case["page"] * kv * case["hd"] * case["layers"] > MOST_MOVED * 2:
            case["pages" if case["pages"] > 8 else "layers"] //= 2
        return case
    case |= {"seqs": _log(rng, 1, 64 if rng.random() < 0.5 else 8), "new": _log(rng, 2, 96) if rng.random() < 0.8 else _log(rng, 1, 512),
             "ctx": _log(rng, 100, 8000) if rng.random() < 0.8 else _log(rng, 1, 100) - 1}
    if kind == "keep":
        case |= {"layers": _log(rng, 1, 32), "branch": rng.choice([4, 5, 6, 8]), "ctx": case["ctx"] // 4}
        while _keys(case) * case["layers"] > MOST_KEYS * 2:
            case["layers" if case["layers"] > 1 else "seqs" if case["seqs"] > 1 else "ctx"] //= 2
        return case
    window = _log(rng, 4, 4096) if rng.random() < 0.3 else 0
    case |= {"branch": rng.choice([0, 0, 1, 2, 3, 4, 8]), "neox": rng.random() < 0.5, "window": window,
             "sinks": rng.choice([0, 1, 4, 64]) if window else 0}
    while _keys(case) > MOST_KEYS or case["seqs"] * heads * case["new"] * (case["new"] + case["ctx"]) > MOST_SCORES or \
            _attention_flops(case) > MOST_FLOPS:
        case["seqs" if case["seqs"] > 1 else "ctx" if case["ctx"] > case["new"] else "new"] //= 2
    return case


# ---------------------------------------------------------------- the batch

def _parts(case, n):
    """What part of the case's largest each of n members has."""
    return [1.0 if not case["ragged"] or i == 0 else 0.25 + 0.75 * ((i * 0.6180339887) % 1) for i in range(n)]


def _lens(case):
    """[(nodes, positions before them)] of the case's sequences."""
    return [(max(1, int(case["new"] * p)), int(case.get("ctx", 0) * p)) for p in _parts(case, case["seqs"])]


def _keys(case):
    return sum(n + c for n, c in _lens(case)) * case["kv"] * case["hd"]


def _parents(case, n):
    """A tree of n nodes in an order that has parents first: node 0 is the root (-1).  branch 1: a chain; b: every
    node has b children, level by level; 0: deep and shallow paths mixed."""
    b = case["branch"]
    if b:
        return [(i - 1) // b if i else -1 for i in range(n)]
    return [i - 1 - int((i * 0.6180339887) % 1 * min(i, 6)) for i in range(n)]


def _depths(parents):
    out = []
    for p in parents:
        out.append(0 if p < 0 else out[p] + 1)
    return out


def _ancestors(parents):
    """[nodes, nodes]: whether the column's node is the row's or an ancestor of it."""
    n = len(parents)
    a = torch.eye(n, dtype=torch.bool)
    for i, p in enumerate(parents):
        if p >= 0:
            a[i] |= a[p]
    return a


def _seen(case, n, ctx):
    """[nodes, ctx + nodes]: which slots each node sees."""
    parents = _parents(case, n)
    depth = torch.tensor(_depths(parents))
    see = torch.cat([torch.ones(n, ctx, dtype=torch.bool), _ancestors(parents)], 1)
    if case["window"]:
        at = torch.cat([torch.arange(ctx), ctx + depth])[None, :]
        see &= (at > (ctx + depth)[:, None] - case["window"]) | (at < case["sinks"])
    return see


def _path(case, n):
    """The path that is kept: the deepest whose later nodes do not lie where it moves to, so that it can be moved
    again."""
    parents = _parents(case, n)
    best = [0]
    for leaf in range(n):
        path = [leaf]
        while parents[path[0]] >= 0:
            path.insert(0, parents[path[0]])
        if len(path) > len(best) and all(i == d or i >= len(path) for d, i in enumerate(path)):
            best = path
    return best


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device=DEV) * std


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device=DEV)


def _keys_values(g, total, kv, hd, layers=1):
    """Keys and values; a few of a head's key channels are large, as models have them."""
    loud = 1 + 3 * (_rand(g, kv, hd) < 0.04)
    return _randn(g, layers, total, kv, hd) * loud, _randn(g, layers, total, kv, hd, std=0.7)


def _inputs(case, seed):
    """What a case computes with.  tree, keep: keys and values of every slot of every sequence (one after the other),
    queries scaled so that a softmax has weight on some tens of positions; copy: of every slot of the pages."""
    g = _gen(seed)
    if case["kind"] in ("tree", "keep"):
        lens = _lens(case)
        k, v = _keys_values(g, sum(n + c for n, c in lens), case["kv"], case["hd"], case.get("layers", 1))
        return k, v, _randn(g, sum(n for n, _ in lens), case["heads"], case["hd"], std=1.6)
    if case["kind"] == "copy":
        return _keys_values(g, sum(_filled_slots(case)), case["kv"], case["hd"], case["layers"])
    if case["kind"] == "pick":
        rows = sum(n for n, _ in _lens(case))
        logits = _randn(g, rows, case["vocab"], std=2.5)
        # drafts are right for a good part: a node's token is what its parent's logits say in three of five
        best = _first_largest(logits)
        parents = _rows_parents(case)
        tokens = torch.randint(0, case["vocab"], (rows,), generator=g, device=DEV)
        right = _rand(g, rows) < 0.6
        tokens = torch.where(right & (parents >= 0), best[parents.clamp(min=0)], tokens)
        return logits, tokens.to(torch.int32)
    rows = case["groups"] * case["beams"]
    logits = _randn(g, rows, case["vocab"], std=2.5)
    if case["masked"]:
        logits = logits.masked_fill(_rand(g, rows, case["vocab"]) < 0.1, -math.inf)
    scores = -8.0 * _rand(g, case["groups"], case["beams"])
    if case["first"]:  # a search starts with one beam
        scores[:, 1:] = -math.inf
    ended = (_rand(g, case["groups"], case["beams"]) < 0.25).to(torch.int32) if case["ended"] else None
    return logits, scores, ended


def _filled_slots(case):
    return [max(1, int(case["page"] * p)) for p in _parts(case, case["pages"])]


def _page_order(count, seed):
    g = torch.Generator()
    g.manual_seed(int(seed))
    return torch.randperm(count, generator=g)


def _rows_parents(case):
    """Parent row of each row of a batch of trees, -1 of roots."""
    out, at = [], 0
    for n, _ in _lens(case):
        out += [p + at if p >= 0 else -1 for p in _parents(case, n)]
        at += n
    return torch.tensor(out, device=DEV)


# ---------------------------------------------------------------- the plain form

def _half(v):
    """f32 to binary16, half rounded up in magnitude, as the framework's quantizers encode scales."""
    u = v.view(torch.int32)
    sign, e, frac = (u >> 16) & 0x8000, ((u >> 23) & 0xff) - 112, u & 0x7fffff
    normal = ((e.clamp(min=0) << 23) + frac + 0x1000) >> 13
    small = (((frac | 0x800000) >> (1 - e).clamp(0, 31)) + 0x1000) >> 13
    mag = torch.where(e > 0, normal, torch.where(e < -10, torch.zeros_like(small), small))
    mag = torch.where((e >= 31) | (mag >= 0x7c00), torch.full_like(mag, 0x7c00), mag)
    return (sign | mag).to(torch.int16).view(torch.float16)


def _round(v):
    """To the nearest whole number, halves away from zero."""
    t = v.trunc()
    return t + torch.where((v - t).abs() >= 0.5, v.sign(), torch.zeros_like(v))


def _blocks(v):
    """[..., hd] as [..., blocks, 32]; a last block's missing elements repeat its last one."""
    hd = v.shape[-1]
    at = torch.arange(-(-hd // QK) * QK, device=v.device).clamp(max=hd - 1)
    return v[..., at].reshape(*v.shape[:-1], -1, QK)


def _quantize(kind, v):
    """Codes and scales of v [..., hd] (f32: the values themselves)."""
    if kind == "f32":
        return (v,)
    b = _blocks(v)
    if kind == "q4_1":
        lo = b.amin(-1, keepdim=True)
        span = b.amax(-1, keepdim=True) - lo
        d, m = _half(span / torch.full_like(span, 15.0)), _half(lo)
    else:
        top = b.abs().amax(-1, keepdim=True)  # a tensor divided by a number would be a product with its inverse
        d = _half(top / torch.full_like(top, 127.0 if kind == "q8_0" else 7.0))
    df = d.float()
    inv = torch.where(df == 0, torch.zeros_like(df), 1.0 / df)
    if kind == "q8_0":
        return _round(b * inv).clamp(-127, 127).to(torch.int8), d
    if kind == "q4_0":
        return _round(b * inv + 8.0).clamp(0, 15).to(torch.uint8), d
    return _round((b - m.float()) * inv).clamp(0, 15).to(torch.uint8), d, m


def _values(kind, parts, hd):
    """The values that codes and scales stand for, f32 [..., hd]."""
    if kind == "f32":
        return parts[0]
    q, d = parts[0].float(), parts[1].float()
    v = d * (q - 8.0) if kind == "q4_0" else d * q if kind == "q8_0" else d * q + parts[2].float()
    return v.flatten(-2)[..., :hd]


def _rotate(x, pos, neox):
    """Rotary embedding of x [tokens, heads, hd] at pos [tokens], in 64 bits, rounded once."""
    hd = x.shape[-1]
    r = torch.arange(hd // 2, device=x.device, dtype=torch.float64)
    a = pos.double()[:, None, None] * THETA ** (-2.0 * r / hd)
    c, s = torch.cos(a), torch.sin(a)
    x = x.double()
    x0, x1 = (x[..., :hd // 2], x[..., hd // 2:]) if neox else (x[..., 0::2], x[..., 1::2])
    y0, y1 = x0 * c - x1 * s, x0 * s + x1 * c
    return (torch.cat([y0, y1], -1) if neox else torch.stack([y0, y1], -1).flatten(-2)).float()


def _first_largest(x):
    """Index of the first largest element of each row."""
    at = torch.arange(x.shape[-1], device=x.device)
    return torch.where(x == x.amax(-1, keepdim=True), at, x.shape[-1]).amin(-1)


def _plain_tree(st):
    """Sequences padded to the longest: scores [seqs, kv, group, nodes, slots]."""
    c = st["case"]
    kv, hd, group = c["kv"], c["hd"], c["heads"] // c["kv"]
    for cache, x in ((st["keys"], _rotate(st["k"], st["pos"], c["neox"])), (st["values"], st["v"])):
        for p, new in zip(cache, _quantize(c["type"], x)):
            p[0, st["slot"]] = new
    rotated = _rotate(st["q"], st["pos"], c["neox"])
    k, v = (_values(c["type"], tuple(p[0, st["padded"]] for p in st[x]), hd) for x in ("keys", "values"))
    k, v = k.permute(0, 2, 3, 1).contiguous(), v.permute(0, 2, 1, 3).contiguous()
    seqs, _, _, t = k.shape
    n = st["qrow"].shape[1]
    q = rotated[st["qrow"]].reshape(seqs, n, kv, group, hd).permute(0, 2, 3, 1, 4).reshape(seqs, kv, group * n, hd)
    s = torch.matmul(q * (1.0 / math.sqrt(hd)), k).view(seqs, kv, group, n, t)
    s = s.masked_fill(st["hidden"], -math.inf)
    s = torch.exp(s - s.amax(-1, keepdim=True))
    s = s / s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(seqs, kv, group * n, t), v).view(seqs, kv, group, n, hd)
    return {"q": rotated, "out": o.permute(0, 3, 1, 2, 4).reshape(seqs, n, c["heads"], hd)[st["qseq"], st["qat"]]}


def _plain_pick(st):
    """Step by step from the roots: the first child whose token is its parent's pick."""
    picks = _first_largest(st["logits"])
    parents, tokens, seq, first = st["parents"], st["tokens"], st["qseq"], st["first"]
    rows, seqs = len(parents), len(first)
    right = (parents >= 0) & (tokens == picks[parents.clamp(min=0)])
    at = torch.arange(rows, device=DEV)
    here, count = first.clone(), torch.ones_like(first)
    kept = torch.full((rows,), -1, device=DEV)
    kept[first] = 0
    for _ in range(st["depth"]):
        child = torch.full((seqs,), rows, device=DEV)
        child.scatter_reduce_(0, seq, torch.where(right & (parents == here[seq]), at, rows), "amin")
        found = child < rows
        # (a sequence that is done writes its last entry again)
        kept[first + count - 1 + found.long()] = torch.where(found, child - first, here - first)
        here, count = torch.where(found, child, here), count + found
    return {"picks": picks.int(), "n_kept": count.int(), "kept": kept.int(), "next": picks[here].int()}


def _plain_keep(st):
    c = st["case"]
    for cache in ("keys", "values"):
        for p in st[cache]:
            p[:, st["to"]] = p[:, st["from"]]
    return {x: _values(c["type"], tuple(p[:, st["read"]] for p in st[x]), c["hd"]) for x in ("keys", "values")}


def _plain_beam(st):
    c = st["case"]
    groups, beams, vocab, keep = c["groups"], c["beams"], c["vocab"], c["keep"]
    x = st["logits"].double().view(groups, beams, vocab)
    top = x.amax(-1, keepdim=True)
    sums = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    s = st["scores"].double()[..., None] + (x - sums)
    if st["ended"] is not None:
        stays = torch.full((vocab,), -math.inf, dtype=torch.float64, device=DEV)
        stays[st["end"]] = 0.0
        s = torch.where(st["ended"][..., None] != 0, st["scores"].double()[..., None] + stays, s)
    s, at = torch.sort(s.view(groups, -1), dim=-1, descending=True, stable=True)
    s, at = s[:, :keep], at[:, :keep]
    none = s == -math.inf
    return {"parents": torch.where(none, -1, at // vocab).int(), "tokens": torch.where(none, -1, at % vocab).int(),
            "scores": s.float()}


# ---------------------------------------------------------------- inputs and one pass

class Dev:
    """A torch tensor's memory in the form the binding takes device buffers."""

    def __init__(self, t):
        self.t, self.ptr, self.nbytes = t, t.data_ptr(), t.numel() * t.element_size()


def _dev(t):
    return None if t is None else Dev(t)


def _hip():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mini-llama-cpp-release_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import mlq_hip
    mlq_hip.init(0)
    return mlq_hip


def _ints(*shape):
    return torch.empty(*shape, dtype=torch.int32, device=DEV)


def _cache(hip, case, n_pages, held, pages, keys, values):
    """The framework's cache holding keys and values [layers, slots ...] of sequences one after the other."""
    layers = case.get("layers", 1)
    cache = hip.KvCache(TYPE[case["type"]], layers, n_pages, case["page"], case["kv"], case["hd"])
    fill = hip.KvPlan(cache, case["heads"], max_seqs=len(held), max_tokens=max(1, sum(held)), max_pages=len(pages))
    fill.set(held, held, pages)
    for layer in range(layers):
        fill.write(layer, Dev(keys[layer]), Dev(values[layer]))
    hip.synchronize(hip.stream(0))
    return cache


def _plain_cache(case, n_pages, slots, keys, values):
    """The same for the plain form: codes and scales [layers, slots of all pages ...]."""
    st = {}
    for name, x in (("keys", keys), ("values", values)):
        parts = _quantize(case["type"], x)
        st[name] = tuple(torch.zeros(x.shape[0], n_pages * case["page"], *p.shape[2:], dtype=p.dtype, device=DEV) for p in parts)
        for p, new in zip(st[name], parts):
            p[:, slots] = new
    return st


def _pages_of(case, held, seed):
    """Pages in a random order over the cache, ids one sequence after the other, where each position lives (slot =
    page id * page size + offset in the page), and the cache's page count, some more than are used."""
    need = [-(-t // case["page"]) for t in held]
    n_pages = sum(need) + 3
    pages = _page_order(n_pages, seed)[:sum(need)]
    slots = torch.cat([pages[sum(need[:i]) + torch.arange(t) // case["page"]] * case["page"] + torch.arange(t) % case["page"]
                       for i, t in enumerate(held)]).to(DEV)
    return pages.tolist(), need, slots, n_pages


def _prepare_tree(case, seed):
    keys, values, q = _inputs(case, seed)
    lens = _lens(case)
    held, new = [n + c for n, c in lens], [n for n, _ in lens]
    trees = [_parents(case, n) for n in new]
    pages, need, slots, n_pages = _pages_of(case, held, seed)
    row = torch.cat([torch.arange(c, c + n) + sum(held[:i]) for i, (n, c) in enumerate(lens)]).to(DEV)
    pos = torch.cat([c + torch.tensor(_depths(t)) for t, (_, c) in zip(trees, lens)]).to(DEV)
    st = {"case": case, "q": q, "k": keys[0, row].contiguous(), "v": values[0, row].contiguous(), "pos": pos}
    if own:
        hip = _hip()
        cache = _cache(hip, case, n_pages, held, pages, keys, values)
        plan = hip.KvPlan(cache, case["heads"], max_seqs=len(lens), max_tokens=len(row), max_pages=len(pages),
                          window=case["window"], sinks=case["sinks"], max_nodes=max(new))
        plan.set(new, held, pages, parents=sum(trees, []))
        hip.synchronize(hip.stream(0))
        return st | {"plan": plan, "q_out": torch.empty_like(q), "out": torch.empty_like(q)}
    longest, most = max(held), max(new)
    at, each = torch.arange(longest, device=DEV), torch.arange(most, device=DEV)
    first = torch.tensor([sum(held[:i]) for i in range(len(lens))], device=DEV)
    qfirst = torch.tensor([sum(new[:i]) for i in range(len(lens))], device=DEV)
    hidden = torch.ones(len(lens), most, longest, dtype=torch.bool)
    for i, (n, c) in enumerate(lens):
        hidden[i, :n, :n + c] = ~_seen(case, n, c)
        hidden[i, n:, 0] = False  # rows of the padding
    seq = torch.repeat_interleave(torch.arange(len(lens), device=DEV), torch.tensor(new, device=DEV))
    st |= _plain_cache(case, n_pages, slots, keys, values)
    return st | {"slot": slots[row], "padded": slots[first[:, None] + torch.minimum(at, torch.tensor(held, device=DEV)[:, None] - 1)],
                 "hidden": hidden.to(DEV)[:, None, None], "qseq": seq,
                 "qrow": qfirst[:, None] + torch.minimum(each, torch.tensor(new, device=DEV)[:, None] - 1),
                 "qat": torch.arange(len(row), device=DEV) - qfirst[seq]}


def _prepare_pick(case, seed):
    logits, tokens = _inputs(case, seed)
    new = [n for n, _ in _lens(case)]
    trees = [_parents(case, n) for n in new]
    st = {"case": case, "logits": logits, "tokens": tokens}
    rows = len(tokens)
    if own:
        hip = _hip()
        cache = hip.KvCache(hip.Q8_0, 1, len(new) * (-(-max(new) // 32)), 32, 1, 64)
        plan = hip.KvPlan(cache, 1, max_seqs=len(new), max_tokens=rows, max_pages=len(new) * (-(-max(new) // 32)),
                          max_nodes=max(new))
        plan.set(new, new, list(range(sum(-(-n // 32) for n in new))), parents=sum(trees, []))
        hip.synchronize(hip.stream(0))
        return st | {"plan": plan, "picks": _ints(rows), "n_kept": _ints(len(new)), "kept": _ints(rows), "next": _ints(len(new))}
    first = torch.tensor([sum(new[:i]) for i in range(len(new))], device=DEV)
    return st | {"parents": _rows_parents(case), "first": first, "depth": max(max(_depths(t)) for t in trees),
                 "qseq": torch.repeat_interleave(torch.arange(len(new), device=DEV), torch.tensor(new, device=DEV))}


def _prepare_keep(case, seed):
    keys, values, _ = _inputs(case, seed)
    lens = _lens(case)
    held, new = [n + c for n, c in lens], [n for n, _ in lens]
    paths = [_path(case, n) for n in new]
    pages, need, slots, n_pages = _pages_of(case, held, seed)
    st = {"case": case, "n_kept": [len(p) for p in paths], "kept": sum(paths, [])}
    if own:
        hip = _hip()
        cache = _cache(hip, case, n_pages, held, pages, keys, values)
        plan = hip.KvPlan(cache, case["heads"], max_seqs=len(lens), max_tokens=sum(new), max_pages=len(pages), max_nodes=max(new))
        plan.set(new, held, pages, parents=sum((_parents(case, n) for n in new), []))
        then = [c + len(p) for (_, c), p in zip(lens, paths)]
        after = hip.KvPlan(cache, case["heads"], max_seqs=len(lens), max_tokens=len(st["kept"]), max_pages=len(pages))
        after.set(st["n_kept"], then, [i for s, t in enumerate(then)
                                       for i in pages[sum(need[:s]):sum(need[:s]) + -(-t // case["page"])]])
        hip.synchronize(hip.stream(0))
        out = [torch.empty(case["layers"], len(st["kept"]), case["kv"], case["hd"], device=DEV) for _ in range(2)]
        return st | {"plan": plan, "after": after, "k_out": out[0], "v_out": out[1]}
    base = [sum(held[:i]) + c for i, (_, c) in enumerate(lens)]
    src = torch.tensor([b + i for b, p in zip(base, paths) for i in p], device=DEV)
    dst = torch.tensor([b + d for b, p in zip(base, paths) for d in range(len(p))], device=DEV)
    return st | _plain_cache(case, n_pages, slots, keys, values) | {"from": slots[src], "to": slots[dst], "read": slots[dst]}


def _prepare_copy(case, seed):
    keys, values = _inputs(case, seed)
    held = _filled_slots(case)
    order = _page_order(2 * len(held) + 3, seed).tolist()
    src, dst = order[:len(held)], order[len(held):2 * len(held)]
    st = {"case": case, "src": src, "dst": dst, "held": held}
    if own:
        hip = _hip()
        cache = _cache(hip, case, len(order), held, src, keys, values)
        after = hip.KvPlan(cache, case["heads"], max_seqs=len(held), max_tokens=1, max_pages=len(held))
        after.set([0] * len(held), held, dst)
        hip.synchronize(hip.stream(0))
        out = [torch.empty(case["layers"], sum(held), case["kv"], case["hd"], device=DEV) for _ in range(2)]
        return st | {"cache": cache, "after": after, "k_out": out[0], "v_out": out[1]}
    slots = [torch.cat([p * case["page"] + torch.arange(t) for p, t in zip(x, held)]).to(DEV) for x in (src, dst)]
    return st | _plain_cache(case, len(order), slots[0], keys, values) | {"from": slots[0], "to": slots[1], "read": slots[1]}


def _prepare_beam(case, seed):
    logits, scores, ended = _inputs(case, seed)
    st = {"case": case, "logits": logits, "scores": scores, "ended": ended, "end": 2}
    if own:
        hip = _hip()
        shape = (case["groups"], case["keep"])
        st |= {"beam": hip.BeamSelect(case["groups"], case["beams"], case["vocab"], case["keep"]), "parents": _ints(*shape),
               "tokens": _ints(*shape), "out": torch.empty(*shape, device=DEV)}
    return st


def prepare(case, seed):
    return {"tree": _prepare_tree, "pick": _prepare_pick, "keep": _prepare_keep, "copy": _prepare_copy,
            "beam": _prepare_beam}[case["kind"]](case, seed)


def run(st):
    c = st["case"]
    if not own:
        return {"tree": _plain_tree, "pick": _plain_pick, "keep": _plain_keep, "copy": _plain_keep,
                "beam": _plain_beam}[c["kind"]](st)
    if c["kind"] == "tree":
        plan = st["plan"]
        plan.write(0, Dev(st["k"]), Dev(st["v"]), q=Dev(st["q"]), q_out=Dev(st["q_out"]), theta=THETA, neox=c["neox"])
        plan.attention(0, Dev(st["q_out"]), Dev(st["out"]))
        return {"q": st["q_out"], "out": st["out"]}
    if c["kind"] == "pick":
        st["plan"].pick(Dev(st["logits"]), c["vocab"], Dev(st["tokens"]), Dev(st["picks"]), Dev(st["n_kept"]),
                        Dev(st["kept"]), Dev(st["next"]))
        return {x: st[x] for x in ("picks", "n_kept", "kept", "next")}
    if c["kind"] == "beam":
        st["beam"].select(Dev(st["logits"]), Dev(st["scores"]), c["groups"], c["beams"], c["vocab"], c["keep"],
                          Dev(st["parents"]), Dev(st["tokens"]), Dev(st["out"]), ended=_dev(st["ended"]), end_token=st["end"])
        return {"parents": st["parents"], "tokens": st["tokens"], "scores": st["out"]}
    if c["kind"] == "keep":
        st["plan"].keep(st["n_kept"], st["kept"])
    else:
        st["cache"].copy_pages(st["src"], st["dst"], st["held"])
    for layer in range(c["layers"]):
        st["after"].read(layer, Dev(st["k_out"][layer]), Dev(st["v_out"][layer]), new_only=c["kind"] == "keep")
    return {"keys": st["k_out"], "values": st["v_out"]}


# ---------------------------------------------------------------- what a pass cannot do without

def _held(case):
    """Bytes of a position's keys and values in a layer."""
    return 2 * case["kv"] * (case["hd"] * 4 if case["type"] == "f32" else -(-case["hd"] // QK) * BLOCK[case["type"]])


def _pairs(case):
    """Positions before the trees that some node sees, and (node, slot it sees) pairs, of all sequences."""
    seen = pairs = 0
    for n, c in _lens(case):
        for i, d in enumerate(_depths(_parents(case, n))):
            lo = max(0, c + d - case["window"] + 1) if case["window"] else 0  # first position of the window
            low, nodes = min(lo, c), c + d + 1 - max(lo, c)  # of the positions before the tree, of the path
            pairs += c - low + nodes + min(case["sinks"], lo)
            if i == 0:
                seen += c - low + min(case["sinks"], low)
    return seen, pairs


def _attention_flops(case):
    return 4 * _pairs(case)[1] * case["heads"] * case["hd"]


def work(case):
    kind = case["kind"]
    if kind in ("tree", "keep"):
        new, kv, hd, heads = sum(n for n, _ in _lens(case)), case["kv"], case["hd"], case["heads"]
    if kind == "tree":
        # queries in, rotated and their results out, keys and values in and into the cache, the cache before them
        return {"bytes": new * (12 * heads * hd + 8 * kv * hd + _held(case)) + _pairs(case)[0] * _held(case),
                "flops": _attention_flops(case) + new * hd * (3 * heads + 7 * kv)}
    if kind == "pick":
        rows = sum(n for n, _ in _lens(case))
        return {"bytes": rows * (case["vocab"] * 4 + 16) + 8 * case["seqs"], "flops": rows * case["vocab"]}
    if kind == "beam":
        rows = case["groups"] * case["beams"]
        return {"bytes": rows * (case["vocab"] * 4 + 8) + case["groups"] * case["keep"] * 12, "flops": rows * case["vocab"] * 4}
    # a slot that moves is read and written; what is read back is read once more as it is and written as f32
    if kind == "keep":
        paths = [_path(case, n) for n, _ in _lens(case)]
        moved, back = sum(i != d for p in paths for d, i in enumerate(p)), sum(map(len, paths))
    else:
        moved = back = sum(_filled_slots(case))
    elements = back * 2 * case["kv"] * case["hd"]
    return {"bytes": case["layers"] * ((2 * moved + back) * _held(case) + 4 * elements), "flops": case["layers"] * 2 * elements}


# ---------------------------------------------------------------- the same in 64 bits

def _f32(v):
    return v.float().double()


def _half64(v):
    """The binary16 next to v (f32 values in 64 bits) with halves rounded up in magnitude."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -14))) - 10)
    step = torch.where(v.abs() / step >= 2048, step * 2, step)  # log2 rounded down below a power of two
    step = torch.where((v.abs() / step < 1024) & (step > 2.0 ** -24), step / 2, step)
    return v.sign() * torch.floor(v.abs() / step + 0.5) * step


def _held64(kind, v):
    """What the cache holds for v (64 bits), by the block formats' definition: scales are
    binary16, and the codes are those of f32 arithmetic, each step of it rounded here."""
    if kind == "f32":
        return v
    hd = v.shape[-1]
    out = torch.empty_like(v)
    for b in range(0, hd, QK):
        x = _f32(v[..., b:b + QK])
        if kind == "q4_1":
            low = x.min(-1, keepdim=True).values
            d = _half64(_f32(_f32(x.max(-1, keepdim=True).values - low) / 15))
            low = _half64(low)
            x = _f32(x - low)
        else:
            d = _half64(_f32(x.abs().max(-1, keepdim=True).values / (127 if kind == "q8_0" else 7)))
        inv = torch.where(d == 0, d, _f32(1 / d))
        y = _f32(x * inv)
        y = _f32(y + 8) if kind == "q4_0" else y
        code = y.sign() * torch.floor(y.abs() + 0.5)
        code = code.clamp(-127, 127) if kind == "q8_0" else code.clamp(0, 15)
        out[..., b:b + QK] = d * (code - 8) if kind == "q4_0" else d * code if kind == "q8_0" else d * code + low
    return out


def _turned64(x, pos, neox):
    """x [tokens, heads, hd] rotated: pairs as complex numbers times e^(i pos theta^(-2r/hd))."""
    hd = x.shape[-1]
    angle = torch.outer(pos.double(), torch.exp(torch.arange(0, hd, 2, device=x.device).double() * (-math.log(THETA) / hd)))
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    x = x.double()
    z = torch.complex(x[..., :hd // 2].contiguous(), x[..., hd // 2:].contiguous()) if neox else \
        torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous())
    z = z * turn
    return torch.cat([z.real, z.imag], -1) if neox else torch.view_as_real(z).flatten(-2)


def _exact_tree(case, seed):
    keys, values, q = _inputs(case, seed)
    out = torch.empty(q.shape, dtype=torch.float64, device=DEV)
    turned = torch.empty_like(out)
    group, at, qat = case["heads"] // case["kv"], 0, 0
    for n, c in _lens(case):
        parents = _parents(case, n)
        # walked upwards from every node, unlike the plain form's
        seen = torch.zeros(n, c + n, dtype=torch.bool)
        pos = torch.empty(n, dtype=torch.long)
        for i in range(n):
            path, p = [], i
            while p >= 0:
                path.append(p)
                p = parents[p]
            pos[i] = c + len(path) - 1
            first = int(pos[i]) - case["window"] + 1 if case["window"] else 0
            seen[i, :c] = (torch.arange(c) >= first) | (torch.arange(c) < case["sinks"])
            for d, node in enumerate(reversed(path)):
                seen[i, c + node] = c + d >= first or c + d < case["sinks"]
        seen, pos = seen.to(DEV), pos.to(DEV)
        new = slice(qat, qat + n)
        turned[new] = _turned64(q[new], pos, case["neox"])
        k = torch.cat([keys[0, at:at + c].double(), _turned64(keys[0, at + c:at + c + n], pos, case["neox"])])
        k, v = _held64(case["type"], k), _held64(case["type"], values[0, at:at + c + n].double())
        for a in range(case["heads"]):
            s = (turned[new, a] @ k[:, a // group].T) / math.sqrt(case["hd"])
            out[new, a] = torch.softmax(s.masked_fill(~seen, -math.inf), -1) @ v[:, a // group]
        at, qat = at + c + n, qat + n
    return {"q": turned, "out": out}


def _exact_pick(case, seed):
    logits, tokens = _inputs(case, seed)
    picks = [int(r.double().cpu().numpy().argmax()) for r in logits]
    tokens, kept, counts, nexts, at = tokens.tolist(), [], [], [], 0
    for n, _ in _lens(case):
        parents = _parents(case, n)
        path = [0]
        while True:
            fit = [i for i in range(n) if parents[i] == path[-1] and tokens[at + i] == picks[at + path[-1]]]
            if not fit:
                break
            path.append(fit[0])
        kept += path + [-1] * (n - len(path))
        counts.append(len(path))
        nexts.append(picks[at + path[-1]])
        at += n
    return {x: torch.tensor(v, dtype=torch.int32, device=DEV) for x, v in
            (("picks", picks), ("n_kept", counts), ("kept", kept), ("next", nexts))}


def _exact_beam(case, seed):
    logits, scores, ended = _inputs(case, seed)
    keep, beams = case["keep"], case["beams"]
    out = {"parents": [], "tokens": [], "scores": []}
    for g in range(case["groups"]):
        found = []
        for b in range(beams):
            score = scores[g, b].double()
            if score == -math.inf:
                continue
            if ended is not None and ended[g, b] != 0:
                found.append((-float(score), b, 2))
                continue
            x = logits[g * beams + b].double()
            s = score + torch.log_softmax(x, -1)
            # all that can be among the best of this beam, ties with the last of them too
            least = torch.sort(s, descending=True).values[min(keep, len(s)) - 1]
            for t in torch.nonzero((s >= least) & (s > -math.inf)).flatten().tolist():
                found.append((-float(s[t]), b, t))
        found = sorted(found)[:keep]
        found += [(math.inf, -1, -1)] * (keep - len(found))
        for name, i, sign in (("scores", 0, -1), ("parents", 1, 1), ("tokens", 2, 1)):
            out[name].append([sign * f[i] for f in found])
    return {x: torch.tensor(v, dtype=torch.float64 if x == "scores" else torch.int32, device=DEV) for x, v in out.items()}


def exact(case, seed):
    kind = case["kind"]
    if kind in ("tree", "pick", "beam"):
        return {"tree": _exact_tree, "pick": _exact_pick, "beam": _exact_beam}[kind](case, seed)
    keys, values = _inputs(case, seed)[:2]
    if kind == "keep":
        rows, at = [], 0
        for n, c in _lens(case):
            rows += [at + c + i for i in _path(case, n)]
            at += n + c
        keys, values = keys[:, rows], values[:, rows]
    return {"keys": _held64(case["type"], keys.double()), "values": _held64(case["type"], values.double())}
