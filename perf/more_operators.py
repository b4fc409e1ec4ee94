"""The operators of a step that checks drafted tokens, and of the pages that it works on, as a
program that serves a language model calls them: the plain forms in elementary torch operations,
and `enceladus.decode`, `enceladus.draft` and `enceladus.pages`.

A case names its operator (`op`):

- `append`: new keys and values into their pages, rotated by positions of their own: the depths
  of a drafted tree, or the time, height and width of a picture's parts;
- `attend`: `nodes` drafted tokens at most of each of `batch` sequences over `length` cached ones
  at most (which count the drafted); a tree, or a chain;
- `accept`: which drafted tokens the model itself would have chosen, from its logits;
- `compact`: the accepted tokens move to the front of the drafted ones' slots, in the caches of
  all layers; or, of a long history, its first tokens and its last ones stay;
- `copy`: pages of all layers' caches into others;
- `fork`: sequences that go on from others, sharing their whole pages, and end again;
- `take`: sequences that grow by tokens, taking the pages for them, and give them back.

Lengths are ragged: they come from the case alone, so that `work` knows them; all values come
from the seed. Trees, ids and bookkeeping are such that a pass can be repeated on its own results.
"""

import math
import random

import numpy as np
import torch

own = False

_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16,
           "float8": torch.float8_e4m3fn}
_SIZE = {"float32": 4, "float16": 2, "bfloat16": 2, "float8": 1}
_K_SCALE, _V_SCALE = 0.03125, 0.0625        # of 8-bit caches


def listed():
    return [
        # a step's drafted trees, rotated by their depths: launches and latency
        {"name": "append_trees", "op": "append", "batch": 32, "new": 27, "past": 1000,
         "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "axes": 1, "woven": False,
         "interleaved": False, "dtype": "bfloat16", "cache": "bfloat16", "page": 16,
         "layout": "token"},
        # prompts of pictures and text, three axes: streaming
        {"name": "append_pictures", "op": "append", "batch": 13, "new": 4001, "past": 300,
         "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "axes": 3, "woven": False,
         "interleaved": False, "dtype": "bfloat16", "cache": "bfloat16", "page": 64,
         "layout": "head"},
        # one request and its drafted tree: the smallest call, latency
        {"name": "attend_one", "op": "attend", "batch": 1, "length": 1999, "nodes": 16,
         "tree": True, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bfloat16",
         "cache": "bfloat16", "page": 16, "layout": "token", "window": 0, "softcap": 0.0},
        # a serving batch with short and long sequences, a tree each
        {"name": "attend_batch", "op": "attend", "batch": 64, "length": 8192, "nodes": 27,
         "tree": True, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bfloat16",
         "cache": "bfloat16", "page": 16, "layout": "token", "window": 0, "softcap": 0.0},
        # one very long document: the length is all there is to split
        {"name": "attend_long", "op": "attend", "batch": 1, "length": 131075, "nodes": 32,
         "tree": True, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "float16",
         "cache": "float16", "page": 128, "layout": "head", "window": 0, "softcap": 0.0},
        # an 8-bit cache, many query heads to a key head, capped scores, a short chain
        {"name": "attend_8bit", "op": "attend", "batch": 24, "length": 16384, "nodes": 5,
         "tree": False, "heads": 64, "kv_heads": 8, "dim": 128, "dtype": "bfloat16",
         "cache": "float8", "page": 64, "layout": "token", "window": 0, "softcap": 30.0},
        # one request: latency
        {"name": "accept_one", "op": "accept", "batch": 1, "nodes": 16, "tree": True,
         "vocab": 32000, "dtype": "float32"},
        # a serving batch: the logits of all drafted tokens are read
        {"name": "accept_batch", "op": "accept", "batch": 64, "nodes": 27, "tree": True,
         "vocab": 128000, "dtype": "bfloat16"},
        # what a batch accepted, in the caches of 16 layers
        {"name": "compact_accepted", "op": "compact", "batch": 64, "length": 300, "nodes": 27,
         "evict": False, "layers": 16, "kv_heads": 8, "dim": 128, "cache": "bfloat16",
         "page": 16, "layout": "token"},
        # pages of 8 layers moved elsewhere: streaming
        {"name": "copy_pages", "op": "copy", "pairs": 300, "pages": 1000, "layers": 8,
         "kv_heads": 8, "dim": 128, "cache": "bfloat16", "page": 64, "layout": "token"},
        # beams: each of 64 requests goes on four times
        {"name": "fork_beams", "op": "fork", "batch": 64, "children": 192, "length": 500,
         "layers": 16, "kv_heads": 8, "dim": 128, "cache": "bfloat16", "page": 16,
         "layout": "token"},
        # a batch grows by its drafted tokens, in a large pool
        {"name": "take_step", "op": "take", "batch": 256, "length": 2000, "nodes": 27,
         "pages": 65536, "page": 16},
    ]


def _log(rng, lo, hi):
    """A whole number between `lo` and `hi`, spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "accept", "compact", "copy", "fork", "take"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    cache = "float8" if dtype != "float32" and rng.random() < 0.25 else dtype
    if op == "accept":
        vocab, nodes = _log(rng, 1000, 262144), _log(rng, 1, 64)
        most = 2.2e8 / (vocab * nodes)
        return {"op": op, "batch": _log(rng, 1, max(1, min(256, int(most)))), "nodes": nodes,
                "tree": rng.random() < 0.7, "vocab": vocab, "dtype": dtype}
    if op == "take":
        return {"op": op, "batch": _log(rng, 1, 512), "length": _log(rng, 1, 4000),
                "nodes": _log(rng, 1, 256), "pages": _log(rng, 20000, 200000),
                "page": rng.choice([16, 24, 64, 128])}
    case = {"op": op, "kv_heads": rng.choice([1, 2, 4, 8, 8, 16]),
            "dim": rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256]), "cache": cache,
            "page": rng.choice([1, 8, 16, 16, 24, 32, 64, 128, 256]),
            "layout": rng.choice(["token", "token", "head"])}
    row, size = case["kv_heads"] * case["dim"], _SIZE[cache]
    if op in ("compact", "copy", "fork"):
        case["layers"] = _log(rng, 1, 40)
        most = 1.2e9 / (2 * case["layers"] * row * size)       # tokens of all sequences
        if op == "copy":
            pages = _log(rng, 4, max(4, min(20000, int(most / case["page"]))))
            return case | {"pages": pages, "pairs": _log(rng, 1, pages // 2)}
        length = _log(rng, 1, min(4000, max(1, int(most))))
        whole = -(-(length + 64) // case["page"]) * case["page"]
        batch = _log(rng, 1, max(1, min(128, int(most / whole))))
        if op == "fork":
            children = max(1, min(4 * batch, int(most / case["page"])))
            return case | {"batch": batch, "length": length, "children": _log(rng, 1, children)}
        evict = length > 8 and rng.random() < 0.4
        return case | {"batch": batch, "length": length, "evict": evict,
                       "nodes": _log(rng, 2, length) if evict else _log(rng, 1, 64)}
    group = rng.choice([1, 2, 4, 4, 5, 7, 8, 16, 24])
    while case["kv_heads"] * group > 64:
        group = max(1, group // 2)
    case |= {"heads": case["kv_heads"] * group, "dtype": dtype}
    if op == "append":
        dim = case["dim"]
        new, past = _log(rng, 1, 4096), _log(rng, 1, 1500)
        most = 2.5e8 / (row * 2 * (new + past) + new * case["heads"] * dim * 2)
        return case | {"batch": _log(rng, 1, max(1, min(512, int(most)))), "new": new,
                       "past": past, "rotary": rng.choice([dim, dim, dim // 2, 16]),
                       "axes": rng.choice([1, 2, 3, 3, 4]), "woven": rng.random() < 0.3,
                       "interleaved": rng.random() < 0.3}
    tree = rng.random() < 0.6
    nodes = _log(rng, 1, 64 if tree else 256)
    length = nodes + _log(rng, 1, 131072)
    most = min(2.6e8 / (row * size * length), 1.7e10 / (nodes * case["heads"] * case["dim"] *
                                                      length))
    while most < 1 and length > nodes:
        length, most = max(nodes, length // 2), most * 2
    return case | {"batch": _log(rng, 1, max(1, min(256, int(most)))), "length": length,
                   "nodes": nodes, "tree": tree,
                   "window": rng.choice([0, 0, 0, _log(rng, 1, 8192)]),
                   "softcap": rng.choice([0.0, 0.0, 0.0, 50.0])}


def _spread(case, most, least=1, salt=0):
    """`batch` ragged lengths up to `most`, the longest among them: they go by the case."""
    rng = random.Random(1000003 * most + 7919 * case["batch"] + salt)
    n = [_log(rng, max(least, most // 64), max(least, most)) for _ in range(case["batch"])]
    n[case["batch"] // 2] = most
    return n


def _lengths(case):
    """(lengths in the cache, tokens of them that are new) of each sequence."""
    if case["op"] == "append":
        new = _spread(case, case["new"])
        return [p + n for p, n in zip(_spread(case, case["past"], salt=1), new)], new
    if case["op"] == "take":
        new = _spread(case, case["nodes"], salt=2)
        return [p + n for p, n in zip(_spread(case, case["length"], salt=1), new)], new
    if case["op"] == "compact" and not case["evict"]:
        new = _spread(case, case["nodes"], least=max(1, 2 * case["nodes"] // 3), salt=2)
        return [p + n for p, n in zip(_spread(case, case["length"], salt=1), new)], new
    if case["op"] == "compact":
        lens = _spread(case, case["length"])
        return lens, [min(n, case["nodes"]) for n in lens]
    new = _spread(case, case["nodes"], least=max(1, 2 * case["nodes"] // 3), salt=2)
    if case["op"] == "accept":
        return new, new
    lens = _spread(case, case["length"]) if case["batch"] > 1 else [case["length"]]
    return [max(p, n) for p, n in zip(lens, new)], new


def _normal(gen, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _cache(case, gen, count, pages, scale):
    """`count` caches of `pages` pages in one array, seen as [cache, page, token, head, element]
    whichever order the tokens and heads of a page are laid out in."""
    page, heads, dim = case["page"], case["kv_heads"], case["dim"]
    shape = (pages, page, heads, dim) if case["layout"] == "token" else \
        (pages, heads, page, dim)
    out = torch.empty((count, *shape), dtype=_DTYPES[case["cache"]], device="cuda")
    for c in out:
        c.copy_(torch.randn(shape, generator=gen, device="cuda") / scale)
    return out if case["layout"] == "token" else out.transpose(2, 3)


def _table(lens, page, gen, pages=None, width=None):
    """(block table, number of pages): the sequences' pages in any order, among others."""
    need = [-(-n // page) for n in lens]
    width, pages = width or max(need), pages or sum(need) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    first = torch.tensor([sum(need[:b]) for b in range(len(need))], device="cuda")
    at = first[:, None] + torch.arange(width, device="cuda")
    used = torch.arange(width, device="cuda") < torch.tensor(need, device="cuda")[:, None]
    table = torch.where(used, order[at.clamp(max=pages - 1)], torch.zeros_like(order[:1]))
    return table.contiguous(), pages


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(new):
    return _int32([sum(new[:b]) for b in range(len(new) + 1)])


def _trees(gen, new, nodes):
    """Random trees in an order in which parents come first: (their nodes' masks, int32
    [tokens, words], node j of a sequence being bit j % 32 of word j // 32; each node's parent
    [sequence, node])."""
    batch, words = len(new), -(-nodes // 32)
    parent = torch.zeros((batch, nodes), dtype=torch.int64, device="cuda")
    anc = torch.zeros((batch, nodes, 32 * words), dtype=torch.bool, device="cuda")
    rows = torch.arange(batch, device="cuda")
    u = torch.rand((batch, nodes), generator=gen, device="cuda")
    for j in range(nodes):
        if j:
            parent[:, j] = (u[:, j] ** 0.5 * j).long().clamp(max=j - 1)
            anc[:, j] = anc[rows, parent[:, j]]
        anc[:, j, j] = True
    bits = torch.ones(32, dtype=torch.int64, device="cuda") << torch.arange(32, device="cuda")
    mask = (anc.view(batch, nodes, words, 32) * bits).sum(-1)
    mask = torch.where(mask >= 1 << 31, mask - (1 << 32), mask).to(torch.int32)
    live = torch.arange(nodes, device="cuda") < torch.tensor(new, device="cuda")[:, None]
    return mask[live], parent


def _rotation(case, gen, lens, new):
    """cos, sin and positions of `append`: depths of a chain or a tree (one axis), or the places
    of pictures' parts (several)."""
    rotary, axes = case["rotary"], case["axes"]
    most = max(lens)
    at = torch.arange(most, device="cuda", dtype=torch.float64)[:, None]
    j = torch.arange(rotary // 2, device="cuda", dtype=torch.float64)
    angle = at * 10000.0 ** (-2 * j / rotary)
    base = torch.cat([torch.arange(n - m, n, device="cuda") for n, m in zip(lens, new)])
    if axes == 1:
        first = torch.cat([torch.full((m,), n - m, device="cuda") for n, m in zip(lens, new)])
        u = torch.rand(base.shape, generator=gen, device="cuda")
        positions = first + ((base - first) * u).long()
    else:
        side = torch.tensor([0, 7, 31, 3], device="cuda")[:axes, None]
        positions = torch.where(side > 0, base // 64 + base % side.clamp(min=1), base // 64)
    return angle.cos().float(), angle.sin().float(), positions.to(torch.int32).contiguous()


def _pair_axes(case):
    """The axis of each rotated pair: sections one after the other, or woven."""
    pairs, axes = case["rotary"] // 2, case["axes"]
    if axes == 1:
        return None
    if case["woven"]:
        return tuple(j % axes for j in range(pairs))
    # the first axis a quarter of the pairs, the others equal shares of the rest
    first = pairs // 4 if axes > 2 else pairs // 2
    return tuple(0 if j < first else min(axes - 1, 1 + (j - first) * (axes - 1) //
                                         max(1, pairs - first)) for j in range(pairs))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": dict(case)}
    op = case["op"]
    if op == "accept":
        new, vocab = _lengths(case)[1], case["vocab"]
        s["logits"] = torch.cat([_normal(gen, n, vocab).mul_(4).to(_DTYPES[case["dtype"]])
                                 for n in new])
        mask, parent = _trees(gen, new, case["nodes"])
        if case["tree"]:
            s["tree"] = mask
        else:
            parent = (torch.arange(case["nodes"], device="cuda") - 1).clamp(min=0).expand(
                len(new), -1)
        s["cu"] = _starts(new)
        live = torch.arange(case["nodes"], device="cuda") < \
            torch.tensor(new, device="cuda")[:, None]
        # most drafted tokens are the ones that the model would choose after their parents
        best = s["logits"].argmax(-1)
        guess = best[(s["cu"][:-1, None] + parent)[live]]
        other = torch.randint(0, vocab, guess.shape, generator=gen, device="cuda")
        hit = torch.rand(guess.shape, generator=gen, device="cuda") < 0.7
        s["tokens"] = torch.where(hit, guess, other).to(torch.int32)
        return s
    if op == "copy":
        s["caches"] = _cache(case, gen, 2 * case["layers"], case["pages"], 1.0)
        order = torch.randperm(case["pages"], generator=gen, device="cuda").to(torch.int32)
        s["source"], s["target"] = order[:case["pairs"]], order[-case["pairs"]:]
        s["list"] = list(s["caches"].unbind(0))
        return s
    if op == "take":
        lens, new = _lengths(case)
        old = [n - m for n, m in zip(lens, new)]
        width = -(-max(lens) // case["page"])
        s["pages"] = max(case["pages"], sum(-(-n // case["page"]) for n in lens) + 3)
        s["table"], _ = _table(old, case["page"], gen, s["pages"], width)
        s["lens"], s["old"], s["grown"] = _int32(old), _int32(old), _int32(lens)
        s["refs"] = _counts(s["table"], old, case["page"], s["pages"])
        return s
    if op == "fork":
        lens = _spread(case, case["length"])
        n, page = case["children"], case["page"]
        rows, width = case["batch"] + n, -(-max(lens) // page)
        pages = sum(-(-x // page) for x in lens) + n + 3
        table, _ = _table(lens + [0] * n, page, gen, pages, width)
        s["table"], s["lens"] = table, _int32(lens + [0] * n)
        s["refs"] = _counts(table, lens + [0] * n, page, pages)
        s["ended"] = _int32(lens + [0] * n)
        s["source"] = torch.arange(n, device="cuda", dtype=torch.int32) % case["batch"]
        s["target"] = case["batch"] + torch.randperm(n, generator=gen, device="cuda").int()
        s["caches"] = _cache(case, gen, 2 * case["layers"], pages, 1.0)
        s["list"] = list(s["caches"].unbind(0))
        assert rows == table.shape[0]
        return s
    lens, new = _lengths(case)
    table, pages = _table(lens, case["page"], gen)
    s["table"] = table
    if op == "compact":
        keep, counts, starts = _kept(case)
        s["keep"], s["counts"], s["starts"] = _int32(keep), _int32(counts), _int32(starts)
        s["lens"] = _int32(lens)
        s["caches"] = _cache(case, gen, 2 * case["layers"], pages, 1.0)
        s["list"] = list(s["caches"].unbind(0))
        return s
    dt = _DTYPES[case["dtype"]]
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    tokens = sum(new)
    s |= {"lens": _int32(lens), "cu": _starts(new)}
    s["k_cache"], s["v_cache"] = (_cache(case, gen, 1, pages, x if case["cache"] == "float8"
                                         else 1.0)[0] for x in (_K_SCALE, _V_SCALE))
    if op == "attend":
        s["q"] = _normal(gen, tokens, heads, dim, dtype=dt)
        if case["tree"]:
            s["tree"] = _trees(gen, new, case["nodes"])[0]
        return s
    row = _normal(gen, tokens, heads + 2 * kv, dim, dtype=dt)       # one fused projection
    s["q"], s["k"], s["v"] = row.split([heads, kv, kv], 1)
    s["cos"], s["sin"], s["positions"] = _rotation(case, gen, lens, new)
    return s


def _counts(table, lens, page, pages):
    """How many sequences hold each page: those of the table, and every third of the others."""
    refs = (torch.arange(pages, device="cuda") % 3 == 0).to(torch.int32)
    for b, n in enumerate(lens):
        if n:
            refs[table[b, :-(-n // page)].long()] = 1
    free = int((refs == 0).sum())
    need = table.shape[0] * (-(-max(lens) // page) + 16)     # no pass runs out of pages
    if free < need:
        held = torch.zeros(pages, dtype=torch.bool, device="cuda")
        for b, n in enumerate(lens):
            if n:
                held[table[b, :-(-n // page)].long()] = True
        refs = held.to(torch.int32)
    return refs


def _kept(case):
    """(tokens kept of each sequence, counted from its start and -1 behind them; how many; the
    starts) of `compact`. None is moved onto a slot that another one is read from."""
    lens, new = _lengths(case)
    rng = random.Random(case["length"] * 31 + case["batch"])
    keep, starts = [], []
    for n, m in zip(lens, new):
        if case["evict"]:                       # the first tokens, and the last ones
            starts.append(0)
            first = min(4, m // 2)
            last = min(m - first, (n - first) // 2)
            keep.append(list(range(first)) + list(range(n - last, n)))
        else:                                   # a path from the first drafted token on
            starts.append(n - m)
            k = min(m, rng.randint(1, 6))
            rest = range(k, m)
            keep.append([0] + sorted(rng.sample(rest, min(len(rest), k - 1))))
    counts = [len(k) for k in keep]
    width = max(counts)
    return [k + [-1] * (width - len(k)) for k in keep], counts, starts


def _scales(case):
    return (_K_SCALE, _V_SCALE) if case["cache"] == "float8" else (1.0, 1.0)


# -- the plain forms ---------------------------------------------------------------------

def _stored(x, scale, dtype):
    x = x / scale
    return x.clamp(-448.0, 448.0).to(dtype) if dtype == torch.float8_e4m3fn else x.to(dtype)


def _rotate(x, cos, sin, rotary, interleaved):
    x = x.float()
    cos, sin = cos[:, None], sin[:, None]
    part, rest = x[..., :rotary], x[..., rotary:]
    a, b = (part[..., ::2], part[..., 1::2]) if interleaved else part.chunk(2, -1)
    y = (a * cos - b * sin, b * cos + a * sin)
    y = torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)
    return torch.cat((y, rest), -1)


def _append(s, case):
    kc, vc, page = s["k_cache"], s["v_cache"], case["page"]
    tokens, lens, cu = s["k"].shape[0], s["lens"].long(), s["cu"].long()
    at = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(cu[1:], at, right=True)
    pos = lens[seq] - (cu[seq + 1] - at)
    turn, axes = s["positions"].long(), _pair_axes(case)
    if axes is None:
        cos, sin = s["cos"][turn], s["sin"][turn]
    else:
        turn = turn[torch.tensor(axes, device="cuda")].t()        # [tokens, pairs]
        cos, sin = (torch.gather(x, 0, turn) for x in (s["cos"], s["sin"]))
    k, q = (_rotate(s[n], cos, sin, case["rotary"], case["interleaved"]) for n in "kq")
    k_scale, v_scale = _scales(case)
    where, off = s["table"][seq, pos // page].long(), pos % page
    kc[where, off] = _stored(k, k_scale, kc.dtype)
    vc[where, off] = _stored(s["v"].float(), v_scale, vc.dtype)
    return q.to(s["q"].dtype), kc, vc


def _padded(cu, nodes):
    """(rows [sequence, node], which of them exist) of the ragged tokens."""
    j, cu = torch.arange(nodes, device="cuda"), cu.long()
    live = j < (cu[1:] - cu[:-1])[:, None]
    return torch.where(live, cu[:-1, None] + j, 0), live


def _ancestors(s, rows, live):
    """Which nodes a node sees, itself among them: [sequence, node, node]."""
    nodes = rows.shape[1]
    j = torch.arange(nodes, device="cuda")
    if "tree" not in s:
        return (j <= j[:, None]) & live[..., None] & live[:, None]
    words = s["tree"][rows]
    return ((words[:, :, j // 32] >> (j % 32)) & 1 != 0) & live[..., None] & live[:, None]


def _attend(s, case):
    table, lens = s["table"].long(), s["lens"].long()
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    rows, live = _padded(s["cu"], case["nodes"])
    batch, nodes = rows.shape
    k_scale, v_scale = _scales(case)
    most = table.shape[1] * case["page"]
    k = s["k_cache"][table].reshape(batch, most, kv, dim).float() * k_scale
    v = s["v_cache"][table].reshape(batch, most, kv, dim).float() * v_scale
    q = s["q"][rows].float().reshape(batch, nodes, kv, heads // kv, dim)
    q = q.permute(0, 2, 1, 3, 4).reshape(batch, kv, nodes * (heads // kv), dim)
    x = q @ k.permute(0, 2, 3, 1).contiguous() * (1.0 / math.sqrt(dim))
    if case["softcap"]:
        x = torch.tanh(x / case["softcap"]) * case["softcap"]
    past = lens - live.sum(1)
    at = torch.arange(most, device="cuda")
    j = at - past[:, None]
    seen = _ancestors(s, rows, live)
    node = j.clamp(0, nodes - 1)[:, None].expand(batch, nodes, most)
    see = torch.where((j < 0)[:, None], True, seen.gather(2, node) & (j < nodes)[:, None])
    if case["window"]:
        # the last of the tokens that a node sees
        behind = see.flip(-1).cumsum(-1).flip(-1)
        see &= behind <= case["window"]
    see = see[:, None, :, None].expand(batch, kv, nodes, heads // kv, most)
    x = x.masked_fill(~see.reshape(x.shape), -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    o = p @ v.permute(0, 2, 1, 3).contiguous() / p.sum(-1, keepdim=True)
    o = o.reshape(batch, kv, nodes, heads // kv, dim).permute(0, 2, 1, 3, 4)
    return o.reshape(batch, nodes, heads, dim)[live].to(s["q"].dtype)


def _accept(s, case):
    x, nodes = s["logits"], case["nodes"]
    vocab = torch.arange(x.shape[1], device="cuda")
    best = torch.where(x == x.amax(-1, keepdim=True), vocab, x.shape[1]).amin(-1)
    rows, live = _padded(s["cu"], nodes)
    best, token = best[rows], s["tokens"].long()[rows]
    seen = _ancestors(s, rows, live)
    depth = seen.sum(-1)
    self_ = torch.eye(nodes, dtype=torch.bool, device="cuda")
    up = seen & ~self_ & (depth[:, None] + 1 == depth[..., None])      # [node, its parent]
    match = (up & (best[:, None] == token[..., None])).any(-1)
    # of children with one token the first
    twin = (up.float() @ up.float().transpose(1, 2).contiguous() > 0) & \
        (token[..., None] == token[:, None])
    match &= ~(twin & torch.tril(torch.ones_like(self_), -1)).any(-1)
    match[:, 0] = True
    good = live & seen[..., 0] & (match[:, None] | ~seen).all(-1)
    count = good.sum(-1)
    path = torch.where(good, depth, nodes + 1).sort(dim=-1, stable=True).indices
    last = path.gather(1, (count - 1).clamp(min=0)[:, None])
    token = best.gather(1, last)[:, 0]
    path = torch.where(torch.arange(nodes, device="cuda") < count[:, None], path, -1)
    return path.int(), count.int(), token.int()


def _compact(s, case):
    keep, counts, starts = s["keep"].long(), s["counts"].long(), s["starts"].long()
    i = torch.arange(keep.shape[1], device="cuda")
    live = (i < counts[:, None]) & (keep != i)
    b = torch.arange(keep.shape[0], device="cuda")[:, None].expand_as(keep)[live]
    old, new = ((starts[:, None] + x)[live] for x in (keep, i.expand_as(keep)))
    c, table, page = s["caches"], s["table"].long(), case["page"]
    c[:, table[b, new // page], new % page] = c[:, table[b, old // page], old % page]
    s["lens"].copy_(starts + counts)
    return s["caches"], s["lens"]


def _copy(s):
    s["caches"][:, s["target"].long()] = s["caches"][:, s["source"].long()]
    return s["caches"]


def _free_pages(refs):
    """The free pages, lowest first, and others behind them."""
    return torch.where(refs == 0, 0, 1).sort(dim=0, stable=True).indices


def _let_go(refs, table, lens, to, page):
    i = torch.arange(table.shape[1], device="cuda")
    gone = (i >= -(-to // page)[:, None]) & (i < -(-lens // page)[:, None])
    refs.index_add_(0, table[gone].long(), torch.full_like(table[gone], -1))
    lens.copy_(torch.minimum(lens, to))


def _fork(s, case):
    refs, table, lens, page = s["refs"], s["table"], s["lens"], case["page"]
    source, target = s["source"].long(), s["target"].long()
    n = lens[source].long()
    need = (n % page != 0).long()
    end = need.cumsum(0)
    served = end <= (refs == 0).sum()
    source, target, n, need, end = (x[served] for x in (source, target, n, need, end))
    fresh = _free_pages(refs)[end - 1].int()
    i = torch.arange(table.shape[1], device="cuda")
    whole = i < (n // page)[:, None]
    shared = table[source]
    refs.index_add_(0, shared[whole].long(), torch.ones_like(shared[whole]))
    part = need > 0
    last = n // page
    old = shared.gather(1, last.clamp(max=table.shape[1] - 1)[:, None])[:, 0]
    table[target] = torch.where(whole, shared, table[target])
    table[target[part], last[part]] = fresh[part]
    refs[fresh[part].long()] = 1
    lens[target] = n.int()
    at = torch.arange(page, device="cuda")
    to = torch.where(part, fresh, 0).long()[:, None].expand(-1, page)
    of = torch.where(part, old, 0).long()[:, None].expand(-1, page)
    off = at.expand(len(to), page)
    some = part[:, None] & (at < (n % page)[:, None])
    s["caches"][:, to[some], off[some]] = s["caches"][:, of[some], off[some]]
    _let_go(refs, table, lens, s["ended"], page)
    return served.int(), table, refs, lens, s["caches"]


def _take(s, case):
    refs, table, lens, page = s["refs"], s["table"], s["lens"], case["page"]
    have, want = -(-lens // page), -(-s["grown"] // page)
    need = (want - have).clamp(min=0).long()
    end = need.cumsum(0)
    served = (end <= (refs == 0).sum()) | (need == 0)
    i = torch.arange(table.shape[1], device="cuda")
    new = (i >= have[:, None]) & (i < want[:, None]) & served[:, None]
    pages = _free_pages(refs)
    which = (end - need)[:, None] + i - have[:, None]
    table[new] = pages[which[new]].int()
    refs[table[new].long()] = 1
    lens.copy_(torch.where(served, s["grown"], lens))
    _let_go(refs, table, lens, s["old"], page)
    return served.int(), table, refs, lens


def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if own:
        from enceladus import decode, draft, pages
        if op == "append":
            k_scale, v_scale = _scales(case)
            q = decode.append_kv(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"],
                                 s["lens"], cu_tokens=s["cu"], q=s["q"], cos=s["cos"],
                                 sin=s["sin"], positions=s["positions"],
                                 pair_axes=_pair_axes(case), interleaved=case["interleaved"],
                                 k_scale=k_scale, v_scale=v_scale)
            return q, s["k_cache"], s["v_cache"]
        if op == "attend":
            k_scale, v_scale = _scales(case)
            return draft.tree_attention(s["q"], s["k_cache"], s["v_cache"], s["table"],
                                        s["lens"], s["cu"], tree=s.get("tree"),
                                        window=case["window"], softcap=case["softcap"],
                                        k_scale=k_scale, v_scale=v_scale)
        if op == "accept":
            return draft.accept(s["logits"], s["tokens"], s["cu"], tree=s.get("tree"),
                                most=case["nodes"])
        if op == "compact":
            pages.compact(s["list"], s["table"], s["starts"], s["keep"], s["counts"],
                          seq_lens=s["lens"])
            return s["caches"], s["lens"]
        if op == "copy":
            pages.copy(s["list"], s["source"], s["target"])
            return s["caches"]
        if op == "fork":
            served = pages.fork(s["list"], s["refs"], s["table"], s["lens"], s["source"],
                                s["target"])
            pages.free(s["refs"], s["table"], s["lens"], s["ended"], page_size=case["page"])
            return served, s["table"], s["refs"], s["lens"], s["caches"]
        served = pages.take(s["refs"], s["table"], s["lens"], s["grown"],
                            page_size=case["page"])
        pages.free(s["refs"], s["table"], s["lens"], s["old"], page_size=case["page"])
        return served, s["table"], s["refs"], s["lens"]
    if op == "copy":
        return _copy(s)
    return {"append": _append, "attend": _attend, "accept": _accept, "compact": _compact,
            "fork": _fork, "take": _take}[op](s, case)


def work(case):
    op = case["op"]
    if op == "accept":
        new = sum(_lengths(case)[1])
        n = new * case["vocab"]
        return {"bytes": n * _SIZE[case["dtype"]] + new * (8 + case["nodes"] // 8), "flops": n}
    if op == "take":
        lens, new = _lengths(case)
        need = sum(-(-n // case["page"]) - -(-(n - m) // case["page"])
                   for n, m in zip(lens, new))
        # free pages are looked for until there are enough; each is counted up and down
        return {"bytes": 4 * need * 6 + 24 * case["batch"], "flops": 4 * need}
    row = case["kv_heads"] * case["dim"]
    if op in ("copy", "fork", "compact"):
        token = 2 * case["layers"] * row * _SIZE[case["cache"]]
        if op == "copy":
            return {"bytes": 2 * case["pairs"] * (case["page"] * token + 4), "flops": 0}
        if op == "compact":
            keep, counts, _ = _kept(case)
            moved = sum(k >= 0 and k != i for row in keep for i, k in enumerate(row))
            return {"bytes": 2 * moved * token + 4 * sum(counts) + 16 * case["batch"],
                    "flops": 0}
        lens, page = _spread(case, case["length"]), case["page"]
        n = [lens[i % case["batch"]] for i in range(case["children"])]
        # a child's part of a page, its row of the table, and the counts up and down
        return {"bytes": sum(2 * (x % page) * token + 24 * -(-x // page) for x in n) +
                24 * len(n), "flops": 0}
    lens, new = _lengths(case)
    cache, size, q = _SIZE[case["cache"]], _SIZE[case["dtype"]], case["heads"] * case["dim"]
    if op == "append":
        tokens = sum(new)
        return {"bytes": tokens * (2 * row * (size + cache) + 2 * q * size + 4 * case["rotary"] +
                                   4 * case["axes"]),
                "flops": tokens * 6 * (row + q)}
    if case["window"]:
        lens = [min(n, case["window"] + m - 1) for n, m in zip(lens, new)]
    tokens, pages = sum(new), sum(-(-n // case["page"]) for n in lens)
    words = -(-case["nodes"] // 32) if case["tree"] else 0
    seen = sum(m * (min(n - m + 1, case["window"]) if case["window"] else n - m + 1)
               for n, m in zip(lens, new))
    return {"bytes": 2 * sum(lens) * row * cache + 2 * tokens * q * size + 4 * pages +
            4 * tokens * words, "flops": 4 * seen * q}


# -- the results in 64 bits ---------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "accept": _exact_accept,
            "compact": _exact_compact, "copy": _exact_copy, "fork": _exact_fork,
            "take": _exact_take}[case["op"]](s, case)


def _exact_append(s, case):
    lens, new = _lengths(case)
    page = case["page"]
    table = s["table"].cpu().numpy()
    k_scale, v_scale = _scales(case)
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    slot = np.concatenate([table[b, np.arange(n - m, n) // page].astype(np.int64) * page +
                           np.arange(n - m, n) % page
                           for b, (n, m) in enumerate(zip(lens, new))])
    slot = torch.from_numpy(slot).cuda()
    q, k = s["q"].double(), s["k"].double()
    r = case["rotary"]
    where = s["positions"].reshape(case["axes"], -1).long()
    axes = _pair_axes(case) or (0,) * (r // 2)
    for j, axis in enumerate(axes):
        z = torch.complex(s["cos"][where[axis], j].double(),
                          s["sin"][where[axis], j].double())[:, None]
        one, two = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + r // 2)
        for x in (q, k):
            y = torch.complex(x[..., one], x[..., two]) * z
            x[..., one], x[..., two] = y.real, y.imag
    k, v = k / k_scale, s["v"].double() / v_scale
    if case["cache"] == "float8":
        k, v = k.clamp(-448, 448), v.clamp(-448, 448)
    kc[slot // page, slot % page] = k
    vc[slot // page, slot % page] = v
    return q, kc, vc


def _bits(s, first, n):
    """[node, node]: which nodes the nodes of the sequence at row `first` see (NumPy)."""
    if "tree" not in s:
        return np.tril(np.ones((n, n), dtype=bool))
    words = s["tree"][first:first + n].contiguous().cpu().numpy().astype("<i4").view(np.uint8)
    return np.unpackbits(words, axis=1, bitorder="little")[:, :n].astype(bool)


def _exact_attend(s, case):
    lens, new = _lengths(case)
    if sum(n * m for n, m in zip(lens, new)) * case["heads"] * case["dim"] > 2e11:
        return None
    page, dim, kv = case["page"], case["dim"], case["kv_heads"]
    group = case["heads"] // kv
    k_scale, v_scale = _scales(case)
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for b, (n, m) in enumerate(zip(lens, new)):
        see = np.ones((m, n), dtype=bool)
        see[:, n - m:] = _bits(s, first, m)
        if case["window"]:
            rank = np.cumsum(see[:, ::-1], axis=1)[:, ::-1]
            see &= rank <= case["window"]
        hide = torch.from_numpy(~see).cuda()[:, None]
        at = torch.arange(n, device="cuda")
        where = s["table"][b].long()[at // page]
        k = s["k_cache"][where, at % page].double() * k_scale
        v = s["v_cache"][where, at % page].double() * v_scale
        for h in range(kv):
            q = s["q"][first:first + m, h * group:(h + 1) * group].double()
            x = (q.reshape(m * group, dim) @ k[:, h].t().contiguous()) / math.sqrt(dim)
            if case["softcap"]:
                x = case["softcap"] * torch.tanh(x / case["softcap"])
            x = x.view(m, group, n).masked_fill(hide, -math.inf)
            y = torch.softmax(x, -1).view(m * group, n) @ v[:, h].contiguous()
            out[first:first + m, h * group:(h + 1) * group] = y.view(m, group, dim)
        first += m
    return out


def _exact_accept(s, case):
    new = _lengths(case)[1]
    top = [torch.nonzero(x == x.max())[0, 0] for x in s["logits"]]
    best, token = torch.stack(top).tolist(), s["tokens"].tolist()
    paths, counts, chosen = [], [], []
    first = 0
    for m in new:
        see = _bits(s, first, m)
        depth = see.sum(1)
        path = [0]
        while True:
            now = path[-1]
            child = [j for j in range(m) if j != now and see[j, now] and
                     depth[j] == depth[now] + 1 and token[first + j] == best[first + now]]
            if not child:
                break
            path.append(child[0])
        paths.append(path + [-1] * (case["nodes"] - len(path)))
        counts.append(len(path))
        chosen.append(best[first + path[-1]])
        first += m
    return _int32(paths), _int32(counts), _int32(chosen)


def _exact_compact(s, case):
    page, c = case["page"], s["caches"].clone()
    for b, (first, count) in enumerate(zip(s["starts"].tolist(), s["counts"].tolist())):
        old = first + s["keep"][b, :count].long()
        new = first + torch.arange(count, device="cuda")
        row = s["table"][b].long()
        c[:, row[new // page], new % page] = s["caches"][:, row[old // page], old % page]
    return c, s["starts"] + s["counts"]


def _exact_copy(s, case):
    c = s["caches"].clone()
    for old, new in zip(s["source"].tolist(), s["target"].tolist()):
        c[:, new] = s["caches"][:, old]
    return c


def _exact_fork(s, case):
    page = case["page"]
    table, refs, lens = (s[n].tolist() for n in ("table", "refs", "lens"))
    c, served, held = s["caches"], [], refs[:]
    for a, b in zip(s["source"].tolist(), s["target"].tolist()):
        n = lens[a]
        whole, rest = n // page, n % page
        fresh = next((p for p, r in enumerate(held) if r == 0), None) if rest else -1
        served.append(int(fresh is not None))
        if fresh is None:
            continue
        table[b][:whole] = table[a][:whole]
        if rest:
            table[b][whole], held[fresh] = fresh, 1
            c[:, fresh, :rest] = c[:, table[a][whole], :rest]
    return _int32(served), _int32(table), s["refs"], s["lens"], c


def _exact_take(s, case):
    page = case["page"]
    table, refs = s["table"].tolist(), s["refs"].tolist()
    served, free = [], (p for p, r in enumerate(refs) if r == 0)
    left = refs.count(0)
    for b, (n, m) in enumerate(zip(s["old"].tolist(), s["grown"].tolist())):
        have, need = -(-n // page), max(0, -(-m // page) - -(-n // page))
        served.append(int(need <= left or need == 0))
        if served[-1]:
            left -= need
            for i in range(need):
                table[b][have + i] = next(free)
    return _int32(served), _int32(table), s["refs"], s["lens"]
