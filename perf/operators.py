"""The operators of a decoding step over a paged cache, as a program that serves a language
model calls them: the plain forms in elementary torch operations, and `enceladus.decode`.

A case names its operator (`op`):

- `append`: the new keys and values of `batch` sequences go into their pages, rotated on the
  way, and the queries are rotated beside them; `new` tokens of each sequence at most (1: a
  decoding step, one token each);
- `attend`: one query token of each of `batch` sequences over `length` cached ones at most;
- `logits`: penalties for repeated tokens, biases, a grammar's mask and the temperature on
  `batch` rows of `vocab` logits.

Lengths are ragged: they come from the case alone, so that `work` knows them; all values come
from the seed.
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
        # one request in its decoding step: launches and latency
        {"name": "append_one", "op": "append", "batch": 1, "new": 1, "past": 1000, "heads": 32,
         "kv_heads": 8, "dim": 128, "rotary": 128, "interleaved": False, "dtype": "bfloat16",
         "cache": "bfloat16", "page": 16, "layout": "token", "fused": True},
        # the decoding step of a full batch, from the rows of one fused projection
        {"name": "append_step", "op": "append", "batch": 256, "new": 1, "past": 1000,
         "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "interleaved": False,
         "dtype": "bfloat16", "cache": "bfloat16", "page": 16, "layout": "token",
         "fused": True},
        # ragged prompts, many tokens at once: streaming
        {"name": "append_prompts", "op": "append", "batch": 13, "new": 4001, "past": 300,
         "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "interleaved": False,
         "dtype": "bfloat16", "cache": "bfloat16", "page": 64, "layout": "head",
         "fused": False},
        # an 8-bit cache, half of each head rotated by neighbouring pairs, pieces of prompts
        {"name": "append_8bit", "op": "append", "batch": 37, "new": 129, "past": 2000,
         "heads": 16, "kv_heads": 16, "dim": 64, "rotary": 32, "interleaved": True,
         "dtype": "float16", "cache": "float8", "page": 32, "layout": "token", "fused": True},
        # one request: the smallest call, latency
        {"name": "attend_one", "op": "attend", "batch": 1, "length": 1999, "spread": False,
         "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bfloat16", "cache": "bfloat16",
         "page": 16, "layout": "token", "window": 0, "softcap": 0.0},
        # a serving batch with short and long sequences
        {"name": "attend_batch", "op": "attend", "batch": 64, "length": 8192, "spread": True,
         "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bfloat16", "cache": "bfloat16",
         "page": 16, "layout": "token", "window": 0, "softcap": 0.0},
        # one very long document: the length is all there is to split
        {"name": "attend_long", "op": "attend", "batch": 1, "length": 131075, "spread": False,
         "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "float16", "cache": "float16",
         "page": 128, "layout": "head", "window": 0, "softcap": 0.0},
        # an 8-bit cache with many query heads to a key head, capped scores
        {"name": "attend_8bit", "op": "attend", "batch": 24, "length": 16384, "spread": True,
         "heads": 64, "kv_heads": 8, "dim": 128, "dtype": "bfloat16", "cache": "float8",
         "page": 64, "layout": "token", "window": 0, "softcap": 30.0},
        # every query head with keys of its own, in 32 bits, smaller heads, pages of odd size
        {"name": "attend_heads", "op": "attend", "batch": 12, "length": 2500, "spread": True,
         "heads": 16, "kv_heads": 16, "dim": 64, "dtype": "float32", "cache": "float32",
         "page": 24, "layout": "token", "window": 0, "softcap": 0.0},
        # one request's row: latency
        {"name": "logits_one", "op": "logits", "batch": 1, "vocab": 32000, "history": 700,
         "biases": 0, "mask": False, "dtype": "float32"},
        # a serving batch with all of it
        {"name": "logits_batch", "op": "logits", "batch": 256, "vocab": 128000,
         "history": 4096, "biases": 20, "mask": True, "dtype": "bfloat16"},
        # long histories, a vocabulary of odd size
        {"name": "logits_long", "op": "logits", "batch": 32, "vocab": 150001,
         "history": 32768, "biases": 300, "mask": False, "dtype": "float16"},
    ]


def _log(rng, lo, hi):
    """A whole number between `lo` and `hi`, spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "logits"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if op == "logits":
        vocab = _log(rng, 1000, 262144)
        return {"op": op, "batch": _log(rng, 1, min(256, (1 << 25) // vocab)), "vocab": vocab,
                "history": _log(rng, 1, 32768) if rng.random() < 0.5 else _log(rng, 1, 2048),
                "biases": rng.choice([0, 0, 7, 300]), "mask": rng.random() < 0.5,
                "dtype": dtype}
    kv_heads = rng.choice([1, 2, 4, 8, 8, 16])
    group = rng.choice([1, 2, 4, 4, 5, 7, 8, 16, 24])
    while kv_heads * group > 64:
        group = max(1, group // 2)
    dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256])
    case = {"op": op, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim,
            "dtype": dtype,
            "cache": "float8" if dtype != "float32" and rng.random() < 0.25 else dtype,
            "page": rng.choice([1, 8, 16, 16, 24, 32, 64, 128, 256]),
            "layout": rng.choice(["token", "token", "head"])}
    size = _SIZE[case["cache"]]
    if op == "append":
        new = 1 if rng.random() < 0.5 else _log(rng, 2, 4096)
        past = _log(rng, 1, 1500)
        most = 2.5e8 / (kv_heads * dim * 2 * (new + past) + new * case["heads"] * dim * 2)
        case |= {"batch": _log(rng, 1, max(1, min(512, int(most)))), "new": new, "past": past,
                 "rotary": rng.choice([dim, dim, dim // 2, 16, 0]),
                 "interleaved": rng.random() < 0.3, "fused": rng.random() < 0.5}
        return case
    length = _log(rng, 1, 131072)
    most = 4e8 / (kv_heads * dim * 2 * size * length)
    while most < 1:
        length, most = max(1, length // 2), most * 2
    case |= {"batch": _log(rng, 1, max(1, min(256, int(most)))), "length": length,
             "spread": rng.random() < 0.7,
             "window": rng.choice([0, 0, 0, _log(rng, 1, 8192)]),
             "softcap": rng.choice([0.0, 0.0, 0.0, 50.0])}
    return case


def _spread(case, most, least=1, salt=0):
    """`batch` ragged lengths up to `most`, the longest among them: they go by the case."""
    rng = random.Random(1000003 * most + 7919 * case["batch"] + salt)
    n = [_log(rng, max(least, most // 64), max(least, most)) for _ in range(case["batch"])]
    n[case["batch"] // 2] = most
    return n


def _lengths(case):
    """(lengths in the cache, tokens that are new) of each sequence."""
    if case["op"] == "attend":
        n = _spread(case, case["length"]) if case["spread"] else \
            [case["length"]] * case["batch"]
        return n, [1] * case["batch"]
    new = _spread(case, case["new"])
    return [p + n for p, n in zip(_spread(case, case["past"], salt=1), new)], new


def _normal(gen, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _cache(case, gen, pages, filled):
    """A cache of `pages` pages, seen as [page, token, head, element] whichever order the
    tokens and heads of a page are laid out in."""
    page, heads, dim = case["page"], case["kv_heads"], case["dim"]
    shape = (pages, page, heads, dim) if case["layout"] == "token" else \
        (pages, heads, page, dim)
    if not filled:
        c = torch.zeros(shape, dtype=torch.float32, device="cuda")
    else:
        c = torch.randn(shape, generator=gen, device="cuda")
        if case["cache"] == "float8":
            c /= filled
    c = c.to(_DTYPES[case["cache"]])
    return c if case["layout"] == "token" else c.permute(0, 2, 1, 3)


def _table(lens, page, gen):
    """(block table, number of pages): the sequences' pages in any order, among others."""
    need = [-(-n // page) for n in lens]
    width, pages = max(need), sum(need) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    first = torch.tensor([sum(need[:b]) for b in range(len(need))], device="cuda")
    at = first[:, None] + torch.arange(width, device="cuda")
    used = torch.arange(width, device="cuda") < torch.tensor(need, device="cuda")[:, None]
    table = torch.where(used, order[at.clamp(max=pages - 1)], torch.zeros_like(order[:1]))
    return table.contiguous(), pages


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": dict(case)}
    dt = _DTYPES[case["dtype"]]
    if case["op"] == "logits":
        rows, vocab, most = case["batch"], case["vocab"], case["history"]
        s["logits"] = _normal(gen, rows, vocab).mul_(4).to(dt)
        # words repeat: the ids of a history follow a steep distribution
        u = torch.rand((rows, most), generator=gen, device="cuda", dtype=torch.float64)
        s["tokens"] = (vocab ** u - 1).to(torch.int32).clamp_(0, vocab - 1)
        lens = _spread(case, most)
        s["token_lens"], s["prompt_lens"] = _int32(lens), _int32([n // 3 for n in lens])
        for name, lo, hi in (("repetition", 1.0, 1.5), ("frequency", 0.0, 0.5),
                             ("presence", 0.0, 0.5), ("temperature", 0.5, 1.5)):
            s[name] = torch.rand(rows, generator=gen, device="cuda") * (hi - lo) + lo
        if case["biases"]:
            n = case["biases"]
            base = torch.randint(0, vocab, (rows, 1), generator=gen, device="cuda")
            ids = (base + torch.arange(n, device="cuda") * 37) % vocab     # distinct ones
            ids[:, n - n // 4:] = -1                    # not every request has as many
            s["bias_ids"] = ids.to(torch.int32)
            s["bias"] = _normal(gen, rows, n)
        if case["mask"]:
            s["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)),
                                         generator=gen, device="cuda").to(torch.int32)
        return s
    lens, new = _lengths(case)
    table, pages = _table(lens, case["page"], gen)
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    attend = case["op"] == "attend"
    s |= {"table": table, "lens": _int32(lens),
          "k_cache": _cache(case, gen, pages, _K_SCALE if attend else 0),
          "v_cache": _cache(case, gen, pages, _V_SCALE if attend else 0)}
    tokens = sum(new)
    if attend:
        s["q"] = _normal(gen, tokens, heads, dim, dtype=dt)
        return s
    if case["fused"]:
        row = _normal(gen, tokens, heads + 2 * kv, dim, dtype=dt)
        s["q"], s["k"], s["v"] = row.split([heads, kv, kv], 1)
    else:
        s["q"], s["k"], s["v"] = (_normal(gen, tokens, n, dim, dtype=dt)
                                  for n in (heads, kv, kv))
    if case["new"] > 1:
        s["cu_tokens"] = _int32([sum(new[:b]) for b in range(len(new) + 1)])
    if case["rotary"]:
        at = torch.arange(max(lens), device="cuda", dtype=torch.float64)[:, None]
        j = torch.arange(case["rotary"] // 2, device="cuda", dtype=torch.float64)
        angle = at * 10000.0 ** (-2 * j / case["rotary"])
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    return s


def _scales(case):
    return (_K_SCALE, _V_SCALE) if case["cache"] == "float8" else (1.0, 1.0)


# -- the plain forms ---------------------------------------------------------------------

def _stored(x, scale, dtype):
    x = x / scale
    return x.clamp(-448.0, 448.0).to(dtype) if dtype == torch.float8_e4m3fn else x.to(dtype)


def _rotate(x, cos, sin, rotary, interleaved):
    x = x.float()
    if not rotary:
        return x
    cos, sin = cos[:, None], sin[:, None]
    part, rest = x[..., :rotary], x[..., rotary:]
    a, b = (part[..., ::2], part[..., 1::2]) if interleaved else part.chunk(2, -1)
    y = (a * cos - b * sin, b * cos + a * sin)
    y = torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)
    return torch.cat((y, rest), -1)


def _append(s, case):
    kc, vc, page = s["k_cache"], s["v_cache"], case["page"]
    tokens, lens = s["k"].shape[0], s["lens"].long()
    at = torch.arange(tokens, device="cuda")
    if case["new"] > 1:
        cu = s["cu_tokens"].long()
        seq = torch.searchsorted(cu[1:], at, right=True)
        pos = lens[seq] - (cu[seq + 1] - at)
    else:
        seq, pos = at, lens - 1
    cos, sin = (s["cos"][pos], s["sin"][pos]) if case["rotary"] else (None, None)
    k, q = (_rotate(s[n], cos, sin, case["rotary"], case["interleaved"]) for n in "kq")
    k_scale, v_scale = _scales(case)
    where, off = s["table"][seq, pos // page].long(), pos % page
    kc[where, off] = _stored(k, k_scale, kc.dtype)
    vc[where, off] = _stored(s["v"].float(), v_scale, vc.dtype)
    return q.to(s["q"].dtype), kc, vc


def _attend(s, case):
    q, table, lens = s["q"].float(), s["table"].long(), s["lens"].long()
    rows, heads, dim = q.shape
    kv = case["kv_heads"]
    k_scale, v_scale = _scales(case)
    most = table.shape[1] * case["page"]
    k = s["k_cache"][table].reshape(rows, most, kv, dim).float() * k_scale
    v = s["v_cache"][table].reshape(rows, most, kv, dim).float() * v_scale
    q = q.reshape(rows, kv, heads // kv, dim)
    x = q @ k.permute(0, 2, 3, 1).contiguous() * (1.0 / math.sqrt(dim))
    if case["softcap"]:
        x = torch.tanh(x / case["softcap"]) * case["softcap"]
    at = torch.arange(most, device="cuda")
    live = at < lens[:, None]
    if case["window"]:
        live &= at >= lens[:, None] - case["window"]
    x = x.masked_fill(~live[:, None, None], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    o = p @ v.permute(0, 2, 1, 3).contiguous() / p.sum(-1, keepdim=True)
    return o.reshape(rows, heads, dim).to(s["q"].dtype)


def _adjust(s, case):
    x, tokens = s["logits"].float(), s["tokens"].long()
    rows, vocab = x.shape
    at = torch.arange(tokens.shape[1], device="cuda")
    live = at < s["token_lens"][:, None]
    said = live & (at >= s["prompt_lens"][:, None])
    count = torch.zeros((2, rows, vocab), dtype=torch.int32, device="cuda")
    count[0].scatter_add_(1, tokens, live.int())
    count[1].scatter_add_(1, tokens, said.int())
    rep, freq, pres, temp = (s[n][:, None] for n in
                             ("repetition", "frequency", "presence", "temperature"))
    x = torch.where(count[0] > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - freq * count[1].float() - pres * (count[1] > 0).float()
    if case["biases"]:
        ids, value = s["bias_ids"].long(), s["bias"]
        x = x.scatter_add(1, ids.clamp(min=0), torch.where(ids >= 0, value, 0.0))
    x = x / temp
    if case["mask"]:
        v = torch.arange(vocab, device="cuda")
        bit = (s["allowed"][:, v // 32] >> (v % 32)) & 1
        x = x.masked_fill(bit == 0, -math.inf)
    return x.to(s["logits"].dtype)


def run(state):
    s, case = state, state["case"]
    if own:
        from enceladus import decode
        if case["op"] == "append":
            k_scale, v_scale = _scales(case)
            q = decode.append_kv(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"],
                                 s["lens"], cu_tokens=s.get("cu_tokens"), q=s["q"],
                                 cos=s.get("cos"), sin=s.get("sin"),
                                 interleaved=case["interleaved"], k_scale=k_scale,
                                 v_scale=v_scale)
            return q, s["k_cache"], s["v_cache"]
        if case["op"] == "attend":
            k_scale, v_scale = _scales(case)
            return decode.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"],
                                          s["lens"], window=case["window"],
                                          softcap=case["softcap"], k_scale=k_scale,
                                          v_scale=v_scale)
        return decode.adjust_logits(s["logits"], tokens=s["tokens"],
                                    token_lens=s["token_lens"], prompt_lens=s["prompt_lens"],
                                    repetition=s["repetition"], frequency=s["frequency"],
                                    presence=s["presence"], bias_ids=s.get("bias_ids"),
                                    bias=s.get("bias"), allowed=s.get("allowed"),
                                    temperature=s["temperature"])
    return {"append": _append, "attend": _attend, "logits": _adjust}[case["op"]](s, case)


def work(case):
    size = _SIZE[case["dtype"]]
    if case["op"] == "logits":
        rows, n = case["batch"], case["batch"] * case["vocab"]
        said = sum(_spread(case, case["history"]))
        return {"bytes": 2 * n * size + 4 * said + (n // 8 if case["mask"] else 0) +
                rows * (8 * case["biases"] + 24), "flops": 6 * n + 2 * said}
    lens, new = _lengths(case)
    row = case["kv_heads"] * case["dim"]
    cache = _SIZE[case["cache"]]
    if case["op"] == "append":
        tokens, q = sum(new), case["heads"] * case["dim"]
        return {"bytes": tokens * (2 * row * (size + cache) + 2 * q * size +
                                   4 * case["rotary"]),
                "flops": tokens * 6 * (row + q)}
    if case["window"]:
        lens = [min(n, case["window"]) for n in lens]
    pages = sum(-(-n // case["page"]) for n in lens)
    q = case["heads"] * case["dim"]
    return {"bytes": 2 * sum(lens) * row * cache + 2 * case["batch"] * q * size + 4 * pages,
            "flops": 4 * sum(lens) * q}


# -- the results in 64 bits ---------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logits":
        return _exact_logits(s, case)
    lens, new = _lengths(case)
    page, dim = case["page"], case["dim"]
    table = s["table"].cpu().numpy()
    k_scale, v_scale = _scales(case)
    if case["op"] == "append":
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        turn = np.concatenate([np.arange(n - m, n) for n, m in zip(lens, new)])
        slot = np.concatenate([table[b, np.arange(n - m, n) // page].astype(np.int64) * page +
                               np.arange(n - m, n) % page
                               for b, (n, m) in enumerate(zip(lens, new))])
        slot, turn = torch.from_numpy(slot).cuda(), torch.from_numpy(turn).cuda()
        q, k = s["q"].double(), s["k"].double()
        r = case["rotary"]
        if r:
            z = torch.complex(s["cos"][turn].double(), s["sin"][turn].double())[:, None]
            for x in (q, k):
                one, two = (slice(0, r, 2), slice(1, r, 2)) if case["interleaved"] else \
                    (slice(0, r // 2), slice(r // 2, r))
                y = torch.complex(x[..., one], x[..., two]) * z
                x[..., one], x[..., two] = y.real, y.imag
        k, v = k / k_scale, s["v"].double() / v_scale
        if case["cache"] == "float8":
            k, v = k.clamp(-448, 448), v.clamp(-448, 448)
        kc[slot // page, slot % page] = k
        vc[slot // page, slot % page] = v
        return q, kc, vc
    kv, group = case["kv_heads"], case["heads"] // case["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        first = max(0, n - case["window"]) if case["window"] else 0
        at = torch.arange(first, n, device="cuda")
        where = s["table"][b].long()[at // page]
        k = s["k_cache"][where, at % page].double() * k_scale
        v = s["v_cache"][where, at % page].double() * v_scale
        for h in range(kv):
            q = s["q"][b, h * group:(h + 1) * group].double()
            x = q @ k[:, h].t().contiguous() / math.sqrt(dim)
            if case["softcap"]:
                x = case["softcap"] * torch.tanh(x / case["softcap"])
            out[b, h * group:(h + 1) * group] = torch.softmax(x, -1) @ v[:, h].contiguous()
    return out


def _exact_logits(s, case):
    vocab = case["vocab"]
    out = s["logits"].double()
    ends, starts = s["token_lens"].tolist(), s["prompt_lens"].tolist()
    numbers = {n: s[n].double().tolist() for n in
               ("repetition", "frequency", "presence", "temperature")}
    for b, x in enumerate(out):
        seen = torch.bincount(s["tokens"][b, :ends[b]].long(), minlength=vocab) > 0
        c = torch.bincount(s["tokens"][b, starts[b]:ends[b]].long(), minlength=vocab)
        rep = numbers["repetition"][b]
        y = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
        y -= numbers["frequency"][b] * c + numbers["presence"][b] * (c > 0)
        if case["biases"]:
            ids = s["bias_ids"][b]
            y.index_add_(0, ids[ids >= 0].long(), s["bias"][b][ids >= 0].double())
        y /= numbers["temperature"][b]
        if case["mask"]:
            words = s["allowed"][b].cpu().numpy().astype("<i4").view(np.uint8)
            bits = np.unpackbits(words, bitorder="little")[:vocab]
            y[torch.from_numpy(bits == 0).cuda()] = -math.inf
        out[b] = y
    return out
