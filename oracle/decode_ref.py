"""64-bit forms of the `enceladus.decode` operators on CPU tensors (TEST INFRASTRUCTURE; see
oracle/__init__.py). They follow the definitions row by row, and share nothing with the kernels.
"""

from __future__ import annotations

import math

import torch


def slots(table, page, pages, first, last):
    """(page, offset) of positions [first, last) of one sequence, and which of them exist."""
    at = torch.arange(first, last)
    row = table.long()
    ids = row[at // page] if len(at) else at
    ok = (ids >= 0) & (ids < pages)
    return torch.where(ok, ids, 0), at % page, ok


def paged_attention(q, k_cache, v_cache, block_table, seq_lens, scale=None, window=0,
                    softcap=0.0, k_scale=1.0, v_scale=1.0):
    """(out, lse, A, S): A is each output's sum of |weight * value|, S the largest
    scale * sum |q k| of each head: what rounding errors are relative to."""
    batch, heads, dim = q.shape
    pages, page, kv, _ = k_cache.shape
    scale = 1 / math.sqrt(dim) if scale is None else scale
    out = torch.zeros(batch, heads, dim, dtype=torch.float64)
    mag = torch.zeros_like(out)
    lse = torch.full((batch, heads), -math.inf, dtype=torch.float64)
    smax = torch.zeros(batch, heads, dtype=torch.float64)
    for b in range(batch):
        n = max(0, min(int(seq_lens[b]), block_table.shape[1] * page))
        first = max(0, n - window) if window else 0
        ids, off, ok = slots(block_table[b], page, pages, first, n)
        ids, off = ids[ok], off[ok]
        if not len(ids):
            continue
        k = k_cache[ids, off].double() * k_scale
        v = v_cache[ids, off].double() * v_scale
        for h in range(heads):
            g = h // (heads // kv)
            qh = q[b, h].double()
            x = (k[:, g] @ qh) * scale
            smax[b, h] = ((k[:, g].abs() @ qh.abs()) * abs(scale)).max()
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            p = torch.softmax(x, 0)
            out[b, h] = p @ v[:, g]
            mag[b, h] = p @ v[:, g].abs()
            lse[b, h] = torch.logsumexp(x, 0)
    return out, lse, mag, smax


def rotate(x, cos, sin, interleaved):
    """x [heads, dim] at one position, cos and sin [R / 2]."""
    x = x.double().clone()
    half = cos.shape[0]
    one = torch.arange(half) * 2 if interleaved else torch.arange(half)
    two = one + 1 if interleaved else one + half
    a, b, c, s = x[:, one].clone(), x[:, two].clone(), cos.double(), sin.double()
    x[:, one], x[:, two] = a * c - b * s, b * c + a * s
    return x


def append_kv(k, v, k_cache, v_cache, block_table, seq_lens, cu_tokens=None, q=None, cos=None,
              sin=None, interleaved=False, k_scale=1.0, v_scale=1.0, q_out=None):
    """(queries, k cache, v cache, written): 64-bit copies, where skipped rows keep what
    `q_out` and the caches held, and `written` marks the slots that were written."""
    pages, page = k_cache.shape[:2]
    kc, vc = k_cache.double(), v_cache.double()
    done = torch.zeros(pages, page, dtype=torch.bool)
    qo = None if q is None else (q if q_out is None else q_out).double().clone()
    batch = block_table.shape[0]
    sat = k_cache.dtype == torch.float8_e4m3fn
    for b in range(batch):
        lo, hi = (b, b + 1) if cu_tokens is None else (int(cu_tokens[b]), int(cu_tokens[b + 1]))
        for t in range(lo, min(hi, k.shape[0])):
            pos = int(seq_lens[b]) - (hi - t)
            if pos < 0 or pos >= block_table.shape[1] * page:
                continue
            if cos is not None and pos >= cos.shape[0]:
                continue
            pg = int(block_table[b, pos // page])
            if not 0 <= pg < pages:
                continue
            kt = k[t].double() if cos is None else rotate(k[t], cos[pos], sin[pos], interleaved)
            kt, vt = kt / k_scale, v[t].double() / v_scale
            kc[pg, pos % page] = kt.clamp(-448, 448) if sat else kt
            vc[pg, pos % page] = vt.clamp(-448, 448) if sat else vt
            done[pg, pos % page] = True
            if q is not None:
                qo[t] = q[t].double() if cos is None else \
                    rotate(q[t], cos[pos], sin[pos], interleaved)
    return qo, kc, vc, done


def adjust_logits(logits, tokens=None, token_lens=None, prompt_lens=None, repetition=1.0,
                  frequency=0.0, presence=0.0, bias_ids=None, bias=None, allowed=None,
                  temperature=0.0):
    rows, vocab = logits.shape
    out = logits.double().clone()

    def of(x, b):
        return float(x[b]) if isinstance(x, torch.Tensor) else float(x)

    for b in range(rows):
        x = out[b]
        if tokens is not None:
            n = tokens.shape[1] if token_lens is None else int(token_lens[b])
            n = max(0, min(n, tokens.shape[1]))
            start = 0 if prompt_lens is None else max(0, int(prompt_lens[b]))
            seen, count = set(), {}
            for i, t in enumerate(tokens[b, :n].tolist()):
                if 0 <= t < vocab:
                    seen.add(t)
                    if i >= start:
                        count[t] = count.get(t, 0) + 1
            for t in seen:
                r = of(repetition, b)
                x[t] = x[t] / r if x[t] > 0 else x[t] * r
                c = count.get(t, 0)
                if c:
                    x[t] = x[t] - of(frequency, b) * c - of(presence, b)
        if bias is not None:
            for t, y in zip(bias_ids[b].tolist(), bias[b].tolist()):
                if 0 <= t < vocab:
                    x[t] += y
        if of(temperature, b) > 0:
            x /= of(temperature, b)
        if allowed is not None:
            v = torch.arange(vocab)
            bit = (allowed[b].long()[v // 32] >> (v % 32)) & 1
            x[bit == 0] = -math.inf
    return out
