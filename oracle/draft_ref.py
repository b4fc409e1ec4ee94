"""64-bit forms of the `enceladus.draft` and `enceladus.pages` operators, and of rotations by
positions of several axes, on CPU tensors (TEST INFRASTRUCTURE; see oracle/__init__.py). They follow
the definitions token by token, and share nothing with the kernels.
"""

from __future__ import annotations

import math

import torch

from oracle.decode_ref import rotate, slots


def seen_by(tree, row, i, n):
    """Which of its sequence's n new tokens the i-th one, at row `row`, sees."""
    j = torch.arange(n)
    if tree is None:
        return j <= i
    words = tree[row].long()
    inside = j // 32 < len(words)
    return inside & ((words[(j // 32).clamp(max=len(words) - 1)] >> (j % 32)) & 1 != 0)


def spans(cu, rows):
    """(first row, number of rows) of each sequence."""
    got = []
    for b in range(len(cu) - 1):
        lo = min(max(int(cu[b]), 0), rows)
        got.append((lo, max(0, min(int(cu[b + 1]), rows) - lo)))
    return got


def tree_attention(q, k_cache, v_cache, block_table, seq_lens, cu, tree=None, scale=None, window=0,
                   softcap=0.0, k_scale=1.0, v_scale=1.0):
    """(out, lse, A, S, done): A is each output's sum of |weight * value|, S the largest
    scale * sum |q k| of each head (what rounding errors are relative to), `done` the rows of
    some sequence."""
    rows, heads, dim = q.shape
    pages, page, kv, _ = k_cache.shape
    group = heads // kv
    scale = 1 / math.sqrt(dim) if scale is None else scale
    out = torch.zeros(rows, heads, dim, dtype=torch.float64)
    mag = torch.zeros_like(out)
    lse = torch.full((rows, heads), -math.inf, dtype=torch.float64)
    smax = torch.zeros(rows, heads, dtype=torch.float64)
    done = torch.zeros(rows, dtype=torch.bool)
    for b, (first, n) in enumerate(spans(cu, rows)):
        length = max(0, int(seq_lens[b]))
        past = length - n
        end = min(length, block_table.shape[1] * page)
        done[first:first + n] = True
        ids, off, ok = slots(block_table[b], page, pages, 0, end)
        at = torch.arange(end)
        for i in range(n):
            see = at < past
            new = seen_by(tree, first + i, i, n)
            for j in range(n):
                if 0 <= past + j < end:
                    see[past + j] = new[j]
            if window:
                rank = torch.flip(torch.cumsum(torch.flip(see.long(), (0,)), 0), (0,))
                see &= rank <= window
            see &= ok
            if not see.any():
                continue
            k = k_cache[ids[see], off[see]].double() * k_scale
            v = v_cache[ids[see], off[see]].double() * v_scale
            for g in range(kv):
                h = slice(g * group, (g + 1) * group)
                qh = q[first + i, h].double()
                x = qh @ k[:, g].T * scale
                smax[first + i, h] = (qh.abs() @ k[:, g].abs().T * abs(scale)).amax(-1)
                if softcap:
                    x = softcap * torch.tanh(x / softcap)
                p = torch.softmax(x, -1)
                out[first + i, h] = p @ v[:, g]
                mag[first + i, h] = p @ v[:, g].abs()
                lse[first + i, h] = torch.logsumexp(x, -1)
    return out, lse, mag, smax, done


def accept(logits, tokens, cu, tree=None, most=None):
    rows = logits.shape[0]
    most = (32 * tree.shape[1] if tree is not None else rows) if most is None else most
    paths, counts, chosen = [], [], []

    def best(row):
        x = logits[row].double()
        nan = torch.isnan(x)
        return int(torch.nonzero(nan if nan.any() else x == x.max())[0, 0])

    for first, n in spans(cu, rows):
        if tree is not None:
            n = min(n, 32 * tree.shape[1])
        if n == 0 or most == 0:
            paths.append([-1] * most), counts.append(0), chosen.append(-1)
            continue
        see = torch.stack([seen_by(tree, first + i, i, n) for i in range(n)])
        depth = see.sum(1)
        path = [0]
        while len(path) < most:
            now = path[-1]
            child = [j for j in range(n) if j != now and see[j, now] and
                     depth[j] == depth[now] + 1 and int(tokens[first + j]) == best(first + now)]
            if not child:
                break
            path.append(child[0])
        paths.append(path + [-1] * (most - len(path)))
        counts.append(len(path))
        chosen.append(best(first + path[-1]))
    shape = (len(paths), most)
    return (torch.tensor(paths, dtype=torch.int32).reshape(shape),
            torch.tensor(counts, dtype=torch.int32), torch.tensor(chosen, dtype=torch.int32))


def turned(x, cos, sin, places, pair_axes, interleaved):
    """x [heads, dim] with pair j turned by row places[pair_axes[j]] of cos and sin."""
    axes = torch.tensor(pair_axes)
    at = torch.tensor(places)[axes]
    j = torch.arange(len(axes))
    return rotate(x, cos[at, j], sin[at, j], interleaved)


def append_kv(k, v, k_cache, v_cache, block_table, seq_lens, cu_tokens=None, q=None, cos=None,
              sin=None, interleaved=False, k_scale=1.0, v_scale=1.0, q_out=None, positions=None,
              pair_axes=None):
    """`decode_ref.append_kv` with positions of the tokens' own."""
    pages, page = k_cache.shape[:2]
    kc, vc = k_cache.double(), v_cache.double()
    done = torch.zeros(pages, page, dtype=torch.bool)
    qo = None if q is None else (q if q_out is None else q_out).double().clone()
    sat = k_cache.dtype == torch.float8_e4m3fn
    positions = positions.reshape(-1, positions.shape[-1])
    pair_axes = (0,) * cos.shape[1] if pair_axes is None else pair_axes
    batch = block_table.shape[0]
    cu = torch.arange(batch + 1) if cu_tokens is None else cu_tokens
    for b, (lo, n) in enumerate(spans(cu, k.shape[0])):
        for t in range(lo, lo + n):
            pos = max(0, int(seq_lens[b])) - (lo + n - t)
            places = positions[:, t].tolist()
            if pos < 0 or pos >= block_table.shape[1] * page or \
                    not all(0 <= p < cos.shape[0] for p in places):
                continue
            pg = int(block_table[b, pos // page])
            if not 0 <= pg < pages:
                continue
            kt = turned(k[t], cos, sin, places, pair_axes, interleaved) / k_scale
            vt = v[t].double() / v_scale
            kc[pg, pos % page] = kt.clamp(-448, 448) if sat else kt
            vc[pg, pos % page] = vt.clamp(-448, 448) if sat else vt
            done[pg, pos % page] = True
            if q is not None:
                qo[t] = turned(q[t], cos, sin, places, pair_axes, interleaved)
    return qo, kc, vc, done


# -- pages: plain lists of whole numbers --------------------------------------------------------

def pages_of(tokens, page):
    return -(-max(tokens, 0) // page)


def take(refs, table, lens, new, page):
    """(served, refs, table, lens) after `pages.take`."""
    refs, table, lens = list(refs), [list(r) for r in table], list(lens)
    width = len(table[0]) if table else 0
    want = []
    for n, m in zip(lens, new):
        have, need = pages_of(n, page), pages_of(m, page)
        want.append(0 if m <= n else None if need > width or have > width else need - have)
    free = [p for p, r in enumerate(refs) if r == 0]
    served, end = [], 0
    for b, need in enumerate(want):
        end += need or 0
        ok = need == 0 or (need is not None and end <= len(free))
        served.append(int(ok))
        if ok and new[b] > lens[b]:
            have = pages_of(lens[b], page)
            for i in range(need):
                table[b][have + i] = free[end - need + i]
                refs[free[end - need + i]] = 1
            lens[b] = new[b]
    return served, refs, table, lens


def free(refs, table, lens, new, page):
    """(refs, lens) after `pages.free`."""
    refs, lens = list(refs), list(lens)
    for b, (n, m) in enumerate(zip(list(lens), new)):
        m = max(m, 0)
        if m >= n:
            continue
        for i in range(pages_of(m, page), min(pages_of(n, page), len(table[b]))):
            p = table[b][i]
            if 0 <= p < len(refs) and refs[p] > 0:
                refs[p] -= 1
        lens[b] = m
    return refs, lens


def fork(refs, table, lens, source, target, page):
    """(served, refs, table, lens, copies) after `pages.fork`; copies are (page, page, tokens)."""
    refs, table, lens = list(refs), [list(r) for r in table], list(lens)
    before, width, rows = list(lens), len(table[0]), len(table)
    unused = [p for p, r in enumerate(refs) if r == 0]
    served, copies, taken, targets = [], [], 0, set()
    for a, b in zip(source, target):
        first = b not in targets
        targets.add(b)
        ok = 0 <= a < rows and 0 <= b < rows and first and b not in source and \
            before[b] <= 0 and pages_of(before[a], page) <= width
        n = max(before[a], 0) if ok else 0
        whole, rest = divmod(n, page)
        part = ok and rest > 0 and 0 <= table[a][whole] < len(refs)
        taken += part
        if part and taken > len(unused):
            ok = False
        served.append(int(ok))
        if not ok:
            continue
        for i in range(pages_of(n, page)):
            p = table[a][i]
            if part and i == whole:
                new = unused[taken - 1]
                copies.append((p, new, rest))
                table[b][i], refs[new] = new, 1
            else:
                table[b][i] = p
                if 0 <= p < len(refs) and refs[p] >= 0:
                    refs[p] += 1
        lens[b] = n
    return served, refs, table, lens, copies


def compact(cache, table, starts, keep, counts):
    """A cache after `pages.compact`, and the new lengths (None: left as it is)."""
    out, lens = cache.clone(), []
    pages, page = cache.shape[:2]
    for b, (start, count) in enumerate(zip(starts, counts)):
        count = min(max(count, 0), len(keep[b]))
        capacity = len(table[b]) * page
        lens.append(None if start < 0 else min(start + count, 2 ** 31 - 1))
        if not 0 <= start < capacity:
            continue
        for i in range(count):
            old, new = start + keep[b][i], start + i
            if keep[b][i] <= i or old >= capacity:
                continue
            p, q = table[b][old // page], table[b][new // page]
            if 0 <= p < pages and 0 <= q < pages:
                out[q, new % page] = cache[p, old % page]
    return out, lens
