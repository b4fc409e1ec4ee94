"""`enceladus.draft`, and appending by positions of several axes, on the GPU against 64-bit forms:
types, head layouts, lengths, trees, windows, masked places that are not finite, ragged and padded
rows, streams, graphs, and a run of the operators together.

Tolerances count the roundings of 32-bit arithmetic (unit 2^-24) relative to the magnitudes that are
summed, and half a step of the output's type.
"""

import math

import numpy as np
import pytest
import torch

import enceladus
from enceladus import decode, draft, pages
from oracle import draft_ref as R
from tests.test_gpu_decode import (BF16, F8, F16, F32, SUB, U, attention_tolerance, cache, close,
                                   half_step, on_gpu, only_live, rand, table_for)

pytestmark = pytest.mark.gpu


def int32(values):
    return torch.tensor(values, dtype=torch.int32)


def starts_of(new, before=0):
    return int32([before + sum(new[:b]) for b in range(len(new) + 1)])


def trees(gen, new, words, empty=0.0):
    """Masks of random trees over each sequence's new tokens, in an order in which parents come
    first; some rows (a share of `empty`) have no bit at all. Bits behind a sequence's tokens are
    wild."""
    rows = []
    for n in new:
        masks = []
        for j in range(n):
            m = 1 << j
            if j:
                m |= masks[int(torch.randint(0, j, (1,), generator=gen))]
            masks.append(m)
        for j in range(n):
            if empty and float(torch.rand(1, generator=gen)) < empty:
                masks[j] = 0
        wild = ((1 << 32 * words) - 1) >> n << n & (0x5A5A5A5A << max(0, 32 * words - 40))
        rows += [[(m | wild) >> 32 * w & 0xFFFFFFFF for w in range(words)] for m in masks]
    t = torch.tensor(rows, dtype=torch.int64).reshape(-1, words)
    return torch.where(t >= 1 << 31, t - (1 << 32), t).to(torch.int32)


def check(q, kc, vc, bt, lens, cu, tree=None, got=None, **kw):
    want, lse, mag, smax, done = R.tree_attention(q, kc, vc, bt, lens, cu, tree, **kw)
    sl = int32(lens)
    got, got_lse = got or draft.tree_attention(
        on_gpu(q), on_gpu(kc), on_gpu(vc), bt.cuda(), sl.cuda(), cu.cuda(),
        tree=None if tree is None else on_gpu(tree), return_lse=True, **kw)
    n = max([1, *lens])
    tol = attention_tolerance(q, want, mag, smax, n + 8, q.dtype)
    close(got[done.cuda()], want[done], tol[done], "out")
    tol = (q.shape[-1] + 16) * U * smax + (n + 64) * U + lse.abs().nan_to_num(0, 0, 0) * 4 * U
    close(got_lse[done.cuda()], lse[done], tol[done], "lse")
    return got


LENS = [0, 1, 15, 16, 33, 64, 129, 300, 700]
NEW = [0, 1, 4, 16, 3, 31, 32, 33, 7]


@pytest.mark.parametrize("dtype,cdtype", [(F32, F32), (F16, F16), (BF16, BF16), (F16, F8),
                                          (BF16, F8)])
@pytest.mark.parametrize("dim,kv,group,page,layout", [
    (64, 2, 4, 16, "token"), (128, 1, 1, 16, "token"), (128, 1, 8, 64, "head"),
    (80, 2, 3, 24, "token"), (256, 1, 2, 32, "token"), (16, 3, 2, 1, "token"),
    (192, 1, 5, 7, "head"), (96, 1, 17, 128, "token"),
])
@pytest.mark.parametrize("tree", [False, True])
def test_attention(dtype, cdtype, dim, kv, group, page, layout, tree):
    gen = torch.Generator().manual_seed(dim * 31 + group)
    bt, count = table_for(gen, LENS, page)
    kc, vc = (only_live(cache(gen, count, page, kv, dim, cdtype, layout), bt, LENS, page)
              for _ in "kv")
    q = rand(gen, sum(NEW), kv * group, dim, dtype=dtype)
    kw = dict(k_scale=0.5, v_scale=2.0) if cdtype is F8 else {}
    check(q, kc, vc, bt, LENS, starts_of(NEW), trees(gen, NEW, 2) if tree else None, **kw)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [8, 24, 104, 136, 248])
def test_attention_odd_head_dims(dtype, dim):
    gen = torch.Generator().manual_seed(dim)
    lens, new = [130, 9, 77], [5, 9, 18]
    bt, count = table_for(gen, lens, 16)
    kc, vc = (only_live(cache(gen, count, 16, 2, dim, dtype), bt, lens, 16) for _ in "kv")
    check(rand(gen, 32, 6, dim, dtype=dtype), kc, vc, bt, lens, starts_of(new),
          trees(gen, new, 1))


@pytest.mark.parametrize("dtype,cdtype", [(F32, F32), (BF16, BF16), (F16, F8)])
@pytest.mark.parametrize("window,softcap,scale", [
    (1, 0.0, None), (2, 0.0, 0.3), (7, 20.0, None), (40, 0.0, -0.2), (100, 0.0, None),
    (1000, 5.0, 1.0), (5000, 0.5, 0.01), (0, 50.0, 0.0)])
@pytest.mark.parametrize("tree", [False, True])
def test_attention_window_softcap_scale(dtype, cdtype, window, softcap, scale, tree):
    gen = torch.Generator().manual_seed(window)
    bt, count = table_for(gen, LENS, 16)
    kc, vc = (only_live(cache(gen, count, 16, 2, 64, cdtype), bt, LENS, 16) for _ in "kv")
    check(rand(gen, sum(NEW), 8, 64, dtype=dtype), kc, vc, bt, LENS, starts_of(NEW),
          trees(gen, NEW, 2, 0.1) if tree else None, window=window, softcap=softcap, scale=scale)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window", [0, 3])
def test_attention_of_rows_that_see_nothing(dtype, window):
    """No past, masks without a bit, more new tokens than the sequence is long, pages that are
    not there, no pages at all."""
    gen = torch.Generator().manual_seed(1)
    lens, new = [9, 3, 0, -4, 40], [9, 8, 5, 2, 6]
    bt, count = table_for(gen, lens, 8)
    bt[4, 2:5] = torch.tensor([-1, 2 ** 31 - 1, count])
    kc, vc = (cache(gen, count, 8, 1, 64, dtype) for _ in "kv")
    tree = trees(gen, new, 1, 0.4)
    q = rand(gen, sum(new), 3, 64, dtype=dtype)
    for t in (tree, None):
        got = check(q, kc, vc, bt, lens, starts_of(new), t, window=window)
        assert (got[9 + 8:9 + 8 + 7] == 0).all()
    empty = torch.zeros(0, 8, 1, 64, dtype=dtype)
    assert (check(q, empty, empty, bt, lens, starts_of(new), tree) == 0).all()


@pytest.mark.parametrize("dtype,cdtype", [(F32, F32), (F16, F16), (BF16, F8)])
@pytest.mark.parametrize("window", [0, 1, 4, 20, 31, 700])
@pytest.mark.parametrize("width", [4, 200])
@pytest.mark.parametrize("tree", [False, True])
def test_attention_of_lengths_beyond_the_table(dtype, cdtype, window, width, tree):
    """Tokens behind the table are absent: a window is of the last ones that are in it. Some, all
    and none of the new ones are."""
    gen = torch.Generator().manual_seed(window + width)
    page, group = 8, 4
    end = width * page
    lens = [end + 8, end + 1, end, end + 68, 2 ** 31 - 1, end - 12, end + 2, 2 * end]
    new = [1, 5, 4, 70, 7, 3, 33, 2]
    bt = torch.randperm(len(lens) * width, generator=gen).to(torch.int32).reshape(-1, width)
    kc, vc = (cache(gen, bt.numel(), page, 1, 64, cdtype) for _ in "kv")
    q = rand(gen, sum(new), group, 64, dtype=dtype)
    mask, cu = trees(gen, new, 3, 0.1) if tree else None, starts_of(new)
    want, lse, mag, smax, _ = R.tree_attention(q, kc, vc, bt, lens, cu, mask, window=window)
    got, got_lse = draft.tree_attention(
        *(x.cuda() for x in (q, kc, vc, bt, int32(lens), cu)),
        tree=None if mask is None else mask.cuda(), window=window, return_lse=True)
    close(got, want, attention_tolerance(q, want, mag, smax, end + 8, dtype), "out")
    close(got_lse, lse, (64 + 16) * U * smax + (end + 64) * U +
          lse.abs().nan_to_num(0, 0, 0) * 4 * U, "lse")


@pytest.mark.parametrize("dtype,cdtype", [(F32, F32), (F16, F16), (BF16, BF16), (BF16, F8)])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("tree,window", [(True, 0), (False, 0), (False, 6), (True, 6)])
def test_attention_values_that_are_not_finite_reach_only_what_sees_them(dtype, cdtype, value,
                                                                        tree, window):
    if cdtype is F8 and not math.isnan(value):
        pytest.skip("e4m3 has no infinities")
    gen = torch.Generator().manual_seed(3)
    lens, new, dim = [70, 33, 20], [13, 33, 9], 64
    bt, count = table_for(gen, lens, 16)
    kc, vc = (cache(gen, count, 16, 2, dim, cdtype) for _ in "kv")
    mask = trees(gen, new, 2) if tree else None
    q = rand(gen, sum(new), 8, dim, dtype=dtype)
    cu = starts_of(new)
    want, lse, mag, smax, _ = R.tree_attention(q, kc, vc, bt, lens, cu, mask, window=window)
    hit = torch.zeros(want.shape, dtype=torch.bool)
    bad = vc.float()
    for b, j, g, d in ((0, 5, 0, 7), (0, 9, 1, 63), (1, 0, 0, 0), (1, 20, 1, 33), (2, -3, 0, 9)):
        at = lens[b] - new[b] + j                          # -3: in the past
        bad[int(bt[b, at // 16]), at % 16, g, d] = value
        for i in range(new[b]):
            row = int(cu[b]) + i
            see = R.seen_by(mask, row, i, new[b])
            line = [1] * (lens[b] - new[b]) + see.int().tolist()
            if line[at] and (not window or sum(line[at:]) <= window):
                hit[row, g * 4:g * 4 + 4, d] = True
    got = draft.tree_attention(q.cuda(), kc.cuda(), bad.to(cdtype).cuda(), bt.cuda(),
                               int32(lens).cuda(), cu.cuda(),
                               tree=None if mask is None else mask.cuda(), window=window)
    assert hit.any() and not torch.isfinite(got[hit.cuda()]).any()
    tol = attention_tolerance(q, want, mag, smax, 100, dtype)
    close(got[~hit.cuda()], want[~hit], tol[~hit])


def deep_trees(gen, new, words):
    """Masks of trees whose nodes follow one of the three before them: paths of hundreds."""
    rows = []
    for n in new:
        masks = []
        for j in range(n):
            up = j - 1 - int(torch.randint(0, min(3, j), (1,), generator=gen)) if j else None
            masks.append(1 << j | (masks[up] if j else 0))
        rows += [[m >> 32 * w & 0xFFFFFFFF for w in range(words)] for m in masks]
    t = torch.tensor(rows, dtype=torch.int64)
    return torch.where(t >= 1 << 31, t - (1 << 32), t).to(torch.int32)


@pytest.mark.parametrize("dtype,cdtype", [(F32, F32), (BF16, BF16), (F16, F8)])
@pytest.mark.parametrize("window", [2, 7, 50, 150, 330])
@pytest.mark.parametrize("make", [trees, deep_trees])
def test_attention_windows_of_masks_of_many_words(dtype, cdtype, window, make):
    """Windows that end among the new tokens, before them, and at the borders of a mask's words;
    lengths with and without a past, and beyond the table; masks that end before the tokens do."""
    gen = torch.Generator().manual_seed(window)
    lens, new = [350, 130, 95, 420], [300, 130, 96, 97]
    bt, count = table_for(gen, lens, 16)
    bt = bt[:, :25]                                        # 400 tokens
    kc, vc = (only_live(cache(gen, count, 16, 1, 64, cdtype), bt, lens, 16) for _ in "kv")
    q = rand(gen, sum(new), 2, 64, dtype=dtype)
    tree = make(gen, new, 10)
    check(q, kc, vc, bt, lens, starts_of(new), tree, window=window)
    check(q, kc, vc, bt, lens, starts_of(new), tree[:, :3].contiguous(), window=window)


@pytest.mark.parametrize("dtype,cdtype", [(F32, F32), (BF16, BF16), (F16, F8)])
@pytest.mark.parametrize("window", [0, 5, 64, 200])
@pytest.mark.parametrize("make", [trees, deep_trees])
def test_attention_values_not_finite_under_masks_of_many_words(dtype, cdtype, window, make):
    gen = torch.Generator().manual_seed(window + 1)
    lens, new, dim = [320, 150], [230, 150], 64
    bt, count = table_for(gen, lens, 16)
    kc, vc = (cache(gen, count, 16, 1, dim, cdtype) for _ in "kv")
    mask, cu = make(gen, new, 8), starts_of(new)
    q = rand(gen, sum(new), 2, dim, dtype=dtype)
    want, _, mag, smax, _ = R.tree_attention(q, kc, vc, bt, lens, cu, mask, window=window)
    hit = torch.zeros(want.shape, dtype=torch.bool)
    bad = vc.float()
    for b, j, d in ((0, -40, 3), (0, 64, 7), (0, 95, 8), (0, 170, 63), (0, 229, 31), (1, 0, 1),
                    (1, 63, 40), (1, 128, 5)):
        at = lens[b] - new[b] + j
        bad[int(bt[b, at // 16]), at % 16, 0, d] = math.nan
        for i in range(new[b]):
            row = int(cu[b]) + i
            line = [1] * (lens[b] - new[b]) + R.seen_by(mask, row, i, new[b]).int().tolist()
            if line[at] and (not window or sum(line[at:]) <= window):
                hit[row, :, d] = True
    got = draft.tree_attention(*(x.cuda() for x in (q, kc, bad.to(cdtype), bt, int32(lens), cu)),
                               tree=mask.cuda(), window=window)
    assert hit.any() and torch.isnan(got[hit.cuda()]).all()
    tol = attention_tolerance(q, want, mag, smax, 330, dtype)
    close(got[~hit.cuda()], want[~hit], tol[~hit])


def test_attention_keys_that_are_not_finite():
    """In masked places they count for nothing; elsewhere the token that sees them is NaN."""
    gen = torch.Generator().manual_seed(4)
    lens, new = [50], [6]
    bt, count = table_for(gen, lens, 16)
    kc, vc = (cache(gen, count, 16, 1, 64, F32) for _ in "kv")
    kc[int(bt[0, 46 // 16]), 46 % 16, 0, 5] = math.nan        # new token 2
    tree = int32([[1], [3], [7], [11], [17], [35]])
    q = rand(gen, 6, 2, 64)
    got = check(q, kc, vc, bt, lens, starts_of(new), tree)
    assert torch.isnan(got[2]).all() and torch.isfinite(got[[0, 1, 3, 4, 5]]).all()


@pytest.mark.parametrize("scale", [1e5, -3e7])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_attention_of_large_scores(scale, dtype):
    """However large the scores are, the largest has its weight."""
    gen = torch.Generator().manual_seed(5)
    lens, new = [100], [4]
    bt, count = table_for(gen, lens, 16)
    kc, vc = (cache(gen, count, 16, 1, 64, dtype) for _ in "kv")
    q = rand(gen, 4, 2, 64, dtype=dtype)
    got = draft.tree_attention(q.cuda(), kc.cuda(), vc.cuda(), bt.cuda(), int32(lens).cuda(),
                               starts_of(new).cuda(), scale=scale)
    at = torch.arange(100)
    k, v = (x[bt[0].long()[at // 16], at % 16, 0].double() for x in (kc, vc))
    for i in range(4):
        x = q[i].double() @ k[:97 + i].T * scale
        close(got[i].cpu(), v[x.argmax(-1)].to(dtype).double(), torch.zeros(2, 64).double())


@pytest.mark.parametrize("dtype,cdtype", [(F32, F32), (F16, F16), (BF16, BF16), (F16, F8),
                                          (BF16, F8)])
@pytest.mark.parametrize("dim", [16, 128, 256])
@pytest.mark.parametrize("new", [1, 5, 12, 30])
def test_attention_weights_keep_32_bits(dtype, cdtype, dim, new):
    """Two nearly equal weights w1, w2 of 0.37 to 0.61 whose values are 1 and -1, beside a weight
    of 1 whose value is 0: the result, (w1 - w2) / (1 + w1 + w2), is about 2^-16, so that it shows
    the weights' errors of 2^-24 and not its own rounding.

    In units of U = 2^-24: the scores are exact; their product with the scale, and that one's
    own rounding, put 2 U of up to 0.73 into the exponent, exp2 is off by at most 2 U of the
    weight: 0.61 (0.73 * 2 + 2) = 2.2 U for each weight, 4.4 U for both. fp16's terms have 14 added
    to the exponent, which rounds it by 2^-21, 5.6 U of the weight, and add 2^-22 = 4 U of it: 11.7
    U for both. The two products' sums are below 1, their terms (up to 6) are added with 1 U each
    or, if the matrix unit cuts off, 2 U: 12 U. All that is divided by 1 + w1 + w2 >= 1.73: 9.5 U,
    and 16.3 U in fp16. Errors of the divisor count by the result, 2^-16."""
    gen = torch.Generator().manual_seed(dim + new)
    batch, group = 8, 4
    kc, vc = (torch.zeros(1, 64, 1, dim) for _ in "kv")
    kc[0, 1, 0, 0] = kc[0, 2, 0, 0] = kc[0, 2, 0, 1] = 1.0
    vc[0, 1], vc[0, 2] = 1.0, -1.0
    kc, vc = kc.to(cdtype), vc.to(cdtype)
    q = torch.zeros(batch * new, group, dim)
    q[..., 0] = -torch.rand(batch * new, group, generator=gen) / 2 - 0.5
    q[..., 1] = -torch.rand(batch * new, group, generator=gen) * 2.0 ** -14
    q = q.to(dtype)
    bt, lens = torch.zeros(batch, 1, dtype=torch.int32), [3 + new] * batch
    cu, tree = starts_of([new] * batch), torch.zeros(batch * new, 1, dtype=torch.int32)
    want, _, _, _, _ = R.tree_attention(q, kc, vc, bt, lens, cu, tree, scale=1.0)
    got = draft.tree_attention(q.cuda(), kc.cuda(), vc.cuda(), bt.cuda(), int32(lens).cuda(),
                               cu.cuda(), tree=tree.cuda(), scale=1.0)
    units = 16.3 if F16 in (dtype, cdtype) or cdtype is F8 else 9.5
    close(got, want, half_step(dtype) * want.abs() + units * U, "out")


@pytest.mark.parametrize("batch", [1, 63, 64, 65, 200])
def test_attention_of_many_sequences(batch):
    gen = torch.Generator().manual_seed(batch)
    lens = torch.randint(0, 200, (batch,), generator=gen).tolist()
    new = torch.randint(0, 6, (batch,), generator=gen).tolist()
    lens[::5] = [0] * len(lens[::5])
    new[1::4] = [0] * len(new[1::4])
    bt, count = table_for(gen, lens, 16)
    kc, vc = (only_live(cache(gen, count, 16, 1, 64, BF16), bt, lens, 16) for _ in "kv")
    check(rand(gen, sum(new), 2, 64, dtype=BF16), kc, vc, bt, lens, starts_of(new),
          trees(gen, new, 1))


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (F16, 200), (F32, 96)])
@pytest.mark.parametrize("batch,kv_heads,group", [(24, 50, 3), (40, 51, 1), (70, 33, 2)])
def test_attention_of_more_sequences_than_fit_at_once(batch, kv_heads, group, dtype, dim):
    """Few workgroups for each key head: sequences are split for two rounds of them, and the parts
    joined by waves of four heads, whose last one has fewer."""
    gen = torch.Generator().manual_seed(batch)
    lens = torch.randint(0, 1500, (batch,), generator=gen).tolist()
    new = [min(n, 1 + i % 4) for i, n in enumerate(lens)]
    bt, count = table_for(gen, lens, 32)
    kc, vc = (only_live(cache(gen, count, 32, kv_heads, dim, dtype), bt, lens, 32) for _ in "kv")
    check(rand(gen, sum(new), kv_heads * group, dim, dtype=dtype), kc, vc, bt, lens,
          starts_of(new), trees(gen, new, 1))


@pytest.mark.parametrize("batch,kv_heads", [(2, 1), (33, 16), (64, 40), (64, 300)])
def test_attention_of_one_long_among_many(batch, kv_heads):
    """Even shares, shares of whole rounds and shares of all of a sequence."""
    gen = torch.Generator().manual_seed(kv_heads)
    lens = [2000] + torch.randint(0, 70, (batch - 1,), generator=gen).tolist()
    lens[1::7] = [0] * len(lens[1::7])
    new = [min(n, 1 + i % 3) for i, n in enumerate(lens)]
    bt, count = table_for(gen, lens, 16)
    kc, vc = (only_live(cache(gen, count, 16, kv_heads, 32, F16), bt, lens, 16) for _ in "kv")
    q = rand(gen, sum(new), kv_heads, 32, dtype=F16)
    check(q, kc, vc, bt, lens, starts_of(new))
    check(q, kc, vc, bt, lens, starts_of(new), window=1500)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("group", [1, 4, 7])
def test_attention_of_prompts(dtype, group):
    """Chains of many tokens, some without a past; a tree as long."""
    gen = torch.Generator().manual_seed(group)
    lens, new = [300, 257, 140], [300, 130, 1]
    bt, count = table_for(gen, lens, 16)
    kc, vc = (only_live(cache(gen, count, 16, 1, 64, dtype), bt, lens, 16) for _ in "kv")
    q = rand(gen, sum(new), group, 64, dtype=dtype)
    check(q, kc, vc, bt, lens, starts_of(new))
    check(q, kc, vc, bt, lens, starts_of(new), window=50)
    check(q, kc, vc, bt, lens, starts_of(new), trees(gen, new, 10))
    one = [300], starts_of(new[:1])
    check(q[:300], kc, vc, bt[:1], *one)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("new", [1, 5, 40])
def test_attention_of_a_long_sequence_is_split_and_joined(dtype, new):
    gen = torch.Generator().manual_seed(6)
    lens, news = [20001, 60], [new, 12]
    bt, count = table_for(gen, lens, 128)
    kc, vc = (cache(gen, count, 128, 1, 64, dtype) for _ in "kv")
    q = rand(gen, new + 12, 3, 64, dtype=dtype)
    tree = trees(gen, news, 2)
    a = check(q, kc, vc, bt, lens, starts_of(news), tree)
    assert torch.equal(a, check(q, kc, vc, bt, lens, starts_of(news), tree))  # the same bits


def test_attention_of_one_token_is_that_of_a_decoding_step():
    gen = torch.Generator().manual_seed(7)
    lens = [1, 40, 333]
    bt, count = table_for(gen, lens, 16)
    kc, vc = (cache(gen, count, 16, 2, 128, F16) for _ in "kv")
    q = rand(gen, 3, 8, 128, dtype=F16)
    args = [x.cuda() for x in (q, kc, vc, bt, int32(lens))]
    a = decode.paged_attention(*args, window=30)
    b = draft.tree_attention(*args, torch.arange(4, dtype=torch.int32).cuda(), window=30)
    assert (a.double() - b.double()).norm() <= 2.0 ** -11 * a.double().norm()


def test_attention_strides_places_and_padding():
    """Queries out of a fused projection, tables, lengths, starts and masks of larger arrays,
    caches inside one array, results into rows of another; rows of no sequence stay."""
    gen = torch.Generator().manual_seed(8)
    lens, new, page, kv, heads, dim = [70, 0, 333], [5, 0, 20], 16, 2, 6, 128
    before, behind = 3, 4
    rows = before + sum(new) + behind
    bt, count = table_for(gen, lens, page)
    both = rand(gen, count, 2, page, kv, dim + 8, dtype=F16).cuda()
    kc, vc = both[:, 0, ..., 3:3 + dim], both[:, 1, ..., 3:3 + dim]
    q = rand(gen, rows, heads + 4, dim, dtype=F16).cuda()[:, 1:1 + heads]
    wide = torch.zeros(3, 40, dtype=torch.int32).cuda()
    wide[:, 5:5 + bt.shape[1]] = bt.cuda()
    lens3 = torch.zeros(3, 4, dtype=torch.int32).cuda()
    lens3[:, 2] = torch.tensor(lens).cuda()
    cu = starts_of(new, before)
    cu2 = torch.stack((cu, cu + 99), 1).cuda()[:, 0]
    tree = torch.zeros(rows, 3, dtype=torch.int32)
    tree[before:before + sum(new), 1:2] = trees(gen, new, 1)
    room = torch.full((rows, heads, dim + 1), 7.0, dtype=F16).cuda()
    out = room[..., :dim]
    args = kc, vc, wide[:, 5:5 + bt.shape[1]], lens3[:, 2], cu2
    got = draft.tree_attention(q, *args, tree=tree.cuda()[:, 1:2], out=out, return_lse=True)
    assert got[0].data_ptr() == out.data_ptr()
    check(q.cpu(), kc.cpu(), vc.cpu(), bt, lens, cu, tree[:, 1:2], got=got)
    assert (room[..., dim] == 7).all()
    assert (room[:before] == 7).all() and (room[-behind:] == 7).all()
    keep = out[before:-behind].clone()
    assert draft.tree_attention(q, *args, tree=tree.cuda()[:, 1:2], out=q).data_ptr() == \
        q.data_ptr()
    assert torch.equal(q[before:-behind], keep)


@pytest.mark.parametrize("length", [500, 1999])
@pytest.mark.parametrize("batch", [1, 3])
def test_attention_workspace_goes_by_the_call(length, batch):
    """No more room for partial results than the sequences have units of 64 tokens."""
    gen = torch.Generator().manual_seed(length)
    kv, group, dim, n = 8, 4, 128, 16
    bt, count = table_for(gen, [length] * batch, 16)
    kc, vc = (cache(gen, count, 16, kv, dim, BF16).cuda() for _ in "kv")
    q = rand(gen, batch * n, kv * group, dim, dtype=BF16).cuda()
    args = [q, kc, vc, bt.cuda(), int32([length] * batch).cuda(), starts_of([n] * batch).cuda()]
    out = draft.tree_attention(*args)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    draft.tree_attention(*args, out=out)
    most = batch * -(-length // 64) * kv * n * group * (dim + 2) * 4 + 16 * batch * n
    blocks = 2 if batch > 1 else 1                         # the host knows the sum of the rows
    assert torch.cuda.max_memory_allocated() - before <= blocks * most + 1024


def test_attention_padded_rows_of_one_long_sequence():
    """Few tokens in rows for many: the split goes by the tokens."""
    gen = torch.Generator().manual_seed(9)
    bt, count = table_for(gen, [5000], 16)
    kc, vc = (cache(gen, count, 16, 1, 64, BF16) for _ in "kv")
    for rows in (3, 40, 3000):
        q = rand(gen, rows, 4, 64, dtype=BF16)
        check(q, kc, vc, bt, [5000], int32([0, 3]))


def test_attention_rows_that_descend_stay_inside():
    """`cu_tokens` that break their rule leave the result open, and nothing else."""
    gen = torch.Generator().manual_seed(10)
    lens = [100, 3000, 50, 70]
    bt, count = table_for(gen, lens, 16)
    kc, vc = (cache(gen, count, 16, 1, 64, BF16).cuda() for _ in "kv")
    for cu in ([0, 8, 2, 9, 12], [5, -3, 2 ** 31 - 1, -2 ** 31, 12], [12, 9, 6, 3, 0]):
        out = torch.full((12 + 2, 2, 64), 5.0, dtype=BF16).cuda()
        draft.tree_attention(rand(gen, 12, 2, 64, dtype=BF16).cuda(), kc, vc, bt.cuda(),
                             int32(lens).cuda(), int32(cu).cuda(), out=out[1:13])
        assert (out[[0, -1]] == 5).all()


def test_attention_far_into_a_cache_beyond_32_bit_offsets():
    page, kv, dim = 64, 8, 128
    count = (1 << 32) // (page * kv * dim) + 40            # 2^32 elements, 4 GiB of e4m3
    gen = torch.Generator().manual_seed(4)
    lens, new = [300, 1000], [6, 9]
    bt = torch.stack([torch.randperm(20, generator=gen)[:16] + count - 40 + 20 * b
                      for b in range(2)]).to(torch.int32)
    bt[:, ::2] -= count - 40                               # near and far in turn
    kc, vc = (torch.zeros(count, page, kv, dim, dtype=torch.uint8, device="cuda").view(F8)
              for _ in "kv")
    small = [rand(gen, 80, page, kv, dim).to(F8) for _ in "kv"]    # the first and last 40 pages
    ids = torch.cat([torch.arange(40), torch.arange(count - 40, count)])
    for c, s in zip((kc, vc), small):
        c.view(torch.uint8)[ids.cuda()] = s.view(torch.uint8).cuda()
    back = torch.where(bt >= 40, bt - (count - 80), bt)
    q = rand(gen, 15, 16, dim, dtype=BF16)
    tree = trees(gen, new, 1)
    got = draft.tree_attention(q.cuda(), kc, vc, bt.cuda(), int32(lens).cuda(),
                               starts_of(new).cuda(), tree=tree.cuda(), return_lse=True)
    check(q, small[0], small[1], back, lens, starts_of(new), tree, got=got)


# -- appending by positions -------------------------------------------------------------------

def append_case(gen, dtype, cdtype, lens, new, page, kv, heads, dim, rotary, axes, layout="token"):
    bt, count = table_for(gen, lens, page)
    tokens, most = sum(new), 200
    d = dict(k=rand(gen, tokens, kv, dim, dtype=dtype), v=rand(gen, tokens, kv, dim, dtype=dtype),
             k_cache=cache(gen, count, page, kv, dim, cdtype, layout),
             v_cache=cache(gen, count, page, kv, dim, cdtype, layout), block_table=bt,
             seq_lens=int32(lens), cu_tokens=starts_of(new),
             q=rand(gen, tokens, heads, dim, dtype=dtype))
    angle = torch.arange(most).double()[:, None] * \
        10000.0 ** (-2 * torch.arange(rotary // 2).double() / rotary)
    d["cos"], d["sin"] = angle.cos().float(), angle.sin().float()
    d["positions"] = torch.randint(0, most, (axes, tokens), generator=gen, dtype=torch.int32)
    return d


def check_append(d, **kw):
    names = ("k", "v", "k_cache", "v_cache", "block_table", "seq_lens")
    q_out = torch.full(d["q"].shape, 3.0).to(d["q"].dtype)
    g = {n: on_gpu(x) for n, x in d.items()}
    want_q, want_k, want_v, done = R.append_kv(*(d[n] for n in names), q_out=q_out,
                                               **{n: d[n] for n in d if n not in names}, **kw)
    got = decode.append_kv(*(g[n] for n in names), q_out=q_out.cuda(),
                           **{n: g[n] for n in g if n not in names}, **kw)

    def tol(x, want, scale=1.0):
        # two products and a sum of 32 bits, a division and the rounding
        top = x.double().abs().max() / scale
        return half_step(want.dtype) * want.double().abs() + 8 * U * top + SUB[want.dtype]

    dt, ct = d["q"].dtype, d["k_cache"].dtype
    close(got, want_q, tol(d["q"], want_q.to(dt)), "q")
    for name, want in (("k", want_k), ("v", want_v)):
        c = g[name + "_cache"].cpu()
        assert torch.equal(c[~done].float(), d[name + "_cache"][~done].float())
        near = half_step(ct) * want.abs() + 8 * U * d[name].double().abs().max() / \
            kw.get(name + "_scale", 1.0) + SUB[ct]
        # a value next to a border of the type may go to either side of it
        close(c[done].double(), want[done], near[done] + 2 * 8 * U * want[done].abs(), name)


@pytest.mark.parametrize("dtype,cdtype", [(F32, F32), (F16, F16), (BF16, BF16), (BF16, F8)])
@pytest.mark.parametrize("dim,rotary,axes,layout", [
    (64, 64, "0" * 32, "token"), (128, 128, "0" * 16 + "1" * 24 + "2" * 24, "token"),
    (128, 128, "012" * 21 + "0", "head"), (80, 48, "3" * 8 + "1" * 8 + "0" * 8, "token"),
    (256, 256, "0" * 60 + "2" * 34 + "1" * 34, "token"), (64, 16, "01010101", "token"),
    (96, 6, "201", "token"),
])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_by_positions(dtype, cdtype, dim, rotary, axes, layout, interleaved):
    gen = torch.Generator().manual_seed(dim + rotary)
    axes = tuple(map(int, axes))
    d = append_case(gen, dtype, cdtype, [40, 7, 130, 0], [17, 7, 40, 0], 16, 2, 5, dim, rotary,
                    max(axes) + 1, layout)
    kw = dict(k_scale=0.25, v_scale=0.5) if cdtype is F8 else {}
    check_append(d, pair_axes=axes, interleaved=interleaved, **kw)


def test_append_positions_that_are_not_in_the_tables():
    """Rows with such a position on any axis are skipped; lengths do not matter for the others."""
    gen = torch.Generator().manual_seed(2)
    d = append_case(gen, F16, F16, [400, 30], [9, 8], 16, 1, 2, 64, 64, 3)
    p = d["positions"]
    p[0, 1], p[1, 3], p[2, 5], p[0, 7], p[2, 16] = 200, -1, 2 ** 31 - 1, -2 ** 31, 199
    check_append(d, pair_axes=(0, 1, 2, 1) * 8)
    d["positions"] = p[0]
    check_append(d)
    check_append(d | {"positions": p.t().contiguous().t()}, pair_axes=(1, 0) * 16)


def test_append_positions_of_slots_are_those_of_none():
    """Positions that are the slots' own turn as without them, bit for bit."""
    gen = torch.Generator().manual_seed(3)
    lens, new = [40, 7, 130], [17, 7, 40]
    for dtype, dim, rotary, inter in ((BF16, 128, 128, False), (F16, 80, 48, True)):
        d = append_case(gen, dtype, dtype, lens, new, 16, 2, 4, dim, rotary, 1)
        own = int32([n - m + i for n, m in zip(lens, new) for i in range(m)])
        runs = []
        for p in (None, own.cuda(), own.cuda()[None]):
            g = {n: on_gpu(x) for n, x in d.items() if n != "positions"}
            q = decode.append_kv(**g, positions=p, interleaved=inter)
            runs.append((q, g["k_cache"], g["v_cache"]))
        for x in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(x, runs[0]))


# -- acceptance -------------------------------------------------------------------------------

def draft_case(gen, new, vocab, words, dtype, tree, hit=0.8):
    logits = rand(gen, sum(new), vocab).to(dtype)
    cu = starts_of(new)
    mask = trees(gen, new, words) if tree else None
    tokens = torch.randint(0, vocab, (sum(new),), generator=gen, dtype=torch.int32)
    for first, n in R.spans(cu, sum(new)):
        for j in range(1, n):
            if float(torch.rand(1, generator=gen)) < hit:
                see = R.seen_by(mask, first + j, j, n)
                parent = int(torch.nonzero(see)[-2]) if tree else j - 1
                tokens[first + j] = int(logits[first + parent].float().argmax())
    return logits, tokens, cu, mask


def check_accept(logits, tokens, cu, tree, most=None):
    want = R.accept(logits, tokens, cu, tree, most)
    got = draft.accept(on_gpu(logits), on_gpu(tokens), cu.cuda(),
                       tree=None if tree is None else on_gpu(tree), most=most)
    for name, a, b in zip(("path", "count", "token"), got, want):
        assert torch.equal(a.cpu(), b), (name, a, b)
    return want


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [1, 7, 1000, 4096, 32001, 70003])
@pytest.mark.parametrize("tree", [False, True])
def test_accept(dtype, vocab, tree):
    gen = torch.Generator().manual_seed(vocab)
    new = [1, 0, 13, 33, 4, 8]
    got = check_accept(*draft_case(gen, new, vocab, 2, dtype, tree))
    assert got[1].max() > 2


@pytest.mark.parametrize("tree", [False, True])
def test_accept_long_drafts_and_short_paths(tree):
    gen = torch.Generator().manual_seed(1)
    new = [600, 300, 2, 256, 257]
    case = draft_case(gen, new, 50, 19, F32, tree, hit=0.995)
    got = check_accept(*case)
    assert tree or got[1].max() > 20
    for most in (0, 1, 2, 7):
        check_accept(*case, most=most)


def test_accept_of_all_of_a_chain():
    gen = torch.Generator().manual_seed(2)
    got = check_accept(*draft_case(gen, [700, 256, 257], 50, 1, BF16, False, hit=1.0))
    assert got[1].tolist() == [700, 256, 257]


def test_accept_ties_infinities_and_nan():
    logits = torch.full((6, 9000), -math.inf)
    logits[1, [70, 8999]] = 3.0
    logits[2, [5000, 100]] = torch.tensor([math.nan, math.inf])
    logits[3, :] = 0.0
    logits[3, :4500] = -0.0
    logits[4, 8191:8193] = 65504.0
    logits[5, [3, 4]] = torch.tensor([-math.nan, math.nan])
    for dtype in (F32, F16, BF16):
        x = logits.to(dtype)
        tokens = int32([9, 0, 70, 5000, 0, 8191])      # each row's choice after the one before
        got = check_accept(x, tokens, int32([0, 6]), None)
        assert got[1].tolist() == [6] and got[2].tolist() == [3]


def test_accept_takes_the_first_of_twins_and_stops_between():
    """Children with one token, children out of order, a grandchild with the token alone."""
    logits = torch.zeros(6, 20)
    for i, t in enumerate((5, 6, 7, 8, 9, 10)):
        logits[i, t] = 1.0
    tree = int32([[1], [3], [5], [1 + 4 + 8], [1 + 2 + 16], [1 + 4 + 8 + 32]])
    tokens = int32([0, 5, 5, 7, 6, 8])
    got = check_accept(logits, tokens, int32([0, 6]), tree)
    assert got[0][0, :3].tolist() == [0, 1, 4]         # node 2 has the token as well
    tokens = int32([0, 4, 5, 7, 6, 8])
    assert check_accept(logits, tokens, int32([0, 6]), tree)[0][0, :4].tolist() == [0, 2, 3, 5]
    tokens = int32([0, 4, 4, 5, 5, 5])
    assert check_accept(logits, tokens, int32([0, 6]), tree)[1].tolist() == [1]


def test_accept_strides_padding_and_wild_rows():
    gen = torch.Generator().manual_seed(3)
    logits, tokens, cu, tree = draft_case(gen, [4, 7, 0, 5], 3001, 1, F16, True)
    wide = torch.zeros(20, 3100, dtype=F16)
    wide[3:19, 7:3008] = logits
    tok2 = torch.zeros(20, 3, dtype=torch.int32)
    tok2[3:19, 1] = tokens
    tree2 = torch.zeros(20, 4, dtype=torch.int32)
    tree2[3:19, 2:3] = tree
    check_accept(wide[:, 7:3008], tok2[:, 1], cu + 3, tree2[:, 2:3])
    for cu in ([0, 8, 2, 9, 12], [5, -3, 2 ** 31 - 1, -2 ** 31, 12], [16, 9, 6, 3, 0]):
        check_accept(logits, tokens, int32(cu), tree)
        check_accept(logits, tokens, int32(cu), None)


# -- as a program uses them -------------------------------------------------------------------

class Model:
    """A small causal model over a paged cache, of one layer: what it says next depends on all
    that came before."""

    def __init__(self, seed, kv=2, heads=4, dim=64, vocab=211, most=300):
        gen = torch.Generator().manual_seed(seed)
        self.kv, self.heads, self.dim, self.vocab = kv, heads, dim, vocab
        self.embed = rand(gen, vocab, (heads + 2 * kv) * dim, scale=0.7).cuda()
        self.head = rand(gen, heads * dim, vocab, scale=0.3).cuda()
        at = torch.arange(most).double()[:, None] * \
            10000.0 ** (-2 * torch.arange(dim // 2).double() / dim)
        self.cos, self.sin = at.cos().float().cuda(), at.sin().float().cuda()

    def project(self, tokens):
        x = self.embed[tokens.long()].view(-1, self.heads + 2 * self.kv, self.dim)
        return x.split([self.heads, self.kv, self.kv], 1)

    def logits(self, o):
        return o.flatten(1) @ self.head

    def plain(self, text, count):
        """`count` more tokens, from whole sequences in 64 bits on the CPU, and the smallest lead
        of a choice."""
        text, lead = list(text), math.inf
        embed, head = self.embed.cpu().double(), self.head.cpu().double()
        cos, sin = self.cos.cpu(), self.sin.cpu()
        for _ in range(count):
            x = embed[torch.tensor(text)].view(len(text), -1, self.dim)
            q, k, v = x.split([self.heads, self.kv, self.kv], 1)
            n = len(text)
            qn = R.rotate(q[-1], cos[n - 1], sin[n - 1], False)
            ks = torch.stack([R.rotate(k[i], cos[i], sin[i], False) for i in range(n)])
            o = torch.zeros(self.heads, self.dim, dtype=torch.float64)
            for h in range(self.heads):
                g = h * self.kv // self.heads
                p = torch.softmax(ks[:, g] @ qn[h] / math.sqrt(self.dim), 0)
                o[h] = p @ v[:, g]
            y = o.flatten() @ head
            top = y.topk(2).values
            lead = min(lead, float(top[0] - top[1]))
            text.append(int(y.argmax()))
        return text, lead


def serve(model, prompts, want, steps, gen, capture=False):
    """Drafted decoding: each step checks a tree of guesses, some of them right. Returns what was
    written for each prompt and how many steps went further than one token."""
    batch, page, width = len(prompts), 8, 40
    pool = batch * width
    caches = [torch.zeros(pool, page, model.kv, model.dim, device="cuda") for _ in "kv"]
    refs = torch.zeros(pool, dtype=torch.int32, device="cuda")
    refs[::7] = -1                                     # not to be taken
    table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    past = torch.zeros(batch, dtype=torch.int32, device="cuda")      # before the new tokens
    lens = past.clone()

    def forward(tokens, cu, n, tree, positions):
        grown = past + n
        served = pages.take(refs, table, lens, grown, page_size=page)
        q, k, v = model.project(tokens)
        q = decode.append_kv(k, v, *caches, table, lens, cu_tokens=cu, q=q, cos=model.cos,
                             sin=model.sin, positions=positions)
        o = draft.tree_attention(q, *caches, table, lens, cu, tree=tree)
        return served, model.logits(o)

    # the prompts, but for their last token
    new = [len(p) - 1 for p in prompts]
    tokens = int32([t for p in prompts for t in p[:-1]]).cuda()
    own = int32([i for n in new for i in range(n)]).cuda()
    served, _ = forward(tokens, starts_of(new).cuda(), int32(new).cuda(), None, own)
    assert served.tolist() == [1] * batch
    past.copy_(lens)
    texts = [list(p) for p in prompts]
    nodes = 7
    tree = int32([[1], [3], [5], [9], [5 + 16], [9 + 32], [5 + 16 + 64]]).cuda()
    depth = int32([0, 1, 1, 1, 2, 2, 3]).cuda()
    parent = [0, 0, 0, 0, 2, 3, 4]
    drafted = torch.zeros(batch * nodes, dtype=torch.int32, device="cuda")
    cu = starts_of([nodes] * batch).cuda()
    count7 = torch.full((batch,), nodes, dtype=torch.int32, device="cuda")
    masks = tree.repeat(batch, 1)

    def step():
        positions = (past[:, None] + depth).flatten()
        served, logits = forward(drafted, cu, count7, masks, positions)
        path, count, token = draft.accept(logits, drafted, cu, tree=masks, most=4)
        pages.compact(caches, table, past, path, count, seq_lens=lens)
        pages.free(refs, table, past.copy_(past + nodes), lens, page_size=page)
        return served, path, count, token

    graph = out = None
    further = 0
    for s in range(steps):
        # guesses: the right continuation on one branch, as far as some place
        guess = []
        for b in range(batch):
            right = want[b][len(texts[b]) - 1:]
            line = [texts[b][-1]] + torch.randint(0, model.vocab, (6,), generator=gen).tolist()
            good = [(), (1,), (2,), (2, 4), (2, 4, 6), (3, 5)][(s + b) % 6]
            for d, j in enumerate(good):
                if d + 1 < len(right):
                    line[j] = right[d + 1]
            guess += line
        drafted.copy_(int32(guess))
        if capture and s == 2:
            graph = torch.cuda.CUDAGraph()
            state = [x.clone() for x in (*caches, refs, table, past, lens)]
            with torch.cuda.graph(graph):
                out = step()
            for x, y in zip((*caches, refs, table, past, lens), state):
                x.copy_(y)
        if graph is not None:
            graph.replay()
            served, path, count, token = out
        else:
            served, path, count, token = step()
        assert served.tolist() == [1] * batch
        for b in range(batch):
            n = int(count[b])
            nodes_of = path[b, :n].tolist()
            assert all(parent[j] == i for i, j in zip(nodes_of, nodes_of[1:]))
            texts[b] += [guess[b * nodes + j] for j in nodes_of[1:]] + [int(token[b])]
            further += n > 1
        assert torch.equal(past, lens) and lens.tolist() == [len(t) - 1 for t in texts]
        torch.randn(1000, device="cuda").sum().item()
    # every page is held once by what is left, and a row's end gives all of them back
    assert int((refs == 1).sum()) == sum(-(-n // page) for n in lens.tolist())
    pages.free(refs, table, lens, page_size=page)
    assert int((refs == 1).sum()) == 0 and int((refs == -1).sum()) == -(-pool // 7)
    return texts, further


@pytest.mark.parametrize("capture", [False, True])
def test_drafted_decoding_writes_what_plain_decoding_does(capture):
    model = Model(0)
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, model.vocab, (n,), generator=gen).tolist() for n in (5, 30, 12)]
    steps = 12
    plain = [model.plain(p, 4 * steps + 4) for p in prompts]
    assert min(lead for _, lead in plain) > 1e-3       # no choice that 32 bits could turn
    texts, further = serve(model, prompts, [t for t, _ in plain], steps, gen, capture)
    assert further > steps
    for got, (want, _) in zip(texts, plain):
        assert got == want[:len(got)]


def serve_short_of_pages(model, prompts, want, most, gen, capture=False):
    """Drafted decoding with fewer pages than all sequences need at once: a row that `take` does not
    serve waits for the next step, and one that has `most` tokens ends, as does the last where none
    can go on. Returns what was written, how often a row waited, and how many wrote to the end."""
    batch, page, width, nodes, pool = len(prompts), 8, 12, 7, 19
    caches = [torch.full((pool, page, model.kv, model.dim), math.nan, device="cuda")
              for _ in "kv"]
    refs = torch.zeros(pool, dtype=torch.int32, device="cuda")
    refs[::7] = -1                                     # not to be taken
    table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(batch, dtype=torch.int32, device="cuda")
    going = torch.ones(batch, dtype=torch.int32, device="cuda")      # 0: the row has ended

    def forward(tokens, cu, tree, positions, live):
        q, k, v = model.project(tokens)
        q = decode.append_kv(k, v, *caches, table, live, cu_tokens=cu, q=q, cos=model.cos,
                             sin=model.sin, positions=positions)
        return model.logits(draft.tree_attention(q, *caches, table, live, cu, tree=tree))

    new = [len(p) - 1 for p in prompts]
    served = pages.take(refs, table, lens, int32(new).cuda(), page_size=page)
    assert served.tolist() == [1] * batch
    forward(int32([t for p in prompts for t in p[:-1]]).cuda(), starts_of(new).cuda(), None,
            int32([i for n in new for i in range(n)]).cuda(), lens)
    tree = int32([[1], [3], [5], [9], [5 + 16], [9 + 32], [5 + 16 + 64]]).cuda()
    depth = int32([0, 1, 1, 1, 2, 2, 3]).cuda()
    cu = starts_of([nodes] * batch).cuda()
    drafted = torch.zeros(batch * nodes, dtype=torch.int32, device="cuda")
    masks = tree.repeat(batch, 1)

    def step():
        starts = lens.clone()
        served = pages.take(refs, table, lens, lens + nodes * going, page_size=page) * going
        held, live = lens.clone(), lens * served
        logits = forward(drafted, cu, masks, (starts[:, None] + depth).flatten(), live)
        path, count, token = draft.accept(logits, drafted, cu, tree=masks, most=4)
        count = count * served
        pages.compact(caches, table, torch.where(served > 0, starts, -1), path, count,
                      seq_lens=lens)
        pages.free(refs, table, held, lens, page_size=page)
        return served, path, count, token

    def guesses(s):
        out = []
        for b in range(batch):
            right = want[b][len(texts[b]) - 1:]
            line = [texts[b][-1]] + torch.randint(0, model.vocab, (6,), generator=gen).tolist()
            good = [(), (1,), (2,), (2, 4), (2, 4, 6), (3, 5)][(s + b) % 6]
            for d, j in enumerate(good):
                if d + 1 < len(right):
                    line[j] = right[d + 1]
            out += line
        return out

    texts, active = [list(p) for p in prompts], list(range(batch))
    graph = out = None
    waited = ended = s = 0
    while active:
        guess = guesses(s)
        drafted.copy_(int32(guess))
        if capture and s == 1:
            graph = torch.cuda.CUDAGraph()
            state = [x.clone() for x in (*caches, refs, table, lens)]
            with torch.cuda.graph(graph):
                out = step()
            for x, y in zip((*caches, refs, table, lens), state):
                x.copy_(y)
        if graph is not None:
            graph.replay()
        else:
            out = step()
        served, path, count, token = (x.cpu() for x in out)
        for b in range(batch):
            assert (int(count[b]) > 0) == (int(served[b]) > 0) and (b in active or not served[b])
            if served[b]:
                texts[b] += [guess[b * nodes + j] for j in path[b, 1:int(count[b])].tolist()]
                texts[b].append(int(token[b]))
        waited += sum(1 - int(served[b]) for b in active)
        assert lens.tolist() == [len(t) - 1 if b in active else 0 for b, t in enumerate(texts)]
        over = [b for b in active if len(texts[b]) >= most]
        ended += len(over)
        if not over and not served.any():
            over = active[-1:]
        for b in over:
            active.remove(b)
            going[b] = 0
            pages.free(refs, table, lens, lens * going, page_size=page)
        # every page is counted as often as rows hold it
        uses = [-1 if p % 7 == 0 else 0 for p in range(pool)]
        for b, n in enumerate(lens.tolist()):
            for p in table[b, :-(-n // page)].tolist():
                uses[p] += 1
        assert refs.tolist() == uses
        s += 1
    return texts, waited, ended


@pytest.mark.parametrize("capture", [False, True])
def test_drafted_decoding_short_of_pages(capture):
    model = Model(5)
    gen = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, model.vocab, (n,), generator=gen).tolist() for n in (17, 5, 20, 9)]
    most = 44
    plain = [model.plain(p, most + 8 - len(p)) for p in prompts]
    assert min(lead for _, lead in plain) > 1e-3       # no choice that 32 bits could turn
    texts, waited, ended = serve_short_of_pages(model, prompts, [t for t, _ in plain], most, gen,
                                                capture)
    assert waited > 5 and ended > 1
    for got, (want, _) in zip(texts, plain):
        assert got == want[:len(got)]


def attend_state(seed, lens):
    gen = torch.Generator().manual_seed(seed)
    new = [5, 9, 2]
    bt, count = table_for(gen, lens, 16)
    kc, vc = (cache(gen, count, 16, 2, 64, BF16).cuda() for _ in "kv")
    q = rand(gen, sum(new), 8, 64, dtype=BF16).cuda()
    return gen, dict(q=q, k_cache=kc, v_cache=vc, block_table=bt.cuda(),
                     seq_lens=int32(lens).cuda(), cu_tokens=starts_of(new).cuda(),
                     tree=trees(gen, new, 1).cuda())


def test_attention_on_two_streams_at_once():
    streams = [torch.cuda.Stream() for _ in range(2)]
    states = [attend_state(seed, [2500, 900, 40])[1] for seed in (40, 41)]
    want = [draft.tree_attention(**s) for s in states]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(states):
            with torch.cuda.stream(streams[i]):
                got[i].append(draft.tree_attention(**s))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(o, w) for o in g)


def test_two_captured_attentions_replayed():
    graphs = []
    for seed in (50, 51):
        gen, s = attend_state(seed, [2500, 900, 40])
        draft.tree_attention(**s)
        logits, tokens, cu, tree = (x.cuda() for x in draft_case(gen, [5, 9], 5000, 1, F32, True))
        draft.accept(logits, tokens, cu, tree=tree)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = (draft.tree_attention(**s), *draft.accept(logits, tokens, cu, tree=tree))
        graphs.append((gen, s, (logits, tokens, cu, tree), g, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    for step in range(4):
        for gen, s, a, _, _ in graphs:
            s["seq_lens"] -= 13
            s["q"].copy_(rand(gen, *s["q"].shape))
            a[0].copy_(rand(gen, *a[0].shape))
        want = [(draft.tree_attention(**s), *draft.accept(*a[:3], tree=a[3]))
                for _, s, a, _, _ in graphs]
        torch.cuda.synchronize()
        for (_, _, _, g, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for w, (_, _, _, _, out) in zip(want, graphs):
            assert all(torch.equal(x, y) for x, y in zip(w, out)), step
        torch.randn(1000, device="cuda").sum().item()


def test_numpy_and_enceladus_arrays():
    gen = torch.Generator().manual_seed(20)
    lens, new = [9, 40], [3, 5]
    bt, count = table_for(gen, lens, 16)
    kc, vc = (cache(gen, count, 16, 2, 64, F32) for _ in "kv")
    q, tree, cu = rand(gen, 8, 4, 64), trees(gen, new, 1), starts_of(new)
    args = (q, kc, vc, bt, int32(lens), cu)
    want = draft.tree_attention(*(x.cuda() for x in args), tree=tree.cuda()).cpu().numpy()
    n = [x.numpy() for x in args]
    got = draft.tree_attention(*n, tree=tree.numpy())
    assert isinstance(got, np.ndarray) and np.array_equal(got, want)
    e = [enceladus.from_numpy(x) for x in n]
    got, lse = draft.tree_attention(*e, tree=enceladus.from_numpy(tree.numpy()), return_lse=True)
    assert isinstance(got, enceladus.Tensor) and np.array_equal(got.numpy(), want)
    assert lse.shape == (8, 4)
    logits, tokens, cu, tree = draft_case(gen, new, 500, 1, F32, True)
    want = [x.cpu().numpy() for x in draft.accept(logits.cuda(), tokens.cuda(), cu.cuda(),
                                                  tree=tree.cuda())]
    got = draft.accept(logits.numpy(), tokens.numpy(), cu.numpy(), tree=tree.numpy())
    assert all(np.array_equal(a, b) for a, b in zip(got, want))


def test_calls_are_timed_and_traced(tmp_path):
    _, s = attend_state(60, [300, 20, 9])
    assert enceladus.testing.do_bench(lambda: draft.tree_attention(**s), rep=3) > 0
    path = tmp_path / "t.json"
    with enceladus.capture(path):
        draft.tree_attention(**s)
    assert "ek_tree_attention" in path.read_text()
