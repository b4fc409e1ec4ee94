"""`enceladus.decode` on the GPU against 64-bit forms: types, head layouts, lengths, pages,
strides, masks, refused pages, streams, graphs, and a run of its operators together.

Tolerances count the roundings of 32-bit arithmetic (unit 2^-24) relative to the magnitudes
that are summed, and half a step of the output's type.
"""

import math

import numpy as np
import pytest
import torch

import enceladus
from enceladus import decode
from oracle import decode_ref as R

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
F8 = torch.float8_e4m3fn
U = 2.0 ** -24
# half of the smallest step of each type
SUB = {F32: 2.0 ** -150, F16: 2.0 ** -25, BF16: 2.0 ** -134, F8: 2.0 ** -10}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, tol, what=""):
    dtype = got.dtype if got.dtype in (F32, F16, BF16) else None
    got, want, tol = got.cpu().double(), want.cpu(), tol.cpu()
    assert got.shape == want.shape
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), what
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what
    off = (got - want).abs()
    ok = (off <= tol) | nan | inf
    if dtype is not None:
        # beyond half a step above the type's largest value a result is its infinity
        edge = torch.finfo(dtype).max * (1 + half_step(dtype) / 2)
        ok |= (got == want.sign() * math.inf) & (want.abs() + tol >= edge)
    assert ok.all(), f"{what}: off by {off[~ok].max():.3g}, {(off / tol)[~ok].max():.3g} times " \
                     f"the tolerance, at {int((~ok).sum())} of {ok.numel()}"


def rand(gen, *shape, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=gen) * scale).to(dtype)


def table_for(gen, lens, page, spare=3, width=None):
    """A block table over shuffled pages; entries behind a sequence's last page are wild."""
    need = [-(-max(n, 0) // page) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=gen).to(torch.int32)
    width = max(max(need), 1) if width is None else width
    bt = torch.full((len(lens), width), 2 ** 31 - 1, dtype=torch.int32)
    bt[:, 1::2] = -7
    at = 0
    for b, n in enumerate(need):
        bt[b, :n] = order[at:at + n]
        at += n
    return bt, pages


def cache(gen, pages, page, kv, dim, dtype, layout="token", fill=None):
    shape = (pages, page, kv, dim) if layout == "token" else (pages, kv, page, dim)
    c = rand(gen, *shape).to(dtype) if fill is None else \
        torch.full(shape, fill).to(dtype)
    return c if layout == "token" else c.permute(0, 2, 1, 3)


def on_gpu(x):
    """The same strides on the GPU."""
    y = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device="cuda")
    return y.copy_(x)


def only_live(c, bt, lens, page):
    """NaN wherever no sequence's length reaches."""
    live = torch.zeros(c.shape[0], c.shape[1], dtype=torch.bool)
    for b, n in enumerate(lens):
        ids, off, ok = R.slots(bt[b], page, c.shape[0], 0, max(0, min(n, bt.shape[1] * page)))
        live[ids[ok], off[ok]] = True
    x = c.float()
    x[~live] = math.nan
    return torch.empty_strided(c.shape, c.stride(), dtype=c.dtype).copy_(x.to(c.dtype))


def attention_tolerance(q, out, mag, smax, n, dtype):
    """Scores: a product over dim and its scale in 32 bits, off by (dim + 16) U S, which the
    weights have as relative error, beside exp2's few units and their own two-term rounding;
    numerator and denominator both, and both sums over n."""
    split = {F32: U, F16: 2.0 ** -22, BF16: 2.0 ** -16}[dtype]
    rel = 2 * ((q.shape[-1] + 16) * U * smax[..., None] + 16 * U + split) + 2 * (n + 8) * U
    return half_step(dtype) * out.abs() + mag * rel * 1.01 + SUB[dtype]


def check_attention(q, kc, vc, bt, lens, **kw):
    sl = torch.tensor(lens, dtype=torch.int32)
    want, lse, mag, smax = R.paged_attention(q, kc, vc, bt, lens, **kw)
    got, got_lse = decode.paged_attention(on_gpu(q), on_gpu(kc), on_gpu(vc), bt.cuda(), sl.cuda(),
                                          return_lse=True, **kw)
    n = max(max(lens), 1)
    close(got, want, attention_tolerance(q, want, mag, smax, n, q.dtype), "out")
    tol = (q.shape[-1] + 16) * U * smax + (n + 64) * U + lse.abs().nan_to_num(0, 0, 0) * 4 * U
    close(got_lse, lse, tol, "lse")
    return got


LENS = [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 1000]


@pytest.mark.parametrize("dtype,cdtype", [(F32, F32), (F16, F16), (BF16, BF16), (F16, F8),
                                          (BF16, F8)])
@pytest.mark.parametrize("dim,kv,group,page,layout", [
    (64, 2, 4, 16, "token"), (128, 2, 1, 16, "token"), (128, 1, 8, 64, "head"),
    (80, 2, 3, 24, "token"), (256, 1, 5, 32, "token"), (16, 3, 2, 1, "token"),
    (192, 1, 16, 7, "head"), (96, 1, 17, 128, "token"), (128, 1, 40, 16, "token"),
])
def test_attention(dtype, cdtype, dim, kv, group, page, layout):
    gen = torch.Generator().manual_seed(dim * 31 + group)
    bt, pages = table_for(gen, LENS, page)
    kc, vc = (only_live(cache(gen, pages, page, kv, dim, cdtype, layout), bt, LENS, page)
              for _ in "kv")
    q = rand(gen, len(LENS), kv * group, dim, dtype=dtype)
    kw = dict(k_scale=0.5, v_scale=2.0) if cdtype is F8 else {}
    check_attention(q, kc, vc, bt, LENS, **kw)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [8, 24, 72, 104, 136, 248])
def test_attention_odd_head_dims(dtype, dim):
    gen = torch.Generator().manual_seed(dim)
    lens = [130, 3, 77]
    bt, pages = table_for(gen, lens, 16)
    kc, vc = (only_live(cache(gen, pages, 16, 2, dim, dtype), bt, lens, 16) for _ in "kv")
    check_attention(rand(gen, 3, 6, dim, dtype=dtype), kc, vc, bt, lens)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window,softcap,scale", [(1, 0.0, None), (7, 0.0, 0.3), (64, 20.0, None),
                                                  (100, 0.0, -0.2), (1000, 5.0, 1.0),
                                                  (5000, 0.5, 0.01), (0, 50.0, 0.0)])
def test_attention_window_softcap_scale(dtype, window, softcap, scale):
    gen = torch.Generator().manual_seed(window)
    bt, pages = table_for(gen, LENS, 16)
    kc, vc = (only_live(cache(gen, pages, 16, 2, 64, dtype), bt, LENS, 16) for _ in "kv")
    check_attention(rand(gen, len(LENS), 8, 64, dtype=dtype), kc, vc, bt, LENS, window=window,
                    softcap=softcap, scale=scale)


@pytest.mark.parametrize("dtype,dim", [(F16, 64), (BF16, 128), (BF16, 240)])
@pytest.mark.parametrize("group", [1, 7, 8, 9, 24])
@pytest.mark.parametrize("window,softcap,scale", [(0, 30.0, None), (71, 0.0, -0.2),
                                                  (200, 2.0, -1.0)])
def test_attention_8_bit_window_softcap_scale(dtype, dim, group, window, softcap, scale):
    gen = torch.Generator().manual_seed(window + group)
    bt, pages = table_for(gen, LENS, 16)
    bt[-1, 3] = -1                                          # a page that is not there
    kc, vc = (only_live(cache(gen, pages, 16, 2, dim, F8), bt, LENS, 16) for _ in "kv")
    check_attention(rand(gen, len(LENS), 2 * group, dim, dtype=dtype), kc, vc, bt, LENS,
                    window=window, softcap=softcap, scale=scale, k_scale=0.5)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_one_large_weight_among_many_small_ones(dtype):
    """One key with nearly all of the weight, thousands that share the rest."""
    gen = torch.Generator().manual_seed(5)
    lens, dim = [6000], 64
    bt, pages = table_for(gen, lens, 16)
    kc, vc = (cache(gen, pages, 16, 1, dim, dtype, fill=0.0) for _ in "kv")
    vc = (vc.float() + 1.0).to(dtype)
    q = torch.zeros(1, 1, dim)
    q[..., 0] = 16.0
    first = int(bt[0, 0])
    kc[first, 3, 0, 0] = 8.0               # its score is 16 above the others' (e^-16 each)
    vc[first, 3, 0, :] = 0.0
    check_attention(q.to(dtype), kc, vc, bt, lens)


def test_attention_of_wild_pages_and_lengths():
    """Pages outside the cache count as absent, a length beyond the table as all of it."""
    gen = torch.Generator().manual_seed(1)
    page, kv, dim = 16, 2, 64
    kc, vc = (cache(gen, 20, page, kv, dim, BF16) for _ in "kv")
    bt = torch.randint(0, 20, (6, 12), generator=gen, dtype=torch.int32)
    bt[0, 3], bt[1, 0], bt[2, :], bt[3, 11] = -1, 2 ** 31 - 1, 20, -2 ** 31
    lens = [192, 100, 150, 192, 2 ** 31 - 1, -5]
    check_attention(rand(gen, 6, 4, dim, dtype=BF16), kc, vc, bt, lens)


def test_attention_values_that_are_not_finite():
    gen = torch.Generator().manual_seed(2)
    lens = [200, 200, 200, 90]
    bt, pages = table_for(gen, lens, 16)
    kc, vc = (only_live(cache(gen, pages, 16, 1, 64, F32), bt, lens, 16) for _ in "kv")
    vc[bt[0, 3], 5, 0, 7] = math.inf           # one element of one sequence
    vc[bt[1, 0], 0, 0, 9] = math.nan
    kc[bt[2, 1], 2, 0, 0] = math.nan           # all of one sequence
    check_attention(rand(gen, 4, 4, 64), kc, vc, bt, lens)


@pytest.mark.parametrize("dtype,value", [(F16, math.inf), (BF16, -math.inf), (BF16, math.nan)])
def test_attention_values_that_are_not_finite_stay_in_their_elements(dtype, value):
    """Infinite or NaN there (a weight is a sum of two 16-bit terms, which may differ in sign),
    and no other element sees it."""
    gen = torch.Generator().manual_seed(3)
    lens = [200, 90]
    bt, pages = table_for(gen, lens, 16)
    kc, vc = (only_live(cache(gen, pages, 16, 1, 64, dtype), bt, lens, 16) for _ in "kv")
    q = rand(gen, 2, 4, 64, dtype=dtype).cuda()
    rest = kc.cuda(), vc.cuda(), bt.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    want = decode.paged_attention(q, *rest)
    rest[1][int(bt[0, 3]), 5, 0, 7] = value
    got = decode.paged_attention(q, *rest)
    assert not torch.isfinite(got[0, :, 7]).any()
    got[0, :, 7] = want[0, :, 7]
    assert torch.equal(got, want)


@pytest.mark.parametrize("batch", [1, 63, 64, 65, 200])
def test_attention_of_many_sequences(batch):
    gen = torch.Generator().manual_seed(batch)
    lens = torch.randint(0, 400, (batch,), generator=gen).tolist()
    lens[::5] = [0] * len(lens[::5])
    bt, pages = table_for(gen, lens, 16)
    kc, vc = (only_live(cache(gen, pages, 16, 1, 64, BF16), bt, lens, 16) for _ in "kv")
    check_attention(rand(gen, batch, 2, 64, dtype=BF16), kc, vc, bt, lens)


def test_attention_strides_and_places():
    """Queries out of a fused projection, tables and lengths of a larger batch, caches inside
    one array, results into rows of another; the result over the queries themselves."""
    gen = torch.Generator().manual_seed(3)
    lens, page, kv, heads, dim = [70, 0, 333], 16, 2, 6, 128
    bt, pages = table_for(gen, lens, page)
    both = rand(gen, pages, 2, page, kv, dim + 8, dtype=F16).cuda()
    kc, vc = both[:, 0, ..., 3:3 + dim], both[:, 1, ..., 3:3 + dim]
    rows = rand(gen, 3, heads + 4, dim, dtype=F16).cuda()
    q = rows[:, 1:1 + heads]
    wide = torch.zeros(3, 40, dtype=torch.int32).cuda()
    wide[:, 5:5 + bt.shape[1]] = bt.cuda()
    lens3 = torch.zeros(3, 4, dtype=torch.int32).cuda()
    lens3[:, 2] = torch.tensor(lens).cuda()
    room = torch.full((3, heads, dim + 1), 7.0, dtype=F16).cuda()
    out = room[..., :dim]
    want, _, mag, smax = R.paged_attention(q.cpu(), kc.cpu(), vc.cpu(), bt, lens)
    tol = attention_tolerance(q, want, mag, smax, 333, F16)
    args = kc, vc, wide[:, 5:5 + bt.shape[1]], lens3[:, 2]
    got = decode.paged_attention(q, *args, out=out)
    assert got.data_ptr() == out.data_ptr()
    close(got, want, tol)
    assert (room[..., dim] == 7).all()
    assert decode.paged_attention(q, *args, out=q).data_ptr() == q.data_ptr()
    close(q, want, tol)


def test_attention_far_into_a_cache_beyond_32_bit_offsets():
    page, kv, dim = 64, 8, 128
    pages = (1 << 32) // (page * kv * dim) + 40            # 2^32 elements, 4 GiB of e4m3
    gen = torch.Generator().manual_seed(4)
    lens = [300, 1000]
    bt = torch.stack([torch.randperm(20, generator=gen)[:16] + pages - 40 + 20 * b
                      for b in range(2)]).to(torch.int32)
    bt[:, ::2] -= pages - 40                               # near and far in turn
    kc, vc = (torch.zeros(pages, page, kv, dim, dtype=torch.uint8, device="cuda").view(F8)
              for _ in "kv")
    small = [rand(gen, 80, page, kv, dim).to(F8) for _ in "kv"]    # the first and last 40 pages
    ids = torch.cat([torch.arange(40), torch.arange(pages - 40, pages)])
    for c, s in zip((kc, vc), small):
        c.view(torch.uint8)[ids.cuda()] = s.view(torch.uint8).cuda()
    back = torch.where(bt >= 40, bt - (pages - 80), bt)
    q = rand(gen, 2, 32, dim, dtype=BF16)
    want, _, mag, smax = R.paged_attention(q, small[0], small[1], back, lens)
    got = decode.paged_attention(q.cuda(), kc, vc, bt.cuda(),
                                 torch.tensor(lens, dtype=torch.int32).cuda())
    close(got, want, attention_tolerance(q, want, mag, smax, 1000, BF16))


def test_attention_of_a_long_sequence_is_split_and_joined():
    gen = torch.Generator().manual_seed(6)
    lens = [70001, 12]
    bt, pages = table_for(gen, lens, 128)
    kc, vc = (cache(gen, pages, 128, 1, 64, F32) for _ in "kv")
    q = rand(gen, 2, 3, 64)
    a = check_attention(q, kc, vc, bt, lens)
    assert torch.equal(a, check_attention(q, kc, vc, bt, lens))       # the same bits again


def attention_variant(call):
    """What `call` returns, and the macros of the one attention kernel that it planned."""
    decode._plans.clear()
    got = call()
    plans = [p for p in decode._plans.values() if p.file == "paged_attention.hip"]
    assert len(plans) == 1
    return got, dict(plans[0].macros)


@pytest.mark.parametrize("dtype,dim", [(F16, 128), (BF16, 128), (F16, 80), (BF16, 80), (F32, 64),
                                       (F32, 48)])
@pytest.mark.parametrize("window,softcap,scale", [(0, 0.0, None), (1200, 0.0, -0.2),
                                                  (1300, 8.0, 0.3)])
def test_attention_16_keys_a_step(dtype, dim, window, softcap, scale, monkeypatch):
    """The step of large calls (here: of a block table far wider than the lengths), with either
    kind of loads: the same bits."""
    gen = torch.Generator().manual_seed(dim + window)
    lens, page, kv = [3000, 0, 1, 777, 64, 2000, 17], 16, 32
    bt, pages = table_for(gen, lens, page, width=190)
    bt[3, 5] = -1                                           # a page that is not there
    kc, vc = (only_live(cache(gen, pages, page, kv, dim, dtype), bt, lens, page) for _ in "kv")
    q = rand(gen, len(lens), kv, dim, dtype=dtype)
    got = []
    for size in (1 << 62, 0):
        monkeypatch.setattr(decode, "_STREAM", size)
        x, macros = attention_variant(lambda: check_attention(
            q, kc, vc, bt, lens, window=window, softcap=softcap, scale=scale))
        assert macros["EK_KT"] == 16 and macros["EK_PAD"] == (dim in (80, 48))
        got.append(x)
    decode._plans.clear()
    assert torch.equal(*got)


@pytest.mark.parametrize("dim", [64, 80, 128, 200])
@pytest.mark.parametrize("window,softcap,scale", [(1, 0.0, None), (64, 20.0, None),
                                                  (100, 0.0, -0.2), (1000, 5.0, -1.0),
                                                  (0, 50.0, 0.0)])
def test_attention_fp16_window_softcap_scale(dim, window, softcap, scale):
    gen = torch.Generator().manual_seed(window + dim)
    bt, pages = table_for(gen, LENS, 16)
    kc, vc = (only_live(cache(gen, pages, 16, 2, dim, F16), bt, LENS, 16) for _ in "kv")
    check_attention(rand(gen, len(LENS), 8, dim, dtype=F16), kc, vc, bt, LENS, window=window,
                    softcap=softcap, scale=scale)


@pytest.mark.parametrize("batch", [256, 257, 320, 1000])
@pytest.mark.parametrize("empty", ["none", "first", "last", "some", "all"])
def test_attention_beyond_256_sequences(batch, empty):
    """With sequences of several chunks among them, and empty ones in the first 256, behind
    them, in both."""
    gen = torch.Generator().manual_seed(batch)
    lens = torch.randint(1, 80, (batch,), generator=gen).tolist()
    lens[7::60] = [900] * len(lens[7::60])
    none = {"none": range(0), "first": range(3, 250, 2), "last": range(251, batch),
            "some": range(0, batch, 3), "all": range(batch)}[empty]
    for b in none:
        lens[b] = 0
    bt, pages = table_for(gen, lens, 16)
    kc, vc = (only_live(cache(gen, pages, 16, 1, 64, BF16), bt, lens, 16) for _ in "kv")
    check_attention(rand(gen, batch, 2, 64, dtype=BF16), kc, vc, bt, lens)


@pytest.mark.parametrize("dtype,cdtype", [(F32, F32), (F16, F16), (BF16, BF16), (F16, F8),
                                          (BF16, F8)])
@pytest.mark.parametrize("dim", [16, 128])
@pytest.mark.parametrize("scale", [1e6, 1e8, -1e10, 2.0 ** 40, 2.0 ** 60])
def test_attention_of_large_scores(dtype, cdtype, dim, scale):
    """Scores far apart in sequences of one chunk and of several: the largest ones, which are
    equal, share the weight. Products of small whole numbers are exact and differ by 1 at least,
    so every weight is 2^0 or 0: what is left to round are the sums over the keys, the division
    and a few products, and in the lse a product."""
    gen = torch.Generator().manual_seed(dim)
    lens, kv = [1, 50, 64, 65, 700, 1500], 2
    bt, pages = table_for(gen, lens, 16)

    def whole(*shape):
        x = torch.randint(-1, 2, shape, generator=gen).float()
        x[..., 16:] = 0
        return x
    kc = only_live(whole(pages, 16, kv, dim).to(cdtype), bt, lens, 16)
    vc = only_live(cache(gen, pages, 16, kv, dim, cdtype), bt, lens, 16)
    q = whole(len(lens), kv * 3, dim).to(dtype)
    kw = dict(scale=scale, k_scale=0.5 if cdtype is F8 else 1.0)
    want, lse, mag, _ = R.paged_attention(q, kc, vc, bt, lens, **kw)
    got, got_lse = decode.paged_attention(on_gpu(q), on_gpu(kc), on_gpu(vc), bt.cuda(),
                                          torch.tensor(lens, dtype=torch.int32).cuda(),
                                          return_lse=True, **kw)
    close(got, want, half_step(dtype) * want.abs() + mag * 2 * (1500 + 16) * U + SUB[dtype], "out")
    close(got_lse, lse, 8 * U * lse.abs() + (1500 + 64) * U, "lse")


@pytest.mark.parametrize("dtype,cdtype", [(F32, F32), (F16, F16), (BF16, BF16), (F16, F8),
                                          (BF16, F8)])
@pytest.mark.parametrize("group", [4, 16])
def test_attention_weights_keep_32_bits(dtype, cdtype, group):
    """Two nearly equal weights w1, w2 of 0.37 to 0.61 whose values are 1 and -1, beside a weight
    of 1 whose value is 0: the result, (w1 - w2) / (1 + w1 + w2), is about 2^-16, so that it shows
    the weights' errors of 2^-24 and not its own rounding.

    In units of U = 2^-24: the scores are exact; their product with the scale, and that one's
    own rounding, put 2 U of up to 0.73 into the exponent, exp2 is off by at most 2 U of the
    weight: 0.61 (0.73 * 2 + 2) = 2.2 U for each weight, 4.4 U for both. fp16's two terms add
    2^-22 = 4 U of it, 4.9 U for both. The two products' sums are below 1, their terms (up to 6)
    are added with 1 U each or, if the matrix unit cuts off, 2 U: 12 U. All that is divided by
    1 + w1 + w2 >= 1.73: 12.4 U. Errors of the divisor count by the result, 2^-16."""
    gen = torch.Generator().manual_seed(group)
    batch, dim = 64, 16
    kc, vc = (torch.zeros(1, 16, 1, dim) for _ in "kv")
    kc[0, 1, 0, 0] = kc[0, 2, 0, 0] = kc[0, 2, 0, 1] = 1.0
    vc[0, 1], vc[0, 2] = 1.0, -1.0
    kc, vc = kc.to(cdtype), vc.to(cdtype)
    q = torch.zeros(batch, group, dim)
    q[..., 0] = -torch.rand(batch, group, generator=gen) / 2 - 0.5
    q[..., 1] = -torch.rand(batch, group, generator=gen) * 2.0 ** -14
    q = q.to(dtype)
    bt, lens = torch.zeros(batch, 1, dtype=torch.int32), [3] * batch
    want, _, _, _ = R.paged_attention(q, kc, vc, bt, lens, scale=1.0)
    got = decode.paged_attention(q.cuda(), kc.cuda(), vc.cuda(), bt.cuda(),
                                 torch.tensor(lens, dtype=torch.int32).cuda(), scale=1.0)
    close(got, want, half_step(dtype) * want.abs() + 12.5 * U, "out")


# -- appending ------------------------------------------------------------------------------

def append_case(gen, dtype, cdtype, lens, new, page, kv, heads, dim, rotary, layout="token",
                behind=0, before=0):
    bt, pages = table_for(gen, lens, page)
    kc, vc = (cache(gen, pages, page, kv, dim, cdtype, layout) for _ in "kv")
    tokens = sum(new) + behind + before
    d = dict(k=rand(gen, tokens, kv, dim, dtype=dtype), v=rand(gen, tokens, kv, dim, dtype=dtype),
             k_cache=kc, v_cache=vc, block_table=bt,
             seq_lens=torch.tensor(lens, dtype=torch.int32))
    if heads:
        d["q"] = rand(gen, tokens, heads, dim, dtype=dtype)
    if any(n != 1 for n in new) or behind or before:
        d["cu_tokens"] = torch.tensor([before + sum(new[:b]) for b in range(len(new) + 1)],
                                      dtype=torch.int32)
    if rotary:
        at = torch.arange(max(max(lens), 1)).double()[:, None]
        j = torch.arange(rotary // 2).double()
        angle = at * 10000.0 ** (-2 * j / rotary)
        d["cos"], d["sin"] = angle.cos().float(), angle.sin().float()
    return d


def check_append(d, q_out=None, **kw):
    names = ("k", "v", "k_cache", "v_cache", "block_table", "seq_lens")
    g = {n: on_gpu(x) for n, x in d.items()}
    if q_out is None and "q" in d:
        q_out = torch.full(d["q"].shape, 3.0).to(d["q"].dtype)
    want_q, want_k, want_v, done = R.append_kv(*(d[n] for n in names),
                                               **{n: d[n] for n in d if n not in names},
                                               q_out=q_out, **kw)
    go = None if q_out is None else on_gpu(q_out)
    got = decode.append_kv(*(g[n] for n in names),
                           **{n: g[n] for n in g if n not in names}, q_out=go, **kw)
    if "q" in d:
        assert got.data_ptr() == go.data_ptr()
        # two products and a sum of 32 bits, and the rounding
        top = d["q"].double().abs().amax(-1, keepdim=True)
        close(got, want_q, half_step(d["q"].dtype) * want_q.abs() + 8 * U * top +
              SUB[d["q"].dtype], "q")
    else:
        assert got is None
    ct = d["k_cache"].dtype
    for name, want, src, s in (("k_cache", want_k, d["k"], kw.get("k_scale", 1.0)),
                               ("v_cache", want_v, d["v"], kw.get("v_scale", 1.0))):
        top = src.double().abs().max() / s
        close(g[name], want, half_step(ct) * want.abs() + 8 * U * top + SUB[ct], name)
        same = g[name].cpu()[~done].view(torch.uint8) == d[name][~done].view(torch.uint8)
        assert same.all(), f"{name}: slots that are not the tokens' were written"
    return g, got


@pytest.mark.parametrize("dtype,cdtype", [(F32, F32), (F16, F16), (BF16, BF16), (F32, F8),
                                          (F16, F8), (BF16, F8)])
@pytest.mark.parametrize("dim,rotary,kv,heads,page,layout,interleaved", [
    (128, 128, 2, 8, 16, "token", False), (64, 32, 3, 3, 24, "head", True),
    (64, 0, 1, 5, 1, "token", False), (80, 20, 2, 2, 7, "token", False),
    (16, 14, 2, 0, 16, "token", False), (256, 256, 1, 16, 64, "head", False),
    (96, 6, 1, 1, 16, "token", True), (192, 128, 4, 4, 128, "token", True),
])
def test_append(dtype, cdtype, dim, rotary, kv, heads, page, layout, interleaved):
    gen = torch.Generator().manual_seed(dim + rotary)
    kw = dict(k_scale=0.25, v_scale=0.3) if cdtype is F8 else {}
    for lens, new, behind, before in (([1, 5, 16, 17, 300], [1] * 5, 0, 0),
                                      ([40, 1, 17, 90], [33, 1, 0, 50], 5, 2)):
        d = append_case(gen, dtype, cdtype, lens, new, page, kv, heads, dim, rotary, layout,
                        behind, before)
        check_append(d, interleaved=interleaved, **kw)


def test_append_in_place_and_strided():
    """Rows of one fused projection, queries rotated where they are."""
    gen = torch.Generator().manual_seed(9)
    d = append_case(gen, BF16, BF16, [10, 30, 64], [1] * 3, 16, 2, 4, 64, 64)
    want, _, _, _ = R.append_kv(*(d[n] for n in ("k", "v", "k_cache", "v_cache", "block_table",
                                                 "seq_lens")), q=d["q"], cos=d["cos"],
                                sin=d["sin"])
    row = torch.cat((d["q"], d["k"], d["v"]), 1)
    wide = torch.zeros(3, 8, 65, dtype=BF16)
    wide[..., 1:] = row
    wide = wide.cuda()
    q, k, v = wide[..., 1:].split([4, 2, 2], 1)
    got = decode.append_kv(k, v, d["k_cache"].cuda(), d["v_cache"].cuda(),
                           d["block_table"].cuda(), d["seq_lens"].cuda(), q=q, q_out=q,
                           cos=d["cos"].cuda(), sin=d["sin"].cuda())
    assert got.data_ptr() == q.data_ptr()
    top = row.double().abs().max()
    close(q, want, half_step(BF16) * want.abs() + 8 * U * top)
    assert torch.equal(k.cpu(), d["k"]) and (wide[..., 0] == 0).all()


def test_append_skips_rows_without_a_slot():
    gen = torch.Generator().manual_seed(10)
    d = append_case(gen, F32, F32, [20, 40, 9, 64], [4, 3, 9, 6], 16, 1, 2, 64, 64, behind=3)
    d["seq_lens"] = torch.tensor([2, 2 ** 31 - 1, 9, 64], dtype=torch.int32)  # 2 tokens early,
    d["block_table"][2, 0] = d["k_cache"].shape[0]                # beyond, no such page,
    d["cos"], d["sin"] = d["cos"][:62], d["sin"][:62]             # positions without a row
    check_append(d)
    d["seq_lens"] = torch.tensor([-3, -2 ** 31, 0, 1 << 30], dtype=torch.int32)
    check_append(d)
    d["cu_tokens"] = torch.tensor([5, 5, 5, 2 ** 31 - 1, 2 ** 31 - 1], dtype=torch.int32)
    d["seq_lens"] = torch.tensor([1, 1, 1, 1], dtype=torch.int32)
    check_append(d)


@pytest.mark.parametrize("batch", [64, 65, 300])
def test_append_many_sequences(batch):
    gen = torch.Generator().manual_seed(batch)
    new = torch.randint(0, 4, (batch,), generator=gen).tolist()
    lens = [n + int(torch.randint(0, 50, (1,), generator=gen)) for n in new]
    check_append(append_case(gen, BF16, BF16, lens, new, 16, 1, 2, 64, 64, behind=1))


def test_append_many_tokens():
    gen = torch.Generator().manual_seed(11)
    check_append(append_case(gen, F16, F16, [9000, 700], [8999, 300], 16, 1, 3, 64, 64))


@pytest.mark.parametrize("heads,dim,rotary,behind", [(37, 24, 8, 3), (9, 136, 0, 0),
                                                     (20, 192, 16, 1)])
def test_append_many_rows_of_many_tokens(heads, dim, rotary, behind):
    """Several waves per token, the last of them with fewer rows than the others."""
    gen = torch.Generator().manual_seed(heads)
    check_append(append_case(gen, F32, F32, [4200, 3, 1], [4199, 1, 0], 16, 3, heads, dim, rotary,
                             behind=behind))


@pytest.mark.parametrize("batch", [256, 257, 600, 16384, 16385, 20011])
def test_append_single_tokens_of_many_sequences(batch):
    gen = torch.Generator().manual_seed(batch)
    new = [1] * batch if batch < 1000 else \
        (torch.rand(batch, generator=gen) < 0.05).int().tolist()
    new[3:40] = [0] * 37
    new[-1] = 1
    lens = [n + int(torch.randint(0, 20, (1,), generator=gen)) for n in new]
    d = append_case(gen, F16, F8, lens, new, 16, 2, 2, 64, 64, before=2, behind=2)
    d["block_table"][::5, 0] = -1                              # pages that are not there
    check_append(d)


@pytest.mark.parametrize("dtype,cdtype", [(F32, F32), (F16, F8), (BF16, BF16)])
def test_loads_past_the_caches_give_the_same(dtype, cdtype, monkeypatch):
    """Large rows and caches are loaded with another hint: the same bits."""
    gen = torch.Generator().manual_seed(12)
    lens, new = [300, 77], [200, 70]
    d = append_case(gen, dtype, cdtype, lens, new, 16, 2, 4, 80, 40)
    got = []
    for size in (1 << 62, 0):
        monkeypatch.setattr(decode, "_STREAM", size)
        monkeypatch.setattr(decode, "_STREAM_ROWS", size)
        decode._plans.clear()
        g, q = check_append(d)
        o = decode.paged_attention(q[[199, 269]], g["k_cache"], g["v_cache"], g["block_table"],
                                   g["seq_lens"]) if dtype is not F32 or cdtype is F32 else q
        x = check_logits(logits_case(torch.Generator().manual_seed(13), 9, 9001, 70, 5, True, dtype))
        got.append((g["k_cache"].view(torch.uint8), g["v_cache"].view(torch.uint8), q, o, x))
    decode._plans.clear()
    for x, y in zip(*got):
        assert torch.equal(x, y)


def test_append_into_caches_of_one_array():
    """Keys and values of a page side by side, call after call; shifted by a page, so that they
    share memory, they are refused also where the plan is known."""
    gen = torch.Generator().manual_seed(15)
    d = append_case(gen, BF16, BF16, [20, 33], [1, 1], 16, 2, 4, 64, 64)
    pages = d["k_cache"].shape[0]
    both = torch.zeros(pages + 1, 2, 16, 2, 64, dtype=BF16)
    d["k_cache"], d["v_cache"] = both[:-1, 0], both[:-1, 1]
    want = [x.clone() for x in R.append_kv(*(d[n] for n in ("k", "v", "k_cache", "v_cache",
                                                            "block_table", "seq_lens")),
                                           q=d["q"], cos=d["cos"], sin=d["sin"])[1:3]]
    g = {n: x.cuda() for n, x in d.items() if "cache" not in n}
    room = both.cuda()
    kw = dict(q=g["q"], cos=g["cos"], sin=g["sin"])
    rest = g["block_table"], g["seq_lens"]
    for _ in range(2):
        room.zero_()
        decode.append_kv(g["k"], g["v"], room[:-1, 0], room[:-1, 1], *rest, **kw)
        for i, w in enumerate(want):
            close(room[:-1, i], w, half_step(BF16) * w.abs() + 8 * U * 5)
    before = room.clone()
    with pytest.raises(ValueError, match="`k_cache` overlaps `v_cache`"):
        decode.append_kv(g["k"], g["v"], room[:-1, 0], room[1:, 0], *rest, **kw)
    assert torch.equal(room, before)


def test_append_rounds_to_8_bits_as_the_type_says():
    """Every neighbourhood of an e4m3 value: its rounding, ties, zeros, overflow, NaN."""
    grid = torch.arange(256, dtype=torch.uint8).view(F8).float()
    grid = grid[~grid.isnan()].sort().values.double()
    mid = (grid[1:] + grid[:-1]) / 2
    x = torch.cat([grid, mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20),
                   torch.tensor([449.0, 464.0, 1e30, -1e30, math.inf, -math.inf, math.nan, 0.0,
                                 -0.0, 2.0 ** -11, 1e-30], dtype=torch.float64)]).float()
    x = torch.cat([x, torch.zeros(-len(x) % 64)]).view(-1, 1, 64)
    n = x.shape[0]
    kc, vc = (torch.zeros(n, 1, 1, 64, dtype=torch.uint8).view(F8).cuda() for _ in "kv")
    bt = torch.arange(n, dtype=torch.int32)[:, None].cuda()
    decode.append_kv(x.cuda(), (-x).cuda(), kc, vc, bt, torch.ones(n, dtype=torch.int32).cuda())
    want = x.clamp(-448, 448).to(F8).float().view(n, 64)
    for got, sign in ((kc, 1), (vc, -1)):
        got = got.float().cpu().view(n, 64)
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(9), (sign * want).nan_to_num(9))
        assert torch.equal(got.signbit()[~want.isnan()], (sign * want).signbit()[~want.isnan()])


@pytest.mark.parametrize("cdtype", [F32, F16, BF16, F8])
@pytest.mark.parametrize("scale", [0.3, 0.7, 1.9, 2.0 - 2.0 ** -23, 2.0 ** -30 * 1.1, 0.25])
def test_append_divides_by_the_scale(cdtype, scale):
    """Cached values are the 32-bit quotients, rounded to the cache's type: around ties, where a
    product with the reciprocal may fall on the other side."""
    gen = torch.Generator().manual_seed(8)
    s = np.float32(scale)
    dtype = F32 if cdtype is F8 else cdtype
    if cdtype is F8:
        grid = torch.arange(256, dtype=torch.uint8).view(F8).float()
        grid = grid[~grid.isnan()].sort().values
        mid = ((grid[1:] + grid[:-1]) / 2).numpy() * s
        x = np.concatenate([mid, np.nextafter(mid, np.float32(1e9)),
                            np.nextafter(mid, np.float32(-1e9))])
    else:
        x = (rand(gen, 64 * 64) * float(s)).to(dtype).float().numpy()
    x = np.concatenate([x, np.float32([math.inf, -math.inf, math.nan, 0.0, -0.0])])
    x = np.concatenate([x, np.zeros(-len(x) % 64, np.float32)]).reshape(-1, 1, 64)
    x = torch.from_numpy(x).to(dtype)
    n = x.shape[0]
    kc, vc = (torch.zeros(n, 1, 1, 64, device="cuda").to(cdtype) for _ in "kv")
    decode.append_kv(x.cuda(), (-x).cuda(), kc, vc,
                     torch.arange(n, dtype=torch.int32)[:, None].cuda(),
                     torch.ones(n, dtype=torch.int32).cuda(), k_scale=float(s),
                     v_scale=float(s))
    want = torch.from_numpy(x.float().numpy() / s)
    if cdtype is F8:
        want = want.clamp(-448, 448)
    want = want.to(cdtype).float().view(n, 64)
    for got, sign in ((kc, 1), (vc, -1)):
        got = got.float().cpu().view(n, 64)
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(9, 1e30, -1e30),
                           (sign * want).nan_to_num(9, 1e30, -1e30))


def test_append_far_below_the_first_position():
    """A length of -2^31 with an end of 2^31 - 1: every position is negative, none wraps round."""
    gen = torch.Generator().manual_seed(14)
    d = append_case(gen, F32, F32, [20, 20], [2, 2], 16, 1, 2, 64, 0)
    d["cu_tokens"] = torch.tensor([0, 2, 2 ** 31 - 1], dtype=torch.int32)
    d["seq_lens"] = torch.tensor([20, -2 ** 31], dtype=torch.int32)
    check_append(d)


# -- logits ---------------------------------------------------------------------------------

def logits_case(gen, rows, vocab, history=0, biases=0, mask=False, dtype=F32, numbers=False):
    d = dict(logits=rand(gen, rows, vocab, scale=4.0).to(dtype))
    if history:
        d["tokens"] = torch.randint(-3, vocab + 3, (rows, history), generator=gen,
                                    dtype=torch.int32)
        d["tokens"][:, ::3] %= 7                               # some come many times
        d["token_lens"] = torch.randint(-1, history + 2, (rows,), generator=gen).int()
        d["prompt_lens"] = torch.randint(-1, history + 1, (rows,), generator=gen).int()
        for n, lo, hi in (("repetition", 0.7, 1.5), ("frequency", -0.2, 0.6),
                          ("presence", -0.2, 0.6)):
            d[n] = 1.3 if numbers else torch.rand(rows, generator=gen) * (hi - lo) + lo
    if biases:
        d["bias_ids"] = torch.randint(-2, min(vocab + 2, 60), (rows, biases), generator=gen,
                                      dtype=torch.int32)       # ids repeat
        d["bias"] = rand(gen, rows, biases, scale=3.0)
    if mask:
        d["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)),
                                     generator=gen).int()
        d["allowed"][rows // 2] = 0                            # a row that allows nothing
    d["temperature"] = 0.7 if numbers else torch.rand(rows, generator=gen) * 1.5
    return d


def check_logits(d, out=None):
    want = R.adjust_logits(**d)
    dtype = d["logits"].dtype
    # what each sum adds up, all of one sign; a dozen 32-bit roundings, and the output's
    mag = dict(d, logits=d["logits"].double().abs().nan_to_num(0, 0, 0))
    mag.pop("allowed", None)
    for n in ("frequency", "presence"):
        if n in d:
            mag[n] = -d[n].abs() if isinstance(d[n], torch.Tensor) else -abs(d[n])
    if "repetition" in d:
        r = torch.as_tensor(d["repetition"]).expand(want.shape[0])
        mag["repetition"] = torch.minimum(r, 1 / r)
    if "bias" in d:
        mag["bias"] = d["bias"].abs()
    top = R.adjust_logits(**mag)
    g = {n: on_gpu(x) if isinstance(x, torch.Tensor) else x for n, x in d.items()}
    got = decode.adjust_logits(g.pop("logits"), out=out, **g)
    assert got.dtype == dtype
    close(got, want, half_step(dtype) * want.abs().nan_to_num(0, 0, 0) + 12 * U * top +
          SUB[dtype], "logits")
    return got


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,vocab,history,biases,mask", [
    (1, 1, 3, 0, False), (2, 7, 5, 3, True), (3, 31, 0, 0, True), (3, 32, 9, 2, True),
    (1, 2047, 100, 5, False), (5, 2049, 1, 300, True), (4, 8191, 1000, 17, True),
    (2, 32000, 5000, 0, False), (40, 50001, 260, 20, True), (300, 8193, 33, 0, True),
    (3, 100003, 0, 0, False), (70000, 3, 2, 1, True), (2, 4097, 30, 1023, False),
    (2, 9000, 0, 513, False), (1, 20000, 2048, 511, True),
])
def test_logits(dtype, rows, vocab, history, biases, mask):
    gen = torch.Generator().manual_seed(rows + vocab)
    check_logits(logits_case(gen, rows, vocab, history, biases, mask, dtype))


def test_logits_numbers_for_all_rows():
    gen = torch.Generator().manual_seed(1)
    d = logits_case(gen, 5, 5000, 200, 4, True, BF16, numbers=True)
    check_logits(d)
    d.pop("token_lens"), d.pop("prompt_lens")                  # the whole row, all generated
    check_logits(d)
    d["temperature"] = 0.0
    check_logits(d)


def test_logits_that_are_not_finite():
    gen = torch.Generator().manual_seed(2)
    d = logits_case(gen, 4, 3000, 500, 8, True, F32)
    d["logits"][0, :1000:3] = math.nan
    d["logits"][1, :1000:3] = -math.inf
    d["logits"][2, :1000:3] = math.inf
    d["logits"][3] = torch.finfo(F32).min
    d["logits"][3, 5] = torch.finfo(F32).max
    d["temperature"] = torch.full((4,), 1.25)
    d["repetition"] = torch.full((4,), 1.0)
    check_logits(d)


def test_logits_of_temperatures_near_zero():
    """Below 2^-128, where the reciprocal is infinite: zeros stay zeros, small logits finite."""
    gen = torch.Generator().manual_seed(5)
    x = rand(gen, 5, 300, scale=4.0)
    x[:, ::7] = 0.0
    x[:, 1::7] *= 2.0 ** -40
    check_logits(dict(logits=x, temperature=torch.tensor([1e-40, 2.0 ** -149, 1e-38, 1e-30,
                                                          2.0 ** -101])))


@pytest.mark.parametrize("lift", [0, 60])
def test_logits_quotients_are_rounded_once(lift):
    """x / temperature, and x / repetition of positive logits, are the 32-bit quotients."""
    gen = torch.Generator().manual_seed(7)
    rows, vocab = 200, 3001
    x = rand(gen, rows, vocab, scale=4.0)
    by = torch.rand(rows, generator=gen) * 1.5 + 0.25
    by[0], by[1], by[2] = 2.0 - 2.0 ** -23, 1.0 + 2.0 ** -23, 1.0
    x[:, 0], x[:, 1], x[:, 2] = math.inf, -math.inf, 0.0
    t = (by.double() * 2.0 ** -lift).float()
    got = decode.adjust_logits(x.cuda(), temperature=t.cuda()).cpu()
    assert torch.equal(got, (x.double() / t.double()[:, None]).float())
    tokens = torch.arange(vocab, dtype=torch.int32).expand(rows, -1).contiguous()
    prompt = torch.full((rows,), vocab, dtype=torch.int32)
    got = decode.adjust_logits(x.cuda(), tokens=tokens.cuda(), prompt_lens=prompt.cuda(),
                               repetition=t.cuda()).cpu()
    r = t.double()[:, None]
    want = torch.where(x > 0, x.double() / r, x.double() * r).float()
    assert torch.equal(got, want)


def test_logits_strides_shared_masks_and_places():
    gen = torch.Generator().manual_seed(3)
    d = logits_case(gen, 6, 4099, 77, 5, True, F16)
    mask = d["allowed"][:1].clone()
    d["allowed"] = mask.expand(6, -1)
    want = check_logits({n: x.contiguous() if isinstance(x, torch.Tensor) else x
                         for n, x in d.items()})
    wide = torch.full((6, 5000), 9.0, dtype=F16).cuda()
    view = wide[:, 1:4100]
    view.copy_(d["logits"])
    g = {n: x.cuda() for n, x in d.items() if n not in ("logits", "allowed")}
    g["allowed"] = mask.cuda().expand(6, -1)
    g["tokens"] = torch.cat((d["tokens"], d["tokens"]), 1).cuda()[:, :77]
    two = torch.stack((d["repetition"], d["repetition"]), 1).cuda()
    g["repetition"] = two[:, 1]
    got = decode.adjust_logits(view, out=view, **g)
    assert got.data_ptr() == view.data_ptr() and torch.equal(got, want)
    assert (wide[:, 0] == 9).all() and (wide[:, 4100:] == 9).all()


def test_logits_biases_add_in_their_order():
    """Entries of one id: 1e8 + 1 - 1e8 in 32 bits is 0, in another order 1."""
    x = torch.zeros(1, 10)
    ids = torch.tensor([[4, 4, 2, 4]], dtype=torch.int32)
    for values, want in (((1e8, 1.0, 0.5, -1e8), 0.0), ((1e8, -1e8, 0.5, 1.0), 1.0)):
        got = decode.adjust_logits(x.cuda(), bias_ids=ids.cuda(),
                                   bias=torch.tensor([values]).cuda())
        assert got[0, 4].item() == want and got[0, 2].item() == 0.5


# -- as a program uses them -------------------------------------------------------------------

def test_numpy_and_enceladus_arrays():
    gen = torch.Generator().manual_seed(20)
    d = append_case(gen, F32, F32, [9, 40], [1, 1], 16, 2, 4, 64, 64)
    order = ("k", "v", "k_cache", "v_cache", "block_table", "seq_lens")
    torch_q = decode.append_kv(*(d[n].cuda() for n in order), q=d["q"].cuda(),
                               cos=d["cos"].cuda(), sin=d["sin"].cuda())
    n = {k: x.numpy().copy() for k, x in d.items()}
    q = decode.append_kv(*(n[k] for k in order), q=n["q"], cos=n["cos"], sin=n["sin"])
    assert isinstance(q, np.ndarray) and np.array_equal(q, torch_q.cpu().numpy())
    assert not np.array_equal(n["k_cache"], d["k_cache"].numpy())
    o = decode.paged_attention(q, n["k_cache"], n["v_cache"], n["block_table"], n["seq_lens"])
    e = {k: enceladus.from_numpy(x) for k, x in n.items()}
    eq = enceladus.from_numpy(q)
    eo, lse = decode.paged_attention(eq, e["k_cache"], e["v_cache"], e["block_table"],
                                     e["seq_lens"], return_lse=True)
    assert isinstance(eo, enceladus.Tensor) and np.array_equal(eo.numpy(), o)
    assert lse.shape == (2, 4)
    lg = logits_case(gen, 3, 500, 20, 2, True, F32)
    want = decode.adjust_logits(**{k: x.cuda() for k, x in lg.items()}).cpu().numpy()
    got = decode.adjust_logits(**{k: x.numpy() for k, x in lg.items()})
    assert np.array_equal(got, want)
    got = decode.adjust_logits(**{k: enceladus.from_numpy(x.numpy()) for k, x in lg.items()})
    assert np.array_equal(got.numpy(), want)


def step_state(seed, batch=3, kv=2, heads=8, dim=64, vocab=997, page=16, most=200):
    gen = torch.Generator().manual_seed(seed)
    width = -(-most // page)
    s = dict(k_cache=torch.zeros(batch * width + 2, page, kv, dim, dtype=BF16),
             v_cache=torch.zeros(batch * width + 2, page, kv, dim, dtype=BF16),
             table=torch.randperm(batch * width + 2, generator=gen)[:batch * width].view(
                 batch, width).int(),
             lens=torch.zeros(batch, dtype=torch.int32),
             w=rand(gen, heads * dim, vocab, scale=0.1),
             tokens=torch.zeros(batch, most, dtype=torch.int32))
    at = torch.arange(most).double()[:, None] * 10000.0 ** (-2 * torch.arange(dim // 2) / dim)
    s["cos"], s["sin"] = at.cos().float(), at.sin().float()
    return gen, {n: x.cuda() for n, x in s.items()}


def one_step(s, q, k, v):
    """A step as a program makes it: append, attend, project, adjust, choose."""
    q = decode.append_kv(k, v, s["k_cache"], s["v_cache"], s["table"], s["lens"], q=q,
                         cos=s["cos"], sin=s["sin"])
    o = decode.paged_attention(q, s["k_cache"], s["v_cache"], s["table"], s["lens"])
    x = decode.adjust_logits(o.flatten(1).float() @ s["w"], tokens=s["tokens"],
                             token_lens=s["lens"], repetition=1.2, frequency=0.3, presence=0.1,
                             temperature=0.8)
    return o, x


def test_a_run_of_steps():
    """Prompts, then single tokens: every step's attention and logits against the whole
    sequences' in 64 bits, kept outside the cache."""
    gen, s = step_state(30)
    batch, kv, heads, dim = 3, 2, 8, 64
    keys, values = ([torch.zeros(0, kv, dim, dtype=torch.float64) for _ in range(batch)]
                    for _ in "kv")
    cos, sin = s["cos"].cpu(), s["sin"].cpu()

    def remember(b, pos, k, v):
        turned = R.rotate(k, cos[pos], sin[pos], False).to(BF16).double()
        keys[b] = torch.cat((keys[b], turned[None]))
        values[b] = torch.cat((values[b], v[None].double()))

    prompts = [70, 1, 33]
    k, v = (rand(gen, sum(prompts), kv, dim, dtype=BF16) for _ in "kv")
    s["lens"].copy_(torch.tensor(prompts))
    cu = torch.tensor([0, 70, 71, 104], dtype=torch.int32).cuda()
    assert decode.append_kv(k.cuda(), v.cuda(), s["k_cache"], s["v_cache"], s["table"],
                            s["lens"], cu_tokens=cu, cos=s["cos"], sin=s["sin"]) is None
    for b, lo in enumerate((0, 70, 71)):
        for i in range(prompts[b]):
            remember(b, i, k[lo + i], v[lo + i])
    for step in range(12):
        s["lens"] += 1
        lens = s["lens"].tolist()
        q, k, v = (rand(gen, batch, n, dim, dtype=BF16) for n in (heads, kv, kv))
        o, x = one_step(s, q.cuda(), k.cuda(), v.cuda())
        want = torch.zeros(batch, heads, dim, dtype=torch.float64)
        for b in range(batch):
            remember(b, lens[b] - 1, k[b], v[b])
            assert len(keys[b]) == lens[b]
            qb = R.rotate(q[b], cos[lens[b] - 1], sin[lens[b] - 1], False).to(BF16).double()
            for h in range(heads):
                p = torch.softmax(keys[b][:, h // 4] @ qb[h] / 8, 0)
                want[b, h] = p @ values[b][:, h // 4]
        # a rotated value next to a border may round to either side in 32 and in 64 bits: a step
        # of 2^-7 of one element; all other errors are far below that
        assert (o.cpu().double() - want).norm() <= 2.0 ** -7 * want.norm()
        logits = o.flatten(1).float() @ s["w"]
        ref = R.adjust_logits(logits.cpu(), s["tokens"].cpu(), lens, repetition=1.2,
                              frequency=0.3, presence=0.1, temperature=0.8)
        close(x, ref, 12 * U * (logits.cpu().double().abs() * 1.2 + 80) / 0.8)
        s["tokens"][torch.arange(batch), s["lens"].long() - 1] = x.argmax(1).int()


def test_steps_on_two_streams_at_once():
    streams = [torch.cuda.Stream() for _ in range(2)]
    runs = []
    for seed in (40, 41):
        gen, s = step_state(seed, most=3000)
        s["lens"].fill_(2500)
        s["k_cache"].copy_(rand(gen, *s["k_cache"].shape))
        s["v_cache"].copy_(rand(gen, *s["v_cache"].shape))
        runs.append((s, [rand(gen, 3, n, 64, dtype=BF16).cuda() for n in (8, 2, 2)]))
    want = [one_step(s, *x) for s, x in runs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (s, x) in enumerate(runs):
            with torch.cuda.stream(streams[i]):
                got[i].append(one_step(s, *x))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        for o, x in g:
            assert torch.equal(o, w[0]) and torch.equal(x, w[1])


def test_two_captured_steps_replayed():
    """Two graphs, replayed in turn and at once, with lengths and caches that move on between
    the replays; each replay against the eager step."""
    graphs = []
    for seed in (50, 51):
        gen, s = step_state(seed, most=1500)
        s["lens"].fill_(700 + seed)
        s["k_cache"].copy_(rand(gen, *s["k_cache"].shape))
        s["v_cache"].copy_(rand(gen, *s["v_cache"].shape))
        x = [rand(gen, 3, n, 64, dtype=BF16).cuda() for n in (8, 2, 2)]
        one_step(s, *x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            one_step(s, *x)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = one_step(s, *x)
        graphs.append((gen, s, x, g, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    for step in range(4):
        for gen, s, x, g, out in graphs:
            s["lens"] += 37
            for t in x:
                t.copy_(rand(gen, *t.shape))
        want = [one_step(s, *x) for _, s, x, _, _ in graphs]
        torch.cuda.synchronize()
        for (_, s, x, g, out), st in zip(graphs, streams):
            if step % 2:
                with torch.cuda.stream(st):
                    g.replay()
            else:
                g.replay()
        torch.cuda.synchronize()
        for w, (_, _, _, _, out) in zip(want, graphs):
            assert torch.equal(out[0], w[0]) and torch.equal(out[1], w[1]), step
        torch.randn(1000, device="cuda").sum().item()


def test_calls_are_timed_and_traced(tmp_path):
    gen = torch.Generator().manual_seed(60)
    d = logits_case(gen, 3, 500, 20)
    g = {n: x.cuda() for n, x in d.items()}
    assert enceladus.testing.do_bench(lambda: decode.adjust_logits(**g), rep=3) > 0
    path = tmp_path / "t.json"
    with enceladus.capture(path):
        decode.adjust_logits(**g)
    assert "ek_adjust_logits" in path.read_text()


def test_settings_by_their_values():
    """A setting given as a tensor or a NumPy scalar counts with the value that it has at the
    call: a plan made before is not taken for the object's sake."""
    gen = torch.Generator().manual_seed(70)
    lens = [50, 9]
    bt, pages = table_for(gen, lens, 16)
    kc, vc = (cache(gen, pages, 16, 1, 64, F32).cuda() for _ in "kv")
    q = rand(gen, 2, 2, 64).cuda()
    args = q, kc, vc, bt.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    scale = torch.tensor(0.25)
    a = decode.paged_attention(*args, scale=scale)
    scale.fill_(0.5)
    b = decode.paged_attention(*args, scale=scale)
    assert torch.equal(a, decode.paged_attention(*args, scale=0.25))
    assert torch.equal(b, decode.paged_attention(*args, scale=np.float32(0.5)))
    assert not torch.equal(a, b)
    x, tokens = rand(gen, 2, 100).cuda(), torch.tensor([[3, 4], [5, 6]], dtype=torch.int32).cuda()
    for _ in range(2):
        a = decode.adjust_logits(x, tokens=tokens, repetition=np.float32(1.5), presence=1)
        b = decode.adjust_logits(x, tokens=tokens, repetition=1.5, presence=True)
        assert torch.equal(a, b)
