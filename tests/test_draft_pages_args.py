"""`enceladus.draft`, `enceladus.pages` and positions of `decode.append_kv`: what they refuse, before
anything is launched (CPU)."""

import numpy as np
import pytest
import torch

import enceladus
from enceladus import decode, draft, pages


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def f8(*shape):
    return torch.zeros(*shape).to(torch.float8_e4m3fn)


def call(fn, defaults, order, kw):
    d = {**defaults(), **kw}
    first = [d.pop(n) for n in order]
    return fn(*first, **d)


def _attend():
    return dict(q=torch.zeros(6, 8, 64), k_cache=torch.zeros(10, 16, 2, 64),
                v_cache=torch.zeros(10, 16, 2, 64), block_table=i32(3, 4), seq_lens=i32(3),
                cu_tokens=i32(4), tree=i32(6, 1))


ATTEND_ORDER = ("q", "k_cache", "v_cache", "block_table", "seq_lens", "cu_tokens")
ATTEND = [
    (dict(q=torch.zeros(6, 8, 64, dtype=torch.float64)), TypeError, "`q` must hold"),
    (dict(q=[1.0]), TypeError, "must be an array"),
    (dict(q=torch.zeros(6, 512)), ValueError, "3 dimensions"),
    (dict(q=torch.zeros(6, 64, 8).transpose(1, 2)), ValueError, "contiguous"),
    (dict(q=torch.zeros(6, 7, 64)), ValueError, "not a multiple"),
    (dict(q=torch.zeros(6, 8, 64).half()), TypeError, "`k_cache` must hold"),
    (dict(k_cache=torch.zeros(10, 16, 2, 32)), ValueError, "`k_cache` must have shape"),
    (dict(v_cache=torch.zeros(10, 8, 2, 64)), ValueError, "`v_cache` must have shape"),
    (dict(v_cache=torch.zeros(10, 2, 16, 64).transpose(1, 2)), ValueError, "same strides"),
    (dict(k_cache=torch.zeros(10, 0, 2, 64), v_cache=torch.zeros(10, 0, 2, 64)), ValueError,
     "at least one token"),
    (dict(k_cache=f8(10, 16, 2, 64)), ValueError, "host"),
    (dict(block_table=torch.zeros(3, 4, dtype=torch.int64)), TypeError, "`block_table`"),
    (dict(block_table=i32(2, 4)), ValueError, "`block_table`"),
    (dict(seq_lens=i32(4)), ValueError, "`seq_lens`"),
    (dict(cu_tokens=i32(0)), ValueError, "one entry more"),
    (dict(cu_tokens=i32(3)), ValueError, "`block_table`"),
    (dict(cu_tokens=torch.zeros(4)), TypeError, "`cu_tokens`"),
    (dict(tree=i32(5, 1)), ValueError, "`tree`"),
    (dict(tree=i32(6)), ValueError, "`tree`"),
    (dict(tree=i32(6, 0)), ValueError, "at least one word"),
    (dict(tree=torch.zeros(6, 1, dtype=torch.int64)), TypeError, "`tree`"),
    (dict(tree=i32(1, 6).t().expand(6, 2)), ValueError, "contiguous"),
    (dict(scale=2.0 ** 61), ValueError, "`scale`"),
    (dict(scale=float("nan")), ValueError, "`scale`"),
    (dict(softcap=-1.0), ValueError, "`softcap`"),
    (dict(softcap=float("inf")), ValueError, "`softcap`"),
    (dict(window=-1), ValueError, "`window`"),
    (dict(window=1.5), TypeError, "integer"),
    (dict(k_scale=0.0), ValueError, "`k_scale`"),
    (dict(v_scale=float("nan")), ValueError, "`v_scale`"),
    (dict(out=torch.zeros(6, 8, 32)), ValueError, "`out`"),
    (dict(out=torch.zeros(6, 8, 64).half()), TypeError, "`out`"),
    (dict(out=torch.zeros(1, 8, 64).expand(6, 8, 64)), ValueError, "expanded"),
    (dict(q=torch.zeros(1, 8, 12).expand(6, 8, 12), k_cache=torch.zeros(1, 1, 2, 12),
          v_cache=torch.zeros(1, 1, 2, 12)), ValueError, "multiple of 8"),
    (dict(q=torch.zeros(1, 8, 264).expand(6, 8, 264), k_cache=torch.zeros(1, 1, 2, 264),
          v_cache=torch.zeros(1, 1, 2, 264)), ValueError, "up to 256"),
    (dict(q=torch.zeros(1, 8, 64).expand((1 << 23) + 1, 8, 64), tree=None), ValueError,
     "tokens are supported"),
    (dict(q=torch.zeros(1, 512, 8).expand(1 << 22, 512, 8), k_cache=torch.zeros(1, 1, 1, 8),
          v_cache=torch.zeros(1, 1, 1, 8), tree=None), ValueError, "too many"),
    (dict(block_table=i32(1, 1).expand(3, 1 << 26)), ValueError, "contiguous"),
]


@pytest.mark.parametrize("kw,error,text", ATTEND)
def test_attention_refuses(kw, error, text):
    with pytest.raises(error, match=text):
        call(draft.tree_attention, _attend, ATTEND_ORDER, kw)


def test_attention_of_too_long_tables():
    kw = dict(block_table=i32(1, 1 << 21).expand(3, 1 << 21), k_cache=torch.zeros(1, 1024, 2, 64),
              v_cache=torch.zeros(1, 1024, 2, 64))
    with pytest.raises(ValueError, match="at most"):
        call(draft.tree_attention, _attend, ATTEND_ORDER, kw)


def test_attention_sequences():
    kw = dict(block_table=i32(1, 4).expand((1 << 16) + 1, 4),
              seq_lens=i32(1).expand((1 << 16) + 1), cu_tokens=i32(1).expand((1 << 16) + 2))
    with pytest.raises(ValueError, match="sequences are supported"):
        call(draft.tree_attention, _attend, ATTEND_ORDER, kw)


def test_attention_of_nothing():
    d = _attend()
    assert call(draft.tree_attention, _attend, ATTEND_ORDER, dict(
        q=torch.zeros(0, 8, 64), tree=i32(0, 1))).shape == (0, 8, 64)
    assert call(draft.tree_attention, _attend, ATTEND_ORDER, dict(
        block_table=i32(0, 4), seq_lens=i32(0), cu_tokens=i32(1))).shape == d["q"].shape
    out, lse = call(draft.tree_attention, _attend, ATTEND_ORDER, dict(
        q=torch.zeros(6, 0, 64), return_lse=True))
    assert out.shape == (6, 0, 64) and lse.shape == (6, 0)


def _accept():
    return dict(logits=torch.zeros(6, 50), tokens=i32(6), cu_tokens=i32(4), tree=i32(6, 1))


ACCEPT = [
    (dict(logits=torch.zeros(6, 50, dtype=torch.int32)), TypeError, "`logits`"),
    (dict(logits=torch.zeros(300)), ValueError, "2 dimensions"),
    (dict(logits=torch.zeros(50, 6).t()), ValueError, "contiguous"),
    (dict(logits=torch.zeros(6, 0)), ValueError, "rows of 1"),
    (dict(tokens=i32(5)), ValueError, "`tokens`"),
    (dict(tokens=torch.zeros(6, dtype=torch.int64)), TypeError, "`tokens`"),
    (dict(cu_tokens=i32(0)), ValueError, "one entry more"),
    (dict(tree=i32(5, 1)), ValueError, "`tree`"),
    (dict(tree=i32(6, 33)), ValueError, "at most 1024"),
    (dict(most=-1), ValueError, "`most`"),
    (dict(most=2.0), TypeError, "integer"),
]


@pytest.mark.parametrize("kw,error,text", ACCEPT)
def test_accept_refuses(kw, error, text):
    with pytest.raises(error, match=text):
        call(draft.accept, _accept, ("logits", "tokens", "cu_tokens"), kw)


def test_accept_of_no_sequences():
    for most, width in ((None, 32), (3, 3)):
        path, count, token = call(draft.accept, _accept, ("logits", "tokens", "cu_tokens"),
                                  dict(cu_tokens=i32(1), most=most))
        assert path.shape == (0, width) and count.shape == (0,) and token.shape == (0,)


def _append():
    return dict(k=torch.zeros(3, 2, 64), v=torch.zeros(3, 2, 64),
                k_cache=torch.zeros(10, 16, 2, 64), v_cache=torch.zeros(10, 16, 2, 64),
                block_table=i32(3, 4), seq_lens=i32(3), cos=torch.zeros(9, 32),
                sin=torch.zeros(9, 32), positions=i32(3))


APPEND = [
    (dict(cos=None, sin=None), "need `cos`"),
    (dict(cos=None, sin=None, positions=None, pair_axes=(0,)), "without `positions`"),
    (dict(positions=None, pair_axes=(0,) * 32), "without `positions`"),
    (dict(positions=i32(4)), "`positions`"),
    (dict(positions=i32(2, 4), pair_axes=(0,) * 32), "`positions`"),
    (dict(positions=i32(1, 1, 3)), "`positions` must have 2 dimensions"),
    (dict(positions=i32(2, 3)), "need `pair_axes`"),
    (dict(positions=i32(0, 3), pair_axes=(0,) * 32), "1 to 4 axes"),
    (dict(positions=i32(5, 3), pair_axes=(0,) * 32), "1 to 4 axes"),
    (dict(positions=i32(2, 3), pair_axes=(0,) * 31), "32 entries"),
    (dict(positions=i32(2, 3), pair_axes=(0,) * 31 + (2,)), "from 0 to 1"),
    (dict(positions=i32(2, 3), pair_axes=(0,) * 31 + (-1,)), "from 0 to 1"),
]


@pytest.mark.parametrize("kw,text", APPEND)
def test_append_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        call(decode.append_kv, _append, ("k", "v", "k_cache", "v_cache", "block_table",
                                         "seq_lens"), kw)


def test_append_refuses_types():
    for kw in (dict(positions=torch.zeros(3)), dict(pair_axes=(0.5,) * 32), dict(pair_axes=3)):
        with pytest.raises(TypeError):
            call(decode.append_kv, _append, ("k", "v", "k_cache", "v_cache", "block_table",
                                             "seq_lens"), kw)


def _caches(n=2, **kw):
    return [torch.zeros(10, 16, 2, 64, **kw) for _ in range(n)]


CACHES = [
    (3, TypeError, "`caches` must be arrays"),
    ([], ValueError, "1 to 256 caches"),
    (_caches(1) * 257, ValueError, "1 to 256 caches"),
    ([3], TypeError, r"`caches\[0\]` must be an array"),
    ([torch.zeros(10, 16, 128)], ValueError, "4 dimensions"),
    (torch.zeros(16, 2, 64), ValueError, "of 4 dimensions, or one of 5"),
    (_caches(1) + [torch.zeros(10, 16, 2, 32)], ValueError, r"`caches\[1\]` differs"),
    (_caches(1) + [torch.zeros(10, 2, 16, 64).transpose(1, 2)], ValueError, "differs"),
    (_caches(1) + _caches(1, dtype=torch.float16), ValueError, "differs"),
    ([torch.zeros(10, 16, 64, 2).transpose(2, 3)], ValueError, "contiguous"),
    ([torch.zeros(1, 16, 2, 64).expand(10, 16, 2, 64)], ValueError, "expanded"),
    ([torch.zeros(10, 0, 2, 64)], ValueError, "at least one token"),
    (_caches(1, dtype=torch.int32), TypeError, "must hold"),
    ([torch.zeros(1, 1, 1, 1).expand(1 << 25, 1, 1, 1)], ValueError, "expanded"),
    ([torch.zeros(10, 16, 2, 64).numpy()[:, ::-1]], ValueError, "negative strides"),
]


@pytest.mark.parametrize("caches,error,text", CACHES)
def test_caches_refused(caches, error, text):
    for fn in (lambda c: pages.copy(c, i32(1), i32(1)),
               lambda c: pages.compact(c, i32(3, 4), i32(3), i32(3, 2), i32(3)),
               lambda c: pages.fork(c, i32(10), i32(3, 4), i32(3), i32(1), i32(1))):
        with pytest.raises(error, match=text):
            fn(caches)


def test_caches_that_share_elements():
    a = torch.zeros(10, 2, 16, 2, 64)
    apart = [a[:, 0], a[:, 1]]
    rows = torch.zeros(11, 16, 2, 64)
    for bad in ([a[:, 0], a[:, 0]], [rows[:10], rows[1:]], [a[:, 0, :, :, :32], a[:, 0, :, :, 31:63]]):
        plan = pages._pages_plan([], [decode._Array("c", x) for x in bad], [], set(), 0,
                                 (0,) * 18)
        with pytest.raises(ValueError, match="share elements"):
            pages._check_apart(plan, [x.data_ptr() for x in bad])
    for good in (apart, [a[:, 0, :, :, :32], a[:, 0, :, :, 32:]], [rows[:5], rows[5:10]]):
        plan = pages._pages_plan([], [decode._Array("c", x) for x in good], [], set(), 0,
                                 (0,) * 18)
        pages._check_apart(plan, [x.data_ptr() for x in good])
    if not torch.cuda.is_available():
        with pytest.raises(ValueError, match="share elements"):
            pages.copy([a[:, 0], a[:, 0]], i32(1), i32(1))


COPY = [
    (dict(source=i32(2)), ValueError, "`target`"),
    (dict(source=torch.zeros(1, dtype=torch.int64)), TypeError, "`source`"),
    (dict(target=i32(1, 1)), ValueError, "`target`"),
    (dict(source=i32(1).expand(1 << 24), target=i32(1).expand(1 << 24)), ValueError, "too many"),
]


@pytest.mark.parametrize("kw,error,text", COPY)
def test_copy_refuses(kw, error, text):
    with pytest.raises(error, match=text):
        call(pages.copy, lambda: dict(caches=_caches(), source=i32(1), target=i32(1)),
             ("caches", "source", "target"), kw)


def _compact():
    return dict(caches=_caches(), block_table=i32(3, 4), starts=i32(3), keep=i32(3, 2),
                counts=i32(3), seq_lens=i32(3))


COMPACT = [
    (dict(block_table=i32(3)), ValueError, "`block_table`"),
    (dict(starts=i32(2)), ValueError, "`starts`"),
    (dict(keep=i32(2, 2)), ValueError, "`keep`"),
    (dict(keep=i32(2, 3).t()), ValueError, "contiguous"),
    (dict(counts=i32(4)), ValueError, "`counts`"),
    (dict(counts=torch.zeros(3)), TypeError, "`counts`"),
    (dict(seq_lens=i32(2)), ValueError, "`seq_lens`"),
    (dict(seq_lens=i32(1).expand(3)), ValueError, "expanded"),
]


@pytest.mark.parametrize("kw,error,text", COMPACT)
def test_compact_refuses(kw, error, text):
    with pytest.raises(error, match=text):
        call(pages.compact, _compact, ("caches", "block_table", "starts", "keep", "counts"), kw)


def _fork():
    return dict(caches=_caches(), refs=i32(10), block_table=i32(3, 4), seq_lens=i32(3),
                source=i32(1), target=i32(1))


FORK = [
    (dict(refs=i32(9)), ValueError, "`refs`"),
    (dict(refs=torch.zeros(10)), TypeError, "`refs`"),
    (dict(refs=i32(1).expand(10)), ValueError, "contiguous"),
    (dict(block_table=i32(3, 0, 4)), ValueError, "`block_table`"),
    (dict(block_table=i32(1, 4).expand(3, 4)), ValueError, "expanded"),
    (dict(block_table=i32(3, 1 << 27)[:, ::1]), ValueError, "at most"),
    (dict(seq_lens=i32(2)), ValueError, "`seq_lens`"),
    (dict(source=i32(2)), ValueError, "`target`"),
    (dict(source=i32(1).expand(1 << 24), target=i32(1).expand(1 << 24)), ValueError, "too many"),
]


@pytest.mark.parametrize("kw,error,text", FORK)
def test_fork_refuses(kw, error, text):
    with pytest.raises(error, match=text):
        call(pages.fork, _fork, ("caches", "refs", "block_table", "seq_lens", "source", "target"),
             kw)


ROWS = [
    (dict(refs=i32(1, 10)), ValueError, "`refs`"),
    (dict(refs=i32(1).expand(1 << 25)), ValueError, "contiguous"),
    (dict(block_table=torch.zeros(3, 4)), TypeError, "`block_table`"),
    (dict(seq_lens=i32(2)), ValueError, "`seq_lens`"),
    (dict(seq_lens=None), ValueError, "`seq_lens`"),
    (dict(new_lens=i32(2)), ValueError, "`new_lens`"),
    (dict(new_lens=torch.zeros(3, dtype=torch.int64)), TypeError, "`new_lens`"),
    (dict(page_size=0), ValueError, "`page_size`"),
    (dict(page_size=-16), ValueError, "`page_size`"),
    (dict(page_size=(1 << 28) + 1), ValueError, "at most"),
    (dict(page_size=16.0), TypeError, "integer"),
]


@pytest.mark.parametrize("fn", [pages.take, pages.free])
@pytest.mark.parametrize("kw,error,text", ROWS)
def test_take_and_free_refuse(fn, kw, error, text):
    with pytest.raises(error, match=text):
        call(fn, lambda: dict(refs=i32(10), block_table=i32(3, 4), seq_lens=i32(3),
                              new_lens=i32(3), page_size=16),
             ("refs", "block_table", "seq_lens", "new_lens"), kw)


def test_take_needs_lengths():
    with pytest.raises(TypeError):
        pages.take(i32(10), i32(3, 4), i32(3), None, page_size=16)


def test_calls_on_nothing():
    """No pairs, rows, forks or elements: nothing is launched."""
    pages.copy(_caches(), i32(0), i32(0))
    pages.copy([torch.zeros(0, 16, 2, 64)], i32(1), i32(1))
    pages.compact(_caches(), i32(0, 4), i32(0), i32(0, 2), i32(0))
    pages.compact(_caches(), i32(3, 4), i32(3), i32(3, 0), i32(3))
    assert pages.fork(_caches(), i32(10), i32(3, 4), i32(3), i32(0), i32(0)).shape == (0,)
    assert pages.take(i32(10), i32(0, 4), i32(0), i32(0), page_size=16).shape == (0,)
    pages.free(i32(10), i32(0, 4), i32(0), page_size=16)


def test_modules_are_public():
    assert enceladus.draft is draft and enceladus.pages is pages
    for module in (draft, pages):
        for name in module.__all__:
            assert getattr(module, name).__doc__


def test_settings_of_any_number_type():
    for one in (1, True, np.float32(1.0), torch.tensor(1.0)):
        with pytest.raises(ValueError, match="not a multiple"):
            call(draft.tree_attention, _attend, ATTEND_ORDER,
                 dict(q=torch.zeros(6, 7, 64), scale=one, k_scale=one))
    for two in (2, np.int64(2)):
        with pytest.raises(ValueError, match="`new_lens`"):
            pages.take(i32(10), i32(3, 4), i32(3), i32(1), page_size=two)
