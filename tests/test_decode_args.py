"""`enceladus.decode`: what its operators refuse, before anything is launched (CPU)."""

import numpy as np
import pytest
import torch

import enceladus
from enceladus import decode


def _attend(**kw):
    d = dict(q=torch.zeros(3, 8, 64), k_cache=torch.zeros(10, 16, 2, 64),
             v_cache=torch.zeros(10, 16, 2, 64),
             block_table=torch.zeros(3, 4, dtype=torch.int32),
             seq_lens=torch.ones(3, dtype=torch.int32))
    d.update(kw)
    return d.pop("q"), d.pop("k_cache"), d.pop("v_cache"), d.pop("block_table"), \
        d.pop("seq_lens"), d


def _append(**kw):
    d = dict(k=torch.zeros(3, 2, 64), v=torch.zeros(3, 2, 64),
             k_cache=torch.zeros(10, 16, 2, 64), v_cache=torch.zeros(10, 16, 2, 64),
             block_table=torch.zeros(3, 4, dtype=torch.int32),
             seq_lens=torch.ones(3, dtype=torch.int32))
    d.update(kw)
    return tuple(d.pop(n) for n in ("k", "v", "k_cache", "v_cache", "block_table",
                                    "seq_lens")) + (d,)


def _f8(*shape):
    return torch.zeros(*shape).to(torch.float8_e4m3fn)


ATTEND = [
    (dict(q=torch.zeros(3, 8, 64, dtype=torch.float64)), TypeError, "`q` must hold"),
    (dict(q=[1.0]), TypeError, "must be an array"),
    (dict(q=torch.zeros(3, 512)), ValueError, "3 dimensions"),
    (dict(q=torch.zeros(3, 64, 8).transpose(1, 2)), ValueError, "contiguous"),
    (dict(q=torch.zeros(3, 7, 64)), ValueError, "not a multiple"),
    (dict(q=torch.zeros(3, 8, 64).half()), TypeError, "`k_cache` must hold"),
    (dict(k_cache=torch.zeros(10, 16, 2, 32)), ValueError, "`k_cache` must have shape"),
    (dict(v_cache=torch.zeros(10, 8, 2, 64)), ValueError, "`v_cache` must have shape"),
    (dict(v_cache=torch.zeros(10, 2, 16, 64).transpose(1, 2)), ValueError, "same strides"),
    (dict(v_cache=torch.zeros(10, 16, 2, 64).half()), TypeError, "`v_cache` must hold"),
    (dict(k_cache=torch.zeros(10, 0, 2, 64), v_cache=torch.zeros(10, 0, 2, 64)), ValueError,
     "at least one token"),
    (dict(k_cache=torch.zeros(10, 16, 0, 64), v_cache=torch.zeros(10, 16, 0, 64)), ValueError,
     "key heads"),
    (dict(k_cache=_f8(10, 16, 2, 64)), ValueError, "host"),
    (dict(block_table=torch.zeros(3, 4, dtype=torch.int64)), TypeError, "`block_table`"),
    (dict(block_table=torch.zeros(2, 4, dtype=torch.int32)), ValueError, "`block_table`"),
    (dict(block_table=torch.zeros(3, 1 << 26, dtype=torch.int32)[:, ::1],
          k_cache=torch.zeros(1, 32, 2, 64), v_cache=torch.zeros(1, 32, 2, 64)), ValueError,
     "at most"),
    (dict(q=torch.zeros(1, 8, 64).expand(1 << 16, 8, 64),
          block_table=torch.zeros(1, 1 << 15, dtype=torch.int32).expand(1 << 16, 1 << 15),
          seq_lens=torch.zeros(1, dtype=torch.int32).expand(1 << 16)), ValueError, "in all"),
    (dict(q=torch.zeros(1, 8, 64).expand((1 << 16) + 1, 8, 64),
          block_table=torch.zeros(1, 4, dtype=torch.int32).expand((1 << 16) + 1, 4),
          seq_lens=torch.zeros(1, dtype=torch.int32).expand((1 << 16) + 1)), ValueError,
     "65536 sequences"),
    (dict(seq_lens=torch.ones(4, dtype=torch.int32)), ValueError, "`seq_lens`"),
    (dict(seq_lens=np.ones(3, np.float32)), TypeError, "`seq_lens`"),
    (dict(seq_lens=np.ones(3, np.int32)[::-1]), ValueError, "negative strides"),
    (dict(window=-1), ValueError, "window"),
    (dict(window=1.5), TypeError, "integer"),
    (dict(softcap=-1.0), ValueError, "softcap"),
    (dict(softcap=float("nan")), ValueError, "softcap"),
    (dict(scale=float("inf")), ValueError, "scale"),
    (dict(k_scale=0.0), ValueError, "k_scale"),
    (dict(k_scale=1e-30), ValueError, "k_scale"),
    (dict(scale=1e30), ValueError, "scale"),
    (dict(scale=float("nan")), ValueError, "scale"),
    (dict(softcap=1e-30), ValueError, "softcap"),
    (dict(q=torch.zeros(3, 8, 64, device="meta")), ValueError, "dense tensor"),
    (dict(q=torch.zeros(3, 8, 64).to_sparse()), ValueError, "dense tensor"),
    (dict(k_cache=torch.zeros(1, 1, 2, 64).expand(1 << 31, 1, 2, 64),
          v_cache=torch.zeros(1, 1, 2, 64).expand(1 << 31, 1, 2, 64)), ValueError, "32-bit"),
    (dict(q=torch.zeros(1, 8, 64).expand(1 << 21, 8, 64),
          block_table=torch.zeros(1, 4, dtype=torch.int32).expand(1 << 21, 4),
          seq_lens=torch.zeros(1, dtype=torch.int32).expand(1 << 21)), ValueError, "sequences"),
    (dict(v_scale=float("nan")), ValueError, "v_scale"),
    (dict(out=torch.zeros(3, 8, 32)), ValueError, "`out`"),
    (dict(out=torch.zeros(3, 8, 64).half()), TypeError, "`out`"),
    (dict(out=torch.zeros(3, 1, 64).expand(3, 8, 64)), ValueError, "expanded"),
    (dict(q=np.zeros((3, 8, 12), np.float32), k_cache=np.zeros((4, 4, 2, 12), np.float32),
          v_cache=np.zeros((4, 4, 2, 12), np.float32)), ValueError, "head dimension"),
    (dict(q=np.zeros((3, 8, 264), np.float32), k_cache=np.zeros((4, 4, 2, 264), np.float32),
          v_cache=np.zeros((4, 4, 2, 264), np.float32)), ValueError, "head dimension"),
]


@pytest.mark.parametrize("change,error,text", ATTEND)
def test_paged_attention_refuses(change, error, text):
    *args, kw = _attend(**change)
    with pytest.raises(error, match=text):
        decode.paged_attention(*args, **kw)


def test_paged_attention_refuses_overlap():
    buf = torch.zeros(4 * 8 * 64)
    q, out = buf[:3 * 512].view(3, 8, 64), buf[512:].view(3, 8, 64)
    *args, _ = _attend(q=q)
    with pytest.raises(ValueError, match="`out` overlaps `q`"):
        decode.paged_attention(*args, out=out)
    *args, kw = _attend()
    with pytest.raises(ValueError, match="overlaps `v_cache`"):
        decode.paged_attention(*args, out=args[2].view(-1)[:1536].view(3, 8, 64))


APPEND = [
    (dict(cu_tokens=torch.zeros(1, dtype=torch.int32).expand((1 << 25) + 2)), ValueError,
     "sequences are supported"),
    (dict(k=torch.zeros(3, 2, 64, dtype=torch.int32)), TypeError, "`k` must hold"),
    (dict(v=torch.zeros(3, 2, 32)), ValueError, "`v` must have shape"),
    (dict(k_cache=torch.zeros(10, 16, 3, 64)), ValueError, "`k_cache`"),
    (dict(k_cache=torch.zeros(10, 16, 2, 64).half()), TypeError, "`k_cache`"),
    (dict(k_cache=torch.zeros(1, 16, 2, 64).expand(10, 16, 2, 64),
          v_cache=torch.zeros(1, 16, 2, 64).expand(10, 16, 2, 64)), ValueError, "expanded"),
    (dict(seq_lens=torch.ones(2, dtype=torch.int32)), ValueError, "seq_lens"),
    (dict(cu_tokens=torch.zeros(3, dtype=torch.int32)), ValueError, "block_table"),
    (dict(cu_tokens=torch.zeros(4)), TypeError, "cu_tokens"),
    (dict(cu_tokens=torch.zeros(0, dtype=torch.int32)), ValueError, "cu_tokens"),
    (dict(cos=torch.zeros(8, 32)), ValueError, "go together"),
    (dict(cos=torch.zeros(8, 32), sin=torch.zeros(8, 16)), ValueError, "`sin`"),
    (dict(cos=torch.zeros(8, 33), sin=torch.zeros(8, 33)), ValueError, "rotates 66"),
    (dict(cos=torch.zeros(8, 0), sin=torch.zeros(8, 0)), ValueError, "rotates 0"),
    (dict(cos=torch.zeros(8, 32).half(), sin=torch.zeros(8, 32).half()), TypeError, "`cos`"),
    (dict(q=torch.zeros(2, 8, 64)), ValueError, "`q`"),
    (dict(q=torch.zeros(3, 8, 64).half()), TypeError, "`q`"),
    (dict(q_out=torch.zeros(3, 8, 64)), ValueError, "without `q`"),
    (dict(q=torch.zeros(3, 8, 64), q_out=torch.zeros(3, 4, 64)), ValueError, "`q_out`"),
    (dict(k_scale=-1.0), ValueError, "k_scale"),
    (dict(k=torch.zeros(1, 2, 64).expand(1 << 26, 2, 64)), ValueError, "tokens"),
]


@pytest.mark.parametrize("change,error,text", APPEND)
def test_append_kv_refuses(change, error, text):
    *args, kw = _append(**change)
    with pytest.raises(error, match=text):
        decode.append_kv(*args, **kw)


def test_overlap_of_rows_side_by_side():
    wide = torch.zeros(3, 100)
    arr = {n: decode._Array(n, x) for n, x in (("a", wide[:, :40]), ("b", wide[:, 40:100]),
                                               ("c", wide[:, 39:60]), ("d", wide[1:, :40]),
                                               ("e", wide.view(-1)[95:215].view(3, 40)))}
    for x, y in ("ab", "ba", "db", "bd"):
        decode._apart(x, arr[x], y, arr[y])
    for x, y in ("ac", "ca", "bc", "cb", "ad", "da", "be", "eb", "ae"):
        with pytest.raises(ValueError, match="overlaps"):
            decode._apart(x, arr[x], y, arr[y])


def test_append_kv_refuses_overlap_and_read_only():
    rows = torch.zeros(4, 8, 64)
    *args, _ = _append()
    with pytest.raises(ValueError, match="`q_out` overlaps `q`"):
        decode.append_kv(*args, q=rows[:3], q_out=rows[1:])
    *args, _ = _append()
    args[3] = args[2]
    with pytest.raises(ValueError, match="are the same"):
        decode.append_kv(*args)
    *args, _ = _append()
    with pytest.raises(ValueError, match="`q_out` overlaps `v_cache`"):
        decode.append_kv(*args, q=rows[:3], q_out=args[3].view(-1)[64:64 + 1536].view(3, 8, 64))
    cache = np.zeros((10, 16, 2, 64), np.float32)
    cache.flags.writeable = False
    *args, _ = _append(k_cache=cache)
    with pytest.raises(ValueError, match="read-only"):
        decode.append_kv(*args)


@pytest.mark.parametrize("views,apart", [
    (lambda x: (x[:, 0], x[:, 1]), True),                      # [pages, 2, page, heads, dim]
    (lambda x: (x[:, 1], x[:, 0]), True),
    (lambda x: (x[0::2, 0], x[1::2, 0]), True),
    (lambda x: (x.view(10, 16, 2, 2, 64)[:, :, 0], x.view(10, 16, 2, 2, 64)[:, :, 1]), True),
    (lambda x: (x.view(10, 16, 2, 128)[..., 64:], x.view(10, 16, 2, 128)[..., :64]), True),
    (lambda x: (x.view(10, 16, 4, 64)[:, :, ::2], x.view(10, 16, 4, 64)[:, :, 1::2]), True),
    (lambda x: (x[:, 0], x[:, 0]), False),
    (lambda x: (x[:-1, 0], x[1:, 0]), False),
    (lambda x: (x[:-1, 1], x[1:, 0]), True),
    (lambda x: (x[:, 0, :, :1], x[:, 0, :, 1:]), True),
    (lambda x: (x[:, 0, :-1], x[:, 0, 1:]), False),
    (lambda x: (x[:, 0, :8], x[:, 0, 8:]), True),
    (lambda x: (x.view(10, 16, 2, 128)[..., :64], x.view(10, 16, 2, 128)[..., 63:127]), False),
    (lambda x: (x.view(10, 16, 2, 128)[..., 8:72], x.view(10, 16, 2, 128)[..., :64]), False),
])
@pytest.mark.parametrize("kind", ["torch", "numpy"])
def test_append_kv_refuses_caches_that_share_memory(views, apart, kind):
    """Caches inside one array: taken where no element is both's. (A `q` without work: nothing is
    launched.)"""
    k, v = views(torch.zeros(10, 2, 16, 2, 64))
    if kind == "numpy":
        k, v = k.numpy(), v.numpy()
    heads = k.shape[2]
    new = torch.zeros(0, heads, 64)
    args = (new, new, k, v, torch.zeros(0, 4, dtype=torch.int32), torch.zeros(0, dtype=torch.int32))
    if apart:
        assert decode.append_kv(*args) is None
    else:
        with pytest.raises(ValueError, match="overlaps `v_cache`|are the same"):
            decode.append_kv(*args)


def test_arrays_that_meet_by_their_strides():
    """Against the sets of their elements' places."""
    rng = np.random.default_rng(1)
    for _ in range(300):
        shape = tuple(int(n) for n in rng.integers(1, 5, 3))
        strides = [int(s) for s in rng.integers(1, 30, 3)]
        a = decode._Array("a", torch.zeros(300).as_strided(shape, strides))
        places = {int(np.dot(i, strides)) for i in np.ndindex(*shape)}
        for gap in range(-60, 61, 7):
            want = any(p + gap in places for p in places)
            assert decode._meet(decode._steps(a), 4, 4 * gap) == want, (shape, strides, gap)


LOGITS = [
    (dict(logits=torch.zeros(3, 100, dtype=torch.int32)), TypeError, "`logits`"),
    (dict(logits=torch.zeros(300)), ValueError, "2 dimensions"),
    (dict(logits=torch.zeros(100, 3).t()), ValueError, "contiguous"),
    (dict(tokens=torch.zeros(2, 5, dtype=torch.int32)), ValueError, "`tokens`"),
    (dict(tokens=torch.zeros(3, 5, dtype=torch.int64)), TypeError, "`tokens`"),
    (dict(tokens=torch.zeros(3, 5, dtype=torch.int32),
          token_lens=torch.zeros(2, dtype=torch.int32)), ValueError, "`token_lens`"),
    (dict(repetition=1.2), ValueError, "need the history"),
    (dict(token_lens=torch.zeros(3, dtype=torch.int32)), ValueError, "need the history"),
    (dict(tokens=torch.zeros(3, 5, dtype=torch.int32), repetition=0.0), ValueError, "repetition"),
    (dict(tokens=torch.zeros(3, 5, dtype=torch.int32), repetition=1e39), ValueError, "repetition"),
    (dict(temperature=1e-40), ValueError, "temperature"),
    (dict(temperature=1e-60), ValueError, "temperature"),
    (dict(temperature=float("nan")), ValueError, "temperature"),
    (dict(tokens=torch.zeros(3, 5, dtype=torch.int32), repetition=torch.zeros(2)), ValueError,
     "`repetition`"),
    (dict(temperature=torch.zeros(3).half()), TypeError, "`temperature`"),
    (dict(bias=torch.zeros(3, 5)), ValueError, "go together"),
    (dict(bias=torch.zeros(3, 5), bias_ids=torch.zeros(3, 4, dtype=torch.int32)), ValueError,
     "`bias`"),
    (dict(bias=torch.zeros(3, 1024), bias_ids=torch.zeros(3, 1024, dtype=torch.int32)),
     ValueError, "at most 1023"),
    (dict(tokens=torch.zeros(3, 1 << 21, dtype=torch.int32)), ValueError, "at most 2097151"),
    (dict(allowed=torch.zeros(3, 3, dtype=torch.int32)), ValueError, "need 4"),
    (dict(allowed=torch.zeros(3, 4, dtype=torch.int64)), TypeError, "`allowed`"),
    (dict(out=torch.zeros(3, 99)), ValueError, "`out`"),
    (dict(logits=torch.zeros(1, 100).expand(1 << 22, 100),
          out=torch.zeros(1, 100).expand(1 << 22, 100)), ValueError, "expanded"),
    (dict(out=torch.zeros(3, 1).expand(3, 100)), ValueError, "contiguous|expanded"),
]


@pytest.mark.parametrize("change,error,text", LOGITS)
def test_adjust_logits_refuses(change, error, text):
    kw = dict(logits=torch.zeros(3, 100))
    kw.update(change)
    with pytest.raises(error, match=text):
        decode.adjust_logits(kw.pop("logits"), **kw)


def test_calls_without_work_launch_nothing():
    *args, kw = _attend(q=torch.zeros(0, 8, 64), seq_lens=torch.ones(0, dtype=torch.int32),
                        block_table=torch.zeros(0, 4, dtype=torch.int32))
    assert decode.paged_attention(*args, **kw).shape == (0, 8, 64)
    *args, kw = _append(k=torch.zeros(0, 2, 64), v=torch.zeros(0, 2, 64),
                        seq_lens=torch.ones(0, dtype=torch.int32),
                        block_table=torch.zeros(0, 4, dtype=torch.int32))
    assert decode.append_kv(*args, **kw) is None
    assert decode.adjust_logits(torch.zeros(0, 50)).shape == (0, 50)
    assert decode.adjust_logits(torch.zeros(3, 0)).shape == (3, 0)


def test_page_division_is_exact():
    """The multiplier that replaces the division by the page size, over all its uses: quotients
    of positions below 2^30."""
    rng = np.random.default_rng(0)
    for page in [1, 2, 3, 5, 7, 8, 16, 24, 31, 64, 100, 127, 128, 1000, 4097, (1 << 29) - 1]:
        mul, shift = decode._page_division(page)
        assert 0 <= mul < 1 << 32
        n = np.concatenate([rng.integers(0, 1 << 30, 20000), np.arange(5000),
                            np.arange(1, 200) * page % (1 << 30),
                            np.arange(1, 200) * page % (1 << 30) - 1,
                            [(1 << 30) - 1]]).astype(object)
        got = [int(x) if page == 1 else (int(x) * mul >> 32) >> shift for x in n]
        assert got == [int(x) // page for x in n], page


def test_module_is_public():
    assert enceladus.decode is decode
    for name in decode.__all__:
        assert getattr(decode, name).__doc__


def test_settings_of_any_number_type():
    """NumPy scalars and tensors of one value count as numbers; a tensor's later value is seen."""
    for one in (1, True, np.float32(1.0), torch.tensor(1.0), torch.tensor(0.5)):
        *args, _ = _attend(q=torch.zeros(3, 7, 64))
        with pytest.raises(ValueError, match="not a multiple"):
            decode.paged_attention(*args, scale=one, k_scale=one)
        with pytest.raises(TypeError, match="`logits`"):
            decode.adjust_logits(torch.zeros(3, 10, dtype=torch.int8),
                                 temperature=one if one.__class__ is not torch.Tensor else 1)
    *args, _ = _attend()
    with pytest.raises(ValueError, match="k_scale"):
        decode.paged_attention(*args, k_scale=torch.tensor(-1.0))
