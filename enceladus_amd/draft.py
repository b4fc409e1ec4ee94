"""The operators that check drafted tokens over a paged key-value cache, as hand-written HIP
kernels.

    q = decode.append_kv(k, v, k_cache, v_cache, block_table, seq_lens, cu_tokens=cu, q=q,
                         cos=cos, sin=sin, positions=positions)
    o = draft.tree_attention(q, k_cache, v_cache, block_table, seq_lens, cu, tree=tree)
    path, count, token = draft.accept(logits, tokens, cu, tree=tree)
    pages.compact(caches, block_table, past, path, count, seq_lens=seq_lens)

(`pages.take` gives the slots before, and says of which rows the new tokens have none: a length of 0
here and a negative `past` keep such a row out.)

Each of `batch` sequences has some new tokens in a row: the last one that was chosen, and drafted
ones that may follow it. Sequence b's are the rows `cu_tokens[b]` to `cu_tokens[b + 1]`, and its
last ones in the cache. `tree` (int32 `[tokens, words]`) says which of them a token sees: bit j % 32
of word j // 32 of its row is its sequence's j-th new token; a token sees itself and its ancestors,
and what was there before the new tokens. Without it they are a chain, each seeing those before it.

Arrays, streams, captures and errors are as in `enceladus.decode`: one device, its current stream,
nothing waits; a call inside a capture needs one before it. There are no gradients.
"""

from __future__ import annotations

import math
import operator
import struct

import numpy as np

from enceladus_amd import decode as _d
from enceladus_amd.runtime import compile as C
from enceladus_amd.runtime import tensor as T

__all__ = ["tree_attention", "accept"]

MAX_NODES = 1024                    # of a tree, in `accept`


def _rows(cu_tokens) -> _d._Array:
    cu = _d._array("cu_tokens", cu_tokens, ("i32",), 1, dense=False)
    _d._need(cu.shape[0] > 0, "`cu_tokens` must have one entry more than there are sequences")
    return cu


def _tree(tree, tokens: int):
    if tree is None:
        return None
    a = _d._array("tree", tree, ("i32",), 2, (tokens, None))
    _d._need(a.shape[1] > 0, "`tree` must have at least one word for each token")
    _d._need(a.shape[1] <= 1 << 20, f"`tree` may have at most {1 << 20} words, got {a.shape[1]}")
    return a


# -- attention -------------------------------------------------------------------------------

_ATTEND = struct.Struct("<11q11iI5iI3f4x")
_UNIT = 64                          # tokens: what a sequence is split in multiples of


def tree_attention(q, k_cache, v_cache, block_table, seq_lens, cu_tokens, *, tree=None,
                   scale: float | None = None, window: int = 0, softcap: float = 0.0,
                   k_scale: float = 1.0, v_scale: float = 1.0, out=None,
                   return_lse: bool = False):
    """Attention of several new tokens per sequence over a paged cache (which holds their own keys
    and values already).

    Token i of the n new ones of sequence b sees the slots before `seq_lens[b] - n` and, of the new
    tokens j, at slot `seq_lens[b] - n + j`, those whose bit is set in its row of `tree` (without
    `tree`: j <= i). Of what it sees only the last `window`, in the order of their slots, count
    when that is above 0 (slots on a page outside the cache are counted among them). For these and
    query head h: s_j = `scale` * q . k_j, made `softcap` * tanh(s_j / `softcap`) when that is above
    0; the result is the sum of softmax(s)_j v_j. Scores, weights and sums have 32 bits; where the
    cache is float16 or float8, a weight is rounded by up to 2^-20 of it before its product. Heads
    are shared as in `decode.paged_attention`. A token that sees nothing, or no score above -inf,
    gives zeros. Tokens on a page outside the cache, beyond the block table or before the sequence's
    first (new ones, where there are more of them than tokens) count as absent. Cache memory that no
    sequence's length reaches may hold anything, NaN included; a value that is not finite reaches
    the tokens that see it alone, whose elements it makes infinite or NaN. Rows of no sequence (padding behind the last, or before the first) are skipped: `out`
    is not written for them (a new one holds anything there).

    Args:
        q: `[tokens, heads, dim]`, float32, float16 or bfloat16; `dim` a multiple of 8 up to 256
            (of 16 with a float8 cache).
        k_cache, v_cache: `[pages, page size, key heads, dim]` of the type of `q`, or
            float8_e4m3fn (not with float32).
        block_table: int32 `[batch, pages of a sequence]`.
        seq_lens: int32 `[batch]`, counting the new tokens; at most 65536 sequences.
        cu_tokens: int32 `[batch + 1]`, not descending.
        tree: int32 `[tokens, words]`; new tokens without a bit in it are seen by none.
        scale: of the scores; 1 / sqrt(dim) without it.
        k_scale, v_scale: what cached values are multiplied by.
        out: where the result goes (`q` itself will do); new without it.
        return_lse: also return the log of each head's sum of exp(s_j), float32 `[tokens, heads]`
            (-inf where nothing is seen).

    Returns:
        The result, `[tokens, heads, dim]` of the type of `q`; `(result, lse)` when `return_lse`.
    """
    # plain numbers from here on: a plan is kept by their values
    scale = None if scale is None else float(scale)
    window, softcap = operator.index(window), float(softcap)
    k_scale, v_scale = float(k_scale), float(v_scale)
    try:
        of = _d._of
        key = (8, of(q), of(k_cache), of(v_cache), of(block_table), of(seq_lens), of(cu_tokens),
               None if tree is None else of(tree), None if out is None else of(out), scale, window,
               softcap, k_scale, v_scale)
        plan = _d._plans.get(key)
    except (AttributeError, TypeError, RuntimeError):
        key = plan = None              # arrays of another kind, or no arrays
    given = out is not None
    if plan is None:
        plan, out = _attention_plan(q, k_cache, v_cache, block_table, seq_lens, cu_tokens, tree,
                                    scale, window, softcap, k_scale, v_scale, out)
        if plan is not None:
            _d._keep(key, plan)
    elif not given:
        out = _d._like(q)
    lse = T.new_empty(q, tuple(q.shape[:2]), np.float32) if return_lse else None
    if plan is not None:
        arrays = [q, k_cache, v_cache, block_table, seq_lens, cu_tokens, tree, out, lse]
        if given:
            plan.check_apart(arrays)
        plan.run(arrays)
    return (out, lse) if return_lse else out


def _shape(columns: float, width: int, size: int) -> tuple[int, int, int, int, int, int]:
    """(keys of a stage, columns of a tile, tiles of a wave, waves over columns, waves over keys,
    workgroups of a CU) for sequences of so many columns of a key head, in heads of `width` cached
    elements of `size` bytes.

    Stages of 16 KB each of keys and values leave the LDS to two workgroups. As many columns as
    there are, in fewer waves and tiles, or else the keys are read again: 8 sequences of up to
    16384, 8 key heads of 128 in bf16, in tiles of 16 by 1 wave, of 16 by 2, of 32 by 2 and of 32 by 4: 11.5
    columns 30.7, 31.6, 36.1, 41.6 us; 27 columns 47.3, 32.6, 37.2, 42.9; 52 columns 74.8, 48.0,
    40.3, 46.3; 111.5 columns 147, 79.0, 58.9, 52.9. Heads of 64 in e4m3 cannot be read in tiles of
    32: two of 16 (111.5 columns 38.3 us, 47.4 in single ones by 2). Heads of 256 and fp32 have no
    registers for either: 52 columns (up to 8192 tokens) by 4 waves 52.3 and 80.3 us, by 2 74.7 and
    99.2; 11.5 columns 46.1 and 76.3, 43.7 and 54.5.
    """
    keys = max(16, min(64, 16384 // (width * size)))
    if size == 4 or width == 256:
        over = 1
        while over < 4 and (columns > 16 * over or keys < 64 // over):
            over *= 2
        return keys, 16, 1, over, 4 // over, 1 if width * size == 1024 else 2
    if columns <= 32:
        # 94 to 113 registers at 64 elements; 129 to 152 at 128, of which only the 8-bit ones'
        # stages leave the LDS to a third workgroup
        at_once = 4 if width == 64 else 3 if size == 1 else 2
        return (keys, 16, 1, 1, 4, at_once) if columns <= 16 else (keys, 16, 1, 2, 2, at_once)
    over = 2 if columns <= 64 else 4
    at_once = 3 if width == 64 and (size == 2 or over == 2) else 2
    return (keys, 16, 2, over, 4 // over, at_once) if width * size == 64 else \
        (keys, 32, 1, over, 4 // over, at_once)


def _macros(q: int, fp8: bool, width: int, pad: bool, shape) -> tuple:
    names = ("EK_Q", "EK_FP8", "EK_DP", "EK_PAD", "EK_KT", "EK_TILE", "EK_CT", "EK_WC", "EK_WK",
             "EK_OCC")
    return tuple(zip(names, (q, int(fp8), width, int(pad), *shape)))


def _attention_plan(q, k_cache, v_cache, block_table, seq_lens, cu_tokens, tree, scale, window,
                    softcap, k_scale, v_scale, out):
    """The checked call's plan (None: nothing to do) and its `out`."""
    need = _d._need
    qa = _d._array("q", q, ("fp32", "fp16", "bf16"), 3)
    tokens, heads, dim = qa.shape
    need(tokens <= 1 << 23, f"at most {1 << 23} tokens are supported, got {tokens}")
    kc, vc = _d._caches(k_cache, v_cache, None, dim,
                        (qa.kind,) if qa.kind == "fp32" else (qa.kind, "fp8"))
    kv_heads = kc.shape[2]
    _d._head_dim(dim, kc.kind)
    need(kv_heads > 0 and heads % kv_heads == 0,
         f"{heads} query heads are not a multiple of {kv_heads} key heads")
    group = heads // kv_heads
    need(tokens * group < 1 << 30, f"{tokens} tokens of {group} heads of a key head are too many "
                                   "for one call")
    cu = _rows(cu_tokens)
    batch = cu.shape[0] - 1
    need(heads <= 65535 and batch <= 1 << 16,
         f"at most 65535 query heads and {1 << 16} sequences are supported, got {heads}, {batch}")
    bt, sl = _d._sequences(block_table, seq_lens, batch)
    ta = _tree(tree, tokens)
    capacity = _d._capacity(bt, kc)
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    need(abs(scale) <= _d._SCALES[1], f"`scale` must be at most 2^60, got {scale}")
    need(softcap == 0 or _d._SCALES[0] <= softcap <= _d._SCALES[1],
         f"`softcap` must be 0 or from 2^-60 to 2^60, got {softcap}")
    need(window >= 0, f"`window` must be at least 0, got {window}")
    _d._positive("k_scale", k_scale)
    _d._positive("v_scale", v_scale)
    if out is None:
        out = T.new_empty(q)
    oa = _d._array("out", out, (qa.kind,), 3, qa.shape)
    _d._written("out", oa)
    arrays = [("q", qa), ("k_cache", kc), ("v_cache", vc), ("block_table", bt),
              ("seq_lens", sl), ("cu_tokens", cu), ("tree", ta), ("out", oa), ("lse", None)]
    _d._device_of(arrays)
    if batch == 0 or heads == 0 or tokens == 0:
        return None, out
    if kc.shape[0] == 0:
        capacity = 0
    window = min(window, _d.MAX_TOKENS)
    width = 64 if dim <= 64 else 128 if dim <= 128 else 256
    shape = _shape(tokens / batch * group, width, kc.size)
    _, tile, tiles, over, split, at_once = shape
    cols = tile * tiles * over
    waves = over * split
    # blocks of columns: each sequence may have one that is not whole
    blocks = -(-tokens * group // cols) if batch == 1 else tokens * group // cols + \
        min(batch, tokens)
    most = -(-capacity // _UNIT)
    if window:
        most = min(most, -(-(window + tokens) // _UNIT))
    need(blocks * max(most, 1) < 1 << 31, f"{tokens} tokens over tables of {capacity} tokens are "
                                          "too many for one call")
    items = max(1, at_once * C.coarsen_cap() // kv_heads)
    # A chunk for every block besides their even shares, and no more than there are units. Room for
    # two rounds of them is there if the blocks are as many as fit at once (workgroups that find
    # nothing to do cost 1 us and more: there are none for its sake).
    x = min(items + blocks, blocks * max(most, 1))
    rounds = 2 if x >= 2 * items else 1
    need(x * 64 * waves < 1 << 32 and kv_heads <= 65535, f"{tokens} tokens are too many for one "
                                                         "call")
    macros = _macros(_d._Q[qa.kind], kc.kind == "fp8", width, dim != width, shape)
    launches = [("ek_tree_attention", (x, kv_heads), 64 * waves)]
    slots = workspace = 0
    join = 1
    # one sequence of as many blocks as there are items has one chunk
    if most > 1 and not (batch == 1 and blocks >= items):
        slots = min(2 * items, x)      # each is a workgroup's
        workspace = slots * kv_heads * cols * (dim + 2) * 4 + 16 * tokens
        # four waves for a token's head where it may have many chunks, one for four heads where it
        # will hardly have more than four
        join = 0 if min(items // blocks, most) > 16 else 4 if rounds * items <= 4 * blocks else 1
        launches.append(("ek_tree_attention_join",
                         (tokens, heads if join == 0 else -(-heads // (4 * join))), 256))
    log2e = 1.4426950408889634
    tail = _ATTEND.pack(
        qa.strides[0], qa.strides[1], oa.strides[0], oa.strides[1],
        *(s * kc.size for s in kc.strides[:3]), bt.strides[0], sl.strides[0], cu.strides[0],
        ta.strides[0] if ta else 0, tokens, batch, heads, kv_heads, group, dim, kc.shape[1],
        kc.shape[0], capacity, window, ta.shape[1] if ta else 0, *_d._page_division(kc.shape[1]),
        items, rounds, slots, join,
        0 if scale >= 0 else 0x80000000 if qa.kind == "fp32" else 0x80008000,
        # so small a scale is as good as none, and keeps -inf (no key there) what it is
        max(abs(scale) * k_scale * log2e, 2.0 ** -126), softcap * log2e, v_scale)
    if not workspace:
        tail = bytes(8) + tail         # the address of the partial results
    return _d._Plan("tree_attention.hip", macros, launches, arrays, {7, 8}, workspace, tail,
                    [(7, 0, True), (7, 1, False), (7, 2, False), (7, 6, False)]), out


# -- acceptance --------------------------------------------------------------------------------

_ACCEPT = struct.Struct("<4q7i4x")


def accept(logits, tokens, cu_tokens, *, tree=None, most: int | None = None):
    """Follows each sequence's drafted tokens as far as they are what the model would choose.

    A token's choice is the place of its row's largest logit (the lowest such place; NaN counts as
    larger than any number). A sequence's walk begins at its first new token, which was chosen
    before; from a token it goes on to the first of its children that is its choice, until there
    is none. A child is a token that sees it and one token more than it does. A chain's only child
    is the next token. Choices of other kinds are made by what is added to the logits before, for
    instance noise to sample.

    Args:
        logits: `[tokens, vocabulary]`, float32, float16 or bfloat16.
        tokens: the new tokens' ids, int32 `[tokens]`.
        cu_tokens: int32 `[batch + 1]`, not descending.
        tree: int32 `[tokens, words]`, at most 32 words; new tokens without a bit in it take no
            part.
        most: the longest path; without it as many as `tree` has bits, or as there are tokens.

    Returns:
        `(path, count, token)`, int32 `[batch, most]`, `[batch]` and `[batch]`: which of its new
        tokens a sequence's walk went through, the first (0) included, and -1 behind them; how
        many; and the choice of the last. 0 and -1 for a sequence without new tokens.
    """
    if most is not None:
        most = operator.index(most)
    try:
        of = _d._of
        key = (9, of(logits), of(tokens), of(cu_tokens), None if tree is None else of(tree), most)
        plan = _d._plans.get(key)
    except (AttributeError, TypeError, RuntimeError):
        key = plan = None              # arrays of another kind, or no arrays
    if plan is None:
        plan = _accept_plan(logits, tokens, cu_tokens, tree, most)
        _d._keep(key, plan)
    shapes = (plan.batch, plan.most), (plan.batch,), (plan.batch,)
    if plan.on_gpu:
        new = [cu_tokens.new_empty(shape) for shape in shapes]
    else:
        new = [T.new_empty(cu_tokens, shape, np.int32) for shape in shapes]
    if plan.launches:
        plan.run([logits, tokens, cu_tokens, tree, *new])
    return tuple(new)


_BEST_THREADS, _BEST_UNROLL = 256, 8     # of a workgroup of accept.hip


def _accept_plan(logits, tokens, cu_tokens, tree, most):
    need = _d._need
    la = _d._array("logits", logits, ("fp32", "fp16", "bf16"), 2)
    rows, vocab = la.shape
    to = _d._array("tokens", tokens, ("i32",), 1, (rows,), dense=False)
    cu = _rows(cu_tokens)
    batch = cu.shape[0] - 1
    ta = _tree(tree, rows)
    need(ta is None or ta.shape[1] * 32 <= MAX_NODES,
         f"trees of at most {MAX_NODES} tokens are supported, got {ta.shape[1] if ta else 0} words")
    need(0 < vocab < 1 << 30, f"rows of 1 to 2^30 logits are supported, got {vocab}")
    need(batch < 1 << 24 and rows < 1 << 24, f"at most {(1 << 24) - 1} sequences and tokens are "
                                             f"supported, got {batch} and {rows}")
    if most is None:
        most = ta.shape[1] * 32 if ta else rows
    need(0 <= most and batch * most < 1 << 40, f"`most` must be at least 0, got {most}")
    most = min(most, (1 << 31) - 1)
    arrays = [("logits", la), ("tokens", to), ("cu_tokens", cu), ("tree", ta), ("path", None),
              ("count", None), ("token", None)]
    _d._device_of(arrays)
    # stretches of a row: whole rounds of a workgroup's loads, fewer where CUs are without one
    vector = _BEST_THREADS * 16 // la.size
    span = vector * _BEST_UNROLL
    while span > vector and rows * -(-vocab // span) < 2 * C.coarsen_cap():
        span //= 2
    pieces = -(-vocab // span)
    need(rows * pieces < 1 << 24, f"logits of shape {la.shape} are too large for one call")
    launches = [("ek_accept", (batch, 1), _BEST_THREADS)] if batch else []
    if rows and batch:
        launches.insert(0, ("ek_row_best", (rows * pieces, 1), _BEST_THREADS))
    tail = _ACCEPT.pack(la.strides[0], to.strides[0], cu.strides[0], ta.strides[0] if ta else 0,
                        rows, vocab, batch, ta.shape[1] if ta else 0, most, pieces, span)
    plan = _d._Plan("accept.hip", (("EK_Q", _d._Q[la.kind]),), launches, arrays, {4, 5, 6},
                    8 * max(1, rows * pieces), tail)
    plan.batch, plan.most = batch, most
    return plan


def specializations():
    """(source, macros) of the kernels that are worth compiling ahead."""
    for q, fp8 in ((2, False), (1, False), (0, False), (2, True), (1, True)):
        size = 1 if fp8 else 2 if q else 4
        for width in (64, 128, 256):
            for shape in sorted({_shape(columns, width, size) for columns in (16, 32, 64, 128)}):
                for pad in (False, True) if size == 2 else (False,):
                    yield "tree_attention.hip", _macros(q, fp8, width, pad, shape)
    for q in (0, 1, 2):
        yield "accept.hip", (("EK_Q", q),)
