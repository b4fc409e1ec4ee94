"""The pages of paged key-value caches, kept on the GPU: copied, shared by several sequences, taken
and given back, and the tokens on them compacted, as hand-written HIP kernels.

    served = pages.take(refs, block_table, seq_lens, new_lens, page_size=16)
    held = seq_lens.clone()
    pages.compact(caches, block_table, torch.where(served > 0, starts, -1), keep, counts,
                  seq_lens=seq_lens)
    served = pages.fork(caches, refs, block_table, seq_lens, source, target)
    pages.free(refs, block_table, held, seq_lens, page_size=16)
    pages.copy(caches, source, target)

`caches` are the arrays `[pages, page size, key heads, head dimension]` of all layers, keys and
values alike (`enceladus.decode` has their form): a list of them, or one array with one more
dimension in front. They have one shape, one type and the same strides, and share no element; the
same pages of all of them move in one launch. `block_table` (int32 `[rows, pages of a sequence]`)
and `seq_lens` (int32 `[rows]`) are those of `enceladus.decode`. `refs` (int32 `[pages]`) counts
the sequences that hold each page: 0 is a free page, and one below 0 is never taken, nor changed
by any call, whichever rows hold it. What decides is on the device, where lengths and counts are, so
nothing waits for them and all of it can be captured: the order in which pages are taken is fixed
(the lowest free ones, by the rows in their order), so that the same calls give the same tables.

Arrays, streams, captures and errors are as in `enceladus.decode`. Ids outside of the cache or the
table are neither read nor written through, a negative length counts as none. `seq_lens`, `refs`
and `block_table` are written in place: calls that use the same ones go to one stream, or wait for
each other.
"""

from __future__ import annotations

import operator
import struct

import numpy as np

from enceladus_amd import decode as _d
from enceladus_amd.runtime import tensor as T

__all__ = ["copy", "compact", "fork", "take", "free"]

_PARAMS = struct.Struct("<8q10i")
_FILE = "pages.hip"
_THREADS, _COPY, _FORK = 256, 1, 8  # of a workgroup that copies, and its accesses: pages.hip
MAX_CACHES = 256                    # of a call: their addresses are kernel arguments
MAX_PAGES = (1 << 25) - 1           # sums over a wave's rows stay in 32 bits
MAX_BLOCKS = (1 << 24) - 1          # of 256 threads: a grid holds fewer than 2^32 threads


# -- arguments -----------------------------------------------------------------------------

def _listed(caches) -> list:
    """The caches as a list: of a list, of an array of them, or of one alone."""
    if isinstance(caches, (list, tuple)):
        return list(caches)
    if T.is_array_like(caches):
        if len(caches.shape) == 4:
            return [caches]
        _d._need(len(caches.shape) == 5, "`caches` must be arrays of 4 dimensions, or one of 5, "
                 f"got shape {tuple(caches.shape)}")
        return [caches[i] for i in range(caches.shape[0])]
    raise TypeError(f"`caches` must be arrays, got {type(caches).__name__}")


def _key(caches):
    """What a plan depends on of the caches; raises where they are none or differ (the checks of
    a new plan say how)."""
    if not isinstance(caches, (list, tuple)):
        return _d._of(caches)
    c = caches[0]
    dtype, shape, strides, device = _d._of(c)
    for x in caches:
        if x.dtype != dtype or x.shape != shape or x.stride() != strides or \
                x.get_device() != device:
            raise TypeError
    return len(caches), dtype, shape, strides, device


def _check_caches(caches: list) -> _d._Array:
    _d._need(0 < len(caches) <= MAX_CACHES,
             f"1 to {MAX_CACHES} caches are supported in a call, got {len(caches)}")
    first = None
    for i, x in enumerate(caches):
        a = _d._array(f"caches[{i}]", x, ("fp32", "fp16", "bf16", "fp8"), 4)
        first = first or a
        _d._need(a.kind == first.kind and a.shape == first.shape and
                 tuple(a.strides) == tuple(first.strides) and a.device == first.device,
                 f"`caches[{i}]` differs from the first in its type, shape, strides or device")
        _d._written(f"caches[{i}]", a)
    _d._need(0 < first.shape[1] <= _d.MAX_TOKENS,
             f"a page must hold at least one token, and at most {_d.MAX_TOKENS}")
    _d._need(first.shape[0] <= MAX_PAGES, f"at most {MAX_PAGES} pages are supported, got "
                                          f"{first.shape[0]}")
    _d._need(first.shape[1] * first.shape[2] * first.shape[3] * first.size < 1 << 31,
             "a page must be smaller than 2^31 bytes")
    return first


def _check_apart(plan, at: list) -> None:
    """Refuses caches that share elements, from their addresses. Whether two do goes by their
    distance alone, so what was found for one is kept."""
    span, at = plan.span, sorted(at)
    if min(map(operator.sub, at[1:], at)) >= span:
        return
    for i, p in enumerate(at):
        for q in at[i + 1:]:
            if q - p >= span:
                break
            meet = plan.gaps.get(q - p)
            if meet is None:
                if len(plan.gaps) > 4096:
                    plan.gaps.clear()
                meet = plan.gaps[q - p] = q == p or \
                    _d._meet(plan.steps, plan.element, q - p)
            _d._need(not meet, "two of `caches` share elements")


def _refs(refs, pages=None):
    a = _d._array("refs", refs, ("i32",), 1, (pages,))
    _d._written("refs", a)
    _d._need(a.shape[0] <= MAX_PAGES, f"at most {MAX_PAGES} pages are supported, got "
                                      f"{a.shape[0]}")
    return a


def _table(block_table, seq_lens, page: int, written=True):
    bt = _d._array("block_table", block_table, ("i32",), 2)
    sl = None
    if seq_lens is not None:
        sl = _d._array("seq_lens", seq_lens, ("i32",), 1, (bt.shape[0],), dense=False)
        _d._written("seq_lens", sl)
    if written:
        _d._written("block_table", bt)
    _d._need(0 < page <= _d.MAX_TOKENS, f"`page_size` must be from 1 to {_d.MAX_TOKENS}, got "
                                        f"{page}")
    _d._need(bt.shape[1] * page <= _d.MAX_TOKENS,
             f"`block_table` covers {bt.shape[1] * page} tokens of a sequence: at most "
             f"{_d.MAX_TOKENS} are supported")
    _d._need(bt.shape[0] <= 1 << 22, f"at most {1 << 22} rows are supported, got {bt.shape[0]}")
    return bt, sl


def _row_form(c: _d._Array) -> tuple:
    """(heads, bytes of a head's row, strides in bytes of pages, tokens and heads), heads that
    follow each other as one."""
    heads, row = c.shape[2], c.shape[3] * c.size
    page, token, head = (s * c.size for s in c.strides[:3])
    if heads <= 1 or head == row:
        heads, row, head = min(heads, 1), row * max(heads, 1), row * max(heads, 1)
    return heads, row, page, token, head


def _access(row: int) -> int:
    """Bytes of an access: up to 16, dividing a row."""
    return min(16, row & -row)


def _slots(count: int) -> int:
    """Addresses that the kernels' arguments have room for: a power of two."""
    return 1 << max(0, count - 1).bit_length()


def _pages_plan(launches, caches, arrays, written, workspace, numbers, access=16, stream=False,
                apart=()):
    """`arrays`: refs, block table, lengths, first, second, counts, served as `_Array`s or None.
    A plan of them and `caches` (as `_Array`s too)."""
    slots = _slots(len(caches))
    named = [(f"caches[{i}]", a) for i, a in enumerate(caches)] + \
        [("caches", None)] * (slots - len(caches)) + arrays
    tail = _PARAMS.pack(*numbers)
    if not workspace:
        tail = bytes(8) + tail
    plan = _d._Plan(_FILE, (("EK_CACHES", slots), ("EK_V", access), ("EK_STREAM", int(stream))),
                    launches, named, set(range(len(caches))) | {slots + i for i in written},
                    workspace, tail)
    # (written, bytes, other, bytes, their names), by their places among `arrays`
    plan.pairs = [(i, arrays[i][1].span(), j, arrays[j][1].span(), (arrays[i][0], arrays[j][0]))
                  for i, j in apart if arrays[i][1] and arrays[j][1]]
    plan.pad = [0] * (slots - len(caches))
    plan.gaps = {}
    if caches:
        plan.span, plan.steps, plan.element = \
            caches[0].span(), _d._steps(caches[0]), caches[0].size
    return plan


def _run(plan, caches, arrays: list) -> None:
    """Launches the plan, unless arrays that it writes overlap others."""
    if not plan.on_gpu:
        caches = _listed(caches)
        at = [_d._Array("caches", x).address() for x in caches]
        rest = [0 if x is None else _d._Array("", x).address() for x in arrays]
    else:
        rest = [0 if x is None else x.data_ptr() for x in arrays]
        if isinstance(caches, (list, tuple)):
            at = [x.data_ptr() for x in caches]
        elif len(caches.shape) == 4:
            at = [caches.data_ptr()]
        else:
            first, step = caches.data_ptr(), caches.stride(0) * plan.element
            at = [first + i * step for i in range(caches.shape[0])]
    if len(at) > 1:
        _check_apart(plan, at)
    for i, n, j, m, names in plan.pairs:
        if rest[i] < rest[j] + m and rest[j] < rest[i] + n:
            _d._apart(names[0], _d._Array(names[0], arrays[i]), names[1],
                      _d._Array(names[1], arrays[j]), False)
    if plan.on_gpu:
        plan.run_at(at + plan.pad + rest)
    else:
        plan.run(caches + [None] * len(plan.pad) + arrays)


def _served(plan, like):
    """A new int32 array of the shape of `like`, which is one."""
    return like.new_empty(like.shape) if plan is not None and plan.on_gpu else \
        T.new_empty(like, tuple(like.shape), np.int32)


def _step(a) -> int:
    return a.strides[0] if a is not None else 0


# -- copying ---------------------------------------------------------------------------------

def copy(caches, source, target) -> None:
    """Copies pages: page `target[i]` becomes page `source[i]`, in every cache.

    Pairs with an id outside of the cache are skipped. All pairs are copied at once, so no target
    may be among the sources; of a target that is there twice, each element is one of the two.

    Args:
        caches: the caches, written in place.
        source, target: int32 `[pairs]`.
    """
    try:
        key = (3, *_key(caches), _d._of(source), _d._of(target))
        plan = _d._plans.get(key)
    except (AttributeError, TypeError, RuntimeError, IndexError):
        key = plan = None
    if plan is None:
        plan = _copy_plan(caches, source, target)
        if plan is None:
            return
        _d._keep(key, plan)
    _run(plan, caches, [None, None, None, source, target, None, None])


def _copy_plan(caches, source, target):
    caches = _listed(caches)
    c = _check_caches(caches)
    sa = _d._array("source", source, ("i32",), 1, dense=False)
    ta = _d._array("target", target, ("i32",), 1, sa.shape, dense=False)
    n = sa.shape[0]
    heads, row, *strides = _row_form(c)
    arrays = [("refs", None), ("block_table", None), ("seq_lens", None), ("source", sa),
              ("target", ta), ("counts", None), ("served", None)]
    _d._device_of([("caches", c), *arrays])
    if n == 0 or heads * row == 0 or c.shape[0] == 0:
        return None
    v = _access(row)
    pieces = -(-(c.shape[1] * heads * row // v) // (_THREADS * _COPY))
    _d._need(n * pieces <= MAX_BLOCKS, f"{n} pages of {c.shape[1] * heads * row} bytes are too "
                                       "many for one call")
    moved = 2 * n * len(caches) * c.shape[1] * heads * row
    return _pages_plan(
        [("ek_copy_pages", (n * pieces, len(caches)), _THREADS)], [c] * len(caches), arrays,
        set(), 0, (*strides, 0, 0, _step(sa), _step(ta), 0, n, 0, 0, c.shape[0], c.shape[1],
                   heads, row, len(caches), pieces, 0), v, moved > _d._STREAM)


# -- compacting ------------------------------------------------------------------------------

def compact(caches, block_table, starts, keep, counts, *, seq_lens=None) -> None:
    """Keeps some tokens of each sequence and moves them together: token `starts[b] + keep[b, i]`
    becomes token `starts[b] + i` for i < `counts[b]`, in every cache.

    `keep[b]` ascends, so tokens move to the front or stay: an entry that is below its index, and
    a token beyond the block table or on a page outside of the cache, does not move. (With entries
    that do not ascend, what the slots from `starts[b]` on hold is left open.) It fits the path
    that `draft.accept` returns, `starts` being the lengths before the drafted tokens, as well as
    the tokens that are kept of a long history. Keys stay as they were rotated. A slot that is
    written to must not be on a page that another sequence holds.

    Args:
        caches: the caches, written in place.
        block_table: int32 `[rows, pages of a sequence]`.
        starts: int32 `[rows]`; rows with a negative one are left as they are.
        keep: int32 `[rows, most]`.
        counts: int32 `[rows]`; at most `most` count.
        seq_lens: int32 `[rows]`, which becomes `starts[b] + counts[b]` (at most 2^31 - 1), also
            where that is beyond the block table; without it nothing is written but the caches.
    """
    try:
        key = (4, *_key(caches), _d._of(block_table), _d._of(starts), _d._of(keep),
               _d._of(counts), None if seq_lens is None else _d._of(seq_lens))
        plan = _d._plans.get(key)
    except (AttributeError, TypeError, RuntimeError, IndexError):
        key = plan = None
    if plan is None:
        plan = _compact_plan(caches, block_table, starts, keep, counts, seq_lens)
        if plan is None:
            return
        _d._keep(key, plan)
    _run(plan, caches, [None, block_table, seq_lens, starts, keep, counts, None])


def _compact_plan(caches, block_table, starts, keep, counts, seq_lens):
    caches = _listed(caches)
    c = _check_caches(caches)
    bt, sl = _table(block_table, seq_lens, c.shape[1], written=False)
    rows = bt.shape[0]
    st = _d._array("starts", starts, ("i32",), 1, (rows,), dense=False)
    ka = _d._array("keep", keep, ("i32",), 2, (rows, None))
    ca = _d._array("counts", counts, ("i32",), 1, (rows,), dense=False)
    _d._need(ka.shape[1] <= _d.MAX_TOKENS, f"at most {_d.MAX_TOKENS} tokens are kept")
    arrays = [("refs", None), ("block_table", bt), ("seq_lens", sl), ("starts", st),
              ("keep", ka), ("counts", ca), ("served", None)]
    _d._device_of([("caches", c), *arrays])
    heads, row, *strides = _row_form(c)
    if rows == 0 or (sl is None and (heads * row == 0 or ka.shape[1] == 0)):
        return None
    v = _access(row) if row else 1
    parts = max(1, -(-(heads * row // v) // 64))
    _d._need(rows * parts * 64 <= MAX_BLOCKS * _THREADS,
             f"{rows} rows of {heads * row} bytes of a token are too many for one call")
    return _pages_plan(
        [("ek_compact", (rows * parts, len(caches)), 64)], [c] * len(caches), arrays, {2}, 0,
        (*strides, bt.strides[0], _step(sl), _step(st), ka.strides[0], _step(ca), rows, rows,
         bt.shape[1], c.shape[0], c.shape[1], heads, row, len(caches), parts, ka.shape[1]), v,
        False, [(2, j) for j in (1, 3, 4, 5)])


# -- sharing ---------------------------------------------------------------------------------

def fork(caches, refs, block_table, seq_lens, source, target):
    """Lets sequences go on from others: row `target[i]` gets the tokens of row `source[i]`.

    Whole pages are shared (their `refs` count one more; one below 0 stays); a last page that is
    not whole is copied to the lowest free one, so that both may append. A target must be an empty
    row (length 0), no source itself, and a row is the target of one fork: of several the first
    counts. A fork with another target, with a row outside of the table, or for which no page is
    left, is not served and changes nothing; forks get pages in their order.

    Args:
        caches: the caches, written in place.
        refs: int32 `[pages]`, written in place.
        block_table: int32 `[rows, pages of a sequence]`, written in place.
        seq_lens: int32 `[rows]`, written in place.
        source, target: int32 `[forks]`, rows of the table.

    Returns:
        int32 `[forks]`: 1 where a fork was served, else 0.
    """
    try:
        key = (5, *_key(caches), _d._of(refs), _d._of(block_table), _d._of(seq_lens),
               _d._of(source), _d._of(target))
        plan = _d._plans.get(key)
    except (AttributeError, TypeError, RuntimeError, IndexError):
        key = plan = None
    if plan is None:
        plan = _fork_plan(caches, refs, block_table, seq_lens, source, target)
        if plan is not None:
            _d._keep(key, plan)
    served = _served(plan, source)
    if plan is not None:
        _run(plan, caches, [refs, block_table, seq_lens, source, target, None, served])
    return served


def _fork_plan(caches, refs, block_table, seq_lens, source, target):
    caches = _listed(caches)
    c = _check_caches(caches)
    ra = _refs(refs, c.shape[0])
    bt, sl = _table(block_table, seq_lens, c.shape[1])
    sa = _d._array("source", source, ("i32",), 1, dense=False)
    ta = _d._array("target", target, ("i32",), 1, sa.shape, dense=False)
    n, rows = sa.shape[0], bt.shape[0]
    arrays = [("refs", ra), ("block_table", bt), ("seq_lens", sl), ("source", sa),
              ("target", ta), ("counts", None), ("served", None)]
    _d._device_of([("caches", c), *arrays])
    if n == 0:
        return None
    heads, row, *strides = _row_form(c)
    v = _access(row) if row else 1
    pieces = max(1, -(-(c.shape[1] * heads * row // v) // (_THREADS * _FORK)))
    _d._need(n * pieces <= MAX_BLOCKS, f"{n} forks of pages of {c.shape[1] * heads * row} bytes "
                                       "are too many for one call")
    _d._need(rows <= 1 << 22, f"at most {1 << 22} rows are supported, got {rows}")
    return _pages_plan(
        [("ek_fork_plan", (1, 1), 1024), ("ek_fork_copy", (n * pieces, len(caches) + 1),
                                          _THREADS)],
        [c] * len(caches), arrays, {0, 1, 2, 6}, 4 * (2 * rows + 3 * n),
        (*strides, bt.strides[0], _step(sl), _step(sa), _step(ta), 0, n, rows, bt.shape[1],
         c.shape[0], c.shape[1], heads, row, len(caches), pieces, 0), v, False,
        [(i, j) for i in (0, 1, 2) for j in range(i + 1, 5)])


# -- taking and giving back --------------------------------------------------------------------

def take(refs, block_table, seq_lens, new_lens, *, page_size: int):
    """Lets sequences grow to `new_lens`: the pages that row b still needs are taken, the lowest
    free ones (`refs` 0, which become 1), by the rows in their order, and entered in its row of the
    table; `seq_lens[b]` becomes `new_lens[b]`.

    A row that does not grow stays as it is. A row is served if the pages for it and all rows
    before it are there; one that is not, or that the table has no room for (it then takes no
    part), keeps its length and its pages.

    A row that is not served must be kept out of what the pages were for, since with its old length
    new tokens would be written over its last ones: `seq_lens * served` as the lengths of
    `decode.append_kv` and `draft.tree_attention` does that (its tokens are skipped and give zeros),
    and in `compact` a start of -1. What it may give back again to `free` are the lengths after this
    call, not `new_lens`.

    Args:
        refs: int32 `[pages]`, written in place.
        block_table: int32 `[rows, pages of a sequence]`, written in place.
        seq_lens: int32 `[rows]`, written in place.
        new_lens: int32 `[rows]`.
        page_size: tokens of a page.

    Returns:
        int32 `[rows]`: 1 where a row has the pages for its new length, else 0.
    """
    page_size = operator.index(page_size)
    try:
        key = (6, _d._of(refs), _d._of(block_table), _d._of(seq_lens), _d._of(new_lens),
               page_size)
        plan = _d._plans.get(key)
    except (AttributeError, TypeError, RuntimeError):
        key = plan = None
    if plan is None:
        plan = _rows_plan(refs, block_table, seq_lens, new_lens, page_size, True)
        if plan is not None:
            _d._keep(key, plan)
    served = _served(plan, seq_lens)
    if plan is not None:
        _run(plan, [], [refs, block_table, seq_lens, new_lens, None, None, served])
    return served


def free(refs, block_table, seq_lens, new_lens=None, *, page_size: int) -> None:
    """Cuts sequences to `new_lens`: the pages behind row b's first `new_lens[b]` tokens lose a
    holder (a page whose count reaches 0 is free), and `seq_lens[b]` becomes `new_lens[b]`. A row
    that is not longer than that stays as it is; a negative length counts as 0. The table keeps its
    entries. A count does not fall below 0, and one below 0 stays.

    Args:
        refs: int32 `[pages]`, written in place.
        block_table: int32 `[rows, pages of a sequence]`.
        seq_lens: int32 `[rows]`, written in place.
        new_lens: int32 `[rows]`; without it all sequences end.
        page_size: tokens of a page.
    """
    page_size = operator.index(page_size)
    try:
        key = (7, _d._of(refs), _d._of(block_table), _d._of(seq_lens),
               None if new_lens is None else _d._of(new_lens), page_size)
        plan = _d._plans.get(key)
    except (AttributeError, TypeError, RuntimeError):
        key = plan = None
    if plan is None:
        plan = _rows_plan(refs, block_table, seq_lens, new_lens, page_size, False)
        if plan is None:
            return
        _d._keep(key, plan)
    _run(plan, [], [refs, block_table, seq_lens, new_lens, None, None, None])


def _rows_plan(refs, block_table, seq_lens, new_lens, page: int, grow: bool):
    ra = _refs(refs)
    bt, sl = _table(block_table, seq_lens, page, written=grow)
    _d._need(sl is not None, "`seq_lens` is needed")
    rows, pages = bt.shape[0], ra.shape[0]
    na = None
    if new_lens is not None or grow:
        na = _d._array("new_lens", new_lens, ("i32",), 1, (rows,), dense=False)
    arrays = [("refs", ra), ("block_table", bt), ("seq_lens", sl), ("new_lens", na),
              ("second", None), ("counts", None), ("served", None)]
    _d._device_of(arrays)
    if rows == 0:
        return None
    numbers = (0, 0, 0, bt.strides[0], _step(sl), _step(na), 0, 0, rows, rows, bt.shape[1],
               pages, page, 0, 0, 0, 0, 0)
    if not grow:
        return _pages_plan([("ek_free_pages", (rows, 1), _THREADS)], [], arrays, {0, 2}, 0,
                           numbers, apart=[(0, 1), (0, 2), (0, 3), (2, 1), (2, 3)])
    most = min(pages, rows * bt.shape[1])
    return _pages_plan([("ek_take_pages", (1, 1), 1024)], [], arrays, {0, 1, 2, 6},
                       4 * (rows + most), numbers,
                       apart=[(i, j) for i in (0, 1, 2) for j in range(i + 1, 4)])


def specializations():
    """(source, macros) of the kernels that are worth compiling ahead."""
    for slots in (1, 2, 4, 8, 16, 32, 64, 128, 256):
        for stream in (0, 1):
            yield _FILE, (("EK_CACHES", slots), ("EK_V", 16), ("EK_STREAM", stream))
