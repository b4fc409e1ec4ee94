"""`enceladus.pages` on the GPU against plain forms, exactly: types and layouts of caches, strides,
pools that run out, wild ids and lengths, the same row or page twice, streams, graphs."""

import numpy as np
import pytest
import torch

import enceladus
from enceladus import pages
from oracle import draft_ref as R
from tests.test_gpu_decode import BF16, F8, F16, F32, cache, on_gpu, rand, table_for

pytestmark = pytest.mark.gpu

WILD = (-1, -2 ** 31, 2 ** 31 - 1)


def int32(values):
    return torch.tensor(values, dtype=torch.int32)


def same(got, want, what=""):
    """Equal bits (whatever they stand for)."""
    got = [x.cpu() for x in got]
    for i, (a, b) in enumerate(zip(got, want)):
        size = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[a.element_size()]
        a, b = a.contiguous().view(size), b.contiguous().view(size)
        assert torch.equal(a, b), (what, i, torch.nonzero(a != b)[:5])


def pool(gen, lens, page, pages_more, width=None, shared=()):
    """(table, refs, lens): rows over shuffled pages, `shared` rows over the pages of row 0."""
    bt, count = table_for(gen, lens, page, spare=pages_more, width=width)
    refs = torch.zeros(count, dtype=torch.int32)
    for b, n in enumerate(lens):
        if b in shared:
            bt[b] = bt[0]
        for p in bt[b, :R.pages_of(n, page)].tolist():
            refs[p] += 1
    return bt, refs, int32(lens)


CACHES = [(F32, 64, 2, 16, "token", 1), (F16, 128, 8, 16, "head", 3), (BF16, 80, 3, 24, "token", 2),
          (F8, 24, 1, 7, "head", 5), (F8, 72, 3, 1, "token", 2), (BF16, 1, 3, 5, "head", 2),
          (F8, 3, 5, 4, "token", 1), (F16, 128, 1, 64, "token", 33), (F32, 256, 16, 8, "head", 4)]


@pytest.mark.parametrize("dtype,dim,kv,page,layout,count", CACHES)
@pytest.mark.parametrize("pairs", [1, 9])
def test_copy(dtype, dim, kv, page, layout, count, pairs):
    gen = torch.Generator().manual_seed(dim)
    caches = [cache(gen, 25, page, kv, dim, dtype, layout) for _ in range(count)]
    order = torch.randperm(25, generator=gen).to(torch.int32)
    source, target = order[:pairs].clone(), order[12:12 + pairs].clone()
    if pairs > 1:
        source[1], target[2], source[3], target[4] = -1, 25, 2 ** 31 - 1, -2 ** 31
        source[5] = source[6]                              # one page to two others
    got = [on_gpu(c) for c in caches]
    pages.copy(got, source.cuda(), target.cuda())
    want = [c.clone() for c in caches]
    for a, b in zip(source.tolist(), target.tolist()):
        if 0 <= a < 25 and 0 <= b < 25:
            for w, c in zip(want, caches):
                w[b] = c[a]
    same(got, want)


def test_copy_of_caches_in_one_array():
    """Keys and values side by side, layers side by side, one array of all caches, one cache."""
    gen = torch.Generator().manual_seed(1)
    whole = rand(gen, 9, 2, 3, 16, 2, 40, dtype=F16)
    source, target = int32([1, 2, 5]), int32([8, 7, 6])
    want = whole.clone()
    want[[8, 7, 6], :, :, :, :, 3:35] = whole[[1, 2, 5], :, :, :, :, 3:35]
    g = whole.cuda()
    pages.copy([g[:, i, j, ..., 3:35] for i in range(2) for j in range(3)], source.cuda(),
               target.cuda())
    same([g], [want])
    stack = rand(gen, 4, 9, 16, 2, 64, dtype=F32)
    want = stack.clone()
    want[:, [8, 7, 6]] = stack[:, [1, 2, 5]]
    g = stack.cuda()
    pages.copy(g, source.cuda()[::1], target.cuda())
    same([g], [want])
    g = stack.cuda()
    pages.copy(g[2], source.cuda(), target.cuda())
    same([g[2]], [want[2]])
    same([g[0]], [stack[0]])


def test_copy_of_strided_ids_and_many_pages():
    gen = torch.Generator().manual_seed(2)
    c = rand(gen, 5000, 16, 2, 64, dtype=BF16)
    order = torch.randperm(5000, generator=gen).to(torch.int32)
    two = torch.stack((order[:2400], order[2500:4900]), 1).cuda()
    g = c.cuda()
    pages.copy([g], two[:, 0], two[:, 1])
    want = c.clone()
    want[order[2500:4900].long()] = c[order[:2400].long()]
    same([g], [want])


def test_copy_far_beyond_32_bit_offsets():
    count = (1 << 32) // (64 * 8 * 128) + 40
    g = torch.zeros(count, 64, 8, 128, dtype=torch.uint8, device="cuda").view(F8)
    gen = torch.Generator().manual_seed(3)
    page = rand(gen, 64, 8, 128).to(F8)
    g.view(torch.uint8)[count - 2] = page.view(torch.uint8).cuda()
    pages.copy([g], int32([count - 2]).cuda(), int32([5]).cuda())
    pages.copy([g], int32([5]).cuda(), int32([count - 1]).cuda())
    for p in (5, count - 1):
        same([g[p]], [page])
    assert not g.view(torch.uint8)[count - 3].any()


@pytest.mark.parametrize("dtype,dim,kv,page,layout,count", CACHES)
def test_compact(dtype, dim, kv, page, layout, count):
    gen = torch.Generator().manual_seed(dim + 1)
    lens = [40, 200, 1, 90, 33, 7, 64]
    bt, total = table_for(gen, lens, page)
    caches = [cache(gen, total, page, kv, dim, dtype, layout) for _ in range(count)]
    starts = [30, 0, 0, 11, 0, -1, 2 ** 31 - 1]
    keep = [[0, 2, 5, 9], list(range(0, 200, 3)), [0], list(range(11, 79)), list(range(33)),
            [1, 2], [1, 2]]
    counts = [len(k) for k in keep]
    counts[3] = 2 ** 31 - 1                                # more than there are entries
    width = max(map(len, keep))
    keep = [k + [10 ** 6 if b == 3 else -1] * (width - len(k)) for b, k in enumerate(keep)]
    wild = bt.clone()
    wild[1, 2::5] = torch.tensor([WILD[i % 3] for i in range(len(wild[1, 2::5]))])
    seq_lens = int32(lens)
    got, gl = [on_gpu(c) for c in caches], seq_lens.cuda()
    pages.compact(got, wild.cuda(), int32(starts).cuda(), int32(keep).cuda(),
                  int32(counts).cuda(), seq_lens=gl)
    want = []
    for c in caches:
        w, new = R.compact(c, wild.tolist(), starts, keep, counts)
        want.append(w)
    same(got, want)
    assert gl.tolist() == [n if m is None else m for n, m in zip(lens, new)]
    again = [on_gpu(c) for c in caches]                    # without lengths the same
    pages.compact(again, wild.cuda(), int32(starts).cuda(), int32(keep).cuda(),
                  int32(counts).cuda())
    same(again, want)


@pytest.mark.parametrize("width", [0, 4])
def test_compact_of_full_rows(width):
    """A sequence that fills its table has no token to move; its length is that of what was kept."""
    c = rand(torch.Generator().manual_seed(12), 4, 8, 1, 16)
    end = 8 * width
    starts = [end, end + 1, end + 100, 2 ** 31 - 2, 2 ** 31 - 1, -1, end]
    counts = [3, 1, 0, 1, 2, 2, -4]
    table = torch.arange(width, dtype=torch.int32).repeat(7, 1)
    keep, lens = int32([[1, 2, 4]]).repeat(7, 1), torch.full((7,), end + 5, dtype=torch.int32)
    g, m = c.cuda(), lens.cuda()
    pages.compact([g], table.cuda(), int32(starts).cuda(), keep.cuda(), int32(counts).cuda(),
                  seq_lens=m)
    same([g], [c])
    assert m.tolist() == [end + 3, end + 2, end + 100, 2 ** 31 - 1, 2 ** 31 - 1, end + 5, end]


@pytest.mark.parametrize("n,share", [(70, 0.9), (1000, 0.5), (5000, 0.03), (3001, 0.99)])
@pytest.mark.parametrize("page", [1, 16, 100])
def test_compact_long_histories(n, share, page):
    """Slots that are read after others were written over their neighbours."""
    gen = torch.Generator().manual_seed(n)
    lens = [n, n // 2 + 3]
    bt, total = table_for(gen, lens, page)
    c = cache(gen, total, page, 2, 64, F32)
    keep = [torch.nonzero(torch.rand(m, generator=gen) < share).flatten().tolist() for m in lens]
    counts = [len(k) for k in keep]
    keep = [k + [-1] * (max(counts) - len(k)) for k in keep]
    g = [c.cuda(), c.cuda() * 2]
    pages.compact(g, bt.cuda(), int32([0, 0]).cuda(), int32(keep).cuda(), int32(counts).cuda())
    want, _ = R.compact(c, bt.tolist(), [0, 0], keep, counts)
    same(g, [want, want * 2])


def test_compact_entries_that_do_not_ascend_stay_inside():
    gen = torch.Generator().manual_seed(4)
    bt, total = table_for(gen, [50, 50], 16)
    room = torch.full((total + 2, 16, 1, 64), 3.0).cuda()
    c = room[1:-1]
    keep = int32([[5, 3, 2 ** 31 - 1, -2 ** 31, 4, 60, 61, 62], list(range(40, 48))])
    pages.compact([c], bt.cuda(), int32([10, 30]).cuda(), keep.cuda(), int32([8, 8]).cuda())
    assert (room == 3).all()


def check_take(refs, table, lens, new, page):
    r, t, n = refs.cuda(), table.cuda(), lens.cuda()
    served = pages.take(r, t, n, int32(new).cuda(), page_size=page)
    want = R.take(refs.tolist(), table.tolist(), lens.tolist(), new, page)
    assert (served.tolist(), r.tolist(), t.tolist(), n.tolist()) == want
    return want


@pytest.mark.parametrize("page", [1, 7, 16])
@pytest.mark.parametrize("spare", [0, 1, 5, 40, 9000])
def test_take(page, spare):
    gen = torch.Generator().manual_seed(spare)
    lens = [0, 5, 16, 17, 100, -3, 7, 32]
    new = [20, 5, 17, 40, 90, 9, 2 ** 31 - 1, 32 + 3 * page]
    bt, refs, n = pool(gen, lens, page, spare, width=R.pages_of(150, page))
    refs[torch.nonzero(refs == 0).flatten()[1::4]] = -5
    check_take(refs, bt, n, new, page)


def test_take_serves_rows_in_their_order_until_one_has_no_pages():
    refs, table = torch.zeros(6, dtype=torch.int32), torch.full((5, 8), -1, dtype=torch.int32)
    refs[2] = 1
    lens = int32([0, 0, 3, 0, 4])
    served, r, _, n = check_take(refs, table, lens, [8, 16, 4, 4, 4], 4)
    assert served == [1, 0, 1, 0, 1] and n == [8, 0, 4, 0, 4]
    served, _, _, _ = check_take(refs, table, lens, [12, 12, 4, 8, 33], 4)
    assert served == [1, 0, 1, 0, 0]


@pytest.mark.parametrize("rows", [1, 1023, 1024, 1025, 5000])
def test_take_of_many_rows(rows):
    gen = torch.Generator().manual_seed(rows)
    refs = torch.randint(-1, 2, (4 * rows + 9000,), generator=gen).to(torch.int32)
    table = torch.full((rows, 6), -1, dtype=torch.int32)
    lens = torch.randint(0, 20, (rows,), generator=gen).to(torch.int32)
    new = (lens + torch.randint(-5, 20, (rows,), generator=gen)).tolist()
    check_take(refs, table, lens, new, 8)


def test_take_of_more_pages_than_32_bits_count():
    """Shares whose sum is beyond 32 bits: the rows before them are served."""
    rows = 70
    refs = torch.zeros(1000, dtype=torch.int32)
    t = torch.full((1, 1 << 20), -1, dtype=torch.int32).repeat(rows, 1)
    lens, new = torch.zeros(rows, dtype=torch.int32), [1 << 30] * rows
    new[:2] = [1024 * 3, 1024 * 5]
    r, g, n = refs.cuda(), t.cuda(), lens.cuda()
    served = pages.take(r, g, n, int32(new).cuda(), page_size=1024)
    assert served.tolist() == [1, 1] + [0] * (rows - 2)
    assert g[0, :4].tolist() == [0, 1, 2, -1] and g[1, :6].tolist() == [3, 4, 5, 6, 7, -1]
    assert r.tolist() == [1] * 8 + [0] * 992 and (g[2:] == -1).all()


@pytest.mark.parametrize("page", [1, 7, 16])
@pytest.mark.parametrize("end", [False, True])
def test_free(page, end):
    gen = torch.Generator().manual_seed(page)
    lens = [40, 40, 17, 0, 300, -2, 40, 16]
    bt, refs, n = pool(gen, lens, page, 5, width=R.pages_of(300, page), shared=(1, 6))
    bt[2, 0], bt[4, 1], bt[4, 2] = WILD[0], WILD[2], len(refs)
    refs[int(bt[7, 0])] = 0                                # counts too low already
    refs[int(bt[4, 0])] = -4
    n[4] = 2 ** 31 - 1                                     # beyond the table: all of the row
    new = [0] * 8 if end else [17, 40, 1, 5, 33, 0, -7, 15]
    r, m = refs.cuda(), n.cuda()
    pages.free(r, bt.cuda(), m, None if end else int32(new).cuda(), page_size=page)
    assert (r.tolist(), m.tolist()) == R.free(refs.tolist(), bt.tolist(), n.tolist(), new, page)


def test_free_of_a_page_that_many_hold_counts_down_to_zero():
    rows = 3000
    table = torch.zeros(rows, 2, dtype=torch.int32).cuda()
    table[:, 1] = 1
    refs = int32([rows, rows - 500, 7]).cuda()             # the second held by fewer than say so
    lens = torch.full((rows,), 32, dtype=torch.int32).cuda()
    pages.free(refs, table, lens, page_size=16)
    assert refs.tolist() == [0, 0, 7] and not lens.any()


def test_free_of_pages_that_are_never_taken():
    """Whatever their count below 0 is, and however many rows hold them."""
    rows = 4000
    refs = int32([-2 ** 31, -1, rows, -2 ** 31 + 1, 0, -7])
    table = torch.arange(6, dtype=torch.int32).repeat(rows, 1).cuda()
    lens = torch.full((rows,), 6 * 16, dtype=torch.int32).cuda()
    r = refs.cuda()
    pages.free(r, table, lens, page_size=16)
    assert r.tolist() == [-2 ** 31, -1, 0, -2 ** 31 + 1, 0, -7] and not lens.any()


FORKS = [
    ([0, 1, 2, 0, 0], [4, 5, 6, 7, 8]),
    ([0, 1, 1, 2], [4, 4, 5, 0]),                          # a row twice, a source as a target
    ([9, -1, 2, 2 ** 31 - 1, 0], [4, 5, 9, 6, -2 ** 31]),  # rows outside of the table
    ([0, 4, 1, 3], [5, 6, 2, 8]),                          # an empty source, a row in use
    ([2], [4]),
]


@pytest.mark.parametrize("source,target", FORKS)
@pytest.mark.parametrize("dtype,dim,kv,page,layout,count", CACHES)
@pytest.mark.parametrize("spare", [0, 2, 30])
def test_fork(source, target, dtype, dim, kv, page, layout, count, spare):
    gen = torch.Generator().manual_seed(spare)
    lens = [33, 48, 7, 100, 0, 0, 0, -1, 0]
    bt, refs, n = pool(gen, lens, page, spare, width=R.pages_of(120, page))
    bt[3, 1] = -1
    caches = [cache(gen, len(refs), page, kv, dim, dtype, layout) for _ in range(count)]
    g, r, t, m = [on_gpu(c) for c in caches], refs.cuda(), bt.cuda(), n.cuda()
    served = pages.fork(g, r, t, m, int32(source).cuda(), int32(target).cuda())
    want = R.fork(refs.tolist(), bt.tolist(), n.tolist(), source, target, page)
    assert (served.tolist(), r.tolist(), t.tolist(), m.tolist()) == want[:4]
    for c in caches:
        old = c.clone()
        for a, b, rest in want[4]:
            c[b, :rest] = old[a, :rest]
    same(g, caches)


def test_fork_of_a_last_page_that_is_not_in_the_cache():
    """Nothing to copy: the child has the parent's entry."""
    refs, n = int32([1, 0, 0]), int32([20, 0])
    for wild in (*WILD, 3):
        bt = int32([[0, wild], [-9, -9]])
        c = torch.zeros(3, 16, 1, 8).cuda()
        r, t, m = refs.cuda(), bt.cuda(), n.cuda()
        assert pages.fork([c], r, t, m, int32([0]).cuda(), int32([1]).cuda()).tolist() == [1]
        assert r.tolist() == [2, 0, 0] and t[1].tolist() == [0, wild] and m.tolist() == [20, 20]


def test_fork_leaves_counts_below_zero():
    """Pages that are never taken stay so, however often rows that hold them are shared, cut and
    ended: whole ones, and one that is not whole, of which children have copies."""
    page, rows = 16, 7
    refs, lens = int32([-1, 1, -2, 0, 0, 0, -2 ** 31, 0]), int32([40, 32, 0, 0, 0, 0, 0])
    table = torch.full((rows, 4), -1, dtype=torch.int32)
    table[0, :3], table[1, :2] = int32([0, 1, 2]), int32([6, 0])
    c = rand(torch.Generator().manual_seed(11), 8, page, 1, 8)
    plain = refs.tolist(), table.tolist(), lens.tolist()
    r, t, m, g = refs.cuda(), table.cuda(), lens.cuda(), c.cuda()
    for source, target in (([0, 1], [2, 3]), ([0, 1, 1], [4, 5, 6])):
        served = pages.fork([g], r, t, m, int32(source).cuda(), int32(target).cuda())
        want, *plain, copies = R.fork(*plain, source, target, page)
        assert (served.tolist(), r.tolist(), t.tolist(), m.tolist()) == (want, *plain)
        assert want == [1] * len(source)
        for a, b, rest in copies:
            c[b, :rest] = c[a, :rest]
    same([g], [c])
    new = [40, 64, 40, 32, 40, 32, 64]                     # no more than one page is left
    served, *plain = R.take(*plain, new, page)
    assert pages.take(r, t, m, int32(new).cuda(), page_size=page).tolist() == served
    assert (r.tolist(), t.tolist(), m.tolist()) == tuple(plain)
    assert not {0, 2, 6} & set(t[1, 2:].tolist() + t[6, 2:].tolist())
    pages.free(r, t, m, page_size=page)
    assert r.tolist() == [-1, 0, -2, 0, 0, 0, -2 ** 31, 0] and not m.any()


@pytest.mark.parametrize("forks", [1, 1024, 1500, 5000])
def test_fork_of_many(forks):
    gen = torch.Generator().manual_seed(forks)
    lens = torch.randint(0, 60, (50,), generator=gen).tolist()
    bt, refs, n = pool(gen, lens + [0] * forks, 8, forks // 2, width=8)
    refs[:5] += 1000
    source = torch.randint(0, 50, (forks,), generator=gen).tolist()
    target = (50 + torch.randperm(forks, generator=gen)).tolist()
    c = cache(gen, len(refs), 8, 1, 8, F16)
    g, r, t, m = c.cuda(), refs.cuda(), bt.cuda(), n.cuda()
    served = pages.fork([g], r, t, m, int32(source).cuda(), int32(target).cuda())
    want = R.fork(refs.tolist(), bt.tolist(), n.tolist(), source, target, 8)
    assert (served.tolist(), r.tolist(), t.tolist(), m.tolist()) == want[:4]
    old = c.clone()
    for a, b, rest in want[4]:
        c[b, :rest] = old[a, :rest]
    same([g], [c])


# -- as a program uses them -------------------------------------------------------------------

def test_strides_of_tables_lengths_and_ids():
    gen = torch.Generator().manual_seed(5)
    lens, page = [33, 48, 7, 0], 16
    bt, refs, n = pool(gen, lens, page, 9, width=6)
    c = cache(gen, len(refs), page, 2, 64, F16)
    wide = torch.full((4, 20), 77, dtype=torch.int32).cuda()
    wide[:, 3:9] = bt.cuda()
    two = torch.stack((n, int32([40, 90, 7, 20]), int32([3, 1, 4, 0]), int32([1, 2, 3, 3])), 1)
    two = two.cuda()
    g, r = c.cuda(), refs.cuda()
    table, m = wide[:, 3:9], two[:, 0]
    state = refs.tolist(), bt.tolist(), lens
    served, *state = R.take(*state, [40, 90, 7, 0], page)
    assert pages.take(r, table, m, int32([40, 90, 7, 0]).cuda(), page_size=page).tolist() == served
    served, *state, copies = R.fork(*state, [2], [3], page)
    assert pages.fork([g], r, table, m, two[2:3, 0] * 0 + 2, two[3:, 3]).tolist() == served
    refs2, lens2 = R.free(state[0], state[1], state[2], [3, 1, 4, 0], page)
    pages.free(r, table, m, two[:, 2], page_size=page)
    assert r.tolist() == refs2 and m.tolist() == lens2 and table.tolist() == state[1]
    assert (wide[:, :3] == 77).all() and (wide[:, 9:] == 77).all()


def random_step(gen, state, page):
    """One call of each kind, on `state` and on plain lists beside it; asserts that they agree."""
    refs, table, lens, caches, plain, held = state
    rows = len(plain[2])
    new = [max(0, n + int(torch.randint(-20, 30, (1,), generator=gen))) for n in plain[2]]
    served = pages.take(refs, table, lens, int32(new).cuda(), page_size=page)
    want, *plain = R.take(*plain, new, page)
    assert served.tolist() == want
    cut = [max(0, n - int(torch.randint(-10, 40, (1,), generator=gen))) for n in plain[2]]
    cut[int(torch.randint(0, rows, (1,), generator=gen))] = 0
    pages.free(refs, table, lens, int32(cut).cuda(), page_size=page)
    plain[0], plain[2] = R.free(*plain, cut, page)
    empty = [b for b, n in enumerate(plain[2]) if n == 0]
    some = [b for b, n in enumerate(plain[2]) if n]
    if empty and some:
        source = [some[int(torch.randint(0, len(some), (1,), generator=gen))] for _ in empty]
        served = pages.fork(caches, refs, table, lens, int32(source).cuda(), int32(empty).cuda())
        want, *plain, copies = R.fork(*plain, source, empty, page)
        assert served.tolist() == want
        for c in held:
            old = c.clone()
            for a, b, rest in copies:
                c[b, :rest] = old[a, :rest]
    assert (refs.tolist(), table.tolist(), lens.tolist()) == tuple(plain)
    return refs, table, lens, caches, plain, held


def test_a_run_of_calls():
    """A small pool that runs out, for many steps: every count, entry and length as in the plain
    form, and every page counted as often as rows hold it."""
    gen = torch.Generator().manual_seed(6)
    page, count, rows = 8, 40, 6
    held = [cache(gen, count, page, 1, 8, F32) for _ in range(3)]
    plain = [[0] * count, [[-1] * 12 for _ in range(rows)], [0] * rows]
    state = (int32(plain[0]).cuda(), int32(plain[1]).cuda(), int32(plain[2]).cuda(),
             [c.cuda() for c in held], plain, held)
    for _ in range(40):
        state = random_step(gen, state, page)
        refs, table, lens = state[4]
        uses = [0] * count
        for b, n in enumerate(lens):
            for p in table[b][:R.pages_of(n, page)]:
                uses[p] += 1
        assert uses == refs
    same(state[3], held)


def test_captured_calls_replayed():
    """A step of all calls as a graph, replayed on states that move on, against eager steps."""
    gen = torch.Generator().manual_seed(7)
    page, rows = 8, 4
    bt, refs, n = pool(gen, [20, 9, 0, 0], page, 60, width=12)
    caches = [cache(gen, len(refs), page, 2, 64, BF16) for _ in range(2)]
    start = [x.cuda() for x in (refs, bt, n, *caches)]
    grow, source, target = (int32(x).cuda() for x in ([30, 12, 0, 0], [0, 1], [2, 3]))
    keep, counts = int32([[0, 2, 5], [0, 1, 4], [3, 5, 7], [0, 0, 0]]).cuda(), \
        int32([3, 2, 3, 0]).cuda()
    moved = int32([0, 0]).cuda(), int32([len(refs) - 1, len(refs) - 2]).cuda()

    def step(r, t, m, *c):
        a = pages.take(r, t, m, grow, page_size=page)
        b = pages.fork(list(c), r, t, m, source, target)
        pages.compact(list(c), t, keep[:, 0], keep, counts, seq_lens=None)
        pages.copy(list(c), *moved)
        pages.free(r, t, m, counts, page_size=page)
        return a, b

    eager, own = [x.clone() for x in start], [x.clone() for x in start]
    step(*[x.clone() for x in start])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(*own)
    for x, y in zip(own, start):
        x.copy_(y)
    for k in range(4):
        want = step(*eager)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want)), k
        same(own, [x.cpu() for x in eager], k)
        grow += 3
        torch.randn(1000, device="cuda").sum().item()


def test_calls_on_two_streams_at_once():
    gen = torch.Generator().manual_seed(8)
    runs, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for i in range(2):
        bt, refs, n = pool(gen, [0] * 300, 4, 3000, width=20)
        runs.append([refs.cuda(), bt.cuda(), n.cuda()])
    want = []
    for i, (r, t, m) in enumerate(runs):
        p = [r.tolist(), t.tolist(), m.tolist()]
        for k in range(1, 9):
            _, *p = R.take(*p, [(7 + i) * k] * 300, 4)
        want.append(p)
    torch.cuda.synchronize()
    for k in range(1, 9):
        for i, (r, t, m) in enumerate(runs):
            with torch.cuda.stream(streams[i]):
                pages.take(r, t, m, torch.full((300,), (7 + i) * k, dtype=torch.int32,
                                               device="cuda"), page_size=4)
    torch.cuda.synchronize()
    for (r, t, m), p in zip(runs, want):
        assert [r.tolist(), t.tolist(), m.tolist()] == p


def test_numpy_and_enceladus_arrays():
    gen = torch.Generator().manual_seed(9)
    bt, refs, n = pool(gen, [20, 9, 0], 8, 9, width=5)
    caches = [cache(gen, len(refs), 8, 1, 16, F32) for _ in range(2)]
    new, source, target = int32([24, 17, 0]), int32([1]), int32([2])
    keep, counts, starts = int32([[0, 3], [1, 2], [0, 0]]), int32([2, 2, 0]), int32([4, 0, 0])

    def run(make):
        r, t, m, nw, s, d, k, c, st = (make(x) for x in (refs, bt, n, new, source, target, keep,
                                                         counts, starts))
        cs = [make(x) for x in caches]
        a = pages.take(r, t, m, nw, page_size=8)
        b = pages.fork(cs, r, t, m, s, d)
        pages.compact(cs, t, st, k, c, seq_lens=m)
        pages.copy(cs, s, d)
        pages.free(r, t, m, c, page_size=8)
        return [a, b, r, t, m, *cs]

    want = [x.cpu().numpy() for x in run(lambda x: x.cuda())]
    got = run(lambda x: x.numpy().copy())
    assert all(isinstance(x, np.ndarray) and np.array_equal(x, w) for x, w in zip(got, want))
    got = run(lambda x: enceladus.from_numpy(x.numpy().copy()))
    assert all(np.array_equal(x.numpy(), w) for x, w in zip(got, want))


def test_calls_are_timed_and_traced(tmp_path):
    gen = torch.Generator().manual_seed(10)
    c = cache(gen, 9, 8, 1, 16, F32).cuda()
    ids = int32([1]).cuda(), int32([2]).cuda()
    assert enceladus.testing.do_bench(lambda: pages.copy([c], *ids), rep=3) > 0
    path = tmp_path / "t.json"
    with enceladus.capture(path):
        pages.copy([c], *ids)
    assert "ek_copy_pages" in path.read_text()
