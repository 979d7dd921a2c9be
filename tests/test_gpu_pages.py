"""Pages of a cache (``sgl_amd_mono.moe.pages``) against a plain pool (``pages_ref``): whole numbers and bytes,
all of them equal."""

import random

import pytest
import torch

import pages_ref

pytestmark = pytest.mark.gpu

I32 = torch.int32


def _i32(v):
    return torch.tensor(v, dtype=I32, device="cuda")


class Both:
    """A pool on the GPU and a plain one, and a table that both keep."""

    def __init__(self, pages, page, seqs, width, layers=2, row=48, seed=0, stride=None):
        from sgl_amd_mono.moe.pages import PagePool

        g = torch.Generator().manual_seed(seed)
        host = [torch.randint(256, (pages, page, row + 16 * i), generator=g, dtype=torch.uint8) for i in range(layers)]
        self.caches = [c.cuda() for c in host]
        self.pool = PagePool(pages, page, caches=self.caches, max_seqs=seqs, max_pages=width, device="cuda")
        self.ref = pages_ref.Pool(pages, page, host)
        wide = torch.full((seqs, stride or width), -7, dtype=I32, device="cuda")
        self.table = wide[:, :width]
        self.rows = [[-7] * width for _ in range(seqs)]
        self.n = [0] * seqs
        self.lens = _i32(self.n)

    def set(self, rows, lens):
        for b, r in enumerate(rows):
            self.rows[b][: len(r)] = r
        self.n = list(lens)
        self.table.copy_(_i32(self.rows))
        self.lens.copy_(_i32(self.n))

    def same(self, data=True):
        torch.cuda.synchronize()
        assert self.lens.tolist() == self.n
        assert self.table.tolist() == self.rows  # entries behind a sequence's pages stay as they were, too
        assert self.pool.refs.tolist() == self.ref.refs
        if data:
            for c, want in zip(self.caches, self.ref.caches):
                assert torch.equal(c.cpu(), want)
        code, where, count, _ = self.pool.read_errors()
        assert count == len(self.ref.errors), (code, where, count, self.ref.errors)
        assert not count or (code, where) in self.ref.errors

    def adopt(self):
        self.pool.adopt(self.table, self.lens)
        self.ref.adopt(self.rows, self.n)

    def grow(self, add, tokens=None, out=None):
        tokens = sum(max(a, 0) for a in add) if tokens is None else tokens
        got = self.pool.grow(self.table, self.lens, _i32(add), tokens, out=out)
        want = self.ref.grow(self.rows, self.n, add, tokens)
        assert [t.tolist() for t in got] == [list(w) for w in want]
        return got

    def trim(self, keep):
        self.pool.trim(self.table, self.lens, _i32(keep))
        self.ref.trim(self.rows, self.n, keep)

    def fork(self, parents):
        self.pool.fork(self.table, self.lens, _i32(parents))
        self.ref.fork(self.rows, self.n, parents)

    def compact(self):
        self.pool.compact(self.table, self.lens)
        self.ref.compact(self.rows, self.n)


@pytest.mark.parametrize("page", [1, 2, 16, 64, 1024])
def test_grow_from_empty(page):
    print(f"\ngrow page={page}", flush=True)
    b = Both(3000, page, 5, 700, layers=0)
    for add in ([1, 0, 3, 2 * page, 5], [1, 1, 1, 1, 1], [page, 0, 600, page - 1, 2 * page + 1], [0, 0, 0, 0, 0]):
        b.grow(add)
        b.same()


def test_grow_lowest_first_in_order_across_blocks():
    b = Both(5000, 1, 3, 4000, layers=0)
    rows = [list(range(0, 2000, 2)), list(range(4999, 3000, -3)), [2500, 2501]]
    b.set(rows, [len(r) for r in rows])
    b.adopt()
    b.same()
    b.grow([1500, 1, 700])
    b.same()


def test_grow_full_room_and_bounds():
    b = Both(10, 4, 5, 3, layers=0)
    b.grow([12, 9, 12, 1, 4])  # 3 + 3 + 3 + 1 pages, then none
    b.same()
    b.trim([12, 9, 0, 1, 0])
    b.grow([1, 3, -2, 3, 13], tokens=30)  # the table's width, in place, below 0, in place, the table's width
    b.same()
    b.grow([0, 0, 12, 0, 0], tokens=11)  # the outputs' rows
    b.same()
    b.grow([0, 0, 12, 0, 4], tokens=20)
    b.same()


def test_grow_with_rows_behind_and_outputs_given():
    b = Both(64, 8, 2, 8, layers=0, stride=13)
    out = tuple(torch.full((n,), 99, dtype=I32, device="cuda") for n in (50, 50, 3))
    assert b.grow([9, 20], tokens=50, out=out)[0] is out[0]
    b.same()
    assert b.pool.grow(b.table, b.lens, _i32([0, 0]), 0)[2].tolist() == [0, 0, 0]


def test_trim_lets_go_and_copies_what_is_shared():
    b = Both(40, 4, 6, 8)
    b.grow([11, 16, 5, 0, 0, 0])
    b.fork([0, 1, 2, 0, 1, 1])
    b.same()
    b.trim([6, 30, 4, 11, 6, 7])  # into shared pages, longer, to a border, as it is, into pages shared thrice
    b.same()
    b.trim([0, -5, 0, 3, 0, 7])
    b.same()
    b.trim([0] * 6)
    b.same()
    assert not b.pool.refs.any()


def test_trim_where_no_page_is_free():
    b = Both(4, 4, 3, 4)
    b.grow([16, 0, 0])
    b.fork([0, 0, 0])
    b.trim([6, 8, 16])
    b.same()  # recorded; the first stays, the second keeps whole pages


def test_fork_shares_and_copies():
    b = Both(60, 4, 8, 6)
    b.grow([7, 8, 21, 1, 0, 0, 0, 0])
    b.same()
    b.fork([0, 1, 2, 3, 0, 0, 2, 1])
    b.same()
    b.fork([7, 7, 6, 6, 6, -1, 2, 0])  # beams: rows dropped, permuted, their own row behind another's
    b.same()
    b.fork([1, -3, 8, 2, 1, 1, 1, 1])  # parents outside the table
    b.same()


def test_fork_where_no_page_is_free():
    b = Both(5, 4, 4, 3)
    b.grow([10, 2, 0, 0])
    b.fork([0, 1, 0, 1])
    b.same()
    b.fork([0, 1, 2, 3])
    b.same()


@pytest.mark.parametrize("pages,page", [(64, 16), (2500, 1), (1024, 4), (1025, 4)])
def test_compact(pages, page):
    print(f"\ncompact {pages} pages of {page}", flush=True)
    rng = random.Random(pages)
    b = Both(pages, page, 9, pages, row=16)
    perm = rng.sample(range(pages), pages)
    rows, lens = [], []
    for i in range(8):
        k = rng.randint(0, pages // 12)
        rows.append([perm.pop() for _ in range(k)])
        lens.append(max(0, k * page - rng.randint(0, page - 1)) if k else 0)
    full = lens[1] // page
    rows.append(rows[1][:full])  # pages of two sequences
    b.set(rows, lens + [full * page])
    b.adopt()
    b.same()
    b.compact()
    b.same()
    b.compact()  # nothing moves
    b.same()
    b.trim([0, 0, 0] + lens[3:] + [0])
    b.compact()
    b.same()
    b.trim([0] * 9)
    b.compact()
    b.same()


def test_compact_a_full_pool():
    b = Both(12, 2, 2, 12)
    b.grow([13, 10])
    b.compact()
    b.same()


def test_compact_needs_every_row():
    b = Both(3000, 2, 3, 900)
    b.grow([600, 40, 1500])
    b.trim([600, 0, 1500])
    b.pool.compact(b.table[:2], b.lens[:2])
    b.ref.errors.append((6, 750))  # the third row's holders
    b.same()
    with pytest.raises(RuntimeError, match="holders missing: 750 "):
        b.pool.raise_on_device_error()
    b.compact()
    b.same()
    b.pool.clear_errors()
    b.ref.errors.clear()
    graph = torch.cuda.CUDAGraph()
    some, lens = b.table[:1], b.lens[:1]
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        b.pool.compact(some, lens)
        b.pool.compact(b.table, b.lens)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        b.ref.errors.append((6, 750))
        b.ref.compact(b.rows, b.n)
        b.same()
        keep = [n - 9 for n in b.n[:1]] + b.n[1:]
        b.trim(keep)


@pytest.mark.parametrize("n", [0, 1, 7, 300])
def test_copy(n):
    from sgl_amd_mono.moe.pages import PagePool

    g = torch.Generator(device="cuda").manual_seed(n)
    shapes = [(700, 1, 656), (700, 1, 16), (700, 3, 1152)]
    caches = [torch.randint(256, s, generator=g, device="cuda", dtype=torch.uint8) for s in shapes]
    want = [c.clone() for c in caches]
    pool = PagePool(700, 1, caches=caches)
    perm = torch.randperm(700, generator=g, device="cuda").int()
    src, dst = perm[:n].contiguous(), perm[n : 2 * n].contiguous()
    pool.copy(src, dst)
    for c, w in zip(caches, want):
        w[dst.long()] = w[src.long()]
        assert torch.equal(c, w)
    pool.raise_on_device_error()


def test_copy_outside_the_pool_is_left_out():
    b = Both(10, 4, 1, 4)
    b.pool.copy(_i32([1, 10, 2, -1]), _i32([5, 6, 11, 7]))
    b.ref.copy([1], [5])
    torch.cuda.synchronize()
    for c, want in zip(b.caches, b.ref.caches):
        assert torch.equal(c.cpu(), want)
    code, where, count, _ = b.pool.read_errors()
    assert (code, count) == (2, 3) and where in (1, 2, 3)


def test_bad_tables_touch_nothing():
    b = Both(10, 4, 3, 4)
    b.set([[1, 99, 2], [3, -1], [4]], [10, 5, 17])  # pages outside the pool, a length past the table
    b.pool.adopt(b.table, b.lens)
    assert b.pool.refs.tolist() == [0, 1, 1, 1, 1, 0, 0, 0, 0, 0]
    code, _, count, _ = b.pool.read_errors()
    assert code in (1, 2) and count == 6  # 99, -1, the length, and the three entries of -7 that it takes in
    b.pool.clear_errors()
    b.pool.compact(b.table, b.lens)
    b.pool.fork(b.table, b.lens, _i32([2, 1, 0]))
    b.pool.trim(b.table, b.lens, _i32([0, 0, 0]))
    torch.cuda.synchronize()
    for c, want in zip(b.caches, b.ref.caches):
        assert torch.equal(c[5:].cpu(), want[5:])  # (pages 1 .. 4 moved to 0 .. 3)
    assert b.pool.read_errors()[2] > 0 and int(b.pool.refs.min()) >= 0


def test_pages_that_nobody_holds_stay_free():
    """Rows forked that name free pages: these get no holders, so that what is free stays counted."""
    b = Both(10, 4, 4, 3)
    b.set([[1, 2], [5, 6, 7]], [8, 12, 0, 0])
    b.pool.adopt(b.table[:1], b.lens[:1])  # the second row holds nothing
    for _ in range(3):
        b.pool.fork(b.table, b.lens, _i32([0, 1, 1, 0]))
        assert b.pool.refs.tolist() == [0, 2, 2, 0, 0, 0, 0, 0, 0, 0]
        b.pool.trim(b.table, b.lens, _i32([8, 0, 0, 0]))
        assert b.pool.refs.tolist() == [0, 1, 1, 0, 0, 0, 0, 0, 0, 0]
        b.lens[1] = 12
    assert b.pool.read_errors()[2] == 3 * (3 + 6)
    b.lens[1] = 0
    slots = b.pool.grow(b.table, b.lens, _i32([0, 12, 12, 12]), 36)[0]
    assert sorted(set((slots // 4).tolist())) == [-1, 0, 3, 4, 5, 6, 7]  # (of 8 free pages two rows take 6)


def test_adopt_finds_shared_partial_pages():
    b = Both(10, 4, 2, 2)
    b.set([[1, 2], [1, 2]], [8, 7])
    b.adopt()
    b.same()


@pytest.mark.parametrize("seed", range(8))
def test_random_lives(seed):
    """Calls in any order, with sequences that come, branch, are cut and go."""
    rng = random.Random(seed)
    page, seqs = rng.choice([1, 2, 4, 16]), rng.randint(1, 40)
    pages, width = rng.randint(20, 1500), rng.randint(4, 60)
    print(f"\nlives seed={seed} pages={pages} page={page} seqs={seqs} width={width}", flush=True)
    b = Both(pages, page, seqs, width, row=16, seed=seed)
    for _ in range(25):
        what = rng.choice(["grow", "grow", "grow", "trim", "fork", "compact", "adopt"])
        if what == "grow":
            add = [rng.choice([0, 1, 1, rng.randint(0, 6 * page)]) for _ in range(seqs)]
            b.grow(add, tokens=sum(add) + rng.choice([0, 0, 3]))
        elif what == "trim":
            b.trim([rng.choice([n, n, 0, rng.randint(0, n)]) for n in b.n])
        elif what == "fork":
            b.fork([rng.choice([i, i, i, rng.randrange(seqs), -1]) for i in range(seqs)])
        elif what == "compact":
            b.compact()
        else:
            b.adopt()
        b.same(data=False)
    b.same()


def test_captured_step():
    """trim and grow in a graph, replayed: each replay gives the step's places, as eager calls do."""
    b = Both(200, 4, 6, 20)
    b.grow([5, 9, 1, 0, 30, 4])
    add, keep = _i32([3, 1, 4, 0, 2, 5]), b.lens.clone()
    out = tuple(torch.empty(n, dtype=I32, device="cuda") for n in (15, 15, 7))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.pool.trim(b.table, b.lens, keep)
        b.pool.grow(b.table, b.lens, add, 15, out=out)
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        keep_now = keep.tolist()
        b.ref.trim(b.rows, b.n, keep_now)
        want = b.ref.grow(b.rows, b.n, add.tolist(), 15)
        assert [t.tolist() for t in out] == [list(w) for w in want]
        b.same()
        add.copy_(_i32([i, 4, 0, 1, 3, 2]))  # a graph replays with other counts
        keep.copy_(b.lens - 1)


def test_outputs_inside_a_capture_have_to_be_given():
    b = Both(20, 4, 2, 4)
    add = _i32([1, 1])
    with pytest.raises(RuntimeError, match="capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            b.pool.grow(b.table, b.lens, add, 2)


def test_on_another_stream():
    b = Both(100, 4, 4, 10)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b.grow([9, 3, 1, 14])
        b.fork([0, 0, 2, 3])
    torch.cuda.current_stream().wait_stream(s)
    b.same()
