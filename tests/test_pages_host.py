"""The page pool on the host side, without a GPU: the C ABI's argument checks (each returns before any HIP call,
so fake device addresses are safe), the structures' layout, and the pool's checks. The plain pool that the GPU
tests compare with is itself checked here."""

import ctypes
import random

import pytest
import torch

import pages_ref

I32 = torch.int32
AT, WS = 0x100000, 0x200000


def _pool(**over):
    from sgl_amd_mono.moe import _lib

    return _lib.PagesPool(**{**dict(pages=100, page_size=16, max_seqs=8, max_pages=20, ncaches=2, caches=AT), **over})


def _table(**over):
    from sgl_amd_mono.moe import _lib

    return _lib.PagesTable(**{**dict(table=AT, lens=AT, stride=20, seqs=8, max_pages=20), **over})


@pytest.fixture(scope="module")
def lib():
    from sgl_amd_mono.moe import _lib

    L = _lib.lib()
    n = ctypes.c_size_t()
    assert L.mkmoe_pages_workspace_bytes(100, 8, 20, ctypes.byref(n)) == 0 and n.value % 256 == 0
    return L, n.value


def _calls(L, n, pool=None, table=None, ws=WS, arg=AT, out=AT, tokens=4):
    r = ctypes.byref
    p, t = r(pool or _pool()), r(table or _table())
    return {
        "adopt": lambda: L.mkmoe_pages_adopt(p, t, ws, n, None),
        "grow": lambda: L.mkmoe_pages_grow(p, t, arg, tokens, out, out, out, ws, n, None),
        "trim": lambda: L.mkmoe_pages_trim(p, t, arg, ws, n, None),
        "fork": lambda: L.mkmoe_pages_fork(p, t, arg, ws, n, None),
        "compact": lambda: L.mkmoe_pages_compact(p, t, ws, n, None),
        "copy": lambda: L.mkmoe_pages_copy(p, arg, arg, tokens, ws, n, None),
    }


def test_workspace_bytes(lib):
    L, n = lib
    size = ctypes.c_size_t()
    for bad in ((0, 1, 1), ((1 << 22) + 1, 1, 1), (1, 0, 1), (1, 1025, 1), (1, 1, 0), (1, 1, (1 << 22) + 1)):
        assert L.mkmoe_pages_workspace_bytes(*bad, ctypes.byref(size)) == -8
    assert L.mkmoe_pages_workspace_bytes(1, 1, 1, None) == -1
    assert L.mkmoe_pages_workspace_bytes(1 << 22, 1024, 1 << 22, ctypes.byref(size)) == 0 and size.value > 1 << 34


@pytest.mark.parametrize("over,code", [
    (dict(pages=0), -8), (dict(pages=-1), -8), (dict(max_seqs=0), -8), (dict(max_seqs=1025), -8), (dict(max_pages=0), -8),
    (dict(page_size=0), -8), (dict(page_size=24), -8), (dict(page_size=2048), -8),
    (dict(pages=1 << 22, page_size=1024), -8),  # 2^32 tokens
    (dict(max_pages=1 << 22, page_size=1024), -8),
    (dict(ncaches=-1), -8), (dict(caches=None), -8),
    (dict(pages=5000), -5), (dict(max_pages=500), -5),
])  # fmt: skip
def test_every_call_checks_the_pool(lib, over, code):
    L, n = lib
    for name, call in _calls(L, n, pool=_pool(**over)).items():
        assert call() == code, name
    for ws, size, e in ((None, n, -1), (WS + 64, n, -4), (WS, n - 1, -5)):
        for name, call in _calls(L, size, ws=ws).items():
            assert call() == e, name


@pytest.mark.parametrize("over,code", [
    (dict(table=None), -1), (dict(lens=None), -1), (dict(seqs=0), -3), (dict(seqs=9), -3), (dict(max_pages=0), -8),
    (dict(max_pages=21, stride=21), -8), (dict(stride=19), -8), (dict(table=AT + 2), -4), (dict(lens=AT + 1), -4),
])  # fmt: skip
def test_every_call_checks_its_table(lib, over, code):
    L, n = lib
    for name, call in _calls(L, n, table=_table(**over)).items():
        if name != "copy":
            assert call() == code, name


def test_other_arguments_are_checked(lib):
    L, n = lib
    for name in ("grow", "trim", "fork", "copy"):
        assert _calls(L, n, arg=None)[name]() == -1, name
        assert _calls(L, n, arg=AT + 2)[name]() == -4, name
    assert _calls(L, n, out=None)["grow"]() == -1 and _calls(L, n, out=AT + 2)["grow"]() == -4
    assert _calls(L, n, tokens=-1)["grow"]() == -3
    assert _calls(L, n, tokens=-1)["copy"]() == -3 and _calls(L, n, tokens=101)["copy"]() == -3
    assert _calls(L, n, tokens=0, arg=None)["copy"]() == 0
    assert _calls(L, n, pool=_pool(ncaches=0, caches=None))["copy"]() == 0
    words = (ctypes.c_int32 * 4)()
    assert L.mkmoe_pages_read_errors(None, words, 4, None) == -1 and L.mkmoe_pages_read_errors(WS, None, 4, None) == -1
    assert L.mkmoe_pages_read_errors(WS, words, 0, None) == -8 and L.mkmoe_pages_read_errors(WS, words, 5, None) == -8
    assert L.mkmoe_pages_adopt(None, None, WS, n, None) == -1


def test_packed_fields_are_the_structure():
    from sgl_amd_mono.moe import _lib

    one, at_once = _lib.PagesTable(1, 2, 3, 4, 5), _lib.PagesTable()
    _lib.PAGES_TABLE.pack_into(at_once, 0, 1, 2, 3, 4, 5)
    assert bytes(one) == bytes(at_once)


# ---------------------------------------------------------------- the pool's class
@pytest.mark.parametrize("args,kw,err", [
    ((0, 16), {}, "0 pages"),
    (((1 << 22) + 1, 1), {}, "pages of 1"),
    ((1 << 22, 1024), {}, "below 2"),
    ((10, 24), {}, "page_size 24"),
    ((10, 2048), {}, "page_size 2048"),
    ((10, 16), dict(max_seqs=0), "max_seqs 0"),
    ((10, 16), dict(max_seqs=1025), "max_seqs 1025"),
    ((10, 16), dict(max_pages=0), "max_pages 0"),
    ((10, 16), dict(device="cpu"), "not a GPU"),
    ((10, 16), dict(caches=[torch.zeros(10, 16)]), "not a GPU"),
])  # fmt: skip
def test_pool_rejects_bad_options(args, kw, err):
    from sgl_amd_mono.moe.pages import PagePool

    with pytest.raises(RuntimeError, match=err):
        PagePool(*args, **kw)


@pytest.fixture
def pool():
    """A pool whose tensors lie on the host; a call that passes its checks is written down."""
    from sgl_amd_mono.moe import _lib
    from sgl_amd_mono.moe.pages import PagePool

    p = PagePool.__new__(PagePool)
    p.pages, p.page_size, p.max_seqs, p.max_pages = 100, 16, 8, 20
    p.device, p._index, p.lib, p._pool, p._table = torch.device("cpu"), -1, _lib.lib(), _pool(), _lib.PagesTable()
    p.calls = []
    p._call = lambda fn, *a: p.calls.append((fn.__name__, a))
    return p


def _i32(*shape):
    return torch.zeros(*shape, dtype=I32)


def test_calls_fill_what_the_library_reads(pool):
    wide, lens, add = _i32(4, 30), _i32(4), _i32(4)
    table, out = wide[:, 5:20], (_i32(9), _i32(9), _i32(5))
    assert pool.grow(table, lens, add, 9, out=out) == out
    pool.trim(table, lens, add)
    pool.fork(table, lens, add)
    pool.compact(table, lens)
    pool.adopt(table, lens)
    pool.adopt()
    pool.copy(add, lens)
    names = [n for n, _ in pool.calls]
    assert names == [f"mkmoe_pages_{x}" for x in ("grow", "trim", "fork", "compact", "adopt", "adopt", "copy")]
    t = pool._table
    assert (t.table, t.lens, t.stride, t.seqs, t.max_pages) == (table.data_ptr(), lens.data_ptr(), 30, 4, 15)
    assert pool.calls[0][1][2:] == (add.data_ptr(), 9, *(x.data_ptr() for x in out))
    assert pool.calls[5][1][1] is None and pool.calls[6][1][1:] == (add.data_ptr(), lens.data_ptr(), 4)


@pytest.mark.parametrize("table,lens,err", [
    (None, _i32(4), "table: missing"),
    (torch.zeros(4, 10, dtype=torch.int64), _i32(4), "table"),
    (_i32(4), _i32(4), "table"),
    (_i32(9, 10), _i32(9), "table"),  # more rows than the pool takes
    (_i32(4, 21), _i32(4), "table"),
    (_i32(10, 4).T, _i32(4), "table"),
    (_i32(1, 10).expand(4, 10), _i32(4), "table"),
    (_i32(4, 10), _i32(5), "lens"),
    (_i32(4, 10), None, "lens: missing"),
    (_i32(4, 10), torch.zeros(4), "lens"),
    (_i32(4, 10), _i32(8)[::2], "lens"),
])  # fmt: skip
def test_tables_are_checked(pool, table, lens, err):
    add = _i32(4)
    for call in (lambda: pool.grow(table, lens, add, 0, out=(_i32(0), _i32(0), _i32(5))), lambda: pool.trim(table, lens, add),
                 lambda: pool.fork(table, lens, add), lambda: pool.compact(table, lens), lambda: pool.adopt(table, lens)):  # fmt: skip
        with pytest.raises(RuntimeError, match=err):
            call()
    assert not pool.calls


def test_other_tensors_are_checked(pool):
    t, n = _i32(4, 10), _i32(4)
    for name in ("trim", "fork"):
        for bad in (None, _i32(3), torch.zeros(4, dtype=torch.int64)):
            with pytest.raises(RuntimeError, match="keep" if name == "trim" else "parents"):
                getattr(pool, name)(t, n, bad)
    with pytest.raises(RuntimeError, match="add"):
        pool.grow(t, n, _i32(5), 3, out=(_i32(3), _i32(3), _i32(5)))
    with pytest.raises(RuntimeError, match="-1 tokens"):
        pool.grow(t, n, n, -1)
    for i, what in enumerate(("slots", "positions", "starts")):
        out = [_i32(3), _i32(3), _i32(5)]
        out[i] = _i32(4)
        with pytest.raises(RuntimeError, match=what):
            pool.grow(t, n, n, 3, out=out)
    for src, dst in ((_i32(3), _i32(4)), (_i32(101), _i32(101)), (None, _i32(3)), (_i32(3, 1), _i32(3))):
        with pytest.raises(RuntimeError, match="src|dst"):
            pool.copy(src, dst)
    assert not pool.calls


# ---------------------------------------------------------------- the plain pool
def test_the_plain_pool_keeps_what_it_should():
    """Through calls in any order: every page is held as often as it is named, a partly filled one once, and a
    sequence's tokens stay what they were."""
    rng = random.Random(1)
    for _ in range(20):
        ps, seqs, width = rng.choice([1, 4]), rng.randint(1, 6), 12
        pool = pages_ref.Pool(40, ps, [torch.zeros(40, ps, dtype=torch.int64)])
        rows, lens, said = [[-1] * width for _ in range(seqs)], [0] * seqs, [[] for _ in range(seqs)]
        for _ in range(30):
            what = rng.choice(["grow", "trim", "fork", "compact"])
            if what == "grow":
                add = [rng.randint(0, 5) for _ in range(seqs)]
                before = list(lens)
                slots, positions, starts = pool.grow(rows, lens, add, sum(add))
                for b in range(seqs):
                    for t in range(starts[b], starts[b] + lens[b] - before[b]):
                        assert positions[t] == len(said[b])
                        said[b].append(rng.randrange(1 << 40))
                        pool.caches[0].view(-1)[slots[t]] = said[b][-1]
            elif what == "trim":
                pool.trim(rows, lens, [rng.randint(0, n) for n in lens])
                said = [s[:n] for s, n in zip(said, lens)]
            elif what == "fork":
                parents = [rng.choice([i, rng.randrange(seqs), -1]) for i in range(seqs)]
                pool.fork(rows, lens, parents)
                said = [list(said[p][:n]) if p >= 0 and n else [] for p, n in zip(parents, lens)]
            else:
                pool.compact(rows, lens)
                live = sum(r > 0 for r in pool.refs)
                assert all(pool.refs[:live]) and not any(pool.refs[live:])
            named = [0] * 40
            for b in range(seqs):
                for p in rows[b][: pool.need(lens[b])]:
                    named[p] += 1
                if lens[b] % ps:
                    assert pool.refs[rows[b][lens[b] // ps]] == 1
                got = [int(pool.caches[0][rows[b][i // ps], i % ps]) for i in range(lens[b])]
                assert got == said[b]
            assert named == pool.refs
