"""Captured calls of a prompt's attention and of the page pool, replayed with other inputs beside eager work: every
replay is what eager calls give from the same state."""

import pytest
import torch

import latent_ref as ref
from test_gpu_latent_prompt import BF, Batch, _cos_sin, _randn, _runner
from test_gpu_pages import Both, _i32

pytestmark = pytest.mark.gpu


def _capture(call):
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    return graph


@pytest.mark.parametrize("fmt,page,width", [("bf16", 16, 64), ("mxfp8", 64, 16), ("mxfp8", 64, 600)])
def test_a_captured_step(fmt, page, width):
    """The step before taken back, the next tokens placed, and a layer's attention of them, in one graph."""
    from sgl_amd_mono.moe.latent import cache_like
    from sgl_amd_mono.moe.pages import PagePool

    heads, seqs, tokens = 4, 5, 300
    b = Batch(61, heads, fmt, page, [1] * seqs, [1] * seqs)  # (its weights and generator)
    pages = 200 * 64 // page
    cache = cache_like(pages, page, fmt)
    pool = PagePool(pages, page, caches=[cache], max_seqs=seqs, max_pages=width)
    run = _runner(heads, max_tokens=tokens, max_context=(8192 if width * page <= 32768 else 40000 * seqs))
    table = torch.zeros(seqs, width, dtype=torch.int32, device="cuda")
    lens, add, keep = (_i32([0] * seqs) for _ in range(3))
    places = tuple(torch.zeros(n, dtype=torch.int32, device="cuda") for n in (tokens, tokens, seqs + 1))
    q, kv = _randn(b.g, tokens, heads, 192), _randn(b.g, tokens, 576)
    cos_sin, out = _cos_sin(2048), torch.zeros(tokens, heads, 128, dtype=BF, device="cuda")

    def call():
        pool.trim(table, lens, keep)
        pool.grow(table, lens, add, tokens, out=places)
        run.attention(b.w, cache, q, kv, cos_sin, places[1], places[0], table, lens, q_starts=places[2], out=out)

    graph = _capture(call)
    states = [table, lens, cache, pool.ws, out, *places]
    for i, (new, cut) in enumerate([([100, 7, 0, 130, 63], [0] * 5), ([1, 250, 3, 0, 4], [90, 7, 0, 64, 63]),
                                    ([60, 60, 60, 60, 60], [0, 200, 3, 5, 1]), ([0] * 5, [60, 60, 60, 60, 0])]):  # fmt: skip
        add.copy_(_i32(new))
        keep.copy_(_i32(cut))
        q.copy_(_randn(b.g, *q.shape))
        kv.copy_(_randn(b.g, *kv.shape))
        out.fill_(7.0)
        torch.cuda.synchronize()
        before = [x.clone() for x in states]
        graph.replay()
        torch.cuda.synchronize()
        after = [x.clone() for x in states]
        for x, y in zip(states, before):
            x.copy_(y)
        call()
        torch.cuda.synchronize()
        for x, y, what in zip(states, after, ("table", "lens", "cache", "pool", "out", "slots", "positions", "starts")):
            if what != "pool":
                assert torch.equal(x, y), (i, what)
        n = sum(new)
        assert lens.tolist() == [c + a for c, a in zip(cut, new)]
        assert torch.isfinite(out[:n].float()).all() and (out[n:] == 7).all()
        held = torch.zeros(pages, dtype=torch.int32, device="cuda")
        for s, length in enumerate(lens.tolist()):
            held[table[s, : -(-length // page)].long()] += 1
        assert torch.equal(held, pool.refs)
    pool.raise_on_device_error()
    run.raise_on_device_error()


def test_two_graphs_of_one_runner():
    """Graphs of other shapes and cuts that share a workspace, replayed in turn."""
    a, b = Batch(62, 4, "bf16", 16, [300, 20], [700, 33]), Batch(63, 4, "mxfp8", 64, [70, 0, 90], [2000, 5, 91], width=1600)
    run = _runner(4, max_context=120000)
    outs = [torch.zeros(x.starts[-1], 4, 128, dtype=BF, device="cuda") for x in (a, b)]
    calls = [lambda x=x, o=o: run.attend(*x.args(), q_starts=x.dev_starts, out=o) for x, o in zip((a, b), outs)]
    graphs = [_capture(c) for c in calls]
    for i in range(4):
        for x in (a, b):
            x.q_nope.copy_(_randn(x.g, *x.q_nope.shape))
            x.cache.copy_(ref.random_cache(x.pages, x.cache.shape[1], "bf16" if x is a else "mxfp8", x.g, "cuda"))
        for o in outs:
            o.fill_(7.0)
        for j in ((0, 1), (1, 0), (0, 0, 1), (1, 1, 0))[i]:
            graphs[j].replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        for c in calls:
            c()
        torch.cuda.synchronize()
        for g, o, x in zip(got, outs, (a, b)):
            assert torch.equal(g, o)
            x.check(g)


def test_captured_calls_of_a_pool():
    """adopt, fork, trim, compact and copy in a graph."""
    b = Both(300, 4, 6, 30, layers=3)
    parents, keep, src, dst = _i32([0] * 6), _i32([0] * 6), _i32([0, 1]), _i32([298, 299])

    def call():
        b.pool.adopt(b.table, b.lens)
        b.pool.fork(b.table, b.lens, parents)
        b.pool.trim(b.table, b.lens, keep)
        b.pool.copy(src, dst)
        b.pool.compact(b.table, b.lens)

    graph = _capture(call)
    torch.cuda.synchronize()
    b.ref.caches = [c.cpu() for c in b.caches]
    steps = [([0, 1, 2, 3, 4, 5], [30, 9, 50, 3, 0, 100]), ([0, 0, 2, 5, 5, 5], [30, 7, 48, 90, 91, 100]),
             ([3, 4, -1, 2, 1, 0], [1000, 89, 3, 41, 7, 30]), ([5, 5, 5, 5, 5, 5], [30, 29, 28, 27, 26, 25])]  # fmt: skip
    rows = [list(range(20 + 40 * i, 20 + 40 * i + 30)) for i in range(6)]
    b.set(rows, [30, 9, 50, 3, 0, 100])
    for p, k in steps:
        for t, v in ((parents, p), (keep, k)):
            t.copy_(_i32(v))
        graph.replay()
        b.ref.adopt(b.rows, b.n)
        b.ref.fork(b.rows, b.n, p)
        b.ref.trim(b.rows, b.n, k)
        b.ref.copy(src.tolist(), dst.tolist())
        b.ref.compact(b.rows, b.n)
        b.same()
        if p == steps[1][0]:  # eager work between
            b.grow([1, 2, 3, 4, 5, 6])
            b.same()


@pytest.mark.parametrize("layers", [1, 128, 129, 300])
def test_pages_of_many_caches(layers):
    """Their places are read 128 at a time; sizes of a page differ between the caches."""
    print(f"\n{layers} caches", flush=True)
    b = Both(12, 2, 3, 5, layers=layers, row=16)
    b.grow([7, 3, 0])
    b.same()
    b.fork([0, 1, 0])
    b.same()
    b.trim([5, 0, 7])
    b.same()
    b.pool.copy(_i32([1]), _i32([11]))
    b.ref.copy([1], [11])
    b.same()
    b.compact()
    b.same()
