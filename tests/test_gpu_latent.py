"""Latent attention's kernels (``sgl_amd_mono.moe.latent``) against a plain 64-bit form
(``latent_ref``), each value within the bound that the kernels' roundings allow."""

import pytest
import torch

import latent_ref as ref

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
SCALE = 192**-0.5
NAN, INF = float("nan"), float("inf")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda").to(BF)


def _runner(heads, **kw):
    from sgl_amd_mono.moe.latent import LatentRunner

    return LatentRunner(heads, scale=SCALE, **kw)


def _cos_sin(n):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    return torch.cat([a.cos(), a.sin()], 1).float().cuda()


def _tables(g, seqs, max_len, page, spare=3):
    per = -(-max_len // page)
    pages = seqs * per + spare
    perm = torch.randperm(pages, generator=g, device="cuda").int()
    return perm[: seqs * per].view(seqs, per).contiguous(), pages


# ---------------------------------------------------------------- append and rows
@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("rope", ["interleaved", "half"])
@pytest.mark.parametrize("tokens,heads,page,index", [(1, 1, 1, torch.int64), (3, 5, 64, torch.int32), (77, 32, 16, torch.int64), (1021, 16, 2, torch.int64)])
def test_append(fmt, rope, tokens, heads, page, index):
    print(f"\nappend {fmt} {rope} tokens={tokens} heads={heads} page={page}", flush=True)
    from sgl_amd_mono.moe.latent import cache_like

    g = _gen(tokens + heads)
    run = _runner(heads, rope=rope)
    pages = -(-2 * tokens // page) + 1
    cache = ref.random_cache(pages, page, fmt, g, "cuda")
    before = cache.clone()
    kv = _randn(g, tokens, 640)[:, 32:608]  # rows of a wider projection
    kv[:, :512] *= 3.0
    w = (1 + 0.1 * torch.randn(512, generator=g, device="cuda")).to(BF)
    q = _randn(g, tokens, heads, 192)
    cs = _cos_sin(4096)
    pos = torch.randint(4096, (tokens,), generator=g, device="cuda").to(index)
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens].to(index)
    out = torch.empty(heads, tokens, 64, dtype=BF, device="cuda").transpose(0, 1)
    run.append(cache, kv, w, cs, pos, slots, q_pe=q[..., 128:], q_out=out)
    got = run.rows(cache, slots)
    torch.cuda.synchronize()
    run.raise_on_device_error()
    flat, keep = cache.view(pages * page, -1), torch.ones(pages * page, dtype=torch.bool, device="cuda")
    keep[slots.long()] = False
    assert torch.equal(flat[keep], before.view(pages * page, -1)[keep])  # no other row was touched
    stored = flat[slots.long()]
    c = ref.norm(kv[:, :512], w, 1e-6)
    cpos = cs[pos.long()]
    pe, size = ref.rotate(kv[:, 512:].double(), cpos, rope == "half")
    vals = ref.row_values(stored)
    # fp32: 512 squares, their mean, the root, the division and two products
    near = c.abs() * 540 * ref.U32
    if fmt == "bf16":
        ref.assert_within(vals[:, :512], c, c.abs() * ref.U16 + 2 * near, "latent")
    else:
        sc = torch.exp2(stored[:, 512:528].double() - 127)
        top = c.view(tokens, 16, 32).abs().amax(-1) / 448
        assert bool((top <= sc * (1 + 1e-4)).all()) and bool((top > sc / 2 * (1 - 1e-4)).all())
        step = torch.maximum(c.abs() * 2.0**-4, (sc * 2.0**-10).repeat_interleave(32, 1))
        ref.assert_within(vals[:, :512], c, step * (1 + 1e-4) + 2 * near, "latent")
    ref.assert_within(vals[:, 512:], pe, pe.abs() * ref.U16 + 3 * ref.U32 * size, "rope part")
    qr, qsize = ref.rotate(q[..., 128:].double(), cpos[:, None], rope == "half")
    ref.assert_within(out, qr, qr.abs() * ref.U16 + 3 * ref.U32 * qsize, "query")
    assert torch.equal(got.double(), vals)  # bf16 holds every row's values exactly
    # the same rows again into an empty cache, the query in place, no norm
    c2 = cache_like(pages, page, fmt)
    q2 = q[..., 128:].contiguous()
    assert run.append(c2, kv, None, cs, pos, slots, q_pe=q2, q_out=q2) is q2
    assert torch.equal(q2, out)
    raw = ref.row_values(c2.view(pages * page, -1)[slots.long()])[:, :512]
    if fmt == "bf16":
        assert torch.equal(raw, kv[:, :512].double())
    else:
        assert float(((raw - kv[:, :512].double()).abs() / kv[:, :512].double().abs().clamp_min(0.05)).max()) <= 2.0**-4


def test_append_codes_are_the_definitions():
    """Each of half a million MXFP8 codes is the nearest one (ties to even) to the 64-bit norm, under
    the least power of two that holds its 32 values: none next to a border falls to the other side."""
    from sgl_amd_mono.moe.latent import cache_like

    g, run, t = _gen(31), _runner(1), 1021
    kv, w = _randn(g, t, 576), (1 + 0.1 * torch.randn(512, generator=g, device="cuda")).to(BF)
    cache, rows = cache_like(t, 1, "mxfp8"), torch.arange(t, device="cuda")
    run.append(cache, kv, w, _cos_sin(1), torch.zeros_like(rows), rows)
    c = ref.norm(kv[:, :512], w, float(torch.tensor(1e-6))).view(t, 16, 32)
    sc = torch.exp2(torch.ceil(torch.log2(c.abs().amax(-1, keepdim=True) / 448)))
    a = (c / sc).abs()
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0**-6))) - 3)
    want = (c.sign() * torch.round(a / step) * step * sc).view(t, 512)
    assert torch.equal(ref.row_values(cache.view(t, -1))[:, :512], want)


def test_append_skips_padding_and_records_bad_indices():
    from sgl_amd_mono.moe.latent import cache_like

    g = _gen(5)
    for fmt in ("bf16", "mxfp8"):
        run = _runner(4)
        cache = cache_like(4, 8, fmt)
        kv, cs = _randn(g, 5, 576), _cos_sin(16)
        q = _randn(g, 5, 4, 64)
        pos = torch.tensor([1, 2, 3, 4, 5], device="cuda")
        slots = torch.tensor([3, -1, 31, -7, 0], device="cuda")
        run.append(cache, kv, None, cs, pos, slots)
        run.raise_on_device_error()
        assert (cache.view(32, -1) != 0).any(1).nonzero().flatten().tolist() == [0, 3, 31]
        # a slot behind the cache, a position behind the table
        before = cache.clone()
        out = torch.full((5, 4, 64), 7.0, dtype=BF, device="cuda")
        run.append(cache, kv, None, cs, torch.tensor([1, 16, 3, -1, 5], device="cuda"),
                   torch.tensor([32, 4, 1 << 40, 5, -1], device="cuda"), q_pe=q, q_out=out)  # fmt: skip
        assert torch.equal(cache, before)
        assert bool((out[1] == 7).all()) and bool((out[3] == 7).all()) and not bool((out[0] == 7).all())
        with pytest.raises(RuntimeError, match="outside"):
            run.raise_on_device_error()
        run.clear_errors()
        run.raise_on_device_error()
        rows = run.rows(cache, torch.tensor([3, -1, 32], device="cuda"))
        assert bool((rows[1:] == 0).all()) and bool((rows[0] != 0).any())
        with pytest.raises(RuntimeError, match="a slot outside the cache, at token 2"):
            run.raise_on_device_error()


def test_append_extremes():
    """Zero rows, the largest values, NaN and infinity in a row."""
    from sgl_amd_mono.moe.latent import cache_like

    run = _runner(1)
    kv = torch.zeros(6, 576, dtype=BF, device="cuda")
    kv[1, :512] = 1e-30
    kv[2, :512] = 3e38  # its squares pass fp32
    kv[3, 5] = NAN
    kv[4, 5] = INF
    kv[5, 0] = 1.0  # one value among zeros
    w = torch.ones(512, dtype=BF, device="cuda")
    pos, slots = torch.zeros(6, dtype=torch.int64, device="cuda"), torch.arange(6, device="cuda")
    for fmt in ("bf16", "mxfp8"):
        cache = cache_like(6, 1, fmt)
        run.append(cache, kv, w, _cos_sin(1), pos, slots)
        got = run.rows(cache, slots).double().cpu()
        assert bool((got[0] == 0).all()) and bool((got[2, :512] == 1).all())
        assert float((got[1, :512] - 1e-27).abs().max()) <= 1e-27 * 2.0**-3
        assert bool(got[3, :512].isnan().all())
        assert bool(got[4, 5].isnan())
        assert abs(float(got[5, 0]) - 512**0.5) <= 512**0.5 * 2.0**-4 and bool((got[5, 1:] == 0).all())


# ---------------------------------------------------------------- attend
def _attend_case(fmt, heads, page, lens, n=1, starts=None, seed=0, stride=0):
    g = _gen(seed)
    seqs, t = len(lens), (len(lens) * n if starts is None else starts[-1])
    table, pages = _tables(g, seqs, max(max(lens), 1), page)
    cache = ref.random_cache(pages, page, fmt, g, "cuda")
    if stride:  # the head axis outermost, rows padded
        q_lat = _randn(g, heads, t, 512 + stride)[..., :512].transpose(0, 1)
        q_pe = _randn(g, t, heads, 128 + 64)[..., 128:]
    else:
        q_lat, q_pe = _randn(g, t, heads, 512), _randn(g, t, heads, 64)
    return cache, q_lat, q_pe, table, torch.tensor(lens, dtype=torch.int32, device="cuda")


def _check_attend(run, fmt, heads, page, lens, n=1, starts=None, seed=0, stride=0, scale=SCALE):
    cache, q_lat, q_pe, table, dl = _attend_case(fmt, heads, page, lens, n, starts, seed, stride)
    t = q_lat.shape[0]
    ds = None if starts is None else torch.tensor(starts, dtype=torch.int32, device="cuda")
    lse = torch.empty(t, heads, device="cuda")
    out = run.attend(cache, q_lat, q_pe, table, dl, q_starts=ds, lse=lse)
    torch.cuda.synchronize()
    run.raise_on_device_error()
    r, rl, bound, lbound = ref.attend(cache, q_lat, q_pe, table, lens, scale, starts)
    ref.assert_within(out, r, bound, "out")
    ref.assert_within(lse, rl, lbound, "lse")


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("heads", [1, 16, 20, 32, 64, 128])
def test_attend_heads(fmt, heads):
    print(f"\nattend {fmt} heads={heads}", flush=True)
    _check_attend(_runner(heads), fmt, heads, 16, [1, 63, 64, 65, 300, 0, 17], seed=heads, stride=8 * (heads % 3))


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("page", [1, 2, 16, 64, 128, 1024])
def test_attend_pages(fmt, page):
    print(f"\nattend {fmt} page={page}", flush=True)
    _check_attend(_runner(8), fmt, 8, page, [1500, 1, 129, 1024, 1023, 2], seed=page)


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("heads,lens,n", [(16, [5, 64, 190, 0, 2], 2), (32, [66, 3, 400], 4), (64, [129, 1000], 5), (1, [200, 70], 65), (128, [4, 260], 3)])
def test_attend_several_queries(fmt, heads, lens, n):
    """A sequence's last n tokens, causal among them; sequences shorter than n leave rows empty."""
    print(f"\nattend {fmt} heads={heads} n={n}", flush=True)
    _check_attend(_runner(heads), fmt, heads, 16, lens, n, seed=n)


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("heads", [8, 64])
def test_attend_ragged_queries(fmt, heads):
    """q_starts: sequences with no, one and many query tokens; rows behind the last stay."""
    print(f"\nattend ragged {fmt} heads={heads}", flush=True)
    run = _runner(heads)
    starts, lens = [0, 3, 3, 4, 24, 24], [70, 50, 129, 40, 9]
    _check_attend(run, fmt, heads, 16, lens, starts=starts, seed=3)
    cache, q_lat, q_pe, table, dl = _attend_case(fmt, heads, 16, lens, starts=starts, seed=3)
    wide = torch.full((30, heads, 512), 7.0, dtype=BF, device="cuda")
    lse = torch.full((30, heads), 7.0, device="cuda")
    pad = lambda q: torch.cat([q, torch.full((6, *q.shape[1:]), NAN, dtype=BF, device="cuda")])  # noqa: E731
    ds = torch.tensor(starts, dtype=torch.int32, device="cuda")
    run.attend(cache, pad(q_lat), pad(q_pe), table, dl, q_starts=ds, out=wide, lse=lse)
    exact = run.attend(cache, q_lat, q_pe, table, dl, q_starts=ds)
    assert torch.equal(wide[:24], exact) and bool((wide[24:] == 7).all()) and bool((lse[24:] == 7).all())


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("heads,lens", [(32, [20011]), (16, [9000, 1, 17000, 0, 300]), (64, [16385, 64])])
def test_attend_long(fmt, heads, lens):
    """Sequences cut into shares over the whole card, and joined."""
    print(f"\nattend long {fmt} heads={heads} {lens}", flush=True)
    _check_attend(_runner(heads), fmt, heads, 64, lens, seed=1)


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
def test_attend_many_sequences(fmt):
    print(f"\nattend many {fmt}", flush=True)
    lens = [(i * 37) % 131 for i in range(512)]
    _check_attend(_runner(4), fmt, 4, 8, lens, seed=2)


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
def test_attend_scores_far_apart(fmt):
    """Scores whose differences pass what exp holds, rising and falling along the sequence: the
    running maximum moves at almost every tile, and the last tokens alone count (or the first)."""
    run, g = _runner(2), _gen(9)
    lens = [700]
    cache, q_lat, q_pe, table, dl = _attend_case(fmt, 2, 1, lens, seed=4)
    rows = table[0, :700].long()
    ramp = torch.linspace(0, 30, 700, device="cuda")[:, None].expand(700, 64).to(BF)
    flat = cache.view(-1, cache.shape[-1])
    if fmt == "bf16":
        flat[rows, 512:] = ramp
    else:
        flat[rows, 528:] = ramp.contiguous().view(torch.uint8)
    q_pe[:, 0] = 30.0
    q_pe[:, 1] = -30.0
    out = run.attend(cache, q_lat, q_pe, table, dl)
    r, _, bound, _ = ref.attend(cache, q_lat, q_pe, table, lens, SCALE)
    ref.assert_within(out, r, bound, "out")


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("heads", [8, 32])
def test_attend_garbage_out_of_sight(fmt, heads):
    """NaN in every row behind a sequence's end, in the rest of its last page and in pages of no
    sequence; page entries behind the length point anywhere."""
    run = _runner(heads)
    lens = [70, 1, 64, 333]
    cache, q_lat, q_pe, table, dl = _attend_case(fmt, heads, 16, lens, seed=6)
    want = run.attend(cache, q_lat, q_pe, table, dl).clone()
    flat = cache.view(-1, cache.shape[-1])
    used = torch.zeros(flat.shape[0], dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens):
        at = torch.arange(n, device="cuda")
        used[table[b].long()[at // 16] * 16 + at % 16] = True
    flat[~used] = NAN if fmt == "bf16" else 0xFF
    t2 = table.clone()
    for b, n in enumerate(lens):
        t2[b, -(-n // 16) :] = [-1, 1 << 30, -(1 << 31), 12345][b]
    assert torch.equal(run.attend(cache, q_lat, q_pe, t2, dl), want)
    run.raise_on_device_error()


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("heads,n", [(8, 4), (32, 3), (64, 2)])
def test_attend_non_finite_tokens_reach_only_their_queries(fmt, heads, n):
    """A later query token's own row holds NaN or infinity: the earlier queries do not see it, and
    their rows stay as they were; those that see it are not finite."""
    run = _runner(heads)
    lens = [70, 64 + n, 200]
    cache, q_lat, q_pe, table, dl = _attend_case(fmt, heads, 16, lens, n, seed=8)
    want = run.attend(cache, q_lat, q_pe, table, dl).clone()
    flat = cache.view(-1, cache.shape[-1])
    for b, length in enumerate(lens):  # the last token of each
        at = int(table[b, (length - 1) // 16]) * 16 + (length - 1) % 16
        if fmt == "bf16":
            flat[at, 100 + b] = [NAN, INF, -INF][b]
        else:
            flat[at, 100 + b] = 0x7F
    out = run.attend(cache, q_lat, q_pe, table, dl)
    last = torch.arange(n - 1, 3 * n, n, device="cuda")
    first = torch.ones(3 * n, dtype=torch.bool, device="cuda")
    first[last] = False
    assert torch.equal(out[first], want[first])
    assert not bool(out[last].isfinite().all(-1).any())


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("scale", [0.0, -0.09, 1.0])
def test_attend_scales(fmt, scale):
    """No scale at all (a plain mean), a negative one, and one that leaves a few tokens."""
    from sgl_amd_mono.moe.latent import LatentRunner

    print(f"\nattend {fmt} scale={scale}", flush=True)
    _check_attend(LatentRunner(24, scale=scale), fmt, 24, 16, [130, 1, 700], 2, seed=18, scale=scale)


@pytest.mark.parametrize("seed", range(24))
def test_attend_at_random(seed):
    """Heads, pages, lengths (some empty), query counts and strides at random."""
    import random

    r = random.Random(seed)
    heads, page = r.choice([1, 3, 8, 12, 17, 32, 40, 64, 127, 128]), r.choice([1, 2, 4, 8, 16, 32, 64, 256])
    seqs = r.choice([1, 2, 5, 13, 37])
    lens = [0 if r.random() < 0.15 else int(10 ** r.uniform(0, 3.5)) for _ in range(seqs)]
    fmt, n, starts = r.choice(["bf16", "mxfp8"]), r.choice([1, 1, 2, 3, 7]), None
    if r.random() < 0.5:
        starts = [0]
        for _ in range(seqs):
            starts.append(starts[-1] + r.choice([0, 1, 1, 2, 4, 9]))
        starts[-1] += starts[-1] == 0
    print(f"\nattend {fmt} heads={heads} page={page} n={n} starts={starts} lens={lens}", flush=True)
    _check_attend(_runner(heads), fmt, heads, page, lens, n, starts, seed=seed, stride=8 * r.choice([0, 1, 5]))


# Work of more than 4096 tiles of 64 query rows (a row tile counts its tiles of 32 cached tokens and 8)
# is taken 64 rows at a time
@pytest.mark.parametrize("fmt,page", [("bf16", 1), ("bf16", 64), ("mxfp8", 1), ("mxfp8", 64)])
@pytest.mark.parametrize("heads,lens,n,starts", [
    (128, [700, 641, 5, 0, 300, 64], 48, None),
    (12, [451, 1000, 460, 9, 77], 0, [0, 451, 451, 902, 1353, 1360]),
    (20, [2500, 1, 129], 0, [0, 600, 601, 605]),
    (64, [32] * 101 + [0, 6000], 5, None),
])  # fmt: skip
def test_attend_tall(fmt, page, heads, lens, n, starts):
    print(f"\nattend tall {fmt} page={page} heads={heads} n={n} {lens[:6]}", flush=True)
    t = [n] * len(lens) if starts is None else [b - a for a, b in zip(starts, starts[1:])]
    tiles = sum(-(-c * heads // 64) * (-(-m // 32) + 8) for c, m in zip(t, lens) if m)
    assert tiles > 4096, tiles
    _check_attend(_runner(heads), fmt, heads, page, lens, n, starts, seed=heads, stride=8 * (heads == 20))


@pytest.mark.parametrize("fmt,page", [("bf16", 16), ("bf16", 64), ("mxfp8", 16), ("mxfp8", 64)])
def test_attend_tall_sees_only_what_it_may(fmt, page):
    """As the two tests above of garbage out of sight and of non-finite tokens, 64 rows at a time."""
    heads, n, lens = 64, 64, [200, 300, 130, 1000]
    run = _runner(heads)
    cache, q_lat, q_pe, table, dl = _attend_case(fmt, heads, page, lens, n, seed=15)
    want = run.attend(cache, q_lat, q_pe, table, dl).clone()
    flat = cache.view(-1, cache.shape[-1])
    used = torch.zeros(flat.shape[0], dtype=torch.bool, device="cuda")
    t2 = table.clone()
    for b, m in enumerate(lens):
        at = torch.arange(m, device="cuda")
        used[table[b].long()[at // page] * page + at % page] = True
        t2[b, -(-m // page) :] = [-1, 1 << 30, -(1 << 31), 12345][b]
    flat[~used] = NAN if fmt == "bf16" else 0xFF
    assert torch.equal(run.attend(cache, q_lat, q_pe, t2, dl), want)
    run.raise_on_device_error()
    for b, m in enumerate(lens):  # the last token of each
        at = int(table[b, (m - 1) // page]) * page + (m - 1) % page
        flat[at, 100 + b] = [NAN, INF, -INF, NAN][b] if fmt == "bf16" else 0x7F
    out = run.attend(cache, q_lat, q_pe, t2, dl)
    last = torch.arange(n - 1, 4 * n, n, device="cuda")
    first = torch.ones(4 * n, dtype=torch.bool, device="cuda")
    first[last] = False
    assert torch.equal(out[first], want[first])
    assert not bool(out[last].isfinite().all(-1).any())
    t2[2, 1] = cache.shape[0]
    run.attend(cache, q_lat, q_pe, t2, dl)
    with pytest.raises(RuntimeError, match="a page outside the cache, at sequence 2"):
        run.raise_on_device_error()
    run.clear_errors()


def test_attend_non_finite_query_stays_in_its_row():
    run = _runner(16)
    cache, q_lat, q_pe, table, dl = _attend_case("bf16", 16, 16, [100, 30], seed=11)
    want = run.attend(cache, q_lat, q_pe, table, dl).clone()
    q_lat[0, 3, 7], q_pe[1, 5, 2] = NAN, INF
    out = run.attend(cache, q_lat, q_pe, table, dl)
    hit = torch.zeros(2, 16, dtype=torch.bool, device="cuda")
    hit[0, 3] = hit[1, 5] = True
    assert torch.equal(out[~hit], want[~hit]) and not bool(out[hit].isfinite().any())


def test_attend_records_bad_pages_lengths_and_starts():
    """Pages outside the cache count as rows of zeros, lengths and starts are clamped; all recorded."""
    run = _runner(8)
    cache, q_lat, q_pe, table, dl = _attend_case("bf16", 8, 16, [40, 100], seed=12)
    bad = table.clone()
    bad[1, 2] = cache.shape[0]
    run.attend(cache, q_lat, q_pe, bad, dl)
    with pytest.raises(RuntimeError, match="a page outside the cache, at sequence 1"):
        run.raise_on_device_error()
    run.clear_errors()
    full = table.shape[1] * 16
    got = run.attend(cache, q_lat, q_pe, table, torch.tensor([full + 1, -5], dtype=torch.int32, device="cuda"))
    assert torch.equal(got, run.attend(cache, q_lat, q_pe, table, torch.tensor([full, 0], dtype=torch.int32, device="cuda")))
    assert bool((got[1] == 0).all())
    with pytest.raises(RuntimeError, match="a length or query start"):
        run.raise_on_device_error()
    run.clear_errors()
    for starts in ([0, 3, 1], [-4, 1, 2], [0, 1, 1 << 30]):
        run.attend(cache, q_lat, q_pe, table, dl, q_starts=torch.tensor(starts, dtype=torch.int32, device="cuda"))
        with pytest.raises(RuntimeError, match="a length or query start"):
            run.raise_on_device_error()
        run.clear_errors()


def test_attend_query_starts_that_run_backwards():
    """They would give rows to several sequences: nothing is attended."""
    run = _runner(64)
    cache, q_lat, q_pe, table, dl = _attend_case("bf16", 64, 16, [40, 100, 60], starts=[0, 2, 4, 6], seed=17)
    for starts in ([0, 6, 0, 6], [0, 4, 3, 6]):
        out = torch.full((6, 64, 512), 7.0, dtype=BF, device="cuda")
        run.attend(cache, q_lat, q_pe, table, dl, q_starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), out=out)
        assert bool((out == 7).all())
        with pytest.raises(RuntimeError, match="a length or query start"):
            run.raise_on_device_error()
        run.clear_errors()
    run.attend(cache, q_lat, q_pe, table, dl, q_starts=torch.tensor([0, 2, 4, 6], dtype=torch.int32, device="cuda"), out=out)
    assert torch.equal(out, run.attend(cache, q_lat, q_pe, table, dl))
    run.raise_on_device_error()


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
def test_attend_offsets_past_32_bits(fmt):
    """A cache of more than 2^32 bytes, its last pages in use."""
    print(f"\nattend far {fmt}", flush=True)
    run, g = _runner(16), _gen(13)
    row = 1152 if fmt == "bf16" else 656
    pages = (1 << 32) // (row * 64) + 20
    small = ref.random_cache(12, 64, fmt, g, "cuda")
    cache = torch.empty(pages, *small.shape[1:], dtype=small.dtype, device="cuda")
    cache[-12:] = small
    table = torch.arange(12, dtype=torch.int32, device="cuda").view(2, 6)
    q_lat, q_pe = _randn(g, 2, 16, 512), _randn(g, 2, 16, 64)
    dl = torch.tensor([380, 200], dtype=torch.int32, device="cuda")
    want = run.attend(small, q_lat, q_pe, table, dl)
    assert torch.equal(run.attend(cache, q_lat, q_pe, table + (pages - 12), dl), want)
    slots = torch.arange(5, device="cuda") + (pages * 64 - 5)
    kv, cs, pos = _randn(g, 5, 576), _cos_sin(8), torch.arange(5, device="cuda")
    run.append(cache, kv, None, cs, pos, slots)
    run.append(small, kv, None, cs, pos, torch.arange(5, device="cuda") + (12 * 64 - 5))
    assert torch.equal(cache[-12:], small)
    assert torch.equal(run.rows(cache, slots), run.rows(small, slots - (pages - 12) * 64))


def test_attend_same_bits_every_time():
    run = _runner(32)
    cache, q_lat, q_pe, table, dl = _attend_case("mxfp8", 32, 64, [5000, 64, 9000, 1], seed=14)
    want = run.attend(cache, q_lat, q_pe, table, dl).clone()
    for _ in range(5):
        assert torch.equal(run.attend(cache, q_lat, q_pe, table, dl), want)


# ---------------------------------------------------------------- the heads' products
@pytest.mark.parametrize("tokens,heads", [(1, 1), (5, 16), (48, 32), (67, 3), (130, 64)])
def test_absorb_and_expand(tokens, heads):
    print(f"\nproject tokens={tokens} heads={heads}", flush=True)
    from sgl_amd_mono.moe.latent import LatentWeights

    g, run = _gen(tokens), _runner(heads)
    w = LatentWeights(norm=_randn(g, 512), kv_b=_randn(g, heads * 256, 512))
    wk = w.kv_b.double().view(heads, 256, 512)
    q = _randn(g, tokens, heads, 192)[..., :128]
    x, a = q.double().transpose(0, 1), q.double().abs().transpose(0, 1)
    want = (x @ wk[:, :128]).transpose(0, 1)
    size = (a @ wk[:, :128].abs()).transpose(0, 1)
    ref.assert_within(run.absorb(w, q), want, want.abs() * ref.U16 + 130 * ref.U32 * size, "absorb")
    o = _randn(g, heads, tokens, 512).transpose(0, 1)
    out = torch.empty(heads, tokens, 128, dtype=BF, device="cuda").transpose(0, 1)
    x, a = o.double().transpose(0, 1), o.double().abs().transpose(0, 1)
    want = (x @ wk[:, 128:].transpose(1, 2)).transpose(0, 1)
    size = (a @ wk[:, 128:].abs().transpose(1, 2)).transpose(0, 1)
    assert run.expand(w, o, out=out) is out
    ref.assert_within(out, want, want.abs() * ref.U16 + 514 * ref.U32 * size, "expand")


# ---------------------------------------------------------------- together
def _layer(fmt, heads, lens, n, page=16, seed=0):
    from sgl_amd_mono.moe.latent import LatentWeights

    g = _gen(seed)
    seqs, t = len(lens), len(lens) * n
    table, pages = _tables(g, seqs, max(lens), page)
    at = torch.tensor([max(0, m - n + i) for m in lens for i in range(n)], device="cuda")
    seq = torch.arange(seqs, device="cuda").repeat_interleave(n)
    slots = table[seq, at // page].long() * page + at % page
    slots[torch.tensor([m - n + i < 0 for m in lens for i in range(n)], device="cuda")] = -1
    return dict(
        w=LatentWeights(norm=(1 + 0.1 * torch.randn(512, generator=g, device="cuda")).to(BF),
                        kv_b=(torch.randn(heads * 256, 512, generator=g, device="cuda") * 512**-0.5).to(BF)),
        cache=ref.random_cache(pages, page, fmt, g, "cuda"), q=_randn(g, t, heads, 192), kv=_randn(g, t, 576),
        cos_sin=_cos_sin(max(lens)), positions=at, slots=slots, table=table,
        lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
    )  # fmt: skip


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("heads,lens,n", [(32, [1, 70, 400, 64], 1), (16, [90, 33], 4), (64, [5, 0, 130], 1), (128, [2000], 2)])
def test_attention_is_its_parts(fmt, heads, lens, n):
    """One call against append, absorb, attend and expand, bit for bit, and against 64 bits.

    Four bf16 roundings lie on the way (absorbed query, rotated query, numerators, output; the
    attended latents stay in fp32), each off by at most 2^-8 of its value and 2^-8 / sqrt(3) in the
    mean square; those of the query reach the output through scores of spread about 1. Their root
    mean square is below sqrt(4 / 3) 2^-8 = 1.16 2^-8 of the output's; twice that is asked for."""
    print(f"\nattention {fmt} heads={heads} lens={lens} n={n}", flush=True)
    d = _layer(fmt, heads, lens, n, seed=heads)
    run = _runner(heads)
    c2 = d["cache"].clone()
    out = run.attention(**d)
    torch.cuda.synchronize()
    run.raise_on_device_error()
    w, q = d["w"], d["q"]
    q_pe = run.append(c2, d["kv"], w.norm, d["cos_sin"], d["positions"], d["slots"], q_pe=q[..., 128:])
    o = torch.empty(q.shape[0], heads, 512, device="cuda")
    run.attend(c2, run.absorb(w, q[..., :128]), q_pe, d["table"], d["lens"], out=o)
    assert torch.equal(c2, d["cache"])
    assert torch.equal(run.expand(w, o), out)
    wk = w.kv_b.double().view(heads, 256, 512)
    ql = (q[..., :128].double().transpose(0, 1) @ wk[:, :128]).transpose(0, 1)
    qr, _ = ref.rotate(q[..., 128:].double(), d["cos_sin"][d["positions"]][:, None], False)
    want, *_ = ref.attend(d["cache"], ql, qr, d["table"], lens, SCALE)
    want = (want.transpose(0, 1) @ wk[:, 128:].transpose(1, 2)).transpose(0, 1)
    err = float((out.double() - want).norm() / want.norm())
    assert err <= 2 * 1.16 * ref.U16, err


@pytest.mark.parametrize("fmt,page", [("bf16", 64), ("mxfp8", 1)])
@pytest.mark.parametrize("heads,lens,n", [(32, [1, 70, 0, 4000], 1), (64, [500, 33], 4)])
def test_attend_in_fp32(fmt, page, heads, lens, n):
    """fp32 outputs, cut sequences' among them, round to the bf16 ones bit for bit; W_UV of them is
    off by the output's rounding 2^-8, the 2^-17 that two bf16 parts leave of a value (each part's
    rounding is within 2^-8 of what it rounds: 2^-16), and 512 fp32 sums."""
    print(f"\nattend fp32 {fmt} page={page} heads={heads} lens={lens} n={n}", flush=True)
    d, run = _layer(fmt, heads, lens, n, seed=3, page=page), _runner(heads)
    w, q_pe = d["w"], d["q"][..., 128:]
    ql = run.absorb(w, d["q"][..., :128])
    wide = torch.full((q_pe.shape[0], heads, 520), 7.0, device="cuda")
    o = run.attend(d["cache"], ql, q_pe, d["table"], d["lens"], out=wide[..., :512])
    assert o.dtype == torch.float32 and bool((wide[..., 512:] == 7).all())
    assert torch.equal(o.to(BF), run.attend(d["cache"], ql, q_pe, d["table"], d["lens"]))
    wv = w.kv_b.double().view(heads, 256, 512)[:, 128:].transpose(1, 2)
    want = (o.double().transpose(0, 1) @ wv).transpose(0, 1)
    size = (o.double().abs().transpose(0, 1) @ wv.abs()).transpose(0, 1)
    bound = (ref.U16 * want.abs() + (2.0**-16 + 520 * ref.U32) * size) * 1.01
    ref.assert_within(run.expand(w, o), want, bound, "expand of fp32")
    run.raise_on_device_error()


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
def test_attention_in_a_graph(fmt):
    """A captured step replayed with new lengths, rows and queries in its buffers, eager work on
    the same runner in between; another stream."""
    d, run = _layer(fmt, 32, [300, 70, 1, 4000], 1, seed=21), _runner(32)
    first, base = d["lens"].clone(), d["cache"].clone()
    out = torch.empty(4, 32, 128, dtype=BF, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        run.attention(**d, out=out)
        with torch.cuda.graph(g, stream=s):
            run.attention(**d, out=out)
    torch.cuda.current_stream().wait_stream(s)
    q0 = d["q"].clone()
    for rep, lens in enumerate([[300, 70, 1, 4000], [10, 70, 1, 64], [300, 1, 0, 2500], [300, 70, 1, 4000]]):
        d["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        d["q"].copy_(q0 * (1 + rep % 3))
        d["cache"].copy_(base)
        out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        got, after = out.clone(), d["cache"].clone()
        d["cache"].copy_(base)
        want = run.attention(**d)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(after, d["cache"]), rep
    d["lens"].copy_(first)
    run.raise_on_device_error()


def test_two_runners_on_two_streams():
    a, b = _layer("bf16", 32, [5000, 80], 1, seed=31), _layer("mxfp8", 32, [300, 7000], 1, seed=32)
    ra, rb = _runner(32), _runner(32)
    wa, wb = ra.attention(**a).clone(), rb.attention(**b).clone()
    torch.cuda.synchronize()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(4):
        with torch.cuda.stream(sa):
            got.append((ra.attention(**a), wa))
        with torch.cuda.stream(sb):
            got.append((rb.attention(**b), wb))
    torch.cuda.synchronize()
    for x, y in got:
        assert torch.equal(x, y)


def test_decode_steps_then_the_moe_block():
    """Three decode steps of a layer's attention, each reading the rows that the last one stored,
    then the MoE block on rows of its output, as a decode layer runs them."""
    from oracle import gen
    from sgl_amd_mono.moe.presets import PRESETS, workload_dict
    from sgl_amd_mono.moe.runner import MoeRunner, MoeWeights

    heads, seqs, page = 8, 3, 4
    d, run = _layer("bf16", heads, [9, 5, 12], 1, page=page, seed=41), _runner(heads)
    g = _gen(42)
    lens = torch.tensor([6, 2, 9], dtype=torch.int32, device="cuda")
    for step in range(3):
        lens = lens + 1
        at = (lens - 1).long()
        slots = d["table"][torch.arange(seqs, device="cuda"), at // page].long() * page + at % page
        q, kv = _randn(g, seqs, heads, 192), _randn(g, seqs, 576)
        out = run.attention(d["w"], d["cache"], q, kv, d["cos_sin"], at, slots, d["table"], lens)
    run.raise_on_device_error()
    wk = d["w"].kv_b.double().view(heads, 256, 512)
    ql = (q[..., :128].double().transpose(0, 1) @ wk[:, :128]).transpose(0, 1)
    qr, _ = ref.rotate(q[..., 128:].double(), d["cos_sin"][at][:, None], False)
    want, *_ = ref.attend(d["cache"], ql, qr, d["table"], lens.tolist(), SCALE)
    want = (want.transpose(0, 1) @ wk[:, 128:].transpose(1, 2)).transpose(0, 1)
    assert float((out.double() - want).norm() / want.norm()) <= 2 * 1.3 * ref.U16
    p = workload_dict("cfg1_plumbing_fp8")
    dense, ex = gen.make_dense(p, 0), gen.LazyExperts(p, 0)
    st = {k: torch.stack([torch.as_tensor(ex.get(e)[i]) for e in range(p["experts"])]).cuda()
          for i, k in enumerate(("w13", "w13_s", "w2", "w2_s"))}  # fmt: skip
    mw = MoeWeights(**{k: v.cuda() for k, v in dense.items() if k != "norm"}, **st)
    moe = MoeRunner(PRESETS["plumbing_fp8"])
    x = out.reshape(seqs, heads * 128)
    assert bool(moe.moe(mw, x).isfinite().all())
    moe.raise_on_device_error()


# ---------------------------------------------------------------- rows of no sequence, tokens that were not stored
def _ragged_layer(fmt, heads, lens, starts, tokens, seed):
    """A step of ``tokens`` rows of which the sequences have those from ``starts``, as in a step padded
    to a captured size; the others are padded tokens (slot -1)."""
    cnt = [b - a for a, b in zip(starts, starts[1:])]
    d = _layer(fmt, heads, lens, 1, seed=seed)
    g = _gen(seed + 1)
    pos, slots = torch.zeros(tokens, dtype=torch.int64, device="cuda"), torch.full((tokens,), -1, device="cuda")
    for b, (s, n) in enumerate(zip(starts, cnt)):
        for i in range(n):
            at = lens[b] - n + i
            if at >= 0:
                pos[s + i] = at
                slots[s + i] = d["table"][b, at // 16].long() * 16 + at % 16
    d.update(q=_randn(g, tokens, heads, 192), kv=_randn(g, tokens, 576), positions=pos, slots=slots,
             q_starts=torch.tensor(starts, dtype=torch.int32, device="cuda"))  # fmt: skip
    return d


def _by_parts(run, d, rows):
    """The step's output by its parts, of the rows that the sequences have."""
    w, q, c2 = d["w"], d["q"], d["cache"].clone()
    q_pe = run.append(c2, d["kv"], w.norm, d["cos_sin"], d["positions"], d["slots"], q_pe=q[..., 128:])
    o = torch.zeros(q.shape[0], run.heads, 512, device="cuda")
    run.attend(c2, run.absorb(w, q[..., :128]), q_pe, d["table"], d["lens"], q_starts=d["q_starts"], out=o)
    return run.expand(w, o)[rows], c2


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("heads", [8, 64])
@pytest.mark.parametrize("starts", [[0, 3, 3, 4, 24], [2, 3, 7, 8, 10], [5, 5, 5, 5, 5]])
def test_attention_leaves_rows_of_no_sequence(fmt, heads, starts):
    """q_starts that cover some of the step's rows: the others stay as they were, also on a runner whose
    last call was another step, whose rows would otherwise come back."""
    print(f"\nattention {fmt} heads={heads} starts={starts}", flush=True)
    t, lens = 30, [70, 50, 129, 400]
    run = _runner(heads)
    first = _ragged_layer(fmt, heads, lens, [0, 10, 20, 29, 30], t, seed=51)
    run.attention(**first)
    d = _ragged_layer(fmt, heads, lens, starts, t, seed=61)
    rows = slice(starts[0], starts[-1])
    want, after = _by_parts(_runner(heads), d, rows)
    out = torch.full((t, heads, 128), 7.0, dtype=BF, device="cuda")
    assert run.attention(**d, out=out) is out
    run.raise_on_device_error()
    assert torch.equal(out[rows], want) and torch.equal(d["cache"], after)
    out[rows] = 7.0
    assert bool((out == 7).all())


def test_attention_of_starts_that_run_backwards():
    run, lens = _runner(32), [70, 50, 129]
    run.attention(**_ragged_layer("bf16", 32, lens, [0, 1, 5, 6], 6, seed=51))
    run.raise_on_device_error()
    d = _ragged_layer("bf16", 32, lens, [0, 2, 4, 6], 6, seed=61)
    for starts in ([0, 4, 3, 6], [0, 6, 0, 6], [4, 5, 6, 0]):
        d["q_starts"].copy_(torch.tensor(starts, dtype=torch.int32))
        out = torch.full((6, 32, 128), 7.0, dtype=BF, device="cuda")
        run.attention(**d, out=out)
        assert bool((out == 7).all())
        with pytest.raises(RuntimeError, match="a length or query start"):
            run.raise_on_device_error()
        run.clear_errors()
    d["q_starts"].copy_(torch.tensor([0, 2, 4, 6], dtype=torch.int32))
    want, _ = _by_parts(_runner(32), d, slice(0, 6))
    assert torch.equal(run.attention(**d), want)
    run.raise_on_device_error()


def test_attention_with_query_starts_in_a_graph():
    """A captured step padded to 16 rows, replayed with other starts."""
    t, heads, lens = 16, 32, [70, 50, 129, 400]
    run, eager = _runner(heads), _runner(heads)
    d = _ragged_layer("mxfp8", heads, lens, [0, 4, 8, 12, 16], t, seed=71)
    out, base = torch.empty(t, heads, 128, dtype=BF, device="cuda"), d["cache"].clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        run.attention(**d, out=out)
        with torch.cuda.graph(g, stream=s):
            run.attention(**d, out=out)
    torch.cuda.current_stream().wait_stream(s)
    for rep, starts in enumerate([[0, 4, 8, 12, 16], [0, 1, 2, 3, 4], [3, 3, 8, 8, 9], [0, 0, 0, 0, 0], [0, 9, 10, 12, 16]]):
        n = _ragged_layer("mxfp8", heads, lens, starts, t, seed=72 + rep)
        for k in ("q", "kv", "positions", "slots", "q_starts"):
            d[k].copy_(n[k])
        d["cache"].copy_(base)
        want, after = _by_parts(eager, d, slice(starts[0], starts[-1]))
        out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[starts[0] : starts[-1]], want) and torch.equal(d["cache"], after), rep
        out[starts[0] : starts[-1]] = 7.0
        assert bool((out == 7).all()), rep
    run.raise_on_device_error()


@pytest.mark.parametrize("heads", [8, 64])
def test_rows_of_no_sequence_are_zeros_in_an_output_of_the_calls_own(heads):
    """Without ``out``, rows that q_starts gives to nobody do not hold what the memory held before."""
    t, lens = 30, [70, 50, 129, 400]
    run = _runner(heads)
    d = _ragged_layer("bf16", heads, lens, [2, 3, 7, 8, 10], t, seed=81)
    q_lat, q_pe = _randn(_gen(82), t, heads, 512), _randn(_gen(83), t, heads, 64)
    keep = torch.zeros(t, dtype=torch.bool, device="cuda")
    keep[2:10] = True
    for call in (lambda: run.attention(**d),
                 lambda: run.attend(d["cache"], q_lat, q_pe, d["table"], d["lens"], q_starts=d["q_starts"])):  # fmt: skip
        for _ in range(3):  # (memory that the allocator gives out again)
            dirty = torch.full((t, heads, 512), NAN, dtype=BF, device="cuda")
            small = torch.full((t, heads, 128), NAN, dtype=BF, device="cuda")
            del dirty, small
            out = call()
            assert bool((out[~keep] == 0).all()) and bool(out[keep].isfinite().all()) and bool((out[keep] != 0).any())
            del out
    run.raise_on_device_error()


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
def test_attention_of_a_token_that_was_not_stored_is_nan(fmt):
    """A position outside cos_sin or a slot outside the cache is recorded, and the token's output says so:
    it is NaN, not what the runner's last step left of its query. The other tokens have theirs."""
    heads, lens = 16, [70, 5, 400, 64, 33]
    run = _runner(heads)
    run.attention(**_layer(fmt, heads, lens, 1, seed=91))
    d = _layer(fmt, heads, lens, 1, seed=92)
    base = d["cache"].clone()
    want = run.attention(**d).clone()
    run.raise_on_device_error()
    ok = torch.tensor([0, 2, 4], device="cuda")
    for name, at, bad, why in (("positions", [1, 3], [d["cos_sin"].shape[0], -1], "a position outside cos_sin"),
                               ("slots", [1, 3], [base.shape[0] * 16, 1 << 40], "a slot outside the cache")):  # fmt: skip
        d["cache"].copy_(base)
        good = d[name].clone()
        d[name][at] = torch.tensor(bad, device="cuda")
        out = run.attention(**d)
        assert torch.equal(out[ok], want[ok])
        assert bool(out[at].isnan().all())
        with pytest.raises(RuntimeError, match=why):
            run.raise_on_device_error()
        run.clear_errors()
        d[name].copy_(good)
    d["cache"].copy_(base)
    assert torch.equal(run.attention(**d), want)
    run.raise_on_device_error()


def test_append_of_a_bad_position_in_an_output_of_its_own():
    """Without ``q_out``, the query rows of a position outside cos_sin are NaN, not what the memory held."""
    from sgl_amd_mono.moe.latent import cache_like

    g, run, t = _gen(97), _runner(4), 5
    cache, kv, q = cache_like(4, 8), _randn(g, t, 576), _randn(g, t, 4, 64)
    pos, slots = torch.tensor([1, 16, 3, -1, 5], device="cuda"), torch.arange(t, device="cuda")
    for _ in range(3):
        dirty = torch.full((t, 4, 64), 7.0, dtype=BF, device="cuda")
        del dirty
        out = run.append(cache, kv, None, _cos_sin(16), pos, slots, q_pe=q)
        assert bool(out[[1, 3]].isnan().all()) and bool(out[[0, 2, 4]].isfinite().all())
        del out
    with pytest.raises(RuntimeError, match="a position outside cos_sin"):
        run.raise_on_device_error()


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
def test_padded_tokens_need_no_position(fmt):
    """A token with a negative slot and a position outside cos_sin is a padded one: nothing is recorded, its
    query rows are zeros. With a position inside, they are rotated as the others are."""
    from sgl_amd_mono.moe.latent import cache_like

    g, run = _gen(95), _runner(4)
    cache, cs = cache_like(4, 8, fmt), _cos_sin(16)
    kv, q = _randn(g, 6, 576), _randn(g, 6, 4, 64)
    pos, slots = torch.tensor([1, -1, 3, 16, 5, 1 << 40], device="cuda"), torch.tensor([3, -1, 31, -7, -1, -1], device="cuda")
    out = torch.full((6, 4, 64), 7.0, dtype=BF, device="cuda")
    run.append(cache, kv, None, cs, pos, slots, q_pe=q, q_out=out)
    run.raise_on_device_error()
    assert (cache.view(32, -1) != 0).any(1).nonzero().flatten().tolist() == [3, 31]
    assert bool((out[[1, 3, 5]] == 0).all())
    real = torch.tensor([0, 2, 4], device="cuda")
    want, size = ref.rotate(q[real].double(), cs[pos[real]][:, None], False)
    ref.assert_within(out[real], want, want.abs() * ref.U16 + 3 * ref.U32 * size, "query")
    # a padded step: the padded sequences are empty, their tokens have neither slot nor position
    d = _layer(fmt, 16, [70, 400, 0, 0], 1, seed=96)
    run = _runner(16)
    base = d["cache"].clone()
    want = run.attention(**d).clone()
    d["cache"].copy_(base)
    d["positions"][2:] = torch.tensor([-1, 1 << 30], device="cuda")
    assert torch.equal(run.attention(**d), want) and bool((want[2:] == 0).all())
    run.raise_on_device_error()


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
def test_append_without_eps(fmt):
    """norm_eps 0 on rows whose root mean square's inverse passes fp32 (bf16's subnormals) or nearly so, and on
    ordinary ones: each is the norm's within the bound of ``test_append``."""
    from sgl_amd_mono.moe.latent import cache_like

    sizes = [2.0**-133, 2.0**-130, 2.0**-127, 2.0**-126, 2.0**-110, 2.0**-100, 2.0**-99, 2.0**-66, 1.0, 2.0**100]
    run, g, t = _runner(1, norm_eps=0.0), _gen(99), len(sizes)
    kv = torch.zeros(t, 576, dtype=BF, device="cuda")
    x = torch.randint(1, 4, (t, 512), generator=g, device="cuda") * (1 - 2 * torch.randint(0, 2, (t, 512), generator=g, device="cuda"))
    kv[:, :512] = (x.double() * torch.tensor(sizes, dtype=torch.float64, device="cuda")[:, None]).to(BF)  # exact
    assert torch.equal(kv[:, :512].double(), x.double() * torch.tensor(sizes, dtype=torch.float64, device="cuda")[:, None])
    w = (1 + 0.1 * torch.randn(512, generator=g, device="cuda")).to(BF)
    rows = torch.arange(t, device="cuda")
    cache = cache_like(t, 1, fmt)
    run.append(cache, kv, w, _cos_sin(1), torch.zeros_like(rows), rows)
    got = ref.row_values(cache.view(t, -1))[:, :512]
    c = ref.norm(kv[:, :512], w, 0.0)
    if fmt == "bf16":
        ref.assert_within(got, c, c.abs() * (ref.U16 + 2 * 540 * ref.U32), "latent")
    else:
        sc = torch.exp2(torch.ceil(torch.log2(c.view(t, 16, 32).abs().amax(-1) / 448))).repeat_interleave(32, 1)
        ref.assert_within(got, c, torch.maximum(c.abs() * 2.0**-4, sc * 2.0**-10) * (1 + 1e-4), "latent")
    run.raise_on_device_error()


@pytest.mark.parametrize("page", [1, 64])
@pytest.mark.parametrize("heads,lens,n", [(32, [1, 70, 0, 400, 3000], 1), (8, [129, 64, 5], 4), (64, [500, 33], 1)])
def test_attend_numerators_of_a_bf16_cache(page, heads, lens, n):
    """32 rows a tile over a bf16 cache take each numerator as two bf16 parts, which leave 2^-16 of it out
    (one leaves up to 2^-8). In fp32 the output has no rounding beside the sums'. A score is a sum of
    576 products in fp32, each addition off by 2^-24 of what is there, less than sum |q k|: in the mean
    square sqrt(576) 2^-24 of that times the scale, and an output twice as much. Twice their sum is asked for."""
    print(f"\nnumerators page={page} heads={heads} lens={lens} n={n}", flush=True)
    run = _runner(heads)
    cache, q_lat, q_pe, table, dl = _attend_case("bf16", heads, page, lens, n, seed=101)
    out = torch.empty(q_lat.shape, device="cuda")
    run.attend(cache, q_lat, q_pe, table, dl, out=out)
    run.raise_on_device_error()
    want, *_ = ref.attend(cache, q_lat, q_pe, table, lens, SCALE)
    most = 0.0
    for b, length in enumerate(lens):
        kv = ref.row_values(ref.sequence_rows(cache, table, b, length)).abs()
        q = torch.cat([q_lat, q_pe], 2)[b * n : b * n + n].double().abs()
        if length:
            most = max(most, float((q @ kv.T).max()) * SCALE)
    asked = 2 * (2.0**-16 + 2 * 576**0.5 * ref.U32 * most + max(lens) ** 0.5 * ref.U32)
    assert asked < 2.0**-11
    err = float((out.double() - want).norm() / want.norm())
    print(f"error {err:.2e}, asked {asked:.2e}", flush=True)
    assert err <= asked
