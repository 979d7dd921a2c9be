"""A prompt's attention (``sgl_amd_mono.moe.latent_prompt``) against a plain 64-bit form (``prompt_ref``), each
value within the bound that the kernels' roundings allow."""

import pytest
import torch

import latent_ref as ref
import prompt_ref

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
SCALE = 192**-0.5
NAN, INF = float("nan"), float("inf")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(BF)


def _runner(heads, **kw):
    from sgl_amd_mono.moe.latent_prompt import LatentPromptRunner

    return LatentPromptRunner(heads, **{"scale": SCALE, "max_tokens": 0, "max_context": 4096, **kw})


def _weights(g, heads):
    from sgl_amd_mono.moe.latent import LatentWeights

    return LatentWeights(norm=(1 + 0.1 * torch.randn(512, generator=g, device="cuda")).to(BF),
                         kv_b=_randn(g, heads * 256, 512, std=512**-0.5))  # fmt: skip


class Batch:
    """New tokens and cached lengths of sequences, their table over a cache of random rows, queries."""

    def __init__(self, seed, heads, fmt, page, new, lens, width=None):
        g = self.g = _gen(seed)
        self.heads, self.new, self.lens = heads, list(new), list(lens)
        self.starts = [sum(new[:i]) for i in range(len(new) + 1)]
        t = self.starts[-1]
        per = max(1, -(-max(self.lens) // page)) if width is None else width
        self.pages = len(new) * per + 3
        perm = torch.randperm(self.pages, generator=g, device="cuda").int()
        self.table = perm[: len(new) * per].view(len(new), per).contiguous()
        self.cache = ref.random_cache(self.pages, page, fmt, g, "cuda")
        self.w = _weights(g, heads)
        self.q_nope, self.q_pe = _randn(g, t, heads, 192)[..., :128], _randn(g, t, heads, 64)
        self.dev_lens = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        self.dev_starts = torch.tensor(self.starts, dtype=torch.int32, device="cuda")

    def args(self):
        return self.w, self.cache, self.q_nope, self.q_pe, self.table, self.dev_lens

    def want(self, scale=SCALE):
        return prompt_ref.attend(self.cache, self.w.kv_b, self.q_nope, self.q_pe, self.table, self.lens, self.starts, scale)

    def check(self, out, lse=None, scale=SCALE):
        torch.cuda.synchronize()
        o, l, bound, lbound = self.want(scale)
        prompt_ref.close(out, o, bound, sigma=abs(scale) * 192**0.5)
        if lse is not None:
            none = torch.isinf(l)
            assert torch.equal(lse[none].double(), l[none])
            assert not (out[none] != 0).any()
            ref.assert_within(lse[~none].double(), l[~none], lbound[~none], "lse")


CASES = [
    # new, lens, heads, page
    ([1], [1], 1, 1),
    ([1], [64], 3, 16),
    ([1], [65], 2, 64),
    ([2, 1, 3], [2, 900, 70], 4, 8),
    ([31], [31], 5, 2),
    ([33], [97], 16, 32),
    ([64, 64], [64, 128], 8, 64),
    ([255], [300], 2, 128),
    ([256], [256], 2, 64),
    ([257], [1000], 2, 64),
    ([300, 1, 17, 0, 513], [301, 1500, 17, 0, 700], 3, 16),
    ([777], [777], 16, 64),
    ([1000, 40], [1100, 2000], 12, 1),
]


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}h-p{c[3]}".replace(" ", ""))
def test_attend(case, fmt):
    new, lens, heads, page = case
    print(f"\nprompt attend {fmt} {case}", flush=True)
    b = Batch(len(new) * 1000 + sum(lens), heads, fmt, page, new, lens)
    run = _runner(heads)
    lse = torch.empty(sum(new), heads, device="cuda")
    out = run.attend(*b.args(), q_starts=b.dev_starts, lse=lse)
    torch.cuda.synchronize()
    run.raise_on_device_error()
    b.check(out, lse)


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("new,lens,heads", [([1], [1], 3), ([33, 0, 2], [97, 50, 1500], 16), ([255, 256, 257], [300, 256, 2000], 2),
                                            ([300, 70], [1300, 700], 2), ([513], [1600], 4), ([777], [777], 16)])  # fmt: skip
def test_tables_of_long_sequences(new, lens, heads, fmt):
    """Where a sequence may be long by its table and by max_context, a call is cut otherwise."""
    print(f"\nlong tables {fmt} {new} {lens} {heads}", flush=True)
    b = Batch(sum(new) + 1, heads, fmt, 64, new, lens, width=520)
    lse = torch.empty(sum(new), heads, device="cuda")
    out = _runner(heads, max_context=33280 * len(new)).attend(*b.args(), q_starts=b.dev_starts, lse=lse)
    b.check(out, lse)


@pytest.mark.parametrize("context", [2048, 65536])  # the call's cut: few query tiles, or cached tokens that may be many
@pytest.mark.parametrize("new,lens,heads", [([130], [130], 3), ([300, 70], [1300, 700], 2), ([513], [1600], 4)])
def test_both_cuts(new, lens, heads, context):
    print(f"\ncuts {new} {lens} {heads} context={context}", flush=True)
    b = Batch(sum(new), heads, "bf16", 16, new, lens)
    lse = torch.empty(sum(new), heads, device="cuda")
    run = _runner(heads, max_context=context)
    b.check(run.attend(*b.args(), q_starts=b.dev_starts, lse=lse), lse)


def test_many_query_tiles():
    """More than one item a share: 128 heads, ragged, joined tiles among them."""
    b = Batch(5, 128, "mxfp8", 64, [700, 3, 260], [700, 900, 261])
    run = _runner(128)
    lse = torch.empty(963, 128, device="cuda")
    b.check(run.attend(*b.args(), q_starts=b.dev_starts, lse=lse), lse)


def test_one_sequence_without_starts():
    b = Batch(6, 8, "bf16", 64, [64, 64, 64], [70, 64, 500])
    out = _runner(8).attend(*b.args())
    b.check(out)


def test_rows_that_see_nothing():
    """More queries than cached tokens, no cached tokens, and sequences without queries."""
    new, lens = [40, 300, 17, 0, 5], [8, 20, 0, 90, 5]
    b = Batch(7, 3, "bf16", 8, new, lens)
    run = _runner(3)
    lse = torch.empty(sum(new), 3, device="cuda")
    out = torch.full((sum(new), 3, 128), 7.0, dtype=BF, device="cuda")
    run.attend(*b.args(), q_starts=b.dev_starts, out=out, lse=lse)
    run.raise_on_device_error()
    b.check(out, lse)
    assert not out[:32].any() and not out[340:357].any()


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.5])
def test_scales(scale):
    b = Batch(8, 4, "mxfp8", 16, [70, 33], [200, 33])
    run = _runner(4, scale=scale)
    lse = torch.empty(103, 4, device="cuda")
    b.check(run.attend(*b.args(), q_starts=b.dev_starts, lse=lse), lse, scale)


def test_strides_and_broadcast():
    b = Batch(9, 6, "bf16", 32, [100, 30], [100, 200])
    run = _runner(6)
    g = b.g
    b.q_pe = _randn(g, 6, 130, 64).transpose(0, 1)  # heads outermost
    b.q_nope = _randn(g, 130, 1, 128).expand(130, 6, 128)  # one row for all heads
    wide = torch.full((6, 130, 160), 7.0, dtype=BF, device="cuda")
    out = wide[:, :, 16:144].transpose(0, 1)
    table = torch.full((2, 20), 99, dtype=torch.int32, device="cuda")  # rows of a wider table
    table[:, : b.table.shape[1]] = b.table
    b.table = table[:, : b.table.shape[1]]
    assert run.attend(*b.args(), q_starts=b.dev_starts, out=out) is out
    b.check(out)
    assert (wide[:, :, :16] == 7).all() and (wide[:, :, 144:] == 7).all()


def test_rows_of_no_sequence_stay():
    b = Batch(10, 4, "bf16", 16, [40, 70], [60, 70])
    run = _runner(4)
    t = 130
    q_nope, q_pe = _randn(b.g, t, 4, 128), _randn(b.g, t, 4, 64)
    q_nope[7:117], q_pe[7:117] = b.q_nope, b.q_pe
    starts = (b.dev_starts + 7).int()
    out = torch.full((t, 4, 128), 7.0, dtype=BF, device="cuda")
    lse = torch.full((t, 4), 7.0, device="cuda")
    run.attend(b.w, b.cache, q_nope, q_pe, b.table, b.dev_lens, q_starts=starts, out=out, lse=lse)
    run.raise_on_device_error()
    assert (out[:7] == 7).all() and (out[117:] == 7).all() and (lse[:7] == 7).all() and (lse[117:] == 7).all()
    b.check(out[7:117], lse[7:117])
    own = run.attend(b.w, b.cache, q_nope, q_pe, b.table, b.dev_lens, q_starts=starts)
    assert not own[:7].any() and not own[117:].any() and torch.equal(own[7:117], out[7:117])


@pytest.mark.parametrize("fmt,bad", [("bf16", NAN), ("bf16", INF), ("bf16", -INF), ("bf16", 3e38), ("mxfp8", NAN)])
@pytest.mark.parametrize("at", [0, 63, 100, 199])
def test_values_that_are_not_finite_reach_only_what_sees_them(fmt, bad, at):
    """A token's latents at their worst, among the new tokens: the queries before it are as without it."""
    heads, n, length = 3, 180, 200
    b = Batch(11, heads, fmt, 16, [n], [length])
    where = b.table[0, at // 16].item(), at % 16
    good = b.cache.clone()
    if fmt == "bf16":
        b.cache[where][:512] = bad
    else:
        b.cache[where][:512] = 0x7F
    run = _runner(heads)
    out = run.attend(*b.args())
    torch.cuda.synchronize()
    b.cache = good
    o, _, bound, _ = b.want()
    first = max(0, at - (length - n))  # the first query that sees it
    ref.assert_within(out[:first], o[:first], bound[:first], "before")
    if bad != 3e38:
        assert not torch.isfinite(out[first:].float()).any()


def test_garbage_behind_the_end_reaches_nothing():
    b = Batch(12, 4, "bf16", 64, [33, 20], [97, 30])
    used = torch.zeros(b.pages * 64, dtype=torch.bool, device="cuda")
    for i, n in enumerate(b.lens):
        at = torch.arange(n, device="cuda")
        used[b.table[i].long()[at // 64] * 64 + at % 64] = True
    b.cache.view(-1, 576)[~used] = NAN
    run = _runner(4)
    first = run.attend(*b.args(), q_starts=b.dev_starts)
    b.check(first)
    run.ws[1 << 20 :].fill_(0xFF)  # what a workspace held before, too (the error words left out)
    assert torch.equal(run.attend(*b.args(), q_starts=b.dev_starts), first)


@pytest.mark.parametrize("size", [1e6, 1e-5, 2.0**-9])
def test_values_outside_what_fp16_holds(size):
    """Values past fp16's range, or so small that it would round them coarsely, of some tiles or of all."""
    b = Batch(13, 4, "bf16", 16, [150, 200], [400, 200])
    b.w.kv_b.view(4, 2, 128, 512)[1:3, 1] *= size  # two heads
    slots = b.table[0].long()[70 // 16 : 130 // 16]
    b.cache[slots, :, :512] *= 64.0  # and a few tokens of all heads
    run = _runner(4)
    torch.cuda.synchronize()
    o, _, bound, _ = b.want()
    out = run.attend(*b.args(), q_starts=b.dev_starts)
    ref.assert_within(out, o, bound, "out")
    for h in range(4):
        prompt_ref.close(out[150:, h], o[150:, h], bound[150:, h], f"head {h}")


@pytest.mark.parametrize("far,length", [(17.0, 6000), (15.25, 60000)])
def test_long_tails_of_small_numerators(far, length):
    """One key that weighs e^far times any other: the others' numerators still count, and in their sum (60000 of
    2^-22 are 1.4 % of it, more than the bound)."""
    heads = 2
    b = Batch(14, heads, "bf16", 64, [130], [length])
    b.cache[..., :] = 0
    b.cache[..., 0] = 1.0  # every token's latents: e_0; the first one's: 32 e_1
    b.cache[b.table[0, 0].item(), 0] = 0
    b.cache[b.table[0, 0].item(), 0, 1] = 32.0
    w = b.w.kv_b.view(heads, 2, 128, 512)
    w[:] = 0
    w[:, 0, 0, 1] = 1.0  # k: dimension 0 is 32 for the first token, 0 for the others
    w[:, 1, :, 0] = 1.0  # v: 1 for the others, 0 for the first one
    b.q_nope, b.q_pe = torch.zeros(130, heads, 128, dtype=BF, device="cuda"), torch.zeros(130, heads, 64, dtype=BF, device="cuda")
    b.q_nope[..., 0] = 1.0
    out = _runner(heads, scale=far / 32, max_context=length + 100).attend(*b.args())
    see = torch.arange(length - 130, length, device="cuda").double()
    want = (see / (see + torch.e**far))[:, None, None].expand(130, heads, 128)
    assert ((out.double() - want).abs() <= want * (2 * ref.U16 + length * ref.U32)).all()


def test_lengths_starts_and_pages_outside_their_bounds():
    b = Batch(15, 4, "bf16", 16, [30, 30, 30], [60, 40, 50])
    run = _runner(4)
    want = run.attend(*b.args(), q_starts=b.dev_starts)
    width = b.table.shape[1] * 16
    lens = b.dev_lens.clone()
    lens[1] = width + 5
    got = run.attend(*b.args()[:5], lens, q_starts=b.dev_starts)
    assert torch.equal(got[:30], want[:30]) and torch.equal(got[60:], want[60:])
    assert run.read_errors()[:2] == [3, 1]
    run.clear_errors()
    starts = b.dev_starts.clone()
    starts[3] = 95  # past the tokens
    got = run.attend(*b.args(), q_starts=starts)
    assert torch.equal(got, want) and run.read_errors()[:2] == [3, 2]
    run.clear_errors()
    starts[2] = 10  # backwards: the second sequence attends nothing
    starts[3] = 90
    out = torch.full_like(want, 7.0)
    run.attend(*b.args(), q_starts=starts, out=out)
    torch.cuda.synchronize()
    assert torch.equal(out[:30][:10], want[:10]) and run.read_errors()[0] == 3
    run.clear_errors()
    table = b.table.clone()
    table[0, 1] = b.pages  # tokens 16 .. 31 read as rows of zeros
    table[2, 0] = -1
    zero = b.cache.clone()
    zero[b.table[0, 1].item()] = 0
    zero[b.table[2, 0].item()] = 0
    got = run.attend(b.w, b.cache, b.q_nope, b.q_pe, table, b.dev_lens, q_starts=b.dev_starts)
    b.cache = zero
    b.check(got)
    assert run.read_errors()[0] == 4
    with pytest.raises(RuntimeError, match="page outside the cache"):
        run.raise_on_device_error()


@pytest.mark.parametrize("starts", [[0, 40, 10, 70, 60, 90], [30, 0, 90, 0, 90, 0], [0, 90] * 2 + [0, 90]])
def test_starts_that_run_backwards(starts):
    """A sequence begins where those before it end: every row is one sequence's, and rows of none stay as they were."""
    b = Batch(16, 4, "bf16", 16, [18] * 5, [200, 70, 65, 130, 90])
    run = _runner(4)
    dev = torch.tensor(starts, dtype=torch.int32, device="cuda")
    out = torch.full((90, 4, 128), 7.0, dtype=BF, device="cuda")
    lse = torch.full((90, 4), 7.0, device="cuda")
    run.attend(*b.args(), q_starts=dev, out=out, lse=lse)
    torch.cuda.synchronize()
    assert run.read_errors()[0] == 3
    b.starts = torch.cummax(torch.tensor(starts), 0).values.tolist()
    first = b.starts[0]
    assert (out[:first] == 7).all() and (lse[:first] == 7).all()
    o, l, bound, lbound = b.want()
    prompt_ref.close(out[first:], o[first:], bound[first:])
    ref.assert_within(lse[first:].double(), l[first:], lbound[first:], "lse")


def test_context_that_the_workspace_does_not_hold():
    new, lens = [20, 30, 40, 10], [200, 300, 100, 0]
    b = Batch(16, 3, "bf16", 16, new, lens)
    run = _runner(3, max_context=400)  # 256 and 320 rows: the second one does not fit, nor the third behind it
    lse = torch.empty(100, 3, device="cuda")
    out = run.attend(*b.args(), q_starts=b.dev_starts, lse=lse)
    o, _, bound, _ = b.want()
    ref.assert_within(out[:20], o[:20], bound[:20], "out")
    assert torch.isnan(out[20:90].float()).all() and torch.isnan(lse[20:90]).all() and not out[90:].any()
    code, where, count, _ = run.read_errors()
    assert code == 5 and where in (1, 2) and count == 2
    run.clear_errors()
    exact = Batch(17, 3, "bf16", 16, [20, 30], [64, 64])
    run = _runner(3, max_context=128)
    exact.check(run.attend(*exact.args(), q_starts=exact.dev_starts))
    run.raise_on_device_error()


def test_512_sequences():
    g = torch.Generator().manual_seed(3)
    new = [int(x) for x in torch.randint(0, 4, (512,), generator=g)]
    lens = [n + int(x) for n, x in zip(new, torch.randint(0, 100, (512,), generator=g))]
    b = Batch(18, 2, "bf16", 16, new, lens)
    run = _runner(2, max_context=512 * 128)
    lse = torch.empty(sum(new), 2, device="cuda")
    out = run.attend(*b.args(), q_starts=b.dev_starts, lse=lse)
    run.raise_on_device_error()
    b.check(out, lse)


def test_offsets_past_32_bits():
    """A cache of 5 GB whose last pages hold the sequences, and keys and values of 4.8 GB, the last head checked."""
    heads, page, length = 128, 64, 36000
    pages = 70000
    g = _gen(19)
    cache = torch.zeros(pages, page, 576, dtype=BF, device="cuda")
    per = -(-length // page)
    cache[-2 * per :] = ref.random_cache(2 * per, page, "bf16", g, "cuda")
    table = (pages - 2 * per + torch.randperm(2 * per, generator=g, device="cuda")).int().view(2, per)
    w = _weights(g, heads)
    q_nope, q_pe = _randn(g, 12, heads, 128), _randn(g, 12, heads, 64)
    lens = torch.tensor([length, length - 77], dtype=torch.int32, device="cuda")
    run = _runner(heads, max_context=2 * length + 128)
    out = run.attend(w, cache, q_nope, q_pe, table, lens)
    run.raise_on_device_error()
    for h in (0, heads - 1):
        z = slice(h, h + 1)
        o, _, bound, _ = prompt_ref.attend(cache, w.kv_b.view(heads, 256, 512)[z], q_nope[:, z], q_pe[:, z], table,
                                           lens.tolist(), [0, 6, 12], SCALE)  # fmt: skip
        ref.assert_within(out[:, z], o, bound, f"head {h}")


@pytest.mark.parametrize("seed", range(10))
def test_random_shapes(seed):
    g = torch.Generator().manual_seed(100 + seed)
    pick = lambda *v: v[int(torch.randint(len(v), (1,), generator=g))]  # noqa: E731
    seqs, heads = pick(1, 1, 2, 3, 7), pick(1, 2, 5, 8, 17)
    most = pick(3, 40, 130, 600)
    new = [int(torch.randint(0, most + 1, (1,), generator=g)) for _ in range(seqs)]
    new[0] = max(1, new[0])
    lens = [max(0, n + int(torch.randint(-5, 700, (1,), generator=g))) for n in new]
    fmt, page = pick("bf16", "mxfp8"), pick(1, 2, 16, 64, 128, 1024)
    print(f"\nrandom {seed}: {new} {lens} heads={heads} {fmt} page={page}", flush=True)
    b = Batch(seed, heads, fmt, page, new, lens)
    lse = torch.empty(sum(new), heads, device="cuda")
    run = _runner(heads, max_context=pick(8192, 100000))
    b.check(run.attend(*b.args(), q_starts=b.dev_starts, lse=lse), lse)
    again = run.attend(*b.args(), q_starts=b.dev_starts)
    assert torch.equal(again, run.attend(*b.args(), q_starts=b.dev_starts))  # the same bits


def test_captured_with_other_lengths():
    b = Batch(20, 4, "bf16", 16, [100, 60, 40], [300, 60, 200], width=40)
    run = _runner(4)
    out = torch.zeros(200, 4, 128, dtype=BF, device="cuda")
    lens, starts = b.dev_lens.clone(), b.dev_starts.clone()
    run.attend(b.w, b.cache, b.q_nope, b.q_pe, b.table, lens, q_starts=starts, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run.attend(b.w, b.cache, b.q_nope, b.q_pe, b.table, lens, q_starts=starts, out=out)
    for new, ln in (([100, 60, 40], [300, 60, 200]), ([10, 160, 30], [640, 170, 30]), ([0, 199, 1], [0, 500, 600])):
        b.new, b.lens = new, ln
        b.starts = [sum(new[:i]) for i in range(4)]
        lens.copy_(torch.tensor(ln, dtype=torch.int32))
        starts.copy_(torch.tensor(b.starts, dtype=torch.int32))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        b.check(out)
        eager = run.attend(b.w, b.cache, b.q_nope, b.q_pe, b.table, lens, q_starts=starts)
        assert torch.equal(eager, out)
    with pytest.raises(RuntimeError, match="capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            run.attend(*b.args())


def test_two_runners_on_two_streams():
    a, b = Batch(21, 4, "bf16", 16, [300], [900]), Batch(22, 8, "mxfp8", 64, [200, 50], [500, 700])
    ra, rb = _runner(4), _runner(8)
    want = ra.attend(*a.args()), rb.attend(*b.args(), q_starts=b.dev_starts)
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(5):
        with torch.cuda.stream(s):
            x = ra.attend(*a.args())
        with torch.cuda.stream(t):
            y = rb.attend(*b.args(), q_starts=b.dev_starts)
        got.append((x, y))
    torch.cuda.synchronize()
    for x, y in got:
        assert torch.equal(x, want[0]) and torch.equal(y, want[1])


# ---------------------------------------------------------------- a layer's whole step
def _cos_sin(n):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    return torch.cat([a.cos(), a.sin()], 1).float().cuda()


def _step(b, rope="interleaved"):
    t = b.starts[-1]
    b.q = _randn(b.g, t, b.heads, 192)
    b.kv = _randn(b.g, t, 640)[:, 32:608]
    pos = torch.cat([torch.arange(n - k, n) for n, k in zip(b.lens, b.new)]).cuda()
    seq = torch.repeat_interleave(torch.arange(len(b.new)), torch.tensor(b.new)).cuda()
    page = b.cache.shape[1]
    b.positions, b.slots = pos, b.table[seq, pos // page].long() * page + pos % page
    b.cos_sin = _cos_sin(max(b.lens))
    b.rope = rope


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("rope", ["interleaved", "half"])
@pytest.mark.parametrize("new,lens,heads", [([1], [1], 2), ([200, 7], [200, 300], 5), ([90, 0, 130], [400, 0, 131], 8)])
def test_attention(new, lens, heads, fmt, rope):
    print(f"\nstep {new} {lens} {heads} {fmt} {rope}", flush=True)
    b = Batch(23 + sum(new), heads, fmt, 16, new, lens)
    _step(b, rope)
    run = _runner(heads, max_tokens=sum(new), rope=rope)
    out = run.attention(b.w, b.cache, b.q, b.kv, b.cos_sin, b.positions, b.slots, b.table, b.dev_lens, q_starts=b.dev_starts)
    torch.cuda.synchronize()
    run.raise_on_device_error()
    # its parts one by one: the rows and the rotated query as append leaves them, then attend over them
    parts = _runner(heads, rope=rope)
    before = b.cache.clone()
    q_pe = parts.append(b.cache, b.kv, b.w.norm, b.cos_sin, b.positions, b.slots, q_pe=b.q[..., 128:])
    assert torch.equal(b.cache, before)
    b.q_nope, b.q_pe = b.q[..., :128], q_pe
    assert torch.equal(out, parts.attend(*b.args(), q_starts=b.dev_starts))
    b.check(out)
    # and the absorbed form of the same step, whose bound is its own: both are near the definition
    from sgl_amd_mono.moe.latent import LatentRunner

    other = LatentRunner(heads, max_tokens=sum(new), scale=SCALE, rope=rope)
    want = other.attention(b.w, b.cache, b.q, b.kv, b.cos_sin, b.positions, b.slots, b.table, b.dev_lens, q_starts=b.dev_starts)
    assert ((out.double() - want.double()).norm() / want.double().norm()).item() < 4 * ref.U16


def test_attention_of_tokens_that_cannot_be_stored():
    b = Batch(24, 4, "bf16", 16, [40], [100])
    _step(b)
    run = _runner(4, max_tokens=40)
    call = lambda: run.attention(b.w, b.cache, b.q, b.kv, b.cos_sin, b.positions, b.slots, b.table, b.dev_lens)  # noqa: E731
    want = call()
    b.slots[3] = b.pages * 16  # outside the cache
    b.positions[5] = 5000  # outside cos_sin
    b.slots[9] = -1  # a padded token: its query is what its position makes it
    b.positions[9] = 10**6
    got = call()
    torch.cuda.synchronize()
    assert torch.isnan(got[[3, 5]].float()).all()
    rest = [i for i in range(40) if i not in (3, 5, 9)]
    assert torch.equal(got[rest], want[rest])  # (their rows were stored by the call before)
    assert torch.isfinite(got[9].float()).all()
    code, where, count, _ = run.read_errors()
    assert (code, where) in ((1, 3), (2, 5)) and count >= 2


def test_no_tokens():
    b = Batch(25, 4, "bf16", 16, [0, 0], [30, 5])
    run = _runner(4)
    assert run.attend(*b.args(), q_starts=b.dev_starts).shape == (0, 4, 128)
