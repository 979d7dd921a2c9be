"""A prompt's attention (``sgl_amd_mono.moe.latent_prompt``) in both cuts of a call: workgroups of 4 waves, and of 8,
where a sequence may be long by its table and by max_context. Every test asserts the cut that its calls took. The plain
form and its bounds are ``prompt_ref``'s."""

import ctypes

import pytest
import torch
import torch.nn.functional as F

import latent_ref as ref
import prompt_ref
from test_gpu_latent_prompt import BF, SCALE, Batch, _runner, _step

pytestmark = pytest.mark.gpu

CUTS = pytest.mark.parametrize("waves", [4, 8])
LONG = 32768 + 1024  # tokens of a sequence, by its table and max_context, that take 8 waves


def waves_of(run):
    """The cut of a runner's last call."""
    from sgl_amd_mono.moe import _lib

    return _lib.testing_lib().mkmoe_host_prompt_waves(ctypes.byref(run._prompt_io))


def _cut(b, waves, tokens=LONG, **kw):
    """A runner for a batch in a cut; its table gets entries behind the sequences' own, which name no page."""
    if waves == 8:
        wide = -(-tokens // b.cache.shape[1]) - b.table.shape[1]
        b.table = F.pad(b.table, (0, max(0, wide)), value=2**30)
        kw = {"max_context": tokens * len(b.lens), **kw}
    return _runner(b.heads, **kw)


@CUTS
@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("new,lens,heads,page", [
    ([1], [1], 1, 1), ([1], [64], 3, 16), ([2, 1, 3], [2, 900, 70], 4, 8), ([31], [31], 5, 2), ([33], [97], 16, 32),
    ([127], [127], 2, 64), ([129], [320], 2, 64), ([255], [300], 2, 128), ([256], [256], 2, 64), ([257], [1000], 2, 64),
    ([300, 1, 17, 0, 513], [301, 1500, 17, 0, 700], 3, 16), ([1000, 40], [1100, 2000], 12, 1), ([2500], [2700], 2, 64),
])  # fmt: skip
def test_attend(new, lens, heads, page, fmt, waves):
    if waves == 4 and new == [2500]:
        new, lens = [2048], [2248]  # (more take 8)
    print(f"\ncut {waves} {fmt} {new} {lens} {heads} page={page}", flush=True)
    b = Batch(sum(lens) + page, heads, fmt, page, new, lens)
    run = _cut(b, waves)
    lse = torch.empty(sum(new), heads, device="cuda")
    out = run.attend(*b.args(), q_starts=b.dev_starts, lse=lse)
    assert waves_of(run) == waves
    b.check(out, lse)
    run.raise_on_device_error()
    assert torch.equal(out, run.attend(*b.args(), q_starts=b.dev_starts))


def test_more_than_2048_tokens_take_8_waves():
    b = Batch(41, 3, "mxfp8", 64, [2600], [3000])
    run = _runner(3)
    out = run.attend(*b.args())
    assert waves_of(run) == 8
    b.check(out)


@CUTS
def test_parts_of_many_shares(waves):
    """Few heads over long keys: a query tile's parts are many shares'; all of them are joined."""
    b = Batch(42, 1, "bf16", 64, [5, 260], [300, 20000])
    run = _cut(b, waves, max_context=40000 if waves == 4 else 2 * LONG)
    lse = torch.empty(265, 1, device="cuda")
    out = run.attend(*b.args(), q_starts=b.dev_starts, lse=lse)
    assert waves_of(run) == waves
    b.check(out, lse)


@CUTS
def test_rows_that_see_nothing(waves):
    new, lens = [40, 300, 17, 0, 5], [8, 20, 0, 90, 5]
    b = Batch(7, 3, "bf16", 8, new, lens)
    run = _cut(b, waves)
    lse = torch.empty(sum(new), 3, device="cuda")
    out = torch.full((sum(new), 3, 128), 7.0, dtype=BF, device="cuda")
    run.attend(*b.args(), q_starts=b.dev_starts, out=out, lse=lse)
    assert waves_of(run) == waves
    b.check(out, lse)
    run.raise_on_device_error()
    assert not out[:32].any() and not out[340:357].any()


@CUTS
@pytest.mark.parametrize("scale", [-0.2, -0.0, 0.0, 1.5, 1e-30])
def test_scales(scale, waves):
    b = Batch(8, 4, "mxfp8", 16, [270, 33], [400, 33])
    run = _cut(b, waves, scale=scale)
    lse = torch.empty(303, 4, device="cuda")
    out = run.attend(*b.args(), q_starts=b.dev_starts, lse=lse)
    assert waves_of(run) == waves
    b.check(out, lse, scale)


@CUTS
def test_strides_and_rows_of_no_sequence(waves):
    b = Batch(9, 6, "bf16", 32, [100, 300], [100, 500])
    run = _cut(b, waves)
    q_pe = torch.zeros(6, 420, 64, dtype=BF, device="cuda").transpose(0, 1)  # heads outermost
    q_nope = torch.zeros(420, 6, 200, dtype=BF, device="cuda")[..., 8:136]
    q_nope[11:411], q_pe[11:411] = b.q_nope, b.q_pe
    wide = torch.full((6, 420, 160), 7.0, dtype=BF, device="cuda")
    out = wide[:, :, 16:144].transpose(0, 1)
    lse = torch.full((420, 6), 7.0, device="cuda")
    run.attend(b.w, b.cache, q_nope, q_pe, b.table, b.dev_lens, q_starts=b.dev_starts + 11, out=out, lse=lse)
    assert waves_of(run) == waves
    b.check(out[11:411], lse[11:411])
    run.raise_on_device_error()
    for rest in (out[:11], out[411:], wide[:, :, :16], wide[:, :, 144:], lse[:11], lse[411:]):
        assert (rest == 7).all()


@CUTS
@pytest.mark.parametrize("starts", [[0, 40, 10, 70, 60, 90], [30, 0, 90, 0, 90, 0], [0, 90] * 2 + [0, 90]])
def test_starts_that_run_backwards(starts, waves):
    b = Batch(16, 4, "bf16", 16, [18] * 5, [200, 70, 65, 130, 90])
    run = _cut(b, waves)
    out = torch.full((90, 4, 128), 7.0, dtype=BF, device="cuda")
    run.attend(*b.args(), q_starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), out=out)
    assert waves_of(run) == waves and run.read_errors()[0] == 3
    b.starts = torch.cummax(torch.tensor(starts), 0).values.tolist()
    first = b.starts[0]
    o, _, bound, _ = b.want()
    assert (out[:first] == 7).all()
    prompt_ref.close(out[first:], o[first:], bound[first:])


@CUTS
def test_pages_and_lengths_outside_their_bounds(waves):
    b = Batch(15, 4, "bf16", 16, [30, 300, 30], [60, 500, 50])
    run = _cut(b, waves)
    lens = b.dev_lens.clone()
    lens[0] = -5
    got = run.attend(*b.args()[:5], lens, q_starts=b.dev_starts)
    assert waves_of(run) == waves and run.read_errors()[:2] == [3, 0]
    b.lens[0] = 0
    b.check(got)  # (the others' bits may differ: the shares' ends lie elsewhere)
    b.lens[0] = 60
    run.clear_errors()
    zero, good = b.cache.clone(), b.table.clone()
    for seq, at, bad in ((0, 1, b.pages), (1, 30, -1), (2, 0, 2**31 - 1)):  # read as rows of zeros
        zero[b.table[seq, at].item()] = 0
        b.table[seq, at] = bad
    got = run.attend(*b.args(), q_starts=b.dev_starts)
    b.cache, b.table = zero, good
    b.check(got)
    assert run.read_errors()[0] == 4


@CUTS
def test_context_that_the_workspace_does_not_hold(waves):
    new, lens = [20, 300, 40, 10], [200, 500, 100, 0]
    b = Batch(16, 3, "bf16", 16, new, lens)
    if waves == 4:
        run = _runner(3, max_context=600)  # 256 and 512 rows: the second one does not fit, nor the third behind it
    else:  # the first one takes most of it
        new, lens = [20, 300, 40, 10], [LONG * 4 - 100, 500, 100, 0]
        b = Batch(16, 3, "bf16", 64, new, lens)
        run = _cut(b, 8)
    lse = torch.empty(370, 3, device="cuda")
    out = run.attend(*b.args(), q_starts=b.dev_starts, lse=lse)
    assert waves_of(run) == waves
    o, _, bound, _ = b.want()
    ref.assert_within(out[:20], o[:20], bound[:20], "out")
    assert torch.isnan(out[20:360].float()).all() and torch.isnan(lse[20:360]).all() and not out[360:].any()
    code, where, count, _ = run.read_errors()
    assert code == 5 and where in (1, 2) and count == 2


@CUTS
def test_captured_with_other_lengths(waves):
    b = Batch(20, 4, "bf16", 16, [300, 60, 40], [300, 60, 200], width=40)
    run = _cut(b, waves)
    out = torch.zeros(400, 4, 128, dtype=BF, device="cuda")
    lens, starts = b.dev_lens.clone(), b.dev_starts.clone()
    call = lambda: run.attend(b.w, b.cache, b.q_nope, b.q_pe, b.table, lens, q_starts=starts, out=out)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    assert waves_of(run) == waves
    for new, ln in (([300, 60, 40], [300, 60, 200]), ([10, 360, 30], [640, 370, 30]), ([0, 399, 1], [0, 500, 600])):
        b.new, b.lens, b.starts = new, ln, [0, new[0], new[0] + new[1], 400]
        lens.copy_(torch.tensor(ln, dtype=torch.int32))
        starts.copy_(torch.tensor(b.starts, dtype=torch.int32))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        b.check(out)
        replayed = out.clone()
        assert torch.equal(call(), replayed)


@CUTS
@pytest.mark.parametrize("seed", range(6))
def test_random_shapes(seed, waves):
    g = torch.Generator().manual_seed(200 + seed)
    pick = lambda *v: v[int(torch.randint(len(v), (1,), generator=g))]  # noqa: E731
    seqs, heads, most = pick(1, 2, 3, 7), pick(1, 2, 5, 8, 17), pick(40, 300, 600)
    new = [int(torch.randint(0, most + 1, (1,), generator=g)) for _ in range(seqs)]
    new[0] = max(1, new[0])
    lens = [max(0, n + int(torch.randint(-20, 900, (1,), generator=g))) for n in new]
    fmt, page = pick("bf16", "mxfp8"), pick(1, 2, 16, 64, 128, 1024)
    print(f"\nrandom {seed} cut {waves}: {new} {lens} heads={heads} {fmt} page={page}", flush=True)
    b = Batch(seed, heads, fmt, page, new, lens)
    run = _cut(b, waves, **({"max_context": 16384} if waves == 4 else {}))
    lse = torch.empty(sum(new), heads, device="cuda")
    out = run.attend(*b.args(), q_starts=b.dev_starts, lse=lse)
    # (a page of many tokens is a long table by itself; then max_context bounds the length)
    assert waves_of(run) == waves
    b.check(out, lse)


@CUTS
def test_attention(waves):
    """A layer's whole step: its parts one by one give the same bits."""
    b = Batch(23, 5, "mxfp8", 16, [200, 7, 0, 130], [200, 300, 0, 131])
    _step(b)
    run = _cut(b, waves, max_tokens=337)
    out = run.attention(b.w, b.cache, b.q, b.kv, b.cos_sin, b.positions, b.slots, b.table, b.dev_lens, q_starts=b.dev_starts)
    assert waves_of(run) == waves
    run.raise_on_device_error()
    q_pe = run.append(b.cache, b.kv, b.w.norm, b.cos_sin, b.positions, b.slots, q_pe=b.q[..., 128:])
    b.q_nope, b.q_pe = b.q[..., :128], q_pe
    assert torch.equal(out, run.attend(*b.args(), q_starts=b.dev_starts))
    b.check(out)


@CUTS
def test_more_items_than_a_share_lists(waves):
    """512 short sequences of 128 heads: 65536 query tiles, 128 or 256 a share, which lists 64 at a time. The cut by 8
    waves is taken where the other's work passes 32 bits: by a max_context of 800000 tokens."""
    g = torch.Generator().manual_seed(5)
    new = [1 + int(x) for x in torch.randint(0, 3, (512,), generator=g)]
    lens = [n + int(x) for n, x in zip(new, torch.randint(0, 60, (512,), generator=g))]
    b = Batch(43, 128, "bf16", 64, new, lens)
    run = _cut(b, waves, tokens=800000, max_context=65536 if waves == 4 else 800000)
    lse = torch.empty(sum(new), 128, device="cuda")
    out = run.attend(*b.args(), q_starts=b.dev_starts, lse=lse)
    assert waves_of(run) == waves
    run.raise_on_device_error()
    for h in (0, 1, 63, 100, 127):
        z = slice(h, h + 1)
        o, l, bound, lbound = prompt_ref.attend(b.cache, b.w.kv_b.view(128, 256, 512)[z], b.q_nope[:, z], b.q_pe[:, z],
                                                b.table, b.lens, b.starts, SCALE)  # fmt: skip
        ref.assert_within(out[:, z], o, bound, f"head {h}")
        ref.assert_within(lse[:, z].double(), l, lbound, f"lse of head {h}")


@CUTS
@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("new,lens,heads", [([777], [777], 16), ([300, 500], [1300, 500], 8), ([200], [6000], 4)])
def test_accuracy(new, lens, heads, fmt, waves):
    """The error in the 2-norm. A rounding to bf16 of values whose logarithms are spread evenly is off by a root mean
    square of r = 2^-8 sqrt((1 - 1/4) / (3 2 ln 2)) = 2^-8 0.4246 of them: an error even over a step, 2^-8 / sqrt 3 of
    the power of two below a value, and the mean of that power's square over the value's own, (1 - 1/4) / (2 ln 2).
    The output is rounded so; each of the 128 key values that the latents make, which moves a score of unit queries and
    keys by r scale sqrt 128, and an output by at most so much of it; a value and a numerator to fp16, by r / 8 each. With 8 % for how
    the values of a case lie: a numerator or value rounded to bf16 instead adds r of it, more than that."""
    b = Batch(50 + sum(new), heads, fmt, 64, new, lens)
    run = _cut(b, waves, **({"max_context": 8192} if waves == 4 else {}))
    out = run.attend(*b.args(), q_starts=b.dev_starts)
    assert waves_of(run) == waves
    want = b.want()[0]
    rel = ((out.double() - want).norm() / want.norm()).item()
    r = ref.U16 * (0.75 / (6 * 0.6931472)) ** 0.5
    print(f"\nerror {rel:.6f}", flush=True)
    assert rel <= 1.08 * r * (1 + 128 * SCALE**2 + 2 / 64) ** 0.5
