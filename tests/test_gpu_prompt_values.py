"""A prompt's attention over values of every size (``sgl_amd_mono.moe.latent_prompt``) against a plain 64-bit form
(``prompt_ref``): what a value loses is its own, whatever stands beside it. Each test runs both cuts of a call: of 4
waves a workgroup, and of 8, where a sequence may be long by its table and by max_context."""

import pytest
import torch

import latent_ref as ref
import prompt_ref
from test_gpu_latent_prompt import BF, Batch, _runner

pytestmark = pytest.mark.gpu

CUTS = pytest.mark.parametrize("waves", [4, 8])


def _batch(seed, heads, fmt, new, lens, waves):
    """A batch and a runner of the cut."""
    long = 32768 + 64
    b = Batch(seed, heads, fmt, 16, new, lens, width=long // 16 if waves == 8 else None)
    return b, lambda **kw: _runner(heads, max_context=long * len(new) if waves == 8 else 4096, **kw)


def _tokens(b, seq, first, end):
    """Pages and places in them of a sequence's tokens first .. end - 1."""
    at = torch.arange(first, end, device="cuda")
    return b.table[seq].long()[at // 16], at % 16


@CUTS
@pytest.mark.parametrize("fmt,log2", [("bf16", -20), ("bf16", -23), ("bf16", -27), ("bf16", -60), ("mxfp8", -19), ("mxfp8", -26)])
@pytest.mark.parametrize("large", [[199], [70], [0, 130]])  # unseen by most of the queries; seen by all
def test_small_tokens_beside_a_large_one(fmt, log2, large, waves):
    b, runner = _batch(31, 3, fmt, [60], [200], waves)
    small = torch.ones(200, dtype=torch.bool, device="cuda")
    small[large] = False
    pages, places = (x[small] for x in _tokens(b, 0, 0, 200))
    if fmt == "bf16":
        b.cache[pages, places, :512] = (b.cache[pages, places, :512].float() * 2.0**log2).to(b.cache.dtype)
    else:
        b.cache[pages, places, 512:528] += log2 % 256  # (of 8 bits)
    lse = torch.empty(60, 3, device="cuda")
    out = runner().attend(*b.args(), lse=lse)
    o, l, bound, lbound = b.want()
    ref.assert_within(out, o, bound, "out")
    # (the sum takes the numerators as they are multiplied, each rounded by up to 2^-8 of it: log(1 + 2^-8) < 2^-8)
    ref.assert_within(lse.double(), l, lbound + ref.U16, "lse")
    if large == [199]:
        prompt_ref.close(out[:59], o[:59], bound[:59], "queries that do not see it")


@CUTS
@pytest.mark.parametrize("log2", [-100, -30, -24, -16, 8, 95])
def test_small_outputs_beside_ordinary_ones(log2, waves):
    """Some of W_UV's rows in another size than the rest: softmax never mixes a head's outputs."""
    b, runner = _batch(32, 2, "bf16", [150, 7], [333, 90], waves)
    rows = [0, 17, 40, 127]
    b.w.kv_b.view(2, 2, 128, 512)[0, 1, rows] *= 2.0**log2
    out = runner().attend(*b.args(), q_starts=b.dev_starts)
    o, _, bound, _ = b.want()
    ref.assert_within(out, o, bound, "out")
    for d in rows:
        prompt_ref.close(out[:, 0, d], o[:, 0, d], bound[:, 0, d], f"output {d}")


@CUTS
def test_values_of_all_sizes(waves):
    """Every token and output has a value of a size of its own, some of them 0: W_UV picks single latents."""
    b, runner = _batch(33, 2, "bf16", [70, 130], [70, 400], waves)
    g = b.g
    size = torch.exp2(torch.rand(b.cache.shape[0], 16, 128, generator=g, device="cuda") * 46 - 40)
    size *= torch.rand(size.shape, generator=g, device="cuda") > 0.1
    b.cache[..., :128] = (b.cache[..., :128].float() * size).to(b.cache.dtype)
    w = b.w.kv_b.view(2, 2, 128, 512)
    w[:, 1] = 0
    w[:, 1, torch.arange(128), torch.arange(128)] = 1.0
    out = runner().attend(*b.args(), q_starts=b.dev_starts)
    o, _, bound, _ = b.want()
    ref.assert_within(out, o, bound, "out")


@CUTS
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("log2,border", [(9, 300), (10, 300), (10, 330), (16, 300), (23, 300), (27, 300), (40, 300), (100, 300)])
def test_scores_far_from_0(log2, border, sign, waves):
    """Scores of 2^log2 and half of it that differ by a few units of their last places, all of them and their sums exact
    in fp32: the weights are those of the differences. A numerator is rounded by up to 2^-11 (and 2^-20 for its
    exponential), in the output's sum and in the weights', a value and the output by 2^-8 each."""
    heads, n, length = 2, 150, 400
    b, runner = _batch(34, heads, "bf16", [n], [length], waves)
    pages, places = _tokens(b, 0, 0, length)
    low = (torch.arange(length, device="cuda") < border) == (sign > 0)  # what weighs more comes later
    size = torch.where(low, 0.5, 1.0).double() * 2.0 ** (log2 - log2 // 2)
    step = 2.0 ** max(-1, log2 - 23)
    units = torch.randint(0, 6, (length,), generator=b.g, device="cuda").double()
    b.cache[pages, places, 0] = size.to(b.cache.dtype)
    b.cache[pages, places, 512:] = 0
    b.cache[pages, places, 512] = units.to(b.cache.dtype)
    w = b.w.kv_b.view(heads, 2, 128, 512)
    w[:, 0] = 0
    w[:, 0, 0, 0] = 1.0  # a key is its latents' first value
    w[:, 1, :, 0] = 0  # values near 1
    b.q_nope, b.q_pe = torch.zeros_like(b.q_nope).contiguous(), torch.zeros_like(b.q_pe)
    b.q_nope[..., 0] = sign * 2.0 ** (log2 // 2)
    b.q_pe[..., 0] = step
    lse = torch.empty(n, heads, device="cuda")
    out = runner(scale=1.0).attend(*b.args(), lse=lse)
    s = sign * size * 2.0 ** (log2 // 2) + units * step
    see = torch.arange(length, device="cuda")[None] <= torch.arange(length - n, length, device="cuda")[:, None]
    s = s.masked_fill(~see, -float("inf"))
    p = torch.softmax(s, 1)
    v = torch.stack([b.cache[pages, places, :512].double() @ w[h, 1].double().T for h in range(heads)])  # [heads, length, 128]
    fine = 514 * ref.U32 * torch.stack([b.cache[pages, places, :512].double().abs() @ w[h, 1].double().abs().T for h in range(heads)])
    o, size_o, fine = ((p[None] @ x).transpose(0, 1) for x in (v, v.abs(), fine))
    ref.assert_within(out, o, (2 * ref.U16 + 2.0**-10 + 2.0**-15) * size_o + 2 * fine, "out")
    want = torch.logsumexp(s, 1)[:, None].expand(n, heads)
    ref.assert_within(lse.double(), want, 2.0**-11 + 2.0**-19 + 4 * ref.U32 * want.abs(), "lse")


@CUTS
@pytest.mark.parametrize("size", [2.0**12, 2.0**-30])
@pytest.mark.parametrize("tiles", [[0], [1, 2, 5], [3, 6, 7, 8, 14], [15], [0, 2, 4, 6, 8, 10, 12, 14], list(range(16))], ids=str)
def test_tiles_that_fp16_does_not_hold(tiles, size, waves):
    """Tiles of 64 tokens whose values are past fp16's range or below it, among others, in all orders."""
    b, runner = _batch(35, 2, "bf16", [290, 40], [1000, 30], waves)
    for t in tiles:
        pages, places = _tokens(b, 0, 64 * t, min(1000, 64 * t + 64))
        b.cache[pages, places, :512] = (b.cache[pages, places, :512].float() * size).to(b.cache.dtype)
    # scores stay near 1: keys are made from the rope values alone, values from the latents
    b.w.kv_b.view(2, 2, 128, 512)[:, 0] = 0
    out = runner().attend(*b.args(), q_starts=b.dev_starts)
    o, _, bound, _ = b.want()
    ref.assert_within(out, o, bound, "out")
    assert torch.equal(out, runner().attend(*b.args(), q_starts=b.dev_starts))


@CUTS
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("at", [800, 830, 959, 999])
def test_values_that_are_not_finite_among_marked_tiles(at, bad, waves):
    """Queries that do not see such a token are as without it, those that do are not finite."""
    b, runner = _batch(36, 2, "bf16", [290], [1000], waves)
    pages, places = _tokens(b, 0, 640, 1000)
    b.cache[pages, places, :512] *= 2.0**12  # finite, and past fp16's range
    b.w.kv_b.view(2, 2, 128, 512)[:, 0] = 0
    pages, places = _tokens(b, 0, at, at + 1)
    good = b.cache.clone()
    b.cache[pages, places, :512] = bad
    out = runner().attend(*b.args())
    b.cache = good
    o, _, bound, _ = b.want()
    first = at - 710
    ref.assert_within(out[:first], o[:first], bound[:first], "before")
    assert not torch.isfinite(out[first:].float()).any()


@CUTS
def test_weights_far_below_the_largest(waves):
    """Every key's value is an output of its own, so the outputs are the weights, from the largest down to less than
    2^-40. A numerator is held to 2^-25, the largest is 2^7 at least: off by 2^-32 beside the rounding's own bound."""
    heads, n, length = 2, 70, 128
    b, runner = _batch(37, heads, "bf16", [n], [length], waves)
    pages, places = _tokens(b, 0, 0, length)
    at = torch.arange(length, device="cuda")
    b.cache[pages, places] = 0
    b.cache[pages, places, at] = 1.0
    b.cache[pages, places, 512 + at % 32] = torch.where(at < 64, 1.0, 0.5).to(b.cache.dtype)
    w = b.w.kv_b.view(heads, 2, 128, 512)
    w[:] = 0
    w[:, 1, at, at] = 1.0
    w[:, 0, 0, :128] = (-0.25 * (at // 32)).to(w.dtype)
    b.q_nope, b.q_pe = torch.zeros_like(b.q_nope).contiguous(), torch.zeros_like(b.q_pe)
    b.q_nope[..., 0] = 32.0
    b.q_pe[..., :32] = (-0.25 * torch.arange(32, device="cuda")).to(BF)
    lse = torch.empty(n, heads, device="cuda")
    out = runner(scale=1.0).attend(*b.args(), lse=lse)
    o, l, bound, lbound = b.want(1.0)
    assert o.max() > 0.1 and o[o > 0].min() < 2.0**-40
    ref.assert_within(out, o, bound + 2.0**-32, "out")
    ref.assert_within(lse.double(), l, lbound + 2.0**-11 + length * 2.0**-32, "lse")
