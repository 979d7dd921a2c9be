"""A prompt's attention over values of every size (``sgl_amd_mono.moe.latent_prompt``) against a plain 64-bit form
(``prompt_ref``): what a value loses is its own, whatever stands beside it. Each test runs both cuts of a call: of 4
waves a workgroup, and of 8, where a sequence may be long by its table and by max_context."""

import pytest
import torch

import latent_ref as ref
import prompt_ref
from test_gpu_latent_prompt import Batch, _runner

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
@pytest.mark.parametrize("log2", [-16, -24, -30, 8])
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
