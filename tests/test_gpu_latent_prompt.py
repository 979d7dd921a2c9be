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
        prompt_ref.close(out, o, bound, self.lens)
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
