"""The page pool, a prompt's attention and single tokens' attention together, as a server runs them: prompts placed
and attended to, samples forked, tokens decoded, drafts taken back, the pool compacted, the next chunk attended to.
Each step against the definition over the sequences' own rows, kept apart from the pages."""

import pytest
import torch

import latent_ref as ref

pytestmark = pytest.mark.gpu

BF, F64 = torch.bfloat16, torch.float64
SCALE = 192**-0.5


class Server:
    def __init__(self, fmt, page, heads, layers=2, pages=120, seqs=6, width=40):
        from sgl_amd_mono.moe.latent import LatentRunner, LatentWeights, cache_like
        from sgl_amd_mono.moe.latent_prompt import LatentPromptRunner
        from sgl_amd_mono.moe.pages import PagePool

        g = self.g = torch.Generator(device="cuda").manual_seed(page)
        rand = lambda *s, std=1.0: (torch.randn(*s, generator=g, device="cuda") * std).to(BF)  # noqa: E731
        self.rand, self.heads = rand, heads
        self.caches = [cache_like(pages, page, fmt) for _ in range(layers)]
        self.pool = PagePool(pages, page, caches=self.caches, max_seqs=seqs, max_pages=width)
        self.w = [LatentWeights(norm=rand(512), kv_b=rand(heads * 256, 512, std=512**-0.5)) for _ in range(layers)]
        self.one = LatentRunner(heads, max_tokens=64, scale=SCALE)
        self.prompt = LatentPromptRunner(heads, max_tokens=2048, max_context=8192, scale=SCALE)
        self.table = torch.zeros(seqs, width, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        a = torch.arange(2048, dtype=F64)[:, None] * 10000.0 ** (-torch.arange(32, dtype=F64) / 32)
        self.cos_sin = torch.cat([a.cos(), a.sin()], 1).float().cuda()
        self.rows = [[torch.zeros(0, 576, dtype=F64, device="cuda")] * seqs for _ in range(layers)]  # by sequence

    def i32(self, v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    def step(self, add, runner):
        """Every layer's step of so many new tokens a sequence, each output near the definition."""
        t = sum(add)
        slots, positions, starts = self.pool.grow(self.table, self.lens, self.i32(add), t)
        for layer, (cache, w) in enumerate(zip(self.caches, self.w)):
            q, kv = self.rand(t, self.heads, 192), self.rand(t, 576)
            out = runner.attention(w, cache, q, kv, self.cos_sin, positions, slots, self.table, self.lens, q_starts=starts)
            new = ref.row_values(runner_rows(runner, cache, slots))
            cs = self.cos_sin[positions.long()]
            q_pe, _ = ref.rotate(q[..., 128:].double(), cs[:, None], False)
            at = 0
            for b, n in enumerate(add):
                rows = self.rows[layer][b] = torch.cat([self.rows[layer][b], new[at : at + n]])
                self.check(out[at : at + n], q[at : at + n, :, :128].double(), q_pe[at : at + n], rows, w)
                at += n
        torch.cuda.synchronize()
        self.pool.raise_on_device_error()
        runner.raise_on_device_error()

    def check(self, out, q_nope, q_pe, rows, w):
        if out.shape[0] == 0:
            return
        kv = w.kv_b.double().view(self.heads, 2, 128, 512)
        n, length = out.shape[0], rows.shape[0]
        see = torch.arange(length, device="cuda") <= (length - n + torch.arange(n, device="cuda"))[:, None]
        for h in range(self.heads):
            k, v = rows[:, :512] @ kv[h, 0].T, rows[:, :512] @ kv[h, 1].T
            s = ((q_nope[:, h] @ k.T + q_pe[:, h] @ rows[:, 512:].T) * SCALE).masked_fill(~see, -float("inf"))
            want = torch.softmax(s, 1) @ v
            # roundings of 2^-8 / sqrt 3 each: the output, numerators, values, and to the scores keys, query (absorbed) and its
            # rotated part: 6 independent ones at most
            assert ((out[:, h].double() - want).norm() / want.norm()).item() <= (6 / 3) ** 0.5 * ref.U16

    def fork(self, parents):
        self.pool.fork(self.table, self.lens, self.i32(parents))
        empty = torch.zeros(0, 576, dtype=F64, device="cuda")
        self.rows = [[r[p] if p >= 0 else empty for p in parents] for r in self.rows]

    def trim(self, keep):
        self.pool.trim(self.table, self.lens, self.i32(keep))
        self.rows = [[x[:n] for x, n in zip(r, keep)] for r in self.rows]

    def stored(self):
        """Every sequence's cached rows are its own."""
        page = self.caches[0].shape[1]
        for layer, cache in enumerate(self.caches):
            for b, rows in enumerate(self.rows[layer]):
                assert int(self.lens[b]) == rows.shape[0]
                if rows.shape[0]:
                    got = ref.row_values(ref.sequence_rows(cache, self.table, b, rows.shape[0]))
                    assert torch.equal(got, rows), (layer, b)
        held = {int(p) for b in range(len(self.lens)) for p in self.table[b, : -(-int(self.lens[b]) // page)]}
        assert {i for i, r in enumerate(self.pool.refs.tolist()) if r} == held


def runner_rows(runner, cache, slots):
    """The cache's own rows at slots, as they are stored."""
    return cache.view(-1, cache.shape[-1])[slots.long()]


@pytest.mark.parametrize("fmt,page", [("bf16", 16), ("mxfp8", 64), ("bf16", 1)])
def test_a_server_s_life(fmt, page):
    print(f"\nserver {fmt} page={page}", flush=True)
    pages = 40 * 64 // page + 60
    s = Server(fmt, page, 3, pages=pages, width=1024 // page)
    s.step([300, 41, 0, 130, 0, 0], s.prompt)  # prompts
    s.stored()
    s.fork([0, 1, 1, 3, 0, 1])  # samples of the first and the second one
    s.stored()
    for _ in range(3):
        s.step([1] * 6, s.one)  # a token each
    s.stored()
    s.step([4, 3, 1, 4, 2, 4], s.one)  # drafts, some of them taken back
    n = s.lens.tolist()
    s.trim([n[0] - 3, n[1], n[2] - 1, n[3] - 4, n[4] - 1, n[5] - 2])
    s.stored()
    s.fork([5, 5, 2, -1, 0, 0])  # beams: rows dropped and permuted
    s.stored()
    s.pool.compact(s.table, s.lens)
    s.stored()
    assert int(s.pool.refs[: int((s.pool.refs > 0).sum())].min()) > 0
    s.step([150, 1, 2, 200, 77, 0], s.prompt)  # a prompt's next chunk beside others
    n = s.lens.tolist()
    s.trim([100, n[1], 20, 0, n[4], n[5] - 1])  # cut into pages that others hold
    s.stored()
    s.step([1, 1, 1, 64, 1, 1], s.prompt)
    s.stored()
    s.trim([0] * 6)
    assert not s.pool.refs.any()
