"""A prompt's attention on the host side, without a GPU: the C ABI's argument checks (each returns before any HIP
call, so fake device addresses are safe), the structure's layout, and the runner's checks."""

import ctypes

import pytest
import torch

from test_latent_host import CACHES, _append, _cache, _weights

BF, I32 = torch.bfloat16, torch.int32
AT, WS = 0x100000, 0x200000


def _prompt(**over):
    from sgl_amd_mono.moe import _lib

    v = dict(
        cache=_cache(), seqs=2, tokens=4, heads=8, max_pages=5, max_context=1000, table_stride=5, qn_token_stride=1536,
        qn_head_stride=192, qp_token_stride=512, qp_head_stride=64, out_token_stride=1024, out_head_stride=128, q_nope=AT,
        q_pe=AT, w=AT, table=AT, lens=AT, q_starts=None, out=AT, lse=None, scale=0.1,
    )  # fmt: skip
    return _lib.LatentPromptIO(**{**v, **over})


@pytest.fixture(scope="module")
def lib():
    from sgl_amd_mono.moe import _lib

    L = _lib.lib()
    n = ctypes.c_size_t()
    assert L.mkmoe_latent_prompt_bytes(8, 1000, ctypes.byref(n)) == 0 and n.value % 256 == 0
    return L, n.value


def test_workspace_bytes(lib):
    L, n = lib
    size = ctypes.c_size_t()
    get = lambda h, c: (L.mkmoe_latent_prompt_bytes(h, c, ctypes.byref(size)), size.value)[::-1]  # noqa: E731
    # 1024 rows at 8 heads: latents, rope values, keys and values, flags
    assert get(8, 1000) == get(8, 1024) == (n, 0)
    assert get(8, 1152)[0] - n == 128 * (1152 + 8 * 512) + 256 * (8 * 18 * 4 > 512)
    assert get(1, 1)[0] < 137 << 20  # (the latent calls' 67 MB are a part of it)
    for h, c in ((0, 1), (129, 1), (1, 0), (1, (1 << 22) + 1)):
        assert get(h, c)[1] == -8
    assert L.mkmoe_latent_prompt_bytes(1, 1, None) == -1
    assert get(128, 1 << 22)[0] > 128 * (1 << 22) * 512  # past 32 bits


@pytest.mark.parametrize("over,code", [(dict(cache=c), e) for c, e in CACHES] + [
    (dict(q_nope=None), -1),
    (dict(q_pe=None), -1),
    (dict(w=None), -1),
    (dict(table=None), -1),
    (dict(lens=None), -1),
    (dict(out=None), -1),
    (dict(seqs=0), -3),
    (dict(seqs=513, tokens=513), -3),
    (dict(tokens=-4), -3),
    (dict(tokens=5), -3),  # not as many for each sequence
    (dict(tokens=(1 << 20) + 2), -3),
    (dict(heads=0), -8),
    (dict(heads=129), -8),
    (dict(max_context=0), -8),
    (dict(max_context=(1 << 22) + 1), -8),
    (dict(max_context=2000), -5),  # the workspace is of 1000
    (dict(heads=9), -5),
    (dict(max_pages=0), -8),
    (dict(table_stride=4), -8),
    (dict(max_pages=1 << 27, table_stride=1 << 27), -8),  # 2^31 tokens a sequence
    (dict(scale=float("nan")), -8),
    (dict(scale=float("-inf")), -8),
    (dict(scale=3e38), -8),  # (times log2 e it is past fp32)
    (dict(q_nope=AT + 8), -4),
    (dict(q_pe=AT + 2), -4),
    (dict(w=AT + 8), -4),
    (dict(out=AT + 8), -4),
    (dict(table=AT + 1), -4),
    (dict(lens=AT + 2), -4),
    (dict(q_starts=AT + 1), -4),
    (dict(lse=AT + 2), -4),
    (dict(qn_head_stride=132), -4),
    (dict(qp_token_stride=-64), -4),
    (dict(out_token_stride=0), -8),
    (dict(out_head_stride=120), -8),
    (dict(out_token_stride=128, out_head_stride=256), -8),  # head 1's rows among token 2's
    (dict(tokens=0), 0),
])  # fmt: skip
def test_prompt_rejects_bad_arguments(lib, over, code):
    L, n = lib
    over = {**over, **({"cache": _cache(**over["cache"])} if "cache" in over else {})}
    assert L.mkmoe_latent_prompt(ctypes.byref(_prompt(**over)), WS, n, None) == code
    assert L.mkmoe_latent_prompt(None, WS, n, None) == -1


def test_more_work_than_32_bits_count(lib):
    L, _ = lib
    io = _prompt(tokens=1 << 20, seqs=1, heads=128, max_pages=1 << 18, table_stride=1 << 18, max_context=1 << 22,
                 out_token_stride=16384, qn_token_stride=24576, qp_token_stride=8192)  # fmt: skip
    assert L.mkmoe_latent_prompt(ctypes.byref(io), WS, 1 << 40, None) == -8
    # (counted: 64 sequences of 1024 that may have 2^20 cached tokens, in one of its two cuts; the next check refuses)
    io = _prompt(tokens=1 << 16, seqs=64, heads=128, max_pages=1 << 14, table_stride=1 << 14, max_context=1 << 20,
                 out_token_stride=16384, qn_token_stride=24576, qp_token_stride=8192, w=AT + 2)  # fmt: skip
    assert L.mkmoe_latent_prompt(ctypes.byref(io), WS, 1 << 40, None) == -4


@pytest.mark.parametrize("ws,size,code", [(None, 0, -1), (WS + 128, 0, -4), (WS, -1, -5)])
def test_workspace_is_checked(lib, ws, size, code):
    L, n = lib
    assert L.mkmoe_latent_prompt(ctypes.byref(_prompt()), ws, n + size, None) == code
    assert L.mkmoe_latent_prompt_step(ctypes.byref(_append()), ctypes.byref(_prompt()), ws, n + size, None) == code


@pytest.mark.parametrize("append,prompt,code", [
    (dict(kv=None), {}, -1),
    (dict(q_out=AT + 2), {}, -4),
    ({}, dict(w=None), -1),
    (dict(tokens=2), {}, -3),
    (dict(heads=4), {}, -8),
    (dict(cache=dict(pages=9)), {}, -8),
    (dict(cache=dict(page_size=8)), {}, -8),
    (dict(cache=dict(data=AT + 256)), {}, -8),
    (dict(cache=dict(fmt=2)), {}, -8),
    (dict(tokens=0), dict(tokens=0), 0),
])  # fmt: skip
def test_step_checks_both_first(lib, append, prompt, code):
    L, n = lib
    append = {**append, **({"cache": _cache(**append["cache"])} if "cache" in append else {})}
    assert L.mkmoe_latent_prompt_step(ctypes.byref(_append(**append)), ctypes.byref(_prompt(**prompt)), WS, n, None) == code
    assert L.mkmoe_latent_prompt_step(None, ctypes.byref(_prompt()), WS, n, None) == -1
    assert L.mkmoe_latent_prompt_step(ctypes.byref(_append()), None, WS, n, None) == -1


def test_packed_fields_are_the_structure():
    from sgl_amd_mono.moe import _lib

    one, at_once, values = _lib.LatentPromptIO(), _lib.LatentPromptIO(), []

    def fill(x):
        for name, t in x._fields_:
            if hasattr(t, "_fields_"):
                fill(getattr(x, name))
            else:
                values.append(0.5 * len(values) if t is ctypes.c_float else 3 * len(values) + 1)
                setattr(x, name, values[-1])

    fill(one)
    _lib.LATENT_PROMPT.pack_into(at_once, 0, *values)
    assert bytes(one) == bytes(at_once)


# ---------------------------------------------------------------- the runner
def test_runner_rejects_bad_options():
    from sgl_amd_mono.moe.latent_prompt import LatentPromptRunner

    for kw, err in (
        (dict(heads=0), "0 heads"), (dict(heads=8, device="cpu"), "not a GPU"), (dict(heads=8, rope="neox"), "rope"),
        (dict(heads=8, max_context=0), "max_context 0"), (dict(heads=8, max_context=1 << 23), "max_context"),
        (dict(heads=8, max_tokens=-1), "max_tokens -1"), (dict(heads=8, max_tokens=1 << 21), "max_tokens"),
        (dict(heads=8, scale=float("nan")), "scale"), (dict(heads=8, norm_eps=-1.0), "norm_eps"),
    ):  # fmt: skip
        with pytest.raises((RuntimeError, ValueError), match=err):
            LatentPromptRunner(**kw)


@pytest.fixture
def runner():
    """A runner whose tensors lie on the host; a call that passes its checks is written down."""
    from sgl_amd_mono.moe import _lib
    from sgl_amd_mono.moe.latent_prompt import LatentPromptRunner

    r = LatentPromptRunner.__new__(LatentPromptRunner)
    r.heads, r.max_tokens, r.max_context, r.scale, r.norm_eps, r.rope = 8, 6, 640, 0.1, 1e-6, 0
    r.device, r._index, r.lib, r._ws = torch.device("cpu"), -1, _lib.lib(), (0, 0)
    r._append_io, r._prompt_io = _lib.LatentAppendIO(), _lib.LatentPromptIO()
    r._q_pe = torch.empty(6, 8, 64, dtype=BF)
    r.calls = []
    r._call = lambda fn, *a: r.calls.append((fn.__name__, a))
    return r


def _args(t=4):
    return dict(
        cache=torch.zeros(10, 16, 576, dtype=BF), q_nope=torch.zeros(t, 8, 192, dtype=BF)[..., :128],
        q_pe=torch.zeros(t, 8, 64, dtype=BF), table=torch.zeros(2, 5, dtype=I32), lens=torch.zeros(2, dtype=I32),
    )  # fmt: skip


def _step(t=4):
    return dict(
        cache=torch.zeros(10, 16, 576, dtype=BF), q=torch.zeros(t, 8, 192, dtype=BF), kv=torch.zeros(t, 576, dtype=BF),
        cos_sin=torch.zeros(50, 64), positions=torch.zeros(t, dtype=I32), slots=torch.zeros(t, dtype=I32),
        table=torch.zeros(2, 5, dtype=I32), lens=torch.zeros(2, dtype=I32),
    )  # fmt: skip


def test_attend_fills_what_the_library_reads(runner):
    d, w = _args(), _weights(False)
    d["q_pe"] = torch.zeros(8, 4, 72, dtype=BF)[..., :64].transpose(0, 1)
    out, lse = torch.empty(4, 8, 128, dtype=BF), torch.empty(4, 8)
    starts = torch.zeros(3, dtype=I32)
    assert runner.attend(w, **d, q_starts=starts, out=out, lse=lse) is out
    ((name, (io, *_)),) = runner.calls
    assert name == "mkmoe_latent_prompt"
    assert (io.seqs, io.tokens, io.heads, io.max_pages, io.max_context, io.table_stride) == (2, 4, 8, 5, 640, 5)
    assert (io.q_nope, io.qn_token_stride, io.qn_head_stride) == (d["q_nope"].data_ptr(), 1536, 192)
    assert (io.q_pe, io.qp_token_stride, io.qp_head_stride) == (d["q_pe"].data_ptr(), 72, 288)
    assert (io.out, io.out_token_stride, io.out_head_stride, io.lse) == (out.data_ptr(), 1024, 128, lse.data_ptr())
    assert (io.w, io.table, io.lens, io.q_starts) == (
        w.kv_b.data_ptr(), d["table"].data_ptr(), d["lens"].data_ptr(), starts.data_ptr())  # fmt: skip
    assert (io.cache.data, io.cache.pages, io.cache.page_size, io.cache.fmt) == (d["cache"].data_ptr(), 10, 16, 1)


def test_attention_fills_what_the_library_reads(runner):
    d, w, out = _step(), _weights(False), torch.empty(4, 8, 128, dtype=BF)
    assert runner.attention(w, **d, out=out) is out
    ((name, (a, io, *_)),) = runner.calls
    assert name == "mkmoe_latent_prompt_step"
    assert (a.tokens, a.heads, a.index_bytes, a.q_out_nan, a.norm_w) == (4, 8, 4, 1, w.norm.data_ptr())
    assert (a.q_pe, a.q_token_stride, a.q_head_stride) == (d["q"].data_ptr() + 256, 1536, 192)
    assert (a.q_out, a.out_token_stride, a.out_head_stride) == (io.q_pe, io.qp_token_stride, io.qp_head_stride)
    assert (io.q_nope, io.qn_token_stride, io.qn_head_stride) == (d["q"].data_ptr(), 1536, 192)
    assert a.q_out == runner._q_pe.data_ptr() and io.q_starts is None and io.lse is None


@pytest.mark.parametrize("over,err", [
    (dict(cache=None), "cache: missing"),
    (dict(cache=torch.zeros(10, 16, 575, dtype=BF)), "cache"),
    (dict(cache=torch.zeros(10, 16, 656, dtype=torch.int8)), "cache"),
    (dict(q_nope=None), "q_nope: missing"),
    (dict(q_nope=torch.zeros(4, 8, 128)), "q_nope"),
    (dict(q_nope=torch.zeros(4, 7, 128, dtype=BF)), "q_nope"),
    (dict(q_nope=torch.zeros(4, 8, 132, dtype=BF)[..., 4:]), "q_nope"),
    (dict(q_pe=None), "q_pe: missing"),
    (dict(q_pe=torch.zeros(3, 8, 64, dtype=BF)), "q_pe"),
    (dict(table=torch.zeros(2, 5, dtype=torch.int64)), "table"),
    (dict(table=torch.zeros(5, 2, dtype=I32).T), "table"),
    (dict(lens=torch.zeros(3, dtype=I32)), "lens"),
    (dict(q_starts=torch.zeros(2, dtype=I32)), "q_starts"),
    (dict(table=torch.zeros(3, 5, dtype=I32), lens=torch.zeros(3, dtype=I32)), "3 sequences of 4"),
    (dict(out=torch.zeros(4, 8, 128)), "out"),
    (dict(out=torch.zeros(4, 1, 128, dtype=BF).expand(4, 8, 128)), "out"),
    (dict(lse=torch.zeros(8, 4)), "lse"),
])  # fmt: skip
def test_attend_refuses(runner, over, err):
    out = dict(out=torch.empty(4, 8, 128, dtype=BF))
    with pytest.raises(RuntimeError, match=err):
        runner.attend(_weights(False), **{**_args(), **out, **over})
    assert not runner.calls


@pytest.mark.parametrize("over,err", [
    (dict(q=None), "q: missing"),
    (dict(q=torch.zeros(7, 8, 192, dtype=BF)), "tokens <= 6"),
    (dict(kv=torch.zeros(3, 576, dtype=BF)), "kv"),
    (dict(kv=None), "kv: missing"),
    (dict(slots=torch.zeros(4, dtype=torch.int64)), "slots"),
    (dict(positions=None), "positions"),
    (dict(cos_sin=torch.zeros(50, 32)), "cos_sin"),
    (dict(lens=None), "lens"),
])  # fmt: skip
def test_attention_refuses(runner, over, err):
    with pytest.raises(RuntimeError, match=err):
        runner.attention(_weights(False), **{**_step(), **over}, out=torch.empty(4, 8, 128, dtype=BF))
    assert not runner.calls


def test_no_tokens_make_no_call(runner):
    runner.attend(_weights(False), **_args(0), out=torch.empty(0, 8, 128, dtype=BF))
    assert not runner.calls
    with pytest.raises(RuntimeError, match="latent norm"):
        runner.attend(_weights(), **_args(), out=torch.empty(4, 8, 128, dtype=BF))
