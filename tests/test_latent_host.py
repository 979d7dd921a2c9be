"""Latent attention's host side without a GPU: the C ABI's argument checks (each returns before any
HIP call, so fake device addresses are safe), the structures' layout, and the runner's checks."""

import ctypes

import pytest
import torch

BF = torch.bfloat16
AT = 0x100000  # a device address that nothing is read from


def _cache(**over):
    from sgl_amd_mono.moe import _lib

    return _lib.LatentCache(**{**dict(data=AT, pages=10, page_size=16, fmt=_lib.LATENT_BF16), **over})


def _append(**over):
    from sgl_amd_mono.moe import _lib

    v = dict(
        cache=_cache(), tokens=4, heads=8, rope=0, index_bytes=8, cos_sin_rows=100, kv_stride=576, q_token_stride=1536,
        q_head_stride=192, out_token_stride=512, out_head_stride=64, kv=AT, norm_w=AT, cos_sin=AT, positions=AT, slots=AT,
        q_pe=AT, q_out=AT, norm_eps=1e-6,
    )  # fmt: skip
    return _lib.LatentAppendIO(**{**v, **over})


def _attend(**over):
    from sgl_amd_mono.moe import _lib

    v = dict(
        cache=_cache(), seqs=2, tokens=4, heads=8, max_pages=5, table_stride=5, ql_token_stride=4096, ql_head_stride=512,
        qp_token_stride=512, qp_head_stride=64, out_token_stride=4096, out_head_stride=512, q_lat=AT, q_pe=AT, table=AT,
        lens=AT, q_starts=None, out=AT, lse=None, scale=0.1, out_f32=0,
    )  # fmt: skip
    return _lib.LatentAttendIO(**{**v, **over})


def _project(which, /, **over):
    from sgl_amd_mono.moe import _lib

    x, y = (512, 128) if which else (128, 512)
    v = dict(tokens=4, heads=8, expand=which, x_f32=0, x_token_stride=8 * x, x_head_stride=x, y_token_stride=8 * y,
             y_head_stride=y, x=AT, w=AT, y=AT)  # fmt: skip
    return _lib.LatentProjectIO(**{**v, **over})


@pytest.fixture(scope="module")
def lib():
    from sgl_amd_mono.moe import _lib

    L = _lib.lib()
    n = ctypes.c_size_t()
    assert L.mkmoe_latent_workspace_bytes(ctypes.byref(n)) == 0 and n.value % 256 == 0
    assert L.mkmoe_latent_workspace_bytes(None) == -1
    return L, n.value


CACHES = [
    (dict(data=None), -1),
    (dict(data=AT + 8), -4),
    (dict(fmt=0), -8),
    (dict(fmt=3), -8),
    (dict(page_size=0), -8),
    (dict(page_size=24), -8),
    (dict(page_size=2048), -8),
    (dict(pages=0), -8),
    (dict(pages=1 << 27), -8),  # 2^31 rows
]


@pytest.mark.parametrize("over,code", [(dict(cache=c), e) for c, e in CACHES] + [
    (dict(kv=None), -1),
    (dict(cos_sin=None), -1),
    (dict(positions=None), -1),
    (dict(slots=None), -1),
    (dict(q_pe=None), -1),
    (dict(q_out=None), -1),
    (dict(tokens=-1), -3),
    (dict(tokens=(1 << 24) + 1), -3),
    (dict(heads=-1), -8),
    (dict(heads=129), -8),
    (dict(rope=2), -8),
    (dict(index_bytes=2), -8),
    (dict(cos_sin_rows=0), -8),
    (dict(norm_eps=-1.0), -8),
    (dict(norm_eps=float("nan")), -8),
    (dict(norm_eps=float("inf")), -8),
    (dict(kv_stride=568), -8),
    (dict(kv_stride=580), -4),
    (dict(kv=AT + 8), -4),
    (dict(norm_w=AT + 2), -4),
    (dict(positions=AT + 4), -4),
    (dict(q_pe=AT + 2), -4),
    (dict(q_head_stride=60), -4),
    (dict(q_token_stride=-64), -4),
    (dict(out_head_stride=0), -8),
    (dict(out_head_stride=56), -8),
    (dict(out_token_stride=504), -8),
    (dict(tokens=0), 0),
])  # fmt: skip
def test_append_rejects_bad_arguments(lib, over, code):
    L, n = lib
    over = {**over, **({"cache": _cache(**over["cache"])} if "cache" in over else {})}
    assert L.mkmoe_latent_append(ctypes.byref(_append(**over)), 0x200000, n, None) == code


@pytest.mark.parametrize("over,code", [(dict(cache=c), e) for c, e in CACHES] + [
    (dict(q_lat=None), -1),
    (dict(q_pe=None), -1),
    (dict(table=None), -1),
    (dict(lens=None), -1),
    (dict(out=None), -1),
    (dict(seqs=0), -3),
    (dict(seqs=513, tokens=513), -3),
    (dict(tokens=-4), -3),
    (dict(tokens=5), -3),  # not as many for each sequence
    (dict(tokens=1 << 22), -3),  # 2^25 rows
    (dict(heads=0), -8),
    (dict(heads=129), -8),
    (dict(max_pages=0), -8),
    (dict(table_stride=4), -8),
    (dict(max_pages=1 << 27, table_stride=1 << 27), -8),  # 2^31 tokens a sequence
    (dict(tokens=1 << 20, max_pages=1 << 25, table_stride=1 << 25), -8),  # more tiles than 32 bits count
    (dict(scale=float("nan")), -8),
    (dict(scale=float("inf")), -8),
    (dict(out_f32=2), -8),
    (dict(q_lat=AT + 8), -4),
    (dict(out=AT + 8), -4),
    (dict(lens=AT + 2), -4),
    (dict(q_starts=AT + 1), -4),
    (dict(lse=AT + 2), -4),
    (dict(ql_head_stride=516), -4),
    (dict(out_token_stride=-8), -4),
    (dict(out_token_stride=0), -8),
    (dict(out_head_stride=504), -8),
    (dict(out_token_stride=512, out_head_stride=1536), -8),  # head 1's rows among token 3's
    (dict(tokens=0), 0),
])  # fmt: skip
def test_attend_rejects_bad_arguments(lib, over, code):
    L, n = lib
    over = {**over, **({"cache": _cache(**over["cache"])} if "cache" in over else {})}
    assert L.mkmoe_latent_attend(ctypes.byref(_attend(**over)), 0x200000, n, None) == code


@pytest.mark.parametrize("expand", [0, 1])
@pytest.mark.parametrize("over,code", [
    (dict(x=None), -1),
    (dict(w=None), -1),
    (dict(y=None), -1),
    (dict(tokens=-1), -3),
    (dict(tokens=(1 << 20) + 1), -3),
    (dict(heads=0), -8),
    (dict(heads=129), -8),
    (dict(expand=2), -8),
    (dict(x_f32=2), -8),
    (dict(x=AT + 4), -4),
    (dict(w=AT + 8), -4),
    (dict(x_token_stride=4), -4),
    (dict(y_head_stride=8), -8),
    (dict(y_token_stride=0), -8),
    (dict(tokens=0), 0),
])  # fmt: skip
def test_project_rejects_bad_arguments(lib, expand, over, code):
    L, _ = lib
    assert L.mkmoe_latent_project(ctypes.byref(_project(expand, **over)), None) == code
    if not expand:
        assert L.mkmoe_latent_project(ctypes.byref(_project(0, x_f32=1)), None) == -8


def test_rows_rejects_bad_arguments(lib):
    L, n = lib
    rows = lambda c=None, slots=AT, ib=8, tokens=3, out=AT, ws=0x200000, size=n: L.mkmoe_latent_rows(  # noqa: E731
        ctypes.byref(c or _cache()), slots, ib, tokens, out, ws, size, None)  # fmt: skip
    assert L.mkmoe_latent_rows(None, AT, 8, 3, AT, 0x200000, n, None) == -1
    assert rows(slots=None) == -1 and rows(out=None) == -1
    for c, e in CACHES:
        assert rows(c=_cache(**c)) == e
    assert rows(tokens=-1) == -3 and rows(ib=3) == -8 and rows(out=AT + 8) == -4 and rows(slots=AT + 4) == -4
    assert rows(tokens=0) == 0


@pytest.mark.parametrize("ws,size,code", [(None, 0, -1), (0x200080, 0, -4), (0x200000, -1, -5)])
def test_workspace_is_checked(lib, ws, size, code):
    L, n = lib
    size += n
    assert L.mkmoe_latent_append(ctypes.byref(_append()), ws, size, None) == code
    assert L.mkmoe_latent_attend(ctypes.byref(_attend()), ws, size, None) == code
    assert L.mkmoe_latent_rows(ctypes.byref(_cache()), AT, 8, 3, AT, ws, size, None) == code
    assert L.mkmoe_latent_step(*map(ctypes.byref, (_append(), _project(0), _attend(), _project(1))), ws, size, None) == code


@pytest.mark.parametrize("parts,code", [
    (dict(append=dict(kv=None)), -1),
    (dict(absorb=dict(w=None)), -1),
    (dict(attend=dict(scale=float("nan"))), -8),
    (dict(expand=dict(y=AT + 2)), -4),
    (dict(absorb=dict(expand=1)), -8),
    (dict(expand=dict(expand=0, y_token_stride=4096, y_head_stride=512)), -8),
    (dict(append=dict(tokens=2)), -3),
    (dict(absorb=dict(tokens=8)), -3),
    (dict(expand=dict(tokens=0)), -3),
    (dict(append=dict(tokens=0), absorb=dict(tokens=0), attend=dict(tokens=0), expand=dict(tokens=0)), 0),
])  # fmt: skip
def test_step_checks_all_of_it_first(lib, parts, code):
    """Whichever part is wrong: nothing is launched (the addresses are fake)."""
    L, n = lib
    get = lambda k: parts.get(k, {})  # noqa: E731
    io = (_append(**get("append")), _project(0, **get("absorb")), _attend(**get("attend")), _project(1, **get("expand")))
    assert L.mkmoe_latent_step(*map(ctypes.byref, io), 0x200000, n, None) == code
    io = (_append(), _project(0), _attend(), _project(1))
    for i in range(4):
        assert L.mkmoe_latent_step(*[None if j == i else ctypes.byref(x) for j, x in enumerate(io)], 0x200000, n, None) == -1


def test_read_errors_rejects_bad_arguments(lib):
    L, _ = lib
    words = (ctypes.c_int32 * 4)()
    assert L.mkmoe_latent_read_errors(None, words, 4, None) == -1
    assert L.mkmoe_latent_read_errors(AT, None, 4, None) == -1
    assert L.mkmoe_latent_read_errors(AT, words, 0, None) == -8
    assert L.mkmoe_latent_read_errors(AT, words, 5, None) == -8


def test_packed_fields_are_the_structure():
    """One value a field, written at once, against the fields set one by one."""
    from sgl_amd_mono.moe import _lib

    for cls, pack in ((_lib.LatentAppendIO, _lib.LATENT_APPEND), (_lib.LatentAttendIO, _lib.LATENT_ATTEND),
                      (_lib.LatentProjectIO, _lib.LATENT_PROJECT)):  # fmt: skip
        one, at_once, values = cls(), cls(), []

        def fill(x):
            for name, t in x._fields_:
                if hasattr(t, "_fields_"):
                    fill(getattr(x, name))
                else:
                    values.append(0.5 * len(values) if t is ctypes.c_float else 3 * len(values) + 1)
                    setattr(x, name, values[-1])

        fill(one)
        pack.pack_into(at_once, 0, *values)
        assert bytes(one) == bytes(at_once)


# ---------------------------------------------------------------- the runner
def test_runner_rejects_bad_options():
    from sgl_amd_mono.moe.latent import LatentRunner, cache_like

    for kw, err in (
        (dict(heads=0), "0 heads"), (dict(heads=129), "129 heads"), (dict(heads=8, device="cpu"), "not a GPU"),
        (dict(heads=8, rope="neox"), "rope"), (dict(heads=8, device="cuda", scale=float("inf")), "scale"),
        (dict(heads=8, device="cuda", norm_eps=-1.0), "norm_eps"),
    ):  # fmt: skip
        with pytest.raises((RuntimeError, ValueError), match=err):
            LatentRunner(**kw)
    with pytest.raises(ValueError, match="bf16 or mxfp8"):
        cache_like(1, 1, "fp8", "cpu")
    assert cache_like(2, 4, "bf16", "cpu").shape == (2, 4, 576)
    assert cache_like(2, 4, "mxfp8", "cpu").shape == (2, 4, 656)


@pytest.fixture
def host_runner():
    """A runner whose tensors lie on the host: its checks are the same, and a call that passes them
    is written down instead of made."""
    from sgl_amd_mono.moe import _lib
    from sgl_amd_mono.moe.latent import LatentRunner

    r = LatentRunner.__new__(LatentRunner)
    r.heads, r.max_tokens, r.scale, r.norm_eps, r.rope = 8, 6, 0.1, 1e-6, 0
    r.device, r._index, r.lib, r._ws = torch.device("cpu"), -1, _lib.lib(), (0, 0)
    r._append_io, r._attend_io = _lib.LatentAppendIO(), _lib.LatentAttendIO()
    r._absorb_io, r._expand_io = _lib.LatentProjectIO(), _lib.LatentProjectIO()
    r._q_lat, r._q_pe = torch.empty(6, 8, 512, dtype=BF), torch.empty(6, 8, 64, dtype=BF)
    r._o_lat = torch.empty(6, 8, 512)
    r.calls = []
    r._call = lambda fn, *a: r.calls.append((fn.__name__, a))
    return r


def _step(t=4):
    i32 = torch.int32
    return dict(
        cache=torch.zeros(10, 16, 576, dtype=BF), q=torch.zeros(t, 8, 192, dtype=BF), kv=torch.zeros(t, 576, dtype=BF),
        cos_sin=torch.zeros(50, 64), positions=torch.zeros(t, dtype=torch.int64), slots=torch.zeros(t, dtype=torch.int64),
        table=torch.zeros(2, 5, dtype=i32), lens=torch.zeros(2, dtype=i32),
    )  # fmt: skip


def _weights(check=True):
    from sgl_amd_mono.moe.latent import LatentWeights

    w = LatentWeights(norm=torch.zeros(512, dtype=BF), kv_b=torch.zeros(8 * 256, 512, dtype=BF))
    if not check:  # (the weights' own check wants a GPU)
        w.check = lambda heads, device=None: None
    return w


def test_weights_are_checked(host_runner):
    w = _weights()
    with pytest.raises(RuntimeError, match="latent norm"):
        w.check(8)
    w.norm = None
    with pytest.raises(RuntimeError, match="norm: missing"):
        w.check(8)
    with pytest.raises(RuntimeError, match="latent norm"):
        host_runner.attention(_weights(), **_step(), out=torch.empty(4, 8, 128, dtype=BF))


def test_attention_fills_what_the_library_reads(host_runner):
    """Pointers, strides and sizes of a step, as the structures that the call is given hold them."""
    r, d, w = host_runner, _step(), _weights(False)
    d["q"] = torch.zeros(8, 4, 200, dtype=BF)[..., :192].transpose(0, 1)  # the head axis outermost
    out = torch.empty(4, 8, 128, dtype=BF)
    assert r.attention(w, **d, out=out) is out
    ((name, (a, k, s, v, *_)),) = r.calls
    assert name == "mkmoe_latent_step"
    assert (a.tokens, a.heads, a.index_bytes, a.cos_sin_rows, a.kv_stride) == (4, 8, 8, 50, 576)
    assert (a.q_pe, a.q_token_stride, a.q_head_stride) == (d["q"].data_ptr() + 256, 200, 800)
    assert (k.x, k.x_token_stride, k.x_head_stride, k.expand) == (d["q"].data_ptr(), 200, 800, 0)
    assert (k.y, k.y_token_stride, k.y_head_stride) == (s.q_lat, s.ql_token_stride, s.ql_head_stride) == (r._q_lat.data_ptr(), 4096, 512)
    assert (a.q_out, a.out_token_stride, a.out_head_stride) == (s.q_pe, s.qp_token_stride, s.qp_head_stride)
    assert (s.out, s.out_f32, s.out_token_stride, s.out_head_stride) == (v.x, v.x_f32, v.x_token_stride, v.x_head_stride)
    assert (s.seqs, s.tokens, s.heads, s.max_pages, s.table_stride, s.q_starts, s.lse) == (2, 4, 8, 5, 5, None, None)
    assert (v.expand, v.y, v.y_token_stride, v.y_head_stride) == (1, out.data_ptr(), 1024, 128)
    assert k.w == v.w == w.kv_b.data_ptr() and a.norm_w == w.norm.data_ptr()
    assert (s.cache.data, s.cache.pages, s.cache.page_size, s.cache.fmt) == (d["cache"].data_ptr(), 10, 16, 1)


BAD_STEPS = [
    ("cache", lambda t: t[..., :575]), ("cache", lambda t: t.float()), ("cache", lambda t: t.transpose(0, 1)),
    ("cache", lambda t: t[:, :, :1].to(torch.uint8)), ("cache", lambda t: None),
    ("q", lambda t: t[..., :191]), ("q", lambda t: t[:, :7]), ("q", lambda t: t.float()), ("q", lambda t: None),
    ("q", lambda t: torch.zeros(4, 8, 196, dtype=BF)[..., :192]), ("q", lambda t: torch.zeros(7, 8, 192, dtype=BF)),
    ("q", lambda t: torch.zeros(4 * 8 * 192 + 1, dtype=BF)[1:].view(4, 8, 192)),
    ("kv", lambda t: t[:3]), ("kv", lambda t: t[:, :512]), ("kv", lambda t: t.half()), ("kv", lambda t: None),
    ("kv", lambda t: torch.zeros(576, 4, dtype=BF).T),
    ("cos_sin", lambda t: t.double()), ("cos_sin", lambda t: t[:, :32]), ("cos_sin", lambda t: None),
    ("positions", lambda t: t[:3]), ("positions", lambda t: t.short()), ("positions", lambda t: None),
    ("slots", lambda t: t.int()), ("slots", lambda t: t.repeat(2)[::2]), ("slots", lambda t: None),
    ("table", lambda t: t.long()), ("table", lambda t: t[0]), ("table", lambda t: t.T), ("table", lambda t: None),
    ("table", lambda t: t[:1]), ("table", lambda t: torch.zeros(513, 5, dtype=torch.int32)),
    ("lens", lambda t: t.long()), ("lens", lambda t: t[:1]), ("lens", lambda t: None),
    ("q_starts", lambda t: torch.zeros(2, dtype=torch.int32)), ("q_starts", lambda t: torch.zeros(3)),
    ("out", lambda t: torch.empty(4, 8, 120, dtype=BF)), ("out", lambda t: torch.empty(4, 8, 128)),
    ("out", lambda t: torch.empty(1, 8, 128, dtype=BF).expand(4, 8, 128)),
    ("out", lambda t: torch.empty(4, 1, 128, dtype=BF).expand(4, 8, 128)),
]  # fmt: skip


@pytest.mark.parametrize("name,change", BAD_STEPS, ids=[f"{n}-{i}" for i, (n, _) in enumerate(BAD_STEPS)])
def test_attention_refuses_before_it_calls(host_runner, name, change):
    d = {**_step(), "out": torch.empty(4, 8, 128, dtype=BF)}
    d[name] = change(d.get(name))
    if name == "table" and d["table"] is not None and d["table"].dim() == 2 and d["table"].shape[0] != 2:
        d["lens"] = torch.zeros(max(1, d["table"].shape[0] - (d["table"].shape[0] == 1)), dtype=torch.int32)
        if d["table"].shape[0] == 1:  # (one sequence of four tokens would be right: the lengths are another's)
            d["lens"] = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="mkmoe latent"):
        host_runner.attention(_weights(False), **d)
    assert not host_runner.calls


def test_calls_refuse_mismatched_tensors(host_runner):
    r, d = host_runner, _step()
    ql, qp = torch.zeros(4, 8, 512, dtype=BF), torch.zeros(4, 8, 64, dtype=BF)
    attend = lambda **k: r.attend(**{**dict(cache=d["cache"], q_lat=ql, q_pe=qp, table=d["table"], lens=d["lens"], out=torch.empty_like(ql)), **k})  # noqa: E731
    for k in (dict(q_pe=qp[:3]), dict(q_lat=ql[..., :64]), dict(out=torch.empty(4, 8, 512, dtype=torch.float16)),
              dict(lse=torch.empty(4, 8, dtype=BF)), dict(lse=torch.empty(8, 4).T), dict(q_lat=None)):  # fmt: skip
        with pytest.raises(RuntimeError, match="mkmoe latent"):
            attend(**k)
    append = lambda **k: r.append(d["cache"], d["kv"], None, d["cos_sin"], d["positions"], d["slots"], **k)  # noqa: E731
    with pytest.raises(RuntimeError, match="without q_pe"):
        append(q_out=qp)
    with pytest.raises(RuntimeError, match="q_out"):
        append(q_pe=qp, q_out=qp[:, :1].expand(4, 8, 64))
    with pytest.raises(RuntimeError, match="slots"):
        r.rows(d["cache"], None)
    with pytest.raises(RuntimeError, match="out"):
        r.rows(d["cache"], d["slots"], out=torch.empty(4, 576))
    with pytest.raises(RuntimeError, match="q_nope"):
        r.absorb(_weights(False), torch.zeros(4, 8, 128))
    with pytest.raises(RuntimeError, match="o_lat"):
        r.expand(_weights(False), ql.half())
    assert not r.calls
    attend(), append(q_pe=qp, q_out=qp), r.expand(_weights(False), ql.float(), out=torch.empty(4, 8, 128, dtype=BF))
    assert [n for n, _ in r.calls] == ["mkmoe_latent_attend", "mkmoe_latent_append", "mkmoe_latent_project"]
    assert r._expand_io.x_f32 == 1


def test_append_rejects_an_unknown_mark(lib):
    L, n = lib
    assert L.mkmoe_latent_append(ctypes.byref(_append(q_out_nan=2)), 0x200000, n, None) == -8
    assert L.mkmoe_latent_append(ctypes.byref(_append(q_out_nan=1, tokens=0)), 0x200000, n, None) == 0


def test_append_marks_an_output_of_its_own(host_runner, monkeypatch):
    """A query that the caller provides keeps the rows of bad positions; one of the call's own has NaN there."""
    r, d, q = host_runner, _step(), torch.zeros(4, 8, 64, dtype=BF)
    monkeypatch.setattr(r, "_new", lambda what, *shape, **kw: torch.zeros(*shape, dtype=BF))
    for q_out in (None, torch.zeros_like(q)):
        r.append(d["cache"], d["kv"], None, d["cos_sin"], d["positions"], d["slots"], q_pe=q, q_out=q_out)
        assert r._append_io.q_out_nan == (q_out is None)


@pytest.mark.parametrize("parts,code", [
    (dict(append=dict(heads=4)), -8),
    (dict(absorb=dict(heads=4)), -8),
    (dict(attend=dict(heads=16, ql_token_stride=8192, qp_token_stride=1024, out_token_stride=8192)), -8),
    (dict(expand=dict(heads=9, x_token_stride=9 * 512, y_token_stride=9 * 128)), -8),
    (dict(expand=dict(x_f32=1)), -8),
    (dict(attend=dict(out_f32=1)), -8),
    (dict(append=dict(cache=dict(data=AT + 16))), -8),
    (dict(append=dict(cache=dict(pages=11))), -8),
    (dict(append=dict(cache=dict(page_size=8))), -8),
    (dict(attend=dict(cache=dict(fmt=2))), -8),
    (dict(append=dict(heads=0, tokens=0), absorb=dict(tokens=0), attend=dict(tokens=0), expand=dict(tokens=0)), 0),
    (dict(append=dict(tokens=0), absorb=dict(tokens=0), attend=dict(tokens=0, out_f32=1), expand=dict(tokens=0, x_f32=1)), 0),
])  # fmt: skip
def test_step_wants_parts_that_fit(lib, parts, code):
    """The same heads (append's may be none: no query), cache and type of the attended latents throughout:
    a part with more heads than the one before wrote would read past its buffer. (Those that fit: no tokens.)"""
    L, n = lib
    get = lambda k: {a: _cache(**b) if a == "cache" else b for a, b in parts.get(k, {}).items()}  # noqa: E731
    io = (_append(**get("append")), _project(0, **get("absorb")), _attend(**get("attend")), _project(1, **get("expand")))
    assert L.mkmoe_latent_step(*map(ctypes.byref, io), 0x200000, n, None) == code


def test_runner_rejects_options_that_fp32_does_not_hold():
    from sgl_amd_mono.moe.latent import LatentRunner

    for kw in (dict(scale=1e39), dict(scale=-1e300), dict(norm_eps=1e39)):
        with pytest.raises(RuntimeError, match="scale .* norm_eps"):
            LatentRunner(8, device="cuda", **kw)
