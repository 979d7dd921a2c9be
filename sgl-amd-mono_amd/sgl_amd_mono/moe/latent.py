"""Host runner of the latent attention that precedes the MoE block in a DeepSeek-V3 decode layer.

A token's keys and values are one shared row of a paged cache: 512 latent values (RMS-normed)
and 64 rotated rope values. ``LatentRunner`` holds one rank's heads and runs, each on the current
stream without a host synchronisation (``include/mkmoe.h``, latent attention):

- ``append``: norm, rotate and store a step's rows; rotate the query's rope part
- ``rows``: the values that cache rows stand for
- ``absorb`` / ``expand``: every head's query through W_UK, its result through W_UV
- ``attend``: the absorbed attention over the cached rows
- ``attention``: a layer's whole step in one call: the first two in one launch, then the others

Caches (``cache_like``): bf16 [pages, page_size, 576], or MXFP8 as uint8 [pages, page_size, 656]
(512 e4m3 codes, 16 E8M0 scales, one per 32 latent values, and the 64 rope values in bf16). The
reference's own attention is another one (``deepseek_v41/gfx950/attention``); the host side follows
its runner's manner (``deepseek_v41/gfx950/runner.py:94-127``): checks that name the tensor, outputs
that the caller may provide, nothing allocated inside a graph capture.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass

import torch

from . import _lib
from .runner import no_capture

LATENT, ROPE, NOPE, V = _lib.LATENT_DIM, _lib.LATENT_ROPE, _lib.LATENT_NOPE, _lib.LATENT_V
ROW, MX_ROW = LATENT + ROPE, _lib.LATENT_MX_ROW
ROPES = {"interleaved": 0, "half": 1}
BF = torch.bfloat16


def cache_like(pages: int, page_size: int, fmt: str = "bf16", device="cuda") -> torch.Tensor:
    """An empty (zeroed) cache of ``pages`` pages, "bf16" or "mxfp8"."""
    if fmt not in ("bf16", "mxfp8"):
        raise ValueError(f"latent cache format {fmt!r}: bf16 or mxfp8")
    if fmt == "bf16":
        return torch.zeros(pages, page_size, ROW, dtype=BF, device=device)
    return torch.zeros(pages, page_size, MX_ROW, dtype=torch.uint8, device=device)


@dataclass
class LatentWeights:
    """One layer's tensors on this rank: ``norm`` bf16 [512] (kv_a_layernorm) and ``kv_b`` bf16
    [heads * 256, 512] (kv_b_proj: per head 128 rows of W_UK, then 128 rows of W_UV), in place."""

    norm: torch.Tensor
    kv_b: torch.Tensor

    def check(self, heads: int, device=None) -> None:
        """Raise unless each tensor has its shape and dtype and is contiguous on one GPU."""
        at = None if device is None else torch.device(device)
        for name, t, shape in (("norm", self.norm, (LATENT,)), ("kv_b", self.kv_b, (heads * (NOPE + V), LATENT))):
            if t is None:
                raise RuntimeError(f"latent {name}: missing, want {shape} {BF}")
            dev_ok = t.is_cuda and (at is None or t.device == at)
            if not (t.shape == shape and t.dtype == BF and t.is_contiguous() and dev_ok):
                raise RuntimeError(
                    f"latent {name}: {tuple(t.shape)} {t.dtype} {t.device} contiguous={t.is_contiguous()}, "
                    f"want {shape} {BF} contiguous on the GPU"
                )


class LatentRunner:
    """Latent attention of one rank's ``heads`` on one GPU: a workspace and the calls.

    ``max_tokens``: query tokens that ``attention`` takes at most (its intermediates' size; the
    other calls have no such bound). ``scale``: of the scores (default 192^-0.5; a model whose rope
    is scaled has another: DeepSeek-V3's is that times (0.1 ln 40 + 1)^2 = 1.874). ``rope``:
    "interleaved" (pairs (2 i, 2 i + 1)) or "half" ((i, i + 32)). One runner serves one stream at
    a time: calls that can overlap need runners of their own."""

    def __init__(self, heads: int, device=None, max_tokens: int = 48, scale: float | None = None,
                 norm_eps: float = 1e-6, rope: str = "interleaved"):  # fmt: skip
        if not 1 <= heads <= _lib.LATENT_MAX_HEADS:
            raise RuntimeError(f"mkmoe latent: {heads} heads, want 1 .. {_lib.LATENT_MAX_HEADS}")
        if rope not in ROPES:
            raise ValueError(f"mkmoe latent: rope {rope!r}, one of {tuple(ROPES)}")
        dev = torch.device("cuda") if device is None else torch.device(device)
        if dev.type != "cuda":
            raise RuntimeError(f"mkmoe latent: {dev} is not a GPU")
        self.heads = int(heads)
        self.max_tokens = int(max_tokens)
        self.scale = (NOPE + ROPE) ** -0.5 if scale is None else float(scale)
        self.norm_eps = float(norm_eps)
        f32 = lambda v: ctypes.c_float(v).value  # noqa: E731  (what the library is given)
        if not math.isfinite(f32(self.scale)) or not (math.isfinite(f32(self.norm_eps)) and self.norm_eps >= 0):
            raise RuntimeError(f"mkmoe latent: scale {self.scale}, norm_eps {self.norm_eps}")
        self.rope = ROPES[rope]
        self.lib = _lib.lib()
        n = ctypes.c_size_t()
        _lib.check(self.lib.mkmoe_latent_workspace_bytes(ctypes.byref(n)), "latent workspace size")
        self.device = torch.device("cuda", torch.cuda.current_device() if dev.index is None else dev.index)
        no_capture("the latent workspace")
        with torch.cuda.device(self.device):
            self.ws = torch.empty(n.value, dtype=torch.uint8, device=self.device)
            self.clear_errors()
            mk = lambda w, t: torch.empty(self.max_tokens, self.heads, w, dtype=t, device=self.device)  # noqa: E731
            # (the attended latents stay in fp32: one rounding less before the output's own)
            self._q_lat, self._q_pe, self._o_lat = mk(LATENT, BF), mk(ROPE, BF), mk(LATENT, torch.float32)
            torch.cuda.current_stream().synchronize()  # whichever stream comes first finds them cleared
        self._index = self.device.index
        self._append_io, self._attend_io = _lib.LatentAppendIO(), _lib.LatentAttendIO()
        self._absorb_io, self._expand_io = _lib.LatentProjectIO(), _lib.LatentProjectIO()
        self._ws = (self.ws.data_ptr(), self.ws.numel())

    # ---- argument checks
    def _bad(self, name: str, t, want: str):
        got = "missing" if t is None else f"{tuple(t.shape)} {t.dtype} {t.device} strides {t.stride()}"
        return RuntimeError(f"mkmoe latent {name}: {got}, want {want} on {self.device}")

    def _rows3(self, name: str, t, tokens: int, width: int, written: bool = False, dtype=BF) -> tuple:
        """(pointer, token stride, head stride) of a [tokens, heads, width] tensor whose last axis is
        contiguous and whose rows start on 16 bytes."""
        h = self.heads
        if t is not None and t.dtype is dtype and t.get_device() == self._index and t.shape == (tokens, h, width):
            ts, hs, last = t.stride()
            at = t.data_ptr()
            if tokens <= 1:
                ts = 0
            if h <= 1:
                hs = 0
            if last == 1 and not (ts | hs) & 7 and not at & 15:
                if not written:
                    return at, ts, hs
                # no two rows of an output share a place
                s0, n0, s1, n1 = (ts, tokens, hs, h) if ts >= hs else (hs, h, ts, tokens)
                if (n1 <= 1 or s1 >= width) and (n0 <= 1 or s0 >= (n1 - 1) * s1 + width):
                    return at, ts, hs
        raise self._bad(name, t, f"[{tokens}, {h}, {width}] {dtype}, rows of whole 16-byte pieces")

    def _vec(self, name: str, t, n: int, dtype) -> int:
        if t is not None and t.dtype is dtype and t.get_device() == self._index and t.shape == (n,) and t.is_contiguous():
            return t.data_ptr()
        raise self._bad(name, t, f"[{n}] {dtype} contiguous")

    def _index_type(self, name: str, t):
        """int32 where ``t`` is, else int64 (which the check then asks for)."""
        if t is None:
            raise self._bad(name, t, "torch.int64 or torch.int32")
        return torch.int32 if t.dtype is torch.int32 else torch.int64

    def _cache(self, t) -> tuple:
        shape = () if t is None else t.shape
        if len(shape) == 3 and t.get_device() == self._index and t.is_contiguous():
            pages, page, row = shape
            if row == ROW and t.dtype is BF:
                return t.data_ptr(), pages, page, _lib.LATENT_BF16
            if row == MX_ROW and t.dtype is torch.uint8:
                return t.data_ptr(), pages, page, _lib.LATENT_MXFP8
        raise self._bad("cache", t, f"[pages, page_size, {ROW}] {BF} or [pages, page_size, {MX_ROW}] torch.uint8 contiguous")

    def _new(self, what: str, *shape, zeros: bool = False) -> torch.Tensor:
        """An output of the call's own. ``zeros``: the call may leave rows of it unwritten."""
        no_capture(what)
        return (torch.zeros if zeros else torch.empty)(*shape, dtype=BF, device=self.device)

    def _call(self, fn, *args) -> None:
        """``fn`` on the current stream of this runner's GPU."""
        stream = torch._C._cuda_getCurrentRawStream(self._index)  # (current_stream()'s, without its object)
        if torch._C._cuda_getDevice() != self._index:
            with torch.cuda.device(self.device):
                rc = fn(*args, stream)
        else:
            rc = fn(*args, stream)
        if rc:
            _lib.check(rc, fn.__name__)

    # ---- the calls' arguments, checked and written into their structures
    def _set_append(self, cache, kv, norm, cos_sin, positions, slots, heads: int, q: tuple, q_out: tuple,
                    nan: int = 0) -> int:  # fmt: skip
        c = self._cache(cache)
        shape = () if kv is None else kv.shape
        if len(shape) != 2 or shape[1] != ROW or kv.dtype is not BF or kv.get_device() != self._index:
            raise self._bad("kv", kv, f"[tokens, {ROW}] {BF}")
        tokens, at = shape[0], kv.data_ptr()
        stride, last = kv.stride()
        if tokens <= 1:
            stride = ROW
        if last != 1 or stride & 7 or stride < ROW or at & 15:
            raise self._bad("kv", kv, f"[tokens, {ROW}] {BF}, rows of whole 16-byte pieces")
        w = 0 if norm is None else self._vec("norm", norm, LATENT, BF)
        turns = () if cos_sin is None else cos_sin.shape
        if (len(turns) != 2 or turns[1] != ROPE or cos_sin.dtype is not torch.float32
                or cos_sin.get_device() != self._index or not cos_sin.is_contiguous()):  # fmt: skip
            raise self._bad("cos_sin", cos_sin, f"[positions, {ROPE}] torch.float32 contiguous")
        index = self._index_type("positions", positions)
        pos = self._vec("positions", positions, tokens, index)
        slot = self._vec("slots", slots, tokens, index)
        _lib.LATENT_APPEND.pack_into(
            self._append_io, 0, *c, tokens, heads, self.rope, 8 if index is torch.int64 else 4, turns[0], stride,
            q[1], q[2], q_out[1], q_out[2], at, w, cos_sin.data_ptr(), pos, slot, q[0], q_out[0], self.norm_eps, nan,
        )  # fmt: skip
        return tokens

    def _set_attend(self, cache, tokens: int, q_lat: tuple, q_pe: tuple, table, lens, q_starts, out: tuple,
                    f32: int, lse: int) -> None:  # fmt: skip
        c = self._cache(cache)
        shape = () if table is None else table.shape
        if len(shape) != 2 or table.dtype is not torch.int32 or table.get_device() != self._index:
            raise self._bad("table", table, "[seqs, max_pages] torch.int32")
        (seqs, max_pages), (stride, last) = shape, table.stride()
        if last != 1 and max_pages > 1:
            raise self._bad("table", table, "[seqs, max_pages] torch.int32, the pages of a sequence contiguous")
        if seqs <= 1:
            stride = max_pages
        at_lens = self._vec("lens", lens, seqs, torch.int32)
        at_starts = 0 if q_starts is None else self._vec("q_starts", q_starts, seqs + 1, torch.int32)
        if not 1 <= seqs <= _lib.LATENT_MAX_SEQS or (q_starts is None and tokens % seqs):
            raise RuntimeError(
                f"mkmoe latent: {seqs} sequences of {tokens} query tokens, want 1 .. {_lib.LATENT_MAX_SEQS} sequences "
                "and, without q_starts, as many tokens in each"
            )
        _lib.LATENT_ATTEND.pack_into(
            self._attend_io, 0, *c, seqs, tokens, self.heads, max_pages, stride, q_lat[1], q_lat[2], q_pe[1], q_pe[2],
            out[1], out[2], q_lat[0], q_pe[0], table.data_ptr(), at_lens, at_starts, out[0], lse, self.scale, f32,
        )  # fmt: skip

    def _set_project(self, io, tokens: int, expand: int, f32: int, x: tuple, w: int, y: tuple) -> None:
        _lib.LATENT_PROJECT.pack_into(io, 0, tokens, self.heads, expand, f32, x[1], x[2], y[1], y[2], x[0], w, y[0])

    # ---- the calls
    def append(
        self,
        cache: torch.Tensor,
        kv: torch.Tensor,  # [T, 576] bf16: latent, rope part before the rotation
        norm: torch.Tensor | None,  # [512] bf16; None: the latent is stored as it is
        cos_sin: torch.Tensor,  # [positions, 64] fp32: 32 cosines, 32 sines
        positions: torch.Tensor,  # [T] int64 or int32
        slots: torch.Tensor,  # [T], as positions: cache rows (page * page_size + offset), distinct
        q_pe: torch.Tensor | None = None,  # [T, heads, 64] bf16
        q_out: torch.Tensor | None = None,
    ) -> torch.Tensor | None:
        """Store the step's rows; -> the query's rope part, rotated (``q_out``, which may be
        ``q_pe`` itself). A token with a negative slot is a padded one and not stored (where its position
        is outside ``cos_sin``, its query is 0). A slot outside the cache or
        a position outside ``cos_sin`` leaves the token unwritten (NaN in a query of the call's own)
        and is recorded (``raise_on_device_error``)."""
        qp = op = (0, 0, 0)
        own = q_out is None
        if q_pe is not None:
            if kv is None:
                raise self._bad("kv", kv, f"[tokens, {ROW}] {BF}")
            tokens = kv.shape[0]
            qp = self._rows3("q_pe", q_pe, tokens, ROPE)
            if q_out is None:
                q_out = self._new("the rotated query", tokens, self.heads, ROPE)
            op = self._rows3("q_out", q_out, tokens, ROPE, written=True)
        elif q_out is not None:
            raise RuntimeError("mkmoe latent q_out: given without q_pe")
        heads = 0 if q_pe is None else self.heads
        if self._set_append(cache, kv, norm, cos_sin, positions, slots, heads, qp, op, int(own)):
            self._call(self.lib.mkmoe_latent_append, self._append_io, *self._ws)
        return q_out

    def rows(self, cache: torch.Tensor, slots: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """-> bf16 [T, 576]: the values that the cache rows ``slots`` stand for (a negative slot's
        are 0), exactly."""
        c = _lib.LatentCache(*self._cache(cache))
        index = self._index_type("slots", slots)
        tokens = slots.numel()
        at = self._vec("slots", slots, tokens, index)
        if out is None:
            out = self._new("the rows", tokens, ROW)
        elif out.shape != (tokens, ROW) or out.dtype is not BF or out.get_device() != self._index or not out.is_contiguous():
            raise self._bad("out", out, f"[{tokens}, {ROW}] {BF} contiguous")
        if tokens:
            self._call(
                self.lib.mkmoe_latent_rows, c, at, 8 if index is torch.int64 else 4, tokens, out.data_ptr(), *self._ws
            )
        return out

    def _project(self, what: str, w, x, out, expand: int) -> torch.Tensor:
        w.check(self.heads, self.device)
        width, wide = (LATENT, V) if expand else (NOPE, LATENT)
        if x is None or x.dim() != 3:
            raise self._bad(what, x, f"[tokens, {self.heads}, {width}] {BF}")
        tokens = x.shape[0]
        f32 = expand and x.dtype == torch.float32
        x = self._rows3(what, x, tokens, width, dtype=torch.float32 if f32 else BF)
        if out is None:
            out = self._new("an output", tokens, self.heads, wide)
        io = self._expand_io if expand else self._absorb_io
        y = self._rows3("out", out, tokens, wide, written=True)
        self._set_project(io, tokens, expand, int(f32), x, w.kv_b.data_ptr(), y)
        if tokens:
            self._call(self.lib.mkmoe_latent_project, io)
        return out

    def absorb(self, w: LatentWeights, q_nope: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """q_nope [T, heads, 128] -> the absorbed query [T, heads, 512]: each head's through W_UK."""
        return self._project("q_nope", w, q_nope, out, 0)

    def expand(self, w: LatentWeights, o_lat: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """The attended latents [T, heads, 512], bf16 or fp32 -> bf16 [T, heads, 128]: each head's through W_UV."""
        return self._project("o_lat", w, o_lat, out, 1)

    def attend(
        self,
        cache: torch.Tensor,
        q_lat: torch.Tensor,  # [T, heads, 512] bf16
        q_pe: torch.Tensor,  # [T, heads, 64] bf16, rotated
        table: torch.Tensor,  # [B, max_pages] int32
        lens: torch.Tensor,  # [B] int32: cached tokens, the queries' own among them
        q_starts: torch.Tensor | None = None,  # [B + 1] int32; None: T / B query tokens each
        out: torch.Tensor | None = None,
        lse: torch.Tensor | None = None,  # [T, heads] fp32: receives log sum exp
    ) -> torch.Tensor:
        """-> [T, heads, 512], bf16 or, where ``out`` is, fp32. A sequence's queries are its last tokens:
        of n, query i sees the first ``len - n + 1 + i`` tokens; one that sees none gives 0 (``lse``
        -inf). Rows of ``out`` that no sequence has by ``q_starts`` (before the first one's queries, behind
        the last one's, all of them where the starts run backwards) stay as they were, 0 without ``out``;
        ``out`` overlaps no input. Pages outside the cache and lengths or starts outside their bounds are recorded
        (``raise_on_device_error``)."""
        if q_lat is None or q_lat.dim() != 3:
            raise self._bad("q_lat", q_lat, f"[tokens, {self.heads}, {LATENT}] {BF}")
        tokens = q_lat.shape[0]
        ql = self._rows3("q_lat", q_lat, tokens, LATENT)
        qp = self._rows3("q_pe", q_pe, tokens, ROPE)
        if out is None:
            out = self._new("the attended rows", tokens, self.heads, LATENT, zeros=q_starts is not None)
        f32 = out.dtype == torch.float32
        op = self._rows3("out", out, tokens, LATENT, written=True, dtype=torch.float32 if f32 else BF)
        at_lse = 0
        if lse is not None:
            if (lse.dtype != torch.float32 or lse.shape != (tokens, self.heads) or lse.device != self.device
                    or not lse.is_contiguous()):  # fmt: skip
                raise self._bad("lse", lse, f"[{tokens}, {self.heads}] torch.float32 contiguous")
            at_lse = lse.data_ptr()
        self._set_attend(cache, tokens, ql, qp, table, lens, q_starts, op, int(f32), at_lse)
        if tokens:
            self._call(self.lib.mkmoe_latent_attend, self._attend_io, *self._ws)
        return out

    def attention(
        self,
        w: LatentWeights,
        cache: torch.Tensor,
        q: torch.Tensor,  # [T, heads, 192] bf16: 128 values without rotation, 64 to rotate
        kv: torch.Tensor,  # [T, 576] bf16
        cos_sin: torch.Tensor,
        positions: torch.Tensor,
        slots: torch.Tensor,
        table: torch.Tensor,
        lens: torch.Tensor,
        q_starts: torch.Tensor | None = None,
        out: torch.Tensor | None = None,
    ) -> torch.Tensor:
        """A layer's whole step -> bf16 [T, heads, 128] (before the output projection): the rows
        appended, then every query's attention over the cache with them. The arguments are those
        of ``append`` and ``attend``; ``lens`` counts the appended tokens. Rows of ``out`` that no
        sequence has stay as they were, as in ``attend``; a token whose slot or position is outside
        its bounds, which is recorded, gives NaN."""
        if q is None or q.dim() != 3 or q.shape[0] > self.max_tokens:
            raise self._bad("q", q, f"[tokens <= {self.max_tokens}, {self.heads}, {NOPE + ROPE}] {BF}")
        tokens, h = q.shape[0], self.heads
        at, ts, hs = self._rows3("q", q, tokens, NOPE + ROPE)
        w.check(h, self.device)
        if out is None:
            out = self._new("the attention's output", tokens, h, V, zeros=q_starts is not None)
        y = self._rows3("out", out, tokens, V, written=True)
        if kv is None or kv.shape[0] != tokens:
            raise self._bad("kv", kv, f"[{tokens}, {ROW}] {BF}")
        parts = (self._q_lat, LATENT), (self._q_pe, ROPE), (self._o_lat, LATENT)
        q_lat, q_pe, o_lat = ((t.data_ptr(), h * n, n) for t, n in parts)
        kv_b = w.kv_b.data_ptr()
        self._set_append(cache, kv, w.norm, cos_sin, positions, slots, h, (at + 2 * NOPE, ts, hs), q_pe)
        self._set_project(self._absorb_io, tokens, 0, 0, (at, ts, hs), kv_b, q_lat)
        self._set_attend(cache, tokens, q_lat, q_pe, table, lens, q_starts, o_lat, 1, 0)
        self._set_project(self._expand_io, tokens, 1, 1, o_lat, kv_b, y)
        if tokens:
            self._call(
                self.lib.mkmoe_latent_step, self._append_io, self._absorb_io, self._attend_io, self._expand_io,
                *self._ws,
            )  # fmt: skip
        return out

    # ---- device errors
    def read_errors(self) -> list[int]:
        """The device error words (synchronises the stream)."""
        words = (ctypes.c_int32 * _lib.LATENT_ERRW_WORDS)()
        self._call(self.lib.mkmoe_latent_read_errors, self._ws[0], words, _lib.LATENT_ERRW_WORDS)
        return list(words)

    def raise_on_device_error(self) -> None:
        """Raise if a call since the last ``clear_errors`` met a slot, position, length, query start
        or page outside its bounds (synchronises the stream)."""
        code, where, count, _ = self.read_errors()
        if code:
            raise RuntimeError(f"mkmoe latent: {_lib.LATENT_ERRORS.get(code, code)} {where} ({count} seen)")

    def clear_errors(self) -> None:
        """Forget recorded errors (on the current stream)."""
        self.ws[: 4 * _lib.LATENT_ERRW_WORDS].zero_()
