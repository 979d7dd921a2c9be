"""Host runner of the latent attention that precedes the MoE block in a DeepSeek-V3 decode layer.

A token's keys and values are one shared row of a paged cache: 512 latent values (RMS-normed)
and 64 rotated rope values. ``LatentRunner`` holds one rank's heads and runs, each on the current
stream without a host synchronisation (``include/mkmoe.h``, latent attention):

- ``append``: norm, rotate and store a step's rows; rotate the query's rope part
- ``rows``: the values that cache rows stand for
- ``absorb`` / ``expand``: every head's query through W_UK, its result through W_UV
- ``attend``: the absorbed attention over the cached rows
- ``attention``: a layer's whole step, the four in turn

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
        for name, shape in (("norm", (LATENT,)), ("kv_b", (heads * (NOPE + V), LATENT))):
            t = getattr(self, name)
            if t is None:
                raise RuntimeError(f"latent {name}: missing, want {shape} {BF}")
            dev_ok = t.is_cuda and (device is None or t.device == torch.device(device))
            if not (tuple(t.shape) == shape and t.dtype == BF and t.is_contiguous() and dev_ok):
                raise RuntimeError(
                    f"latent {name}: {tuple(t.shape)} {t.dtype} {t.device} contiguous={t.is_contiguous()}, "
                    f"want {shape} {BF} contiguous on the GPU"
                )


class LatentRunner:
    """Latent attention of one rank's ``heads`` on one GPU: a workspace and the calls.

    ``max_tokens``: query tokens that ``attention`` takes at most (its intermediates' size; the
    other calls have no such bound). ``scale``: of the scores (default 192^-0.5). ``rope``:
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
        if not math.isfinite(self.scale) or not (math.isfinite(self.norm_eps) and self.norm_eps >= 0):
            raise RuntimeError(f"mkmoe latent: scale {self.scale}, norm_eps {self.norm_eps}")
        self.rope = ROPES[rope]
        self.lib = _lib.lib()
        n = ctypes.c_size_t()
        _lib.check(self.lib.mkmoe_latent_workspace_bytes(ctypes.byref(n)), "latent workspace size")
        self.device = torch.device("cuda", torch.cuda.current_device() if dev.index is None else dev.index)
        no_capture("the latent workspace")
        with torch.cuda.device(self.device):
            self.ws = torch.zeros(n.value, dtype=torch.uint8, device=self.device)
            mk = lambda w: torch.empty(self.max_tokens, self.heads, w, dtype=BF, device=self.device)  # noqa: E731
            self._q_lat, self._q_pe, self._o_lat = mk(LATENT), mk(ROPE), mk(LATENT)
            torch.cuda.current_stream().synchronize()  # whichever stream comes first finds it zeroed

    # ---- argument checks
    def _bad(self, name: str, t, want: str):
        got = "missing" if t is None else f"{tuple(t.shape)} {t.dtype} {t.device} strides {t.stride()}"
        return RuntimeError(f"mkmoe latent {name}: {got}, want {want} on {self.device}")

    def _rows3(self, name: str, t, tokens: int, width: int, written: bool = False) -> tuple:
        """(pointer, token stride, head stride) of a bf16 [tokens, heads, width] tensor whose last
        axis is contiguous and whose rows start on 16 bytes."""
        h = self.heads
        if t is not None and t.dtype == BF and t.device == self.device and t.shape == (tokens, h, width):
            ts, hs, last = t.stride()
            ts, hs = ts if tokens > 1 else 0, hs if h > 1 else 0
            ok = last == 1 and ts % 8 == 0 and hs % 8 == 0 and t.data_ptr() % 16 == 0
            if ok and written:  # no two rows of an output share a place
                a, b = (ts, tokens), (hs, h)
                (s0, n0), (s1, n1) = (a, b) if ts >= hs else (b, a)
                ok = (n1 == 1 or s1 >= width) and (n0 == 1 or s0 >= (n1 - 1) * s1 + width)
            if ok:
                return t.data_ptr(), ts, hs
        raise self._bad(name, t, f"[{tokens}, {h}, {width}] {BF}, rows of whole 16-byte pieces")

    def _vec(self, name: str, t, n: int, dtypes: tuple) -> int:
        if t is None or t.device != self.device or t.dtype not in dtypes or t.shape != (n,) or not t.is_contiguous():
            raise self._bad(name, t, f"[{n}] {dtypes[0]} contiguous")
        return t.data_ptr()

    def _cache(self, t) -> _lib.LatentCache:
        if t is not None and t.dim() == 3 and t.device == self.device and t.is_contiguous():
            pages, page, row = t.shape
            if (t.dtype, row) == (BF, ROW):
                return _lib.LatentCache(t.data_ptr(), pages, page, _lib.LATENT_BF16)
            if (t.dtype, row) == (torch.uint8, MX_ROW):
                return _lib.LatentCache(t.data_ptr(), pages, page, _lib.LATENT_MXFP8)
        raise self._bad("cache", t, f"[pages, page_size, {ROW}] {BF} or [pages, page_size, {MX_ROW}] torch.uint8 contiguous")

    def _new(self, what: str, *shape) -> torch.Tensor:
        no_capture(what)
        return torch.empty(*shape, dtype=BF, device=self.device)

    def _call(self, fn, *args) -> None:
        """``fn`` on the current stream of this runner's GPU."""
        if torch.cuda.current_device() != self.device.index:
            with torch.cuda.device(self.device):
                rc = fn(*args, torch.cuda.current_stream().cuda_stream)
        else:
            rc = fn(*args, torch.cuda.current_stream().cuda_stream)
        if rc:
            _lib.check(rc, fn.__name__)

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
        ``q_pe`` itself). A token with a negative slot is not stored. A slot outside the cache or
        a position outside ``cos_sin`` leaves the token unwritten and is recorded
        (``raise_on_device_error``)."""
        c = self._cache(cache)
        if kv is None or kv.dim() != 2 or kv.shape[1] != ROW or kv.dtype != BF or kv.device != self.device:
            raise self._bad("kv", kv, f"[tokens, {ROW}] {BF}")
        tokens = kv.shape[0]
        stride = kv.stride(0) if tokens > 1 else ROW
        if kv.stride(1) != 1 or stride % 8 or stride < ROW or kv.data_ptr() % 16:
            raise self._bad("kv", kv, f"[tokens, {ROW}] {BF}, rows of whole 16-byte pieces")
        if norm is not None:
            self._vec("norm", norm, LATENT, (BF,))
        if (cos_sin is None or cos_sin.dim() != 2 or cos_sin.shape[1] != ROPE or cos_sin.dtype != torch.float32
                or cos_sin.device != self.device or not cos_sin.is_contiguous()):  # fmt: skip
            raise self._bad("cos_sin", cos_sin, f"[positions, {ROPE}] torch.float32 contiguous")
        pos = self._vec("positions", positions, tokens, (torch.int64, torch.int32))
        slot = self._vec("slots", slots, tokens, (positions.dtype,))
        qp = qts = qhs = op = ots = ohs = 0
        if q_pe is not None:
            qp, qts, qhs = self._rows3("q_pe", q_pe, tokens, ROPE)
            if q_out is None:
                q_out = self._new("the rotated query", tokens, self.heads, ROPE)
            op, ots, ohs = self._rows3("q_out", q_out, tokens, ROPE, written=True)
        elif q_out is not None:
            raise RuntimeError("mkmoe latent q_out: given without q_pe")
        io = _lib.LatentAppendIO(
            c, tokens, self.heads if q_pe is not None else 0, self.rope, 8 if positions.dtype == torch.int64 else 4,
            cos_sin.shape[0], stride, qts, qhs, ots, ohs, kv.data_ptr(), None if norm is None else norm.data_ptr(),
            cos_sin.data_ptr(), pos, slot, qp or None, op or None, self.norm_eps, 0,
        )  # fmt: skip
        if tokens:
            self._call(self.lib.mkmoe_latent_append, ctypes.byref(io), self.ws.data_ptr(), self.ws.numel())
        return q_out

    def rows(self, cache: torch.Tensor, slots: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """-> bf16 [T, 576]: the values that the cache rows ``slots`` stand for (a negative slot's
        are 0), exactly."""
        c = self._cache(cache)
        tokens = slots.shape[0]
        at = self._vec("slots", slots, tokens, (torch.int64, torch.int32))
        if out is None:
            out = self._new("the rows", tokens, ROW)
        if out.shape != (tokens, ROW) or out.dtype != BF or out.device != self.device or not out.is_contiguous():
            raise self._bad("out", out, f"[{tokens}, {ROW}] {BF} contiguous")
        if tokens:
            self._call(
                self.lib.mkmoe_latent_rows, ctypes.byref(c), at, 8 if slots.dtype == torch.int64 else 4, tokens,
                out.data_ptr(), self.ws.data_ptr(), self.ws.numel(),
            )  # fmt: skip
        return out

    def _project(self, what: str, w, x, out, expand: int) -> torch.Tensor:
        w.check(self.heads, self.device)
        width, wide = (LATENT, V) if expand else (NOPE, LATENT)
        if x is None or x.dim() != 3:
            raise self._bad(what, x, f"[tokens, {self.heads}, {width}] {BF}")
        tokens = x.shape[0]
        xp, xts, xhs = self._rows3(what, x, tokens, width)
        if out is None:
            out = self._new("an output", tokens, self.heads, wide)
        yp, yts, yhs = self._rows3("out", out, tokens, wide, written=True)
        io = _lib.LatentProjectIO(tokens, self.heads, expand, 0, xts, xhs, yts, yhs, xp, w.kv_b.data_ptr(), yp)
        if tokens:
            self._call(self.lib.mkmoe_latent_project, ctypes.byref(io))
        return out

    def absorb(self, w: LatentWeights, q_nope: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """q_nope [T, heads, 128] -> the absorbed query [T, heads, 512]: each head's through W_UK."""
        return self._project("q_nope", w, q_nope, out, 0)

    def expand(self, w: LatentWeights, o_lat: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """The attended latents [T, heads, 512] -> [T, heads, 128]: each head's through W_UV."""
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
        """-> bf16 [T, heads, 512]. A sequence's queries are its last tokens: of n, query i sees the
        first ``len - n + 1 + i`` tokens; one that sees none gives 0 (``lse`` -inf). Rows of ``out``
        behind the last sequence's queries stay as they were. Pages outside the cache and lengths
        or starts outside their bounds are recorded (``raise_on_device_error``)."""
        c = self._cache(cache)
        if q_lat is None or q_lat.dim() != 3:
            raise self._bad("q_lat", q_lat, f"[tokens, {self.heads}, {LATENT}] {BF}")
        tokens = q_lat.shape[0]
        ql, ql_ts, ql_hs = self._rows3("q_lat", q_lat, tokens, LATENT)
        qp, qp_ts, qp_hs = self._rows3("q_pe", q_pe, tokens, ROPE)
        i32 = torch.int32
        if (table is None or table.dim() != 2 or table.dtype != i32 or table.device != self.device
                or table.stride(1) != 1 and table.shape[1] > 1):  # fmt: skip
            raise self._bad("table", table, "[seqs, max_pages] torch.int32")
        seqs, max_pages = table.shape
        t_stride = table.stride(0) if seqs > 1 else max_pages
        at_lens = self._vec("lens", lens, seqs, (i32,))
        at_starts = None if q_starts is None else self._vec("q_starts", q_starts, seqs + 1, (i32,))
        if not 1 <= seqs <= _lib.LATENT_MAX_SEQS or (q_starts is None and tokens % seqs):
            raise RuntimeError(
                f"mkmoe latent: {seqs} sequences of {tokens} query tokens, want 1 .. {_lib.LATENT_MAX_SEQS} sequences "
                "and, without q_starts, as many tokens in each"
            )
        if out is None:
            out = self._new("the attended rows", tokens, self.heads, LATENT)
        op, o_ts, o_hs = self._rows3("out", out, tokens, LATENT, written=True)
        at_lse = None
        if lse is not None:
            if (lse.dtype != torch.float32 or lse.shape != (tokens, self.heads) or lse.device != self.device
                    or not lse.is_contiguous()):  # fmt: skip
                raise self._bad("lse", lse, f"[{tokens}, {self.heads}] torch.float32 contiguous")
            at_lse = lse.data_ptr()
        io = _lib.LatentAttendIO(
            c, seqs, tokens, self.heads, max_pages, t_stride, ql_ts, ql_hs, qp_ts, qp_hs, o_ts, o_hs, ql, qp,
            table.data_ptr(), at_lens, at_starts, op, at_lse, self.scale, 0,
        )  # fmt: skip
        if tokens:
            self._call(self.lib.mkmoe_latent_attend, ctypes.byref(io), self.ws.data_ptr(), self.ws.numel())
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
        of ``append`` and ``attend``; ``lens`` counts the appended tokens."""
        if q is None or q.dim() != 3 or q.shape[0] > self.max_tokens:
            raise self._bad("q", q, f"[tokens <= {self.max_tokens}, {self.heads}, {NOPE + ROPE}] {BF}")
        tokens = q.shape[0]
        self._rows3("q", q, tokens, NOPE + ROPE)
        w.check(self.heads, self.device)
        if out is None:
            out = self._new("the attention's output", tokens, self.heads, V)
        self._rows3("out", out, tokens, V, written=True)
        q_lat, q_pe, o_lat = self._q_lat[:tokens], self._q_pe[:tokens], self._o_lat[:tokens]
        self.append(cache, kv, w.norm, cos_sin, positions, slots, q_pe=q[..., NOPE:], q_out=q_pe)
        self.absorb(w, q[..., :NOPE], out=q_lat)
        self.attend(cache, q_lat, q_pe, table, lens, q_starts=q_starts, out=o_lat)
        return self.expand(w, o_lat, out=out)

    # ---- device errors
    def read_errors(self) -> list[int]:
        """The device error words (synchronises the stream)."""
        words = (ctypes.c_int32 * _lib.LATENT_ERRW_WORDS)()
        self._call(self.lib.mkmoe_latent_read_errors, self.ws.data_ptr(), words, _lib.LATENT_ERRW_WORDS)
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
