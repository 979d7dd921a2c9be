"""Host runner of a prompt's attention over the paged latent cache (``include/mkmoe.h``, a prompt's tokens).

The rows and the cache are those of ``latent``. Where a sequence brings one or a few tokens,
``latent.LatentRunner`` attends in the absorbed form, every head against the row itself. A prompt
brings hundreds: here each head's keys and values are made from the cached rows once a call, and the
attention over them takes 640 operations a score instead of 2176. ``LatentPromptRunner`` runs, each
on the current stream without a host synchronisation:

- ``append``, ``rows``: as ``LatentRunner``
- ``attend``: new tokens' attention over the cached rows, theirs among them
- ``attention``: a layer's whole step: the tokens' rows appended, their query rotated, then ``attend``

A batch that has both kinds of sequences is two calls, each with its sequences' rows of the table.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .latent import BF, NOPE, ROPE, ROW, LatentWeights, V, _LatentCalls


class LatentPromptRunner(_LatentCalls):
    """A prompt's attention of one rank's ``heads`` on one GPU: a workspace and the calls.

    ``max_tokens``: new tokens that ``attention`` takes at most. ``max_context``: cached tokens whose
    keys and values the workspace holds: those of a call's sequences with new tokens, each one's
    rounded up to 64 (135 MB, and a token 1152 bytes and 512 a head); where it is large for a call, and the call's
    table wide, the work is cut as for long sequences, and short ones take up to a fifth longer. ``scale``,
    ``norm_eps``, ``rope``: as ``LatentRunner``. One runner serves one stream at a time: calls that can overlap need
    runners of their own."""

    def __init__(self, heads: int, device=None, max_tokens: int = 8192, max_context: int = 32768,
                 scale: float | None = None, norm_eps: float = 1e-6, rope: str = "interleaved"):  # fmt: skip
        super().__init__(heads, device, scale, norm_eps, rope)
        if not 1 <= max_context <= _lib.LATENT_MAX_CONTEXT:
            raise RuntimeError(f"mkmoe latent: max_context {max_context}, want 1 .. {_lib.LATENT_MAX_CONTEXT}")
        if not 0 <= max_tokens <= _lib.LATENT_MAX_PROMPT:
            raise RuntimeError(f"mkmoe latent: max_tokens {max_tokens}, want 0 .. {_lib.LATENT_MAX_PROMPT}")
        self.max_tokens, self.max_context = int(max_tokens), int(max_context)
        n = ctypes.c_size_t()
        _lib.check(
            self.lib.mkmoe_latent_prompt_bytes(self.heads, self.max_context, ctypes.byref(n)), "prompt workspace size"
        )
        (self._q_pe,) = self._take_workspace(n.value, (BF, (self.max_tokens, self.heads, ROPE)))
        self._prompt_io = _lib.LatentPromptIO()

    def _set_prompt(self, cache, tokens: int, w, q_nope: tuple, q_pe: tuple, table, lens, q_starts, out: tuple,
                    lse: int) -> None:  # fmt: skip
        c = self._cache(cache)
        w.check(self.heads, self.device)
        if tokens > _lib.LATENT_MAX_PROMPT:
            raise RuntimeError(f"mkmoe latent: {tokens} query tokens, want at most {_lib.LATENT_MAX_PROMPT}")
        seqs, max_pages, stride, at_table, at_lens, at_starts = self._batch(tokens, table, lens, q_starts)
        _lib.LATENT_PROMPT.pack_into(
            self._prompt_io, 0, *c, seqs, tokens, self.heads, max_pages, self.max_context, 0, stride, q_nope[1], q_nope[2],
            q_pe[1], q_pe[2], out[1], out[2], q_nope[0], q_pe[0], w.kv_b.data_ptr(), at_table, at_lens, at_starts, out[0],
            lse, self.scale, 0,
        )  # fmt: skip

    def attend(
        self,
        w: LatentWeights,
        cache: torch.Tensor,
        q_nope: torch.Tensor,  # [T, heads, 128] bf16
        q_pe: torch.Tensor,  # [T, heads, 64] bf16, rotated
        table: torch.Tensor,  # [B, max_pages] int32
        lens: torch.Tensor,  # [B] int32: cached tokens, the queries' own among them
        q_starts: torch.Tensor | None = None,  # [B + 1] int32; None: T / B query tokens each
        out: torch.Tensor | None = None,
        lse: torch.Tensor | None = None,  # [T, heads] fp32: receives log sum exp
    ) -> torch.Tensor:
        """-> bf16 [T, heads, 128], before the output projection. A sequence's queries are its last
        tokens: of n, query i sees the first ``len - n + 1 + i`` tokens; one that sees none gives 0
        (``lse`` -inf). Rows of ``out`` that no sequence has by ``q_starts`` stay as they were, 0 without
        ``out``; ``out`` overlaps no input. Pages outside the cache and lengths or starts outside
        their bounds are recorded (``raise_on_device_error``), and so is a sequence whose cached tokens
        ``max_context`` does not hold, in the order of the batch: its queries give NaN."""
        if q_nope is None or q_nope.dim() != 3:
            raise self._bad("q_nope", q_nope, f"[tokens, {self.heads}, {NOPE}] {BF}")
        tokens = q_nope.shape[0]
        qn = self._rows3("q_nope", q_nope, tokens, NOPE)
        qp = self._rows3("q_pe", q_pe, tokens, ROPE)
        if out is None:
            out = self._new("the attended rows", tokens, self.heads, V, zeros=q_starts is not None)
        y = self._rows3("out", out, tokens, V, written=True)
        self._set_prompt(cache, tokens, w, qn, qp, table, lens, q_starts, y, self._lse(lse, tokens))
        if tokens:
            self._call(self.lib.mkmoe_latent_prompt, self._prompt_io, *self._ws)
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
        """A layer's whole step of prompts -> bf16 [T, heads, 128] (before the output projection): the
        rows appended, then every query's attention over the cache with them. The arguments are
        those of ``append`` and ``attend``; ``lens`` counts the appended tokens. A token whose slot
        or position is outside its bounds is recorded and not stored, and its query is NaN."""
        if q is None or q.dim() != 3 or q.shape[0] > self.max_tokens:
            raise self._bad("q", q, f"[tokens <= {self.max_tokens}, {self.heads}, {NOPE + ROPE}] {BF}")
        tokens, h = q.shape[0], self.heads
        at, ts, hs = self._rows3("q", q, tokens, NOPE + ROPE)
        if out is None:
            out = self._new("the attention's output", tokens, h, V, zeros=q_starts is not None)
        y = self._rows3("out", out, tokens, V, written=True)
        if kv is None or kv.shape[0] != tokens:
            raise self._bad("kv", kv, f"[{tokens}, {ROW}] {BF}")
        q_pe = self._q_pe.data_ptr(), h * ROPE, ROPE
        self._set_append(cache, kv, w.norm, cos_sin, positions, slots, h, (at + 2 * NOPE, ts, hs), q_pe, 1)
        self._set_prompt(cache, tokens, w, (at, ts, hs), q_pe, table, lens, q_starts, y, 0)
        if tokens:
            self._call(self.lib.mkmoe_latent_prompt_step, self._append_io, self._prompt_io, *self._ws)
        return out
