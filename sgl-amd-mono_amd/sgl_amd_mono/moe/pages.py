"""Pages of a paged cache: who holds them, where a step's tokens go, and their copies (``include/mkmoe.h``, pages
of a cache).

``LatentRunner`` and ``LatentPromptRunner`` attend by a table of pages and lengths that the caller keeps.
``PagePool`` keeps them, on the GPU and without a host synchronisation, for one or several caches
(a model's layers) that the same pages index:

- ``adopt``: the pool as a table says, or empty
- ``grow``: the next tokens' places: slots, positions and query starts as the runners take them
- ``trim``: sequences cut to a length: tokens of a draft that were not accepted, or all of them (freed)
- ``fork``: rows that go on from others, sharing their full pages: samples of a prompt, beams
- ``compact``: the pages held moved to the front of the pool
- ``copy``: pages' bytes to other pages

A page that is partly filled belongs to one sequence: its next token is written there. ``fork`` and
``trim`` copy it where it would be shared. Pages are taken lowest first, in the sequences' order, so
the same calls give the same tables. The reference's caches are SGLang's, with pages kept on the host; the
checks follow its runner's manner (``deepseek_v41/gfx950/runner.py:94-127``).
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .runner import no_capture

I32 = torch.int32


class PagePool:
    """A pool of ``pages`` pages of ``page_size`` tokens, all free at first.

    ``caches``: tensors whose first axis is the pages (``latent.cache_like``'s, a layer each), whose bytes
    ``fork``, ``trim``, ``compact`` and ``copy`` move; they are used in place and kept alive. ``max_seqs``,
    ``max_pages``: the largest table that a call takes ([B, max_pages], a sequence a row; by default sequences
    of 131072 tokens, or the pool's): the pool keeps a copy of so many entries (4 bytes each), and 16 bytes a
    page. One pool serves one stream at a time."""

    def __init__(self, pages: int, page_size: int, caches=(), max_seqs: int = 512, max_pages: int | None = None, device=None):
        if not 1 <= page_size <= 1024 or page_size & (page_size - 1):
            raise RuntimeError(f"mkmoe pages: page_size {page_size}, want a power of two, 1 .. 1024")
        if not 1 <= pages <= _lib.PAGES_MAX_PAGES or pages * page_size >= 1 << 31:
            raise RuntimeError(
                f"mkmoe pages: {pages} pages of {page_size}, want 1 .. {_lib.PAGES_MAX_PAGES} and below 2^31 tokens"
            )
        max_pages = min(pages, max(1, 131072 // page_size)) if max_pages is None else max_pages
        if not 1 <= max_pages <= _lib.PAGES_MAX_PAGES or max_pages * page_size >= 1 << 31:
            raise RuntimeError(
                f"mkmoe pages: max_pages {max_pages} of {page_size}, want 1 .. {_lib.PAGES_MAX_PAGES} and below 2^31 tokens"
            )
        if not 1 <= max_seqs <= _lib.PAGES_MAX_SEQS:
            raise RuntimeError(f"mkmoe pages: max_seqs {max_seqs}, want 1 .. {_lib.PAGES_MAX_SEQS}")
        caches = list(caches)
        dev = torch.device("cuda") if device is None else torch.device(device)
        if device is None and caches:
            dev = caches[0].device
        if dev.type != "cuda":
            raise RuntimeError(f"mkmoe pages: {dev} is not a GPU")
        self.pages, self.page_size, self.max_seqs, self.max_pages = int(pages), int(page_size), int(max_seqs), int(max_pages)
        self.lib = _lib.lib()
        n = ctypes.c_size_t()
        _lib.check(self.lib.mkmoe_pages_workspace_bytes(pages, max_seqs, max_pages, ctypes.byref(n)), "pages workspace size")
        self.device = torch.device("cuda", torch.cuda.current_device() if dev.index is None else dev.index)
        self._index = self.device.index
        places = []
        for i, c in enumerate(caches):
            size = c.numel() * c.element_size() // max(1, pages)
            if (c.device != self.device or c.dim() < 1 or c.shape[0] != pages or not c.is_contiguous() or size == 0
                    or size % 16 or c.data_ptr() % 16):  # fmt: skip
                raise RuntimeError(
                    f"mkmoe pages caches[{i}]: {tuple(c.shape)} {c.dtype} {c.device}, want [{pages}, ...] contiguous on "
                    f"{self.device}, pages of whole 16-byte pieces"
                )
            places.append((c.data_ptr(), size))
        spans = sorted((at, at + size * pages, i) for i, (at, size) in enumerate(places))
        for (_, end, i), (at, _, j) in zip(spans, spans[1:]):
            if at < end:
                raise RuntimeError(f"mkmoe pages: caches[{i}] and caches[{j}] share memory")
        no_capture("the page pool")
        self.caches = caches
        with torch.cuda.device(self.device):
            self.ws = torch.zeros(n.value, dtype=torch.uint8, device=self.device)
            self._places = torch.tensor(places, dtype=torch.int64).to(self.device) if places else None
        # how many sequences hold each page, int32 [pages]; read-only
        self.refs = self.ws[_lib.PAGES_REFS_AT : _lib.PAGES_REFS_AT + 4 * pages].view(I32)
        self._ws = (self.ws.data_ptr(), self.ws.numel())
        at = 0 if self._places is None else self._places.data_ptr()
        self._pool = _lib.PagesPool(self.pages, self.page_size, self.max_seqs, self.max_pages, len(caches), 0, at)
        self._table = _lib.PagesTable()
        self._call(self.lib.mkmoe_pages_adopt, self._pool, None)
        with torch.cuda.device(self.device):
            torch.cuda.current_stream().synchronize()  # whichever stream comes first finds it so

    # ---- argument checks
    def _bad(self, name: str, t, want: str):
        got = "missing" if t is None else f"{tuple(t.shape)} {t.dtype} {t.device} strides {t.stride()}"
        return RuntimeError(f"mkmoe pages {name}: {got}, want {want} on {self.device}")

    def _vec(self, name: str, t, n: int | None = None) -> int:
        if (t is not None and t.dtype is I32 and t.get_device() == self._index and t.dim() == 1
                and (n is None or t.shape[0] == n) and t.is_contiguous()):  # fmt: skip
            return t.data_ptr()
        raise self._bad(name, t, f"[{'n' if n is None else n}] {I32} contiguous")

    def _set_table(self, table, lens) -> int:
        """The table's structure filled; -> its sequences."""
        shape = () if table is None else table.shape
        if len(shape) != 2 or table.dtype is not I32 or table.get_device() != self._index:
            raise self._bad("table", table, f"[seqs, max_pages] {I32}")
        (seqs, max_pages), (stride, last) = shape, table.stride()
        if not 1 <= seqs <= self.max_seqs or not 1 <= max_pages <= self.max_pages:
            raise self._bad("table", table, f"[1 .. {self.max_seqs}, 1 .. {self.max_pages}] {I32}")
        if seqs == 1:
            stride = max_pages
        if (last != 1 and max_pages > 1) or stride < max_pages:
            raise self._bad("table", table, f"[seqs, max_pages] {I32}, the pages of a sequence contiguous, rows apart")
        _lib.PAGES_TABLE.pack_into(self._table, 0, table.data_ptr(), self._vec("lens", lens, seqs), stride, seqs, max_pages)
        return seqs

    def _call(self, fn, *args) -> None:
        """``fn`` on the current stream of this pool's GPU."""
        stream = torch._C._cuda_getCurrentRawStream(self._index)
        if torch._C._cuda_getDevice() != self._index:
            with torch.cuda.device(self.device):
                rc = fn(*args, *self._ws, stream)
        else:
            rc = fn(*args, *self._ws, stream)
        if rc:
            _lib.check(rc, fn.__name__)

    # ---- the calls
    def adopt(self, table: torch.Tensor | None = None, lens: torch.Tensor | None = None) -> None:
        """The pool as ``table`` [B, max_pages] and ``lens`` [B] (int32) say: every page held as often as
        the sequences name it. None: all free. What the pool held before is forgotten."""
        if table is None and lens is None:
            self._call(self.lib.mkmoe_pages_adopt, self._pool, None)
            return
        self._set_table(table, lens)
        self._call(self.lib.mkmoe_pages_adopt, self._pool, self._table)

    def grow(self, table, lens, add: torch.Tensor, tokens: int, out=None) -> tuple:
        """``add`` [B] int32 tokens more for each sequence -> (slots [tokens], positions [tokens], starts
        [B + 1]), int32, as the runners' ``append`` and ``attend`` take them. ``lens`` grows and ``table`` gets the
        pages taken, in place. ``tokens``: rows of the outputs; those behind the sum of ``add`` have slot -1.
        ``out``: the three tensors. A sequence for which no pages are left, no entries in the table or no rows in
        the outputs stays as it was, its tokens' slots are -1 and it is recorded (``raise_on_device_error``). Pages
        are given in the rows' order, and none past a row that goes without for want of them: the rows behind it
        that need a page go without too, though some may be free. What has to go on (decode steps) belongs in the
        rows before what may wait (prompts), or in a call before."""
        seqs = self._set_table(table, lens)
        at_add = self._vec("add", add, seqs)
        if not 0 <= tokens < 1 << 31:
            raise RuntimeError(f"mkmoe pages: {tokens} tokens")
        if out is None:
            no_capture("the tokens' places")
            out = tuple(torch.empty(n, dtype=I32, device=self.device) for n in (tokens, tokens, seqs + 1))
        slots, positions, starts = out
        places = (self._vec("slots", slots, tokens), self._vec("positions", positions, tokens),
                  self._vec("starts", starts, seqs + 1))  # fmt: skip
        self._call(self.lib.mkmoe_pages_grow, self._pool, self._table, at_add, tokens, *places)
        return slots, positions, starts

    def trim(self, table, lens, keep: torch.Tensor) -> None:
        """Sequences cut to their first ``keep`` [B] int32 tokens, in place: their other pages are let go (0 frees
        a sequence; ``lens`` or more leaves it as it is). Where the last page kept is then partly filled and
        others held it too before the call, the sequence gets a copy; it stays as it was, and is recorded, where no
        page was free. That holds where the call lets the others go as well: with no page to spare, free them in
        a call before."""
        seqs = self._set_table(table, lens)
        self._call(self.lib.mkmoe_pages_trim, self._pool, self._table, self._vec("keep", keep, seqs))

    def fork(self, table, lens, parents: torch.Tensor) -> None:
        """Row b goes on from row ``parents[b]`` (int32 [B], -1: empty) as it was before the call, in place. Full
        pages are shared; a last page that is not full stays with the lowest of its rows and the others get
        copies. A row that none goes on from lets go of its pages, which the next call can take. A row for whose
        copy no page is free becomes empty and is recorded."""
        seqs = self._set_table(table, lens)
        self._call(self.lib.mkmoe_pages_fork, self._pool, self._table, self._vec("parents", parents, seqs))

    def compact(self, table, lens) -> None:
        """The n pages held moved to the pool's first n, the table's entries with them: those behind to the free
        ones before, both in order. ``table`` has every sequence that holds pages; where their number shows that
        it does not, nothing is moved and it is recorded."""
        self._set_table(table, lens)
        self._call(self.lib.mkmoe_pages_compact, self._pool, self._table)

    def copy(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Pages ``src`` [n] int32 copied to ``dst`` in every cache. ``dst`` are distinct and none of them is among
        ``src``; who holds them is not changed. Pairs outside the pool are left out and recorded."""
        at = self._vec("src", src)
        n = src.shape[0]
        if n > self.pages:
            raise self._bad("src", src, f"[n <= {self.pages}] {I32}")
        self._call(self.lib.mkmoe_pages_copy, self._pool, at, self._vec("dst", dst, n), n)

    # ---- device errors
    def read_errors(self) -> list[int]:
        """The device error words (synchronises the stream)."""
        words = (ctypes.c_int32 * _lib.PAGES_ERRW_WORDS)()
        stream = torch._C._cuda_getCurrentRawStream(self._index)
        with torch.cuda.device(self.device):
            _lib.check(self.lib.mkmoe_pages_read_errors(self._ws[0], words, len(words), stream), "pages errors")
        return list(words)

    def raise_on_device_error(self) -> None:
        """Raise if a call since the last ``clear_errors`` met a value outside its bounds or found no room
        (synchronises the stream)."""
        code, where, count, _ = self.read_errors()
        if code:
            raise RuntimeError(f"mkmoe pages: {_lib.PAGES_ERRORS.get(code, code)} {where} ({count} seen)")

    def clear_errors(self) -> None:
        """Forget recorded errors (on the current stream)."""
        self.ws[: 4 * _lib.PAGES_ERRW_WORDS].zero_()
