"""A prompt's attention over the paged latent cache, and the cache's pages, as timed cases.

A token's keys and values are one shared latent row: 512 latent values (after an RMSNorm) and 64
rotated rope values, kept in a paged cache as bf16 (576 values a row) or as MXFP8 (512 e4m3 codes,
16 E8M0 scales, one per 32 values, and the 64 rope values in bf16: 656 bytes a row). A chunk of a
prompt's new tokens attends over it with a key and a value for each head and token, made from the
latents by W_UK and W_UV. A page of the cache belongs to one or several sequences.

Fields of a case:
- ``op``: "chunk" (new tokens' attention over the cached rows, theirs among them), "step" (a layer's
  whole attention of such tokens: norm, rotate and store their rows first), "grow" (the step before
  taken back, then every sequence's next tokens given their places), "fork" (the samples before freed,
  then new ones forked), "compact" (tables taken over, their pages moved to the front of the pool)
  or "copy" (pages to other pages)
- ``fmt``: the cache's, "bf16" or "mxfp8"; ``page``: tokens a page; ``heads``: of one rank
- chunk, step: ``seqs``, ``new``, ``past``: sequences, the most new and earlier tokens of one;
  ``lens``: "one" (all have so many), "ragged" (spread over 1 .. new, 0 .. past) or "padded" (ragged, and a quarter
  of the sequences empty)
- pages: ``pages``: the pool's; ``layers``: caches that its pages index; ``seqs``, ``max_len``:
  sequences, of 1 .. max_len tokens; ``add`` (grow): the most new tokens of one; ``ways`` (fork):
  samples of each prompt; ``moved`` (copy): pages copied

``own`` false: elementary torch operations. True: ``LatentPromptRunner``'s and ``PagePool``'s calls.
"""

import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
LATENT, ROPE, ROW = 512, 64, 576
NOPE, VDIM = 128, 128  # a head's query part without rotation, and its value
MX_ROW = LATENT + LATENT // 32 + 2 * ROPE
EPS = 1e-6
SCALE = (NOPE + ROPE) ** -0.5
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def _chunk(name, op, seqs, new, past, heads, fmt, page, lens="ragged", rope="interleaved"):
    return dict(name=name, op=op, seqs=seqs, new=new, past=past, heads=heads, fmt=fmt, page=page, lens=lens, rope=rope)


def _pages(name, op, pages, page, fmt, layers, seqs, max_len, **more):
    return dict(name=name, op=op, pages=pages, page=page, fmt=fmt, layers=layers, seqs=seqs, max_len=max_len, **more)


def listed():
    return [
        # one user's short message behind a short chat: latency
        _chunk("chunk_small", "chunk", 1, 193, 700, 16, "bf16", 64, lens="one"),
        # a question about a long document: few rows, so the keys are split over the card
        _chunk("chunk_long_past", "chunk", 1, 300, 65000, 16, "bf16", 64, lens="one"),
        # the largest: a chunk of a long prompt in its second half, 8-bit cache
        _chunk("chunk_large_mxfp8", "chunk", 1, 8191, 8192, 32, "mxfp8", 64, lens="one"),
        # a layer's step over whole short prompts, ragged, padded, in single-token pages
        _chunk("step_prompts", "step", 16, 1000, 0, 32, "bf16", 1, lens="padded"),
        # a layer's step over a few prompts' next chunks, 8-bit cache, many heads
        _chunk("step_chunks_mxfp8", "step", 4, 1024, 4096, 64, "mxfp8", 16, rope="half"),
        # places for a verify step's tokens: latency
        _pages("grow_verify", "grow", 8192, 64, "bf16", 0, 45, 8192, add=4),
        # places for whole prompts in a pool of single-token pages
        _pages("grow_prompts", "grow", 1 << 20, 1, "mxfp8", 0, 24, 20000, add=8192),
        # a few samples of one prompt, a single cache
        _pages("fork_few", "fork", 300, 64, "bf16", 1, 1, 4001, ways=3),
        # a batch of prompts with eight samples each, a model's layers
        _pages("fork_layers", "fork", 1500, 32, "bf16", 24, 40, 1000, ways=8),
        # a fragmented pool of one cache, 8-bit
        _pages("compact_one", "compact", 2048, 64, "mxfp8", 1, 24, 3000),
        # a fragmented pool, a model's layers
        _pages("compact_layers", "compact", 1200, 64, "bf16", 24, 24, 1500),
        # a document's pages duplicated in a model's layers
        _pages("copy_layers", "copy", 1000, 64, "mxfp8", 24, 0, 0, moved=301),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["chunk", "chunk", "chunk", "step", "grow", "fork", "compact", "copy"])
    fmt = rng.choice(["bf16", "mxfp8"])
    page = rng.choice([1, 2, 8, 16, 32, 64, 128])
    if op in ("chunk", "step"):
        heads = rng.choice([8, 12, 16, 24, 32, 40, 64, 128])
        seqs = _log(rng, 1, 24)
        # no more keys and values, and no more scores, than the largest listed cases have
        top = (1 << 20) // (heads * seqs)
        new = _log(rng, 1, min(8192, max(2, top // 2)))
        past = rng.choice([0, _log(rng, 1, max(1, top - new))])
        past = min(past, max(0, int(3.0e9 / (heads * seqs * new)) - new // 2))
        c = _chunk("", op, seqs, new, past, heads, fmt, page, rng.choice(["one", "ragged", "ragged", "padded"]),
                   rng.choice(["interleaved", "half"]))  # fmt: skip
    elif op == "grow":
        seqs, max_len, add = _log(rng, 1, 64), _log(rng, 1, 16384), _log(rng, 1, 4096)
        pages = seqs * (-(-(max_len + add) // page)) + _log(rng, 1, 4096)
        c = _pages("", op, pages, page, fmt, 0, seqs, max_len, add=add)
    else:
        layers = rng.choice([1, 2, 5, 16, 24])
        row = 2 * ROW if fmt == "bf16" else MX_ROW
        most = max(12, int(1.8e9 / (layers * row * page)))  # the pool's pages
        pages = min(_log(rng, 12, 4096), most)
        if op == "copy":
            c = _pages("", op, pages, page, fmt, layers, 0, 0, moved=_log(rng, 1, pages // 3))
        else:
            ways = rng.choice([1, 2, 3, 4, 8]) if op == "fork" else 0
            seqs = _log(rng, 1, max(1, min(48, pages // (2 * (ways + 1)))))
            max_len = _log(rng, 1, max(1, (pages - seqs * ways) * page // (2 * seqs)))
            c = _pages("", op, pages, page, fmt, layers, seqs, max_len, **({"ways": ways} if ways else {}))
    del c["name"]
    return c


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed * 7919 + 23)


def _randn(g, *shape, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(BF)


def _cos_sin(positions):
    """[positions, 64] fp32: 32 cosines, then 32 sines, of angles formed in 64 bits."""
    inv = 10000.0 ** (-torch.arange(0, ROPE, 2, dtype=F64, device=DEV) / ROPE)
    a = torch.arange(positions, dtype=F64, device=DEV)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], 1).float()


def _mx_cache(latent, rope):
    """Rows of a cache [n, 656] from latent values [n, 512] and bf16 rope values."""
    v = latent.unflatten(-1, (-1, 32))
    top = v.abs().amax(-1).clamp_min(torch.finfo(F32).tiny) / 448
    m, e = torch.frexp(top)  # top = m 2^e, m in [0.5, 1): the least power of two not below it
    e = torch.where(m == 0.5, e - 1, e).clamp(-126, 127)
    q = (v * torch.exp2(-e.to(v.dtype))[..., None]).clamp(-448, 448).float().to(torch.float8_e4m3fn)
    return torch.cat([q.view(torch.uint8).flatten(-2), (e + 127).to(torch.uint8), rope.contiguous().view(torch.uint8)], 1)


def _cache(g, fmt, pages, page):
    """A cache as earlier steps left it: latents of RMS 1, rope values of the same size."""
    n = pages * page
    out = torch.empty(n, ROW if fmt == "bf16" else MX_ROW, dtype=BF if fmt == "bf16" else torch.uint8, device=DEV)
    for part in out.split(1 << 17):
        row = _randn(g, part.shape[0], ROW)
        part.copy_(row if fmt == "bf16" else _mx_cache(row[:, :LATENT].float(), row[:, LATENT:]))
    return out.view(pages, page, -1)


def _spread(most, count, least=1):
    """``count`` whole numbers from ``least`` to ``most``, evenly apart."""
    return [most - (most - least) * i // max(1, count - 1) for i in range(count)]


def _new_tokens(case):
    """How many new tokens the sequences of a case have, by size: every seed's inputs have as many."""
    b = case["seqs"]
    if case["lens"] == "one":
        return [case["new"]] * b
    empty = b // 4 if case["lens"] == "padded" else 0
    return _spread(case["new"], b - empty) + [0] * empty


def _chunk_data(case, seed):
    g, rng = _gen(seed), random.Random(seed * 31 + 5)
    b, page, h = case["seqs"], case["page"], case["heads"]
    new = _new_tokens(case)
    past = [case["past"]] * b
    if case["lens"] != "one":
        live = sum(n > 0 for n in new)
        new = rng.sample(new[:live], live) + new[live:]  # the empty ones stay at the end
        past = [rng.randint(0, case["past"]) if n else 0 for n in new]
    lens = [n + p for n, p in zip(new, past)]
    starts = [sum(new[:i]) for i in range(b + 1)]
    t = starts[-1]
    per = -(-(case["new"] + case["past"]) // page)
    pages = b * per
    table = torch.randperm(pages, generator=g, device=DEV).view(b, per).int()
    dev = lambda v, dt=torch.int32: torch.tensor(v, dtype=dt, device=DEV)  # noqa: E731
    d = dict(new=new, past=past, at=starts, table=table, lens=dev(lens), tokens=t)
    d["starts"] = None if case["lens"] == "one" else dev(starts)
    d["kv_b"] = _randn(g, h * (NOPE + VDIM), LATENT, std=LATENT**-0.5)
    d["norm"] = (1 + 0.1 * torch.randn(LATENT, generator=g, device=DEV)).to(BF)
    d["q"] = _randn(g, t, h, NOPE + ROPE)
    if case["op"] == "chunk":
        d["q_pe"] = _randn(g, t, h, ROPE)  # rotated, as the rows' append gave it
    else:
        d["kv"] = _randn(g, t, ROW)
        d["cos_sin"] = _cos_sin(max(1, case["new"] + case["past"]))
        pos = [torch.arange(p, p + n) for n, p in zip(new, past)]
        d["positions"] = torch.cat(pos).to(DEV)
        seq = torch.repeat_interleave(torch.arange(b), torch.tensor(new)).to(DEV)
        d["slots"] = table[seq, d["positions"] // page].long() * page + d["positions"] % page
    d["cache"] = _cache(g, case["fmt"], pages, page)
    return d


def _pages_data(case, seed):
    g, rng = _gen(seed), random.Random(seed * 37 + 11)
    op, pages, page, b = case["op"], case["pages"], case["page"], case["seqs"]
    d = dict(caches=[_cache(g, case["fmt"], pages, page) for _ in range(case["layers"])])
    perm = torch.randperm(pages, generator=g, device=DEV).int()
    if op == "copy":
        n = case["moved"]
        d["src"], d["dst"] = perm[:n].contiguous(), perm[n : 2 * n].contiguous()
        return d
    lens = [rng.randint(1, case["max_len"]) for _ in range(b)]
    rows = b * (1 + case.get("ways", 0))
    width = -(-(case["max_len"] + case.get("add", 0)) // page)
    table = torch.zeros(rows, width, dtype=torch.int32)
    at, host = 0, perm.cpu()
    for i, n in enumerate(lens):
        k = -(-n // page)
        table[i, :k] = host[at : at + k]
        at += k
    d["table"] = table.to(DEV)
    d["lens"] = torch.tensor(lens + [0] * (rows - b), dtype=torch.int32, device=DEV)
    d["table0"], d["lens0"] = d["table"].clone(), d["lens"].clone()
    if op == "grow":
        add = rng.sample(_spread(case["add"], b, 0), b)
        d["add"], d["tokens"] = torch.tensor(add, dtype=torch.int32, device=DEV), sum(add)
    if op == "fork":
        ways = case["ways"]
        parents = list(range(b)) + [i // ways for i in range(b * ways)]
        d["parents"] = torch.tensor(parents, dtype=torch.int32, device=DEV)
        # rows that get a page of their own: the samples of prompts whose last page is not full
        d["own_page"] = torch.tensor([i for i in range(b, rows) if lens[parents[i]] % page], dtype=torch.int64, device=DEV)
    return d


def _data(case, seed):
    return _chunk_data(case, seed) if case["op"] in ("chunk", "step") else _pages_data(case, seed)


def prepare(case, seed):
    d = _data(case, seed)
    st = dict(case=case, d=d)
    op = case["op"]
    if own:
        sys.path.insert(1, os.path.join(os.getcwd(), "sgl-amd-mono_amd"))
    if op in ("chunk", "step"):
        st["out"] = torch.empty(d["tokens"], case["heads"], VDIM, dtype=BF, device=DEV)
        if own:
            from sgl_amd_mono.moe.latent import LatentWeights
            from sgl_amd_mono.moe.latent_prompt import LatentPromptRunner

            context = sum(-(-(n + p) // 64) * 64 for n, p in zip(d["new"], d["past"]))
            st["w"] = LatentWeights(norm=d["norm"], kv_b=d["kv_b"])
            st["runner"] = LatentPromptRunner(
                case["heads"], max_tokens=max(1, d["tokens"]), max_context=context, scale=SCALE, norm_eps=EPS,
                rope=case["rope"],
            )  # fmt: skip
    elif own:
        from sgl_amd_mono.moe.pages import PagePool

        seqs, width = d["table"].shape if "table" in d else (1, 1)
        st["pool"] = PagePool(case["pages"], case["page"], caches=d["caches"], max_seqs=seqs, max_pages=width)
        if "table" in d:
            st["pool"].adopt(d["table"], d["lens"])
        if op == "grow":
            st["places"] = [torch.empty(n, dtype=torch.int32, device=DEV) for n in (d["tokens"], d["tokens"], case["seqs"] + 1)]
    elif "table" in d:
        st["refs"] = _plain_refs(case, d)
    return st


# ---------------------------------------------------------------- the calls
def _run_own(st):
    case, d = st["case"], st["d"]
    op = case["op"]
    if op == "chunk":
        return st["runner"].attend(
            st["w"], d["cache"], d["q"][..., :NOPE], d["q_pe"], d["table"], d["lens"], q_starts=d["starts"], out=st["out"]
        )
    if op == "step":
        r = st["runner"]
        r.attention(
            st["w"], d["cache"], d["q"], d["kv"], d["cos_sin"], d["positions"], d["slots"], d["table"], d["lens"],
            q_starts=d["starts"], out=st["out"],
        )  # fmt: skip
        # 8-bit rows are handed on as the values that they stand for
        return st["out"], r.rows(d["cache"], d["slots"]) if case["fmt"] == "mxfp8" else d["cache"]
    pool = st["pool"]
    if op == "copy":
        pool.copy(d["src"], d["dst"])
        return list(d["caches"])
    if op == "compact":
        d["table"].copy_(d["table0"])
        d["lens"].copy_(d["lens0"])
        pool.adopt(d["table"], d["lens"])
        pool.compact(d["table"], d["lens"])
    else:
        pool.trim(d["table"], d["lens"], d["lens0"])
        if op == "grow":
            return *pool.grow(d["table"], d["lens"], d["add"], d["tokens"], out=st["places"]), d["table"], d["lens"], pool.refs
        pool.fork(d["table"], d["lens"], d["parents"])
    return d["table"], d["lens"], pool.refs, list(d["caches"])


def run(state):
    if own:
        return _run_own(state)
    return _plain_chunk(state) if state["case"]["op"] in ("chunk", "step") else _plain_pages(state)


# ---------------------------------------------------------------- the plain form: attention
def _rotate(x, cos, sin, rope):
    if rope == "half":
        a, b = x[..., : ROPE // 2], x[..., ROPE // 2 :]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    a, b = x[..., ::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)


def _plain_rows(cache):
    """The values of cache rows [..., row] in 32 bits."""
    if cache.dtype == BF:
        return cache.float()
    q = cache[..., :LATENT].contiguous().view(torch.float8_e4m3fn).float().unflatten(-1, (-1, 32))
    e = torch.exp2(cache[..., LATENT : LATENT + LATENT // 32].float() - 127)
    pe = cache[..., LATENT + LATENT // 32 :].contiguous().view(BF).float()
    return torch.cat([(q * e[..., None]).flatten(-2), pe], -1)


def _plain_append(d, rope, fmt):
    """Writes the rows; returns the rotation's cosines and sines."""
    dt = F64 if fmt == "mxfp8" else F32  # codes sit next to a border: 64 bits
    c = d["kv"][:, :LATENT].to(dt)
    c = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS) * d["norm"].to(dt)
    cs = d["cos_sin"][d["positions"]]
    cos, sin = cs[:, : ROPE // 2], cs[:, ROPE // 2 :]
    pe = _rotate(d["kv"][:, LATENT:].float(), cos, sin, rope).to(BF)
    row = torch.cat([c.to(BF), pe], 1) if fmt == "bf16" else _mx_cache(c, pe)
    d["cache"].view(-1, row.shape[1])[d["slots"]] = row
    return cos[:, None], sin[:, None]


def _plain_chunk(st):
    case, d, out = st["case"], st["d"], st["out"]
    h, page = case["heads"], case["page"]
    q = d["q"].float()
    if case["op"] == "chunk":
        q_pe = d["q_pe"].float()
    else:
        cos, sin = _plain_append(d, case["rope"], case["fmt"])
        q_pe = _rotate(q[..., NOPE:], cos, sin, case["rope"])
    w = d["kv_b"].float().view(h, NOPE + VDIM, LATENT)
    flat = d["cache"].view(-1, d["cache"].shape[-1])
    for i, (n, past) in enumerate(zip(d["new"], d["past"])):
        if n == 0:
            continue
        t0, length = d["at"][i], n + past
        key = torch.arange(length, device=DEV)
        rows = _plain_rows(flat[d["table"][i].long()[key // page] * page + key % page])
        qs = torch.cat([q[t0 : t0 + n, :, :NOPE], q_pe[t0 : t0 + n]], -1).transpose(0, 1)  # [h, n, 192]
        heads = max(1, min(h, (1 << 28) // length // 640))
        for h0 in range(0, h, heads):
            hs = slice(h0, h0 + heads)
            kv = rows[:, :LATENT] @ w[hs].flatten(0, 1).T  # [len, heads x 256]
            kv = kv.view(length, -1, NOPE + VDIM).transpose(0, 1)
            k = torch.cat([kv[..., :NOPE], rows[:, LATENT:].expand(kv.shape[0], -1, -1)], -1)
            v = kv[..., NOPE:].contiguous()
            step = max(1, (1 << 27) // (length * k.shape[0]))
            for a in range(0, n, step):
                s = qs[hs, a : a + step].contiguous() @ k.transpose(1, 2) * SCALE
                at = past + a + torch.arange(s.shape[1], device=DEV)
                s.masked_fill_(key > at[:, None], -math.inf)
                p = torch.exp(s - s.amax(-1, keepdim=True))
                o = (p @ v) / p.sum(-1, keepdim=True)
                out[t0 + a : t0 + a + s.shape[1], hs] = o.transpose(0, 1).to(BF)
    if case["op"] == "chunk":
        return out
    if case["fmt"] == "bf16":
        return out, d["cache"]
    return out, _plain_rows(flat[d["slots"]]).to(BF)


# ---------------------------------------------------------------- the plain form: pages
def _plain_refs(case, d):
    """How many sequences hold each page."""
    held = -(-d["lens"] // case["page"])
    live = torch.arange(d["table"].shape[1], device=DEV) < held[:, None]
    refs = torch.zeros(case["pages"], dtype=torch.int32, device=DEV)
    return refs.index_add_(0, d["table"].flatten(), live.flatten().int())


def _plain_trim(st):
    """Back to lens0; a page that is then partly filled is held by this sequence alone."""
    d, page = st["d"], st["case"]["page"]
    col = torch.arange(d["table"].shape[1], device=DEV)
    gone = (col < (-(-d["lens"] // page))[:, None]) & (col >= (-(-d["lens0"] // page))[:, None])
    st["refs"].index_add_(0, d["table"].flatten(), -gone.flatten().int())
    d["lens"].copy_(torch.minimum(d["lens"], d["lens0"]))


def _plain_free(refs):
    """Pages, the free ones first, in order."""
    return torch.sort((refs > 0).to(torch.int8), stable=True).indices.int()


def _plain_pages(st):
    case, d = st["case"], st["d"]
    op, page = case["op"], case["page"]
    if op == "copy":
        for c in d["caches"]:
            c[d["dst"]] = c[d["src"]]
        return list(d["caches"])
    table, lens = d["table"], d["lens"]
    if op == "compact":
        table.copy_(d["table0"])
        lens.copy_(d["lens0"])
        refs = st["refs"].copy_(_plain_refs(case, d))
        live = refs > 0
        count = live.sum()
        at = torch.arange(case["pages"], device=DEV)
        src = (live & (at >= count)).nonzero()[:, 0]
        dst = (~live & (at < count)).nonzero()[:, 0]
        for c in d["caches"]:
            c[dst] = c[src]
        to = at.int()
        to[src] = dst.int()
        refs[dst] = refs[src]
        refs[src] = 0
        held = torch.arange(table.shape[1], device=DEV) < (-(-lens // page))[:, None]
        table.copy_(torch.where(held, to[table], table))
        return table, lens, refs, list(d["caches"])
    _plain_trim(st)
    refs = st["refs"]
    free = _plain_free(refs)
    if op == "fork":
        rows, parents = d["own_page"], d["parents"].long()
        table.copy_(table[parents])
        lens.copy_(lens[parents])
        new, last = free[: rows.shape[0]], (lens[rows] // page).long()
        for c in d["caches"]:
            c[new] = c[table[rows, last]]
        table[rows, last] = new
        refs.copy_(_plain_refs(case, d))
        return table, lens, refs, list(d["caches"])
    # grow: token r of the call belongs to sequence seq[r], as its token at[r]
    t, add = d["tokens"], d["add"]
    ends = add.cumsum(0)
    r = torch.arange(t, device=DEV)
    seq = torch.searchsorted(ends, r, right=True)
    at = (lens[seq] + r - (ends - add)[seq]).int()
    held = -(-lens // page)
    need = -(-(lens + add) // page) - held
    first = need.cumsum(0) - need
    k = at // page - held[seq]  # which of the sequence's new pages; below 0 its last one before
    got = torch.where(k >= 0, free[(first[seq] + k).clamp_min(0)], table[seq, (at // page).long()])
    table[seq, (at // page).long()] = got
    refs[got] = 1
    lens += add
    starts = torch.cat([ends.new_zeros(1), ends]).int()
    return got * page + at % page, at, starts, table, lens, refs


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    op, row = case["op"], 2 * ROW if case["fmt"] == "bf16" else MX_ROW
    page = case["page"]
    if op in ("chunk", "step"):
        h, new = case["heads"], [n for n in _new_tokens(case) if n]
        past = case["past"] if case["lens"] == "one" else case["past"] / 2
        t, cached = sum(new), sum(n + past for n in new)
        pairs = sum(n * past + n * (n + 1) / 2 for n in new)
        w = h * (NOPE + VDIM) * LATENT
        b = cached * (row + 4 / page) + 8 * case["seqs"] + 2 * w + t * h * 2 * (NOPE + ROPE + VDIM)
        # the keys and values of every cached token, once a call, then 192 + 128 products for each score
        f = cached * 2 * w + 2 * pairs * h * (NOPE + ROPE + VDIM)
        if op == "step":
            back = row + 2 * ROW + 8 if case["fmt"] == "mxfp8" else 0
            b += t * (2 * ROW + row + 8 * ROPE // 2 + 16 + back)
            f += t * (5 * LATENT + 6 * ROPE // 2 * (h + 1))
        return {"bytes": b, "flops": f}
    if op == "copy":
        return {"bytes": 2 * case["moved"] * case["layers"] * page * row + 8 * case["moved"], "flops": 0}
    b, mean = case["seqs"], (case["max_len"] + 1) / 2
    entries = b * mean / page + b / 2
    if op == "grow":
        t = sum(_spread(case["add"], b, 0))
        # slots, positions and starts, new pages' entries and counts, taken back and given anew
        return {"bytes": 8 * t + 16 * b + 16 * (t / page + b / 2), "flops": 0}
    if op == "fork":
        ways = case["ways"]
        moved = b * ways * (1 - 1 / page)
        return {"bytes": 2 * moved * case["layers"] * page * row + 16 * entries * ways + 16 * b * (1 + ways), "flops": 0}
    moved = entries * max(0.0, 1 - entries / case["pages"])  # pages behind the first ones, dealt at random
    return {"bytes": 2 * moved * case["layers"] * page * row + 8 * case["pages"] + 24 * entries + 16 * b, "flops": 0}


# ---------------------------------------------------------------- the definition in 64 bits
def _turn(x, pos, cos_sin, rope):
    """x [t, k, 64] as 32 complex numbers, each turned by its angle."""
    cs = cos_sin[pos].double()
    turn = torch.complex(cs[:, :32], cs[:, 32:])[:, None]
    z = x.double()
    if rope == "half":
        z = torch.complex(z[..., :32], z[..., 32:]) * turn
        return torch.cat([z.real, z.imag], -1)
    z = torch.complex(z[..., 0::2].contiguous(), z[..., 1::2].contiguous()) * turn
    return torch.view_as_real(z).flatten(-2)


def _fp8_near(v):
    """The nearest e4m3 value (ties to even), |v| <= 448."""
    a = v.abs()
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0**-6))) - 3)
    return torch.sign(v) * torch.round(a / step) * step


def _exact_rows(raw, fmt):
    """Cached rows' values [n, 576] in 64 bits."""
    if fmt == "bf16":
        return raw.double()
    code = raw[:, :LATENT].int()
    m, e = code & 7, (code >> 3) & 15
    v = torch.where(e > 0, torch.exp2(e.double() - 7) * (1 + m.double() / 8), m.double() * 2.0**-9)
    v = torch.where(code >= 128, -v, v)
    sc = torch.exp2(raw[:, LATENT : LATENT + 16].double() - 127).repeat_interleave(32, 1)
    pe = raw[:, LATENT + 16 :].contiguous().view(BF).double()
    return torch.cat([v * sc, pe], 1)


def _new_rows(d, rope, fmt):
    """The step's rows in 64 bits (MXFP8: the values that they are held as)."""
    x = d["kv"].double()
    c = x[:, :LATENT]
    c = c / ((c**2).sum(1, keepdim=True) / LATENT + EPS).sqrt() * d["norm"].double()
    pe = _turn(x[:, None, LATENT:], d["positions"], d["cos_sin"], rope)[:, 0]
    if fmt == "mxfp8":
        g = c.view(-1, 16, 32)
        s = torch.exp2(torch.ceil(torch.log2(g.abs().amax(-1, keepdim=True) / 448)))
        c = (_fp8_near(g / s) * s).flatten(1)
    return torch.cat([c, pe], 1)


def exact(case, seed):
    op, fmt, page = case["op"], case["fmt"], case["page"]
    if op not in ("chunk", "step"):
        return None  # whole numbers, and bytes moved as they are
    d = _data(case, seed)
    h, q = case["heads"], d["q"].double()
    raw = d["cache"].view(-1, d["cache"].shape[-1])
    if op == "chunk":
        qp, held = d["q_pe"].double(), None
    else:
        qp = _turn(q[..., NOPE:], d["positions"], d["cos_sin"], case["rope"])
        new = _new_rows(d, case["rope"], fmt)
        stored = new.to(BF).double()  # a bf16 row; an MXFP8 row's values fit bf16 as they are
        held = new
        if fmt == "bf16":
            held = d["cache"].double().view(-1, ROW)
            held[d["slots"]] = new
            held = held.view(d["cache"].shape)
    w = d["kv_b"].double().view(h, 2, 128, LATENT)
    out = torch.zeros(d["tokens"], h, VDIM, dtype=F64, device=DEV)
    for i, (n, past) in enumerate(zip(d["new"], d["past"])):
        if n == 0:
            continue
        t0 = d["at"][i]
        at = torch.arange(n + past, device=DEV)
        kv = _exact_rows(raw[d["table"][i].long()[at // page] * page + at % page], fmt)
        if op == "step":
            kv[past:] = stored[t0 : t0 + n]
        c, pe = kv[:, :LATENT], kv[:, LATENT:]
        late = torch.arange(past, past + n, device=DEV)
        for hh in range(h):
            k, v = torch.cat([c @ w[hh, 0].T, pe], 1), c @ w[hh, 1].T
            for a in range(0, n, 4096):
                z = slice(t0 + a, t0 + min(n, a + 4096))
                s = torch.cat([q[z, hh, :NOPE], qp[z, hh]], 1) @ k.T * SCALE
                s = torch.where(at[None] <= late[a : a + 4096, None], s, torch.full_like(s[:1, :1], -math.inf))
                out[z, hh] = torch.softmax(s, -1) @ v
    return out if op == "chunk" else (out, held)
