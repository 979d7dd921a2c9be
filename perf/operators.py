"""The latent-attention operators of a decode layer, as timed cases.

One token's keys and values are one shared latent row: 512 latent values (after an RMSNorm) and
64 rotated rope values, kept in a paged cache as bf16 (576 values a row) or as MXFP8 (512 e4m3
codes, 16 E8M0 scales, one per 32 values, and the 64 rope values in bf16: 656 bytes a row).

Fields of a case:
- ``op``: "append" (norm, rotate, write the step's rows into the cache, rotate the query's rope
  part), "attend" (the absorbed form: every head's 512 + 64 query values against the cached rows,
  whose latent part is also the value) or "step" (a layer's whole attention: append, the query
  through W_UK, attend, the result through W_UV)
- ``fmt``: the cache's, "bf16" or "mxfp8"; ``page``: tokens a page; ``heads``: of one rank
- ``tokens`` (append): the call's tokens; ``rope``: "interleaved" or "half"
- ``seqs``, ``max_len``: sequences, and the longest one's cached tokens; ``lens``: "one" (all of
  them that long), "ragged" (spread over 1 .. max_len) or "padded" (ragged, and a quarter of the
  sequences empty, as in a step padded to a captured batch)
- ``n``: query tokens a sequence, the last of its tokens (1: decode; more: tokens to verify);
  ``mixed``: 1 .. n of them, differing by sequence

``own`` false: elementary torch operations in 32 bits. True: the calls of ``LatentRunner``.
"""

import math
import os
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


def _append(name, tokens, heads, fmt, page, rope="interleaved"):
    return dict(name=name, op="append", tokens=tokens, heads=heads, fmt=fmt, page=page, rope=rope)


def _over(name, op, seqs, max_len, heads, fmt, page, lens="ragged", n=1, mixed=False):
    return dict(
        name=name, op=op, seqs=seqs, max_len=max_len, heads=heads, fmt=fmt, page=page, lens=lens, n=n, mixed=mixed
    )


def listed():
    return [
        # a small decode step's rows: a launch's latency
        _append("append_decode", 7, 32, "bf16", 64),
        # a verify step's rows, three tokens for each of 15 sequences, 8-bit cache
        _append("append_verify_mxfp8", 45, 64, "mxfp8", 16, "half"),
        # a long prompt's rows, an odd number of them
        _append("append_prompt", 8191, 32, "bf16", 64),
        # one user's chat: latency, a page that ends inside the last tile
        _over("attend_one_short", "attend", 1, 1025, 32, "bf16", 64, lens="one"),
        # one user's long document: one row of work split over the whole card
        _over("attend_one_long", "attend", 1, 131071, 32, "bf16", 64, lens="one"),
        # a full decode step of ragged sequences, padded to a captured batch; a table of single tokens
        _over("attend_padded", "attend", 48, 8192, 32, "bf16", 1, lens="padded"),
        # a verify step: 4 x 64 rows read each cached token
        _over("attend_verify", "attend", 12, 8192, 64, "bf16", 64, n=4),
        # a few users, 8-bit cache, small pages
        _over("attend_mxfp8_few", "attend", 8, 2500, 64, "mxfp8", 16),
        # the largest: a full batch of long sequences in 8 bits
        _over("attend_mxfp8_large", "attend", 64, 16384, 32, "mxfp8", 64),
        # a verify step in which the sequences bring 1 .. 4 tokens each
        _over("attend_mxfp8_mixed", "attend", 24, 4096, 16, "mxfp8", 1, n=4, mixed=True),
        # a layer's whole attention in a small and in a full decode step
        _over("step_few", "step", 8, 2048, 32, "bf16", 64),
        _over("step_full_mxfp8", "step", 48, 4096, 64, "mxfp8", 64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "step"])
    fmt = rng.choice(["bf16", "mxfp8"])
    page = rng.choice([1, 2, 8, 16, 32, 64, 128])
    heads = rng.choice([8, 12, 16, 24, 32, 40, 64, 128])
    if op == "append":
        c = _append("", _log(rng, 1, 8192), heads, fmt, page, rng.choice(["interleaved", "half"]))
    else:
        n = rng.choice([1, 1, 2, 3, 4, 5])
        seqs = _log(rng, 1, 64) if op == "attend" else _log(rng, 1, max(1, 48 // n))
        # no more cached tokens, and no more rows against each, than the largest listed cases have
        top = min(131072, 64 * 16384 // seqs if op == "attend" else 48 * 4096 // seqs)
        if n * heads > 64:
            top = min(top, max(2 * n, 12 * 8192 * 256 // (seqs * n * heads)))
        lens = rng.choice(["one", "ragged", "ragged", "padded"])
        c = _over("", op, seqs, _log(rng, n, top), heads, fmt, page, lens, n, n > 1 and rng.random() < 0.4)
    del c["name"]
    return c


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed * 7919 + 17)


def _randn(g, *shape, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(BF)


def _cos_sin(positions):
    """[positions, 64] fp32: 32 cosines, then 32 sines, of angles formed in 64 bits."""
    inv = 10000.0 ** (-torch.arange(0, ROPE, 2, dtype=F64, device=DEV) / ROPE)
    a = torch.arange(positions, dtype=F64, device=DEV)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], 1).float()


def _mx_pack(x):
    """Latent values [n, 512] -> codes [n, 512] and scales [n, 16] (uint8)."""
    v = x.unflatten(-1, (-1, 32))
    top = v.abs().amax(-1).clamp_min(torch.finfo(F32).tiny) / 448
    m, e = torch.frexp(top)  # top = m 2^e, m in [0.5, 1): the least power of two not below it
    e = torch.where(m == 0.5, e - 1, e).clamp(-126, 127)
    q = (v * torch.exp2(-e.to(v.dtype))[..., None]).clamp(-448, 448).float().to(torch.float8_e4m3fn)
    return q.view(torch.uint8).flatten(-2), (e + 127).to(torch.uint8)


def _mx_cache(latent, rope):
    """Rows of a cache [n, 656] from latent values and bf16 rope values."""
    q, e = _mx_pack(latent)
    return torch.cat([q, e, rope.contiguous().view(torch.uint8)], 1)


def _cache(g, fmt, pages, page):
    """A cache as earlier steps left it: latents of RMS 1, rope values of the same size."""
    n = pages * page
    out = torch.empty(n, ROW if fmt == "bf16" else MX_ROW, dtype=BF if fmt == "bf16" else torch.uint8, device=DEV)
    for part in out.split(1 << 17):
        row = _randn(g, part.shape[0], ROW)
        part.copy_(row if fmt == "bf16" else _mx_cache(row[:, :LATENT].float(), row[:, LATENT:]))
    return out.view(pages, page, -1)


def _batch(case, g):
    """Lengths, the page table over a cache whose pages are dealt at random, query starts."""
    b, page, n = case["seqs"], case["page"], case["n"]
    cpu = torch.Generator().manual_seed(int(torch.randint(1 << 30, (1,), generator=g, device=DEV)))
    lens = torch.full((b,), case["max_len"])
    if case["lens"] != "one":
        lens = (torch.rand(b, generator=cpu) * (case["max_len"] - n + 1)).int() + n
    live = torch.ones(b, dtype=torch.bool)
    if case["lens"] == "padded":
        live[b - b // 4 :] = False
        lens = torch.where(live, lens, torch.zeros_like(lens))
    per = -(-case["max_len"] // page)
    pages = b * per
    table = torch.randperm(pages, generator=g, device=DEV).view(b, per).int()
    starts = None
    if case["mixed"]:
        cnt = (torch.arange(b) % n + 1)[torch.randperm(b, generator=cpu)]
        starts = torch.cat([torch.zeros(1, dtype=torch.int64), cnt.cumsum(0)]).int()
    tokens = b * n if starts is None else int(starts[-1])
    return lens.int(), table, pages, starts, tokens


def _data(case, seed):
    """The tensors that a program has before the call, by name."""
    g = _gen(seed)
    h, page = case["heads"], case["page"]
    d = dict(norm=(1 + 0.1 * torch.randn(LATENT, generator=g, device=DEV)).to(BF))
    if case["op"] == "append":
        t = case["tokens"]
        pages = -(-2 * t // page)
        limit = 131072
        d["positions"] = torch.randint(limit, (t,), generator=g, device=DEV)
        d["slots"] = torch.randperm(pages * page, generator=g, device=DEV)[:t].contiguous()
        d["q_pe"] = _randn(g, t, h, NOPE + ROPE)[..., NOPE:]  # the rope part of a projection's rows
    else:
        lens, table, pages, starts, t = _batch(case, g)
        d["lens"], d["table"] = lens.to(DEV), table
        d["starts"] = None if starts is None else starts.to(DEV)
        limit = case["max_len"]
        if case["op"] == "attend":
            d["q_lat"] = _randn(g, t, h, LATENT)
            d["q_pe"] = _randn(g, t, h, ROPE)
        else:
            q0 = torch.arange(0, t + 1, case["n"]) if starts is None else starts.long()
            seq = torch.repeat_interleave(torch.arange(case["seqs"]), q0.diff())
            at = lens[seq].long() - q0[seq + 1] + torch.arange(t)  # each query's own place
            live = (lens[seq] > 0).to(DEV)
            seq, at = seq.to(DEV), at.to(DEV).clamp_min(0)
            d["positions"] = at
            slot = table[seq, at // page].long() * page + at % page
            d["slots"] = torch.where(live, slot, torch.full_like(slot, -1))
            d["q"] = _randn(g, t, h, NOPE + ROPE)
            d["kv_b"] = _randn(g, h * (NOPE + VDIM), LATENT, std=LATENT**-0.5)
    if case["op"] != "attend":
        d["kv"] = _randn(g, t, ROW)
        d["cos_sin"] = _cos_sin(limit)
    d["cache"] = _cache(g, case["fmt"], pages, page)
    return d


def prepare(case, seed):
    d = _data(case, seed)
    st = dict(case=case, d=d)
    if own:
        sys.path.insert(1, os.path.join(os.getcwd(), "sgl-amd-mono_amd"))
        from sgl_amd_mono.moe.latent import LatentRunner, LatentWeights

        h, op = case["heads"], case["op"]
        t = d["q_lat" if op == "attend" else "kv"].shape[0]
        st["runner"] = LatentRunner(h, max_tokens=t, scale=SCALE, norm_eps=EPS, rope=case.get("rope", "interleaved"))
        st["out"] = torch.empty(t, h, dict(append=ROPE, attend=LATENT, step=VDIM)[op], dtype=BF, device=DEV)
        if op == "step":
            st["w"] = LatentWeights(norm=d["norm"], kv_b=d["kv_b"])
    return st


# ---------------------------------------------------------------- the calls
def _run_own(st):
    case, d, r, out = st["case"], st["d"], st["runner"], st["out"]
    cache, mx = d["cache"], case["fmt"] == "mxfp8"
    if case["op"] == "attend":
        return r.attend(cache, d["q_lat"], d["q_pe"], d["table"], d["lens"], q_starts=d["starts"], out=out)
    if case["op"] == "append":
        r.append(cache, d["kv"], d["norm"], d["cos_sin"], d["positions"], d["slots"], q_pe=d["q_pe"], q_out=out)
    else:
        r.attention(
            st["w"], cache, d["q"], d["kv"], d["cos_sin"], d["positions"], d["slots"], d["table"], d["lens"],
            q_starts=d["starts"], out=out,
        )  # fmt: skip
    # 8-bit rows are handed on as the values that they stand for
    return out, r.rows(cache, d["slots"]) if mx else cache


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------- the plain form
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
    q = cache[..., :LATENT].view(torch.float8_e4m3fn).float().unflatten(-1, (-1, 32))
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
    flat = d["cache"].view(-1, row.shape[1])
    at = d["slots"].clamp_min(0)  # rows with no slot write what is there
    flat[at] = torch.where(d["slots"][:, None] >= 0, row, flat[at])
    return cos[:, None], sin[:, None]


def _plain_attend(case, d, ql, qp):
    """Absorbed queries [t, h, 512] and [t, h, 64] -> [t, h, 512], in 32 bits."""
    b, page, n, h, t = case["seqs"], case["page"], case["n"], case["heads"], ql.shape[0]
    lens = d["lens"].long()
    flat = d["cache"].view(-1, d["cache"].shape[-1])
    key = torch.arange(case["max_len"], device=DEV)
    row = d["table"].long()[:, key // page] * page + key % page
    q = torch.cat([ql, qp], -1)
    if d["starts"] is None:
        grid, first = torch.arange(b * n, device=DEV).view(b, n), torch.zeros_like(lens)
        cnt = torch.full_like(lens, n)
    else:  # each sequence's queries at the end of n places
        s = d["starts"].long()
        cnt = s.diff()
        first = n - cnt
        grid = (s[1:, None] - n + torch.arange(n, device=DEV)).clamp_min(0)
    out = torch.zeros_like(ql)
    step = max(1, (1 << 20) // max(1, case["max_len"]))
    for i in range(0, b, step):
        kv = _plain_rows(flat[row[i : i + step]])
        ix = grid[i : i + step]
        qs = q[ix].flatten(1, 2)  # [b, n h, 576]
        s = qs @ kv.transpose(1, 2) * SCALE
        limit = lens[i : i + step, None] - n + 1 + torch.arange(n, device=DEV)
        seen = key < limit[:, :, None]
        s = s.unflatten(1, (n, h)).masked_fill(~seen[:, :, None], -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(torch.finfo(F32).min))
        p = p / p.sum(-1, keepdim=True).clamp_min(torch.finfo(F32).tiny)
        o = (p.flatten(1, 2) @ kv[..., :LATENT]).unflatten(1, (n, h))
        real = torch.arange(n, device=DEV) >= first[i : i + step, None]
        out.index_put_((ix,), torch.where(real[..., None, None], o, torch.zeros_like(o)), accumulate=True)
    return out


def _run_plain(st):
    case, d = st["case"], st["d"]
    if case["op"] == "attend":
        return _plain_attend(case, d, d["q_lat"].float(), d["q_pe"].float()).to(BF)
    rope = case.get("rope", "interleaved")
    cos, sin = _plain_append(d, rope, case["fmt"])
    if case["op"] == "append":
        out = _rotate(d["q_pe"].float(), cos, sin, rope)
    else:
        w = d["kv_b"].float().view(case["heads"], NOPE + VDIM, LATENT)
        q = d["q"].float()
        ql = (q[..., :NOPE].transpose(0, 1).contiguous() @ w[:, :NOPE]).transpose(0, 1)
        o = _plain_attend(case, d, ql, _rotate(q[..., NOPE:], cos, sin, rope))
        out = (o.transpose(0, 1).contiguous() @ w[:, NOPE:].transpose(1, 2)).transpose(0, 1).contiguous()
    if case["fmt"] == "bf16":
        return out.to(BF), d["cache"]
    flat = d["cache"].view(-1, MX_ROW)
    rows = _plain_rows(flat[d["slots"].clamp_min(0)])
    return out.to(BF), torch.where(d["slots"][:, None] >= 0, rows, torch.zeros_like(rows)).to(BF)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    h, row = case["heads"], 2 * ROW if case["fmt"] == "bf16" else MX_ROW
    per_append = 2 * ROW + row + 8 * ROPE // 2 + 16  # kv, the row, cosines and sines, position and slot
    back = row + 2 * ROW + 8 if case["fmt"] == "mxfp8" else 0  # rows handed on as values
    if case["op"] == "append":
        t = case["tokens"]
        b = t * (per_append + back + 2 * h * ROPE * 2) + 2 * LATENT
        return {"bytes": b, "flops": t * (5 * LATENT + 6 * ROPE // 2 * (h + 1))}
    n, seqs = case["n"], case["seqs"]
    mean = case["max_len"] if case["lens"] == "one" else (case["max_len"] + n) / 2
    live = seqs - (seqs // 4 if case["lens"] == "padded" else 0)
    per = (n + 1) / 2 if case["mixed"] else n
    t = seqs * per
    b = live * mean * row + live * mean / case["page"] * 4 + 8 * seqs
    f = live * per * mean * h * 2 * (ROW + LATENT)
    if case["op"] == "attend":
        return {"bytes": b + t * h * 2 * (ROW + LATENT), "flops": f}
    b += t * (per_append + back + h * 2 * (NOPE + ROPE + VDIM)) + h * (NOPE + VDIM) * LATENT * 2 + 2 * LATENT
    return {"bytes": b, "flops": f + t * h * 2 * (NOPE + VDIM) * LATENT}


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
    d = _data(case, seed)
    op, fmt, h, page = case["op"], case["fmt"], case["heads"], case["page"]
    rope = case.get("rope", "interleaved")
    if op != "attend":
        new = _new_rows(d, rope, fmt)
        keep = d["slots"] >= 0
        if fmt == "bf16":
            held = d["cache"].double().view(-1, ROW)
            held[d["slots"][keep]] = new[keep]
            held = held.view(d["cache"].shape)
        else:
            held = torch.where(keep[:, None], new, torch.zeros_like(new))
    if op == "append":
        return _turn(d["q_pe"], d["positions"], d["cos_sin"], rope), held
    lens, table = d["lens"].tolist(), d["table"].long()
    t = d["q_lat" if op == "attend" else "q"].shape[0]
    starts = list(range(0, t + 1, case["n"])) if d["starts"] is None else d["starts"].tolist()
    raw = d["cache"].view(-1, d["cache"].shape[-1])
    if op == "step":
        q = d["q"].double()
        qp = _turn(q[..., NOPE:], d["positions"], d["cos_sin"], rope)
        w = d["kv_b"].double().view(h, NOPE + VDIM, LATENT)
        stored = new.to(BF).double()  # a bf16 row; an MXFP8 row's values fit bf16 as they are
    out = torch.zeros(t, h, LATENT if op == "attend" else VDIM, dtype=F64, device=DEV)
    for i, length in enumerate(lens):
        q0, q1 = starts[i], starts[i + 1]
        if length == 0 or q0 == q1:
            continue
        at = torch.arange(length, device=DEV)
        kv = _exact_rows(raw[table[i, at // page] * page + at % page], fmt)
        cnt = min(q1 - q0, length)
        if op == "step":
            kv[length - cnt :] = stored[q1 - cnt : q1]
        c, pe = kv[:, :LATENT], kv[:, LATENT:]
        for j in range(q1 - cnt, q1):
            m = length - (q1 - 1 - j)
            if op == "attend":
                s = (d["q_lat"][j].double() @ c[:m].T + d["q_pe"][j].double() @ pe[:m].T) * SCALE
                out[j] = torch.softmax(s, -1) @ c[:m]
            else:  # every key and value expanded, as the model defines them
                for hh in range(h):
                    k = c[:m] @ w[hh, :NOPE].T
                    s = (k @ q[j, hh, :NOPE] + pe[:m] @ qp[j, hh]) * SCALE
                    out[j, hh] = torch.softmax(s, -1) @ (c[:m] @ w[hh, NOPE:].T)
    return out if op == "attend" else (out, held)
