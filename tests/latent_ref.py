"""Plain 64-bit latent attention for the tests of ``sgl_amd_mono.moe.latent``, and the error bounds
that the kernels' roundings allow.

A rounding is off by at most half a step: 2^-8 of the value in bf16, 2^-24 in fp32, 2^-4 in e4m3
(2^-10 of the scale below e4m3's normal range)."""

import torch

L, R, ROW, MX_ROW = 512, 64, 576, 656
U16, U32 = 2.0**-8, 2.0**-24
BF, F64 = torch.bfloat16, torch.float64


def e4m3_values(codes):
    """The values of e4m3 codes (uint8), fp64; NaN for 0x7f and 0xff."""
    c = codes.to(torch.int64)
    e, m = (c >> 3) & 15, (c & 7).to(F64)
    v = torch.where(e > 0, torch.exp2(e.to(F64) - 7) * (1 + m / 8), m * 2.0**-9)
    v = torch.where((c & 127) == 127, torch.full_like(v, float("nan")), v)
    return torch.where(c >= 128, -v, v)


def row_values(rows):
    """Cache rows [n, 576] bf16 or [n, 656] uint8 -> their values [n, 576] fp64."""
    if rows.dtype == BF:
        return rows.to(F64)
    v = e4m3_values(rows[:, :L]) * torch.exp2(rows[:, L : L + 16].to(F64) - 127).repeat_interleave(32, 1)
    pe = rows[:, L + 16 :].contiguous().view(BF).to(F64)
    return torch.cat([v, pe], 1)


def random_cache(pages, page, fmt, gen, device):
    """Rows of values near 1 in every place; MXFP8: random codes (no NaN), scales near 2^-8."""
    if fmt == "bf16":
        return torch.randn(pages, page, ROW, generator=gen, device=device).to(BF)
    c = torch.empty(pages, page, MX_ROW, dtype=torch.uint8, device=device)
    # codes of magnitude up to 448, their scales 2^-8 or 2^-7: values near 1
    mag = torch.randint(40, 127, (pages, page, L), generator=gen, device=device)
    sign = torch.randint(0, 2, (pages, page, L), generator=gen, device=device) * 128
    c[..., :L] = (mag + sign).to(torch.uint8)
    c[..., L : L + 16] = torch.randint(119, 121, (pages, page, 16), generator=gen, device=device).to(torch.uint8)
    pe = torch.randn(pages, page, R, generator=gen, device=device).to(BF)
    c[..., L + 16 :] = pe.view(torch.uint8)
    return c


def sequence_rows(cache, table, b, length):
    page = cache.shape[1]
    at = torch.arange(length, device=cache.device)
    flat = cache.view(-1, cache.shape[-1])
    return flat[table[b].long()[at // page] * page + at % page]


def attend(cache, q_lat, q_pe, table, lens, scale, starts=None):
    """-> (out fp64 [T, h, 512], lse fp64 [T, h], bound on |out|'s error, bound on lse's).

    The kernel's scores are fp32 sums of exact products of bf16 values (any order, 576 terms), times
    a scale, so they are off by at most ds = (576 + 4) 2^-24 scale sum |q k|, with 2^-22 |s| for
    the scale's and the exponent's roundings; a numerator exp(s - max) is then off by a factor
    exp(2 ds') of itself (the maximum's error cancels between numerator and sum), 2^-22 for the
    exponential, and 2^-8 for its bf16 rounding, which the sum does not have. Sums of up to len
    fp32 terms add len 2^-24; the output's own rounding is 2^-8."""
    t, h, _ = q_lat.shape
    dev = q_lat.device
    out = torch.zeros(t, h, L, dtype=F64, device=dev)
    lse = torch.full((t, h), -float("inf"), dtype=F64, device=dev)
    bound, lbound = torch.zeros_like(out), torch.zeros_like(lse)
    seqs = len(lens)
    if starts is None:
        starts = [i * (t // seqs) for i in range(seqs + 1)]
    for b, length in enumerate(lens):
        n = starts[b + 1] - starts[b]
        kv = row_values(sequence_rows(cache, table, b, length))
        for i in range(n):
            m = length - n + 1 + i
            if m <= 0:
                continue
            j = starts[b] + i
            q = torch.cat([q_lat[j], q_pe[j]], 1).to(F64)
            s = q @ kv[:m].T * scale
            p = torch.softmax(s, -1)
            out[j] = p @ kv[:m, :L]
            lse[j] = torch.logsumexp(s, -1)
            ds = 580 * U32 * abs(scale) * (q.abs() @ kv[:m].abs().T).amax(-1) + 2.0**-22 * (s.abs().amax(-1) + 1)
            a = p @ kv[:m, :L].abs()
            rel = (torch.expm1(2 * ds) * 2 + m * U32 * 2 + 2.0**-20)[:, None]
            bound[j] = (U16 + rel) * a * 1.01 + U16 * (1 + U16) * out[j].abs() + 1e-30
            lbound[j] = 2 * ds + m * U32 + 2.0**-21 * (lse[j].abs() + 1)
    return out, lse, bound, lbound


def rotate(x, cs, half):
    """x [..., 64] fp64 by the rows cs [..., 64] -> (values, sum of the two products' sizes)."""
    c, s = cs[..., :32].to(F64), cs[..., 32:].to(F64)
    if half:
        a, b = x[..., :32], x[..., 32:]
        join = lambda u, v: torch.cat([u, v], -1)  # noqa: E731
    else:
        a, b = x[..., ::2], x[..., 1::2]
        join = lambda u, v: torch.stack([u, v], -1).flatten(-2)  # noqa: E731
    return join(a * c - b * s, b * c + a * s), join((a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs())


def norm(c, w, eps):
    c = c.to(F64)
    return c if w is None else c * torch.rsqrt((c * c).mean(-1, keepdim=True) + eps) * w.to(F64)


def assert_within(got, ref, bound, what):
    got = got.to(F64)
    bad = ~((got - ref).abs() <= bound) & ~(torch.isnan(got) & torch.isnan(ref)) & ~(got == ref)
    if bool(bad.any()):
        at = bad.nonzero()[0].tolist()
        i = tuple(at)
        raise AssertionError(
            f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds, first at {at}: {got[i].item()} for "
            f"{ref[i].item()}, bound {bound[i].item() if bound.shape == got.shape else bound}"
        )
