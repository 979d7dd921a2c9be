"""Plain 64-bit attention of a prompt's tokens for the tests of ``sgl_amd_mono.moe.latent_prompt``, and the
error bounds that the kernels' roundings allow (a rounding: 2^-8 of the value in bf16, 2^-24 in fp32)."""

import torch

import latent_ref as ref

U16, U32 = ref.U16, ref.U32
F64 = torch.float64


def attend(cache, kv_b, q_nope, q_pe, table, lens, starts, scale):
    """-> (out fp64 [T, h, 128], lse [T, h], bound on out's error, bound on lse's).

    A key's value is an fp32 sum of 512 products, rounded to bf16: off by dk = 2^-8 |k| + 514 2^-24 sum |w c|;
    a value's, dv, likewise. A score is an fp32 sum of 192 products of such keys: off by
    ds = scale (sum |q| dk + 196 2^-24 sum |q| (|k| + dk)) + 2^-21 |s|, its numerator by a factor d = exp(2 ds) - 1,
    2^-21 for the exponential and 2^-8 for its bf16 rounding (the sum takes the unrounded one); the sums of up to
    len terms add len 2^-24 each, joined parts 2^-21, the output's rounding 2^-8 and what bf16's smallest
    normal value leaves."""
    t, h, _ = q_nope.shape
    dev = q_nope.device
    w = kv_b.double().view(h, 2, 128, 512)
    out = torch.zeros(t, h, 128, dtype=F64, device=dev)
    lse = torch.full((t, h), -float("inf"), dtype=F64, device=dev)
    bound, lbound = torch.zeros_like(out), torch.zeros_like(lse)
    for b, length in enumerate(lens):
        n = starts[b + 1] - starts[b]
        if n <= 0 or length <= 0:
            continue
        rows = ref.row_values(ref.sequence_rows(cache, table, b, length))
        c, pe = rows[:, :512], rows[:, 512:]
        see = torch.arange(length, device=dev)[None] <= (length - n + torch.arange(n, device=dev))[:, None]
        some = see.any(1)
        z = slice(starts[b], starts[b + 1])
        for hh in range(h):
            k, v = c @ w[hh, 0].T, c @ w[hh, 1].T
            fine = 514 * U32 * (c.abs() @ w[hh].abs().transpose(1, 2))
            dk, dv = U16 * k.abs() + fine[0], U16 * v.abs() + fine[1]
            qn, qp = q_nope[z, hh].double(), q_pe[z, hh].double()
            s = (qn @ k.T + qp @ pe.T) * scale
            size = qn.abs() @ (k.abs() + dk).T + qp.abs() @ pe.abs().T
            ds = abs(scale) * (qn.abs() @ dk.T + 196 * U32 * size) + 2.0**-21 * s.abs()
            s = s.masked_fill(~see, -float("inf"))
            top = s.amax(1, keepdim=True).clamp_min(-1e300)
            p = torch.where(see, torch.exp(s - top), torch.zeros_like(s))
            total = p.sum(1, keepdim=True).clamp_min(1e-300)
            p = p / total
            o = p @ v
            d = torch.expm1(2 * ds) + 2.0**-21 + length * U32
            d = torch.where(see, d, torch.zeros_like(d))
            err = (p * (d + U16)) @ (v.abs() + dv) + p @ dv + (p * d).sum(1, keepdim=True) * (o.abs() + p @ dv)
            out[z, hh] = o
            bound[z, hh] = err * (1 + U16) + U16 * o.abs() + 2.0**-126
            lse[z, hh] = torch.where(some, (top + torch.log(total))[:, 0], lse[z, hh])
            lbound[z, hh] = torch.log1p((p * d).sum(1)) + 4 * U32 * lse[z, hh].abs().clamp_max(1e300) + 2.0**-20
    return out, lse, bound, lbound


def close(got, want, bound, what="out", sigma=1.0):
    """Every value within its bound, and the whole within what independent roundings make: u = 2^-8 / sqrt 3 of it
    each for the output's, its numerators' and its values', and for the keys', which move a score by u times the
    scores' own standard deviation sigma and the output by as much of it: u sqrt(3 + sigma^2) together (2 u at
    sigma 1: queries and keys of values near 1 have sigma = |scale| sqrt 192)."""
    ref.assert_within(got, want, bound, what)
    rel = ((got.double() - want).norm() / want.norm().clamp_min(1e-300)).item()
    assert rel <= U16 / 3**0.5 * (3 + sigma**2) ** 0.5, (what, rel)
