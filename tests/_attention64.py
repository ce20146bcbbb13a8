"""Attention of one request in 64 bits, with how far a kernel's result may be off.

A kernel's scores are f32 sums of d products of 16-bit values, each off by at most d 2^-24 of the sum of magnitudes; its weights
are off by that (times ln 2 a unit of the log2 domain), by 2e-6 for the exponential and, rounded to the element type for the value
product, by half a step, or in f16 by half the smallest step, 2^-25, beside a largest weight of at least 1; the sum of the weights is
not rounded, the result is, once.  Weighted sums in f32 add n 2^-24 of their magnitude."""

import math

import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def attend(q, k, v, scale, seen=None):
    """``q`` (rows, heads, d), ``k`` / ``v`` (keys, kv heads, d), ``seen`` (rows, keys) truth values or None ->
    ``(out, lse, tolerance of out, tolerance of lse)``; a row without keys: zeros and -inf."""
    rows, heads, d = q.shape
    keys, kv = k.shape[:2]
    half = HALF_STEP[q.dtype]
    if keys == 0 or rows == 0:
        out, lse = torch.zeros(rows, heads, d, dtype=torch.float64, device=q.device), torch.full((rows, heads), -math.inf, dtype=torch.float64, device=q.device)
        return out, lse, torch.zeros_like(out), torch.zeros_like(lse)
    if seen is None:
        seen = torch.ones(rows, keys, dtype=torch.bool, device=q.device)
    q64 = q.double().reshape(rows, kv, heads // kv, d).permute(1, 2, 0, 3).reshape(kv, -1, d)
    k64, v64 = k.double().permute(1, 2, 0).contiguous(), v.double().transpose(0, 1).contiguous()
    mask = seen[None].expand(heads // kv, rows, keys).reshape(1, -1, keys)
    live = seen.any(-1)[None].expand(heads // kv, rows).reshape(-1)
    logits = torch.bmm(q64, k64) * scale
    size = (torch.bmm(q64.abs(), k64.abs()) * abs(scale)).masked_fill(~mask, 0).amax(-1, keepdim=True)
    off = d * 2.0 ** -24 * size                                   # of a logit, natural units
    logits = logits.masked_fill(~mask, -math.inf)
    lse = torch.logsumexp(logits, -1, keepdim=True)
    w = torch.where(mask & (logits != -math.inf), torch.exp(logits - lse), torch.zeros_like(logits))
    # (a value that is not finite: the rows that see its key, by what it is; others by the finite values)
    clean = torch.where(v64.isfinite(), v64, torch.zeros_like(v64))
    out = torch.bmm(w, clean)
    sees = mask.double().expand(kv, -1, -1).contiguous()
    for flag, value in ((v64 == math.inf, math.inf), (v64 == -math.inf, -math.inf), (v64.isnan(), math.nan)):
        if bool(flag.any()):
            out = torch.where(torch.bmm(sees, flag.double()) > 0, out + value, out)
    out = torch.where(w.isnan().any(-1, keepdim=True), torch.full_like(out, math.nan), out)
    spread = torch.bmm(w.nan_to_num(0), clean.abs())
    rel = half + 2 * off + 4e-6 + keys * 2.0 ** -24
    tiny = (2.0 ** -25 * keys if q.dtype == torch.float16 else 0.0) * clean.abs().amax()
    tol = rel * spread + tiny
    tol = tol + half * (out.abs() + tol) + (2.0 ** -25 if q.dtype == torch.float16 else 0.0)
    lse2 = lse[..., 0] / math.log(2.0)
    lse_tol = (off[..., 0] + 4e-6 + keys * 2.0 ** -24) / math.log(2.0) + lse2.abs().nan_to_num(0, posinf=0, neginf=0) * 2.0 ** -22

    def back(x):
        return x.reshape(kv, heads // kv, rows, -1).permute(2, 0, 1, 3).reshape(rows, heads, -1)

    out = torch.where(live[None, :, None], out, torch.zeros_like(out))
    return back(out), back(lse2[..., None])[..., 0], back(tol), back(lse_tol[..., None])[..., 0]


def same(got, want, tol, what):
    """``got`` within ``tol`` of ``want``; undefined and infinite elements at the same places."""
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf()), f"{what}: infinite or undefined elsewhere"
    finite = want.isfinite()
    assert torch.equal(got[want.isinf()] > 0, want[want.isinf()] > 0), f"{what}: an infinite value's sign"
    worst = ((got - want).abs() / tol.clamp_min(1e-30))[finite]
    assert worst.numel() == 0 or float(worst.max()) <= 1.0, f"{what}: off by {float(worst.max()):.2f} times the tolerance"
