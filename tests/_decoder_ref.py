"""Plain 64-bit forms of the decoder operators, and the tolerances of their tests.

Tolerances. Let u be half the spacing of a type at 1 (2^-9 of a value for bf16
after rounding to nearest gives a relative error of at most u = 2^-8, 2^-11 for
f16, 2^-24 for f32). A result in a 2-byte type carries its own rounding (u) and,
in the attention, that of the softmax weights or score gradients which enter the
second product in the same type (u, in a sum of independent terms); h re-read
from storage in the norm's backward carries one more. So 2-norms are compared
with 3 u. In float32 the products' sums (up to a few thousand terms, error
growing as their root) and the scores in the exponent (|s| up to about 16, each
with a relative error of some u times the root of dim) dominate: 2e-5 covers
16 * 2^-24 * sqrt(256) = 1.5e-5. Single elements may be off by 8 times that of
max(|element|, root mean square): the largest of some 10^5 normal deviates is
below 6 standard deviations.
"""

from __future__ import annotations

import torch

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2e-5 / 3}


def close(got: torch.Tensor, want: torch.Tensor, dtype: torch.dtype | None = None, what: str = "") -> None:
    dtype = dtype or got.dtype
    tol = 3 * U[dtype]
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if got.numel() == 0:
        return
    g, w = got.double().cpu(), want.double().cpu()
    assert torch.equal(torch.isnan(g), torch.isnan(w)), what + ": NaN in other places"
    assert torch.equal(torch.isinf(g), torch.isinf(w)), what + ": infinities in other places"
    fine = torch.isfinite(w)
    g, w = g[fine], w[fine]
    if w.numel() == 0:
        return
    norm = w.norm().item()
    off = (g - w).norm().item()
    assert off <= tol * norm + 1e-30, f"{what}: relative error {off / max(norm, 1e-300):.3g} > {tol:.3g}"
    rms = norm / w.numel() ** 0.5
    worst = ((g - w).abs() / torch.maximum(w.abs(), torch.full_like(w, rms + 1e-300))).max().item()
    assert worst <= 8 * tol, f"{what}: an element is {worst:.3g} off, > {8 * tol:.3g}"


def attention(q, k, v, ql, kl, scale, mask=None):
    """Packed cross attention in 64 bits, differentiable. Masked keys take no part at all."""

    group = q.size(1) // k.size(1)
    out = []
    qa = ka = 0
    for t, s in zip(ql, kl):
        qs = q[qa:qa + t]
        idx = torch.arange(ka, ka + s, device=q.device)
        if mask is not None:
            idx = idx[mask[idx]]
        qa, ka = qa + t, ka + s
        if idx.numel() == 0:
            out.append(torch.zeros_like(qs))
            continue
        ks, vs = k[idx].repeat_interleave(group, 1), v[idx].repeat_interleave(group, 1)
        p = torch.softmax(torch.einsum("thd,shd->hts", qs, ks) * scale, -1)
        out.append(torch.einsum("hts,shd->thd", p, vs))
    return torch.cat(out) if out else q * 0


def norm(x, weight, residual, eps):
    h = x if residual is None else x + residual
    return h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * weight, h


def dequantize(codes, scales, zeros, group):
    c = torch.stack((codes & 15, codes >> 4), -1).reshape(codes.size(0), -1).double()
    z = torch.full_like(scales, 8).double() if zeros is None else zeros.double()
    return (c - z.repeat_interleave(group, 1)) * scales.double().repeat_interleave(group, 1)
