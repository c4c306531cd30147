"""Plain float64 forms of the operators around a DiT block, and how far a float32 evaluation may lie from them.

A tolerance counts roundings: half a step of the output's type relative to the value (finfo.eps / 2), and for the float32
arithmetic before it 2^-24 for each operation, relative to the magnitude of the terms (not of their possibly cancelling
sum).  A sum over C values, accumulated by at least 64 lanes and joined in a tree, takes at most C / 64 + 6 additions on
the longest path; SLACK covers the other operations of an output."""

import math

import torch

U32 = 2.0 ** -24
SLACK = 26


def half_step(dtype, value):
    """Rounding of a value to dtype: half a step relative, half the smallest step near zero."""
    f = torch.finfo(dtype)
    return value.abs() * (f.eps / 2) + f.tiny * f.eps / 2


def norm(kind, v, mag, eps):
    """(n, how large the terms of its error are) for rows v whose own terms have magnitude mag >= |v|."""
    if kind is None:
        return v, mag
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    d = v - mean
    rstd = 1 / torch.sqrt(d.square().mean(-1, keepdim=True) + eps)
    n = d * rstd
    d_err = mag + (mag.mean(-1, keepdim=True) if kind == "layer" else 0)  # error of a centred value, in U32 per step
    # the variance's own error is twice the mean of |d| times the error of d, and that of its sum
    var_err = 2 * (d.abs() * d_err).mean(-1, keepdim=True) * rstd.square()
    return n, d_err * rstd + n.abs() * (2 + var_err)


def affine(n, mag, weight, bias, scale, shift):
    for w in (weight,):
        if w is not None:
            n, mag = n * w.double(), mag * w.double().abs()
    if bias is not None:
        n, mag = n + bias.double(), mag + bias.double().abs()
    if scale is not None:
        s = scale.double()
        n, mag = n * (1 + s), mag * (1 + s.abs())
    if shift is not None:
        n, mag = n + shift.double(), mag + shift.double().abs()
    return n, mag


def block(x, y=None, gate=None, residual_scale=1.0, post_norm=None, post_weight=None, post_bias=None, post_eps=1e-6,
          weight=None, bias=None, scale=None, shift=None, norm_kind="layer", eps=1e-6):
    """(h, error of h before rounding, z, error of z before rounding), float64."""
    k = (x.shape[-1] / 64 + SLACK) * U32
    h = x.double()
    mag = h.abs()
    if y is not None:
        p = y.double()
        p, pm = norm(post_norm, p, p.abs(), post_eps)
        p, pm = affine(p, pm, post_weight, post_bias, None, None)
        if gate is not None:
            p, pm = p * gate.double(), pm * gate.double().abs()
        h, mag = residual_scale * h + p, abs(residual_scale) * mag + pm
    z, zm = norm(norm_kind, h, mag, eps)
    z, zm = affine(z, zm, weight, bias, scale, shift)
    return h, mag * k, z, zm * k


def check(out, ref, err, what):
    """out against the float64 ref: within err and the rounding of out's type."""
    d = (out.double() - ref).abs()
    tol = err + half_step(out.dtype, ref.abs() + err)
    bad = ~(d <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((d / tol).nan_to_num(9e9).max()):.3g} x the tolerance"


def check_rows(rows, z, err, what):
    """Int8Rows against the float64 z they hold: no value further than half a step (and z's own error) from its code."""
    top = z.abs().amax(-1, keepdim=True)
    terr = err.amax(-1, keepdim=True)
    s = rows.scale.double().unsqueeze(-1)
    assert ((s * 127 - top).abs() <= terr + 2 * U32 * top + 1e-44).all(), f"{what}: scale"
    codes = rows.codes[..., :rows.cols].double()
    assert (codes.abs() <= 127).all()
    d = (codes * s - z).abs()
    tol = s / 2 + err + terr + 8 * U32 * top
    assert (d <= tol).all(), f"{what}: codes, worst {float((d / tol).nan_to_num(9e9).max()):.3g} x the tolerance"
    assert (rows.codes[..., rows.cols:] == 0).all(), f"{what}: the padding is not zero"


def codes_of(x):
    """(codes, scale) of the rows of x in float64 arithmetic."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    return torch.round(127 * x / torch.where(top > 0, top, 1.0)), (top / 127).squeeze(-1)


def linear(rows_codes, rows_scale, codes, scale, bias, act):
    """(out, error before rounding) from INT8 codes [..., K] and [N, K], float64 (integer sums are exact in it)."""
    s = rows_codes.double() @ codes.double().t().contiguous()
    p = s * rows_scale.double().unsqueeze(-1) * scale.double()
    y = p if bias is None else p + bias.double()
    err = U32 * (4 * p.abs() + 2 * y.abs())
    if act in (None, "none"):
        return y, err
    t = y if act == "silu" else 2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)
    out = y * torch.sigmoid(t)
    # exp(-t): its argument carries a few roundings, each an absolute error of |t| U32 in the exponent; the derivative of
    # either activation stays below 1.13
    return out, 1.13 * err + out.abs() * U32 * (16 + 8 * t.abs()) + 1e-30
