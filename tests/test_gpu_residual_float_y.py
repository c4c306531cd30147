"""gated_residual and gated_residual_norm of a float32 y beside a half x: what int8_linear(..., out_dtype=torch.float32) gives
reaches the sum unrounded."""

import pytest
import torch

from tests import block_plain as P
from tests.gpu_util import require_gpu

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _rand(shape, seed, dtype=FP32, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


# narrow rows of 8, 16 and 32 lanes, one to eight waves a row, a wide row; dividing into nothing
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("B,L,C", [(1, 1, 1), (2, 3, 65), (1, 5, 200), (3, 7, 520), (2, 33, 1027), (1, 9, 1536), (2, 2, 5120),
                                   (1, 2, 8200), (1, 2, 13824), (1, 1, 20481)])
@pytest.mark.parametrize("post", [None, "layer", "rms"])
def test_float_y_beside_a_half_x(B, L, C, dtype, post):
    require_gpu()
    from telefuser_amd.norm import gated_residual, gated_residual_norm

    x, y = _rand((B, L, C), C, dtype), _rand((B, L, C), C + 1)
    gate, scale, shift = (_rand((B, 1, C), i, std=0.3) for i in range(3))
    how = {} if post is None else {"post_norm": post, "post_weight": _rand((C,), 5) + 1, "post_bias": _rand((C,), 6)}
    h, z = gated_residual_norm(x, y, gate, scale=scale, shift=shift, **how)
    assert h.dtype == dtype and z.dtype == dtype
    rh, eh, rz, ez = P.block(x, y, gate, scale=scale, shift=shift, **how)
    P.check(h, rh, eh, "h")
    P.check(z, rz, ez, "z")
    rows = gated_residual_norm(x, y, gate, scale=scale, shift=shift, out_dtype=torch.int8, **how)[1]
    P.check_rows(rows, rz, ez, "int8 z")
    assert torch.equal(gated_residual(x, y, gate, **how), h)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("L,C", [(16384, 260), (16390, 1536), (16400, 2565), (17000, 5120), (16400, 8192)])
def test_long_sequences(L, C, dtype):
    require_gpu()
    from telefuser_amd.norm import gated_residual_norm

    x, y = _rand((1, L, C), C, dtype), _rand((1, L, C), C + 1)
    gate, scale, shift = (_rand((C,), i, std=0.3) for i in range(3))
    at = torch.cat([torch.arange(0, 40), torch.arange(L - 40, L)]).cuda()
    for how in ({}, {"post_norm": "rms", "post_weight": gate + 1}):
        h, z = gated_residual_norm(x, y, gate, scale=scale, shift=shift, **how)
        rh, eh, rz, ez = P.block(x[:, at], y[:, at], gate, scale=scale, shift=shift, **how)
        P.check(h[:, at], rh, eh, "h")
        P.check(z[:, at], rz, ez, "z")
        # every row is written, once: the sum of each against that of the plain form, both of rounded values
        ref = x.float() + (P.norm(how.get("post_norm"), y.double(), 0, 1e-6)[0].float() * (gate + 1) if how else y) * gate
        assert ((h.float().sum(-1) - ref.sum(-1)).abs() <= (ref.abs() * torch.finfo(dtype).eps + 1e-5).sum(-1)).all()


def test_strides_of_a_float_y():
    require_gpu()
    from telefuser_amd.norm import gated_residual_norm

    x, big = _rand((2, 6, 1536), 1, BF16), _rand((2, 9, 3100), 2)
    for y in (big[:, 1:7, :1536], big[:, :6, 1:1537], big[:, 2:8, 3:3075:2], big[:1, :6, 8:1544].expand(2, 6, 1536)):
        h, z = gated_residual_norm(x, y, norm="rms")
        rh, eh, rz, ez = P.block(x, y, norm_kind="rms")
        P.check(h, rh, eh, "h")
        P.check(z, rz, ez, "z")


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("M,K,C", [(3, 640, 256), (300, 1536, 640)])
def test_product_and_residual_round_once(M, K, C, dtype):
    """h and z of a product that cancels against x: a rounding of the product alone would be seen."""
    require_gpu()
    from telefuser_amd.linear import Int8Weight, int8_linear
    from telefuser_amd.norm import gated_residual_norm, per_token_int8

    u = _rand((M, K), 1, dtype)
    weight = Int8Weight.quantize(_rand((C, K), 2, std=K ** -0.5), _rand((C,), 3, std=0.1))
    rows = per_token_int8(u)
    ref, err = P.linear(rows.codes[:, :K], rows.scale, weight.codes[:, :K], weight.scale, weight.bias, None)
    x = (-1.01 * ref).to(dtype)
    y = int8_linear(u, weight, out_dtype=FP32)
    h, z = gated_residual_norm(x, y, norm="rms")
    rh, eh, rz, ez = P.block(x, ref, norm_kind="rms")
    # z = h / sqrt(mean(h^2) + eps) is 1 / |h| steep at most in each of its values, the row's others included
    rstd = 1 / torch.sqrt(rh.square().mean(-1, keepdim=True) + 1e-6)
    P.check(h, rh, eh + err, "h")
    P.check(z, rz, ez + rstd * (err + rz.abs() * err.square().mean(-1, keepdim=True).sqrt()), "z")
    rounded = x.double() + y.to(dtype).double()
    assert ((rounded - rh).abs() > eh + err + P.half_step(dtype, rh.abs() + eh + err)).any()


def test_other_types_are_refused():
    require_gpu()
    from telefuser_amd.norm import gated_residual

    x = _rand((2, 3, 64), 1, BF16)
    for y in (x.to(FP16), x.double()):
        with pytest.raises(ValueError, match="y must"):
            gated_residual(x, y)
    with pytest.raises(ValueError, match="y must"):
        gated_residual(x.to(FP16), x)
