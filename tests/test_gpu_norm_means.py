"""LayerNorm of rows whose mean is large beside their deviation, constant rows the extreme: the mean is removed to the last bit
that the row's own values have.

A constant row's result is 0 exactly.  A float32 sum of C equal values v lies k steps of v's from C v, its mean therefore a few
steps from v, and v minus that is exact (the two are within a factor of two).  Those differences are the same small whole
number of steps in every channel, so their own sum is exact, its C-th part is the difference, and subtracting it leaves 0."""

import pytest
import torch

from tests import block_plain as P
from tests.gpu_util import require_gpu

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
VALUES = (171.0, 241.0, -2736.0, 10944.0, 0.0, 3.0)
# narrow rows, one to eight waves a row, wide rows; 1 / C rounded moves the mean of one of VALUES in 896, 3584 and 7040
WIDTHS = (1, 24, 65, 200, 260, 896, 1027, 3584, 5120, 7040, 8200, 13824, 20480, 20608, 40001)


def _constant(L, C, dtype):
    v = torch.tensor(VALUES, device="cuda")
    v = v.repeat(-(-L // len(VALUES)))[:L]
    if dtype is FP32:
        v = v / 3 + 1e-3
    return v.to(dtype)[None, :, None].expand(1, L, C).contiguous()


def _zero(t):
    return not t.any().item()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("C", WIDTHS)
def test_constant_rows(C, dtype):
    require_gpu()
    from telefuser_amd.norm import block_norm, gated_residual, gated_residual_norm

    x = _constant(len(VALUES), C, dtype)
    shift = torch.randn(C, generator=torch.Generator(device="cuda").manual_seed(C), device="cuda")
    assert _zero(block_norm(x))
    assert torch.equal(block_norm(x, shift + 2, shift=shift, scale=shift), shift.to(dtype).expand_as(x))
    rows = block_norm(x, shift, out_dtype=torch.int8)
    assert _zero(rows.scale) and _zero(rows.codes)
    h, z = gated_residual_norm(x, x, shift, post_norm="layer", post_weight=shift)
    assert torch.equal(h, x) and _zero(z)
    assert torch.equal(gated_residual(x, x, post_norm="layer"), x)
    h, z = gated_residual_norm(x, x.flip(1), residual_scale=0.5)  # the sum is what is constant
    assert _zero(z)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("C", [896, 2565, 3584, 7040])
def test_constant_rows_of_long_sequences(C, dtype):
    require_gpu()
    from telefuser_amd.norm import block_norm, gated_residual_norm

    x = _constant(16384 + 7, C, dtype)
    weight = torch.randn(C, generator=torch.Generator(device="cuda").manual_seed(C), device="cuda")
    assert _zero(block_norm(x, weight))
    rows = block_norm(x, weight, out_dtype=torch.int8)
    assert _zero(rows.scale) and _zero(rows.codes)
    h, z = gated_residual_norm(x, x, weight, post_norm="layer", post_weight=weight)
    assert torch.equal(h, x) and _zero(z)


@pytest.mark.parametrize("L,C", [(5, 65), (5, 200), (5, 896), (5, 1536), (5, 5120), (5, 13824), (5, 20608), (16384, 65),
                                 (16384, 200), (16384, 896), (16384, 1536), (16384, 5120)])
def test_small_deviation_beside_the_mean(L, C):
    """Float32 rows 1000 +- 0.01: their values minus a mean that lies within a few steps of 1000 are exact, so the result
    carries only the roundings of the deviations' own sums, relative to the deviations."""
    require_gpu()
    from telefuser_amd.norm import block_norm, gated_residual

    g = torch.Generator(device="cuda").manual_seed(C)
    x = 1000 + 0.01 * torch.randn((1, L, C), generator=g, device="cuda")
    weight = torch.ones(C, device="cuda")
    z, p = block_norm(x, weight), gated_residual(torch.zeros_like(x), x, post_norm="layer", post_weight=weight)
    at = torch.cat([torch.arange(0, min(L, 50)), torch.arange(max(0, L - 50), L)]).cuda()
    d = x[:, at].double()
    d = d - d.mean(-1, keepdim=True)
    ref = d / torch.sqrt(d.square().mean(-1, keepdim=True) + 1e-6)
    # (C / 64 + 26) roundings of a deviation, of the deviations' mean and, relative to z, of the deviation's root; the first
    # mean is up to (C / 64 + 26) 2^-24 1000 off, which the deviations carry until it is removed: m of their size
    k = (C / 64 + P.SLACK) * P.U32
    m = k * 1000 / 0.01
    tol = k * (1 + m) * (2 + 3 * ref.abs() * (1 + m)) + P.half_step(FP32, ref)
    assert ((z[:, at].double() - ref).abs() <= tol).all()
    assert ((p[:, at].double() - ref).abs() <= tol).all()
