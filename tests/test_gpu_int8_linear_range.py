"""int8_linear of activations near the ends of the float range: finite results are finite, and tiny ones keep their bits."""

import pytest
import torch

from tests import block_plain as P
from tests.gpu_util import require_gpu

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


# few tokens (quantized on the way, and from rows), a product split along K, and tiles of the three sizes
@pytest.mark.parametrize("M,K,N", [(1, 1024, 64), (3, 16000, 40), (16, 4096, 9000), (64, 8192, 96), (130, 9000, 129), (300, 1024, 999),
                                   (1560, 1024, 1536), (3000, 1024, 3001)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("size", [1e35, 1e-30])
def test_large_and_tiny_rows(M, K, N, dtype, size):
    require_gpu()
    from telefuser_amd.linear import Int8Weight, int8_linear
    from telefuser_amd.norm import per_token_int8

    g = torch.Generator(device="cuda").manual_seed(M + N)
    x = (torch.rand((M, K), generator=g, device="cuda") * 0.25 + 0.75).mul_(size).to(dtype)  # codes of one sign: large sums
    codes = torch.randint(64, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
    codes[::2] *= -1
    scale = (torch.rand(N, generator=g, device="cuda") + 0.5) * 1e-5
    weight = Int8Weight(codes, scale)
    rows = per_token_int8(x)
    ref, err = P.linear(rows.codes[:, :K], rows.scale, codes, scale, None, None)
    largest = (rows.codes[:, :K].double().sum(-1) * 64 * rows.scale.double()).max()
    assert size < 1 or largest > torch.finfo(FP32).max  # the sum times the row's scale alone leaves the range
    for out in (int8_linear(x, weight), int8_linear(rows, weight, out_dtype=FP32)):
        assert torch.isfinite(out).all()
        P.check(out, ref, err, f"{out.dtype}")
    out = int8_linear(rows, weight, act="silu", out_dtype=FP32)
    if size > 1:  # y or 0, as y is positive or negative
        P.check(out, ref.clamp(min=0), err, "silu")
    big = Int8Weight(codes, scale * 1e18)  # beyond the range: an infinity of the result's sign
    if size > 1:
        out = int8_linear(rows, big, out_dtype=FP32)
        ref = ref * 1e18
        over = ref.abs() > 2 * torch.finfo(FP32).max
        assert over.any() and torch.equal(out[over], torch.sign(ref[over]).float() * float("inf"))
