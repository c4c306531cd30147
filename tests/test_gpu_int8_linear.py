"""int8_linear and Int8Weight against float64 products of the same codes."""

import pytest
import torch

from tests import block_plain as P
from tests.gpu_util import log, require_gpu

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _x(shape, seed, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _weight(n, k, seed, bias=True):
    g = torch.Generator(device="cuda").manual_seed(seed + 5)
    codes = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    scale = (torch.rand(n, generator=g, device="cuda") + 0.5) / (73 * k ** 0.5)
    return codes, scale, torch.randn(n, generator=g, device="cuda") if bias else None


def _check(x, w, act, out, what):
    codes, scale = P.codes_of(x)
    ref, err = P.linear(codes, scale.float(), *w, act)
    P.check(out, ref, err, what)


SIZES = [(1, 1, 1), (1, 128, 3), (1, 1536, 1536), (2, 129, 33), (3, 64, 5120), (5, 4096, 64), (8, 640, 200), (15, 1027, 129),
         (16, 256, 17), (17, 128, 64), (31, 300, 100), (33, 127, 65), (64, 512, 96), (65, 256, 128), (100, 2048, 129), (127, 128, 999),
         (128, 1536, 256), (129, 256, 513), (200, 8960, 96), (255, 384, 257), (256, 128, 256), (257, 1024, 640),
         (300, 1027, 999), (600, 128, 1100), (1024, 512, 513), (1560, 640, 1536), (2049, 256, 1025),
         (1300, 2000, 1537), (2500, 13824, 640), (3000, 300, 3001), (9000, 200, 4000)]


@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_linear(M, K, N, dtype):
    require_gpu()
    from telefuser_amd.linear import Int8Weight, int8_linear

    x = _x((M, K), M + K + N, dtype)
    w = _weight(N, K, N)
    weight = Int8Weight(*w)
    for act in (None, "gelu_tanh", "silu"):
        out = int8_linear(x, weight, act=act)
        assert out.dtype == dtype and out.shape == (M, N)
        if dtype is FP32:  # a float32 value may take the other of two equally near codes: compare from the codes
            from telefuser_amd.norm import per_token_int8

            rows = per_token_int8(x)
            ref, err = P.linear(rows.codes[:, :K], rows.scale, *w, act)
            P.check(out, ref, err, f"{act}")
        else:
            _check(x, w, act, out, f"{act}")
    out = int8_linear(x, Int8Weight(w[0], w[1]), out_dtype=FP32)
    if dtype is not FP32:
        _check(x, (w[0], w[1], None), None, out, "without bias, float32")


@pytest.mark.parametrize("M", [1, 3, 16, 40, 130, 700])
def test_sums_are_exact(M):
    """The largest sums: every code 127 over the longest K, scale 1."""
    require_gpu()
    from telefuser_amd.linear import Int8Rows, Int8Weight, int8_linear

    K = 131072
    ones = torch.full((M, K), 127, dtype=torch.int8, device="cuda")
    w = torch.full((3, K), 127, dtype=torch.int8, device="cuda")
    w[1] = -127
    w[2, ::2] = -128
    rows = Int8Rows(ones, torch.ones(M, device="cuda"), K)
    out = int8_linear(rows, Int8Weight(w, torch.ones(3, device="cuda")), out_dtype=FP32)
    want = torch.tensor([127 * 127 * K, -127 * 127 * K, 127 * (127 - 128) * K // 2], dtype=torch.float64)
    assert torch.equal(out.cpu(), want.float().expand(M, 3))


@pytest.mark.parametrize("M,N", [(1, 200), (7, 64), (70, 300), (300, 520)])
def test_rows_without_a_value(M, N):
    """Rows of zeros give the bias, rows with NaN or infinity give NaN, and leave their neighbours alone."""
    require_gpu()
    from telefuser_amd.linear import Int8Weight, int8_linear

    K = 256
    x = _x((M, K), 3, BF16)
    w = _weight(N, K, 4)
    weight = Int8Weight(*w)
    good = int8_linear(x, weight)
    y = x.clone()
    y[M // 2] = 0
    out = int8_linear(y, weight)
    assert torch.equal(out[M // 2], w[2].to(BF16))
    keep = torch.arange(M, device="cuda") != M // 2
    assert torch.equal(out[keep], good[keep])
    for v in (float("nan"), float("inf"), float("-inf")):
        y = x.clone()
        y[M // 2, 7] = v
        for act in (None, "silu"):
            out = int8_linear(y, weight, act=act)
            assert torch.isnan(out[M // 2]).all()
            assert torch.equal(out[keep], int8_linear(x, weight, act=act)[keep])


def test_shapes_strides_and_quantized_weights():
    require_gpu()
    from telefuser_amd.linear import Int8Weight, int8_linear
    from telefuser_amd.norm import block_norm, per_token_int8

    w = _x((96, 200), 1, BF16) * 0.1
    weight = Int8Weight.quantize(w, _x((96,), 2, BF16))
    assert (weight.in_features, weight.out_features) == (200, 96)
    codes, scale = P.codes_of(w)
    assert torch.equal(weight.codes[:, :200].double(), codes) and torch.equal(weight.scale, scale.float())
    big = _x((2, 40, 440), 3, BF16)
    for v in (big[:, :30, :200], big[:, :, 1:201], big[:, :, 0:400:2], big.transpose(0, 1)[:, :, :200], big[0, ::3, 8:208]):
        out = int8_linear(v, weight, act="silu")
        assert out.shape == (*v.shape[:-1], 96)
        assert torch.equal(out, int8_linear(v.contiguous(), weight, act="silu"))
        assert torch.equal(out, int8_linear(per_token_int8(v), weight, act="silu"))
    rows = block_norm(big[:, :, :200], out_dtype=torch.int8)
    ref, err = P.linear(rows.codes[..., :200], rows.scale, weight.codes[:, :200], weight.scale, weight.bias, None)
    P.check(int8_linear(rows, weight), ref, err, "norm to rows")
    for shape in ((0, 200), (2, 0, 200)):
        assert int8_linear(torch.empty(shape, dtype=BF16, device="cuda"), weight).shape == (*shape[:-1], 96)
    strided = Int8Weight(torch.cat([codes, codes], 1).to(torch.int8)[:, :200], scale[:, None], None)
    assert torch.equal(strided.codes, weight.codes)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("B,L,K", [(1, 1, 1), (1, 1, 16384), (1, 16, 1024), (2, 8, 1000), (4, 4, 1024), (3, 5, 130),
                                   (1, 7, 2049), (5, 1, 3200), (1, 17, 100), (1, 9, 1920)])
def test_few_tokens_quantized_on_the_way(B, L, K, dtype):
    """A floating x of few values (and just more than a few) gives the bits of its INT8 rows, whatever its strides."""
    require_gpu()
    from telefuser_amd.linear import Int8Weight, int8_linear
    from telefuser_amd.norm import per_token_int8

    weight = Int8Weight(*_weight(100, K, 2))
    big = _x((B + 1, L + 2, K + 9), K, dtype)
    big[0, 0, 0] = float("inf")
    for v in (big[1:, :L, :K], big[1:, 1:L + 1, 3:K + 3], big[1:, 2:, 8:K + 8].clone(), big.transpose(0, 1)[1:L + 1, 1:, :K]):
        for act in (None, "silu"):
            assert torch.equal(int8_linear(v, weight, act=act), int8_linear(per_token_int8(v), weight, act=act,
                                                                            out_dtype=dtype))
    zero = torch.zeros((B, L, K), dtype=dtype, device="cuda")
    zero[0, 0, K // 2] = float("nan")
    out = int8_linear(zero, weight, out_dtype=FP32)
    assert torch.isnan(out[0, 0]).all()
    assert torch.equal(out.reshape(B * L, -1)[1:], weight.bias.expand(B * L - 1, -1))


def test_offsets_past_32_bits():
    require_gpu()
    from telefuser_amd.linear import Int8Rows, Int8Weight, int8_linear

    M, N, K = 140000, 16500, 128  # 2.3e9 outputs
    g = torch.Generator(device="cuda").manual_seed(1)
    codes = torch.randint(-127, 128, (M, K), generator=g, device="cuda", dtype=torch.int8)
    rows = Int8Rows(codes, torch.rand(M, generator=g, device="cuda"), K)
    w = _weight(N, K, 2)
    out = int8_linear(rows, Int8Weight(*w))
    for part in (slice(0, 300), slice(130000, 130300), slice(M - 300, M)):
        ref, err = P.linear(codes[part], rows.scale[part], *w, None)
        P.check(out[part], ref, err, f"{part}")
    del out
    M, K = 20000, 131072  # 2.6e9 codes
    codes = torch.ones((M, K), dtype=torch.int8, device="cuda")
    codes[-1] = 3
    out = int8_linear(Int8Rows(codes, torch.ones(M, device="cuda"), K),
                      Int8Weight(torch.ones((40, K), dtype=torch.int8, device="cuda"), torch.ones(40, device="cuda")),
                      out_dtype=FP32)
    assert (out[:-1] == K).all() and (out[-1] == 3 * K).all()
    log("offsets past 32 bits: done")


@pytest.mark.parametrize("M,K,N", [(1, 1536, 640), (12, 2048, 96), (100, 4096, 256), (1560, 640, 1536)])
def test_repeats_bit_for_bit_on_another_stream_and_in_graphs(M, K, N):
    require_gpu()
    from telefuser_amd.linear import Int8Weight, int8_linear

    x, x2 = _x((M, K), 1, BF16), _x((M, K), 2, BF16)
    weight = Int8Weight(*_weight(N, K, 3))
    out = int8_linear(x, weight, act="gelu_tanh")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):  # two streams at once
        with torch.cuda.stream(side):
            a = int8_linear(x, weight, act="gelu_tanh")
        b = int8_linear(x2, weight, act="gelu_tanh")
    torch.cuda.synchronize()
    assert torch.equal(a, out) and torch.equal(b, int8_linear(x2, weight, act="gelu_tanh"))
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    pool = torch.cuda.graph_pool_handle()
    with torch.cuda.graph(g1, pool=pool):
        o1 = int8_linear(x, weight, act="gelu_tanh")
    with torch.cuda.graph(g2, pool=pool):
        o2 = int8_linear(x2, weight, act="gelu_tanh")
    for seed in (11, 12, 13):
        x.copy_(_x((M, K), seed, BF16))
        x2.copy_(_x((M, K), seed + 50, BF16))
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(o1, int8_linear(x, weight, act="gelu_tanh"))
        assert torch.equal(o2, int8_linear(x2, weight, act="gelu_tanh"))
