"""block_norm, gated_residual, gated_residual_norm and per_token_int8 against their float64 forms."""

import itertools

import pytest
import torch

from tests import block_plain as P
from tests.gpu_util import log, require_gpu

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _x(shape, seed, dtype, offset=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=g, device="cuda")
    c = torch.rand(shape[-1], generator=g, device="cuda")
    return (x * torch.where(c > 0.98, 12.0, 0.4 + c) + offset).to(dtype)


def _p(shape, seed, dtype=FP32, std=0.3):
    g = torch.Generator(device="cuda").manual_seed(seed + 77)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


# lengths and widths at the borders of lanes, vectors and register blocks, dividing into nothing, and one channel
SIZES = [(1, 1, 1), (1, 1, 64), (2, 3, 65), (1, 5, 511), (1, 4, 512), (3, 7, 520), (2, 33, 1027), (1, 9, 1536),
         (1, 3, 2047), (1, 2, 2048), (2, 2, 2056), (1, 3, 5120), (1, 2, 8192), (1, 2, 8200), (1, 2, 13824),
         (1, 2, 16384), (1, 1, 16392), (1, 1, 40001)]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("B,L,C", SIZES)
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_block_norm(B, L, C, dtype, kind):
    require_gpu()
    from telefuser_amd.norm import block_norm

    x = _x((B, L, C), C + L, dtype)
    scale, shift, w, b = _p((B, 1, C), 1), _p((B, 1, C), 2), _p((C,), 3) + 1, _p((C,), 4)
    for how in ({}, {"weight": w}, {"scale": scale, "shift": shift},
                {"weight": w, "bias": b, "scale": scale, "shift": shift}):
        z = block_norm(x, **how, norm=kind)
        assert z.dtype == dtype and z.shape == x.shape
        _, _, ref, err = P.block(x, **how, norm_kind=kind)
        P.check(z, ref, err, f"{kind} {sorted(how)}")
        rows = block_norm(x, **how, norm=kind, out_dtype=torch.int8)
        P.check_rows(rows, ref, err, f"int8 {kind} {sorted(how)}")


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("B,L,C", SIZES)
@pytest.mark.parametrize("post", [None, "layer", "rms"])
def test_gated_residual_norm(B, L, C, dtype, post):
    require_gpu()
    from telefuser_amd.norm import gated_residual, gated_residual_norm

    x, y = _x((B, L, C), C + L, dtype), _x((B, L, C), C + L + 9, dtype)
    gate, scale, shift = _p((B, 1, C), 1), _p((B, 1, C), 2), _p((B, 1, C), 3)
    how = {} if post is None else {"post_norm": post, "post_weight": _p((C,), 5) + 1, "post_bias": _p((C,), 6)}
    h, z = gated_residual_norm(x, y, gate, residual_scale=0.75, scale=scale, shift=shift, **how)
    rh, eh, rz, ez = P.block(x, y, gate, 0.75, scale=scale, shift=shift, **how)
    P.check(h, rh, eh, "h")
    P.check(z, rz, ez, "z")
    h2, rows = gated_residual_norm(x, y, gate, residual_scale=0.75, scale=scale, shift=shift, out_dtype=torch.int8, **how)
    assert torch.equal(h, h2)
    P.check_rows(rows, rz, ez, "int8 z")
    assert torch.equal(gated_residual(x, y, gate, residual_scale=0.75, **how), h)
    rh, eh, _, _ = P.block(x, y, **how)
    P.check(gated_residual(x, y, **how), rh, eh, "h without gate")


@pytest.mark.parametrize("C", [96, 512, 1027, 1536, 5120])
def test_parameter_shapes_and_types(C):
    require_gpu()
    from telefuser_amd.norm import gated_residual_norm

    B, L = 2, 5
    x, y = _x((B, L, C), 1, FP16), _x((B, L, C), 2, FP16)
    shapes = [(C,), (1,), (1, C), (L, C), (L, 1), (B, 1, C), (1, L, C), (B, L, C), (B, L, 1), (B, 1, 1), (1, 1, 1)]
    for i, (a, b) in enumerate(zip(shapes, shapes[3:] + shapes[:3])):
        dt = (FP32, FP16, BF16)[i % 3]
        gate, scale, shift, w = _p(a, 1, dt), _p(b, 2, FP32), _p(a, 3, dt), _p(b, 4, dt)
        h, z = gated_residual_norm(x, y, gate, scale=scale, shift=shift, weight=w, norm="rms", out_dtype=FP32)
        rh, eh, rz, ez = P.block(x, y, gate, scale=scale, shift=shift, weight=w, norm_kind="rms")
        P.check(h, rh, eh, f"h {a} {b}")
        P.check(z, rz, ez, f"z {a} {b}")
    e = _p((B, 6, C), 9)  # the six modulation vectors of a block side by side, as views
    h, z = gated_residual_norm(x, y, e[:, 2:3], scale=e[:, 4:5], shift=e[:, 3:4])
    rh, eh, rz, ez = P.block(x, y, e[:, 2:3], scale=e[:, 4:5], shift=e[:, 3:4])
    P.check(h, rh, eh, "h of views")
    P.check(z, rz, ez, "z of views")
    wide = _p((2, C * 2), 5)[:, 1::2]  # strided channels
    h, z = gated_residual_norm(x[0, :2], y[0, :2], wide, weight=wide[1])
    rh, eh, rz, ez = P.block(x[0, :2], y[0, :2], wide, weight=wide[1])
    P.check(h, rh, eh, "h, strided channels")
    P.check(z, rz, ez, "z, strided channels")


@pytest.mark.parametrize("C", [64, 1536, 5120])
def test_strides_alignment_and_types(C):
    require_gpu()
    from telefuser_amd.norm import block_norm, gated_residual_norm

    B, L = 2, 6
    big = _x((B, L + 3, 2 * C + 24), 3, BF16)
    views = {"rows apart": big[:, 1:L + 1, :C], "off 16 bytes": big[:, :L, 1:C + 1], "odd rows": big[:, 0:2 * 3:2, 8:C + 8],
             "channels apart": big[:, :L, 0:2 * C:2], "batch first": big.transpose(0, 1)[:, :, :C],
             "one batch entry": big[1, :L, 8:C + 8], "repeated row": big[:, :1, :C].expand(B, L, C)}
    # the same float64 tolerance as everywhere, not the bits of the contiguous call: how a row lies in memory decides which
    # lane sums which of its channels, and float32 sums in another order differ within the counted roundings
    def same(z, what, x, y=None, h=None, **how):
        rh, eh, rz, ez = P.block(x, y, **how)
        P.check(z, rz, ez, f"z {what}")
        if h is not None:
            P.check(h, rh, eh, f"h {what}")

    for what, v in views.items():
        same(block_norm(v), what, v)
        h, z = gated_residual_norm(v, v, norm="rms")
        same(z, what, v, v, h, norm_kind="rms")
    flat = torch.zeros(B * L * C + 8, dtype=FP32, device="cuda")
    off = flat[1:1 + B * L * C].view(B, L, C)
    off.copy_(_x((B, L, C), 4, FP32))
    same(block_norm(off), "off 4 bytes", off)
    x = _x((B, L, C), 5, FP32)
    odd = _p((C + 1,), 6)[1:]  # a parameter off 16 bytes
    same(block_norm(x, odd), "odd parameter", x, weight=odd)
    for yt, zt in itertools.product((BF16, FP16, FP32), (BF16, FP16, FP32)):  # a float32 residual stream
        y = _x((B, L, C), 6, yt)
        h, z = gated_residual_norm(x, y, out_dtype=zt)
        rh, eh, rz, ez = P.block(x, y)
        assert h.dtype == FP32 and z.dtype == zt
        P.check(h, rh, eh, f"h {yt}")
        P.check(z, rz, ez, f"z {yt} {zt}")


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("M,K", [(1, 1), (3, 16), (2, 127), (5, 128), (7, 129), (33, 1027), (4, 1536), (2, 8960),
                                 (3, 13824), (1, 40001)])
def test_per_token_int8(M, K, dtype):
    require_gpu()
    from telefuser_amd.norm import per_token_int8

    x = _x((M, K), K, dtype, offset=0.0)
    x[0, K // 2] = x[0].abs().max() * 2  # half of it is a value half-way between two codes
    if K > 16:
        x[0, 3], x[0, 5] = x[0, K // 2] / 2, -x[0, K // 2] / 2
    rows = per_token_int8(x)
    assert rows.codes.shape == (M, -(-K // 128) * 128) and rows.scale.shape == (M,) and rows.cols == K
    codes, scale = P.codes_of(x)
    assert torch.equal(rows.scale, scale.float())  # (in float64: torch divides float32 by a scalar through its reciprocal)
    assert (rows.codes[:, K:] == 0).all()
    if dtype is not FP32:  # the quotients of half values are never near a border without lying on it
        assert torch.equal(rows.codes[:, :K].double(), codes)
    else:
        P.check_rows(rows, x.double(), torch.zeros_like(x, dtype=torch.float64), "fp32")
    d = rows.dequantize(FP32)
    assert d.shape == x.shape and ((d.double() - x.double()).abs() <= scale[:, None] * 0.5001).all()


@pytest.mark.parametrize("dtype,bits", [(FP16, 10), (BF16, 7)])
def test_codes_of_every_pair_of_half_values(dtype, bits):
    """A row for every mantissa of the maximum, holding every mantissa at the ten exponents below it (values further below
    have code 0): the codes are those of the real numbers."""
    require_gpu()
    from telefuser_amd.norm import per_token_int8

    m = 1 + torch.arange(2 ** bits, device="cuda", dtype=torch.float64) / 2 ** bits
    x = torch.cat([m * 2.0 ** -e for e in range(10)]).expand(len(m), -1)
    x = torch.where(x <= m[:, None], x, 0.0)
    x = torch.cat([m[:, None], x, -x], 1).to(dtype)
    rows = per_token_int8(x)
    codes, scale = P.codes_of(x)
    assert torch.equal(rows.scale, scale.float())
    assert torch.equal(rows.codes[:, :x.shape[1]].double(), codes)


@pytest.mark.parametrize("K", [8, 100, 1536, 9000])
def test_int8_rows_of_extreme_values(K):
    require_gpu()
    from telefuser_amd.norm import block_norm, per_token_int8

    x = torch.ones((8, K), device="cuda")
    x[0] = 0.0
    x[1, 2] = float("nan")
    x[2, 3] = float("inf")
    x[3, 4] = float("-inf")
    x[4] *= 3e38
    x[4, ::2] *= -1
    x[5] *= 1e-38
    x[6] *= 1e-44
    x[7] *= 5e-5
    rows = per_token_int8(x)
    assert rows.scale[0] == 0 and (rows.codes[0] == 0).all()
    assert torch.isnan(rows.scale[1:4]).all() and (rows.codes[1:4] == 0).all()
    assert torch.isfinite(rows.scale[4:]).all()
    c = rows.codes[4, :K]
    assert (c[0::2] == -127).all() and (c[1::2] == 127).all()
    assert (rows.codes[5:, :K] == 127).all()
    for dt in (FP16, BF16):
        r = per_token_int8(x.to(dt))
        assert r.scale[0] == 0 and torch.isnan(r.scale[1:4]).all() and (r.codes[1:4] == 0).all()
    z = block_norm(x[:5], norm="rms")  # a row's infinity or NaN stays in its row
    assert (z[0] == 0).all() and torch.isnan(z[1]).all() and torch.isnan(z[2, 3]) and torch.isnan(z[3, 4])
    assert (z[2, :3] == 0).all()
    rows = block_norm(x[:4], out_dtype=torch.int8)
    assert rows.scale[0] == 0 and torch.isnan(rows.scale[1:]).all()


@pytest.mark.parametrize("C", [40, 200, 1536])
@pytest.mark.parametrize("w", [1e-38, 1e-33, 1e-20, 1e20, 1e35])
def test_int8_rows_of_tiny_and_huge_weights(C, w):
    require_gpu()
    from telefuser_amd.norm import block_norm

    x = _x((5, C), 1, BF16)
    x[3] = 0.0  # beside the others in its wave
    weight = torch.full((C,), w, device="cuda")
    rows = block_norm(x, weight, norm="rms", out_dtype=torch.int8)
    _, _, z, err = P.block(x, weight=weight, norm_kind="rms")
    keep = torch.tensor([0, 1, 2, 4], device="cuda")
    # a scale near the smallest float32 has few bits: the codes, not their products with it
    top = z.abs().amax(-1, keepdim=True)
    d = (rows.codes[keep, :C].double() - 127 * z[keep] / top[keep]).abs()
    assert (d <= 0.5 + 127 * (err / top)[keep] * 2 + 127 * 8 * P.U32).all()
    assert (rows.codes[3] == 0).all() and rows.scale[3] == 0
    assert torch.isfinite(rows.scale).all()


def test_constant_rows_and_large_means():
    require_gpu()
    from telefuser_amd.norm import block_norm

    for C in (64, 1536, 5120):
        x = torch.full((3, C), 100.0, device="cuda")
        x[1] += torch.randn(C, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) * 1e-2
        x[2] = -7.0
        z = block_norm(x)
        _, _, ref, err = P.block(x)
        P.check(z, ref, err, "large mean")


def test_empty_and_many_rows():
    require_gpu()
    from telefuser_amd.norm import block_norm, gated_residual_norm, per_token_int8

    for shape in ((0, 64), (2, 0, 64), (0, 3, 64)):
        x = torch.empty(shape, dtype=BF16, device="cuda")
        assert block_norm(x).shape == shape
        h, z = gated_residual_norm(x, x, out_dtype=torch.int8)
        assert h.shape == shape and z.codes.shape == (*shape[:-1], 128) and z.scale.shape == shape[:-1]
        assert per_token_int8(x).scale.shape == shape[:-1]
    x = _x((1, 70001, 64), 1, BF16)
    _, _, ref, err = P.block(x)
    P.check(block_norm(x), ref, err, "many rows")


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("B,L,C", [(1, 16384, 260), (2, 16400, 520), (1, 20011, 1027), (1, 16390, 1536), (1, 17000, 2565),
                                   (1, 16384, 4097), (2, 16387, 5120), (1, 16400, 8192)])
def test_many_rows_of_shared_parameters(B, L, C, dtype):
    """Long sequences with the parameters of a batch entry: rows from all over, and none written twice or left out."""
    require_gpu()
    from telefuser_amd.norm import block_norm, gated_residual, gated_residual_norm

    x, y = _x((B, L, C), C, dtype), _x((B, L, C), C + 1, dtype)
    at = torch.cat([torch.arange(0, 20), torch.randint(20, L - 20, (60,), generator=torch.Generator().manual_seed(C)),
                    torch.arange(L - 20, L)]).cuda()
    xs, ys = x[:, at], y[:, at]
    gate, scale, shift, w, b, pw = (_p(s, i) for i, s in enumerate([(B, 1, C), (B, 1, C), (1, 1, C), (C,), (C,), (C,)]))
    for how in ({"scale": scale, "shift": shift}, {"weight": w, "norm": "rms"},
                {"weight": w, "bias": b, "scale": scale, "shift": shift}):
        ref = {**how, "norm_kind": how.get("norm", "layer")}
        ref.pop("norm", None)
        _, _, rz, ez = P.block(xs, **ref)
        P.check(block_norm(x, **how)[:, at], rz, ez, f"z {sorted(how)}")
        rows = block_norm(x, **how, out_dtype=torch.int8)
        P.check_rows(type(rows)(rows.codes[:, at], rows.scale[:, at], C), rz, ez, f"int8 {sorted(how)}")
    for how in ({}, {"post_norm": "rms", "post_weight": pw}, {"post_norm": "layer", "post_weight": pw, "post_bias": b}):
        h, z = gated_residual_norm(x, y, gate, scale=scale, shift=shift, **how)
        rh, eh, rz, ez = P.block(xs, ys, gate, scale=scale, shift=shift, **how)
        P.check(h[:, at], rh, eh, f"h {sorted(how)}")
        P.check(z[:, at], rz, ez, f"z {sorted(how)}")
        # (not the bits of h: without the norm's parameters another kernel may run, which sums a row in another order)
        P.check(gated_residual(x, y, gate, **how)[:, at], rh, eh, f"h alone {sorted(how)}")
    full = block_norm(x, scale=scale, shift=shift)  # every row, against the same rows in short calls
    for i in range(0, L, 8000):
        part = block_norm(x[:, i:i + 8000], scale=scale, shift=shift)
        assert ((full[:, i:i + 8000].float() - part.float()).abs() <= 0.02 * (part.float().abs() + 1)).all()


@pytest.mark.parametrize("C", [260, 1027, 1536])
@pytest.mark.parametrize("L", [40, 16384])
def test_infinite_gate_of_the_last_channel(L, C):
    """The lanes past a row's end keep zeros: an infinite value leaves 0 in the other channels of an RMS norm, NaN in its
    own."""
    require_gpu()
    from telefuser_amd.norm import gated_residual_norm

    x, y, gate = _x((1, L, C), 1, BF16), _x((1, L, C), 2, BF16).abs() + 1, _p((C,), 3)
    gate[-1] = float("inf")
    h, z = gated_residual_norm(x, y, gate, norm="rms")
    assert (h[..., -1] == float("inf")).all() and z[..., -1].isnan().all()
    assert h[..., :-1].isfinite().all() and (z[..., :-1] == 0).all()


def test_offsets_past_32_bits():
    require_gpu()
    from telefuser_amd.norm import gated_residual_norm

    L, C = 70000, 32768  # 2.3e9 values
    x = torch.zeros((1, L, C), dtype=BF16, device="cuda")
    x[:, -3:] = _x((1, 3, C), 1, BF16)
    gate = _p((C,), 2)
    h, z = gated_residual_norm(x, x, gate)
    rh, eh, rz, ez = P.block(x[:, -4:], x[:, -4:], gate)
    P.check(h[:, -4:], rh, eh, "h")
    P.check(z[:, -4:], rz, ez, "z")
    assert not h[:, :4].any() and not z[:, :4].any()
    del h, z
    rows = gated_residual_norm(x, x, gate, out_dtype=torch.int8)[1]
    P.check_rows(type(rows)(rows.codes[:, -4:], rows.scale[:, -4:], C), rz, ez, "int8 z")
    log("offsets past 32 bits: done")


def test_repeats_bit_for_bit_on_another_stream_and_in_a_graph():
    require_gpu()
    from telefuser_amd.norm import gated_residual_norm

    x, y = _x((2, 300, 1536), 1, BF16), _x((2, 300, 1536), 2, BF16)
    gate, scale, shift = _p((2, 1, 1536), 1), _p((2, 1, 1536), 2), _p((2, 1, 1536), 3)

    def call():
        return gated_residual_norm(x, y, gate, scale=scale, shift=shift, out_dtype=torch.int8)

    h, z = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        h1, z1 = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(h, h1) and torch.equal(z.codes, z1.codes) and torch.equal(z.scale, z1.scale)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        hg, zg = call()
    for seed in (5, 6, 7):  # each replay on new values, against eager calls
        x.copy_(_x((2, 300, 1536), seed, BF16))
        g.replay()
        torch.cuda.synchronize()
        h, z = call()
        assert torch.equal(h, hg) and torch.equal(z.codes, zg.codes) and torch.equal(z.scale, zg.scale)
