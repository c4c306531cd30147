"""The operators around the attention as a DiT block runs them: norm and modulation to INT8 rows, the Q, K, V projections,
the fused self-attention, its output projection, the gated residual with the next norm, and the feed-forward layers.  Every
operator of the pass is checked against its float64 form on the values that it met in the pass."""

import pytest
import torch

from tests import block_plain as P
from tests.gpu_util import require_gpu

pytestmark = pytest.mark.gpu


def _block(B, L, H, F, seed):
    from telefuser_amd.linear import Int8Weight

    C = H * 128
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape, std=1.0):
        return torch.randn(shape, generator=g, device="cuda") * std

    p = {n: Int8Weight.quantize(rand(o, i, std=i ** -0.5).bfloat16(), rand(o, std=0.1).bfloat16())
         for n, i, o in (("q", C, C), ("k", C, C), ("v", C, C), ("o", C, C), ("up", C, F), ("down", F, C))}
    p["wq"], p["wk"] = rand(C, std=0.1) + 1, rand(C, std=0.1) + 1
    p["e"] = rand(B, 6, C, std=0.2)  # shift, scale, gate of the attention and of the feed-forward layers
    angle = torch.arange(L, device="cuda")[:, None] * 0.9 ** torch.arange(64, device="cuda")
    p["cos"], p["sin"] = angle.cos(), angle.sin()
    return rand(B, L, C).bfloat16(), p


def _run(x, p, H):
    """The block's output, and what each operator took and gave."""
    from telefuser_amd.linear import int8_linear, per_token_int8
    from telefuser_amd.norm import block_norm, gated_residual, gated_residual_norm
    from telefuser_amd.prologue import wan_self_attention

    e = [p["e"][:, i:i + 1] for i in range(6)]
    rows = block_norm(x, scale=e[1], shift=e[0], out_dtype=torch.int8)
    q, k, v = (int8_linear(rows, p[n]) for n in "qkv")
    a = wan_self_attention(q, k, v, p["wq"], p["wk"], p["cos"], p["sin"], H)
    o = int8_linear(a, p["o"])
    h, rows2 = gated_residual_norm(x, o, e[2], scale=e[4], shift=e[3], out_dtype=torch.int8)
    u = int8_linear(rows2, p["up"], act="gelu_tanh")
    d = int8_linear(u, p["down"])
    y = gated_residual(h, d, e[5])
    return y, dict(rows=rows, q=q, k=k, v=v, a=a, o=o, h=h, rows2=rows2, u=u, d=d, a_rows=per_token_int8(a),
                   u_rows=per_token_int8(u))


@pytest.mark.parametrize("B,L,H,F", [(1, 300, 2, 640), (2, 1000, 4, 1100), (1, 17000, 3, 1024)])
def test_block(B, L, H, F):
    require_gpu()
    x, p = _block(B, L, H, F, L)
    y, t = _run(x, p, H)
    e = [p["e"][:, i:i + 1] for i in range(6)]
    at = torch.cat([torch.arange(0, 100), torch.arange(L - 100, L)]).cuda()

    def rows_at(r):
        return type(r)(r.codes[:, at], r.scale[:, at], r.cols)

    def linear(rows, name, out, act=None):
        w = p[name]
        ref, err = P.linear(rows.codes[:, at, :rows.cols], rows.scale[:, at], w.codes[:, :w.in_features], w.scale, w.bias,
                            act)
        P.check(out[:, at], ref, err, name)

    _, _, rz, ez = P.block(x[:, at], scale=e[1], shift=e[0])
    P.check_rows(rows_at(t["rows"]), rz, ez, "norm before the attention")
    for n in "qkv":
        linear(t["rows"], n, t[n])
    linear(t["a_rows"], "o", t["o"])
    rh, eh, rz, ez = P.block(x[:, at], t["o"][:, at], e[2], scale=e[4], shift=e[3])
    P.check(t["h"][:, at], rh, eh, "residual after the attention")
    P.check_rows(rows_at(t["rows2"]), rz, ez, "norm before the feed-forward layers")
    linear(t["rows2"], "up", t["u"], "gelu_tanh")
    linear(t["u_rows"], "down", t["d"])
    rh, eh, _, _ = P.block(t["h"][:, at], t["d"][:, at], e[5])
    P.check(y[:, at], rh, eh, "residual after the feed-forward layers")
    assert torch.isfinite(y.float()).all()


def test_block_replays_in_a_graph():
    require_gpu()
    x, p = _block(1, 700, 2, 640, 3)
    _run(x, p, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _run(x, p, 2)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, _ = _run(x, p, 2)
    for seed in (4, 5, 6):
        x.copy_(_block(1, 700, 2, 640, seed)[0])
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, _run(x, p, 2)[0])
