"""What the operators around a DiT block refuse, without a GPU: the Python checks and the C entries' status codes."""

import ctypes

import pytest
import torch

from telefuser_amd import _lib
from telefuser_amd.linear import Int8Rows, Int8Weight, int8_linear
from telefuser_amd.norm import block_norm, gated_residual, gated_residual_norm, per_token_int8

X = torch.zeros(2, 3, 64, dtype=torch.bfloat16)


@pytest.mark.parametrize("call,words", [
    (lambda: block_norm(X.double()), "bfloat16, float16 or float32"),
    (lambda: block_norm(X.to(torch.int8)), "bfloat16, float16 or float32"),
    (lambda: block_norm(X[0, 0]), r"\[L, C\] or \[B, L, C\]"),
    (lambda: block_norm(X[None]), r"\[L, C\] or \[B, L, C\]"),
    (lambda: block_norm(X[..., :0]), "no channels"),
    (lambda: block_norm(X, norm="group"), "'layer' or 'rms'"),
    (lambda: block_norm(X, norm=None), "'layer' or 'rms'"),
    (lambda: gated_residual_norm(X, X, norm=None), "'layer' or 'rms'"),
    (lambda: gated_residual(X, X, post_norm="batch"), "'layer' or 'rms'"),
    (lambda: gated_residual(X, X, post_weight=X[0, 0]), "need post_norm"),
    (lambda: block_norm(X, eps=-1.0), "eps"),
    (lambda: block_norm(X, eps=float("nan")), "eps"),
    (lambda: gated_residual(X, X, post_norm="rms", post_eps=-1e-6), "eps"),
    (lambda: block_norm(X), "on a GPU"),
    (lambda: per_token_int8(X), "on a GPU"),
    (lambda: block_norm(X.clone().requires_grad_()), "no backward"),
    (lambda: block_norm(X, torch.ones(64, requires_grad=True)), "no backward"),
    (lambda: gated_residual(X, X, torch.ones(64, requires_grad=True)), "no backward"),
    (lambda: per_token_int8(X.clone().requires_grad_()), "no backward"),
    (lambda: int8_linear(X, None), "Int8Weight"),
    (lambda: Int8Weight(X[0], torch.ones(3)), "int8"),
    (lambda: Int8Weight(torch.zeros(3, 0, dtype=torch.int8), torch.ones(3)), "int8"),
    (lambda: Int8Weight(torch.zeros(3, 8, dtype=torch.int8), torch.ones(4)), "scale"),
    (lambda: Int8Weight(torch.zeros(3, 8, dtype=torch.int8), torch.ones(3, dtype=torch.int32)), "scale"),
    (lambda: Int8Weight(torch.zeros(3, 8, dtype=torch.int8), torch.ones(3), torch.ones(8)), "bias"),
    (lambda: Int8Weight(torch.zeros(1, 131073, dtype=torch.int8), torch.ones(1)), "int32"),
    (lambda: Int8Weight(torch.zeros(3, 8, dtype=torch.int8), torch.ones(3, requires_grad=True)), "no backward"),
    (lambda: Int8Weight.quantize(X), r"\[N, K\]"),
])
def test_refusals(call, words):
    with pytest.raises(ValueError, match=words):
        call()


W = Int8Weight(torch.ones(5, 64, dtype=torch.int8), torch.ones(5), torch.zeros(5))


def test_weight_layout():
    assert W.codes.shape == (5, 128) and (W.codes[:, 64:] == 0).all() and W.codes.is_contiguous()
    assert (W.out_features, W.in_features) == (5, 64) and W.bias.dtype == torch.float32
    with torch.no_grad():  # parameters of a module, as they are at inference
        w = Int8Weight(torch.ones(5, 64, dtype=torch.int8), torch.ones(5, requires_grad=True))
    assert not w.scale.requires_grad and w.bias is None


@pytest.mark.parametrize("rows,kw,words", [
    (X[..., :32], {}, "64 channels"),
    (X, {"act": "relu"}, "act must be"),
    (X, {}, "on a GPU"),
    (Int8Rows(torch.zeros(2, 128, dtype=torch.int8), torch.ones(2), 64), {}, "on one GPU"),
    (Int8Rows(torch.zeros(2, 128, dtype=torch.int8), torch.ones(2), 64), {"out_dtype": torch.float64}, "out_dtype"),
    (Int8Rows(torch.zeros(2, 128, dtype=torch.int8), torch.ones(2), 100), {}, "channels"),
    (Int8Rows(torch.zeros(2, 64, dtype=torch.int8), torch.ones(2), 64), {}, "channels"),
    (Int8Rows(torch.zeros(2, 128, dtype=torch.int8), torch.ones(3), 64), {}, "a scale|scale for each"),
    (Int8Rows(torch.zeros(2, 128, dtype=torch.int8), torch.ones(2).double(), 64), {}, "float32 scale"),
    (Int8Rows(torch.zeros(2, 256, dtype=torch.int8)[:, :128], torch.ones(2), 64), {}, "contiguous"),
    (Int8Rows(torch.zeros(2, 128), torch.ones(2), 64), {}, "int8 codes"),
    (Int8Rows(torch.zeros(2, 128, dtype=torch.int8), torch.ones(2, requires_grad=True), 64), {}, "no backward"),
])
def test_linear_refusals(rows, kw, words):
    with pytest.raises(ValueError, match=words):
        int8_linear(rows, W, **kw)


@pytest.mark.parametrize("p", [torch.ones(63), torch.ones(3, 3, 64), torch.ones(1, 2, 3, 64), torch.ones(2, 2, 64)])
def test_parameter_shapes(p, monkeypatch):
    from telefuser_amd import norm

    with pytest.raises(ValueError, match="broadcast"):
        norm._param(p, X, "scale", [])


def test_parameter_strides():
    from telefuser_amd import norm

    def strides(t):
        keep = []
        _, sb, sl, _ = norm._param(t, X, "gate", keep)
        return sb, sl, len(keep)

    assert strides(torch.ones(64)) == (0, 0, 0)
    assert strides(torch.ones(3, 64)) == (0, 64, 0)
    assert strides(torch.ones(2, 1, 64)) == (64, 0, 0)
    assert strides(torch.ones(1, 3, 64)) == (0, 64, 0)
    assert strides(torch.ones(2, 3, 64)) == (192, 64, 0)
    assert strides(torch.ones(2, 6, 64)[:, 2:3]) == (384, 0, 0)
    assert strides(torch.ones(2, 3, 1)) == (192, 64, 1)
    assert strides(torch.ones(1)) == (0, 0, 1)
    assert strides(torch.tensor(1.0)) == (0, 0, 1)
    with pytest.raises(ValueError, match="float32"):
        norm._param(torch.ones(64, dtype=torch.float64), X, "gate", [])


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _norm_args(**kw):
    none = _lib.QattnParam(None, 0, 0, 0)
    a = _lib.QattnBlockNormArgs(ctypes.sizeof(_lib.QattnBlockNormArgs), 4096, None, None, 8192, 4096, 0, 64, 0, 0, 128, 1, 2,
                                64, none, none, none, none, none, none, none, 0, 0, 0, 1, 0, 1e-6, 0.0, 1.0)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def test_packed_args_are_the_struct():
    a = _lib.QattnBlockNormArgs
    assert _lib.BLOCK_NORM_ARGS.size == ctypes.sizeof(a)
    param = (11, 12, 13, 2)
    values = (1, 2, 3, 4, 5, 6, *range(21, 29), *param * 7, 31, 32, 33, 34, 35, 0.5, 0.25, 2.0)
    got = a.from_buffer_copy(_lib.BLOCK_NORM_ARGS.pack(*values))
    flat = []
    for name, kind in a._fields_:
        v = getattr(got, name)
        flat += [getattr(v, n) for n, _ in kind._fields_] if kind is _lib.QattnParam else [v]
    assert tuple(flat) == values


@pytest.mark.parametrize("kw,code", [
    ({"size": 8}, 9), ({"x_dtype": 3}, 1), ({"x_dtype": -1}, 1), ({"y": 4096, "y_dtype": 1}, 1), ({"z_dtype": 4}, 1),
    ({"y": 4096, "y_dtype": 2}, 1), ({"C": 0}, 2), ({"C": 1 << 25}, 2), ({"B": -1}, 2), ({"B": 1 << 20, "L": 1 << 20}, 2),
    ({"norm": 3}, 9), ({"post_norm": -1}, 9), ({"z": None}, 9), ({"x": None}, 9), ({"x": 4097}, 4), ({"z": 8200}, 4),
    ({"h": 8}, 4), ({"z_dtype": 3, "z_scale": None}, 9), ({"z_dtype": 3, "z_pitch": 48}, 3),
    ({"z_dtype": 3, "z_pitch": 72}, 3), ({"gate": _lib.QattnParam(4096, 0, 0, 3)}, 1),
    ({"scale": _lib.QattnParam(4098, 0, 0, 2)}, 4), ({"bias": _lib.QattnParam(4096, 0, -1, 2)}, 3),
])
def test_block_norm_status(lib, kw, code):
    assert lib.qattn_block_norm(_norm_args(**kw), None) == code, lib.qattn_last_error()


def test_empty_calls_launch_nothing(lib):
    assert lib.qattn_block_norm(_norm_args(B=0), None) == 0
    assert lib.qattn_block_norm(_norm_args(L=0), None) == 0
    assert lib.qattn_block_norm(None, None) == 9
    assert _linear(lib, M=0) == 0


def _linear(lib, **kw):
    a = dict(x=4096, xp=128, sx=4096, w=4096, wp=128, sw=4096, bias=None, out=4096, dt=0, os=64, M=2, N=64, K=128, act=0, ws=None, wb=0)
    a.update(kw)
    return lib.qattn_linear_int8(a["x"], a["xp"], a["sx"], a["w"], a["wp"], a["sw"], a["bias"], a["out"], a["dt"], a["os"],
                                 a["M"], a["N"], a["K"], a["act"], a["ws"], a["wb"], None)


@pytest.mark.parametrize("kw,code", [
    ({"dt": 3}, 1), ({"dt": -1}, 1), ({"N": 0}, 2), ({"M": -1}, 2), ({"K": 64}, 2), ({"K": 0}, 2), ({"K": 192, "xp": 192}, 2),
    ({"K": 131200, "xp": 131200, "wp": 131200}, 2), ({"act": 3}, 9), ({"act": -1}, 9), ({"x": None}, 9), ({"sx": None}, 9),
    ({"w": None}, 9), ({"sw": None}, 9), ({"out": None}, 9), ({"xp": 64}, 3), ({"wp": 136}, 3), ({"os": 63}, 3),
    ({"x": 4104}, 4), ({"w": 4097}, 4), ({"out": 4097}, 4), ({"out": 4098, "dt": 2}, 4), ({"sw": 4098}, 4),
    ({"bias": 4098}, 4), ({"xp": 1 << 23}, 3), ({"M": 64, "K": 8192, "xp": 8192, "wp": 8192}, 7),
    ({"M": 64, "K": 8192, "xp": 8192, "wp": 8192, "ws": 4104, "wb": 1 << 30}, 7),
    ({"M": 64, "K": 8192, "xp": 8192, "wp": 8192, "ws": 4096, "wb": 2 * 128 * 128 * 4 - 1}, 7),
])
def test_linear_status(lib, kw, code):
    assert _linear(lib, **kw) == code, lib.qattn_last_error()


@pytest.mark.parametrize("kw,code", [
    ({"xd": 3}, 1), ({"cols": 0}, 2), ({"cols": 131073}, 2), ({"B": -1}, 2), ({"L": 1 << 40}, 2), ({"x": None}, 9),
    ({"x": 4097}, 4), ({"w": None}, 9), ({"wp": 128}, 3), ({"os": 63}, 3), ({"act": 7}, 9), ({"ws": None}, 7),
    ({"wb": 99 * 260 + 3}, 7), ({"ws": 4104}, 7), ({"dt": 9}, 1),
])
def test_linear_rows_status(lib, kw, code):
    a = dict(x=4096, xd=0, B=1, L=99, cols=200, w=4096, wp=256, out=4096, dt=0, os=64, N=64, act=0, ws=4096, wb=99 * 260 + 4)
    a.update(kw)
    rc = lib.qattn_linear_int8_rows(a["x"], a["xd"], 0, 200, a["B"], a["L"], a["cols"], a["w"], a["wp"], 4096, None,
                                    a["out"], a["dt"], a["os"], a["N"], a["act"], a["ws"], a["wb"], None)
    assert rc == code, lib.qattn_last_error()


def test_linear_workspaces(lib):
    rows, split = lib.qattn_linear_int8_rows_workspace_size, lib.qattn_linear_int8_workspace_size
    assert rows(0, 64, 100) == rows(5, 0, 100) == rows(5, 64, 0) == rows(1, 64, 16384) == rows(16, 64, 1024) == 0
    assert rows(1, 64, 16385) == 16528 and rows(99, 64, 200) == 99 * 260 + 4 and rows(75600, 64, 5120) == 75600 * 5124
    # split along K: few tiles and many stages, whole tiles of int32 sums
    assert split(75600, 13824, 5120) == split(1560, 1536, 8960) == split(200, 64, 256) == split(16, 64, 8960) == 0
    for m, n, k in ((17, 100, 4096), (64, 1536, 8960), (100, 9216, 13824), (300, 300, 13824)):
        tile = -(-m // 64) * -(-n // 64) * 64 * 64 * 4  # (a larger tile holds whole ones of these)
        assert split(m, n, k) >= 2 * tile and split(m, n, k) % (64 * 64 * 4) == 0
        assert rows(m, n, k) == (m * k + m * 4 + 15) // 16 * 16 + split(m, n, k)


@pytest.mark.parametrize("current,index,entered", [(0, 0, []), (0, 2, [2]), (1, 0, [0])])
def test_launch_on_the_tensors_device(monkeypatch, current, index, entered):
    """A launch takes the current stream of the tensors' GPU, with that GPU made current for it if it is not."""
    seen, inside = [], []

    class Device:
        def __init__(self, i):
            self.i = i

        def __enter__(self):
            inside.append(self.i)

        def __exit__(self, *exc):
            inside.append("left")

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 1000 + i, raising=False)
    monkeypatch.setattr(torch.cuda, "device", Device)
    _lib.launch(index, lambda *a: seen.append((a, list(inside))), "x", 5)
    assert seen == [(("x", 5, 1000 + index), entered)]
    assert inside == (entered + ["left"] if entered else [])
