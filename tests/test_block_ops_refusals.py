"""Further refusals of the operators around a DiT block, without a GPU."""

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from telefuser_amd import _lib
from telefuser_amd.linear import Int8Rows, Int8Weight, int8_linear
from telefuser_amd.norm import block_norm, gated_residual, gated_residual_norm, per_token_int8


def _args(**kw):
    none = _lib.QattnParam(None, 0, 0, 0)
    a = _lib.QattnBlockNormArgs(ctypes.sizeof(_lib.QattnBlockNormArgs), 4096, 4096, 8192, 8192, 4096, 0, 64, 0, 64, 128, 1, 2,
                                64, none, none, none, none, none, none, none, 0, 0, 0, 1, 0, 1e-6, 0.0, 1.0)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


@pytest.mark.parametrize("x,y", [(0, 1), (1, 0), (0, 3), (1, 3), (2, 3), (2, -1), (0, 4)])
def test_type_of_y(x, y):
    """An x of one half type takes y of the other nowhere, and a float32 y in the second entry only."""
    lib = _lib.load()
    for entry in (lib.qattn_block_norm, lib.qattn_block_norm_ex):
        assert entry(_args(x_dtype=x, y_dtype=y), None) == 1, lib.qattn_last_error()
    assert lib.qattn_block_norm(_args(x_dtype=0, y_dtype=2), None) == 1


@pytest.mark.parametrize("kw,code", [({"size": 8}, 9), ({"x_dtype": 3}, 1), ({"C": 0}, 2), ({"y_dtype": 2, "y": 4098}, 4),
                                     ({"h": None, "z": None}, 9), ({"post_norm": 3}, 9)])
def test_second_entry_checks_as_the_first(kw, code):
    lib = _lib.load()
    assert lib.qattn_block_norm_ex(_args(**kw), None) == code, lib.qattn_last_error()
    assert lib.qattn_block_norm_ex(_args(B=0, y_dtype=2), None) == 0
    assert lib.qattn_block_norm_ex(None, None) == 9


X = torch.zeros(2, 3, 64, dtype=torch.bfloat16)
CODES = torch.ones(5, 64, dtype=torch.int8)


@pytest.mark.parametrize("call", [
    lambda d: block_norm(d(X)),
    lambda d: block_norm(X, d(torch.ones(64))),
    lambda d: block_norm(X, bias=d(torch.ones(64))),
    lambda d: block_norm(X, scale=d(torch.ones(64)), shift=torch.ones(64)),
    lambda d: block_norm(X, shift=d(torch.ones(64))),
    lambda d: gated_residual(d(X), X),
    lambda d: gated_residual(X, d(X)),
    lambda d: gated_residual(X, X, d(torch.ones(64))),
    lambda d: gated_residual_norm(X, X, post_norm="rms", post_weight=d(torch.ones(64))),
    lambda d: gated_residual_norm(X, X, post_norm="layer", post_bias=d(torch.ones(64))),
    lambda d: per_token_int8(d(X)),
    lambda d: Int8Weight(CODES, d(torch.ones(5))),
    lambda d: Int8Weight(CODES, torch.ones(5), d(torch.ones(5))),
    lambda d: int8_linear(d(X), Int8Weight(CODES, torch.ones(5))),
    lambda d: int8_linear(Int8Rows(torch.zeros(2, 128, dtype=torch.int8), d(torch.ones(2)), 64), Int8Weight(CODES, torch.ones(5))),
])
@pytest.mark.parametrize("no_grad", [False, True])
def test_tangents_are_refused(call, no_grad):
    """A dual tensor's tangent would be lost: no requires_grad shows it, and no_grad does not switch it off."""
    with forward_ad.dual_level():
        with torch.set_grad_enabled(not no_grad), pytest.raises(ValueError, match="no forward-mode derivative"):
            call(lambda t: forward_ad.make_dual(t, torch.ones_like(t)))
        assert Int8Weight(CODES, torch.ones(5)).out_features == 5  # plain tensors are fine within a level
        with pytest.raises(ValueError, match="on a GPU"):
            block_norm(X)
