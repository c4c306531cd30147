"""Further refusals of the operators around a DiT block, without a GPU."""

import ctypes

import pytest

from telefuser_amd import _lib


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
