"""INT8 linear layers: activations in INT8 with a scale per token, weights in INT8 with a scale per output channel.

``int8_linear(x, weight)`` takes a floating x (quantized per token on the way) or the ``Int8Rows`` that
``telefuser_amd.norm.block_norm(..., out_dtype=torch.int8)`` and ``per_token_int8`` give.  The products are summed
exactly in int32; both scales, the bias and the activation are applied in float32 before the one rounding.
"""

from __future__ import annotations

from typing import Optional, Union

import torch

from . import _lib
from .norm import _DTYPE, Int8Rows, _check_input, _gpu, _no_grad, _rows, per_token_int8

_ACT = {None: 0, "none": 0, "gelu_tanh": 1, "silu": 2}
_MAX_K = 131072  # 127 * 127 * K stays in int32


class Int8Weight:
    """The weight [N, K] of a linear layer in INT8: codes (rows zero-padded to a multiple of 128), a float32 scale per
    output channel and the bias, laid out once.

    ``Int8Weight(codes, scale, bias)`` takes what a quantized checkpoint holds (codes int8 [N, K] in -127 .. 127, scale
    [N] or [N, 1]); ``Int8Weight.quantize(weight, bias)`` quantizes a floating weight on the GPU."""

    def __init__(self, codes: torch.Tensor, scale: torch.Tensor, bias: Optional[torch.Tensor] = None):
        if codes.dim() != 2 or codes.dtype != torch.int8 or 0 in codes.shape:
            raise ValueError(f"codes must be int8 [N, K], got {codes.dtype} {tuple(codes.shape)}")
        n, k = codes.shape
        if k > _MAX_K:
            raise ValueError(f"K = {k}: sums of more than {_MAX_K} products may not fit int32")
        if tuple(scale.shape) not in ((n,), (n, 1)) or not scale.is_floating_point():
            raise ValueError(f"scale must be floating [N] or [N, 1] with N = {n}, got {scale.dtype} "
                             f"{tuple(scale.shape)}")
        if bias is not None and (tuple(bias.shape) != (n,) or not bias.is_floating_point()):
            raise ValueError(f"bias must be floating [N] with N = {n}, got {bias.dtype} {tuple(bias.shape)}")
        _no_grad(scale, bias)
        dev = codes.device
        if scale.device != dev or (bias is not None and bias.device != dev):
            raise ValueError("codes, scale and bias must be on one device")
        kpad = -(-k // 128) * 128
        if kpad != k:
            codes = torch.nn.functional.pad(codes, (0, kpad - k))
        self.codes = codes if codes.is_contiguous() and codes.data_ptr() % 16 == 0 else codes.clone(
            memory_format=torch.contiguous_format)
        self.scale = scale.detach().reshape(n).to(torch.float32).contiguous()
        self.bias = None if bias is None else bias.detach().to(torch.float32).contiguous()
        self.out_features, self.in_features = n, k

    @classmethod
    def quantize(cls, weight: torch.Tensor, bias: Optional[torch.Tensor] = None) -> "Int8Weight":
        """From a floating weight [N, K] on the GPU: per row, scale = max|w| / 127 and codes = round(127 w / max|w|).  The
        weight and the bias are detached: a module's parameters go in as they are."""
        if weight.dim() != 2:
            raise ValueError(f"weight must be [N, K], got {tuple(weight.shape)}")
        rows = per_token_int8(weight.detach())
        made = cls(rows.codes, rows.scale, None if bias is None else bias.detach())
        made.in_features = rows.cols
        return made


def int8_linear(x: Union[torch.Tensor, Int8Rows], weight: Int8Weight, *, act: Optional[str] = None,
                out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """act(x @ weight.T + bias) in INT8: [..., K] -> [..., N].

    x: floating [B, L, K] or [M, K], or ``Int8Rows`` of them.  act: None, "gelu_tanh" or "silu".  out_dtype: bfloat16,
    float16 or float32; x's by default, bfloat16 for ``Int8Rows``."""
    if not isinstance(weight, Int8Weight):
        raise ValueError(f"weight must be an Int8Weight, got {type(weight).__name__}")
    act_code = _ACT.get(act)
    if act_code is None:
        raise ValueError(f"act must be None, 'gelu_tanh' or 'silu', got {act!r}")
    lib, n, w, bias = _lib.load(), weight.out_features, weight.codes, weight.bias
    kpad = w.shape[1]
    if isinstance(x, Int8Rows):
        return _linear_rows(lib, x, weight, act_code, out_dtype)
    x_dt = _check_input(x, "x")
    shape = x.shape
    if shape[-1] != weight.in_features:
        raise ValueError(f"x has {tuple(shape)}, the weight takes {weight.in_features} channels")
    _no_grad(x)
    dev = _gpu(x)
    if w.get_device() != dev:
        raise ValueError(f"x is on {x.device}, the weight on {w.device}")
    out_dtype = out_dtype or x.dtype
    out_dt = _out_code(out_dtype)
    out = x.new_empty((*shape[:-1], n), dtype=out_dtype)
    B, L = 1 if len(shape) == 2 else shape[0], shape[-2]
    if B and L:
        xr, sb, sl = _rows(x)
        size = lib.qattn_linear_int8_rows_workspace_size(B * L, n, shape[-1])
        ws = x.new_empty(size, dtype=torch.uint8) if size else None
        _lib.launch(dev, lib.qattn_linear_int8_rows, xr.data_ptr(), x_dt, sb, sl, B, L, shape[-1], w.data_ptr(), kpad,
                    weight.scale.data_ptr(), None if bias is None else bias.data_ptr(), out.data_ptr(), out_dt, n, n,
                    act_code, None if ws is None else ws.data_ptr(), size)
    return out


def _out_code(out_dtype: torch.dtype) -> int:
    code = _DTYPE.get(out_dtype)
    if code is None:
        raise ValueError(f"out_dtype must be bfloat16, float16 or float32, got {out_dtype}")
    return code


def _linear_rows(lib, x: Int8Rows, weight: Int8Weight, act_code: int, out_dtype):
    codes, x_scale, cols = x
    out_dtype = out_dtype or torch.bfloat16
    out_dt = _out_code(out_dtype)
    kpad, n = weight.codes.shape[1], weight.out_features
    if cols != weight.in_features or codes.shape[-1] != kpad:
        raise ValueError(f"x has {cols} channels in rows of {codes.shape[-1]}, the weight takes {weight.in_features} "
                         f"in rows of {kpad}")
    dev = codes.get_device()
    if codes.dtype != torch.int8 or x_scale.dtype != torch.float32 or codes.shape[:-1] != x_scale.shape or \
            not codes.is_contiguous() or not x_scale.is_contiguous() or x_scale.get_device() != dev:
        raise ValueError("Int8Rows must hold contiguous int8 codes and a contiguous float32 scale for each row")
    _no_grad(x_scale)
    if not codes.is_cuda or weight.codes.get_device() != dev:
        raise ValueError(f"x is on {codes.device}, the weight on {weight.codes.device}: both must be on one GPU")
    out = codes.new_empty((*codes.shape[:-1], n), dtype=out_dtype)
    m = x_scale.numel()
    if m:
        bias = weight.bias
        size = lib.qattn_linear_int8_workspace_size(m, n, kpad)
        ws = codes.new_empty(size) if size else None
        _lib.launch(dev, lib.qattn_linear_int8, codes.data_ptr(), kpad, x_scale.data_ptr(), weight.codes.data_ptr(), kpad,
                    weight.scale.data_ptr(), None if bias is None else bias.data_ptr(), out.data_ptr(), out_dt, n, m, n,
                    kpad, act_code, None if ws is None else ws.data_ptr(), size)
    return out


__all__ = ["Int8Rows", "Int8Weight", "int8_linear", "per_token_int8"]
