"""The row operators around a DiT block: the norm before it and the gated residual after it.

A block runs ``norm -> modulate(scale, shift) -> layers -> x + gate * y``; as separate elementwise kernels each arrow
reads and writes the whole residual stream.  Here they are one pass over the rows:

``block_norm``           z = norm(x) * weight + bias, then z * (1 + scale) + shift; optionally straight to INT8 rows for
                         ``int8_linear``
``gated_residual``       h = residual_scale * x + gate * y, y normalized first with ``post_norm``
``gated_residual_norm``  both: (h, z), z from the float32 h before it is rounded
``per_token_int8``       INT8 rows of an activation (or of a weight), one scale per row

Forward only, like the attention they surround: inputs that need a gradient are refused.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib

_NORM = {None: 0, "layer": 1, "rms": 2}
_DTYPE = {torch.bfloat16: _lib.QATTN_BF16, torch.float16: _lib.QATTN_FP16, torch.float32: _lib.QATTN_F32}
_NO_PARAM = _lib.QattnParam(None, 0, 0, 0)


class Int8Rows(NamedTuple):
    """Rows of a [..., K] tensor in INT8: value = codes * scale, scale = max|row| / 127.

    ``codes`` [..., Kpad] int8 contiguous, K rounded up to 128 and the columns past ``cols`` zero; ``scale`` [...]
    float32."""

    codes: torch.Tensor
    scale: torch.Tensor
    cols: int

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        return (self.codes[..., :self.cols].float() * self.scale.unsqueeze(-1)).to(dtype)


def _no_grad(*tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError("no backward: call under torch.no_grad() or detach the inputs")


def _check_input(x: torch.Tensor, name: str) -> None:
    if x.dtype not in _DTYPE:
        raise ValueError(f"{name} must be bfloat16, float16 or float32, got {x.dtype}")
    if x.dim() not in (2, 3):
        raise ValueError(f"{name} must be [L, C] or [B, L, C], got {tuple(x.shape)}")
    if x.shape[-1] == 0:
        raise ValueError(f"{name} has no channels")


def _rows(x: torch.Tensor):
    """x with contiguous channels, and its strides over (b, l)."""
    if x.stride(-1) != 1 and x.shape[-1] > 1:
        x = x.contiguous()
    return (x, 0, x.stride(0)) if x.dim() == 2 else (x, x.stride(0), x.stride(1))


def _param(t: Optional[torch.Tensor], x: torch.Tensor, name: str, keep: list):
    """A parameter that broadcasts against x, as the kernels read it; tensors that must outlive the call go to keep."""
    if t is None:
        return _NO_PARAM
    if t.dtype not in _DTYPE:
        raise ValueError(f"{name} must be bfloat16, float16 or float32, got {t.dtype}")
    if t.device != x.device:
        raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    shape, c = t.shape, x.shape[-1]
    if len(shape) > x.dim() or any(n not in (1, m) for n, m in zip(shape[::-1], x.shape[::-1])):
        raise ValueError(f"{name} {tuple(shape)} does not broadcast against x {tuple(x.shape)}")
    if c > 1 and (not shape or shape[-1] != c or t.stride(-1) != 1):  # one value for all channels, or strided channels
        t = t.expand(*shape[:-1], c).contiguous()
        keep.append(t)
    n = t.dim()
    sl = t.stride(-2) if n > 1 and t.shape[-2] > 1 else 0
    sb = t.stride(0) if n > 2 and t.shape[0] > 1 else 0
    return _lib.QattnParam(t.data_ptr(), sb, sl, _DTYPE[t.dtype])


def _run(x, y, gate, residual_scale, post, post_weight, post_bias, post_eps, want_h, norm, weight, bias, scale, shift,
         eps, z_dtype):
    _check_input(x, "x")
    if norm not in _NORM or post not in _NORM:
        raise ValueError(f"a norm is 'layer' or 'rms', got {norm!r}, {post!r}")
    if not eps >= 0 or not post_eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}, {post_eps}")
    _no_grad(x, y, gate, post_weight, post_bias, weight, bias, scale, shift)
    dev = x.device
    if dev.type != "cuda":
        raise ValueError(f"x must be on a GPU, got {dev}")
    keep = []
    xr, x_sb, x_sl = _rows(x)
    y_ptr = y_sb = y_sl = y_dt = 0
    if y is not None:
        _check_input(y, "y")
        if y.shape != x.shape or y.device != dev:
            raise ValueError(f"y must be {tuple(x.shape)} on {dev}, got {tuple(y.shape)} on {y.device}")
        if y.dtype != x.dtype and x.dtype != torch.float32:
            raise ValueError(f"y must have x's dtype {x.dtype} (or x be float32), got {y.dtype}")
        yr, y_sb, y_sl = _rows(y)
        keep.append(yr)
        y_ptr, y_dt = yr.data_ptr(), _DTYPE[y.dtype]
    B, (L, C) = (1 if x.dim() == 2 else x.shape[0]), x.shape[-2:]
    h = z = codes = z_scale = None
    pitch = 0
    if want_h:
        h = torch.empty(x.shape, dtype=x.dtype, device=dev)
    if z_dtype == torch.int8:
        pitch = -(-C // 128) * 128
        codes = torch.empty((*x.shape[:-1], pitch), dtype=torch.int8, device=dev)
        z_scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev)
        z = Int8Rows(codes, z_scale, C)
    elif z_dtype is not None:
        if z_dtype not in _DTYPE:
            raise ValueError(f"out_dtype must be bfloat16, float16, float32 or int8, got {z_dtype}")
        z = codes = torch.empty(x.shape, dtype=z_dtype, device=dev)
    params = [_param(t, x, n, keep) for t, n in ((gate, "gate"), (weight, "weight"), (bias, "bias"), (scale, "scale"),
                                                 (shift, "shift"), (post_weight, "post_weight"),
                                                 (post_bias, "post_bias"))]
    if B and L:
        args = _lib.QattnBlockNormArgs(
            ctypes.sizeof(_lib.QattnBlockNormArgs), xr.data_ptr(), y_ptr, h.data_ptr() if want_h else None,
            codes.data_ptr() if codes is not None else None, z_scale.data_ptr() if z_scale is not None else None, x_sb,
            x_sl, y_sb, y_sl, pitch, B, L, C, *params, _DTYPE[x.dtype], y_dt,
            _lib.QATTN_I8 if z_scale is not None else _DTYPE.get(z_dtype, 0), _NORM[norm], _NORM[post], eps, post_eps,
            residual_scale)
        with _lib.on_device(dev):
            _lib.check(_lib.load().qattn_block_norm(args, _lib.stream_of(x)))
    return h, z


def block_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
               scale: Optional[torch.Tensor] = None, shift: Optional[torch.Tensor] = None, norm: str = "layer",
               eps: float = 1e-6, out_dtype: Optional[torch.dtype] = None):
    """The norm before a block: norm(x) * weight + bias, then * (1 + scale) + shift, in float32, rounded once.

    x: [B, L, C] or [L, C] in bf16 / fp16 / fp32, any strides.  weight, bias, scale and shift broadcast against x ([C],
    [B, 1, C], [B, L, C], ...) and are float32 or half.  norm: "layer" or "rms".  out_dtype: x's by default, another
    floating one, or torch.int8 for ``Int8Rows`` (what ``int8_linear`` takes) quantized from the float32 result."""
    if norm is None:
        raise ValueError("a norm is 'layer' or 'rms', got None")
    return _run(x, None, None, 1.0, None, None, None, 0.0, False, norm, weight, bias, scale, shift, eps,
                out_dtype or x.dtype)[1]


def gated_residual(x: torch.Tensor, y: torch.Tensor, gate: Optional[torch.Tensor] = None, *,
                   residual_scale: float = 1.0, post_norm: Optional[str] = None,
                   post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None,
                   post_eps: float = 1e-6) -> torch.Tensor:
    """The residual after a block: residual_scale * x + gate * y in x's dtype, computed in float32.

    y has x's shape and dtype (any of the three beside a float32 x); gate broadcasts against x.  post_norm ("layer" or
    "rms", with post_weight and post_bias) normalizes y's rows first."""
    return _run(x, y, gate, residual_scale, _post(post_norm, post_weight, post_bias), post_weight, post_bias, post_eps,
                True, None, None, None, None, None, 0.0, None)[0]


def gated_residual_norm(x: torch.Tensor, y: torch.Tensor, gate: Optional[torch.Tensor] = None, *,
                        residual_scale: float = 1.0, post_norm: Optional[str] = None,
                        post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None,
                        post_eps: float = 1e-6, weight: Optional[torch.Tensor] = None,
                        bias: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None,
                        shift: Optional[torch.Tensor] = None, norm: str = "layer", eps: float = 1e-6,
                        out_dtype: Optional[torch.dtype] = None):
    """``gated_residual`` after one block and ``block_norm`` before the next in one pass: (h, z).  z is the norm of the
    float32 sum, before h is rounded to x's dtype."""
    if norm is None:
        raise ValueError("a norm is 'layer' or 'rms', got None")
    return _run(x, y, gate, residual_scale, _post(post_norm, post_weight, post_bias), post_weight, post_bias, post_eps,
                True, norm, weight, bias, scale, shift, eps, out_dtype or x.dtype)


def _post(post_norm, post_weight, post_bias):
    if post_norm is None and (post_weight is not None or post_bias is not None):
        raise ValueError("post_weight and post_bias need post_norm")
    return post_norm


def per_token_int8(x: torch.Tensor) -> Int8Rows:
    """INT8 rows of x [B, L, K] or [M, K] (bf16 / fp16 / fp32, any strides): scale = max|row| / 127, codes =
    round(127 x / max|row|), ties to even.  A row of zeros has scale 0; one with an infinity or a NaN has scale NaN, so
    that its products are NaN."""
    return _run(x, None, None, 1.0, None, None, None, 0.0, False, None, None, None, None, None, 0.0, torch.int8)[1]


__all__ = ["Int8Rows", "block_norm", "gated_residual", "gated_residual_norm", "per_token_int8"]
