"""The row operators around a DiT block: the norm before it and the gated residual after it.

A block runs ``norm -> modulate(scale, shift) -> layers -> x + gate * y``; as separate elementwise kernels each arrow
reads and writes the whole residual stream.  Here they are one pass over the rows:

``block_norm``           z = norm(x) * weight + bias, then z * (1 + scale) + shift; optionally straight to INT8 rows for
                         ``int8_linear``
``gated_residual``       h = residual_scale * x + gate * y, y normalized first with ``post_norm``
``gated_residual_norm``  both: (h, z), z from the float32 h before it is rounded
``per_token_int8``       INT8 rows of an activation (or of a weight), one scale per row

Forward only, like the attention they surround: inputs that need a gradient, or carry a tangent, are refused.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _lib

_NORM = {None: 0, "layer": 1, "rms": 2}
_DTYPE = {torch.bfloat16: _lib.QATTN_BF16, torch.float16: _lib.QATTN_FP16, torch.float32: _lib.QATTN_F32}
_NO_PARAM = (0, 0, 0, 0)
_pack_args, _ARGS_SIZE = _lib.BLOCK_NORM_ARGS.pack, _lib.BLOCK_NORM_ARGS.size


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
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError("no backward: call under torch.no_grad() or detach the inputs")
    if forward_ad._current_level >= 0:  # (a tangent has neither requires_grad nor a part in no_grad)
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError("no forward-mode derivative: detach the inputs")


def _check_input(x: torch.Tensor, name: str) -> int:
    """The dtype code of x after the checks that every input takes."""
    code = _DTYPE.get(x.dtype)
    if code is None:
        raise ValueError(f"{name} must be bfloat16, float16 or float32, got {x.dtype}")
    shape = x.shape
    if len(shape) not in (2, 3):
        raise ValueError(f"{name} must be [L, C] or [B, L, C], got {tuple(shape)}")
    if shape[-1] == 0:
        raise ValueError(f"{name} has no channels")
    return code


def _gpu(x: torch.Tensor) -> int:
    if not x.is_cuda:
        raise ValueError(f"x must be on a GPU, got {x.device}")
    return x.get_device()


def _rows(x: torch.Tensor):
    """x with contiguous channels, and its strides over (b, l)."""
    st = x.stride()
    if st[-1] != 1 and x.shape[-1] > 1:
        x = x.contiguous()
        st = x.stride()
    return (x, 0, st[0]) if len(st) == 2 else (x, st[0], st[1])


def _param(t: torch.Tensor, x: torch.Tensor, name: str, keep: list):
    """A parameter that broadcasts against x, as the fields of qattn_param; tensors that must outlive the call go to
    keep."""
    code = _DTYPE.get(t.dtype)
    if code is None:
        raise ValueError(f"{name} must be bfloat16, float16 or float32, got {t.dtype}")
    if t.get_device() != x.get_device():
        raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    shape, st, like = t.shape, t.stride(), x.shape
    n, c = len(shape), like[-1]
    if shape != like:
        fits = n <= len(like)
        for size, want in zip(shape[::-1], like[::-1]):
            if size != want and size != 1:
                fits = False
        if not fits:
            raise ValueError(f"{name} {tuple(shape)} does not broadcast against x {tuple(like)}")
    if c > 1 and (n == 0 or shape[-1] != c or st[-1] != 1):  # one value for all channels, or strided channels
        t = t.expand(*shape[:-1], c).contiguous()
        keep.append(t)
        st = t.stride()
    sl = st[-2] if n > 1 and shape[-2] > 1 else 0
    sb = st[0] if n > 2 and shape[0] > 1 else 0
    return t.data_ptr(), sb, sl, code


def _run(x, y, gate, residual_scale, post, post_weight, post_bias, post_eps, want_h, norm, weight, bias, scale, shift,
         eps, z_dtype):
    x_dt = _check_input(x, "x")
    if norm not in _NORM or post not in _NORM:
        raise ValueError(f"a norm is 'layer' or 'rms', got {norm!r}, {post!r}")
    if not eps >= 0 or not post_eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}, {post_eps}")
    _no_grad(x, y, gate, post_weight, post_bias, weight, bias, scale, shift)
    dev = _gpu(x)
    shape = x.shape
    keep = []
    xr, x_sb, x_sl = _rows(x)
    y_ptr = y_sb = y_sl = y_dt = 0
    if y is not None:
        y_dt = _check_input(y, "y")
        if y.shape != shape or y.get_device() != dev:
            raise ValueError(f"y must be {tuple(shape)} on {x.device}, got {tuple(y.shape)} on {y.device}")
        if y_dt != x_dt and _lib.QATTN_F32 not in (x_dt, y_dt):
            raise ValueError(f"y must have x's dtype {x.dtype} (or one of them be float32), got {y.dtype}")
        yr, y_sb, y_sl = _rows(y)
        keep.append(yr)
        y_ptr = yr.data_ptr()
    B, (L, C) = (1 if len(shape) == 2 else shape[0]), shape[-2:]
    h = z = None
    h_ptr = z_ptr = s_ptr = pitch = z_dt = 0
    if want_h:
        h = torch.empty_like(x, memory_format=torch.contiguous_format)
        h_ptr = h.data_ptr()
    if z_dtype is torch.int8:
        pitch, z_dt = -(-C // 128) * 128, _lib.QATTN_I8
        z = Int8Rows(x.new_empty((*shape[:-1], pitch), dtype=torch.int8), x.new_empty(shape[:-1], dtype=torch.float32), C)
        z_ptr, s_ptr = z.codes.data_ptr(), z.scale.data_ptr()
    elif z_dtype is not None:
        z_dt = _DTYPE.get(z_dtype)
        if z_dt is None:
            raise ValueError(f"out_dtype must be bfloat16, float16, float32 or int8, got {z_dtype}")
        z = torch.empty_like(x, dtype=z_dtype, memory_format=torch.contiguous_format)
        z_ptr = z.data_ptr()
    if B and L:
        args = _pack_args(
            _ARGS_SIZE, xr.data_ptr(), y_ptr, h_ptr, z_ptr, s_ptr, x_sb, x_sl, y_sb, y_sl, pitch, B, L, C,
            *(_NO_PARAM if gate is None else _param(gate, x, "gate", keep)),
            *(_NO_PARAM if weight is None else _param(weight, x, "weight", keep)),
            *(_NO_PARAM if bias is None else _param(bias, x, "bias", keep)),
            *(_NO_PARAM if scale is None else _param(scale, x, "scale", keep)),
            *(_NO_PARAM if shift is None else _param(shift, x, "shift", keep)),
            *(_NO_PARAM if post_weight is None else _param(post_weight, x, "post_weight", keep)),
            *(_NO_PARAM if post_bias is None else _param(post_bias, x, "post_bias", keep)),
            x_dt, y_dt, z_dt, _NORM[norm], _NORM[post], eps, post_eps, residual_scale)
        _lib.launch(dev, _lib.load().qattn_block_norm_ex, args)
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

    y has x's shape, and its dtype or float32 (any of the three beside a float32 x); gate broadcasts against x.  post_norm
    ("layer" or "rms", with post_weight and post_bias) normalizes y's rows first.  A float32 y, as
    ``int8_linear(..., out_dtype=torch.float32)`` gives it, is not rounded on its way into the sum."""
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
