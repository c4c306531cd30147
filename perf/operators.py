"""Performance cases of the operators around the attention of a DiT block: adaLN norms, gated residuals and the
INT8 projections.

``listed`` names the cases, ``draw`` gives further ones of the same ranges, ``prepare`` makes what a program holds
before the call (inputs on the GPU, the weight in INT8), ``run`` is one pass, ``work`` the bytes and operations that
no implementation can do without and ``exact`` the same result in 64 bits.  ``own`` chooses what ``run`` calls: the
framework's operators, or their plain form in elementary torch operations.

Kinds of a case:
  norm      ``block_norm``: the norm before a block, modulated by the timestep's scale and shift.
  residual  ``gated_residual_norm``: x + gate * y after a block (y normalized first with ``post``) and the norm before
            the next one.
  linear    ``int8_linear`` of an activation: INT8 rows with a scale per token, times an INT8 weight with a scale per
            channel, bias and activation.
  enter     ``block_norm`` to INT8 rows, then ``int8_linear``: how a block's projections start.
  leave     ``int8_linear``, then ``gated_residual_norm``: how a block's projections end.

Activations have a few channels much larger than the others, as a DiT's have; the modulation is in float32 and small.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EPS = 1e-6
_MOST = 75600 * 5120  # values of the largest activation
_MOST_OPS = 2 * 75600 * 5120 * 13824


def _norm(name, B, L, C, dtype="bf16", norm="layer", affine=False, mod="batch"):
    return {"name": name, "kind": "norm", "B": B, "L": L, "C": C, "dtype": dtype, "norm": norm, "affine": affine,
            "mod": mod}


def _residual(name, B, L, C, dtype="bf16", norm="layer", affine=False, mod="batch", post=False):
    return {**_norm(name, B, L, C, dtype, norm, affine, mod), "kind": "residual", "post": post}


def _linear(name, M, K, N, dtype="bf16", act="none", bias=True):
    return {"name": name, "kind": "linear", "M": M, "K": K, "N": N, "dtype": dtype, "act": act, "bias": bias}


def listed():
    return [
        # one token through the smaller model's width: launch and host time
        _residual("residual_one_token", 1, 1, 1536),
        # Wan2.1-1.3B 480p x 81 frames: the norm before the self-attention
        _norm("wan1.3b_480p_norm", 1, 32760, 1536),
        # Wan2.1-14B 720p x 81 frames: the gated residual after the attention and the norm before the FFN
        _residual("wan14b_720p_residual", 1, 75600, 5120),
        # two clips of three 480p frames with a timestep of its own for every token, the block's output normalized
        # before it is added, RMS norms with weights, fp16
        _residual("token_timesteps", 2, 4680, 5120, "fp16", "rms", True, "token", True),
        # a width and a length that divide into nothing, float32
        _norm("odd_width_fp32", 3, 777, 1027, "fp32", "rms", True, "batch"),
        # one token: the conditioning vector's projection, the weight is what is read
        _linear("linear_one_token", 1, 1536, 9216, "bf16", "silu"),
        # the text embedding of 512 context tokens (4096 -> 5120), GELU
        _linear("text_embedding", 512, 4096, 5120, "bf16", "gelu_tanh"),
        # one 480p latent frame of a streaming model through the FFN's second product
        _linear("frame_ffn_down", 1560, 8960, 1536),
        # sizes that divide into nothing, fp16
        _linear("odd_linear", 777, 1027, 999, "fp16", "none", False),
        # Wan2.1-14B 720p: the FFN's first product, the largest call
        _linear("wan14b_720p_ffn_up", 75600, 5120, 13824, "bf16", "gelu_tanh"),
        # Wan2.1-1.3B 480p: norm, modulation and the Q, K, V projections
        {"name": "wan1.3b_480p_qkv", "kind": "enter", "B": 1, "L": 32760, "C": 1536, "N": 4608, "dtype": "bf16",
         "norm": "layer", "affine": False, "mod": "batch", "act": "none"},
        # ... and the FFN's second product, the gated residual and the next block's norm
        {"name": "wan1.3b_480p_ffn_end", "kind": "leave", "B": 1, "L": 32760, "K": 8960, "C": 1536, "dtype": "bf16",
         "norm": "layer", "affine": False, "mod": "batch"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng):
    w = _log_int(rng, 64, 14000)
    return w if rng.random() < 0.3 else max(64, w // 128 * 128)


def draw(rng):
    kind = rng.choice(["norm", "norm", "residual", "residual", "linear", "linear", "linear", "enter", "leave"])
    c = {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if kind in ("linear", "enter", "leave"):
        c["dtype"] = rng.choice(["bf16", "bf16", "fp16"])
    rows = _log_int(rng, 1, 75600)
    if kind == "linear":
        K, N = _width(rng), _width(rng)
        while 2 * rows * K * N > _MOST_OPS or rows * max(K, N) > 2 * _MOST:
            rows = rows // 2 + 1
        return {**c, "M": rows, "K": K, "N": N, "act": rng.choice(["none", "gelu_tanh", "silu"]),
                "bias": rng.random() < 0.7}
    B = rng.choice([1, 1, 2, 3])
    C = min(_width(rng), 8192)
    most = _MOST if c["dtype"] != "fp32" else _MOST // 2
    mod = rng.choice(["none", "batch", "batch", "token"])
    if mod == "token":
        most //= 4
    rows = max(1, min(rows, most // C) // B)
    c.update(B=B, L=rows, C=C, norm=rng.choice(["layer", "rms"]), affine=rng.random() < 0.4, mod=mod)
    if kind == "residual":
        c["post"] = rng.random() < 0.3
    elif kind == "enter":
        c.update(N=_width(rng), act="none")
    elif kind == "leave":
        c["K"] = _width(rng)
    other = c.get("N", c.get("K", 0))
    while other and 2 * B * c["L"] * C * other > _MOST_OPS:
        c["L"] = c["L"] // 2 + 1
    return c


def _activation(g, shape, dtype):
    x = torch.randn(shape, generator=g, device="cuda")
    c = torch.rand(shape[-1], generator=g, device="cuda")
    return x.mul_(torch.where(c > 0.99, 12.0, 0.4 + c)).to(dtype)


def _weight(g, N, K):
    """An INT8 weight [N, K] and the scale of each channel, as a quantized checkpoint holds them."""
    w = torch.randn((N, K), generator=g, device="cuda") * (0.5 + torch.rand((N, 1), generator=g, device="cuda"))
    t = w.abs().amax(1, keepdim=True) / (127.0 * math.sqrt(K))
    return torch.round(w / (t * math.sqrt(K))).to(torch.int8), t.squeeze(1).contiguous()


def _modulation(g, case, std, one=0.0):
    mod = case["mod"]
    if mod == "none":
        return None
    shape = (case["B"], case["L"] if mod == "token" else 1, case["C"])
    return torch.randn(shape, generator=g, device="cuda").mul_(std).add_(one)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPE[case["dtype"]]
    s = {"case": case}
    kind = case["kind"]
    if kind == "linear":
        s["x"] = _activation(g, (case["M"], case["K"]), dtype)
        w = _weight(g, case["N"], case["K"])
        bias = torch.randn(case["N"], generator=g, device="cuda") * 0.2 if case["bias"] else None
    else:
        shape = (case["B"], case["L"], case["C"])
        s["x"] = _activation(g, shape, dtype)
        s["scale"], s["shift"] = _modulation(g, case, 0.2), _modulation(g, case, 0.2)
        s["w"] = torch.rand(case["C"], generator=g, device="cuda") + 0.5 if case["affine"] else None
        s["b"] = None
        if case["affine"] and case["norm"] == "layer":
            s["b"] = torch.randn(case["C"], generator=g, device="cuda") * 0.1
        if kind in ("residual", "leave"):
            s["gate"] = _modulation(g, case, 0.3, 0.2)
        if kind == "residual":
            s["y"] = torch.randn(shape, generator=g, device="cuda").to(dtype)
            s["post"] = torch.rand(case["C"], generator=g, device="cuda") + 0.5 if case["post"] else None
        elif kind == "enter":
            w = _weight(g, case["N"], case["C"])
            bias = torch.randn(case["N"], generator=g, device="cuda") * 0.2
        elif kind == "leave":
            s["y"] = _activation(g, (case["B"], case["L"], case["K"]), dtype)
            w = _weight(g, case["C"], case["K"])
            bias = torch.randn(case["C"], generator=g, device="cuda") * 0.2
    if kind in ("linear", "enter", "leave"):
        s["codes"], s["channel"] = w
        s["bias"] = bias
        if own:
            from telefuser_amd.linear import Int8Weight

            s["weight"] = Int8Weight(*w, bias)
    return s


# ---- the plain form ------------------------------------------------------------------------------------------------
def _plain_norm(h, s):
    if s["case"]["norm"] == "layer":
        h = h - h.mean(-1, keepdim=True)
    n = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + _EPS)
    if s["w"] is not None:
        n = n * s["w"]
    if s["b"] is not None:
        n = n + s["b"]
    if s["scale"] is not None:
        n = n * (1 + s["scale"]) + s["shift"]
    return n


def _plain_linear(x, s, act="none"):
    """x in 64 bits, where a value next to the border of two codes would otherwise take the other one."""
    top = x.abs().amax(-1, keepdim=True)
    codes = torch.round(x * 127 / torch.where(top > 0, top, 1.0))
    y = codes.float().reshape(-1, codes.shape[-1]) @ s["codes"].float().t()
    y = y.reshape(*codes.shape[:-1], -1) * (top / 127).float() * s["channel"]
    if s["bias"] is not None:
        y = y + s["bias"]
    if act == "gelu_tanh":
        y = y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y))
    elif act == "silu":
        y = y * torch.sigmoid(y)
    return y


def _plain_residual(y, s):
    if s.get("post") is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + _EPS) * s["post"]
    return s["x"].float() + (y if s["gate"] is None else y * s["gate"])


def _run_plain(s):
    kind, dtype = s["case"]["kind"], s["x"].dtype
    if kind == "norm":
        return _plain_norm(s["x"].float(), s).to(dtype)
    if kind == "residual":
        h = _plain_residual(s["y"].float(), s)
        return h.to(dtype), _plain_norm(h, s).to(dtype)
    if kind == "linear":
        return _plain_linear(s["x"].double(), s, s["case"]["act"]).to(dtype)
    if kind == "enter":
        return _plain_linear(_plain_norm(s["x"].double(), s), s).to(dtype)
    h = _plain_residual(_plain_linear(s["y"].double(), s), s)
    return h.to(dtype), _plain_norm(h, s).to(dtype)


# ---- the framework's operators -------------------------------------------------------------------------------------
def _run_own(s):
    from telefuser_amd.linear import int8_linear
    from telefuser_amd.norm import block_norm, gated_residual_norm

    c = s["case"]
    kind = c["kind"]
    if kind == "linear":
        return int8_linear(s["x"], s["weight"], act=c["act"])
    how = {"norm": c["norm"], "weight": s["w"], "bias": s["b"], "scale": s["scale"], "shift": s["shift"], "eps": _EPS}
    if kind == "norm":
        return block_norm(s["x"], **how)
    if kind == "enter":
        return int8_linear(block_norm(s["x"], **how, out_dtype=torch.int8), s["weight"], out_dtype=s["x"].dtype)
    if kind == "leave":  # the product reaches the sum in float32, as in the plain form
        y = int8_linear(s["y"], s["weight"], out_dtype=torch.float32)
        return gated_residual_norm(s["x"], y, s["gate"], **how)
    post = {} if s["post"] is None else {"post_norm": "rms", "post_weight": s["post"]}
    return gated_residual_norm(s["x"], s["y"], s["gate"], **post, **how)


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": M * K * e + N * K + 4 * N * (1 + case["bias"]) + M * N * e, "flops": 2 * M * N * K}
    R, C = case["B"] * case["L"], case["C"]
    params = {"none": 0, "batch": case["B"] * C * 4, "token": R * C * 4}[case["mod"]]
    vectors = 4 * C * (case["affine"] * (2 if case["norm"] == "layer" else 1) + bool(case.get("post")))
    if case["kind"] == "norm":
        return {"bytes": 2 * R * C * e + 2 * params + vectors, "flops": 8 * R * C}
    if case["kind"] == "residual":
        return {"bytes": 4 * R * C * e + 3 * params + vectors, "flops": (10 + 4 * case["post"]) * R * C}
    if case["kind"] == "enter":
        N = case["N"]
        return {"bytes": R * C * e + 2 * params + vectors + N * C + 8 * N + R * N * e, "flops": 2 * R * N * C + 8 * R * C}
    K = case["K"]
    return {"bytes": R * K * e + K * C + 8 * C + 3 * R * C * e + 3 * params + vectors,
            "flops": 2 * R * K * C + 10 * R * C}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------
def _exact_product(x, s):
    largest = torch.linalg.vector_norm(x, math.inf, dim=-1, keepdim=True)
    step = largest / 127
    q = torch.where(largest > 0, (127 * x / largest).round(), torch.zeros_like(x))
    out = torch.mm(q.flatten(0, -2), s["codes"].double().t().contiguous()).unflatten(0, x.shape[:-1])
    out.mul_(step).mul_(s["channel"].double())
    return out if s["bias"] is None else out.add_(s["bias"].double())


def _exact_norm(x, s):
    if s["case"]["norm"] == "rms":
        z = x / torch.sqrt(x.square().mean(-1, keepdim=True) + _EPS)
    else:
        var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
        z = (x - mean) / torch.sqrt(var + _EPS)
    if s["w"] is not None:
        z *= s["w"].double()
    if s["b"] is not None:
        z += s["b"].double()
    return z if s["scale"] is None else z + z * s["scale"].double() + s["shift"].double()


def exact(case, seed):
    s = prepare(case, seed)
    x, kind = s["x"].double(), case["kind"]
    if kind == "norm":
        return _exact_norm(x, s)
    if kind == "enter":
        return _exact_product(_exact_norm(x, s), s)
    if kind == "linear":
        y = _exact_product(x, s)
        if case["act"] == "silu":
            return y / (1 + torch.exp(-y))
        if case["act"] == "gelu_tanh":
            inner = torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y.pow(3)))
            return inner.add_(1).mul_(y).mul_(0.5)
        return y
    y = s["y"].double()
    if kind == "leave":
        y = _exact_product(y, s)
    elif s["post"] is not None:
        y = s["post"].double() * y / torch.sqrt(y.square().mean(-1, keepdim=True) + _EPS)
    h = x + y if s["gate"] is None else torch.addcmul(x, y, s["gate"].double())
    return h, _exact_norm(h, s)
