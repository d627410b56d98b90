"""LayerNorm of the last dimension for rows of any width in float32, bfloat16
or float16, with its backward pass (cign_layer_norm_fwd/_bwd).

``fused_block_ops`` has the block's norms (float32, up to 1024 wide, with
dropout or an addend) and ``jk_norm`` the output norm over the block states
(float32, up to 2048 wide); :func:`layer_norm` takes the rows they refuse: a
deeper model's output norm, half-precision rows, rows of a wider buffer, norms
without weight or bias.  Statistics and sums are float32 for every type, the
weight and bias gradients are summed in a fixed order, and y, grad x, grad
weight and grad bias are rounded once.  A row whose level is far above its
spread keeps its digits: what the mean's own rounding leaves is taken out.
Rows with a spread above about 1e19, whose squares leave float32's range, come
out as the bias.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib


def _ptr(t):
    return None if t is None else t.data_ptr()


def _forward(x, ldx, weight, bias, eps, need_stats):
    n, d = x.shape
    y = x.new_empty((n, d))
    param = x if weight is None and bias is None else (bias if weight is None else weight)
    stats = mean = rstd = None
    if need_stats:  # mean [n], then rstd [n]
        stats = torch.empty((2 * n,), dtype=torch.float32, device=x.device)
        mean = stats.data_ptr()
        rstd = mean + 4 * n
    _lib.launch("cign_layer_norm_fwd", x, n, d, _lib.TYPE_CODES[x.dtype],
                _lib.TYPE_CODES[param.dtype], x.data_ptr(), ldx, _ptr(weight), _ptr(bias), eps,
                y.data_ptr(), mean, rstd)
    return y, stats


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        rows, ldx = _lib.rows_of(x)
        y, stats = _forward(rows, ldx, weight, bias, eps, True)
        ctx.save_for_backward(rows, weight, stats)
        ctx.ldx = ldx
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @_lib.once
    def backward(ctx, gy):
        x, weight, stats = ctx.saved_tensors
        n, d = x.shape
        gy, ldg = _lib.rows_of(gy)
        want_x, want_w, want_b, _ = ctx.needs_input_grad
        param = ctx.bias_dtype or (x if weight is None else weight).dtype
        gx = x.new_empty((n, d)) if want_x else None
        gw = weight.new_empty((d,)) if want_w else None
        gb = torch.empty((d,), dtype=ctx.bias_dtype, device=x.device) if want_b else None
        ws, ws_bytes = None, 0
        if want_w or want_b:
            ws_bytes = _lib.load_library().cign_layer_norm_bwd_workspace_bytes(n, d)
            ws = _lib.workspace(ws_bytes, x.device)
        mean = stats.data_ptr()
        _lib.launch("cign_layer_norm_bwd", x, n, d, _lib.TYPE_CODES[x.dtype],
                    _lib.TYPE_CODES[param], gy.data_ptr(), ldg, x.data_ptr(), ctx.ldx,
                    _ptr(weight), mean, mean + 4 * n, _ptr(gx), _ptr(gw), _ptr(gb), _ptr(ws),
                    ws_bytes)
        return gx, gw, gb, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """LayerNorm of x's last dimension: (x - mean) / sqrt(var + eps) * weight + bias.

    x: CUDA float32, bfloat16 or float16, any leading dimensions; the rows may
    lie in a wider buffer.  weight, bias: [D] or None, both of one type, x's or
    float32.  Gradients flow to x, weight and bias (once: a second derivative
    raises, as forward mode does)."""
    if x.device.type != "cuda" or x.dtype not in _lib.TYPE_CODES:
        raise TypeError("x must be CUDA float32, bfloat16 or float16")
    if x.dim() < 1 or x.size(-1) < 1:
        raise ValueError(f"x must be [..., D] with D >= 1, got {tuple(x.shape)}")
    d = x.size(-1)
    eps = float(eps)
    if not (0.0 <= eps < float("inf")):
        raise ValueError("eps must be finite and not negative")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.device != x.device or p.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"{name} must be on x's device, of x's type or float32")
        if p.shape != (d,):
            raise ValueError(f"{name} must be [{d}], got {tuple(p.shape)}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError("weight and bias must have the same type")
    rows = x if x.dim() == 2 else x.reshape(-1, d)
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        y = _LayerNormFn.apply(rows, weight, bias, eps)
    else:
        _lib.refuse_tangents("layer_norm", x, weight, bias)
        rows, ldx = _lib.rows_of(rows)
        y = _forward(rows, ldx, weight, bias, eps, False)[0]
    return y if x.dim() == 2 else y.view(x.shape)
