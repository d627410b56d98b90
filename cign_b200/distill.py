"""Distillation of a node classifier from a teacher's best few classes of each
node, as ``node_log_probs(teacher_logits, top_k=...)`` or ``torch.topk`` keeps
them, with the gradient of the student's logits (cign_distill_fwd/_bwd).
"""
from __future__ import annotations

import torch

from . import _lib

MAX_KEPT = 256
MAX_CLASSES = 1 << 20
_TAILS = {"drop": 0, "bucket": 1}
_INDEX_CODES = {torch.int32: 0, torch.int64: 1}


def _teacher_args(values, ld_v, index, ld_i):
    return (values.size(1), _lib.TYPE_CODES[values.dtype], values.data_ptr(), ld_v,
            _INDEX_CODES[index.dtype], index.data_ptr(), ld_i)


def _forward(logits, ld, values, ld_v, index, ld_i, temperature, tail, need_stats):
    n, c = logits.shape
    dev = logits.device
    loss = torch.empty((n,), dtype=torch.float32, device=dev)
    stats = torch.empty((n, 8), dtype=torch.float32, device=dev) if need_stats else None
    _lib.launch("cign_distill_fwd", logits, n, c, _lib.TYPE_CODES[logits.dtype], logits.data_ptr(),
                ld, *_teacher_args(values, ld_v, index, ld_i), temperature, tail, loss.data_ptr(),
                None if stats is None else stats.data_ptr())
    return loss, stats


class _DistillFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, values, index, temperature, tail):
        rows, ld = _lib.rows_of(logits)
        values, ld_v = _lib.rows_of(values)
        index, ld_i = _lib.rows_of(index)
        loss, stats = _forward(rows, ld, values, ld_v, index, ld_i, temperature, tail, True)
        ctx.save_for_backward(rows, values, index, stats)
        ctx.args = ld, ld_v, ld_i, temperature, tail
        return loss

    @_lib.once
    def backward(ctx, g_loss):
        logits, values, index, stats = ctx.saved_tensors
        ld, ld_v, ld_i, temperature, tail = ctx.args
        n, c = logits.shape
        grad = logits.new_empty((n, c))
        _lib.launch("cign_distill_bwd", logits, n, c, _lib.TYPE_CODES[logits.dtype],
                    logits.data_ptr(), ld, *_teacher_args(values, ld_v, index, ld_i), temperature,
                    tail, stats.data_ptr(), g_loss.data_ptr(), g_loss.stride(0), grad.data_ptr())
        return grad, None, None, None, None


def distill_top_logits(logits: torch.Tensor, teacher_values: torch.Tensor,
                       teacher_index: torch.Tensor, temperature: float = 1.0,
                       tail: str = "drop") -> torch.Tensor:
    """temperature^2 * KL(teacher || student) per node, float32 [N].

    logits: [N, C], CUDA float32, bfloat16 or float16 (rows may lie in a wider
    buffer, C <= 2^20); the student is softmax(logits / temperature), temperature
    between 1e-3 and 1e6.
    teacher_values, teacher_index: [N, K] (K <= 256; float32, bfloat16 or
    float16; int32 or int64), the kept classes in any order.  An entry with a
    negative index or the value -inf is absent; an index >= C makes its row
    NaN; a class that occurs twice counts with both entries.

    tail "drop": the teacher is softmax(teacher_values / temperature) over the
    kept classes.  tail "bucket": teacher_values are the teacher's log
    probabilities at the temperature, and what they leave of 1 is one more
    class, compared with the student's probability of all the other classes.

    The student's log sum is float32: at temperatures far above the logits'
    spread, where p and q are nearly equal, the gradient of a kept class,
    temperature * (p - q), is known to about temperature * 2^-22.

    A node without entries has loss 0 and gradient 0; a student row of -inf
    only has loss inf and gradient 0.  A kept class that the student masks
    (-inf) gives loss inf, unless the teacher's probability of it is 0 in 64
    bits (its logarithm below about -745, as a mask of -1e4 leaves it): then
    the class takes no part.  The gradient flows to logits (once: a
    second derivative raises, as forward mode does); the teacher's tensors are
    constants."""
    if logits.device.type != "cuda" or logits.dtype not in _lib.TYPE_CODES:
        raise TypeError("logits must be CUDA float32, bfloat16 or float16")
    if teacher_values.device != logits.device or teacher_values.dtype not in _lib.TYPE_CODES:
        raise TypeError("teacher_values must be float32, bfloat16 or float16 on the logits' device")
    if teacher_index.device != logits.device or teacher_index.dtype not in _INDEX_CODES:
        raise TypeError("teacher_index must be int32 or int64 on the logits' device")
    if logits.dim() != 2 or not (1 <= logits.size(1) <= MAX_CLASSES):
        raise ValueError(f"logits must be [N, C] with 1 <= C <= {MAX_CLASSES}, "
                         f"got {tuple(logits.shape)}")
    if teacher_values.dim() != 2 or teacher_values.size(0) != logits.size(0) or \
            not (1 <= teacher_values.size(1) <= MAX_KEPT):
        raise ValueError(f"teacher_values must be [{logits.size(0)}, K] with 1 <= K <= {MAX_KEPT}, "
                         f"got {tuple(teacher_values.shape)}")
    if teacher_index.shape != teacher_values.shape:
        raise ValueError("teacher_values and teacher_index must have the same shape")
    if teacher_values.requires_grad:
        raise ValueError("teacher_values are constants here: detach them")
    temperature = float(temperature)
    if not (1e-3 <= temperature <= 1e6):
        raise ValueError(f"temperature must be between 1e-3 and 1e6, got {temperature}")
    if tail not in _TAILS:
        raise ValueError(f"tail must be 'drop' or 'bucket', got {tail!r}")
    if torch.is_grad_enabled() and logits.requires_grad:
        return _DistillFn.apply(logits, teacher_values, teacher_index, temperature, _TAILS[tail])
    _lib.refuse_tangents("distill_top_logits", logits, teacher_values)
    rows, ld = _lib.rows_of(logits)
    values, ld_v = _lib.rows_of(teacher_values)
    index, ld_i = _lib.rows_of(teacher_index)
    return _forward(rows, ld, values, ld_v, index, ld_i, temperature, _TAILS[tail], False)[0]
