"""Log probabilities of the nodes' labels, entropy and best classes from the
classifier's logits, with the gradient of the logits
(cign_node_log_probs_fwd/_bwd).

``-node_log_probs(logits, labels).log_prob`` is the reference's cross entropy
per node (generic_engine/train_cign.py:2103-2148) in one pass over the logits;
a node without a label carries a negative one, so neither a mask nor a gather
of the training rows is needed and the call can be captured in a graph.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib

MAX_TOP = 64


class NodeLogProbs(NamedTuple):
    log_prob: Optional[torch.Tensor]       # [N] float32; None without labels
    entropy: torch.Tensor                  # [N] float32
    top_log_probs: Optional[torch.Tensor]  # [N, top_k] float32; None for top_k = 0
    top_index: Optional[torch.Tensor]      # [N, top_k] int64


def _ptr(t):
    return None if t is None else t.data_ptr()


def _forward(logits, ld, labels, top_k, need_stats):
    n, c = logits.shape
    dev = logits.device
    log_prob = None if labels is None else torch.empty((n,), dtype=torch.float32, device=dev)
    entropy = torch.empty((n,), dtype=torch.float32, device=dev)
    stats = torch.empty((n, 2), dtype=torch.float32, device=dev) if need_stats else None
    top = index = None
    if top_k:
        top = torch.empty((n, top_k), dtype=torch.float32, device=dev)
        index = torch.empty((n, top_k), dtype=torch.int64, device=dev)
    _lib.launch("cign_node_log_probs_fwd", logits, n, c, _lib.TYPE_CODES[logits.dtype],
                logits.data_ptr(), ld, _ptr(labels), top_k, _ptr(log_prob), entropy.data_ptr(),
                _ptr(stats), _ptr(top), _ptr(index))
    return log_prob, entropy, top, index, stats


class _NodeLogProbsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, top_k):
        rows, ld = _lib.rows_of(logits)
        log_prob, entropy, top, index, stats = _forward(rows, ld, labels, top_k, True)
        ctx.save_for_backward(rows, labels, stats, entropy, index)
        ctx.ld = ld
        ctx.top_k = top_k
        ctx.set_materialize_grads(False)
        if index is not None:
            ctx.mark_non_differentiable(index)
        return log_prob, entropy, top, index

    @_lib.once
    def backward(ctx, g_log_prob, g_entropy, g_top, _):
        if g_log_prob is None and g_entropy is None and g_top is None:
            return None, None, None
        logits, labels, stats, entropy, index = ctx.saved_tensors
        n, c = logits.shape
        grad = logits.new_empty((n, c))
        g_top = None if g_top is None else g_top.contiguous()
        _lib.launch("cign_node_log_probs_bwd", logits, n, c, _lib.TYPE_CODES[logits.dtype],
                    logits.data_ptr(), ctx.ld, _ptr(labels), stats.data_ptr(), entropy.data_ptr(),
                    ctx.top_k, _ptr(index), _ptr(g_log_prob),
                    0 if g_log_prob is None else g_log_prob.stride(0), _ptr(g_entropy),
                    0 if g_entropy is None else g_entropy.stride(0), _ptr(g_top), grad.data_ptr())
        return grad, None, None


def node_log_probs(logits: torch.Tensor, labels: Optional[torch.Tensor] = None,
                   top_k: int = 0) -> NodeLogProbs:
    """Per node (row of logits [N, C], CUDA float32, bfloat16 or float16; the
    rows may lie in a wider buffer):

    * log_prob: log softmax at labels[n] (int64 [N]).  A negative label is no
      label: 0, and no gradient.  A label >= C gives NaN.
    * entropy of the softmax.
    * top_log_probs, top_index: the top_k (at most 64) classes, best first;
      equal logits go to the lower class, NaN before everything.

    Logits of -inf mask classes.  A row that masks all of them has log_prob
    -inf (0 without a label), entropy 0 and gradient 0; a row with NaN or +inf
    gives NaN.  Gradients flow from log_prob, entropy and top_log_probs to
    logits (once: a second derivative raises, as forward mode does)."""
    if logits.device.type != "cuda" or logits.dtype not in _lib.TYPE_CODES:
        raise TypeError("logits must be CUDA float32, bfloat16 or float16")
    if logits.dim() != 2 or logits.size(1) < 1:
        raise ValueError(f"logits must be [N, C] with C >= 1, got {tuple(logits.shape)}")
    n, c = logits.shape
    if labels is not None:
        if labels.device != logits.device or labels.dtype != torch.int64:
            raise TypeError("labels must be int64 on the logits' device")
        if labels.shape != (n,):
            raise ValueError(f"labels must be [{n}], got {tuple(labels.shape)}")
        labels = labels.contiguous()
    top_k = int(top_k)
    if not (0 <= top_k <= min(c, MAX_TOP)):
        raise ValueError(f"top_k must be between 0 and min(C, {MAX_TOP}), got {top_k}")
    if torch.is_grad_enabled() and logits.requires_grad:
        return NodeLogProbs(*_NodeLogProbsFn.apply(logits, labels, top_k))
    _lib.refuse_tangents("node_log_probs", logits)
    rows, ld = _lib.rows_of(logits)
    return NodeLogProbs(*_forward(rows, ld, labels, top_k, False)[:4])
