"""Cross entropy of feature rows over a large vocabulary of embeddings (MI355X matrix cores).

What the clip head's unit features (``FieldHeads.get_clip_outputs_from_feature``, ``pogs/fields/gaussian_field.py:194-204``)
are trained and scored on when every pixel has a label in a table of phrase embeddings.  The value and the gradients of
``torch.nn.functional.cross_entropy(scale * features @ vocabulary.T, labels)``, without the ``[rows, words]`` logits: the
forward pass keeps one maximum and sum a row, the backward pass makes the products again for one piece of the vocabulary
at a time.  (Up to 128 rows of a large vocabulary do keep them for it, 4 bytes each, and read the vocabulary as it is.)
Products take 16-bit operands and add in float32.  Of float32 input 2^-21 of a product at most is left out: few rows take it
in three bfloat16 pieces, all 24 bits; otherwise the logits take every row and every word by a power of two of its own, in 22
bits (a value below 2^-15 of its row's largest to 2^-38 of that).  The gradients' products are made of bfloat16 pieces, which
hold each softmax entry to 2^-24 (float32 input) or 2^-16, beside rows, words and weights up to 2^130 times as large.
Results do not depend on the order in which workgroups run; a call with gradients to come and one without may take different
kernels and differ in the last bits.  HIP kernels only (``pr_vocab_ce_fwd``, ``pr_vocab_ce_bwd``); there is no CPU path.
"""
from __future__ import annotations

import math
from typing import Tuple, Union

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib
from .rendering import _call, _on, _ptr, _raw_stream, _refuse_dual

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}     # PR_F32, PR_F16, PR_BF16
_REDUCTIONS = ("none", "sum", "mean")


def _scratch(nbytes: int, device) -> Tensor:
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def _forward(x, w, labels, scale, ignore_index, reduction, want_lse, with_grad, stream):
    """``x [P, D]``, ``w [V, D]``, ``labels [P]`` int64 -> loss (``[P]`` or 0-d), lse ``[P]`` or None, what backward keeps."""
    (P, D), V, dev = x.shape, w.shape[0], x.device
    lse = torch.empty(P, dtype=torch.float32, device=dev) if want_lse else None
    loss = torch.empty(P if reduction == "none" else (), dtype=torch.float32, device=dev)
    if P == 0:
        if reduction != "none":
            loss.fill_(math.nan if reduction == "mean" else 0.0)
        return loss, lse, None
    lib, t = _lib.load(), _TYPES[x.dtype]
    # few rows and no gradient to come: nothing is packed and nothing kept
    plain = not with_grad and (P <= lib.pr_vocab_ce_score_rows() or not lib.pr_vocab_ce_keeps_vocabulary(P, V, D))
    kept = None if plain else _scratch(lib.pr_vocab_ce_kept_bytes(t, P, V, D), dev)
    scratch = _scratch(lib.pr_vocab_ce_fwd_scratch_bytes(t, P, V, D), dev)
    per_row, scalar = (loss, None) if reduction == "none" else (None, loss)
    with _on(dev):
        _call("pr_vocab_ce_fwd", t, P, V, D, _ptr(x), *x.stride(), _ptr(w), *w.stride(), _ptr(labels), ignore_index, scale,
              int(reduction == "mean"), _ptr(kept), 0 if plain else kept.numel(), _ptr(scratch), scratch.numel(),
              _ptr(per_row), _ptr(lse), _ptr(scalar), stream)
    return loss, lse, kept


class _VocabularyCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, labels, scale, ignore_index, reduction, want_lse, stream):
        ctx.set_materialize_grads(False)
        ctx.args = x.shape, w.shape[0], x.dtype, scale, ignore_index, reduction
        loss, lse, kept = _forward(x, w, labels, scale, ignore_index, reduction, want_lse, True, stream)
        # kept has its own copy of the features and, but for few rows, of the vocabulary
        again = kept is not None and ctx.needs_input_grad[0] and not _lib.load().pr_vocab_ce_keeps_vocabulary(len(x), *w.shape)
        ctx.save_for_backward(labels, kept, w if again else None)
        return loss, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, g_loss, g_lse):
        labels, kept, w = ctx.saved_tensors
        (P, D), V, dtype, scale, ignore_index, reduction = ctx.args
        want_x, want_w = ctx.needs_input_grad[:2]
        dev = labels.device
        empty = P == 0 or (g_loss is None and g_lse is None)
        make = torch.zeros if empty else torch.empty
        dx = make(P, D, dtype=dtype, device=dev) if want_x else None
        dw = make(V, D, dtype=dtype, device=dev) if want_w else None
        if not empty:
            g_loss = None if g_loss is None else g_loss.float().contiguous()
            g_lse = None if g_lse is None else g_lse.float().contiguous()
            lib, t = _lib.load(), _TYPES[dtype]
            scratch = _scratch(lib.pr_vocab_ce_bwd_scratch_bytes(t, P, V, D, int(want_x), int(want_w)), dev)
            with _on(dev):
                _call("pr_vocab_ce_bwd", t, P, V, D, _ptr(w), *(w.stride() if w is not None else (0, 0)), _ptr(labels),
                      ignore_index, scale, int(reduction == "mean"), int(reduction == "none"), _ptr(kept), kept.numel(),
                      _ptr(g_loss), _ptr(g_lse), _ptr(scratch), scratch.numel(), _ptr(dx), _ptr(dw), _raw_stream(dev.index))
        return (dx, dw) + (None,) * 6


_STREAM_KEY = "pogs_amd.stream"


def _mark_leaves(output: Tensor, stream: int, reshaped: bool) -> None:
    """Marks the gradient nodes of the leaves among features and vocabulary with the stream that they came up on.  A leaf's
    node lives as long as any graph of it does and keeps its first stream; a backward pass captured on another stream would
    make that one part of the capture, which ends the process.  So the call that would lead there is refused.
    ``reshaped``: the features are a leaf, and the call has made rows of them itself."""
    for node, _ in output.grad_fn.next_functions[:2]:
        while reshaped and node is not None and not hasattr(node, "variable"):
            node = node.next_functions[0][0]
        reshaped = False
        if node is not None and hasattr(node, "variable"):     # a leaf's
            if node.metadata.setdefault(_STREAM_KEY, stream) != stream and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a graph of the same features or vocabulary, made outside the capture, is still alive: "
                                   "its backward pass cannot be captured; drop that graph's outputs first")


def _check(features: Tensor, vocabulary: Tensor, labels: Tensor, scale: float, reduction: str) -> float:
    if vocabulary.dim() != 2 or 0 in vocabulary.shape:
        raise ValueError(f"the vocabulary must be [words, dims] and not empty, got {tuple(vocabulary.shape)}")
    if features.dim() < 1 or features.shape[-1] != vocabulary.shape[1]:
        raise ValueError(f"features {tuple(features.shape)} do not end in the vocabulary's {vocabulary.shape[1]} dims")
    if labels.shape != features.shape[:-1]:
        raise ValueError(f"labels must be {tuple(features.shape[:-1])}, one a feature row, got {tuple(labels.shape)}")
    if labels.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"labels must be int64 or int32, got {labels.dtype}")
    if features.dtype != vocabulary.dtype or features.dtype not in _TYPES:
        raise TypeError("features and vocabulary must both be float32, float16 or bfloat16, got "
                        f"{features.dtype} and {vocabulary.dtype}")
    if isinstance(scale, Tensor):
        raise TypeError("scale is a plain number; multiply the features by a learned one")
    if not abs(scale) <= 1e38:
        raise ValueError(f"scale must be finite (within 1e38), got {scale}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {_REDUCTIONS}, got {reduction!r}")
    _refuse_dual("vocabulary_cross_entropy", (features, vocabulary))
    if not features.is_cuda:
        raise RuntimeError("pogs_amd.vocabulary runs on a HIP device only (no CPU fallback)")
    if not features.device == vocabulary.device == labels.device:
        raise RuntimeError("features, vocabulary and labels are on different devices")
    return float(scale)


def vocabulary_cross_entropy(features: Tensor, vocabulary: Tensor, labels: Tensor, scale: float = 1.0,
                             ignore_index: int = -100, reduction: str = "mean",
                             return_lse: bool = False) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """Cross entropy of ``scale * features @ vocabulary.T`` against ``labels``, without the logits.

    ``features``: ``[..., D]`` and ``vocabulary``: ``[V, D]``, both float32, float16 or bfloat16, any strides;
    ``labels``: ``[...]`` int64 or int32.  Returns float32: the mean over the rows whose label is not ``ignore_index``
    (NaN if there are none, as in torch), their ``"sum"``, or with ``"none"`` one value a row (0 for an ignored one);
    with ``return_lse`` also every row's ``log sum_v exp(scale <x, w_v>)`` (0 for an ignored row).  Differentiable in
    features and vocabulary, through the loss and the log-sum (gradients in the inputs' type, from the formula; not
    twice, and not in forward mode, which is refused).  Ignored rows contribute nothing, even if their features are not finite; the loss and log-sum of a row with an
    infinite logit are NaN.  A label that is neither in
    ``0..V-1`` nor ``ignore_index`` makes its row's loss NaN and the gradients with it: nothing is read out of range,
    and the host does not wait to look.  Features may be changed in place before the backward pass, labels may not, and
    neither may the vocabulary where it is large and the rows are at most 128 (autograd refuses).  Safe in a captured
    graph, gradients included, as long as no graph of the same leaves made outside the capture is alive (refused where one
    of this function is)."""
    scale = _check(features, vocabulary, labels, scale, reduction)
    D = features.shape[-1]
    x = features if features.dim() == 2 else features.reshape(-1, D)
    flat = labels if labels.dim() == 1 else labels.reshape(-1)
    if flat.dtype != torch.int64 or not flat.is_contiguous():
        flat = flat.to(torch.int64).contiguous()
    stream = _raw_stream(x.device.index)
    args = x, vocabulary, flat, scale, int(ignore_index), reduction, return_lse
    if torch.is_grad_enabled() and (x.requires_grad or vocabulary.requires_grad):
        loss, lse = _VocabularyCrossEntropy.apply(*args, stream)
        _mark_leaves(loss, stream, x is not features and features.is_leaf)
    else:
        loss, lse, _ = _forward(*args, False, stream)
    if reduction == "none" and labels.dim() != 1:
        loss = loss.reshape(labels.shape)
    return (loss, lse.reshape(labels.shape)) if return_lse else loss
