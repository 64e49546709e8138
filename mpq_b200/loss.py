"""Softmax cross entropy of an output head over its whole vocabulary, from the hidden states, with its gradients.

    loss = vocab_cross_entropy(hidden, model.lm_head.weight, labels)        # mean over the labels that count
    nll = vocab_cross_entropy(hidden, weight, labels, reduction="none")     # scores of tokens, for a perplexity

The logits (tokens x vocabulary) are not stored: the forward pass reduces them tile by tile inside the product.  The
backward pass takes the vocabulary in pieces.  It computes a piece's logits again, except for the first columns, which
the forward pass keeps in 16 bits where a gradient is wanted and ``keep_bytes`` has room: that saves their product and
costs digits (probabilities within 2^-12.5 of themselves, and none below 2^-32 of the largest beside them).  With
``keep_bytes=0`` nothing of the logits' size outlives a call.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import ops
from ._lib import call_on, load, ptr

_DTYPES = {torch.bfloat16: 1, torch.float16: 2}
_REDUCTIONS = ("none", "sum", "mean")
PIECE_BYTES = 1 << 30  # default room for the piece of the logits' gradient that the backward pass holds at a time
KEEP_BYTES = 1 << 31   # default room for what the forward pass keeps for the backward pass


def _operand(x: torch.Tensor) -> torch.Tensor:
    """x (2-D, 16 bits) as the tensor loads take it: unit column stride, rows and base on 16-byte boundaries.  Whole
    multiples of 8 columns pass as they are; other widths are copied into padded rows."""
    rows, cols = x.shape
    if x.numel() == 0 or (x.stride(1) == 1 and x.stride(0) % 8 == 0 and x.stride(0) >= cols and x.data_ptr() % 16 == 0):
        return x
    padded = torch.empty(rows, (cols + 7) // 8 * 8, device=x.device, dtype=x.dtype)
    padded[:, :cols].copy_(x)
    return padded[:, :cols]


def _piece(tokens: int, vocab: int, piece: Optional[int]) -> int:
    """Columns of the vocabulary that the backward pass takes at a time, a multiple of 256."""
    most = (vocab + 255) // 256 * 256
    if piece is None:
        piece = max(PIECE_BYTES // (2 * max(tokens, 1)), 256) // 256 * 256
    return max(256, min((int(piece) + 255) // 256 * 256, most))


def _keep(tokens: int, vocab: int, keep_bytes: int) -> int:
    """Columns of the vocabulary that fit in keep_bytes at two bytes a token: all, or a multiple of 256."""
    cols = int(keep_bytes) // (2 * max(tokens, 1))
    return vocab if cols >= (vocab + 7) // 8 * 8 else cols // 256 * 256


def _forward(hidden, weight, labels, ignore_index, reduction, keep_bytes):
    """(result, work, keep, keep_cols) of a checked call.  ``work`` holds, as floats: lse (T), the count of labels, the
    scores for the backward pass (T), the scores (T, unless they are the result) and, from 8 bytes on, the tiles' partial
    sums."""
    t, h = hidden.shape
    v = weight.shape[0]
    dev = hidden.device
    x, w = _operand(hidden), _operand(weight)
    tiles = load().mpq_xent_tiles(t, v)
    each = reduction == "none"
    out = torch.empty(t, device=dev, dtype=torch.float32) if each else torch.empty((), device=dev, dtype=torch.float32)
    work = torch.empty(_part_at(t) + 2 * t * tiles, device=dev, dtype=torch.float32)
    at, at_out = work.data_ptr(), out.data_ptr()
    keep_cols = _keep(t, v, keep_bytes) if keep_bytes and t else 0
    ldk = (keep_cols + 7) // 8 * 8
    keep = torch.empty(t, ldk, device=dev, dtype=hidden.dtype) if keep_cols else None
    call_on(dev.index, "mpq_xent_forward", t, v, h, _DTYPES[hidden.dtype], x.data_ptr(), x.stride(0), w.data_ptr(),
            w.stride(0), labels.data_ptr(), ignore_index, at + 4 * _part_at(t), 2 * t * tiles, at + 4 * (t + 1), at,
            at_out if each else at + 4 * (2 * t + 1), _REDUCTIONS.index(reduction), at_out, at + 4 * t, ptr(keep), ldk,
            keep_cols, ops.status_word(dev).data_ptr())
    return out, work, keep, keep_cols


def _part_at(t: int) -> int:
    return (3 * t + 2) // 2 * 2


class _VocabCrossEntropy(torch.autograd.Function):

    @staticmethod
    def forward(ctx, hidden, weight, labels, ignore_index, reduction, piece, keep_bytes):
        out, work, keep, keep_cols = _forward(hidden, weight, labels, ignore_index, reduction, keep_bytes)
        ctx.save_for_backward(hidden, weight, labels)
        ctx.ignore_index, ctx.piece, ctx.mean = ignore_index, piece, reduction == "mean"
        ctx.work, ctx.kept = work, (keep, keep_cols)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, gout):
        hidden, weight, labels = ctx.saved_tensors
        t, h = hidden.shape
        v = weight.shape[0]
        dev = hidden.device
        need_h, need_w = ctx.needs_input_grad[:2]
        dh = torch.empty(t, h, device=dev, dtype=hidden.dtype) if need_h else None
        dw = torch.empty(v, h, device=dev, dtype=weight.dtype) if need_w else None
        if t == 0:
            return dh, dw if dw is None else dw.zero_(), None, None, None, None, None
        x, w = _operand(hidden), _operand(weight)
        gout = gout.to(torch.float32).contiguous()
        # the kept columns turn into their gradient in place: a second pass through the graph computes them again
        (keep, keep_cols), ctx.kept = ctx.kept, (None, 0)
        piece = _piece(t, v - keep_cols, ctx.piece)
        each = gout.dim() > 0  # one upstream gradient a token: d is scaled by the largest
        planes = load().mpq_xent_planes(t, v, h, piece, keep_cols) if need_h else 0
        # FP32 sums of dhidden, and the scale
        acc = torch.empty(planes * t * h + 1, device=dev, dtype=torch.float32) if planes or each else None
        d = torch.empty(t, piece, device=dev, dtype=hidden.dtype) if keep_cols < v else None
        at = ctx.work.data_ptr()
        at_acc = 0 if acc is None else acc.data_ptr()
        call_on(dev.index, "mpq_xent_backward", t, v, h, _DTYPES[hidden.dtype], x.data_ptr(), x.stride(0), w.data_ptr(),
                w.stride(0), labels.data_ptr(), ctx.ignore_index, at, gout.data_ptr(), int(each),
                at + 4 * t if ctx.mean else None, at + 4 * _part_at(t), at + 4 * (t + 1), ptr(keep),
                0 if keep is None else keep.shape[1], keep_cols, at_acc + 4 * planes * t * h if each else None, ptr(d),
                piece, at_acc if planes else None, ptr(dh), h, ptr(dw), h, ops.status_word(dev).data_ptr())
        return dh, dw, None, None, None, None, None


def vocab_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, *, ignore_index: int = -100,
                        reduction: str = "mean", piece: Optional[int] = None,
                        keep_bytes: int = KEEP_BYTES) -> torch.Tensor:
    """Cross entropy of softmax(hidden @ weight.T) at ``labels``, in float32.

    ``hidden`` (..., H) and ``weight`` (V, H): bfloat16 or float16; ``labels`` (...): integers.  Labels equal to
    ``ignore_index`` do not count (their score is 0, their gradient 0; the mean over no labels is NaN); labels outside
    the vocabulary give NaN.  ``reduction``: "mean" over the labels that count, "sum" or "none" (one score a token).
    Differentiable once in ``hidden`` and ``weight``, whose gradients come in their own type (for the head's, rows of
    ``hidden`` that do not count must be finite all the same: they meet a zero).  ``keep_bytes`` bounds what the forward
    pass keeps for the backward pass (by default 2 GiB; 0: nothing; what was kept serves one backward pass, another through
    the same graph computes it again and may differ in its last digits), ``piece`` the columns of the vocabulary that the
    backward pass computes again at a time (by default what fits in 1 GiB).  Waits inside the kernels are bounded:
    ``ops.check_status`` raises, once the caller synchronises by it, if one ran out and left a result undefined."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {_REDUCTIONS}, got {reduction!r}")
    if not (hidden.is_cuda and weight.is_cuda and labels.is_cuda):
        raise ValueError("mpq_b200 kernels require CUDA tensors (there is no CPU path)")
    if not hidden.device == weight.device == labels.device:
        raise ValueError("vocab_cross_entropy: the tensors are on different devices")
    if hidden.dtype not in _DTYPES or weight.dtype != hidden.dtype:
        raise ValueError(f"vocab_cross_entropy takes bfloat16 or float16 tensors of one type, got {hidden.dtype} and "
                         f"{weight.dtype}")
    if weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"vocab_cross_entropy: hidden {tuple(hidden.shape)} does not fit the head {tuple(weight.shape)}")
    if 0 in weight.shape:
        raise ValueError("vocab_cross_entropy: the head is empty")
    if labels.shape != hidden.shape[:-1]:
        raise ValueError(f"vocab_cross_entropy: labels {tuple(labels.shape)} for hidden {tuple(hidden.shape)}")
    if labels.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"labels must be int64 or int32, got {labels.dtype}")
    if piece is not None and int(piece) < 1:
        raise ValueError("piece must be positive")
    if int(keep_bytes) < 0:
        raise ValueError("keep_bytes must not be negative")
    flat = labels.reshape(-1).to(torch.int64).contiguous()
    rows = hidden if hidden.dim() == 2 else hidden.reshape(-1, hidden.shape[-1])
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        out = _VocabCrossEntropy.apply(rows, weight, flat, int(ignore_index), reduction, piece, int(keep_bytes))
    else:
        out = _forward(rows, weight, flat, int(ignore_index), reduction, 0)[0]
    return out.view(labels.shape) if reduction == "none" else out


__all__ = ["vocab_cross_entropy"]
