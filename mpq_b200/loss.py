"""Softmax cross entropy of an output head over its whole vocabulary, from the hidden states, with its gradients.

    loss = vocab_cross_entropy(hidden, model.lm_head.weight, labels)        # mean over the labels that count
    nll = vocab_cross_entropy(hidden, weight, labels, reduction="none")     # scores of tokens, for a perplexity

The logits (tokens x vocabulary) are never stored: the forward pass reduces them tile by tile inside the product, and
the backward pass computes them again a piece of the vocabulary at a time.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import ops
from ._lib import call, load, ptr

_DTYPES = {torch.bfloat16: 1, torch.float16: 2}
_REDUCTIONS = ("mean", "sum", "none")
PIECE_BYTES = 1 << 30  # default room for the piece of the logits' gradient that the backward pass holds at a time


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


class _VocabCrossEntropy(torch.autograd.Function):

    @staticmethod
    def forward(ctx, hidden, weight, labels, ignore_index, reduction, piece):
        t, h = hidden.shape
        v = weight.shape[0]
        dev = hidden.device
        code = _DTYPES[hidden.dtype]
        x, w = _operand(hidden), _operand(weight)
        tiles = int(load().mpq_xent_tiles(v))
        lse = torch.empty(t, device=dev, dtype=torch.float32)
        nll = torch.empty(t, device=dev, dtype=torch.float32)
        part = torch.empty(2 * t * tiles + t, device=dev, dtype=torch.float32)
        tgt = part[2 * t * tiles:]
        with torch.cuda.device(dev):
            call("mpq_xent_forward", t, v, h, code, ptr(x), x.stride(0), ptr(w), w.stride(0), ptr(labels), ignore_index,
                 ptr(part), 2 * t * tiles, ptr(tgt), ptr(lse), ptr(nll), ptr(ops.status_word(dev)))
            if reduction == "none":
                out, count = nll, None
            else:
                both = torch.empty(2, device=dev, dtype=torch.float32)
                out, count = both[0], both[1]
                call("mpq_xent_reduce", t, ptr(nll), ptr(labels), ignore_index, int(reduction == "mean"), ptr(out),
                     ptr(count))
        ctx.save_for_backward(hidden, weight, labels, lse, count if reduction == "mean" else None)
        ctx.ignore_index, ctx.piece = ignore_index, piece
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, gout):
        hidden, weight, labels, lse, count = ctx.saved_tensors
        t, h = hidden.shape
        v = weight.shape[0]
        dev = hidden.device
        need_h, need_w = ctx.needs_input_grad[:2]
        dh = torch.empty(t, h, device=dev, dtype=hidden.dtype) if need_h else None
        dw = torch.empty(v, h, device=dev, dtype=weight.dtype) if need_w else None
        if t == 0:
            return dh, dw if dw is None else dw.zero_(), None, None, None, None
        x, w = _operand(hidden), _operand(weight)
        gout = gout.to(torch.float32).contiguous()
        piece = _piece(t, v, ctx.piece)
        d = torch.empty(t, piece, device=dev, dtype=hidden.dtype)
        gmax = torch.empty(1, device=dev, dtype=torch.float32)
        acc = torch.empty(t, h, device=dev, dtype=torch.float32) if need_h and v > piece else None
        with torch.cuda.device(dev):
            call("mpq_xent_backward", t, v, h, _DTYPES[hidden.dtype], ptr(x), x.stride(0), ptr(w), w.stride(0),
                 ptr(labels), ctx.ignore_index, ptr(lse), ptr(gout), int(gout.dim() > 0), ptr(count), ptr(gmax), ptr(d),
                 piece, ptr(acc), ptr(dh), h, ptr(dw), h, ptr(ops.status_word(dev)))
        return dh, dw, None, None, None, None


def vocab_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, *, ignore_index: int = -100,
                        reduction: str = "mean", piece: Optional[int] = None) -> torch.Tensor:
    """Cross entropy of softmax(hidden @ weight.T) at ``labels``, in float32.

    ``hidden`` (..., H) and ``weight`` (V, H): bfloat16 or float16; ``labels`` (...): integers.  Labels equal to
    ``ignore_index`` do not count (their score is 0, their gradient 0; the mean over no labels is NaN); labels outside
    the vocabulary give NaN.  ``reduction``: "mean" over the labels that count, "sum" or "none" (one score a token).
    Differentiable once in ``hidden`` and ``weight``, whose gradients come in their own type; ``piece`` sets how many
    columns of the vocabulary the backward pass holds at a time (by default what fits in 1 GiB)."""
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
    flat = labels.reshape(-1).to(torch.int64).contiguous()
    out = _VocabCrossEntropy.apply(hidden.reshape(-1, hidden.shape[-1]), weight, flat, int(ignore_index), reduction, piece)
    return out.view(labels.shape) if reduction == "none" else out


__all__ = ["vocab_cross_entropy"]
