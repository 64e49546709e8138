"""Scores of token sequences under a decoder LM, in floating point or with its linears in microscaled 4 bits.

    perplexity(model, ids)                       # of a loaded decoder
    convert_linears_mx4(model.model)             # every linear of the layers in MX4, in place
    perplexity(model, ids)
    tune_head(model, ids, steps=20)              # final norm and output head, the 4-bit layers as they are

and the same from the command line, on a registered synthetic shape or a local checkpoint directory:

    python -m mpq_b200.evaluate --model tiny_llama --sequences 8 --seqlen 512 --tune 20

The output head's logits are not stored: the loss is ``vocab_cross_entropy`` on the hidden states.  Decoders whose logits
are another function of them than hidden @ head.T (a head with a bias; a soft cap or a scale in the configuration) are
refused, and so are heads of another type than bfloat16 and float16, which the loss takes.
"""
from __future__ import annotations

import argparse
import copy
import json
from typing import Any, Dict, List, Optional

import torch

from . import ops
from .loss import vocab_cross_entropy
from .mx4 import convert_linears_mx4


def _checked_ids(model, ids: torch.Tensor) -> torch.Tensor:
    dev = next(model.parameters()).device
    if dev.type != "cuda":
        raise ValueError("mpq_b200 kernels require CUDA tensors (there is no CPU path)")
    ids = torch.as_tensor(ids, dtype=torch.long)
    if ids.dim() != 2 or ids.shape[1] < 2:
        raise ValueError("ids must be (sequences, tokens) with two tokens at least")
    _check_range(ids, model.get_input_embeddings().weight.shape[0])
    return ids.to(dev)


def _check_range(ids: torch.Tensor, words: int) -> None:
    """Looking up an id that the embedding does not hold would be a device-side failure, which ends the process's GPU
    context."""
    if ids.numel() and not (0 <= int(ids.min()) and int(ids.max()) < words):
        raise ValueError(f"ids must be in [0, {words}), got {int(ids.min())} to {int(ids.max())}")


# What a decoder's configuration says about its logits beyond the head's product, and the values that leave them alone.
_ON_LOGITS = {"final_logit_softcapping": (None, 0.0), "logit_scale": (None, 1.0), "logits_scaling": (None, 1.0),
              "lm_head_multiplier": (None, 1.0)}


def _checked_head(model) -> torch.Tensor:
    """The head's weight, where the decoder's logits are hidden @ head.T as far as its head and configuration tell."""
    head = getattr(model, "lm_head", None)
    if not isinstance(head, torch.nn.Linear):
        raise ValueError(f"the loss needs the output head as an nn.Linear named lm_head, got {type(head).__name__} (convert "
                         "the linears of the decoder's layers, model.model, and leave the head as it is)")
    if head.bias is not None:
        raise ValueError("the loss is that of hidden @ head.T: a head with a bias is not supported")
    config = getattr(model, "config", None)
    for name, neutral in _ON_LOGITS.items():
        value = getattr(config, name, None)
        if value not in neutral:
            raise ValueError(f"the loss is that of hidden @ head.T: a decoder with {name} = {value} is not supported")
    return head.weight


@torch.no_grad()
def _check_logits(model, ids: torch.Tensor, out) -> None:
    """Raise where the decoder's own logits of two tokens of ``ids`` are not hidden @ head.T.  ``out``: what its layers gave
    for ``ids``; they do not run again (the decoder gets the two tokens' hidden states handed back).  A decoder that calls
    its layers past ``model.forward`` runs them on the two tokens, whose hidden states then differ by the rounding of other
    kernels."""
    inner, head = model.model, model.lm_head.weight
    short = copy.copy(out)
    short.last_hidden_state = out.last_hidden_state[:1, :2]
    before = inner.__dict__.get("forward")
    handed = []

    def hand_back(*args, **kwargs):
        handed.append(True)
        return short

    inner.forward = hand_back
    try:
        own = model(ids[:1, :2]).logits.float()
    finally:
        if before is None:
            del inner.forward
        else:
            inner.forward = before
    plain = torch.nn.functional.linear(short.last_hidden_state.to(head.dtype), head).float()
    room = 2.0 ** -8 if handed else 2.0 ** -4
    if own.shape != plain.shape or bool(((own - plain).abs().amax(-1) > room * plain.abs().amax(-1)).any()):
        raise ValueError(f"{type(model).__name__}'s logits are not hidden @ head.T: its loss is not supported")


@torch.no_grad()
def token_scores(model, ids: torch.Tensor, batch_size: int = 8) -> torch.Tensor:
    """Negative log-likelihood of every token but the first of each sequence: (sequences, tokens - 1) in float32."""
    ids = _checked_ids(model, ids)
    head = _checked_head(model)
    out: List[torch.Tensor] = []
    for part in ids.split(int(batch_size)):
        states = model.model(part[:, :-1])
        if not out:
            _check_logits(model, part[:, :-1], states)
        hidden = states.last_hidden_state.to(head.dtype)
        del states  # its key/value cache
        out.append(vocab_cross_entropy(hidden, head, part[:, 1:], reduction="none"))
    ops.check_status(ids.device)
    return torch.cat(out)


def perplexity(model, ids: torch.Tensor, batch_size: int = 8) -> float:
    """exp of the mean score over all scored tokens (infinity beyond float64)."""
    return float(token_scores(model, ids, batch_size).double().mean().exp())


def _untied_head(model) -> torch.Tensor:
    """The head's weight, a copy where it was the input embedding's as well."""
    head = model.lm_head
    embedding = model.get_input_embeddings()
    if embedding is not None and embedding.weight.data_ptr() == head.weight.data_ptr():
        head.weight = torch.nn.Parameter(head.weight.detach().clone(), requires_grad=head.weight.requires_grad)
        model.config.tie_word_embeddings = False
    return head.weight


def tune_head(model, ids: torch.Tensor, steps: int = 20, lr: float = 1e-2, batch_size: int = 8) -> List[float]:
    """Train the final norm and the output head on ``ids`` (SGD on the mean loss), with the layers as they are; returns
    the loss of each step.  The layers run forward only, so their linears may be in any format.  The weights are summed up
    in float32 while the steps run: a step of 16-bit weights by themselves rounds to nothing for most of them.  A head that
    is tied to the input embedding gets weights of its own first: training the embedding would change the layers' inputs,
    and by a part of its gradient only."""
    ids = _checked_ids(model, ids)
    inner = model.model
    _checked_head(model)
    head = _untied_head(model)
    params = [p for p in (*inner.norm.parameters(), head)]
    wanted = [p.requires_grad for p in params]
    seen: Dict[str, torch.Tensor] = {}
    hook = inner.norm.register_forward_pre_hook(lambda mod, args: seen.__setitem__("x", args[0].detach()))
    losses: List[torch.Tensor] = []
    try:
        for p in params:
            p.requires_grad_(True)
        sums = [p.detach().float() for p in params]
        parts = ids.split(int(batch_size))
        for step in range(int(steps)):
            part = parts[step % len(parts)]
            with torch.no_grad():
                states = inner(part[:, :-1])
            if step == 0:
                _check_logits(model, part[:, :-1], states)
            del states  # its key/value cache
            loss = vocab_cross_entropy(inner.norm(seen["x"]).to(head.dtype), head, part[:, 1:])
            grads = torch.autograd.grad(loss, params)
            with torch.no_grad():
                for p, total, g in zip(params, sums, grads):
                    p.copy_(total.add_(g, alpha=-float(lr)))
            losses.append(loss.detach())
    finally:
        hook.remove()
        for p, w in zip(params, wanted):
            p.requires_grad_(w)
    ops.check_status(ids.device)
    return [float(v) for v in losses]


def main(argv: Optional[List[str]] = None) -> Dict[str, Any]:
    from .model import calibration_ids
    from .quantization import _load_model
    ap = argparse.ArgumentParser(prog="mpq_b200.evaluate", description=__doc__.split("\n\n")[0])
    ap.add_argument("--model", default="tiny_llama", help="a registered synthetic shape or a local checkpoint directory")
    ap.add_argument("--sequences", type=int, default=8)
    ap.add_argument("--seqlen", type=int, default=512)
    ap.add_argument("--batch-size", type=int, default=8)
    ap.add_argument("--seed", type=int, default=0)
    ap.add_argument("--tune", type=int, default=0, help="training steps of the final norm and the head afterwards")
    ap.add_argument("--lr", type=float, default=1e-2, help="step size of --tune")
    a = ap.parse_args(argv)
    dev = torch.device("cuda", torch.cuda.current_device())
    model, name = _load_model(a.model, dev, a.seed)
    ids = calibration_ids(a.sequences, a.seqlen, int(model.config.vocab_size), seed=a.seed + 1)
    out: Dict[str, Any] = {"model": name, "tokens": a.sequences * (a.seqlen - 1),
                           "perplexity": perplexity(model, ids, a.batch_size)}
    out["mx4_linears"] = convert_linears_mx4(model.model)
    out["perplexity_mx4"] = perplexity(model, ids, a.batch_size)
    if a.tune:
        out["tune_losses"] = tune_head(model, ids, a.tune, a.lr, a.batch_size)
        out["perplexity_mx4_tuned"] = perplexity(model, ids, a.batch_size)
    print(json.dumps(out))
    return out


if __name__ == "__main__":
    main()
