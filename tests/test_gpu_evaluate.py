"""The 4-bit linears and the vocabulary loss together, as a user scores a decoder."""
import math

import pytest
import torch


@pytest.fixture(scope="module")
def decoder():
    from mpq_b200.model import build_synthetic_decoder
    return lambda: build_synthetic_decoder("tiny_llama", device=torch.device("cuda:0"), seed=3)


def plain_scores(model, ids):
    """Scores from whole logits in float32 of the same hidden states."""
    with torch.no_grad():
        hidden = model.model(ids[:, :-1]).last_hidden_state.float()
        logits = hidden @ model.lm_head.weight.float().T
        return torch.nn.functional.cross_entropy(logits.flatten(0, 1), ids[:, 1:].flatten(), reduction="none"
                                                 ).view(ids.shape[0], -1)


@pytest.mark.gpu
def test_scores_match_whole_logits(cuda_dev, decoder):
    from mpq_b200.evaluate import perplexity, token_scores
    from mpq_b200.model import calibration_ids
    model = decoder()
    ids = calibration_ids(5, 70, 1000, seed=1).to(cuda_dev)
    want = plain_scores(model, ids)
    got = token_scores(model, ids, batch_size=5)
    # logits within 1e-5 of sum |h| |w| (< 16 here), twice, and 1e-5 for the exponentials
    assert got.shape == (5, 69) and float((got - want).abs().max()) <= 2 * 16e-5 + 1e-5
    # another batch size runs other kernels of the library that computes the layers
    assert abs(perplexity(model, ids, batch_size=2) - math.exp(float(want.double().mean()))) <= 0.01 * math.exp(float(want.mean()))


@pytest.mark.gpu
def test_converted_decoder_runs_on_its_quantised_values(cuda_dev, decoder):
    """Each converted linear against plain products of the values it stands for, inside the decoder's forward pass."""
    from mpq_b200.evaluate import token_scores
    from mpq_b200.model import calibration_ids
    from mpq_b200.mx4 import Mx4Linear, convert_linears_mx4, dequantize_mx4, quantize_mx4
    model = decoder()
    weights = {n: m.weight.detach().clone() for n, m in model.model.named_modules() if isinstance(m, torch.nn.Linear)}
    assert convert_linears_mx4(model.model) == len(weights) == 14
    ids = calibration_ids(3, 40, 1000, seed=2).to(cuda_dev)
    seen = []
    hooks = [m.register_forward_hook(lambda mod, args, out, n=n: seen.append((n, args[0], out)))
             for n, m in model.model.named_modules() if isinstance(m, Mx4Linear)]
    scores = token_scores(model, ids)
    for h in hooks:
        h.remove()
    assert len(seen) == 14 and bool(scores.isfinite().all())
    for name, x, y in seen:
        x = x.reshape(-1, x.shape[-1])
        a = dequantize_mx4(quantize_mx4(x)).double()
        b = dequantize_mx4(quantize_mx4(weights[name])).double()
        ref, size = a @ b.T, a.abs() @ b.abs().T
        err = (y.reshape(ref.shape).double() - ref).abs()
        assert bool((err <= 1e-5 * size + 2.0 ** -8 * ref.abs()).all()), name
    assert float((scores - plain_scores(model, ids)).abs().max()) <= 2 * 16e-5 + 1e-5


@pytest.mark.gpu
def test_tuning_the_head_of_a_4_bit_decoder_lowers_its_loss(cuda_dev, decoder):
    from mpq_b200.evaluate import main, tune_head
    from mpq_b200.model import calibration_ids
    from mpq_b200.mx4 import convert_linears_mx4
    model = decoder()
    convert_linears_mx4(model.model)
    ids = calibration_ids(2, 33, 1000, seed=4).to(cuda_dev)
    norm = model.model.norm.weight
    before = norm.requires_grad
    losses = tune_head(model, ids, steps=12, lr=1.0)
    assert losses[-1] < losses[0] - 0.05 and all(math.isfinite(v) for v in losses)
    assert norm.requires_grad == before
    out = main(["--sequences", "2", "--seqlen", "33", "--tune", "2"])
    assert out["mx4_linears"] == 14 and 500 < out["perplexity_mx4"] < 2000 and len(out["tune_losses"]) == 2


def test_refusals():
    from mpq_b200.evaluate import perplexity, tune_head
    model = torch.nn.Module()
    model.lm_head = torch.nn.Linear(4, 8)
    with pytest.raises(ValueError, match="CUDA"):
        perplexity(model, torch.zeros(1, 4, dtype=torch.long))
    with pytest.raises(ValueError, match="CUDA"):
        tune_head(model, torch.zeros(1, 4, dtype=torch.long))


@pytest.mark.gpu
def test_refuses_ids_without_a_next_token(cuda_dev, decoder):
    from mpq_b200.evaluate import perplexity
    model = decoder()
    for bad in (torch.zeros(3, 1, dtype=torch.long), torch.zeros(5, dtype=torch.long)):
        with pytest.raises(ValueError, match="two tokens"):
            perplexity(model, bad)
