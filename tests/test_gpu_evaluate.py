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


def small_decoder(family, **changes):
    """A random decoder of another family on the CPU in float32, with logits of some size."""
    transformers = pytest.importorskip("transformers")
    sizes = dict(vocab_size=120, hidden_size=32, intermediate_size=48, num_hidden_layers=1, num_attention_heads=2,
                 num_key_value_heads=2, max_position_embeddings=64, initializer_range=0.5, pad_token_id=0, bos_token_id=1,
                 eos_token_id=2)
    if family in ("Gemma2", "Llama"):
        sizes["head_dim"] = 16
    config = getattr(transformers, family + "Config")(**{**sizes, **changes})
    torch.manual_seed(0)
    return getattr(transformers, family + "ForCausalLM")(config).eval()


@pytest.mark.parametrize("family,changes,plain", [
    ("Llama", {}, True), ("Llama", {"tie_word_embeddings": True}, True), ("Qwen3", {"head_dim": 16}, True),
    ("Gemma2", {"final_logit_softcapping": None}, True), ("Granite", {"logits_scaling": 1.0}, True),
    ("Gemma2", {}, False), ("Granite", {"logits_scaling": 8.0}, False), ("Cohere", {}, False), ("Phi", {}, False)])
def test_heads_that_are_more_than_a_product_are_refused(family, changes, plain):
    """By what the head and the configuration say, and by comparing the decoder's own logits; the layers do not run again and
    the decoder is left as it was."""
    from mpq_b200.evaluate import _check_logits, _checked_head
    model = small_decoder(family, **changes)
    if family == "Phi":
        torch.nn.init.normal_(model.lm_head.bias)
    ids = torch.arange(3, 33).view(2, 15)
    with torch.no_grad():
        states, logits = model.model(ids), model(ids).logits
    calls = []
    hook = model.model.layers[0].register_forward_hook(lambda *a: calls.append(1))
    if plain:
        assert _checked_head(model) is model.lm_head.weight
        _check_logits(model, ids, states)
    else:
        with pytest.raises(ValueError, match="hidden @ head.T"):
            _checked_head(model)
        with pytest.raises(ValueError, match="hidden @ head.T"):
            _check_logits(model, ids, states)
    hook.remove()
    assert not calls and "forward" not in model.model.__dict__ and states.last_hidden_state.shape[:2] == (2, 15)
    with torch.no_grad():
        assert torch.equal(model(ids).logits, logits)


def test_logits_changed_in_a_way_that_nothing_tells():
    from mpq_b200.evaluate import _check_logits, _checked_head
    model = small_decoder("Llama")
    ids = torch.arange(3, 33).view(2, 15)
    with torch.no_grad():
        states = model.model(ids)
    _checked_head(model)
    hook = model.lm_head.register_forward_hook(lambda mod, args, out: 0.9 * out)
    with pytest.raises(ValueError, match="hidden @ head.T"):
        _check_logits(model, ids, states)
    hook.remove()
    _check_logits(model, ids, states)


@pytest.mark.gpu
def test_scores_of_another_function_are_refused(cuda_dev):
    from mpq_b200.evaluate import perplexity, token_scores, tune_head
    model = small_decoder("Gemma2").to(cuda_dev).to(torch.bfloat16)
    ids = torch.arange(3, 33).view(2, 15)
    for call in (perplexity, token_scores, tune_head):
        with pytest.raises(ValueError, match="final_logit_softcapping"):
            call(model, ids)
    plain = small_decoder("Gemma2", final_logit_softcapping=None, hidden_size=256).to(cuda_dev).to(torch.bfloat16)
    with torch.no_grad():
        logits = plain(ids[:, :-1].to(cuda_dev)).logits.float()
    want = torch.nn.functional.cross_entropy(logits.flatten(0, 1), ids[:, 1:].flatten().to(cuda_dev), reduction="none")
    got = token_scores(plain, ids)
    # the decoder's own logits are rounded to bfloat16: two of them differ by 2^-8 of the largest at most
    assert float((got.flatten() - want).abs().max()) <= 2.0 ** -8 * 2 * float(logits.abs().max())


def test_a_head_that_is_no_linear_layer_is_refused():
    """As it is after converting a whole decoder instead of its layers."""
    from mpq_b200.evaluate import _checked_head
    from mpq_b200.mx4 import Mx4Linear, Mx4Tensor
    model = small_decoder("Llama")
    codes, scales = torch.zeros(120, 16, dtype=torch.uint8), torch.zeros(1, 1, 512, dtype=torch.uint8)
    model.lm_head = Mx4Linear(Mx4Tensor(codes, scales, (120, 32)))
    with pytest.raises(ValueError, match="nn.Linear named lm_head, got Mx4Linear"):
        _checked_head(model)
    with pytest.raises(ValueError, match="nn.Linear named lm_head"):
        _checked_head(torch.nn.Module())


@pytest.mark.gpu
def test_tuning_by_its_default_step_moves_the_weights(cuda_dev, decoder):
    """The first step's gradient promises lr |g|^2 a step; half of that has to arrive over twenty (the loss is convex in the
    head, its curvature at this step size takes a few per cent, the rounding of the weights to bfloat16 some more)."""
    from mpq_b200.evaluate import tune_head
    from mpq_b200.model import calibration_ids
    model = decoder()
    ids = calibration_ids(8, 512, 1000, seed=1).to(cuda_dev)
    with torch.no_grad():
        hidden = model.model(ids[:, :-1]).last_hidden_state.float()
        logits = hidden @ model.lm_head.weight.float().T
        d = torch.softmax(logits, -1) - torch.nn.functional.one_hot(ids[:, 1:], 1000)
        g = (d.flatten(0, 1).T @ hidden.flatten(0, 1)) / d.shape[:2].numel()
    losses = tune_head(model, ids)
    assert len(losses) == 20 and losses[0] - losses[-1] >= 0.5 * 19 * 1e-2 * float(g.square().sum())


def test_untying_a_head():
    from mpq_b200.evaluate import _untied_head
    tied = small_decoder("Llama", tie_word_embeddings=True)
    before = tied.lm_head.weight
    head = _untied_head(tied)
    assert head is tied.lm_head.weight and head is not before and torch.equal(head, before)
    assert tied.get_input_embeddings().weight is before and not tied.config.tie_word_embeddings
    assert _untied_head(tied) is head


@pytest.mark.gpu
def test_tuning_a_tied_head_leaves_the_embedding(cuda_dev):
    from mpq_b200.evaluate import tune_head
    model = small_decoder("Llama", tie_word_embeddings=True, hidden_size=64).to(cuda_dev).to(torch.bfloat16)
    embedding = model.get_input_embeddings().weight
    assert embedding is model.lm_head.weight
    before = embedding.detach().clone()
    losses = tune_head(model, torch.arange(3, 33).view(2, 15), steps=5, lr=0.1)
    assert losses[-1] < losses[0]
    assert torch.equal(model.get_input_embeddings().weight, before) and not torch.equal(model.lm_head.weight, before)


def test_range_of_ids():
    from mpq_b200.evaluate import _check_range
    _check_range(torch.tensor([[0, 119], [3, 4]]), 120)
    _check_range(torch.zeros(0, 4, dtype=torch.long), 120)
    for bad in (120, -1, -100, 2 ** 40):
        with pytest.raises(ValueError, match="ids must be in"):
            _check_range(torch.tensor([[0, 1], [bad, 2]]), 120)


@pytest.mark.gpu
def test_refuses_ids_outside_the_vocabulary(cuda_dev, decoder):
    from mpq_b200.evaluate import perplexity, token_scores, tune_head
    model = decoder()
    for bad in (1000, -100):
        for ids in (torch.tensor([[1, 2, bad]]), torch.tensor([[1, bad, 2]], device=cuda_dev)):
            for call in (perplexity, token_scores, tune_head):
                with pytest.raises(ValueError, match="ids must be in"):
                    call(model, ids)
    assert token_scores(model, torch.tensor([[0, 999]])).shape == (1, 1)


def test_a_wait_that_ran_out_is_named():
    """The word that the kernels leave, faked: whose wait it was, once."""
    from mpq_b200 import ops
    cpu = torch.device("cpu")
    word = ops.status_word(cpu)
    for code, whose in ((3, "FP32-faithful product"), (15, "mx4_linear"), (24, "vocab_cross_entropy"), (99, "tensor-core")):
        word.fill_(code)
        with pytest.raises(RuntimeError, match=f"{whose}.*timed out .code {code}.; its results are undefined"):
            ops.check_status(cpu)
        ops.check_status(cpu)


def test_perplexities_of_any_score(monkeypatch):
    from mpq_b200 import evaluate
    for scores, want in ((torch.tensor([[1.0, 3.0]]), math.exp(2.0)), (torch.tensor([[900.0]]), math.inf),
                         (torch.tensor([[math.inf]]), math.inf)):
        monkeypatch.setattr(evaluate, "token_scores", lambda *args: scores)
        assert evaluate.perplexity(None, None) == pytest.approx(want, rel=1e-12)
    monkeypatch.setattr(evaluate, "token_scores", lambda *args: torch.tensor([[math.nan, 1.0]]))
    assert math.isnan(evaluate.perplexity(None, None))


def test_a_decoder_that_runs_its_layers_itself():
    """Its hidden states of the two tokens come from other kernels: a difference like theirs is no other function."""
    transformers = pytest.importorskip("transformers")
    from mpq_b200.evaluate import _check_logits
    torch.manual_seed(0)
    model = transformers.OPTForCausalLM(transformers.OPTConfig(
        vocab_size=120, hidden_size=32, word_embed_proj_dim=32, ffn_dim=48, num_hidden_layers=1, num_attention_heads=2,
        max_position_embeddings=64, init_std=0.5)).eval()
    ids = torch.arange(3, 33).view(2, 15)
    with torch.no_grad():
        states = model.model(ids)
    states.last_hidden_state = states.last_hidden_state * (1 + 2.0 ** -7 * torch.randn(2, 15, 32))
    _check_logits(model, ids, states)
    hook = model.lm_head.register_forward_hook(lambda mod, args, out: 0.8 * out)
    with pytest.raises(ValueError, match="hidden @ head.T"):
        _check_logits(model, ids, states)
    hook.remove()


@pytest.mark.gpu
def test_no_batch_keeps_its_cache(cuda_dev, decoder):
    """What the layers gave for one batch (its key/value cache with it) is gone when the next one runs."""
    import weakref
    from mpq_b200.evaluate import token_scores, tune_head
    model = decoder()
    caches, alive = [], []

    def before(mod, args):
        if "forward" not in mod.__dict__:  # not while the check of the logits hands a batch's states back
            alive.append(sum(r() is not None for r in caches))

    hooks = [model.model.register_forward_pre_hook(before),
             model.model.register_forward_hook(lambda mod, args, out: caches.append(weakref.ref(out.past_key_values)))]
    ids = torch.arange(3, 123, device=cuda_dev).view(6, 20)
    token_scores(model, ids, batch_size=2)
    tune_head(model, ids, steps=3, batch_size=2)
    for h in hooks:
        h.remove()
    assert len(alive) == 6 and not any(alive)
