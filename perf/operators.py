"""What is measured of the microscaled 4-bit operators and of the vocabulary loss.

Three operators that stand next to the post-training quantisation of a decoder:

* ``quantize``: a matrix into microscaled 4-bit floating point (4-bit E2M1 elements, one power-of-two scale for 32
  consecutive elements of a row) and back into its own type;
* ``linear``: y = Q(x) W^T + b, with W held in that format and x quantised within the call;
* ``xent``: the softmax cross entropy of a decoder's output head over its whole vocabulary, from the hidden states,
  as scores of tokens (direction "score") or as a mean loss with its gradients (direction "train").

``run`` computes them in plain torch operations in 32 bits, or, where ``own`` is true, by the package's operators.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
LOSS_IGNORED = -100

# The sizes are those of the registered decoder shapes (hidden 1024, 2048 and 4096, intermediate 8192 and 14336,
# vocabularies 128256 and 151936, calibration batches of 8 x 2048 tokens), of single tokens, and generic odd ones.
MOST_ELEMENTS = 16384 * 4096            # of quantize: the largest listed case's
MOST_LINEAR = 16384 * 4096 * 14336      # of linear: tokens x inputs x outputs
MOST_SCORED = 2047 * 151936 * 1024      # of xent, score: tokens x vocabulary x hidden
MOST_TRAINED = 8192 * 128256 * 4096     # of xent, train


def listed():
    return [
        # one token's activations on their way into a product
        {"name": "quantize_token", "op": "quantize", "rows": 1, "cols": 4096, "dtype": "bfloat16"},
        # an odd matrix: a last block of 10 elements in each row
        {"name": "quantize_ragged", "op": "quantize", "rows": 1021, "cols": 2730, "dtype": "float16"},
        # the weights of a down projection, in the type that a solver holds them in
        {"name": "quantize_weight", "op": "quantize", "rows": 4096, "cols": 14336, "dtype": "float32"},
        # the activations of one calibration batch
        {"name": "quantize_batch", "op": "quantize", "rows": 16384, "cols": 4096, "dtype": "bfloat16"},
        # one new token through an up projection: serving's smallest call
        {"name": "linear_token", "op": "linear", "tokens": 1, "cols": 4096, "out": 14336, "dtype": "bfloat16",
         "bias": False},
        # a few sequences' new tokens through a down projection
        {"name": "linear_few", "op": "linear", "tokens": 7, "cols": 14336, "out": 4096, "dtype": "bfloat16",
         "bias": False},
        # a ragged prompt through an odd layer with a bias, K ending inside a block
        {"name": "linear_ragged", "op": "linear", "tokens": 333, "cols": 1000, "out": 1531, "dtype": "float16",
         "bias": True},
        # a calibration batch through an up projection
        {"name": "linear_batch", "op": "linear", "tokens": 16384, "cols": 4096, "out": 14336, "dtype": "bfloat16",
         "bias": False},
        # the score of one token
        {"name": "xent_token", "op": "xent", "way": "score", "tokens": 1, "vocab": 128256, "hidden": 4096,
         "dtype": "bfloat16", "ignored": 0.0},
        # the scores of one sequence's next tokens, for a perplexity
        {"name": "xent_sequence", "op": "xent", "way": "score", "tokens": 2047, "vocab": 151936, "hidden": 1024,
         "dtype": "bfloat16", "ignored": 0.0},
        # a short padded batch's training step, odd sizes
        {"name": "xent_train_ragged", "op": "xent", "way": "train", "tokens": 511, "vocab": 32003, "hidden": 2048,
         "dtype": "float16", "ignored": 0.3},
        # a batch's training step at the largest head
        {"name": "xent_train_batch", "op": "xent", "way": "train", "tokens": 8192, "vocab": 128256, "hidden": 4096,
         "dtype": "bfloat16", "ignored": 0.05},
    ]


def _between(rng, low, high):
    """A whole number, uniform over the logarithm of the range."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "xent", "xent"])
    if op == "quantize":
        cols = _between(rng, 32, 14336)
        rows = min(_between(rng, 1, 16384), MOST_ELEMENTS // cols)
        return {"op": op, "rows": rows, "cols": cols, "dtype": rng.choice(["float32", "bfloat16", "float16"])}
    if op == "linear":
        cols, out = _between(rng, 128, 14336), _between(rng, 128, 14336)
        if rng.random() < 0.5:  # most layers are whole numbers of blocks wide
            cols, out = (cols + 63) // 64 * 64, (out + 63) // 64 * 64
        tokens = min(_between(rng, 1, 16384), MOST_LINEAR // (cols * out))
        return {"op": op, "tokens": tokens, "cols": cols, "out": out,
                "dtype": rng.choice(["float32", "bfloat16", "bfloat16", "float16"]), "bias": rng.random() < 0.3}
    way = rng.choice(["score", "train"])
    hidden, vocab = 8 * _between(rng, 16, 512), _between(rng, 1000, 151936)
    most = MOST_SCORED if way == "score" else MOST_TRAINED
    tokens = max(1, min(_between(rng, 1, 8192), most // (hidden * vocab)))
    return {"op": op, "way": way, "tokens": tokens, "vocab": vocab, "hidden": hidden,
            "dtype": rng.choice(["bfloat16", "bfloat16", "float16"]), "ignored": rng.choice([0.0, 0.05, 0.5])}


# ---- inputs ----


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _activations(g, rows, cols):
    """Normed hidden states: unit normal rows whose channels differ in scale, with a few large ones."""
    return _normal(g, rows, cols) * torch.exp(0.5 * _normal(g, cols))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "quantize":
        return {"case": case, "x": _activations(g, case["rows"], case["cols"]).to(dtype)}
    if case["op"] == "linear":
        w = 0.02 * _normal(g, case["out"], case["cols"]) * torch.exp(0.3 * _normal(g, case["out"], 1))
        codes, scales = _pack(w)
        return {"case": case, "x": _activations(g, case["tokens"], case["cols"]).to(dtype), "codes": codes,
                "scales": scales, "bias": _normal(g, case["out"]).to(dtype) if case["bias"] else None}
    t, v, h = case["tokens"], case["vocab"], case["hidden"]
    weight = 0.02 * _normal(g, v, h)
    labels = torch.randint(0, v, (t,), generator=g, device="cuda")
    # from a guess to a certainty: the hidden state leans towards its label's row by up to 14 in the logit
    lean = 14 * torch.rand(t, 1, generator=g, device="cuda")
    rows = weight[labels]
    hidden = _normal(g, t, h) + lean * rows / (rows * rows).sum(1, keepdim=True)
    labels = torch.where(torch.rand(t, generator=g, device="cuda") < case["ignored"], LOSS_IGNORED, labels)
    labels[0] = 0  # one label at least counts
    train = case["way"] == "train"
    return {"case": case, "hidden": hidden.to(dtype).requires_grad_(train),
            "weight": weight.to(dtype).requires_grad_(train), "labels": labels}


# ---- microscaled 4-bit floating point in plain operations ----


def _blocks(x):
    """Rows padded by zeros to whole blocks, as rows x blocks x 32 in 32 bits."""
    rows, cols = x.shape
    padded = torch.nn.functional.pad(x.float(), (0, -cols % 32))
    return padded.view(rows, -1, 32)


def _encode(x):
    """(codes, scale codes) of a matrix: the block's scale is 2^(e - 127), with e the biased exponent of its largest
    magnitude less 2 (and 0 at least; 255, which stands for NaN, where the block is not finite); the elements are
    rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times the scale, ties to the even code, larger ones to 6."""
    b = _blocks(x)
    largest = b.abs().amax(2)
    e = largest.view(torch.int32) >> 23
    e = torch.where(e == 255, 255, (e - 2).clamp(min=0))
    inverse = ((254 - e.clamp(max=253)) << 23).view(torch.float32)
    a = b.abs() * inverse.unsqueeze(2)
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int()
            + (a >= 3.5).int() + (a > 5.0).int())
    return code + 8 * torch.signbit(b).int(), e


def _decode(code, e):
    """The values that codes (rows x blocks x 32) and scale codes (rows x blocks) stand for."""
    m = code & 7
    size = torch.where(m < 4, 0.5 * m.float(), torch.where(m < 6, m.float() - 2, 2 * m.float() - 8))
    scale = torch.where(e == 0, 0x00400000, e << 23).to(torch.int32).view(torch.float32)
    scale = torch.where(e == 255, float("nan"), scale)
    return torch.where(code >= 8, -size, size) * scale.unsqueeze(2)


def _pack(x):
    """The stored form: two codes to a byte, the even column's in the low half, rows x (whole blocks x 16) bytes; the
    scales in tiles of 128 rows x 4 blocks, each 512 bytes, byte (r % 32) * 16 + (r // 32) * 4 + block % 4 of it."""
    code, e = _encode(x)
    rows, blocks = e.shape
    pairs = code.view(rows, -1, 2)
    codes = (pairs[:, :, 0] + 16 * pairs[:, :, 1]).to(torch.uint8)
    padded = torch.nn.functional.pad(e, (0, -blocks % 4, 0, -rows % 128)).to(torch.uint8)
    tiles = padded.view(padded.shape[0] // 128, 4, 32, padded.shape[1] // 4, 4).permute(0, 3, 2, 1, 4)
    return codes, tiles.reshape(padded.shape[0] // 128, padded.shape[1] // 4, 512).contiguous()


def _unpack(codes, scales):
    rows, half = codes.shape
    code = torch.stack([codes & 15, codes >> 4], 2).int().view(rows, -1, 32)
    tiles = scales.view(scales.shape[0], scales.shape[1], 32, 4, 4).permute(0, 3, 2, 1, 4)
    e = tiles.reshape(scales.shape[0] * 128, scales.shape[1] * 4)[:rows, :half // 16].int()
    return _decode(code, e)


# ---- one pass ----


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    case = state["case"]
    if case["op"] == "quantize":
        from mpq_b200.mx4 import dequantize_mx4, quantize_mx4
        return dequantize_mx4(quantize_mx4(state["x"]), dtype=state["x"].dtype)
    if case["op"] == "linear":
        from mpq_b200.mx4 import Mx4Tensor, mx4_linear
        w = Mx4Tensor(state["codes"], state["scales"], (case["out"], case["cols"]))
        return mx4_linear(state["x"], w, bias=state["bias"])
    from mpq_b200.loss import vocab_cross_entropy
    if case["way"] == "score":
        return vocab_cross_entropy(state["hidden"], state["weight"], state["labels"], reduction="none")
    loss = vocab_cross_entropy(state["hidden"], state["weight"], state["labels"])
    grads = torch.autograd.grad(loss, (state["hidden"], state["weight"]))
    return {"loss": loss.detach(), "hidden": grads[0], "weight": grads[1]}


def _run_plain(state):
    case = state["case"]
    if case["op"] == "quantize":
        x = state["x"]
        return _decode(*_encode(x)).view(x.shape[0], -1)[:, :x.shape[1]].to(x.dtype)
    if case["op"] == "linear":
        x = state["x"]
        y = _decode(*_encode(x)).view(x.shape[0], -1) @ _unpack(state["codes"], state["scales"]).flatten(1).T
        return (y if state["bias"] is None else y + state["bias"].float()).to(x.dtype)
    h, w, labels = state["hidden"].detach(), state["weight"].detach(), state["labels"]
    counted = labels != LOSS_IGNORED
    target = torch.where(counted, labels, 0).unsqueeze(1)
    logits = h.float() @ w.float().T
    largest = logits.amax(1, keepdim=True)
    lse = largest + (logits - largest).exp().sum(1, keepdim=True).log()
    scores = torch.where(counted, (lse - logits.gather(1, target))[:, 0], 0.0)
    if case["way"] == "score":
        return scores
    share = counted.float() / counted.sum()
    d = (logits - lse).exp() * share.unsqueeze(1)
    d = d.scatter_add(1, target, -share.unsqueeze(1))
    return {"loss": (scores * share).sum(), "hidden": (d @ w.float()).to(h.dtype), "weight": (d.T @ h.float()).to(w.dtype)}


# ---- the definition in 64 bits ----


def _exact_mx4(x):
    """The values of a matrix in microscaled 4 bits, by the spacing of the grid around each element."""
    rows, cols = x.shape
    b = torch.zeros(rows, -(-cols // 32) * 32, dtype=torch.float64, device=x.device)
    b[:, :cols] = x.double()
    b = b.view(rows, -1, 32)
    _, e = torch.frexp(b.abs().amax(2, keepdim=True))
    s = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=x.device), (e - 3).clamp(min=-127).double())
    s = torch.where(b.abs().amax(2, keepdim=True) == 0, 2.0 ** -127, s)
    a = b.abs() / s
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    q = (torch.round(a / step) * step).clamp(max=6.0)
    return (torch.sign(b) * q * s).view(rows, -1)[:, :cols]


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "quantize":
        return _exact_mx4(state["x"])
    if case["op"] == "linear":
        grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64,
                            device="cuda")
        codes, n, k = state["codes"].long(), case["out"], case["cols"]
        w = torch.stack([grid[codes % 16], grid[codes // 16]], 2).view(n, -1)[:, :k]
        r, j = torch.arange(n, device="cuda")[:, None], (torch.arange(k, device="cuda") // 32)[None, :]
        at = (r % 32) * 16 + (r % 128) // 32 * 4 + j % 4
        w = w * torch.pow(2.0, state["scales"][r // 128, j // 4, at].double() - 127)
        y = _exact_mx4(state["x"]) @ w.T
        return y if state["bias"] is None else y + state["bias"].double()
    h, w, labels = state["hidden"].detach().double(), state["weight"].detach().double(), state["labels"]
    keep = (labels >= 0).double()
    one = torch.arange(labels.numel(), device="cuda")
    logits = h @ w.T
    lse = torch.logsumexp(logits, 1)
    scores = (lse - logits[one, labels.clamp(min=0)]) * keep
    if case["way"] == "score":
        return scores
    p = logits.sub_(lse[:, None]).exp_()
    p[one, labels.clamp(min=0)] -= 1
    p *= (keep / keep.sum())[:, None]
    return {"loss": scores.sum() / keep.sum(), "hidden": p @ w, "weight": p.T @ h}


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "quantize":  # the matrix in, its codes and scales out, its values out
        n, blocks = case["rows"] * case["cols"], case["rows"] * -(-case["cols"] // 32)
        return {"bytes": 2 * size * n + 17 * blocks, "flops": 3 * n}
    if case["op"] == "linear":
        t, k, n = case["tokens"], case["cols"], case["out"]
        return {"bytes": size * t * (k + n) + 17 * n * -(-k // 32) + (size * n if case["bias"] else 0),
                "flops": 2 * t * k * n}
    t, v, h = case["tokens"], case["vocab"], case["hidden"]
    once = size * h * (t + v)
    if case["way"] == "score":
        return {"bytes": once + 12 * t, "flops": 2 * t * v * h}
    return {"bytes": 2 * once + 8 * t, "flops": 6 * t * v * h}
