"""The vocabulary loss and its gradients against the formulas in 64 bits.

Bounds, before any run: a logit off the tensor cores is within 1e-5 of sum |h| |w| (the bound that this package's other
tensor-core products are held to) = delta_t at most for token t; a score is then within 2 delta_t, plus 1e-5 for the
FP32 exponentials and logarithm.  The logits' gradient d is off by 2 delta_t + 1e-5 of p, and by one rounding u (2^-8
for bf16, 2^-11 for f16) of itself; a product with it adds 1e-5 of the sum of magnitudes and the output's rounding u.
"""
import math

import pytest
import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def inputs(t, v, h, dtype, dev, seed=0, ignored=0.2, lean=8.0):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(v, h, generator=g) * (1.5 / h ** 0.5)
    y = torch.randint(0, v, (t,), generator=g)
    x = torch.randn(t, h, generator=g) + lean * torch.rand(t, 1, generator=g) * w[y] / w[y].square().sum(1, keepdim=True)
    y = torch.where(torch.rand(t, generator=g) < ignored, -100, y)
    return x.to(dtype).to(dev), w.to(dtype).to(dev), y.to(dev)


def formulas(x, w, y, gout=None, reduction="mean", ignore=-100):
    """Scores and gradients in 64 bits, with the bounds above."""
    u = U[x.dtype]
    x, w, y = x.double().cpu(), w.double().cpu(), y.cpu()
    keep = y != ignore
    logits = x @ w.T
    delta = 1e-5 * (x.abs() @ w.abs().T).amax(1)
    lse = torch.logsumexp(logits, 1)
    at = torch.where(keep, y, 0)[:, None]
    nll = torch.where(keep, lse - logits.gather(1, at)[:, 0], 0.0)
    share = keep.double() / (keep.sum() if reduction == "mean" else 1)
    gout = torch.ones(()) if gout is None else gout.double().cpu()
    g = share * gout
    p = torch.exp(logits - lse[:, None])
    d = p.scatter_add(1, at, -torch.ones_like(p[:, :1])) * g[:, None]
    off = (p * (2 * delta + 1e-5)[:, None]) * g.abs()[:, None] + u * d.abs()
    if x.shape[0] and u == 2.0 ** -11:  # f16 holds multiples of 2^-24 in units of 2^-15 of the largest g
        off = off + 2.0 ** -40 * g.abs().max()
    dh, dw = d @ w, d.T @ x
    tol_h = off @ w.abs() + 1e-5 * (d.abs() @ w.abs()) + u * dh.abs() + (2.0 ** -24 if u == 2.0 ** -11 else 0)
    tol_w = off.T @ x.abs() + 1e-5 * (d.abs().T @ x.abs()) + u * dw.abs() + (2.0 ** -24 if u == 2.0 ** -11 else 0)
    return {"nll": nll, "tol": torch.where(keep, 2 * delta + 1e-5, 0.0), "share": share, "dh": dh, "dw": dw, "tol_h": tol_h,
            "tol_w": tol_w}


def within(got, want, tol):
    err = (got.detach().cpu().double() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


SHAPES = [(1, 1, 8), (1, 1000, 64), (2, 7, 24), (5, 257, 128), (31, 300, 8), (127, 511, 200), (128, 512, 64),
          (129, 2049, 136), (200, 1000, 256), (300, 777, 1024), (513, 4100, 72)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(U), ids=str)
@pytest.mark.parametrize("t,v,h", SHAPES)
def test_scores(cuda_dev, t, v, h, dtype):
    from mpq_b200.loss import vocab_cross_entropy
    x, w, y = inputs(t, v, h, dtype, cuda_dev)
    ref = formulas(x, w, y)
    nll = vocab_cross_entropy(x, w, y, reduction="none")
    assert nll.dtype == torch.float32
    within(nll, ref["nll"], ref["tol"])
    total = vocab_cross_entropy(x, w, y, reduction="sum")
    within(total, ref["nll"].sum(), ref["tol"].sum() + 1e-6 * ref["nll"].sum())
    mean = vocab_cross_entropy(x, w, y)
    if bool((y != -100).any()):
        within(mean, (ref["nll"] * ref["share"]).sum(), (ref["tol"] * ref["share"]).sum() + 1e-6 * ref["nll"].max())
    else:
        assert bool(mean.isnan())


@pytest.mark.gpu
@pytest.mark.parametrize("piece,keep", [(None, 1 << 31), (None, 0), (256, 0), (600, 0), (256, 150000), (None, 700000)])
@pytest.mark.parametrize("dtype", list(U), ids=str)
@pytest.mark.parametrize("t,v,h", SHAPES)
def test_gradients(cuda_dev, t, v, h, dtype, piece, keep):
    from mpq_b200.loss import vocab_cross_entropy
    x, w, y = inputs(t, v, h, dtype, cuda_dev, 1)
    y[0] = v - 1
    x.requires_grad_(), w.requires_grad_()
    ref = formulas(x.detach(), w.detach(), y)
    dh, dw = torch.autograd.grad(vocab_cross_entropy(x, w, y, piece=piece, keep_bytes=keep), (x, w))
    assert dh.dtype == dtype and dw.dtype == dtype
    within(dh, ref["dh"], ref["tol_h"])
    within(dw, ref["dw"], ref["tol_w"])
    gout = torch.randn(t, generator=torch.Generator().manual_seed(3)).to(cuda_dev)
    ref = formulas(x.detach(), w.detach(), y, gout, "none")
    nll = vocab_cross_entropy(x, w, y, reduction="none", piece=piece, keep_bytes=keep)
    dh, dw = torch.autograd.grad(nll, (x, w), gout)
    within(dh, ref["dh"], ref["tol_h"])
    within(dw, ref["dw"], ref["tol_w"])


@pytest.mark.gpu
@pytest.mark.parametrize("keep", [1 << 31, 0, 100000])
@pytest.mark.parametrize("dtype", list(U), ids=str)
@pytest.mark.parametrize("t", [16, 17, 32, 33, 48, 63, 64, 65, 96, 129])
def test_numbers_of_tokens_between_the_forms(cuda_dev, t, dtype, keep):
    """Token counts at and around those where the products change sides."""
    from mpq_b200.loss import vocab_cross_entropy
    x, w, y = inputs(t, 1003, 264, dtype, cuda_dev, t)
    y[0], y[-1] = 1002, 0
    x.requires_grad_(), w.requires_grad_()
    ref = formulas(x.detach(), w.detach(), y)
    within(vocab_cross_entropy(x, w, y, reduction="none"), ref["nll"], ref["tol"])
    loss = vocab_cross_entropy(x, w, y, keep_bytes=keep)
    within(loss, (ref["nll"] * ref["share"]).sum(), (ref["tol"] * ref["share"]).sum() + 1e-6 * ref["nll"].max())
    dh, dw = torch.autograd.grad(loss, (x, w))
    within(dh, ref["dh"], ref["tol_h"])
    within(dw, ref["dw"], ref["tol_w"])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(U), ids=str)
def test_gradients_against_differences(cuda_dev, dtype):
    """Central differences of the 64-bit loss along a direction: eps = 1e-5 leaves 1e-9 of curvature and rounding, so the
    bound is the gradients' own summed along the direction."""
    from mpq_b200.loss import vocab_cross_entropy
    x, w, y = inputs(70, 900, 96, dtype, cuda_dev, 2)
    x.requires_grad_(), w.requires_grad_()
    dh, dw = torch.autograd.grad(vocab_cross_entropy(x, w, y), (x, w))
    ref = formulas(x.detach(), w.detach(), y)
    xd, wd, yd = x.detach().double().cpu(), w.detach().double().cpu(), y.cpu()
    g = torch.Generator().manual_seed(0)
    for _ in range(4):
        a, b = torch.randn(xd.shape, generator=g).double(), torch.randn(wd.shape, generator=g).double()
        loss = lambda e: torch.nn.functional.cross_entropy((xd + e * a) @ (wd + e * b).T, yd)  # noqa: E731
        slope = (loss(1e-5) - loss(-1e-5)) / 2e-5
        got = (dh.cpu().double() * a).sum() + (dw.cpu().double() * b).sum()
        tol = (ref["tol_h"] * a.abs()).sum() + (ref["tol_w"] * b.abs()).sum() + 1e-7
        assert abs(float(got - slope)) <= float(tol)


@pytest.mark.gpu
def test_one_gradient_at_a_time_and_scaled_loss(cuda_dev):
    from mpq_b200.loss import vocab_cross_entropy
    x, w, y = inputs(60, 700, 64, torch.bfloat16, cuda_dev, 4)
    both = torch.autograd.grad(vocab_cross_entropy(x.requires_grad_(), w.requires_grad_(), y), (x, w))
    only_h = torch.autograd.grad(vocab_cross_entropy(x, w.detach(), y), x)[0]
    only_w = torch.autograd.grad(vocab_cross_entropy(x.detach(), w, y), w)[0]
    assert torch.equal(both[0], only_h) and torch.equal(both[1], only_w)
    scaled = torch.autograd.grad(64.0 * vocab_cross_entropy(x, w, y), (x, w))
    assert torch.equal(scaled[0], 64 * both[0]) and torch.equal(scaled[1], 64 * both[1])


@pytest.mark.gpu
def test_a_second_pass_through_the_graph(cuda_dev):
    from mpq_b200.loss import vocab_cross_entropy
    x, w, y = inputs(90, 1200, 64, torch.bfloat16, cuda_dev, 12)
    x.requires_grad_(), w.requires_grad_()
    loss = vocab_cross_entropy(x, w, y)
    one = torch.autograd.grad(loss, (x, w), retain_graph=True)
    two = torch.autograd.grad(loss, (x, w))
    again = torch.autograd.grad(vocab_cross_entropy(x, w, y, keep_bytes=0), (x, w))
    ref = formulas(x.detach(), w.detach(), y)
    within(one[0], ref["dh"], ref["tol_h"])
    within(one[1], ref["dw"], ref["tol_w"])
    assert torch.equal(two[0], again[0]) and torch.equal(two[1], again[1])


@pytest.mark.gpu
def test_small_upstream_gradients_in_f16(cuda_dev):
    """A mean over many tokens: every entry of d is far below f16's normal range, its gradients are not lost."""
    from mpq_b200.loss import vocab_cross_entropy
    x, w, y = inputs(400, 3000, 64, torch.float16, cuda_dev, 5, ignored=0.0, lean=0.0)
    x.requires_grad_()
    ref = formulas(x.detach(), w, y)
    scale = 2.0 ** 12
    dh = torch.autograd.grad(scale * vocab_cross_entropy(x, w, y), x)[0]
    within(dh / scale, ref["dh"], ref["tol_h"])
    off = (dh.cpu().double() / scale - ref["dh"]).norm() / ref["dh"].norm()
    assert float(off) <= 2 * U[torch.float16]


@pytest.mark.gpu
def test_rows_that_do_not_count(cuda_dev):
    from mpq_b200.loss import vocab_cross_entropy
    x, w, y = inputs(40, 500, 64, torch.bfloat16, cuda_dev, 6, ignored=0.0)
    x[3] = float("nan")  # a padded position may hold anything
    x[5] = float("inf")
    y[3] = y[5] = y[7] = -100
    x.requires_grad_()
    loss = vocab_cross_entropy(x, w, y)
    dh = torch.autograd.grad(loss, x)[0]
    assert bool(loss.isfinite()) and bool(dh.isfinite().all())
    assert not dh[[3, 5, 7]].any()
    other = vocab_cross_entropy(x, w, torch.where(y == -100, 2 ** 40, y), ignore_index=2 ** 40)
    assert torch.equal(other, loss)
    seven = torch.where(y == -100, 7, y)
    assert torch.equal(vocab_cross_entropy(x, w, seven, ignore_index=7, reduction="none") == 0, seven == 7)
    none = torch.full_like(y, -100)
    total = vocab_cross_entropy(x, w, none, reduction="sum")
    assert float(total) == 0 and not torch.autograd.grad(total, x)[0].any()
    mean = vocab_cross_entropy(x, w, none)
    assert bool(mean.isnan()) and not torch.autograd.grad(mean, x)[0].any()


@pytest.mark.gpu
def test_labels_outside_the_vocabulary_give_nan(cuda_dev):
    from mpq_b200.loss import vocab_cross_entropy
    x, w, y = inputs(20, 300, 64, torch.bfloat16, cuda_dev, 7, ignored=0.0)
    good = vocab_cross_entropy(x, w, y, reduction="none")
    y[4], y[9] = 300, -1
    x.requires_grad_()
    nll = vocab_cross_entropy(x, w, y, reduction="none")
    bad = torch.zeros(20, dtype=torch.bool, device=cuda_dev)
    bad[[4, 9]] = True
    assert torch.equal(nll.isnan(), bad) and torch.equal(nll[~bad], good[~bad])
    dh = torch.autograd.grad(nll.sum(), x)[0]
    assert torch.equal(dh.isnan().any(1), bad)


@pytest.mark.gpu
def test_large_logits_and_infinities(cuda_dev):
    """Logits of +-3000: the running maximum keeps every exponential finite; a row with an infinity scores NaN alone."""
    from mpq_b200.loss import vocab_cross_entropy
    x, w, y = inputs(33, 600, 64, torch.bfloat16, cuda_dev, 8, ignored=0.0)
    x = x * 400
    ref = formulas(x, w, y)
    nll = vocab_cross_entropy(x, w, y, reduction="none")
    within(nll, ref["nll"], ref["tol"] + 1e-6 * ref["nll"])
    x[2, 3] = float("inf")
    again = vocab_cross_entropy(x, w, y, reduction="none")
    keep = torch.arange(33, device=cuda_dev) != 2
    assert torch.equal(again[keep], nll[keep]) and not bool(again[2].isfinite())


@pytest.mark.gpu
@pytest.mark.parametrize("t", [1, 40])
def test_small_scores_of_large_logits(cuda_dev, t):
    """Scores of 0.05 from logits of 200, which are exact here.  What may be off: 16 roundings of a sum near 1 (2^-24
    each), and 2e-6 of the score (exponents near -14 rounded at 2^-21, 2^-22 of the exponentials, 1.3e-8 of log2(e))."""
    from mpq_b200.loss import vocab_cross_entropy
    v, h = 1000, 64
    x = torch.zeros(t, h)
    x[:, 0] = 1.0
    w = torch.zeros(v, h)
    w[:, 0] = 189.0 + torch.arange(v) % 3
    y = torch.arange(t) * 7 + 5
    x[torch.arange(t), 1 + torch.arange(t)] = 1.0
    w[y, 1 + torch.arange(t)] = 200.0 - w[y, 0]
    logits = x.double() @ w.double().T
    want = torch.logsumexp(logits, 1) - logits[torch.arange(t), y]
    nll = vocab_cross_entropy(x.to(cuda_dev, torch.bfloat16), w.to(cuda_dev, torch.bfloat16), y.to(cuda_dev),
                              reduction="none")
    within(nll, want, 2.0 ** -20 + 2e-6 * want)


@pytest.mark.gpu
@pytest.mark.parametrize("keep", [1 << 31, 0])
@pytest.mark.parametrize("dtype", list(U), ids=str)
@pytest.mark.parametrize("t", [1, 64, 70])
def test_nearly_certain_labels(cuda_dev, t, dtype, keep):
    """Scores of 1e-4 and their gradients, from logits that are exact: token t's are column t of the head, its d is
    column t of the head's gradient.  The score is off by 5e-6 of itself (exponents near -24 rounded at 2^-20, and some
    rounding of sums), d by one rounding for itself, one for the gradient and 2^-12.5 for a kept distance."""
    from mpq_b200.loss import vocab_cross_entropy
    v, h = 1000, 72
    g = torch.Generator().manual_seed(t)
    x = torch.eye(t, h, dtype=torch.float64)
    w = 3.0 + torch.randint(0, 3, (v, h), generator=g).double()
    y = torch.randint(0, v, (t,), generator=g)
    w[y, torch.arange(t)] = 20.0
    logits = x @ w.T
    rest = torch.exp(logits - 20.0).scatter(1, y[:, None], 0.0)
    want = torch.log1p(rest.sum(1))
    d = (rest / (1 + rest.sum(1, keepdim=True))).scatter(1, y[:, None], -(1 - torch.exp(-want))[:, None])
    xs, ws = x.to(cuda_dev, dtype), w.to(cuda_dev, dtype).requires_grad_()
    within(vocab_cross_entropy(xs, ws, y.to(cuda_dev), reduction="none"), want, 5e-6 * want)
    loss = vocab_cross_entropy(xs, ws, y.to(cuda_dev), reduction="sum", keep_bytes=keep)
    dw, = torch.autograd.grad(loss, ws)
    u = U[dtype]
    within(dw[:, :t].T, d, (2 * u + u * u + 2.0 ** -12.4) * d.abs() + (2.0 ** -24 if dtype == torch.float16 else 0))


def exact_logits(t, base, label, v=1000, h=72):
    """Operands whose logits are `base` everywhere but `label` at each token's own, exactly (the two parts are small whole
    numbers); column 1 + i of the head's gradient is token i's d."""
    x, w = torch.zeros(t, h), torch.zeros(v, h)
    x[:, 0] = 1.0
    x[torch.arange(t), 1 + torch.arange(t)] = 1.0
    y = (torch.arange(t) * 7 + 5) % v
    w[:, 0] = base
    w[y, 1 + torch.arange(t)] = label - base
    return x, w, y


@pytest.mark.gpu
@pytest.mark.parametrize("keep", [1 << 31, 0])
@pytest.mark.parametrize("dtype", list(U), ids=str)
@pytest.mark.parametrize("base,label", [(-60.0, -50.0), (-60.0, -45.0), (-60.0, -70.0), (-110.0, -100.0), (-112.0, -240.0),
                                        (-1000.0, -990.0), (-1000.0, -1000.0)])
@pytest.mark.parametrize("t", [1, 40, 64, 70])
def test_logits_that_are_all_negative(cuda_dev, t, base, label, dtype, keep):
    """The softmax does not change when all logits are shifted.  A score is off by 5e-6 of itself (as of nearly certain
    labels).  A d rests on lse in FP32: 2^-22 |lse| of it for two roundings in log2 and ln units, one rounding for itself
    and one for the gradient, 2^-12.4 where distances are kept, 1e-5 for the exponentials; in f16 d is a multiple of 2^-24
    of its unit 2^-15 and a gradient of 2^-24."""
    from mpq_b200.loss import vocab_cross_entropy
    x, w, y = exact_logits(t, base, label)
    logits = x.double() @ w.double().T
    gap = torch.full((t,), base - label).double()
    want = torch.log1p(999 * torch.exp(gap))
    p = torch.exp(logits - label - want[:, None])
    d = p.scatter(1, y[:, None], torch.expm1(-want)[:, None])
    lse = label + want
    xs, ws = x.to(cuda_dev, dtype).requires_grad_(), w.to(cuda_dev, dtype).requires_grad_()
    within(vocab_cross_entropy(xs, ws, y.to(cuda_dev), reduction="none"), want, 5e-6 * want)
    loss = vocab_cross_entropy(xs, ws, y.to(cuda_dev), reduction="sum", keep_bytes=keep)
    dh, dw = torch.autograd.grad(loss, (xs, ws))
    u, f16 = U[dtype], dtype == torch.float16
    off = (u + 2.0 ** -12.4 + 1e-5 + 2.0 ** -22 * lse.abs()[:, None]) * d.abs() + (2.0 ** -40 if f16 else 0)
    within(dw[:, 1:1 + t].T, d, (1 + u) * off + u * d.abs() + (2.0 ** -24 if f16 else 0))
    ref = d @ w.double()
    within(dh, ref, off @ w.double().abs() + 1e-5 * (d.abs() @ w.double().abs()) + u * ref.abs() + (2.0 ** -24 if f16 else 0))


@pytest.mark.gpu
@pytest.mark.parametrize("t", [1, 64, 65])
def test_one_word_of_any_logit(cuda_dev, t):
    """A vocabulary of one: every score and gradient is 0, whatever the logit."""
    from mpq_b200.loss import vocab_cross_entropy
    y = torch.zeros(t, dtype=torch.int64, device=cuda_dev)
    for size in (-500.0, -10.0, 0.0, 10.0):
        x = torch.ones(t, 8, device=cuda_dev, dtype=torch.bfloat16).requires_grad_()
        w = torch.full((1, 8), size, device=cuda_dev, dtype=torch.bfloat16).requires_grad_()
        nll = vocab_cross_entropy(x, w, y, reduction="none")
        dh, dw = torch.autograd.grad(nll.sum(), (x, w))
        assert not nll.any() and not dh.any() and not dw.any()


@pytest.mark.gpu
@pytest.mark.parametrize("keep", [1 << 31, 0])
@pytest.mark.parametrize("dtype", list(U), ids=str)
@pytest.mark.parametrize("base", [3008.0, -3008.0, 12032.0, -12032.0])
@pytest.mark.parametrize("t", [1, 13, 64, 65, 70])
def test_gradients_of_large_logits(cuda_dev, t, base, dtype, keep):
    """Logits in the thousands whose largest is not the label's, exactly known: d of the largest column is what matters.
    Bounds as for logits that are all negative; a kept distance counts from a maximum in log2 units that is off by another
    2^-24 of itself, which 2^-22 |lse| still covers."""
    from mpq_b200.loss import vocab_cross_entropy
    v = 1000
    x, w, y = exact_logits(t, base, base)
    i = torch.arange(t)
    top = 1.0 + i % 13
    w[y, 1 + i] = top - 2
    w[(y + 391) % v, 1 + i] = top
    logits = x.double() @ w.double().T
    lse = torch.logsumexp(logits, 1)
    want = lse - logits[i, y]
    d = torch.exp(logits - lse[:, None]).scatter(1, y[:, None], torch.expm1(-want)[:, None])
    xs, ws = x.to(cuda_dev, dtype).requires_grad_(), w.to(cuda_dev, dtype).requires_grad_()
    loss = vocab_cross_entropy(xs, ws, y.to(cuda_dev), reduction="sum", keep_bytes=keep)
    dh, dw = torch.autograd.grad(loss, (xs, ws))
    u, f16 = U[dtype], dtype == torch.float16
    off = (u + 2.0 ** -12.4 + 1e-5 + 2.0 ** -22 * lse.abs()[:, None]) * d.abs() + (2.0 ** -40 if f16 else 0)
    within(dw[:, 1:1 + t].T, d, (1 + u) * off + u * d.abs() + (2.0 ** -24 if f16 else 0))
    ref = d @ w.double()
    within(dh, ref, off @ w.double().abs() + 1e-5 * (d.abs() @ w.double().abs()) + u * ref.abs() + (2.0 ** -24 if f16 else 0))


@pytest.mark.gpu
@pytest.mark.parametrize("keep", [1 << 31, 0])
@pytest.mark.parametrize("dtype", list(U), ids=str)
@pytest.mark.parametrize("t", [1, 64, 65, 130])
def test_gradients_beside_masked_words(cuda_dev, t, dtype, keep):
    """Every third word of the head is masked by its type's lowest value (logits at most -3e4, probability 0 in 64 bits):
    the loss and the gradients are those of the other words alone, and a masked word's gradient is 0."""
    from mpq_b200.loss import vocab_cross_entropy
    x, w, y = inputs(t, 900, 72, dtype, cuda_dev, 15)
    y[0] = 1
    x[:, 0] = 0.5
    w[:, 0] = 0
    masked = torch.arange(900, device=cuda_dev) % 3 == 0
    y = torch.where((y >= 0) & masked[y], y + 1, y)
    w[masked] = 0
    w[masked, 0] = torch.finfo(dtype).min
    at = torch.cumsum(~masked, 0) - 1
    ref = formulas(x, w[~masked], torch.where(y >= 0, at[y], y))
    x.requires_grad_(), w.requires_grad_()
    loss = vocab_cross_entropy(x, w, y, keep_bytes=keep)
    within(loss, (ref["nll"] * ref["share"]).sum(), (ref["tol"] * ref["share"]).sum() + 1e-6 * ref["nll"].max())
    dh, dw = torch.autograd.grad(loss, (x, w))
    within(dh, ref["dh"], ref["tol_h"])
    within(dw[~masked], ref["dw"], ref["tol_w"])
    assert not dw[masked].any()


@pytest.mark.gpu
@pytest.mark.parametrize("keep", [1 << 31, 0])
@pytest.mark.parametrize("t", [1, 64, 65, 130])
def test_logits_of_bfloat16s_lowest_value(cuda_dev, t, keep):
    """Stretches of words whose logits are -3.39e38, further from 0 than FP32 holds in log2 units: scores and gradients are
    those of the other words; a masked label scores its distance from them; where all words are masked, none is."""
    from mpq_b200.loss import vocab_cross_entropy
    low = torch.finfo(torch.bfloat16).min
    x, w, y = inputs(t, 1000, 72, torch.bfloat16, cuda_dev, 16)
    y[0] = 1
    x[:, 0] = 1
    w[:, 0] = 0
    masked = torch.zeros(1000, dtype=torch.bool, device=cuda_dev)
    masked[200:800] = True
    y = torch.where((y >= 0) & masked[y], y % 200, y)
    w[masked] = 0
    w[masked, 0] = low
    at = torch.cumsum(~masked, 0) - 1
    ref = formulas(x, w[~masked], torch.where(y >= 0, at[y], y))
    x.requires_grad_(), w.requires_grad_()
    loss = vocab_cross_entropy(x, w, y, keep_bytes=keep)
    within(loss, (ref["nll"] * ref["share"]).sum(), (ref["tol"] * ref["share"]).sum() + 1e-6 * ref["nll"].max())
    dh, dw = torch.autograd.grad(loss, (x, w))
    within(dh, ref["dh"], ref["tol_h"])
    within(dw[~masked], ref["dw"], ref["tol_w"])
    assert not dw[masked].any()
    nll = vocab_cross_entropy(x, w, torch.full_like(y, 500), reduction="none")
    within(nll, torch.full((t,), -low).double(), -1e-6 * low)
    alone = torch.zeros_like(w)
    alone[:, 0] = low
    nll = vocab_cross_entropy(x, alone, torch.full_like(y, 500), reduction="none", keep_bytes=keep)
    within(nll, torch.full((t,), math.log(1000)).double(), 1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("keep", [1 << 31, 0])
@pytest.mark.parametrize("dtype", list(U), ids=str)
@pytest.mark.parametrize("t", [5, 70, 140])
def test_upstream_gradients_that_are_not_finite(cuda_dev, t, dtype, keep):
    """One token's upstream gradient is infinite or NaN (a loss scaled too far): its own row of dhidden is not finite, the
    others are what they are without it; also where all other upstream gradients are 0."""
    from mpq_b200.loss import vocab_cross_entropy
    x, w, y = inputs(t, 700, 72, dtype, cuda_dev, 17, ignored=0.0)
    x.requires_grad_()
    gout = torch.randn(t, generator=torch.Generator().manual_seed(4)).to(cuda_dev)
    gout[2] = 0
    ref = formulas(x.detach(), w, y, gout, "none")
    others = torch.arange(t, device=cuda_dev) != 2
    for bad in (float("inf"), float("-inf"), float("nan")):
        for size in (1.0, 0.0):
            nll = vocab_cross_entropy(x, w, y, reduction="none", keep_bytes=keep)
            dh = torch.autograd.grad(nll, x, torch.where(others, size * gout, bad))[0]
            within(dh[others], size * ref["dh"][others.cpu()], ref["tol_h"][others.cpu()])
            assert not dh[2].isfinite().any()


@pytest.mark.gpu
def test_shapes_strides_and_types_of_labels(cuda_dev):
    from mpq_b200.loss import vocab_cross_entropy
    x, w, y = inputs(60, 400, 128, torch.bfloat16, cuda_dev, 9)
    want = vocab_cross_entropy(x, w, y, reduction="none")
    assert torch.equal(vocab_cross_entropy(x.view(3, 20, 128), w, y.view(3, 20), reduction="none"), want.view(3, 20))
    assert torch.equal(vocab_cross_entropy(x, w, y.int(), reduction="none"), want)
    wide = torch.zeros(60, 300, device=cuda_dev, dtype=x.dtype)
    wide[:, 5:133] = x                                   # rows off the 16-byte boundary
    assert torch.equal(vocab_cross_entropy(wide[:, 5:133], w, y, reduction="none"), want)
    assert torch.equal(vocab_cross_entropy(x.T.contiguous().T, w.T.contiguous().T, y, reduction="none"), want)
    lots = torch.stack([y, y], 1)[:, 0]
    assert torch.equal(vocab_cross_entropy(x, w, lots, reduction="none"), want)
    row = x[:1].expand(60, 128).requires_grad_()
    assert vocab_cross_entropy(row, w, y, reduction="none").shape == (60,)
    for h in (1, 7, 130):                                # widths that are not whole 16-byte lines
        xs, ws, ys = inputs(37, 333, h, torch.bfloat16, cuda_dev, 10)
        ys[0] = 5
        ref = formulas(xs, ws, ys)
        xs.requires_grad_(), ws.requires_grad_()
        loss = vocab_cross_entropy(xs, ws, ys)
        dh, dw = torch.autograd.grad(loss, (xs, ws))
        within(dh, ref["dh"], ref["tol_h"])
        within(dw, ref["dw"], ref["tol_w"])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(U), ids=str)
@pytest.mark.parametrize("t", [5, 130])
def test_neighbours_of_narrow_operands_are_not_read(cuda_dev, t, dtype):
    """Rows that end inside 16 bytes, between NaNs: views of wider matrices, taken as they are."""
    from mpq_b200.loss import vocab_cross_entropy
    x, w, y = inputs(t, 300, 20, dtype, cuda_dev, 5)
    ref = formulas(x, w, y)
    wide = [torch.full((r.shape[0], 32), float("nan"), device=cuda_dev, dtype=dtype) for r in (x, w)]
    for big, part in zip(wide, (x, w)):
        big[:, :20] = part
    x, w = (big[:, :20].requires_grad_() for big in wide)
    loss = vocab_cross_entropy(x, w, y)
    within(loss, (ref["nll"] * ref["share"]).sum(), (ref["tol"] * ref["share"]).sum() + 1e-6 * ref["nll"].max())
    dh, dw = torch.autograd.grad(loss, (x, w))
    within(dh, ref["dh"], ref["tol_h"])
    within(dw, ref["dw"], ref["tol_w"])


@pytest.mark.gpu
@pytest.mark.parametrize("t,keep_cols", [(5, 0), (130, 0), (130, 300)])
def test_gradients_into_wider_rows(cuda_dev, t, keep_cols):
    """The C entries with leading dimensions beyond the columns: what lies between the rows is left alone."""
    from mpq_b200 import _lib, ops
    v, h, ld, dtype = 300, 20, 24, torch.bfloat16
    x, w, y = inputs(t, v, h, dtype, cuda_dev, 6)
    ref = formulas(x, w, y)
    xp, wp = (torch.nn.functional.pad(m, (0, ld - h)) for m in (x, w))
    f32 = lambda *n: torch.zeros(*n, device=cuda_dev)  # noqa: E731
    lib, status = _lib.load(), ops.status_word(cuda_dev).data_ptr()
    tiles = lib.mpq_xent_tiles(t, v)
    part, tgt, lse, nll, loss, count, gmax = f32(2 * t * tiles), f32(t), f32(t), f32(t), f32(1), f32(1), f32(1)
    keep = torch.zeros(t, 304, device=cuda_dev, dtype=dtype) if keep_cols else None
    d = torch.zeros(t, 512, device=cuda_dev, dtype=dtype)
    acc = f32(max(1, lib.mpq_xent_planes(t, v, h, 512, keep_cols)) * t * h)
    dh, dw = (torch.full((r, ld), 7.0, device=cuda_dev, dtype=dtype) for r in (t, v))
    _lib.call("mpq_xent_forward", t, v, h, 1, xp.data_ptr(), ld, wp.data_ptr(), ld, y.data_ptr(), -100, part.data_ptr(),
              part.numel(), tgt.data_ptr(), lse.data_ptr(), nll.data_ptr(), 2, loss.data_ptr(), count.data_ptr(),
              _lib.ptr(keep), 304, keep_cols, status)
    gout = torch.ones(1, device=cuda_dev)
    _lib.call("mpq_xent_backward", t, v, h, 1, xp.data_ptr(), ld, wp.data_ptr(), ld, y.data_ptr(), -100, lse.data_ptr(),
              gout.data_ptr(), 0, count.data_ptr(), part.data_ptr(), tgt.data_ptr(), _lib.ptr(keep), 304, keep_cols,
              gmax.data_ptr(), d.data_ptr(), 512, acc.data_ptr(), dh.data_ptr(), ld, dw.data_ptr(), ld, status)
    within(dh[:, :h], ref["dh"], ref["tol_h"])
    within(dw[:, :h], ref["dw"], ref["tol_w"])
    assert (dh[:, h:] == 7.0).all() and (dw[:, h:] == 7.0).all()


@pytest.mark.gpu
def test_streams_and_repeatability(cuda_dev):
    from mpq_b200.loss import vocab_cross_entropy
    x, w, y = inputs(300, 2000, 128, torch.bfloat16, cuda_dev, 11)
    x.requires_grad_(), w.requires_grad_()

    def step():
        loss = vocab_cross_entropy(x, w, y, piece=512)
        return (loss.detach(), *torch.autograd.grad(loss, (x, w)))

    first = step()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        runs = [step() for _ in range(5)]
    s.synchronize()
    for r in runs:
        assert all(torch.equal(a, b) for a, b in zip(first, r))


@pytest.mark.gpu
@pytest.mark.parametrize("t", [9, 200])
def test_step_in_a_cuda_graph(cuda_dev, t):
    """A captured step on new inputs gives what the same step gives outside, bit for bit."""
    from mpq_b200.loss import vocab_cross_entropy
    x, w, y = inputs(t, 700, 128, torch.bfloat16, cuda_dev, 12)
    x.requires_grad_(), w.requires_grad_()

    def step():
        loss = vocab_cross_entropy(x, w, y, piece=256, keep_bytes=2 * 256 * t)
        return (loss.detach(), *torch.autograd.grad(loss, (x, w)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (13, 14):
        new = inputs(t, 700, 128, torch.bfloat16, cuda_dev, seed)
        with torch.no_grad():
            x.copy_(new[0]), w.copy_(new[1]), y.copy_(new[2])
        graph.replay()
        got = [r.clone() for r in held]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.gpu
def test_empty(cuda_dev):
    from mpq_b200.loss import vocab_cross_entropy
    w = torch.randn(30, 16, device=cuda_dev).to(torch.bfloat16).requires_grad_()
    x = torch.zeros(0, 16, device=cuda_dev, dtype=torch.bfloat16, requires_grad=True)
    y = torch.zeros(0, device=cuda_dev, dtype=torch.int64)
    assert vocab_cross_entropy(x, w, y, reduction="none").shape == (0,)
    assert bool(vocab_cross_entropy(x, w, y).isnan())
    dh, dw = torch.autograd.grad(vocab_cross_entropy(x, w, y, reduction="sum"), (x, w))
    assert dh.shape == (0, 16) and not dw.any()


def test_refusals_without_a_gpu():
    from mpq_b200 import _lib
    from mpq_b200.loss import vocab_cross_entropy
    with pytest.raises(ValueError, match="CUDA"):
        vocab_cross_entropy(torch.zeros(2, 8), torch.zeros(4, 8), torch.zeros(2, dtype=torch.int64))
    lib = _lib.load()
    f = lambda **k: lib.mpq_xent_forward(*{**dict(T=4, V=9, H=8, dtype=1, h=16, ldh=8, w=16, ldw=8, y=16, ignore=-100,  # noqa: E731
                                                  part=16, n=16, tgt=16, lse=16, nll=16, red=0, loss=None,
                                                  count=None, keep=None, ldk=0, kc=0,
                                                  status=16, stream=None), **k}.values())
    assert f(red=1) == 10001 and f(red=3) == 10001
    assert f(kc=9) == 10001 and f(keep=16, ldk=8, kc=9) == 10001 and f(keep=16, ldk=8, kc=8) == 10001
    assert f(dtype=0) == 10001 and f(ldh=12) == 10001 and f(h=8) == 10001 and f(n=15) == 10001 and f(status=None) == 10001
    assert f(T=0) == 0
    b = lambda **k: lib.mpq_xent_backward(*{**dict(T=4, V=600, H=8, dtype=1, h=16, ldh=8, w=16, ldw=8, y=16, ignore=-100,  # noqa: E731
                                                   lse=16, gout=16, gs=0, count=None, part=16, tgt=16,
                                                   keep=None, ldk=0, kc=0, gmax=16, d=16, piece=256, acc=16, dh=16,
                                                   lddh=8, dw=16, lddw=8, status=16, stream=None), **k}.values())
    assert b(gs=1, gmax=None) == 10001
    assert b(kc=256) == 10001 and b(keep=16, ldk=256, kc=256, part=None) == 10001
    assert b(piece=100) == 10001 and b(acc=None) == 10001 and b(lddh=7) == 10001 and b(d=None) == 10001 and b(dtype=3) == 10001


@pytest.mark.gpu
def test_refusals(cuda_dev):
    from mpq_b200.loss import vocab_cross_entropy
    x, w, y = inputs(4, 30, 16, torch.bfloat16, cuda_dev)
    for bad, match in (((x.float(), w.float(), y), "bfloat16 or float16"), ((x, w.half(), y), "one type"),
                       ((x[:, :8], w, y), "does not fit"), ((x, w[:0], y), "empty"), ((x, w, y[:3]), "labels"),
                       ((x, w, y.float()), "int64"), ((x, w, y.cpu()), "CUDA")):
        with pytest.raises(ValueError, match=match):
            vocab_cross_entropy(*bad)
    with pytest.raises(ValueError, match="reduction"):
        vocab_cross_entropy(x, w, y, reduction="avg")
    with pytest.raises(ValueError, match="piece"):
        vocab_cross_entropy(x, w, y, piece=0)
    with pytest.raises(ValueError, match="keep_bytes"):
        vocab_cross_entropy(x, w, y, keep_bytes=-1)
