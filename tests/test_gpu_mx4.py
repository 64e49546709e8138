"""Microscaled 4-bit operators against a plain 64-bit implementation of the format.

The format's own rounding is exact (power-of-two scales, ties defined), so codes and scales are compared bit for bit.
A product accumulates in the tensor cores' FP32: 1e-5 of sum |a| |b| (the bound that this package's other tensor-core
products are held to), plus one rounding to the output's type, 2^-8 (bf16), 2^-11 (f16) or 2^-24 (f32) of the result;
f16 results below its normal range round to multiples of 2^-24.
"""
import math

import pytest
import torch

GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = list(ROUND)


def plain_quantize(x):
    """(codes rows x padded cols, scale codes rows x blocks), by search over the grid in 64 bits."""
    rows, cols = x.shape
    nb = -(-cols // 32)
    b = torch.zeros(rows, nb * 32, dtype=torch.float64)
    b[:, :cols] = x.double().cpu()
    b = b.view(rows, nb, 32)
    finite = torch.isfinite(b).all(2)
    top = torch.where(finite, b.abs().amax(2), 1.0)
    mantissa, e = torch.frexp(top)  # top = m 2^e, m in [0.5, 1): floor(log2 top) = e - 1
    c = torch.where(top == 0, 0, (e - 3 + 127).clamp(min=0))
    a = torch.where(finite[..., None], b.abs() / torch.pow(2.0, c.double() - 127)[..., None], 0.0)
    gap = (a[..., None] - GRID).abs()
    near = gap == gap.amin(-1, keepdim=True)
    even = near & (torch.arange(8) % 2 == 0)
    code = torch.where(even.any(-1), even.double().argmax(-1), near.double().argmax(-1))
    code = code + 8 * torch.signbit(b).long()
    return torch.where(finite[..., None], code, 0).view(rows, -1), torch.where(finite, c.long(), 255)


def plain_values(code, c):
    q = GRID[code & 7] * torch.where(code >= 8, -1.0, 1.0)
    s = torch.where(c == 255, float("nan"), torch.pow(2.0, c.double() - 127))
    return (q.view(code.shape[0], -1, 32) * s[..., None]).view(code.shape)


def unpack(q):
    """Codes and scale codes of an Mx4Tensor from its stored form."""
    codes, scales, (rows, cols) = q.codes.cpu().long(), q.scales.cpu().long(), q.shape
    nb = -(-cols // 32)
    code = torch.stack([codes % 16, codes // 16], 2).view(rows, -1)
    r, j = torch.arange(rows)[:, None], torch.arange(nb)[None]
    return code, scales[r // 128, j // 4, (r % 32) * 16 + r % 128 // 32 * 4 + j % 4]


def same_but_zero_sign(a, b):
    return bool(((a == b) | ((a & 7) == 0) & ((b & 7) == 0)).all())


def values(rows, cols, dtype, dev, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp(spread * torch.randn(rows, max(-(-cols // 8), 1), generator=g)
                                                         ).repeat_interleave(8, 1)[:, :cols]
    return x.clamp(-6e4, 6e4).to(dtype).to(dev)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (1, 32), (3, 31), (2, 33), (127, 100), (129, 256), (257, 1000), (64, 4096)])
def test_quantize_codes_and_values(cuda_dev, shape, dtype):
    from mpq_b200.mx4 import dequantize_mx4, quantize_mx4
    x = values(*shape, dtype, cuda_dev)
    q = quantize_mx4(x)
    code, c = unpack(q)
    want_code, want_c = plain_quantize(x)
    assert torch.equal(c, want_c)
    assert same_but_zero_sign(code, want_code)
    want = plain_values(want_code, want_c)[:, :shape[1]]
    for out in DTYPES:
        got = dequantize_mx4(q, out)
        assert got.dtype == out and torch.equal(got.cpu().double(), want.to(out).double())


@pytest.mark.gpu
def test_quantize_pads_are_zero(cuda_dev):
    from mpq_b200.mx4 import quantize_mx4, stored_shapes
    from mpq_b200._lib import call, ptr
    x = values(130, 70, torch.float32, cuda_dev)
    codes_shape, scales_shape = stored_shapes(130, 70)
    codes = torch.full(codes_shape, 0xAB, device=cuda_dev, dtype=torch.uint8)
    scales = torch.full(scales_shape, 0xFF, device=cuda_dev, dtype=torch.uint8)
    call("mpq_mx4_quantize", ptr(x), 0, 70, 130, 70, ptr(codes), ptr(scales))
    q = quantize_mx4(x)
    assert torch.equal(q.codes, codes) and torch.equal(q.scales, scales)
    code, _ = unpack(q)
    assert not (code[:, 70:] & 7).any()
    real = torch.zeros(scales_shape, dtype=torch.bool)
    r, j = torch.arange(130)[:, None], torch.arange(3)[None]
    real[r // 128, j // 4, (r % 32) * 16 + r % 128 // 32 * 4 + j % 4] = True
    assert not scales.cpu()[~real].any()


@pytest.mark.gpu
def test_every_tie_and_edge_value(cuda_dev):
    """Midpoints of the grid, their neighbours in bf16 and f32, saturation, and the ends of the scale's range."""
    from mpq_b200.mx4 import dequantize_mx4, quantize_mx4
    mids = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.9]
    for dtype in (torch.float32, torch.bfloat16):
        eps = 2.0 ** -22 if dtype == torch.float32 else 2.0 ** -7
        near = [m * (1 + s * eps) for m in mids for s in (-1, 0, 1)]
        rows = []
        for e in (-124, -60, 0, 60, 122):
            body = [sign * v * 2.0 ** e for v in near for sign in (1, -1)]
            for i in range(0, len(body), 31):
                part = body[i:i + 31]
                rows.append([4.0 * 2.0 ** e] + part + [0.0] * (31 - len(part)))
        x = torch.tensor(rows, dtype=torch.float64).to(dtype).to(cuda_dev)
        code, c = unpack(quantize_mx4(x))
        want_code, want_c = plain_quantize(x)
        assert torch.equal(c, want_c) and same_but_zero_sign(code, want_code)
        assert torch.equal(dequantize_mx4(quantize_mx4(x)).cpu().double(), plain_values(want_code, want_c))
    tiny = torch.zeros(4, 32)
    tiny[0, 3] = 2.0 ** -149
    tiny[1, :] = 2.0 ** -127
    tiny[2, 5] = 3.0e38
    x = tiny.to(cuda_dev)
    want_code, want_c = plain_quantize(x)
    code, c = unpack(quantize_mx4(x))
    assert torch.equal(c, want_c) and same_but_zero_sign(code, want_code)
    assert c[3, 0] == 0  # an empty block


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_non_finite_blocks_read_back_as_nan(cuda_dev, dtype):
    from mpq_b200.mx4 import Mx4Tensor, dequantize_mx4, mx4_linear, quantize_mx4
    x = values(5, 100, dtype, cuda_dev, spread=0.5)
    x[1, 40], x[2, 99], x[4, 0] = float("nan"), float("inf"), float("-inf")
    back = dequantize_mx4(quantize_mx4(x))
    bad = torch.zeros(5, 100, dtype=torch.bool)
    bad[1, 32:64] = bad[2, 96:] = bad[4, :32] = True
    assert torch.equal(back.cpu().isnan(), bad)
    w = quantize_mx4(values(70, 100, dtype, cuda_dev, 1, 0.5))
    y = mx4_linear(x, w)
    assert torch.equal(y.isnan().all(1).cpu(), bad.any(1)) and torch.equal(y.isnan().any(1).cpu(), bad.any(1))
    assert isinstance(w, Mx4Tensor)


def check_linear(x, w, bias=None):
    from mpq_b200.mx4 import mx4_linear, quantize_mx4
    k = x.shape[-1]
    a = plain_values(*plain_quantize(x.reshape(-1, k)))
    b = plain_values(*plain_quantize(w))
    ref, size = a @ b.T, a.abs() @ b.abs().T
    if bias is not None:
        ref, size = ref + bias.double().cpu(), size + bias.double().cpu().abs()
    y = mx4_linear(x, quantize_mx4(w), bias)
    assert y.dtype == x.dtype and y.shape == (*x.shape[:-1], w.shape[0])
    err = (y.reshape(ref.shape).cpu().double() - ref).abs()
    tol = 1e-5 * size + ROUND[x.dtype] * ref.abs() + (2.0 ** -24 if x.dtype == torch.float16 else 0)
    assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 128, 256), (1, 300, 4096), (2, 129, 96), (3, 1000, 520), (7, 257, 2048),
                                   (8, 64, 33), (9, 512, 1056), (16, 200, 640), (33, 700, 128), (64, 1024, 992),
                                   (127, 130, 700), (128, 128, 512), (129, 383, 1000), (256, 256, 2304), (333, 1531, 1000),
                                   (700, 900, 224), (1100, 2100, 160)])
def test_linear(cuda_dev, m, n, k, dtype):
    x = values(m, k, dtype, cuda_dev, 2, 0.7)
    w = values(n, k, dtype, cuda_dev, 3, 0.7) * 0.05
    check_linear(x, w)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m,n,k", [(12, 4096, 2048), (5, 192, 4128), (128, 1000, 8200), (4, 96, 32), (2, 31, 20000), (3, 40, 20000),
                                   (1, 5, 180000), (2600, 1153, 288), (3000, 2000, 1000), (2049, 4097, 96), (1537, 3900, 2080)])
def test_linear_split_and_wide(cuda_dev, m, n, k, dtype):
    """K shared by a cluster, K too long for the kernel of few tokens, and tiles of CTA pairs with ragged ends."""
    x = values(m, k, dtype, cuda_dev, 4, 0.4)
    w = values(n, k, dtype, cuda_dev, 5, 0.4) * 0.05
    check_linear(x, w)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 5, 40, 200])
def test_linear_bias_strides_and_leading_dimensions(cuda_dev, m):
    g = torch.Generator().manual_seed(5)
    w = (torch.randn(193, 416, generator=g) * 0.1).to(cuda_dev)
    bias = torch.randn(193, generator=g).to(cuda_dev).to(torch.bfloat16)
    x = torch.randn(m, 3, 416, generator=g).to(cuda_dev).to(torch.bfloat16)
    check_linear(x, w, bias)
    wide = torch.randn(m, 500, generator=g).to(cuda_dev).to(torch.bfloat16)
    check_linear(wide[:, 3:419], w, bias)                   # rows at odd offsets
    check_linear(torch.randn(416, m, generator=g).to(cuda_dev).to(torch.bfloat16).T, w)  # columns along the rows
    check_linear(x[:, 1], w)                                # every third row
    check_linear(x[:1, :1].expand(m, 1, 416), w)            # one row, broadcast


@pytest.mark.gpu
def test_linear_masked_inputs_of_lowest_value(cuda_dev):
    """Rows of zeros, and blocks that hold a type's lowest value next to ordinary ones (the scale follows it)."""
    x = values(6, 256, torch.bfloat16, cuda_dev, 7, 0.5)
    x[2] = 0
    x[3, 64:96] = 0
    x[4, 5] = torch.finfo(torch.bfloat16).min
    w = values(130, 256, torch.bfloat16, cuda_dev, 8, 0.5) * 0.01
    check_linear(x[:4], w)
    check_linear(x.float(), w.float() * 1e-3)


@pytest.mark.gpu
def test_scales_at_the_ends_of_their_range_in_a_product(cuda_dev):
    """Denormal inputs against large weights: scales 2^-127 .. 2^100, the result in FP32's range."""
    x = values(4, 96, torch.float32, cuda_dev, 9, 0.3) * 2.0 ** -124
    w = values(40, 96, torch.float32, cuda_dev, 10, 0.3) * 2.0 ** 100
    check_linear(x, w)
    check_linear(x.repeat(20, 1), w)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 2, 3, 130])
def test_scales_whose_product_leaves_the_range(cuda_dev, m):
    """Finite results of scales whose product is beyond FP32: a 0 in the weights where x holds its type's lowest value, sums
    of a quarter, and weights near the largest value against small inputs."""
    low = torch.finfo(torch.bfloat16).min
    x = values(m, 160, torch.float32, cuda_dev, 11, 0.3)
    x[::2, 5] = low
    w = 40 * values(50, 160, torch.float32, cuda_dev, 12, 0.3)
    w[:, 5] = 0
    check_linear(x, w)
    check_linear(x.bfloat16(), w.bfloat16())
    x[:, :32], w[:, :32] = 0, 0
    x[:, 0], x[:, 1] = 2.0 ** 127, 2.0 ** 124
    w[:, 1], w[:, 2] = 4.0, 32.0
    w[:, 32:] = 0
    check_linear(x, w)  # (1/2 2^125) (1/2 2^3) = 2^126
    for big, small in ((126, -100), (122, -126), (118, 0), (0, 118), (-100, 126)):
        a = values(m, 160, torch.float32, cuda_dev, 13, 0.1).clamp(-2, 2) * 2.0 ** small
        b = values(50, 160, torch.float32, cuda_dev, 14, 0.1).clamp(-2, 2) * 2.0 ** big
        check_linear(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 2])
def test_results_below_the_normal_range(cuda_dev, m):
    """Few tokens: block sums are exact down to FP32's smallest number, so a result is off by 2^-149 a block and lane."""
    from mpq_b200.mx4 import mx4_linear, quantize_mx4
    a = values(m, 160, torch.float32, cuda_dev, 15, 0.3) * 2.0 ** -70
    b = values(50, 160, torch.float32, cuda_dev, 16, 0.3) * 2.0 ** -60
    want = plain_values(*plain_quantize(a)) @ plain_values(*plain_quantize(b)).T
    err = (mx4_linear(a, quantize_mx4(b)).cpu().double() - want).abs()
    assert bool((err <= 2.0 ** -149 * 10).all()) and bool(want.abs().min() > 0)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k", [(1, 32 * nb) for nb in (600, 718, 722, 723, 724)] + [(2, 32 * nb) for nb in (301, 361, 362)])
def test_rows_around_the_default_limit_of_shared_memory(cuda_dev, m, k):
    """x takes 68 bytes a block and token of shared memory; 48 KB is where a launch has to ask for more."""
    x = values(m, k, torch.bfloat16, cuda_dev, 8, 0.4)
    check_linear(x, values(9, k, torch.bfloat16, cuda_dev, 9, 0.4) * 0.05)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m,n,k", [(8, 4096, 4096), (100, 4096, 4096), (128, 2000, 8192), (64, 4100, 1500), (6, 130, 2050)])
def test_linear_with_a_bias_and_parts_of_k(cuda_dev, m, n, k, dtype):
    """Shapes whose K a cluster of two or four shares, tiles of 64 and of 128 columns."""
    x = values(m, k, dtype, cuda_dev, 10, 0.4)
    check_linear(x, values(n, k, dtype, cuda_dev, 11, 0.4) * 0.05, values(1, n, dtype, cuda_dev, 12, 0.4)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 2, 3, 130])
def test_every_code_at_every_place_of_a_block(cuda_dev, m):
    """Products with a single element of x: y is the weight itself, exactly, for each of the 16 codes at each of the 96
    places of a row (three blocks of different scales), whichever kernel the number of tokens selects."""
    from mpq_b200.mx4 import Mx4Tensor, mx4_linear, stored_shapes
    rows, cols = 16 * 3 + 1, 96
    r, j = torch.arange(rows)[:, None], torch.arange(cols)[None]
    code = (r * 5 + j * 7 + j // 16) % 16
    c = (120 + 5 * (j // 32) + r % 3).expand(rows, cols)[:, ::32]
    pairs = code.view(rows, -1, 2)
    codes = (pairs[..., 0] + 16 * pairs[..., 1]).to(torch.uint8)
    scales = torch.zeros(stored_shapes(rows, cols)[1], dtype=torch.uint8)
    b = torch.arange(3)[None]
    scales[r // 128, b // 4, (r % 32) * 16 + r % 128 // 32 * 4 + b % 4] = c.to(torch.uint8)
    w = Mx4Tensor(codes.to(cuda_dev), scales.to(cuda_dev), (rows, cols))
    want = plain_values(code, c)
    for start in range(0, cols, m):
        x = torch.zeros(m, cols)
        places = [(start + t) % cols for t in range(m)]
        x[torch.arange(m), places] = 1.0
        y = mx4_linear(x.to(cuda_dev), w)
        assert torch.equal(y.cpu().double(), want[:, places].T + 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m", [1, 2])
@pytest.mark.parametrize("n,k", [(70, 9000), (1800, 4128), (15001, 1056), (16000, 64)])
def test_every_code_in_slices_and_rounds(cuda_dev, n, k, m, dtype):
    """Few tokens, K in slices of several steps and rows in several rounds of a CTA: x has one element in each block, at every
    place in turn, so that y is a sum of one code of each block, exactly (multiples of 1/8 below 2^16)."""
    from mpq_b200.mx4 import Mx4Tensor, mx4_linear, stored_shapes
    nb = -(-k // 32)
    r, j = torch.arange(n, device=cuda_dev)[:, None], torch.arange(32 * nb, device=cuda_dev)[None]
    code = ((r * 5 + j * 7 + j // 16 + r * j // 97) % 16) * (j < k)
    b = torch.arange(nb, device=cuda_dev)[None]
    c = 125 + (r + 3 * b) % 6
    scales = torch.zeros(stored_shapes(n, k)[1], dtype=torch.uint8, device=cuda_dev)
    scales[r // 128, b // 4, (r % 32) * 16 + r % 128 // 32 * 4 + b % 4] = c.to(torch.uint8)
    pairs = code.view(n, -1, 2)
    w = Mx4Tensor((pairs[..., 0] + 16 * pairs[..., 1]).to(torch.uint8), scales, (n, k))
    q = GRID.to(cuda_dev)[code & 7] * torch.where(code >= 8, -1.0, 1.0) * torch.pow(2.0, c.double() - 127).repeat_interleave(32, 1)
    for place in range(0, 32, m):
        x = torch.zeros(m, k, device=cuda_dev, dtype=dtype)
        for t in range(m):
            at = 32 * torch.arange(nb, device=cuda_dev) + (place + t + 11 * torch.arange(nb, device=cuda_dev)) % 32
            x[t, at[at < k]] = 1.0
        want = (x.double() @ q[:, :k].T + 0.0).to(dtype)
        assert torch.equal(mx4_linear(x, w) + 0.0, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m,n,k", [(1, 40, 70), (2, 129, 300), (300, 1000, 520)])
def test_product_of_two_stored_matrices(cuda_dev, m, n, k, dtype):
    """mpq_mx4_gemm against the same product of the values that the two matrices stand for: both operands are exact, so
    only the FP32 sums (K 2^-23 of the sum of magnitudes, 2^-22 for sums that truncate) and one rounding are off."""
    from mpq_b200 import _lib, ops
    from mpq_b200.mx4 import dequantize_mx4, quantize_mx4
    g = torch.Generator().manual_seed(m + n + k)
    a, b = (quantize_mx4(torch.randn(r, k, generator=g).to(cuda_dev)) for r in (m, n))
    out = torch.full((m, n + 3), 7.0, device=cuda_dev, dtype=dtype)
    _lib.call("mpq_mx4_gemm", m, n, k, a.codes.data_ptr(), a.scales.data_ptr(), b.codes.data_ptr(), b.scales.data_ptr(),
              None, out.data_ptr(), {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype], n + 3,
              ops.status_word(cuda_dev).data_ptr())
    av, bv = dequantize_mx4(a).double(), dequantize_mx4(b).double()
    want, size = av @ bv.T, av.abs() @ bv.abs().T
    room = size * k * 2.0 ** -22 + want.abs() * {torch.float32: 0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    assert ((out[:, :n].double() - want).abs() <= room).all()
    assert (out[:, n:] == 7.0).all()


@pytest.mark.gpu
def test_empty_and_repeatable(cuda_dev):
    from mpq_b200.mx4 import dequantize_mx4, mx4_linear, quantize_mx4
    w = quantize_mx4(values(64, 96, torch.bfloat16, cuda_dev))
    assert mx4_linear(torch.zeros(0, 96, device=cuda_dev), w).shape == (0, 64)
    assert mx4_linear(torch.zeros(2, 0, 96, device=cuda_dev), w).shape == (2, 0, 64)
    none = quantize_mx4(torch.zeros(5, 0, device=cuda_dev))
    assert dequantize_mx4(none).shape == (5, 0)
    bias = torch.ones(5, device=cuda_dev)
    assert torch.equal(mx4_linear(torch.zeros(3, 0, device=cuda_dev), none, bias), torch.ones(3, 5, device=cuda_dev))
    assert dequantize_mx4(quantize_mx4(torch.zeros(0, 33, device=cuda_dev))).shape == (0, 33)
    for m in (1, 6, 50, 300):
        x = values(m, 96, torch.bfloat16, cuda_dev, m)
        assert torch.equal(mx4_linear(x, w), mx4_linear(x, w))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0,), (4, 0), (2, 3, 0), (2, 0, 0), (0, 3, 0)])
def test_linear_over_no_columns(cuda_dev, shape):
    """Sums over nothing, for every token there is: the bias alone, or zeros."""
    from mpq_b200.mx4 import dequantize_mx4, mx4_linear, quantize_mx4
    none = quantize_mx4(torch.zeros(5, 0, device=cuda_dev))
    bias = torch.arange(5.0, device=cuda_dev)
    x = torch.zeros(shape, device=cuda_dev)
    assert torch.equal(mx4_linear(x, none), torch.zeros(*shape[:-1], 5, device=cuda_dev))
    assert torch.equal(mx4_linear(x, none, bias), bias.expand(*shape[:-1], 5))
    assert dequantize_mx4(quantize_mx4(x)).shape == (math.prod(shape[:-1]), 0)


@pytest.mark.parametrize("cols,blocks", [(1, 1), (64, 2), (70, 3), (128, 4), (300, 10)])
def test_scales_are_padded_by_zeros(cols, blocks):
    """Whatever a caller's padding held; the caller's tensor and the scales that count stay as they are."""
    from mpq_b200.mx4 import Mx4Linear, Mx4Tensor, stored_shapes
    shape_codes, shape_scales = stored_shapes(130, cols)
    scales = torch.full(shape_scales, 255, dtype=torch.uint8)
    q = Mx4Tensor(torch.zeros(shape_codes, dtype=torch.uint8), scales, (130, cols))
    assert bool((scales == 255).all())
    real = torch.arange(4 * shape_scales[1]).view(1, -1, 1, 1, 4) < blocks
    want = torch.where(real, 255, 0).expand(2, -1, 32, 4, 4).reshape(shape_scales).to(torch.uint8)
    assert torch.equal(q.scales, want) and torch.equal(q.to("cpu").scales, want)
    layer = Mx4Linear(q)
    layer.load_state_dict({"codes": q.codes, "scales": scales})
    assert torch.equal(layer.mx4_weight.scales, want) and bool((scales == 255).all())


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 2, 3, 300, 2000])
def test_padding_of_a_callers_scales_does_not_matter(cuda_dev, m):
    from mpq_b200.mx4 import Mx4Linear, Mx4Tensor, mx4_linear, quantize_mx4
    for cols in (33, 70, 220):
        q = quantize_mx4(values(1000, cols, torch.float32, cuda_dev, cols, 0.3))
        over = -(-cols // 32) % 4
        scales = q.scales.clone()
        scales.view(*scales.shape[:2], 32, 4, 4)[:, -1, :, :, over:] = 255
        x = values(m, cols, torch.float32, cuda_dev, 3, 0.3)
        want = mx4_linear(x, q)
        assert bool(want.isfinite().all())
        assert torch.equal(mx4_linear(x, Mx4Tensor(q.codes, scales, q.shape)), want)
        layer = Mx4Linear(q)
        layer.load_state_dict({"codes": q.codes, "scales": scales})
        assert torch.equal(layer(x), want)


@pytest.mark.gpu
def test_another_stream_and_layers(cuda_dev):
    """Work queued on a stream of its own, and the module form against the function."""
    from mpq_b200.mx4 import Mx4Linear, convert_linears_mx4, mx4_linear, quantize_mx4
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(160, 96), torch.nn.Sequential(torch.nn.Linear(96, 40, bias=False))
                              ).to(cuda_dev).to(torch.bfloat16)
    x = values(37, 160, torch.bfloat16, cuda_dev, 1, 0.3)
    want = mx4_linear(mx4_linear(x, quantize_mx4(net[0].weight), net[0].bias), quantize_mx4(net[1][0].weight))
    assert convert_linears_mx4(net) == 2 and isinstance(net[1][0], Mx4Linear)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        outs = [net(x) for _ in range(20)]
    s.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    state = net.state_dict()
    assert math.prod(state["0.codes"].shape) == 96 * 160 // 2


@pytest.mark.gpu
def test_conversion_of_shared_layers(cuda_dev):
    """A layer with several places, in one module or in two, is converted once and stands at all of them."""
    from mpq_b200.mx4 import Mx4Linear, convert_linears_mx4
    shared = torch.nn.Linear(64, 64, device=cuda_dev)
    net = torch.nn.Sequential(shared, shared, torch.nn.Sequential(shared, torch.nn.Linear(64, 8, device=cuda_dev)))
    x = torch.randn(3, 64, device=cuda_dev)
    assert convert_linears_mx4(net) == 2
    assert isinstance(net[0], Mx4Linear) and net[1] is net[0] and net[2][0] is net[0] and isinstance(net[2][1], Mx4Linear)
    assert torch.equal(net(x), net[2][1](net[0](net[0](net[0](x)))))
    assert convert_linears_mx4(net) == 0


@pytest.mark.gpu
def test_product_in_a_cuda_graph(cuda_dev):
    from mpq_b200.mx4 import mx4_linear, quantize_mx4
    w = quantize_mx4(values(300, 512, torch.bfloat16, cuda_dev, 3, 0.3))
    for m in (1, 30, 150):
        x = values(m, 512, torch.bfloat16, cuda_dev, 4, 0.3)
        mx4_linear(x, w)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = mx4_linear(x, w)
        x.copy_(values(m, 512, torch.bfloat16, cuda_dev, 5, 0.3))
        graph.replay()
        assert torch.equal(y, mx4_linear(x, w))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 64), (5, 64), (300, 64), (2, 3, 64)])
def test_a_backward_pass_raises(cuda_dev, shape):
    """A linear in 4 bits has no gradient: through a skip connection, for x or the bias alone, or below other layers; what
    lies above it trains, and the forward pass is what it is without gradients."""
    from mpq_b200.mx4 import Mx4Linear, mx4_linear, quantize_mx4
    w = quantize_mx4(values(64, 64, torch.float32, cuda_dev, 1, 0.3))
    x, bias = torch.randn(*shape, device=cuda_dev), torch.randn(64, device=cuda_dev)
    want = mx4_linear(x, w, bias)
    assert not want.requires_grad
    for x_grad, bias_grad in ((True, False), (False, True), (True, True)):
        xs, bs = x.clone().requires_grad_(x_grad), bias.clone().requires_grad_(bias_grad)
        with torch.no_grad():
            assert not mx4_linear(xs, w, bs).requires_grad
        y = mx4_linear(xs, w, bs)
        assert y.requires_grad and torch.equal(y, want)
        y += x  # in place, as a residual stream may do
        with pytest.raises(RuntimeError, match="forward only"):
            (xs + y).sum().backward()
        assert xs.grad is None and bs.grad is None
    layer = Mx4Linear(w, bias)
    with pytest.raises(RuntimeError, match="forward only"):
        layer(x.clone().requires_grad_()).sum().backward()
    above = torch.nn.Linear(64, 3, device=cuda_dev)
    above(layer(x)).sum().backward()
    assert above.weight.grad is not None


def test_refusals_without_a_gpu():
    from mpq_b200 import _lib
    from mpq_b200.mx4 import Mx4Tensor, dequantize_mx4, mx4_linear, quantize_mx4
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="CUDA"):
        quantize_mx4(x)
    with pytest.raises(ValueError, match="uint8"):
        Mx4Tensor(torch.zeros(4, 32), torch.zeros(1, 1, 512, dtype=torch.uint8), (4, 64))
    with pytest.raises(ValueError, match="codes"):
        Mx4Tensor(torch.zeros(4, 31, dtype=torch.uint8), torch.zeros(1, 1, 512, dtype=torch.uint8), (4, 64))
    q = Mx4Tensor(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(1, 1, 512, dtype=torch.uint8), (4, 64))
    with pytest.raises(ValueError, match="CUDA"):
        dequantize_mx4(q)
    with pytest.raises(ValueError, match="CUDA"):
        mx4_linear(x, q)
    lib = _lib.load()
    assert lib.mpq_mx4_quantize(16, 7, 64, 4, 64, 16, 16, None) == 10001
    assert lib.mpq_mx4_quantize(16, 0, 63, 4, 64, 16, 16, None) == 10001
    assert lib.mpq_mx4_quantize(None, 0, 64, 4, 64, 16, 16, None) == 10001
    assert lib.mpq_mx4_quantize(16, 0, 64, 4, 64, 8, 16, None) == 10001 and b"aligned" in lib.mpq_last_error()
    assert lib.mpq_mx4_dequantize(16, 16, 4, 64, 16, 0, 63, None) == 10001
    assert lib.mpq_mx4_gemm(4, 4, 0, 16, 16, 16, 16, None, 16, 0, 4, 16, None) == 10001
    assert lib.mpq_mx4_gemm(4, 4, 64, 16, 16, 16, 16, None, 16, 0, 4, None, None) == 10001
    assert lib.mpq_mx4_quantize(None, 0, 64, 0, 64, None, None, None) == 0


@pytest.mark.gpu
def test_refusals(cuda_dev):
    from mpq_b200.mx4 import mx4_linear, quantize_mx4
    w = quantize_mx4(torch.zeros(8, 64, device=cuda_dev))
    with pytest.raises(ValueError, match="columns"):
        mx4_linear(torch.zeros(2, 65, device=cuda_dev), w)
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        mx4_linear(torch.zeros(2, 64, device=cuda_dev, dtype=torch.float64), w)
    with pytest.raises(ValueError, match="bias"):
        mx4_linear(torch.zeros(2, 64, device=cuda_dev), w, torch.zeros(8, device=cuda_dev, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="bias"):
        mx4_linear(torch.zeros(2, 64, device=cuda_dev), w, torch.zeros(7, device=cuda_dev))
    with pytest.raises(ValueError, match="different devices"):
        mx4_linear(torch.zeros(2, 64, device=cuda_dev), w.to("cpu"))
    with pytest.raises(ValueError, match="dimension"):
        quantize_mx4(torch.zeros((), device=cuda_dev))
