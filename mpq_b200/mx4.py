"""Microscaled 4-bit floating point (MX4): quantisation, reading back, and linear layers on it.

A row is cut into blocks of 32 elements; a block holds 4-bit E2M1 elements (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
negatives) and one power-of-two scale.  It is the 4-bit format that the tensor cores multiply directly, so it serves
next to the solved formats of this package as the round-to-nearest baseline at 4.25 bits a weight:

    w4 = quantize_mx4(layer.weight)         # once
    y = mx4_linear(x, w4, layer.bias)       # x is quantised within the call, token by token
    convert_linears_mx4(model.model)        # every nn.Linear below, in place

The operators run forward only: a backward pass through a linear raises.  Tensors must be on the GPU (there is no CPU
path).
"""
from __future__ import annotations

import math
from typing import Dict, List, Optional, Tuple

import torch

from . import ops
from ._lib import call_on, load, ptr

BLOCK = 32
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _dtype_code(dtype: torch.dtype) -> int:
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"MX4 operators take float32, bfloat16 or float16 tensors, not {dtype}")
    return code


def stored_shapes(rows: int, cols: int) -> Tuple[Tuple[int, int], Tuple[int, int, int]]:
    """Shapes of the codes and the scales (uint8) of a rows x cols matrix: two codes to a byte, rows padded to whole
    blocks; scales in tiles of 128 rows x 4 blocks, (row, block) at byte (row % 32) * 16 + (row % 128 // 32) * 4 +
    block % 4 of its tile (the layout in which the tensor cores take them).  Scales of blocks beyond a row's last, up to
    the tile's four, are 0."""
    blocks = -(-cols // BLOCK)
    return (rows, 16 * blocks), (-(-rows // 128), -(-blocks // 4), 512)


def _ends_inside_a_tile(cols: int) -> int:
    """Blocks of the last scale tile that a row fills, 0 where it fills all four."""
    return -(-cols // BLOCK) % 4


def _clear_padding(scales: torch.Tensor, cols: int) -> None:
    """Zeros in place of the scales beyond a row's last block.  The tensor cores multiply them with codes of 0, which a scale
    of 255 would make NaN."""
    over = _ends_inside_a_tile(cols)
    if over:
        scales.view(*scales.shape[:2], 32, 4, 4)[:, -1, :, :, over:] = 0


class Mx4Tensor:
    """A quantised matrix: ``codes`` and ``scales`` in the stored form (see ``stored_shapes``) and its ``shape``.  Scales that
    end inside a tile are copied, with zeros as their padding whatever it held."""

    __slots__ = ("codes", "scales", "shape")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape: Tuple[int, int]):
        self._hold(codes, scales, shape)
        if _ends_inside_a_tile(self.shape[1]):
            if self.scales is scales:
                self.scales = scales.clone()
            _clear_padding(self.scales, self.shape[1])

    def _hold(self, codes, scales, shape) -> None:
        rows, cols = int(shape[0]), int(shape[1])
        want_codes, want_scales = stored_shapes(rows, cols)
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise ValueError("MX4 codes and scales are uint8 tensors")
        if codes.shape != want_codes or scales.shape != want_scales:
            raise ValueError(f"a {rows} x {cols} MX4 matrix has codes {want_codes} and scales {want_scales}, got "
                             f"{tuple(codes.shape)} and {tuple(scales.shape)}")
        if codes.device != scales.device:
            raise ValueError("MX4 codes and scales are on different devices")
        if not codes.is_contiguous() or codes.data_ptr() % 16:
            codes = codes.clone(memory_format=torch.contiguous_format)
        if not scales.is_contiguous() or scales.data_ptr() % 16:
            scales = scales.clone(memory_format=torch.contiguous_format)
        self.codes, self.scales, self.shape = codes, scales, (rows, cols)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @classmethod
    def _checked(cls, codes, scales, shape) -> "Mx4Tensor":
        """A tensor whose parts are known to fit (they were just made)."""
        q = cls.__new__(cls)
        q.codes, q.scales, q.shape = codes, scales, shape
        return q

    @classmethod
    def _padded(cls, codes, scales, shape) -> "Mx4Tensor":
        """A tensor whose scales are known to be padded by zeros."""
        q = cls.__new__(cls)
        q._hold(codes, scales, shape)
        return q

    def to(self, device) -> "Mx4Tensor":
        return Mx4Tensor._padded(self.codes.to(device), self.scales.to(device), self.shape)

    def __repr__(self) -> str:
        return f"Mx4Tensor({self.shape[0]} x {self.shape[1]}, {self.codes.device})"


def _rows_of(x: torch.Tensor, what: str) -> torch.Tensor:
    """x as a matrix of rows with unit column stride (a copy only where the strides ask for one)."""
    if not x.is_cuda:
        raise ValueError("mpq_b200 kernels require CUDA tensors (there is no CPU path)")
    dims = x.dim()
    if dims < 1:
        raise ValueError(f"{what} needs at least one dimension")
    if dims != 2:
        x = x.reshape(math.prod(x.shape[:-1]), x.shape[-1])
    cols, (step, unit) = x.shape[1], x.stride()
    if (unit != 1 and cols != 1 or step < cols) and x.numel():
        x = x.contiguous()
    return x


def quantize_mx4(x: torch.Tensor) -> Mx4Tensor:
    """Quantise the rows of x (..., cols): block scale 2^(floor(log2 max|x|) - 2), elements to the nearest E2M1 value
    (ties to even), values beyond 6 scales saturate.  A block with an infinity or a NaN reads back as NaN."""
    x = _rows_of(x, "quantize_mx4")
    code = _dtype_code(x.dtype)
    rows, cols = x.shape
    shape_codes, shape_scales = stored_shapes(rows, cols)
    codes = torch.empty(*shape_codes, device=x.device, dtype=torch.uint8)
    scales = torch.empty(*shape_scales, device=x.device, dtype=torch.uint8)
    call_on(x.device.index, "mpq_mx4_quantize", x.data_ptr(), code, max(x.stride(0), cols), rows, cols, codes.data_ptr(),
            scales.data_ptr())
    return Mx4Tensor._checked(codes, scales, (rows, cols))


def dequantize_mx4(q: Mx4Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values a quantised matrix stands for (exact in float32 and bfloat16; float16 rounds or overflows where the
    scale leaves its range)."""
    code = _dtype_code(dtype)
    if not q.codes.is_cuda:
        raise ValueError("mpq_b200 kernels require CUDA tensors (there is no CPU path)")
    rows, cols = q.shape
    out = torch.empty(rows, cols, device=q.device, dtype=dtype)
    call_on(out.device.index, "mpq_mx4_dequantize", q.codes.data_ptr(), q.scales.data_ptr(), rows, cols,
            out.data_ptr(), code, max(cols, 1))
    return out


class _ForwardOnly(torch.autograd.Function):
    """Ties a result to the inputs whose gradient it does not have: a backward pass that needs it raises, where a detached
    result would leave their gradients short of its part."""

    @staticmethod
    def forward(ctx, out, *inputs):
        ctx.mark_dirty(out)
        return out

    @staticmethod
    def backward(ctx, grad):
        raise RuntimeError("mx4_linear runs forward only: it has no gradients for x or the bias (freeze what lies below the "
                           "4-bit linears, or run them under torch.no_grad())")


def mx4_linear(x: torch.Tensor, weight: Mx4Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y = Q(x) W^T + b for x (..., K) and a quantised W (N x K): x is quantised row by row, the products accumulate in
    FP32, and y (x's dtype) is rounded once.  Forward only: a backward pass that needs the gradient of x or of the bias
    raises.  Waits inside the kernels are bounded: ``ops.check_status`` raises, once the caller synchronises by it, if one
    ran out and left a result undefined."""
    tied = torch.is_grad_enabled() and (x.requires_grad or bias is not None and bias.requires_grad)
    given = (x, bias)
    rows = _rows_of(x, "mx4_linear")
    code = _dtype_code(x.dtype)
    n, k = weight.shape
    if rows.shape[1] != k:
        raise ValueError(f"mx4_linear: x has {rows.shape[1]} columns, the weight {k}")
    if weight.device != x.device:
        raise ValueError("mx4_linear: x and the weight are on different devices")
    if bias is not None:
        if bias.shape != (n,) or bias.dtype != x.dtype or bias.device != x.device:
            raise ValueError(f"mx4_linear: the bias must be {n} values of x's dtype on x's device")
        bias = bias.detach().contiguous()
    m = rows.shape[0]
    out = torch.empty(m, n, device=x.device, dtype=x.dtype)
    if m and n:
        if k == 0:
            out.zero_() if bias is None else out.copy_(bias.expand(m, n))
        else:
            need = load().mpq_mx4_linear_work(m, k)
            work = torch.empty(need, device=x.device, dtype=torch.uint8) if need else None
            call_on(x.device.index, "mpq_mx4_linear", rows.data_ptr(), code, max(rows.stride(0), k), m, n, k,
                    weight.codes.data_ptr(), weight.scales.data_ptr(), ptr(bias), ptr(work), out.data_ptr(), n,
                    ops.status_word(x.device).data_ptr())
    if x.dim() != 2:
        out = out.view(*x.shape[:-1], n)
    return _ForwardOnly.apply(out, *given) if tied else out


class Mx4Linear(torch.nn.Module):
    """A linear layer with its weight in MX4 (forward only: see ``mx4_linear``)."""

    def __init__(self, weight: Mx4Tensor, bias: Optional[torch.Tensor] = None):
        super().__init__()
        self.out_features, self.in_features = weight.shape
        self.register_buffer("codes", weight.codes)
        self.register_buffer("scales", weight.scales)
        self.register_buffer("bias", None if bias is None else bias.detach().clone())

    @classmethod
    def from_linear(cls, linear: torch.nn.Linear) -> "Mx4Linear":
        return cls(quantize_mx4(linear.weight), linear.bias)

    @property
    def mx4_weight(self) -> Mx4Tensor:
        return Mx4Tensor._padded(self.codes, self.scales, (self.out_features, self.in_features))

    def _load_from_state_dict(self, *args, **kwargs) -> None:
        super()._load_from_state_dict(*args, **kwargs)
        _clear_padding(self.scales, self.in_features)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return mx4_linear(x, self.mx4_weight, self.bias)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"


def convert_linears_mx4(module: torch.nn.Module) -> int:
    """Replace every ``nn.Linear`` below ``module`` by an ``Mx4Linear`` of its weight, at all of its places by the same one
    where it has several; returns how many there were."""
    places: Dict[int, List[Tuple[torch.nn.Module, str]]] = {}
    for parent in module.modules():
        for name, child in parent._modules.items():
            if isinstance(child, torch.nn.Linear):
                places.setdefault(id(child), []).append((parent, name))
    for at in places.values():
        parent, name = at[0]
        layer = Mx4Linear.from_linear(getattr(parent, name))
        for parent, name in at:
            setattr(parent, name, layer)
    return len(places)


__all__ = ["Mx4Tensor", "Mx4Linear", "convert_linears_mx4", "dequantize_mx4", "mx4_linear", "quantize_mx4",
           "stored_shapes"]
