"""8-bit activation checkpoints for the layers the optimizer trains.

Between a forward and a backward pass, training holds the input of every
linear layer for the weight gradient and the input of every activation
function for its derivative.  This module holds them in 8 bits:

    packed = pack_input(x)              # int8 values, one power-of-two scale per 32 columns
    q, k, v = (linear(x, w, packed=packed) for w in (wq, wk, wv))   # one checkpoint, three layers
    y, packed_y = gelu(h, pack_output=True)                         # h and y held in 8 bits
    out = linear(y, w2, packed=packed_y)

Packing rounds x to x^ = q * 2^e with |x - x^| <= 2^(e-1) < max|x| / 127 over
each group of 32 columns of a row; outputs are computed from x itself, and only
weight gradients and GELU's derivative see x^.  A group with an infinity or a
NaN stands for NaN.  `pack` can return the column sums that the optimizer's
forward hook needs from the same read of x (stats=True); the optimizers of this
package do so by themselves for every `PackedLinear` they select.

`PackedLinear` is nn.Linear with a packed input.  Everything runs on CUDA
(sm_100) tensors in float32, bfloat16 or float16; there is no CPU path.
Forward-mode derivatives (torch.autograd.forward_ad) and tracing
(torch.jit.trace, make_fx) are refused.
"""
from __future__ import annotations

import math

import torch
from torch import nn

from . import _lib

__all__ = ["PackedActivation", "PackedLinear", "gelu", "gelu_backward", "linear", "pack", "pack_input", "unpack",
           "weight_gradient"]

GROUP = 32  # columns that share a scale
_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_GELU_FORMS = {"none": _lib.SM_GELU_ERF, "tanh": _lib.SM_GELU_TANH}


def values_ld(cols: int) -> int:
    """Bytes of one row of a checkpoint's int8 values."""
    return -(-cols // 16) * 16


def exponents_ld(cols: int) -> int:
    """Bytes of one row of a checkpoint's exponents."""
    return -(-cols // (4 * GROUP)) * 4


class PackedActivation:
    """An activation held in 8 bits.

    values: int8 [rows, columns rounded up to 16]; exponents: uint8 [rows,
    groups of 32 columns rounded up to 4], e + 127 (255: the group is NaN);
    shape, dtype: of the activation; sums: float32 [2, columns] (column sums of
    x^2 and of x) or None."""

    __slots__ = ("values", "exponents", "shape", "dtype", "sums", "_shared")

    def __init__(self, values: torch.Tensor, exponents: torch.Tensor, shape, dtype: torch.dtype,
                 sums: torch.Tensor | None = None):
        shape = tuple(shape)
        if not shape:
            raise ValueError("an activation has at least one dimension")
        rows, cols = math.prod(shape[:-1]), shape[-1]
        if dtype not in _DTYPES:
            raise TypeError(f"an activation must be float32, bfloat16 or float16; got {dtype}")
        if values.dtype != torch.int8 or values.shape != (rows, values_ld(cols)) or not values.is_contiguous():
            raise ValueError(f"values must be contiguous int8 [{rows}, {values_ld(cols)}]; "
                             f"got {values.dtype} {tuple(values.shape)}")
        if exponents.dtype != torch.uint8 or exponents.shape != (rows, exponents_ld(cols)) \
                or not exponents.is_contiguous() or exponents.device != values.device:
            raise ValueError(f"exponents must be contiguous uint8 [{rows}, {exponents_ld(cols)}] on the "
                             f"values' device; got {exponents.dtype} {tuple(exponents.shape)}")
        if sums is not None and (sums.dtype != torch.float32 or sums.shape != (2, cols)):
            raise ValueError(f"sums must be float32 [2, {cols}]")
        self.values, self.exponents, self.shape, self.dtype, self.sums = values, exponents, shape, dtype, sums
        self._shared = None

    @classmethod
    def _made(cls, parts, shape, dtype: torch.dtype, shared=None) -> "PackedActivation":
        """From what the binding returns, which needs no checks.  shared: through
        which layers called with the checkpoint sum their input gradients."""
        self = object.__new__(cls)
        self.values, self.exponents, self.sums = parts
        self.shape, self.dtype, self._shared = tuple(shape), dtype, shared
        return self

    def __getstate__(self):  # a copy is of the values alone
        return self.values, self.exponents, self.sums, self.shape, self.dtype

    def __setstate__(self, state):
        self.values, self.exponents, self.sums, self.shape, self.dtype = state
        self._shared = None

    @property
    def device(self) -> torch.device:
        return self.values.device

    @property
    def nbytes(self) -> int:
        """Bytes held for the backward pass."""
        return self.values.numel() + self.exponents.numel()

    def unpack(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        return unpack(self, dtype)


def _fits(packed: PackedActivation, delta: torch.Tensor, shape, what: str) -> None:
    if delta.dim() == 0:
        raise ValueError("a cotangent has at least one dimension")
    if delta.device != packed.values.device:
        raise ValueError(f"cotangent on {delta.device}, checkpoint on {packed.device}")
    if packed.shape != shape and (packed.shape[-1] != shape[-1] or packed.values.shape[0] != math.prod(shape[:-1])):
        raise ValueError(f"the checkpoint of a {packed.shape} activation does not fit {what} {tuple(shape)}")


def pack(x: torch.Tensor, *, stats: bool = False) -> PackedActivation:
    """The 8-bit checkpoint of x [..., columns] (any strides; not
    differentiable).  stats: also return the column sums of x^2 and x
    (PackedActivation.sums), from the same read of x."""
    parts, shared = _lib.binding().pack(x, stats)
    return PackedActivation._made(parts, x.shape, x.dtype, shared)


def pack_input(x: torch.Tensor, *, stats: bool = False) -> PackedActivation:
    """The checkpoint that linear layers reading x take under the current
    autocast state: of x as it comes, or of its float16 values where the layers
    compute in float16 (their cotangents then need those).  stats: the column
    sums of x as it comes, as the optimizers' hooks of plain layers take them."""
    parts, half, shared = _lib.binding().pack_input(x, stats)
    return PackedActivation._made(parts, x.shape, torch.float16 if half else x.dtype, shared)


def unpack(packed: PackedActivation, dtype: torch.dtype | None = None) -> torch.Tensor:
    """The values a checkpoint stands for, in the activation's type or `dtype`
    (float32 always holds them exactly; float16 only those packed from it)."""
    dtype = packed.dtype if dtype is None else dtype
    if dtype == torch.float16 and packed.dtype != torch.float16:
        raise TypeError(f"a checkpoint of {packed.dtype} values does not fit float16")
    return _lib.binding().unpack(packed.values, packed.exponents, packed.shape, dtype)


def weight_gradient(delta: torch.Tensor, packed: PackedActivation, *,
                    dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """dW [d_out, d_in] = delta^T x^ of a linear layer with output cotangent
    delta [..., d_out] and packed input [..., d_in], summed in FP32.  A float16
    cotangent needs a checkpoint packed from float16 values.  Not
    differentiable: with a delta that takes a gradient the result raises once
    something differentiates through it."""
    cols = packed.shape[-1]
    _fits(packed, delta, (*delta.shape[:-1], cols), "the rows of a cotangent with")
    if delta.dtype == torch.float16 and packed.dtype != torch.float16:
        raise TypeError(f"a float16 cotangent needs a checkpoint of float16 values; got {packed.dtype}")
    return _lib.binding().weight_gradient(delta, packed.values, packed.exponents, cols, dtype)


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
           packed: PackedActivation | None = None) -> torch.Tensor:
    """x W^T + b, holding x in 8 bits for the weight gradient.

    Computes in x's type, or autocast's where it is on; weight and bias are
    cast to it, and their gradients come in their own types, the weight's
    straight from the FP32 sum.  `packed`: x's checkpoint, where the caller has
    it already (several layers that read one x share one checkpoint; where it
    was packed while x takes a gradient, their input gradients are summed in
    FP32 and rounded once); else x is packed here if the weight needs a gradient.
    Differentiable once."""
    if packed is None:
        return _lib.binding().linear(x, weight, bias, None, None, 0, False, None)
    return _lib.binding().linear(x, weight, bias, packed.values, packed.exponents, packed.shape[-1],
                                 packed.dtype == torch.float16, packed._shared)


class PackedLinear(nn.Linear):
    """nn.Linear that holds its input in 8 bits between forward and backward
    (see `linear`).  forward(x, packed) takes the input's checkpoint where the
    caller has it.  Selected by the optimizers of this package like any
    nn.Linear; their forward hook then takes the activation statistics from the
    packing pass instead of reading x again."""

    def forward(self, x: torch.Tensor, packed: PackedActivation | None = None) -> torch.Tensor:
        return linear(x, self.weight, self.bias, packed=packed)

    @classmethod
    def from_linear(cls, module: nn.Linear) -> "PackedLinear":
        """A PackedLinear that shares `module`'s parameters."""
        out = cls(module.in_features, module.out_features, bias=module.bias is not None, device="meta")
        out.weight, out.bias = module.weight, module.bias
        return out.train(module.training)


def _gelu_form(approximate: str) -> int:
    form = _GELU_FORMS.get(approximate)
    if form is None:
        raise ValueError(f'approximate must be "none" or "tanh"; got {approximate!r}')
    return form


def gelu(x: torch.Tensor, *, approximate: str = "none", pack_output: bool = False, stats: bool = False):
    """GELU of x [..., columns], holding x in 8 bits for the derivative.

    approximate: "none" (x Phi(x)) or "tanh", as in torch.  pack_output: return
    (y, the checkpoint of y) for the layer that reads y, with y's column sums
    if `stats`.  One pass over x writes all of it.  Differentiable once."""
    if stats and not pack_output:
        raise ValueError("stats needs pack_output")
    y, parts = _lib.binding().gelu(x, _gelu_form(approximate), pack_output, stats)
    return (y, PackedActivation._made(parts, x.shape, x.dtype)) if pack_output else y


def gelu_backward(delta: torch.Tensor, packed: PackedActivation, *, approximate: str = "none") -> torch.Tensor:
    """delta * gelu'(x^) for the checkpoint of GELU's input, in delta's type:
    what `gelu` runs in its backward pass.  Not differentiable, as
    `weight_gradient`."""
    _fits(packed, delta, delta.shape, "a cotangent")
    return _lib.binding().gelu_backward(delta, packed.values, packed.exponents, _gelu_form(approximate))
