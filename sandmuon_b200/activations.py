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
"""
from __future__ import annotations

import math

import torch
from torch import nn

from . import _lib, engine

__all__ = ["PackedActivation", "PackedLinear", "gelu", "gelu_backward", "linear", "pack", "pack_input", "unpack",
           "weight_gradient"]


class PackedActivation:
    """An activation held in 8 bits.

    values: int8 [rows, columns rounded up to 16]; exponents: uint8 [rows,
    groups of 32 columns rounded up to 4], e + 127 (255: the group is NaN);
    shape, dtype: of the activation; sums: float32 [2, columns] (column sums of
    x^2 and of x) or None."""

    __slots__ = ("values", "exponents", "shape", "dtype", "sums")

    def __init__(self, values: torch.Tensor, exponents: torch.Tensor, shape, dtype: torch.dtype,
                 sums: torch.Tensor | None = None):
        shape = tuple(shape)
        if not shape:
            raise ValueError("an activation has at least one dimension")
        rows, cols = math.prod(shape[:-1]), shape[-1]
        if dtype not in engine.ACTIVATION_DTYPES:
            raise TypeError(f"an activation must be float32, bfloat16 or float16; got {dtype}")
        if values.dtype != torch.int8 or values.shape != (rows, engine.activation_ld(cols)) \
                or not values.is_contiguous():
            raise ValueError(f"values must be contiguous int8 [{rows}, {engine.activation_ld(cols)}]; "
                             f"got {values.dtype} {tuple(values.shape)}")
        if exponents.dtype != torch.uint8 or exponents.shape != (rows, engine.activation_lde(cols)) \
                or not exponents.is_contiguous() or exponents.device != values.device:
            raise ValueError(f"exponents must be contiguous uint8 [{rows}, {engine.activation_lde(cols)}] on the "
                             f"values' device; got {exponents.dtype} {tuple(exponents.shape)}")
        if sums is not None and (sums.dtype != torch.float32 or sums.shape != (2, cols)):
            raise ValueError(f"sums must be float32 [2, {cols}]")
        self.values, self.exponents, self.shape, self.dtype, self.sums = values, exponents, shape, dtype, sums

    @property
    def device(self) -> torch.device:
        return self.values.device

    @property
    def nbytes(self) -> int:
        """Bytes held for the backward pass."""
        return self.values.numel() + self.exponents.numel()

    def unpack(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        return unpack(self, dtype)


def _flat(t: torch.Tensor) -> torch.Tensor:
    return t if t.dim() == 2 else t.reshape(math.prod(t.shape[:-1]), t.shape[-1])


def _of_shape(packed: PackedActivation, shape, what: str) -> None:
    if packed.shape != shape and (packed.shape[-1] != shape[-1]
                                  or packed.values.shape[0] != math.prod(shape[:-1])):
        raise ValueError(f"the checkpoint of a {packed.shape} activation does not fit {what} {tuple(shape)}")


def pack(x: torch.Tensor, *, stats: bool = False) -> PackedActivation:
    """The 8-bit checkpoint of x [..., columns] (any strides; not
    differentiable).  stats: also return the column sums of x^2 and x
    (PackedActivation.sums), from the same read of x."""
    if x.dim() == 0:
        raise ValueError("an activation has at least one dimension")
    x = x.detach()
    values, exponents, sums = engine.pack_activations(_flat(x), stats)
    return PackedActivation(values, exponents, x.shape, x.dtype, sums)


def unpack(packed: PackedActivation, dtype: torch.dtype | None = None) -> torch.Tensor:
    """The values a checkpoint stands for, in the activation's type or `dtype`
    (float32 always holds them exactly; float16 only those packed from it)."""
    dtype = packed.dtype if dtype is None else dtype
    if dtype == torch.float16 and packed.dtype != torch.float16:
        raise TypeError(f"a checkpoint of {packed.dtype} values does not fit float16")
    out = engine.unpack_activations(packed.values, packed.exponents, packed.shape[-1], dtype)
    return out if len(packed.shape) == 2 else out.view(packed.shape)


def weight_gradient(delta: torch.Tensor, packed: PackedActivation, *,
                    dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """dW [d_out, d_in] = delta^T x^ of a linear layer with output cotangent
    delta [..., d_out] and packed input [..., d_in], summed in FP32.  A float16
    cotangent needs a checkpoint packed from float16 values."""
    if delta.dim() == 0:
        raise ValueError("a cotangent has at least one dimension")
    if delta.device != packed.device:
        raise ValueError(f"cotangent on {delta.device}, checkpoint on {packed.device}")
    if delta.dtype == torch.float16 and packed.dtype != torch.float16:
        raise TypeError(f"a float16 cotangent needs a checkpoint of float16 values; got {packed.dtype}")
    _of_shape(packed, (*delta.shape[:-1], packed.shape[-1]), "the rows of a cotangent with")
    return engine.weight_gradient(_flat(delta.detach()), packed.values, packed.exponents, packed.shape[-1], dtype)


# ---------------------------------------------------------------- linear layer

class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, packed):
        dtype = x.dtype
        cast = weight if weight.dtype == dtype else weight.to(dtype)
        ctx.save_for_backward(cast, packed.values, packed.exponents)
        ctx.x_shape, ctx.weight_dtype = x.shape, weight.dtype
        if bias is None:
            return torch.nn.functional.linear(x, cast)
        ctx.bias_dtype = bias.dtype
        return torch.nn.functional.linear(x, cast, bias.to(dtype))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, delta):
        cast, values, exponents = ctx.saved_tensors
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        rows = _flat(delta)
        dx = dw = db = None
        if need_x:
            dx = torch.mm(rows, cast)
            if dx.shape != ctx.x_shape:
                dx = dx.view(ctx.x_shape)
        if need_w:
            dw = engine.weight_gradient(rows, values, exponents, ctx.x_shape[-1], ctx.weight_dtype)
        if need_b:
            db = engine.column_sums(rows)
            if ctx.bias_dtype != torch.float32:
                db = db.to(ctx.bias_dtype)
        return dx, dw, db, None


def _compute_dtype(x: torch.Tensor) -> torch.dtype:
    """The type a linear layer computes in: autocast's where it is on, else x's."""
    return torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else x.dtype


def pack_input(x: torch.Tensor, *, stats: bool = False) -> PackedActivation:
    """The checkpoint that linear layers reading x take under the current
    autocast state: of x as it comes, or of its float16 values where the layers
    compute in float16 (their cotangents then need those)."""
    return pack(x.to(torch.float16) if _compute_dtype(x) == torch.float16 else x, stats=stats)


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
           packed: PackedActivation | None = None) -> torch.Tensor:
    """x W^T + b, holding x in 8 bits for the weight gradient.

    Computes in x's type, or autocast's where it is on; weight and bias are
    cast to it, and their gradients come in their own types, the weight's
    straight from the FP32 sum.  `packed`: x's checkpoint, where the caller has
    it already (several layers that read one x share one checkpoint); else x is
    packed here if the weight needs a gradient."""
    if weight.dim() != 2 or x.dim() == 0 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear: input {tuple(x.shape)} does not fit weight {tuple(weight.shape)}")
    if bias is not None and bias.shape != (weight.shape[0],):
        raise ValueError(f"linear: bias {tuple(bias.shape)} does not fit weight {tuple(weight.shape)}")
    _lib.ensure_device(x.device)
    dtype = _compute_dtype(x)
    types = engine.ACTIVATION_DTYPES
    if dtype not in types or weight.dtype not in types or (bias is not None and bias.dtype not in types):
        raise TypeError(f"linear computes in float32, bfloat16 or float16, with weight and bias of these types; got "
                        f"{dtype}, {weight.dtype}, {None if bias is None else bias.dtype}")
    if packed is not None:
        if packed.device != x.device:
            raise ValueError(f"input on {x.device}, checkpoint on {packed.device}")
        _of_shape(packed, x.shape, "an input")
        if dtype == torch.float16 and packed.dtype != torch.float16:
            raise TypeError(f"a float16 layer needs a checkpoint of float16 values; got {packed.dtype}")
    if not (torch.is_grad_enabled() and weight.requires_grad):
        # nothing reads the checkpoint, and torch's own layer keeps no x
        return torch.nn.functional.linear(x.to(dtype), weight.to(dtype), None if bias is None else bias.to(dtype))
    if packed is None:
        packed = pack_input(x)
    return _Linear.apply(x if x.dtype == dtype else x.to(dtype), weight, bias, packed)


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


# ------------------------------------------------------------------------ GELU

class _Gelu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, approximate, pack_output, stats):
        y, kept, packed = engine.gelu_forward(_flat(x), approximate, True, pack_output, stats)
        ctx.save_for_backward(*kept)
        ctx.approximate, ctx.x_shape = approximate, x.shape
        y = y.view(x.shape)
        if not pack_output:
            return y
        values, exponents, sums = packed
        ctx.mark_non_differentiable(values, exponents, *(() if sums is None else (sums,)))
        ctx.set_materialize_grads(False)
        return y, values, exponents, sums

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, delta, *_):
        if delta is None:
            return None, None, None, None
        values, exponents = ctx.saved_tensors
        dx = engine.gelu_backward(_flat(delta), values, exponents, ctx.approximate)
        return dx.view(ctx.x_shape), None, None, None


def gelu(x: torch.Tensor, *, approximate: str = "none", pack_output: bool = False, stats: bool = False):
    """GELU of x [..., columns], holding x in 8 bits for the derivative.

    approximate: "none" (x Phi(x)) or "tanh", as in torch.  pack_output: return
    (y, the checkpoint of y) for the layer that reads y, with y's column sums
    if `stats`.  One pass over x writes all of it."""
    if x.dim() == 0:
        raise ValueError("an activation has at least one dimension")
    if stats and not pack_output:
        raise ValueError("stats needs pack_output")
    if torch.is_grad_enabled() and x.requires_grad:
        out = _Gelu.apply(x, approximate, pack_output, stats)
        if not pack_output:
            return out
        y, values, exponents, sums = out
    else:
        y, _, packed = engine.gelu_forward(_flat(x.detach()), approximate, False, pack_output, stats)
        y = y.view(x.shape)
        if not pack_output:
            return y
        values, exponents, sums = packed
    return y, PackedActivation(values, exponents, x.shape, x.dtype, sums)


def gelu_backward(delta: torch.Tensor, packed: PackedActivation, *, approximate: str = "none") -> torch.Tensor:
    """delta * gelu'(x^) for the checkpoint of GELU's input, in delta's type:
    what `gelu` runs in its backward pass."""
    if delta.dim() == 0:
        raise ValueError("a cotangent has at least one dimension")
    if delta.device != packed.device:
        raise ValueError(f"cotangent on {delta.device}, checkpoint on {packed.device}")
    _of_shape(packed, delta.shape, "a cotangent")
    return engine.gelu_backward(_flat(delta.detach()), packed.values, packed.exponents, approximate).view(delta.shape)
