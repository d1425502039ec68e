"""8-bit activation checkpoints on the GPU against the FP64 oracle: pack and
its column sums, unpack, weight gradient, GELU forward and backward.

Tolerances, from the arithmetic:
  pack, unpack      none: the quantiser and x^ are exact arithmetic
  column sums       FP32 partial sums: n terms in any order are off by at most
                    n * 2^-24 * sum|term|
  weight gradient   exact products; an FP32 sum of n terms (n cut at a tensor
                    core step of 16, three planes for FP32) that may truncate
                    is off by at most n * 2^-23 * sum|term|; then half a step
                    of the result's type
  GELU              erfc / tanh / exp of a few units in the last place, and an
                    argument rounded to FP32 that moves the tail by x^2 units:
                    (16 + 2 x^2) * 2^-24 relative to the sum of the magnitudes
                    of its terms, then half a step of the result's type"""
import numpy as np
import pytest
import torch

from oracle import activation_oracle as orc
from sandmuon_b200 import _lib, activations

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def name(dtype):
    return str(dtype).removeprefix("torch.")


def f64(t):
    return t.detach().double().cpu().numpy()


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def activation(rows, cols, dtype, seed=0, scale=0.5):
    g = torch.Generator().manual_seed(seed * 1000003 + rows * 131 + cols)
    x = torch.randn(rows, cols, generator=g) * torch.exp(torch.randn(cols, generator=g) * scale) + 0.1
    return x.to(dtype).to(DEV)


def cotangent(rows, cols, dtype, seed=1):
    g = torch.Generator().manual_seed(seed * 1000003 + rows * 137 + cols)
    scale = 0.25 if dtype == torch.float16 else 1e-3
    return (torch.randn(rows, cols, generator=g) * torch.exp(torch.randn(cols, generator=g) * .5) * scale).to(dtype).to(DEV)


def check_packed(packed, x):
    values, codes, hat = orc.checkpoint(f64(x).reshape(-1, x.shape[-1]), name(x.dtype))
    np.testing.assert_array_equal(packed.values.cpu().numpy(), values)
    np.testing.assert_array_equal(packed.exponents.cpu().numpy(), codes)
    np.testing.assert_array_equal(f64(packed.unpack(torch.float32)).reshape(hat.shape), hat)
    np.testing.assert_array_equal(f64(packed.unpack()).reshape(hat.shape), hat)
    return hat


def check_sums(sums, x):
    v = f64(x).reshape(-1, x.shape[-1])
    n = v.shape[0] + 8
    got = f64(sums)
    assert (np.abs(got[0] - (v ** 2).sum(0)) <= n * 2.0 ** -24 * (v ** 2).sum(0)).all()
    assert (np.abs(got[1] - v.sum(0)) <= n * 2.0 ** -24 * np.abs(v).sum(0)).all()


SHAPES = [(1, 1), (1, 768), (3, 31), (5, 32), (7, 33), (64, 16), (130, 40), (257, 129), (33, 1000), (1000, 264),
          (2049, 768), (17, 8200)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_pack_is_the_definition(rows, cols, dtype):
    x = activation(rows, cols, dtype)
    packed = activations.pack(x, stats=True)
    check_packed(packed, x)
    check_sums(packed.sums, x)
    plain = activations.pack(x)
    assert plain.sums is None
    assert torch.equal(plain.values, packed.values) and torch.equal(plain.exponents, packed.exponents)


@pytest.mark.parametrize("dtype", DTYPES)
def test_pack_strides_and_shapes(dtype):
    base = activation(96, 200, dtype)
    for x in (base[:, 3:180], base[::3], base.t(), base[:, ::2], base[5:6].expand(40, 200), base[:, 7:8].expand(96, 64),
              base.view(4, 24, 200), base.view(4, 24, 200).transpose(0, 1), base[0], base.view(2, 3, 16, 200)[:, :, ::2]):
        packed = activations.pack(x, stats=True)
        check_packed(packed, x)
        check_sums(packed.sums, x)
        assert packed.unpack().shape == x.shape


@pytest.mark.parametrize("dtype", DTYPES)
def test_pack_of_nothing(dtype):
    for shape in ((0, 40), (4, 0), (0, 0), (2, 0, 8)):
        packed = activations.pack(torch.empty(shape, dtype=dtype, device=DEV), stats=True)
        assert packed.unpack().shape == shape
        assert torch.equal(packed.sums, torch.zeros(2, shape[-1], device=DEV))


@pytest.mark.parametrize("dtype", DTYPES)
def test_pack_extremes(dtype):
    """Zeros, the type's largest and smallest magnitudes, exact borders
    127 * 2^e and the next number above, ties, infinities and NaN."""
    info = torch.finfo(dtype)
    x = torch.zeros(10, 96, dtype=dtype)
    x[1, 0], x[1, 40], x[1, 70] = info.max, -info.max, info.tiny
    x[2, 3] = info.smallest_normal * info.eps      # the smallest subnormal
    x[3, :32] = torch.linspace(-127, 127, 32)
    x[3, 32:64] = torch.linspace(-127, 127, 32) / 2 ** 7
    x[4, :32] = 127.0
    x[4, 1] = 127.0 * (1 + 2 * info.eps)
    x[5, :32] = (torch.arange(32) - 16 + 0.5).to(dtype)
    x[5, 31] = 127.0
    x[6, 10], x[6, 50], x[6, 90] = float("inf"), float("-inf"), float("nan")
    x[7, :] = info.max
    x[8, ::2] = info.smallest_normal
    x = x.to(DEV)
    for t in (x, x[:, :95], x.t().contiguous().t()):
        hat = check_packed(activations.pack(t), t)
        assert np.isnan(hat[6]).all()
    packed = activations.pack(x[:6], stats=True)
    if dtype != torch.float32 and dtype != torch.bfloat16:
        check_sums(packed.sums, x[:6])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("rows,d_in,d_out", [(1, 1, 1), (1, 64, 32), (3, 40, 7), (64, 128, 128), (65, 130, 260),
                                              (200, 257, 100), (1000, 300, 513), (4100, 96, 64), (777, 1000, 264)])
def test_weight_gradient(rows, d_in, d_out, dtype, out_dtype):
    x, delta = activation(rows, d_in, dtype), cotangent(rows, d_out, dtype)
    packed = activations.pack(x)
    check_weight_gradient(activations.weight_gradient(delta, packed, dtype=out_dtype), delta, packed, out_dtype)


def check_weight_gradient(got, delta, packed, out_dtype=torch.float32):
    d = f64(delta).reshape(-1, delta.shape[-1])
    hat = f64(packed.unpack(torch.float32)).reshape(d.shape[0], packed.shape[-1])
    want, size = d.T @ hat, np.abs(d).T @ np.abs(hat)
    bound = (d.shape[0] + 64) * 3 * 2.0 ** -23 * size + half_step(out_dtype) * np.abs(want)
    if out_dtype == torch.float16:
        bound = bound + 2.0 ** -25  # half a step of its subnormals
    assert got.shape == want.shape and got.dtype == out_dtype
    assert (np.abs(f64(got) - want) <= bound).all()
    if out_dtype == torch.float32 and np.linalg.norm(want) > 0:
        assert np.linalg.norm(f64(got) - want) <= 4e-6 * np.linalg.norm(want)
    assert _lib.device_status(DEV) == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_weight_gradient_strides(dtype):
    """Cotangents that cannot be read in place: transposed, sliced, broadcast
    along rows or columns (zero strides), higher-dimensional."""
    packed = activations.pack(activation(120, 72, dtype))
    base = cotangent(130, 150, dtype)
    for delta in (base[3:123, 5:70], cotangent(48, 120, dtype).t(), base[:120, ::3], base[:1, :56].expand(120, 56),
                  base[:120, :1].expand(120, 40), base[:120, :64], base[:120, :8].reshape(2, 60, 8)):
        check_weight_gradient(activations.weight_gradient(delta, packed), delta, packed)


def test_weight_gradient_without_rows_or_columns():
    for rows, d_in, d_out in ((0, 40, 24), (5, 0, 24), (5, 40, 0)):
        packed = activations.pack(torch.randn(rows, d_in, device=DEV))
        got = activations.weight_gradient(torch.randn(rows, d_out, device=DEV), packed)
        assert torch.equal(got, torch.zeros(d_out, d_in, device=DEV))


@pytest.mark.parametrize("dtype", DTYPES)
def test_weight_gradient_nonfinite(dtype):
    """A NaN group reaches its 32 columns of dW and no others; an infinite or
    NaN cotangent its row of dW."""
    x, delta = activation(100, 96, dtype), cotangent(100, 40, dtype)
    x[50, 40] = float("inf")
    got = activations.weight_gradient(delta, activations.pack(x))
    assert torch.isnan(got[:, 32:64]).all() and torch.isfinite(got[:, :32]).all() and torch.isfinite(got[:, 64:]).all()
    x = activation(100, 96, dtype).abs() + 1
    delta[7, 3], delta[8, 4], delta[9, 5] = float("inf"), float("-inf"), float("nan")
    got = activations.weight_gradient(delta, activations.pack(x))
    assert (got[3] == float("inf")).all() and (got[4] == float("-inf")).all() and torch.isnan(got[5]).all()
    assert torch.isfinite(got[:3]).all() and torch.isfinite(got[6:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_weight_gradient_is_deterministic(dtype):
    x, delta = activation(3000, 520, dtype), cotangent(3000, 300, dtype)
    packed = activations.pack(x)
    first = activations.weight_gradient(delta, packed)
    for _ in range(5):
        assert torch.equal(first, activations.weight_gradient(delta, packed))


def test_weight_gradient_adversarial_checkpoint():
    """Values a packer never writes (-128, scattered exponents, padding that is
    not zero) still multiply out as int8 times a power of two, and padding
    reaches no result."""
    g = torch.Generator().manual_seed(5)
    rows, d_in, d_out = 90, 37, 20
    values = torch.randint(-128, 128, (rows, 48), generator=g, dtype=torch.int8).to(DEV)
    codes = torch.randint(100, 150, (rows, 4), generator=g, dtype=torch.uint8).to(DEV)
    for dtype in (torch.bfloat16, torch.float32):
        packed = activations.PackedActivation(values, codes, (rows, d_in), dtype)
        scale = torch.pow(2.0, codes.cpu().double() - 127).repeat_interleave(32, 1)
        hat = values.cpu().double()[:, :d_in] * scale[:, :d_in]
        assert torch.equal(packed.unpack(torch.float32).cpu().double(), hat)
        delta = cotangent(rows, d_out, dtype)
        check_weight_gradient(activations.weight_gradient(delta, packed), delta, packed)


# ----------------------------------------------------------------------- GELU

def gelu_bounds(x, approximate):
    """(y, slope, allowance of y, allowance of the slope), relative errors of
    the FP32 evaluation as in the module docstring."""
    y, slope = orc.gelu(x, approximate)
    c = (16 + 2 * np.minimum(x * x, 400.0)) * 2.0 ** -24
    phi = np.abs(y) / np.maximum(np.abs(x), 1e-300) + (x == 0) * 0.5
    if approximate == "tanh":  # 1 + tanh cancels for negative x
        return y, slope, c * np.abs(x), c * (1 + np.abs(x) + np.abs(x) ** 3 * (np.abs(x) < 12))
    dense = np.abs(x) * np.exp(-x * x / 2)
    return y, slope, c * np.abs(y) + 2.0 ** -120, c * (phi + dense) + 2.0 ** -120


@pytest.mark.parametrize("approximate", ["none", "tanh"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 64), (5, 33), (64, 128), (130, 257), (999, 1000)])
def test_gelu(rows, cols, dtype, approximate):
    x = activation(rows, cols, dtype, scale=1.0)
    delta = cotangent(rows, cols, dtype)
    leaf = x.clone().requires_grad_()
    y, packed = activations.gelu(leaf, approximate=approximate, pack_output=True, stats=True)
    dx, = torch.autograd.grad(y, leaf, delta)
    alone = activations.gelu(x, approximate=approximate)
    assert torch.equal(alone, y) and not alone.requires_grad
    want, _, allowed, _ = gelu_bounds(f64(x), approximate)
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert (np.abs(f64(y) - want) <= allowed + half_step(dtype) * np.abs(want) + tiny / 2).all()
    check_packed(packed, y)
    check_sums(packed.sums, y)
    hat = orc.checkpoint(f64(x), name(dtype))[2]
    _, slope, _, allowed = gelu_bounds(hat, approximate)
    d = f64(delta)
    assert dx.dtype == dtype
    assert (np.abs(f64(dx) - d * slope) <= np.abs(d) * (allowed + half_step(dtype) * np.abs(slope)) + tiny).all()
    assert torch.equal(dx, activations.gelu_backward(delta, activations.pack(x), approximate=approximate))


@pytest.mark.parametrize("approximate", ["none", "tanh"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gelu_extremes(dtype, approximate):
    """Far arguments: y is x or 0, the slope 1 or 0, never NaN; NaN stays NaN
    and takes its group's derivative along."""
    top = torch.finfo(dtype).max
    x = torch.tensor([[top, -top, 1000.0, -1000.0, 40.0, -40.0, 0.0, -0.0]], dtype=dtype, device=DEV)
    rows = x.t().expand(8, 32).contiguous()  # a group for each
    leaf = rows.clone().requires_grad_()
    y = activations.gelu(leaf, approximate=approximate)
    want = torch.clamp(rows, min=0)
    assert torch.equal(y, want)
    dx, = torch.autograd.grad(y, leaf, torch.ones_like(y))
    assert torch.equal(dx, torch.where(rows > 0, 1.0, torch.where(rows < 0, 0.0, 0.5)).to(dtype))
    leaf = torch.ones(2, 64, dtype=dtype, device=DEV)
    leaf[1, 3] = float("nan")
    leaf.requires_grad_()
    y = activations.gelu(leaf, approximate=approximate)
    dx, = torch.autograd.grad(y, leaf, torch.ones_like(y))
    assert torch.isnan(y).sum() == 1 and torch.isnan(dx).sum() == 32 and torch.isnan(dx[1, :32]).all()


def test_gelu_strides_broadcast_cotangent_and_shapes():
    base = activation(60, 100, torch.float32)
    for x in (base.t(), base[:, 3:40], base.view(3, 20, 100), base[0], base[:, ::2], base[:0]):
        leaf = x.detach().requires_grad_()
        y = activations.gelu(leaf)
        assert y.shape == x.shape
        y.sum().backward()  # an expanded cotangent
        want = activations.gelu_backward(torch.ones(x.shape, device=DEV), activations.pack(x))
        assert torch.equal(leaf.grad, want)


def test_gelu_derivative_against_differences():
    """dx of the packed input against central differences of the oracle at x^."""
    x = activation(8, 64, torch.float32).requires_grad_()
    y = activations.gelu(x)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    hat, h = orc.checkpoint(f64(x), "float32")[2], 1e-5
    diff = (orc.gelu(hat + h, "none")[0] - orc.gelu(hat - h, "none")[0]) / (2 * h)
    assert np.abs(f64(dx) - diff).max() < 1e-6
