"""Numerics of the 8-bit checkpoint operators beyond single calls: statistics
under autocast, long sums, negative views, infinities, and what is left when a
wait of the weight gradient runs out.

Tolerances, from the arithmetic: an FP32 chain of n additions of terms of one
sign is off by at most n * 2^-24 relative; FP64 joins add one rounding to FP32."""
import numpy as np
import pytest
import torch

from sandmuon_b200 import DiagonalWeightedPE, RankOneAWeightedPE, _lib, activations
from test_gpu_activations import DTYPES, activation, check_packed, check_sums, check_weight_gradient, cotangent, f64

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


# ------------------------------------------------------------------ statistics

def between_halves(rows, cols):
    """FP32 values that FP16 rounds all the same way (by 2^-12 relative), and
    some that it cannot hold."""
    x = torch.full((rows, cols), 1 + 2.0 ** -12, device=DEV)
    x[:, ::3] *= -1
    return x


@pytest.mark.parametrize("cols", [40, 128])
def test_statistics_under_autocast_are_of_the_input_itself(cols):
    """FP16 layers keep a checkpoint of the FP16 values; the column sums are
    those of the FP32 input, as a plain layer's hook takes them."""
    x = between_halves(64, cols)
    x[3, 1], x[5, 2] = 7e4, -3e5  # past FP16's range
    for dtype in (torch.float16, torch.bfloat16):
        with torch.autocast("cuda", dtype=dtype):
            packed = activations.pack_input(x, stats=True)
            assert activations.pack_input(x).sums is None
        source = x.half() if dtype == torch.float16 else x
        assert packed.dtype == source.dtype
        plain = activations.pack(source)
        assert torch.equal(packed.values, plain.values) and torch.equal(packed.exponents, plain.exponents)
        check_sums(packed.sums, x)
    for shape in ((0, cols), (2, 0, cols), (cols,)):
        with torch.autocast("cuda", dtype=torch.float16):
            packed = activations.pack_input(torch.ones(shape, device=DEV), stats=True)
        assert packed.shape == shape and packed.sums.shape == (2, cols)
        assert torch.equal(packed.sums, torch.full((2, cols), float(shape == (cols,)), device=DEV))


@pytest.mark.parametrize("rank_one", [True, False])
def test_hook_statistics_of_packed_and_plain_layers_agree_under_autocast(rank_one):
    """150 terms of one sign: both sums are within 158 * 2^-24 of the exact one."""
    x = between_halves(150, 64)
    make = RankOneAWeightedPE if rank_one else DiagonalWeightedPE
    keys = ("a_sum", "a_first_sum") if rank_one else ("a_sum",)
    seen = []
    for layer in (torch.nn.Linear(64, 48), activations.PackedLinear(64, 48)):
        model = torch.nn.Sequential(layer).to(DEV)
        opt = make(model, lr=1e-2)
        with torch.autocast("cuda", dtype=torch.float16):
            model(x).float().sum().backward()
        seen.append([f64(opt.state[layer.weight][k]) for k in keys])
        opt.close()
    for a, b in zip(*seen):
        assert (np.abs(a - b) <= 2 * 158 * 2.0 ** -24 * np.abs(a)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_column_sums_of_a_tall_and_wide_input(dtype):
    """A lane adds at most 128 rows in FP32 before the FP64 join, whatever the
    shape: equal terms, whose rounding errors add up, stay within 132 * 2^-24.
    (One broadcast row: the input itself takes no memory.)"""
    rows, cols = 16384, 131072
    row = (torch.arange(cols, device=DEV) % 977 + 300).float().mul_(0.001).to(dtype)
    x = row.expand(rows, cols)
    packed = activations.pack(x, stats=True)
    v = row.double()
    want = torch.stack((v * v, v)) * rows
    assert float(((packed.sums.double() - want).abs() / want).max()) <= 132 * 2.0 ** -24
    del packed
    odd = row[1:].expand(rows, cols - 1)  # the element mapping
    sums = activations.pack(odd, stats=True).sums
    assert float(((sums.double() - want[:, 1:]).abs() / want[:, 1:]).max()) <= 132 * 2.0 ** -24


# ------------------------------------------------------ waits that run out

@pytest.fixture
def expired():
    """Lets a worker (a CTA pair) of the following weight gradients take its
    first wait as run out; the library does no work and waits for nothing
    there, so nothing hangs."""
    yield _lib.load().sm_inject_expired_wait
    _lib.load().sm_inject_expired_wait(-1)
    _lib.device_status(DEV)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,d_in,d_out", [
    (300, 40, 24),         # one worker, one tile
    (20000, 64, 300),      # two tiles in equal parts
    (1100, 2048, 1280),    # stretches across tile borders
    (2000, 2304, 2304),    # whole tiles and shared ones
])
def test_a_wait_that_ran_out_leaves_nan(rows, d_in, d_out, dtype, expired):
    """Every element is the right one or NaN: no memory that was never written
    is returned as a gradient, and the status word says what happened."""
    x, delta = activation(rows, d_in, dtype), cotangent(rows, d_out, dtype)
    packed = activations.pack(x)
    for out_dtype in (torch.float32, torch.bfloat16):
        want = activations.weight_gradient(delta, packed, dtype=out_dtype)
        assert _lib.device_status(DEV) == 0
        for worker in (0, 1, 5, 71):
            assert expired(worker) == 0
            # memory of the result: full of a value that is not the gradient's
            torch.full((d_out, d_in), 7.0, dtype=out_dtype, device=DEV)
            got = activations.weight_gradient(delta, packed, dtype=out_dtype)
            assert expired(-1) == 0
            bad = torch.isnan(got)
            assert torch.equal(got[~bad], want[~bad])
            assert (_lib.device_status(DEV) != 0) == bool(bad.any())
            if worker == 0:
                assert bad.any()
            # whole 256 x 256 tiles
            tiles = torch.nn.functional.max_pool2d(bad[None].float(), 256, ceil_mode=True)[0]
            full = tiles.repeat_interleave(256, 0).repeat_interleave(256, 1)[:d_out, :d_in]
            assert torch.equal(full > 0, bad)
        assert torch.equal(activations.weight_gradient(delta, packed, dtype=out_dtype), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_views_that_stand_for_their_negative(dtype):
    """The imaginary part of a conjugate is a real tensor whose memory holds
    the opposite sign."""
    kind = torch.complex64 if dtype == torch.float32 else torch.complex32
    base = activation(40, 64, dtype)
    z = torch.zeros(40, 64, dtype=kind, device=DEV)
    torch.view_as_real(z)[..., 1] = base
    x = z.conj().imag
    assert x.is_neg() and x.dtype == dtype
    want = -base
    packed = activations.pack(x, stats=True)
    check_packed(packed, want)
    check_sums(packed.sums, want)
    check_weight_gradient(activations.weight_gradient(x, packed), want, packed)
    assert torch.equal(activations.gelu(x), activations.gelu(want))
    assert torch.equal(activations.gelu_backward(x, packed), activations.gelu_backward(want, packed))


# ------------------------------------------------------------------ long sums

@pytest.mark.parametrize("dtype", DTYPES)
def test_long_sums_are_cut_into_chains(dtype):
    """Tensor cores truncate as they add, so their error grows with the length
    of a chain; the kernel ends chains after 128 steps (2048 tokens, or 672 for
    the three products of an FP32 cotangent) and adds them with rounding.  A
    whole tile of a long sum is therefore, bit for bit, the FP32 sum of what
    the chains' tokens give on their own.  (Of the 81 tiles the first few are
    shared out by tokens instead.)"""
    chain, chains, width = 672 if dtype == torch.float32 else 2048, 8, 2304
    rows = chain * chains
    x, delta = activation(rows, width, dtype), cotangent(rows, width, dtype)
    got = activations.weight_gradient(delta, activations.pack(x))
    want = 0
    for i in range(0, rows, chain):
        want = want + activations.weight_gradient(delta[i:i + chain], activations.pack(x[i:i + chain]))
    assert torch.equal(got[1024:], want[1024:])


# ------------------------------------------------------------------ infinities

@pytest.mark.parametrize("approximate", ["none", "tanh"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [64, 33])
def test_gelu_of_infinities(cols, dtype, approximate):
    """+inf gives inf and -inf NaN, as x Phi(x) does in floating point and
    torch's own GELU; their group's derivative is NaN, and no other's."""
    x = activation(6, cols, dtype)
    x[1, 3], x[2, 5] = float("inf"), float("-inf")
    leaf = x.clone().requires_grad_()
    y, packed = activations.gelu(leaf, approximate=approximate, pack_output=True)
    ours, torchs = f64(y), f64(torch.nn.functional.gelu(x, approximate=approximate))
    assert np.array_equal(np.isnan(ours), np.isnan(torchs)) and np.array_equal(np.isinf(ours), np.isinf(torchs))
    assert ours[1, 3] == np.inf and np.isnan(ours[2, 5]) and np.isfinite(np.delete(ours, [1, 2], 0)).all()
    hat = f64(packed.unpack(torch.float32))
    dx = f64(torch.autograd.grad(y, leaf, torch.ones_like(y))[0])
    for got in (hat, dx):
        assert np.isnan(got[1:3, :32]).all() and np.isfinite(got[1:3, 32:]).all()
        assert np.isfinite(np.delete(got, [1, 2], 0)).all()
