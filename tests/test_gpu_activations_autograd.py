"""The 8-bit checkpoint operators inside autograd: second and forward
derivatives, tracing, in-place changes of outputs, memory of a backward pass.

An operator that cannot give what is asked of it raises; it never returns a
constant in its place."""
import pytest
import torch
import torch.fx.experimental.proxy_tensor

from sandmuon_b200 import activations
from test_gpu_activations import DTYPES, activation, cotangent

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def weight(d_out, d_in, seed=0):
    g = torch.Generator().manual_seed(seed + 7 * d_out + d_in)
    return (torch.randn(d_out, d_in, generator=g) * .05).to(DEV).requires_grad_()


# --------------------------------------------------------- second derivatives

def test_a_penalty_on_the_input_gradient_of_a_linear_layer_raises():
    """d(sum y)/dx = 1^T W depends on the weight although the cotangent is a
    constant."""
    x, w = activation(40, 64, torch.float32).requires_grad_(), weight(16, 64)
    b = torch.zeros(16, device=DEV, requires_grad=True)
    for bias in (None, b):
        y = activations.linear(x, w, bias)
        g, = torch.autograd.grad(y.sum(), x, create_graph=True)
        assert torch.equal(g, torch.ones(40, 16, device=DEV) @ w.detach())
        with pytest.raises(RuntimeError, match="differentiate"):
            (y.sum() + g.square().sum()).backward()


def test_a_penalty_on_the_weight_gradient_raises_where_the_input_has_a_gradient():
    """d(sum y)/dW = 1^T x depends on x: an error for an x with a gradient, a
    constant for data."""
    w = weight(16, 64)
    x = activation(40, 64, torch.float32)
    for leaf in (x.clone().requires_grad_(), x):
        y = activations.linear(leaf, w)
        g, = torch.autograd.grad(y.sum(), w, create_graph=True)
        assert torch.equal(g, activations.weight_gradient(torch.ones(40, 16, device=DEV), activations.pack(x)))
        if leaf.requires_grad:
            with pytest.raises(RuntimeError, match="differentiate"):
                g.square().sum().backward()
        else:
            assert not g.requires_grad


def test_a_recorded_bias_gradient_of_a_constant_cotangent_is_a_constant():
    x, w = activation(40, 64, torch.float32).requires_grad_(), weight(16, 64)
    b = torch.zeros(16, device=DEV, requires_grad=True)
    g, = torch.autograd.grad(activations.linear(x, w, b).sum(), b, create_graph=True)
    assert torch.equal(g, torch.full((16,), 40.0, device=DEV)) and not g.requires_grad
    loss = activations.linear(x, w, b).square().sum()  # a cotangent that depends on the bias
    g, = torch.autograd.grad(loss, b, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate"):
        g.sum().backward()


@pytest.mark.parametrize("approximate", ["none", "tanh"])
def test_a_penalty_on_the_gradient_of_gelu_raises(approximate):
    x = activation(40, 64, torch.float32).requires_grad_()
    for pack_output in (False, True):
        y = activations.gelu(x, approximate=approximate, pack_output=pack_output)
        y = y[0] if pack_output else y
        g, = torch.autograd.grad(y.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate"):
            (y.sum() + g.square().sum()).backward()


def test_recorded_gradients_are_the_plain_ones():
    x, w = activation(40, 64, torch.float32).requires_grad_(), weight(16, 64)
    b = torch.zeros(16, device=DEV, requires_grad=True)
    delta = cotangent(40, 16, torch.float32)
    y = activations.linear(x, w, b)
    plain = torch.autograd.grad(y, [x, w, b], delta, retain_graph=True)
    recorded = torch.autograd.grad(y, [x, w, b], delta, create_graph=True)
    for p, r in zip(plain, recorded):
        assert torch.equal(p, r) and not p.requires_grad


@pytest.mark.parametrize("dtype", DTYPES)
def test_operators_on_a_cotangent_with_a_gradient(dtype):
    """Their results can be used, and raise once something differentiates
    through them: they depend on the cotangent."""
    delta = cotangent(40, 64, dtype)
    packed = activations.pack(activation(40, 64, dtype))
    for call in (activations.weight_gradient, activations.gelu_backward):
        got = call(delta.clone().requires_grad_(), packed)
        assert torch.equal(got, call(delta, packed))
        with pytest.raises(RuntimeError, match="differentiate"):
            got.float().sum().backward()
        with torch.no_grad():
            assert not call(delta.clone().requires_grad_(), packed).requires_grad


# -------------------------------------------------- forward mode and tracing

def test_tangents_are_refused():
    """No operator carries a forward-mode tangent; none drops it."""
    x, delta = activation(8, 64, torch.float32), cotangent(8, 64, torch.float32)
    w = weight(16, 64)
    packed = activations.pack(x)
    calls = (activations.gelu, lambda t: activations.gelu(t, approximate="tanh", pack_output=True),
             lambda t: activations.weight_gradient(t, packed), lambda t: activations.gelu_backward(t, packed),
             lambda t: activations.linear(t, w), lambda t: activations.linear(x, w, t[0, :16]))
    with torch.autograd.forward_ad.dual_level():
        for leaf in (False, True):
            dual = torch.autograd.forward_ad.make_dual(x.clone().requires_grad_(leaf), torch.ones_like(x))
            for call in calls:
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(dual)
        with pytest.raises(RuntimeError, match="forward-mode"):
            activations.linear(x, torch.autograd.forward_ad.make_dual(w, torch.ones_like(w)))
        # with a weight that takes no gradient, linear is torch's own layer
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        out = torch.autograd.forward_ad.unpack_dual(activations.linear(dual, w.detach()))
        assert torch.equal(out.tangent, torch.nn.functional.linear(torch.ones_like(x), w.detach()))


def test_tracing_is_refused():
    """A trace would record the allocation of an output and not the kernel that
    fills it."""
    make_fx = torch.fx.experimental.proxy_tensor.make_fx
    x, w = activation(8, 64, torch.float32), weight(16, 64)
    packed = activations.pack(x)
    calls = (activations.gelu, lambda t: activations.pack(t).values, lambda t: activations.pack_input(t).values,
             lambda t: activations.unpack(packed) + t, lambda t: activations.weight_gradient(t, packed),
             lambda t: activations.gelu_backward(t, packed), lambda t: activations.linear(t, w))
    for call in calls:
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(call, x, check_trace=False)
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(lambda t: call(t))(x)
    frozen = w.detach()
    traced = torch.jit.trace(lambda t: activations.linear(t, frozen), x)  # torch's own layer
    assert torch.equal(traced(2 * x), torch.nn.functional.linear(2 * x, frozen))


# ------------------------------------------------------------ in-place changes

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(48,), (5, 48), (2, 5, 48), (2, 3, 5, 48), (0, 48)])
def test_outputs_can_be_changed_in_place(shape, dtype):
    """relu_, residual additions and scalings of an output, as after nn.Linear."""
    base = torch.randn(*shape, generator=torch.Generator().manual_seed(3)).to(dtype).to(DEV)
    w = weight(32, 48)
    b = torch.zeros(32, device=DEV, requires_grad=True)
    for bias in (None, b):
        x = base.clone().requires_grad_()
        want = torch.nn.functional.linear(x, w.to(dtype), None if bias is None else bias.to(dtype)).detach()
        y = activations.linear(x, w, bias)
        y += 1
        y.relu_()
        assert torch.equal(y, (want + 1).relu())
        y.sum().backward()
        kept = (want + 1 > 0).to(dtype)
        assert torch.equal(x.grad, (kept.reshape(-1, 32) @ w.detach().to(dtype)).view(shape))
        assert torch.equal(w.grad, activations.weight_gradient(kept, activations.pack(base)))
        w.grad = None
    for pack_output in (False, True):
        x = base.clone().requires_grad_()
        y = activations.gelu(x, pack_output=pack_output)
        y = y[0] if pack_output else y
        want = y.detach().clone()
        y.mul_(2)
        y += 1
        assert torch.equal(y, want * 2 + 1)
        y.sum().backward()
        assert torch.equal(x.grad, activations.gelu_backward(torch.full_like(base, 2), activations.pack(base)))


def test_inplace_modules_after_a_packed_layer():
    layer = activations.PackedLinear(48, 32).to(DEV)
    plain = torch.nn.Linear(48, 32).to(DEV)
    plain.load_state_dict(layer.state_dict())
    x = activation(10, 48, torch.float32).view(2, 5, 48)
    outs = [torch.nn.Sequential(m, torch.nn.ReLU(inplace=True))(x) for m in (layer, plain)]
    assert torch.equal(*outs)
    outs[0].sum().backward()
    outs[1].sum().backward()
    assert torch.equal(layer.bias.grad, plain.bias.grad)


# --------------------------------------------------------------------- memory

def test_backward_of_gelu_allocates_its_result_alone():
    """No zero gradients for the output's checkpoint and sums, which take
    none."""
    x = activation(4096, 4096, torch.bfloat16).requires_grad_()
    delta = cotangent(4096, 4096, torch.bfloat16)
    for stats in (False, True):
        y, packed = activations.gelu(x, pack_output=True, stats=stats)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        dx, = torch.autograd.grad(y, x, delta)
        used = torch.cuda.max_memory_allocated() - before
        # dx and allocation granularity; the checkpoint would add half of dx again
        assert used <= dx.numel() * dx.element_size() + (1 << 20)
        del y, packed, dx


def test_a_gradient_that_nothing_gives():
    """A cotangent that is left undefined behind an output stays so, as with
    torch's own layers."""
    class Nothing(torch.autograd.Function):
        @staticmethod
        def forward(ctx, y):
            return y.clone()

        @staticmethod
        def backward(ctx, delta):
            return None

    w = weight(32, 48)
    b = torch.zeros(32, device=DEV, requires_grad=True)
    calls = (lambda x: activations.linear(x, w, b), activations.gelu,
             lambda x: activations.gelu(x, pack_output=True, stats=True)[0])
    for call in calls:
        x = activation(10, 48, torch.float32).requires_grad_()
        assert torch.autograd.grad(Nothing.apply(call(x)).sum(), x, allow_unused=True) == (None,)
        Nothing.apply(call(x)).sum().backward()
        assert w.grad is None and b.grad is None


# ------------------------------------------------- layers that share an input

def shared_exact(deltas, ws, dtype):
    """(sum of delta W, sum of |delta| |W|) in FP64."""
    pairs = [(d.double(), w.detach().to(dtype).double()) for d, w in zip(deltas, ws)]
    return sum(d @ w for d, w in pairs), sum(d.abs() @ w.abs() for d, w in pairs)


def check_shared(got, deltas, ws, dtype, out_dtype=None):
    """FP32 sums of 3 x 96 terms in any order (library products may truncate: a
    step of 2^-23 a term, and the joins), then half a step of the result's
    type."""
    want, size = shared_exact(deltas, ws, dtype)
    bound = 300 * 2.0 ** -23 * size + torch.finfo(out_dtype or dtype).eps / 2 * want.abs()
    assert got.dtype == (out_dtype or dtype)
    assert bool(((got.double().reshape(want.shape) - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(500, 80), (5, 100, 80), (80,), (0, 80)])
def test_input_gradients_of_layers_that_share_a_checkpoint_are_summed_in_fp32(shape, dtype):
    ws = [weight(96, 80, seed) for seed in range(3)]
    rows = 1 if len(shape) == 1 else torch.Size(shape[:-1]).numel()
    base = activation(max(rows, 1), 80, dtype)[:rows].view(shape)
    deltas = [cotangent(max(rows, 1), 96, dtype, seed=k)[:rows] for k in range(3)]
    shaped = [d.view(*shape[:-1], 96) for d in deltas]
    x = base.clone().requires_grad_()
    packed = activations.pack(x)
    outs = [activations.linear(x, w, packed=packed) for w in ws]
    first = torch.autograd.grad(outs, [x, *ws], shaped, retain_graph=True)
    check_shared(first[0], deltas, ws, dtype)
    for w, dw, d in zip(ws, first[1:], shaped):
        assert torch.equal(dw, activations.weight_gradient(d, activations.pack(base)))
    # again, one layer alone, and through x's own graph
    assert torch.equal(torch.autograd.grad(outs, x, shaped, retain_graph=True)[0], first[0])
    check_shared(torch.autograd.grad(outs[1], x, shaped[1])[0], deltas[1:2], ws[1:2], dtype)
    h = x * 2
    packed = activations.pack(h)
    got, = torch.autograd.grad([activations.linear(h, w, packed=packed) for w in ws], h, shaped)
    assert torch.equal(got, first[0])
    # a checkpoint kept over several passes
    packed = activations.pack(x)
    for _ in range(2):
        got, = torch.autograd.grad([activations.linear(x, w, packed=packed) for w in ws], x, shaped)
        assert torch.equal(got, first[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_shared_input_gradients_under_autocast(dtype):
    """FP32 inputs: the sum is not rounded to the layers' type at all."""
    ws = [weight(96, 80, seed) for seed in range(3)]
    x = activation(500, 80, torch.float32).requires_grad_()
    deltas = [cotangent(500, 96, dtype, seed=k) for k in range(3)]
    with torch.autocast("cuda", dtype=dtype):
        packed = activations.pack_input(x, stats=True)
        outs = [activations.linear(x, w, packed=packed) for w in ws]
    got, = torch.autograd.grad(outs, x, deltas)
    check_shared(got, deltas, ws, dtype, torch.float32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,d_in,d_out", [(7, 33, 5), (257, 129, 1), (1, 1, 1), (40, 24, 0), (64, 8, 1000)])
def test_shared_input_gradients_of_odd_sizes_and_strides(rows, d_in, d_out, dtype):
    """Weights and cotangents of any strides (a transposed weight, a broadcast
    cotangent), sizes without alignment, a layer without outputs."""
    x = activation(rows, d_in, dtype).requires_grad_()
    base = weight(d_in, d_out, 1).detach()
    ws = [base.t().requires_grad_(), weight(d_out, d_in, 2)]
    deltas = [cotangent(rows, d_out, dtype), cotangent(rows, 1, dtype).expand(rows, d_out)]
    packed = activations.pack(x)
    outs = [activations.linear(x, w, packed=packed) for w in ws]
    got = torch.autograd.grad(outs, [x, *ws], deltas)
    want, size = shared_exact(deltas, ws, dtype)
    bound = (2 * d_out + 20) * 2.0 ** -23 * size + torch.finfo(dtype).eps / 2 * want.abs()
    assert bool(((got[0].double() - want).abs() <= bound + torch.finfo(dtype).smallest_normal).all())
    for dw, d in zip(got[1:], deltas):
        assert torch.equal(dw, activations.weight_gradient(d, packed))


def test_a_checkpoint_of_another_tensor_sends_no_gradient_there():
    """The gradient goes to the x that a layer is called with, whatever its
    checkpoint was packed from."""
    dtype = torch.bfloat16
    w, delta = weight(96, 80), cotangent(500, 96, dtype)
    base = activation(500, 80, dtype)
    other = base.clone().requires_grad_()
    packed = activations.pack(other)
    for make in (lambda: base.clone().requires_grad_(), lambda: (base / 2).requires_grad_() * 2):
        x = make()
        got, elsewhere = torch.autograd.grad(activations.linear(x, w, packed=packed), [x, other], delta,
                                             allow_unused=True)
        check_shared(got, [delta], [w], dtype)
        assert elsewhere is None
    y = activations.linear(base, w, packed=packed)  # data
    assert torch.autograd.grad(y, [w, other], delta, allow_unused=True)[1] is None
    # an input changed in place since: its gradient is scaled on its way
    h = other * 1
    packed = activations.pack(h)
    h *= 0.5
    got, = torch.autograd.grad(activations.linear(h, w, packed=packed), other, delta)
    check_shared(got * 2, [delta], [w], dtype)
    # packed where nothing is recorded
    with torch.no_grad():
        packed = activations.pack(other)
    check_shared(torch.autograd.grad(activations.linear(other, w, packed=packed), other, delta)[0], [delta], [w], dtype)


def test_checkpoints_of_graph_tensors_can_be_copied():
    import copy
    import pickle
    x = activation(20, 80, torch.bfloat16).requires_grad_()
    packed = activations.pack(x * 2, stats=True)
    for again in (copy.copy(packed), copy.deepcopy(packed), pickle.loads(pickle.dumps(packed))):
        assert torch.equal(again.values, packed.values) and torch.equal(again.exponents, packed.exponents)
        assert torch.equal(again.sums, packed.sums) and again.shape == packed.shape and again.dtype == packed.dtype
        assert torch.equal(again.unpack(), packed.unpack())


def test_a_penalty_on_a_shared_input_gradient_raises():
    x, w = activation(40, 80, torch.bfloat16).requires_grad_(), weight(96, 80)
    packed = activations.pack(x)
    y = activations.linear(x, w, packed=packed)
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate"):
        (y.sum() + g.square().sum()).backward()


CAPTURED = """
import torch
from sandmuon_b200 import activations
g = torch.Generator(device="cuda").manual_seed(1)
x = torch.randn(300, 80, generator=g, device="cuda").bfloat16().requires_grad_()
ws = [torch.randn(96, 80, generator=g, device="cuda").mul_(.05).requires_grad_() for _ in range(2)]
d = torch.randn(300, 96, generator=g, device="cuda").bfloat16()

def work(packed=None):
    packed = packed or activations.pack(x)
    outs = [activations.linear(x, w, packed=packed) for w in ws]
    y, py = activations.gelu(x, pack_output=True)
    return torch.autograd.grad([*outs, y], [x, *ws], [d, d, x.detach()])

want = work()
kept = activations.pack(x)  # on another stream than the capture's
[activations.linear(x, w, packed=kept) for w in ws]
for packed in (None, kept):
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work(packed)
    for t in got:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
print("ok")
"""


def test_a_captured_backward_with_a_checkpoint_from_outside():
    """In a process of its own, which a failed capture would leave unusable.
    (An eager graph of the same leaves must not live meanwhile, with torch's own
    layers neither.)"""
    import subprocess
    import sys
    from pathlib import Path
    out = subprocess.run([sys.executable, "-c", CAPTURED], capture_output=True, text=True, timeout=300,
                         cwd=Path(__file__).resolve().parents[1])
    assert out.returncode == 0 and out.stdout.strip().endswith("ok"), out.stderr[-2000:]


def test_a_kept_checkpoint_keeps_no_graph_alive():
    x = activation(1024, 1024, torch.bfloat16).requires_grad_()
    w = weight(96, 1024)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    h = x.exp().exp()  # keeps two results for its backward
    packed = activations.pack(h)
    outs = [activations.linear(h, w, packed=packed) for _ in range(2)]
    assert torch.autograd.grad(outs, x, [torch.ones_like(y) for y in outs], retain_graph=True)[0].shape == x.shape
    del h, outs
    assert torch.cuda.memory_allocated() - before <= packed.nbytes + 4096
