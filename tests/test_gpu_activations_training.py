"""The 8-bit checkpoint operators as a training loop uses them: linear layers
sharing a checkpoint, autocast, captured graphs, other streams, the optimizer's
hooks on packed layers, and the GPT-2 workload with checkpoints="int8".

Tolerances: a layer's weight gradient is held to delta^T x^ with the bounds of
the operator's own tests; what torch computes (outputs, input gradients) to the
same torch products, rounded alike.  Statistics: 1e-5 relative, as for the
hooks of plain layers."""
import numpy as np
import pytest
import torch

from oracle import activation_oracle as orc
from sandmuon_b200 import DiagonalWeightedPE, RankOneAWeightedPE, _lib, activations
from sandmuon_b200.workloads import GPT2, gpt2_matrix_filter, gpt2_train_step
from test_gpu_activations import DTYPES, activation, check_sums, check_weight_gradient, cotangent, f64, name

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


# ------------------------------------------------ sizes that fill the machine

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,d_in,d_out", [
    (5000, 2304, 2304),    # 81 tiles: whole waves, chains that are cut, a remainder
    (1100, 2048, 1280),    # 40 tiles: stretches across tile borders
    (20000, 64, 300),      # two tiles, a long sum in many parts
    (260, 5200, 10),       # one row of tiles
    (130, 8, 5000),        # one column of tiles
])
def test_weight_gradient_of_many_tiles(rows, d_in, d_out, dtype):
    x, delta = activation(rows, d_in, dtype), cotangent(rows, d_out, dtype)
    packed = activations.pack(x)
    got = activations.weight_gradient(delta, packed)
    d, hat = delta.double(), packed.unpack(torch.float32).double()
    want, size = d.t() @ hat, d.abs().t() @ hat.abs()
    assert ((got.double() - want).abs() <= (rows + 64) * 3 * 2.0 ** -23 * size).all()
    # chains of 128 steps, joined by rounded additions
    assert float((got.double() - want).norm() / want.norm()) <= 4e-6
    for out_dtype in (torch.bfloat16, torch.float16):
        low = activations.weight_gradient(delta, packed, dtype=out_dtype)
        assert torch.equal(low, got.to(out_dtype))
    assert _lib.device_status(DEV) == 0


# --------------------------------------------------------------------- linear

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,d_out", [((1, 24), 8), ((5, 7, 33), 70), ((130, 264), 513), ((0, 24), 8), ((48,), 5)])
def test_linear_and_its_gradients(shape, d_out, dtype):
    g = torch.Generator().manual_seed(len(shape) + d_out)
    x = torch.randn(*shape, generator=g).to(dtype).to(DEV).requires_grad_()
    w = (torch.randn(d_out, shape[-1], generator=g) * .05).to(DEV).requires_grad_()
    b = torch.randn(d_out, generator=g).to(DEV).requires_grad_()
    delta = cotangent(max(1, x[..., 0].numel()), d_out, dtype)[:x[..., 0].numel()].view(*shape[:-1], d_out)
    y = activations.linear(x, w, b)
    assert torch.equal(y, torch.nn.functional.linear(x, w.to(dtype), b.to(dtype)))
    dx, dw, db = torch.autograd.grad(y, [x, w, b], delta)
    assert dx.shape == x.shape and dx.dtype == dtype and dw.dtype == db.dtype == torch.float32
    flat = delta.reshape(-1, d_out)
    assert torch.equal(dx.reshape(-1, shape[-1]), torch.mm(flat, w.detach().to(dtype)))
    packed = activations.pack(x)
    assert torch.equal(dw, activations.weight_gradient(delta, packed))
    check_weight_gradient(dw, flat, activations.pack(x.detach().reshape(-1, shape[-1])))
    n = flat.shape[0] + 8
    assert (np.abs(f64(db) - f64(flat).sum(0)) <= n * 2.0 ** -24 * np.abs(f64(flat)).sum(0)).all()


def test_linear_shares_a_checkpoint_and_takes_any_needed_gradients():
    x = activation(200, 96, torch.bfloat16).requires_grad_()
    ws = [torch.randn(n, 96, device=DEV).mul_(.05).requires_grad_() for n in (64, 40, 8)]
    packed = activations.pack(x, stats=True)
    check_sums(packed.sums, x)
    outs = [activations.linear(x, w, packed=packed) for w in ws]
    deltas = [cotangent(200, w.shape[0], torch.bfloat16) for w in ws]
    grads = torch.autograd.grad(outs, [x, *ws], deltas)
    for delta, dw in zip(deltas, grads[1:]):
        check_weight_gradient(dw, delta, packed)
    want = sum(d.double() @ w.detach().to(torch.bfloat16).double() for d, w in zip(deltas, ws))
    # three rounded products, two rounded sums
    size = sum((d.double().abs() @ w.detach().to(torch.bfloat16).double().abs()) for d, w in zip(deltas, ws))
    assert ((grads[0].double() - want).abs() <= 5 * 2.0 ** -8 * size).all()
    w = ws[0]
    only_w, = torch.autograd.grad(activations.linear(x.detach(), w), w, deltas[0])
    assert torch.equal(only_w, grads[1])
    frozen = activations.linear(x, w.detach())
    only_x, = torch.autograd.grad(frozen, x, deltas[0])
    assert torch.equal(only_x, torch.mm(deltas[0], w.detach().to(torch.bfloat16)))
    with torch.no_grad():
        assert not activations.linear(x, w).requires_grad
    with pytest.raises(ValueError, match="does not fit"):
        activations.linear(x[:100], w, packed=packed)
    with pytest.raises(TypeError, match="float16"):
        activations.linear(x.half(), w, packed=packed)
    with pytest.raises(TypeError):
        activations.linear(x.double(), w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_linear_under_autocast(dtype):
    """FP32 inputs and weights: the layer computes in autocast's type, the
    checkpoint is of the FP32 input (of its FP16 values for FP16)."""
    x = activation(150, 64, torch.float32).requires_grad_()
    layer = activations.PackedLinear(64, 48).to(DEV)
    with torch.autocast("cuda", dtype=dtype):
        y = layer(x)
        want = torch.nn.functional.linear(x, layer.weight, layer.bias)
    assert y.dtype == dtype and torch.equal(y, want)
    delta = cotangent(150, 48, dtype)
    y.backward(delta)
    assert x.grad.dtype == layer.weight.grad.dtype == torch.float32
    source = x.detach() if dtype == torch.bfloat16 else x.detach().half()
    check_weight_gradient(layer.weight.grad, delta, activations.pack(source))


def test_linear_holds_an_eighth_of_fp32_memory():
    """Between forward and backward a packed layer holds 1 + 1/32 bytes per
    input element instead of four."""
    x = torch.randn(4096, 2048, device=DEV)
    layers = [activations.PackedLinear(2048, 2048, bias=False).to(DEV) for _ in range(4)]
    torch.cuda.synchronize()

    def held(build):
        before = torch.cuda.memory_allocated()
        keep = build()
        return torch.cuda.memory_allocated() - before, keep

    def chain(step):
        h = x
        for layer in layers:
            h = step(layer, h)
        return h

    packed, out = held(lambda: chain(lambda layer, h: layer(h)))
    del out
    plain, out = held(lambda: chain(lambda layer, h: torch.nn.functional.linear(h, layer.weight)))
    n = x.numel()
    # the last output stays in both; plain holds three FP32 inputs besides x
    assert plain >= 4 * n * 4 and packed <= 4 * n + 4 * n * 33 / 32 + (1 << 20)


def test_in_place_change_of_a_saved_weight_is_noticed():
    x = activation(40, 32, torch.float32)
    w = torch.randn(16, 32, device=DEV).requires_grad_()
    y = activations.linear(x, w)
    with torch.no_grad():
        w.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


# ---------------------------------------------------------- streams and graphs

def test_captured_graphs_replay_with_new_inputs_and_share_nothing():
    """Two graphs captured one after the other on one stream, replayed at the
    same time on two: each owns its workspaces."""
    cases = [(3000, 264, 520), (2500, 136, 260)]
    state = []
    capture = torch.cuda.Stream()
    for k, (rows, d_in, d_out) in enumerate(cases):
        s = dict(x=activation(rows, d_in, torch.bfloat16, seed=k), d=cotangent(rows, d_out, torch.bfloat16, seed=k),
                 e=cotangent(rows, d_in, torch.bfloat16, seed=k + 7))

        def work(s=s):
            leaf = s["x"].detach().requires_grad_()
            packed = activations.pack(s["x"], stats=True)
            y, py = activations.gelu(leaf, pack_output=True, stats=True)
            dx, = torch.autograd.grad(y, leaf, s["e"])
            return [activations.weight_gradient(s["d"], packed), packed.sums, packed.unpack(),
                    activations.weight_gradient(s["d"], py), py.sums, dx]

        capture.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(capture):
            work()
            capture.synchronize()
            s["graph"] = torch.cuda.CUDAGraph()
            with torch.cuda.graph(s["graph"], stream=capture):
                s["out"] = work()
        s["work"] = work
        state.append(s)
    torch.cuda.synchronize()
    for s, (rows, d_in, d_out) in zip(state, cases):
        s["x"].copy_(activation(rows, d_in, torch.bfloat16, seed=11))
        s["d"].copy_(cotangent(rows, d_out, torch.bfloat16, seed=12))
        s["want"] = s["work"]()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for st, s in zip(streams, state):
            with torch.cuda.stream(st):
                s["graph"].replay()
    torch.cuda.synchronize()
    for s in state:
        for got, want in zip(s["out"], s["want"]):
            assert torch.equal(got, want)
    assert _lib.device_status(DEV) == 0


def test_calls_on_another_stream():
    x, d = activation(4000, 520, torch.float32), cotangent(4000, 260, torch.float32)
    want = activations.weight_gradient(d, activations.pack(x))
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for st in streams:
        with torch.cuda.stream(st):
            got.append(activations.weight_gradient(d, activations.pack(x)))
    torch.cuda.synchronize()
    for g in got:
        assert torch.equal(g, want)


# ------------------------------------------------------------------- optimizer

@pytest.mark.parametrize("rank_one", [True, False])
def test_hooks_take_packed_statistics(rank_one):
    """An optimizer over packed layers accumulates the same statistics and
    counts as over plain ones, and steps."""
    torch.manual_seed(1)
    plain = torch.nn.Sequential(torch.nn.Linear(64, 96), torch.nn.GELU(), torch.nn.Linear(96, 32)).to(DEV)
    packed = torch.nn.Sequential(activations.PackedLinear.from_linear(plain[0]), torch.nn.GELU(),
                                 activations.PackedLinear.from_linear(plain[2]))
    make = RankOneAWeightedPE if rank_one else DiagonalWeightedPE
    states = []
    before = [p.detach().clone() for p in plain.parameters()]
    for model in (plain, packed):
        opt = make(model, lr=1e-2)
        for k in range(3):
            x = activation(50 + k, 64, torch.float32, seed=k)
            (model(x).square().sum() / 3).backward()
        keys = ("a_sum", "a_first_sum", "b_sum") if rank_one else ("a_sum", "b_sum")
        states.append([{k: opt.state[p][k].clone() for k in keys} | {k: opt.state[p][k] for k in ("a_count", "b_count")}
                       for p in opt.named_matrices.values()])
        with torch.no_grad():
            model.eval()
            model(x)
            model.train()
        opt.step()
        for key in ("a_count", "b_count"):
            assert all(opt.state[p][key] == 0 for p in opt.named_matrices.values())
        assert all(torch.isfinite(p).all() for p in model.parameters())
        opt.close()
        with torch.no_grad():
            for p, b in zip(plain.parameters(), before):
                p.copy_(b)
                p.grad = None
    for a, b in zip(*states):
        assert a["a_count"] == b["a_count"] == 153 and a["b_count"] == b["b_count"]
        for key in a:
            if torch.is_tensor(a[key]):
                assert float((a[key] - b[key]).norm() / a[key].norm()) < 1e-5, key


def test_gpt2_workload_with_int8_checkpoints():
    """The training path: every block matrix's gradient is delta^T x^ of what
    the layer saw, q/k/v share one checkpoint, statistics equal the tensors'
    own sums, a step runs, and less memory is held."""
    torch.manual_seed(3)
    model = GPT2(layers=2, width=128, heads=4, vocab=512, context=64, checkpoints="int8").to(DEV)
    opt = RankOneAWeightedPE(model, lr=1e-2, module_filter=gpt2_matrix_filter)
    seen_in, seen_packed, seen_out, probes = {}, {}, {}, []
    for key, module in model.named_modules():
        if gpt2_matrix_filter(key, module):
            def fwd(mod, args, kwargs, out, key=key):
                seen_in[key] = args[0].detach().reshape(-1, args[0].shape[-1]).clone()
                seen_packed[key] = args[1] if len(args) > 1 else kwargs["packed"]
                out.register_hook(lambda g, key=key: seen_out.__setitem__(key, g.detach().reshape(-1, g.shape[-1]).clone()))
            probes.append(module.register_forward_hook(fwd, with_kwargs=True))
    gen = torch.Generator(device=DEV).manual_seed(4)
    idx = torch.randint(0, 512, (4, 64), generator=gen, device=DEV)
    tgt = torch.randint(0, 512, (4, 64), generator=gen, device=DEV)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        logits = model(idx)
        loss = torch.nn.functional.cross_entropy(logits.view(-1, 512), tgt.view(-1))
    loss.backward()
    for p in probes:
        p.remove()
    params = dict(model.named_parameters())
    assert len(seen_in) == 12
    for key, x in seen_in.items():
        p = params[key + ".weight"]
        packed = seen_packed[key]
        values, codes, _ = orc.checkpoint(f64(x), name(x.dtype))
        np.testing.assert_array_equal(packed.values.cpu().numpy(), values)
        check_weight_gradient(p.grad, seen_out[key], packed)
        st = opt.state[p]
        if opt.a_sources[id(p)] is p:
            assert st["a_count"] == x.shape[0]
            want = x.double().square().sum(0)
            assert float((st["a_sum"].double() - want).norm() / want.norm()) < 1e-5
            want = x.double().sum(0)
            assert float((st["a_first_sum"].double() - want).norm() / want.norm()) < 1e-5
        want = seen_out[key].double().square().sum(0)
        assert float((st["b_sum"].double() - want).norm() / want.norm()) < 1e-5
    for i in range(2):
        q = f"transformer.h.{i}.attn."
        assert seen_packed[q + "q_proj"] is seen_packed[q + "k_proj"] is seen_packed[q + "v_proj"]
    opt.step()
    opt.zero_grad(set_to_none=True)
    total = gpt2_train_step(model, opt, [idx, idx], [tgt, tgt])
    assert torch.isfinite(total) and _lib.device_status(DEV) == 0
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        model.eval()
        quiet = model(idx)
    assert torch.isfinite(quiet.float()).all()
    opt.close()


def test_gpt2_memory():
    def peak(checkpoints):
        torch.manual_seed(3)
        model = GPT2(layers=6, width=256, heads=4, vocab=256, context=512, checkpoints=checkpoints).to(DEV)
        idx = torch.zeros(16, 512, dtype=torch.long, device=DEV)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            out = model(idx)
        return torch.cuda.memory_allocated() - before - out.numel() * out.element_size(), out

    plain, out = peak(None)
    del out
    packed, out = peak("int8")
    assert packed < 0.75 * plain


# ------------------------------------------------------------------ edge cases

@pytest.mark.parametrize("dtype", DTYPES)
def test_weight_gradient_of_one_row_of_a_wider_tensor(dtype):
    """A single row keeps whatever row stride its tensor had."""
    base = cotangent(4, 21, dtype)
    packed = activations.pack(activation(1, 50, dtype))
    for delta in (base[:1, :16], base[0, :16], base[:1]):
        check_weight_gradient(activations.weight_gradient(delta, packed), delta.reshape(1, -1), packed)


def test_offsets_past_32_bits():
    """More than 2^31 elements: the last rows are packed, unpacked, summed and
    multiplied like a small tensor of their own."""
    rows, cols, tail = 70000, 32768, 96
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=DEV)
    x[-tail:] = activation(tail, cols, torch.bfloat16)
    last = x[-tail:].clone()
    packed = activations.pack(x, stats=True)
    small = activations.pack(last, stats=True)
    assert torch.equal(packed.values[-tail:], small.values) and torch.equal(packed.exponents[-tail:], small.exponents)
    assert float((packed.sums - small.sums).norm() / small.sums.norm()) < 1e-6
    delta = torch.zeros(rows, 40, dtype=torch.bfloat16, device=DEV)
    delta[-tail:] = cotangent(tail, 40, torch.bfloat16)
    dw, want = activations.weight_gradient(delta, packed), activations.weight_gradient(delta[-tail:], small)
    assert float((dw - want).norm() / want.norm()) < 2e-6
    del delta
    out = activations.unpack(packed)
    assert torch.equal(out[-tail:], small.unpack()) and not out[:1000].any()
    del out
    y, py = activations.gelu(x, pack_output=True)
    assert torch.equal(y[-tail:], activations.gelu(last)) and not y[:1000].any()
    del x
    dx = activations.gelu_backward(y, packed)
    assert torch.equal(dx[-tail:], activations.gelu_backward(y[-tail:], small))


def test_first_call_inside_a_capture():
    """A process whose first operator call is captured: nothing the library
    sets up on first use breaks the capture."""
    import subprocess
    import sys
    from pathlib import Path
    code = """
import torch
from sandmuon_b200 import activations
x = torch.randn(3000, 300, device="cuda").bfloat16()
d = torch.randn(3000, 200, device="cuda").bfloat16()
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    packed = activations.pack(x, stats=True)
    dw = activations.weight_gradient(d, packed)
    dw32 = activations.weight_gradient(d.float(), packed)
    y, py = activations.gelu(x, pack_output=True, stats=True)
    dx = activations.gelu_backward(y, packed)
g.replay()
torch.cuda.synchronize()
assert torch.equal(dw, activations.weight_gradient(d, activations.pack(x)))
assert torch.equal(dx, activations.gelu_backward(y, activations.pack(x)))
print("ok")
"""
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                         cwd=Path(__file__).resolve().parents[1])
    assert out.returncode == 0 and out.stdout.strip().endswith("ok"), out.stderr[-2000:]


def test_gradients_can_be_recorded_but_not_differentiated():
    x = activation(40, 64, torch.float32).requires_grad_()
    w = torch.randn(16, 64, device=DEV).requires_grad_()
    for y, leaves in ((activations.linear(x, w).square().sum(), [x, w]), (activations.gelu(x).square().sum(), [x])):
        plain = torch.autograd.grad(y, leaves, retain_graph=True)
        recorded = torch.autograd.grad(y, leaves, create_graph=True)
        for a, b in zip(plain, recorded):
            assert torch.equal(a, b)
        with pytest.raises(RuntimeError, match="differentiate"):
            torch.autograd.grad(recorded[0].sum(), leaves[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_weight_gradient_of_the_largest_and_smallest_values(dtype):
    """Checkpoints at both ends of their exponents, next to ordinary ones."""
    g = torch.Generator().manual_seed(8)
    x = torch.randn(300, 160, generator=g).double()
    top = 6e4 if dtype == torch.float16 else 3e38
    x[:, :32] *= top / x[:, :32].abs().max()
    x[:, 32:64] *= 5000 if dtype == torch.float16 else 1e30
    x[:, 64:96] *= torch.finfo(dtype).smallest_normal * 64
    x[7, 96:128] = 0
    x = x.to(dtype).to(DEV)
    delta = (torch.randn(300, 70, generator=g) * (1e-3 if dtype == torch.float16 else 1e-6)).to(dtype).to(DEV)
    packed = activations.pack(x)
    got = activations.weight_gradient(delta, packed)
    d, hat = delta.double(), packed.unpack(torch.float32).double()
    want, size = d.t() @ hat, d.abs().t() @ hat.abs()
    # a subnormal product or plane of the cotangent is off by at most 2^-133 a term
    assert ((got.double() - want).abs() <= 400 * 3 * 2.0 ** -23 * size + 900 * 2.0 ** -133 * (1 + hat.abs().max())).all()
    assert float(((got.double() - want) / size.clamp_min(1e-300))[:, :64].abs().max()) < 1e-5
    assert float(((got.double() - want) / size.clamp_min(1e-300))[:, 96:].abs().max()) < 1e-5


@pytest.mark.parametrize("dtype", DTYPES)
def test_weight_gradient_repeats_bit_for_bit_under_load(dtype):
    """Back-to-back calls over two sets of inputs that fill every SM: the sums
    run in a fixed order, so each call returns the same bits.  (A k-block that
    is read before it is complete, or after its slot was given back, shows
    here; it took about one k-block in a million.)"""
    rows, d_in, d_out = 16384, 2048, 4096 if dtype == torch.float32 else 8192
    sets = []
    for seed in (1, 2):
        g = torch.Generator(device=DEV).manual_seed(seed)
        x = torch.randn(rows, d_in, generator=g, device=DEV) * torch.exp(torch.randn(rows, 1, generator=g, device=DEV))
        delta = torch.randn(rows, d_out, generator=g, device=DEV) * 0.1
        packed, delta = activations.pack(x.to(dtype)), delta.to(dtype)
        sets.append((delta, packed, activations.weight_gradient(delta, packed)))
    del x
    wrong = torch.zeros((), dtype=torch.int64, device=DEV)
    for _ in range(60):
        for delta, packed, want in sets:
            wrong += (activations.weight_gradient(delta, packed) != want).sum()
    assert int(wrong) == 0
    assert _lib.device_status(DEV) == 0
