"""8-bit activation checkpoints without a GPU: refusals of the Python entry
points and of the C-ABI (each before any device work), the oracle's own
properties, and how the optimizer and the GPT-2 workload take packed layers."""
import ctypes

import numpy as np
import pytest
import torch
from torch import nn

from oracle import activation_oracle as orc
from sandmuon_b200 import RankOneAWeightedPE, _lib, activations
from sandmuon_b200.workloads import GPT2, gpt2_matrix_filter


def cpu_packed(rows=3, cols=40, dtype=torch.bfloat16, **change):
    parts = dict(values=torch.zeros(rows, 48, dtype=torch.int8), exponents=torch.zeros(rows, 4, dtype=torch.uint8),
                 shape=(rows, cols), dtype=dtype)
    parts.update(change)
    return activations.PackedActivation(**parts)


def test_layout_sizes():
    for cols, ld, lde in ((1, 16, 4), (16, 16, 4), (17, 32, 4), (128, 128, 4), (129, 144, 8), (768, 768, 24)):
        assert (activations.values_ld(cols), activations.exponents_ld(cols)) == (ld, lde)
        values, codes, _ = orc.checkpoint(np.ones((2, cols)), "float32")
        assert values.shape == (2, ld) and codes.shape == (2, lde)
    assert cpu_packed(shape=(1, 3, 40)).nbytes == 3 * 52


def test_oracle_rounds_within_half_a_step():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, 100)) * np.exp(rng.standard_normal((50, 100)) * 4)
    values, codes, hat = orc.checkpoint(x, "float32")
    step = np.repeat(np.ldexp(1.0, codes[:, :4].astype(int) - 127), 32, 1)[:, :100]
    assert (np.abs(x - hat) <= step / 2).all()
    top = np.abs(np.pad(x, ((0, 0), (0, 28))).reshape(50, 4, 32)).max(-1)
    e = codes[:, :4].astype(int) - 127
    assert (top <= 127 * np.ldexp(1.0, e)).all() and (top > 127 * np.ldexp(1.0, e - 1)).all()


@pytest.mark.parametrize("change,error", [
    (dict(shape=()), ValueError),
    (dict(dtype=torch.float64), TypeError),
    (dict(values=torch.zeros(3, 40, dtype=torch.int8)), ValueError),
    (dict(values=torch.zeros(3, 48, dtype=torch.uint8)), ValueError),
    (dict(values=torch.zeros(48, 3, dtype=torch.int8).t()), ValueError),
    (dict(exponents=torch.zeros(3, 2, dtype=torch.uint8)), ValueError),
    (dict(exponents=torch.zeros(3, 4, dtype=torch.int8)), ValueError),
    (dict(shape=(2, 40)), ValueError),
    (dict(sums=torch.zeros(2, 39)), ValueError),
    (dict(sums=torch.zeros(2, 40, dtype=torch.float64)), ValueError),
])
def test_packed_activation_refuses(change, error):
    with pytest.raises(error):
        cpu_packed(**change)


def test_cpu_tensors_fail_loudly(built_library):
    x = torch.randn(3, 40)
    for call in (lambda: activations.pack(x), lambda: activations.gelu(x), lambda: cpu_packed().unpack(),
                 lambda: activations.weight_gradient(x.bfloat16(), cpu_packed()),
                 lambda: activations.gelu_backward(x.bfloat16(), cpu_packed()),
                 lambda: activations.linear(x, torch.randn(5, 40)),
                 lambda: activations.PackedLinear(40, 5)(x)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_argument_checks(built_library):
    x = torch.randn(3, 40)
    scalar = torch.tensor(1.0)
    with pytest.raises(ValueError):
        activations.pack(scalar)
    with pytest.raises(ValueError):
        activations.gelu(scalar)
    with pytest.raises(ValueError, match="pack_output"):
        activations.gelu(x, stats=True)
    with pytest.raises(TypeError, match="float16"):
        activations.weight_gradient(x.half(), cpu_packed())
    with pytest.raises(TypeError, match="float16"):
        activations.unpack(cpu_packed(), torch.float16)
    with pytest.raises(ValueError, match="does not fit"):
        activations.weight_gradient(torch.randn(4, 7), cpu_packed())
    with pytest.raises(ValueError, match="does not fit"):
        activations.gelu_backward(torch.randn(3, 41), cpu_packed())
    with pytest.raises(ValueError, match="fit weight"):
        activations.linear(x, torch.randn(5, 41))
    with pytest.raises(ValueError, match="bias"):
        activations.linear(x, torch.randn(5, 40), torch.randn(4))
    with pytest.raises(ValueError, match="approximate"):
        activations._gelu_form("sigmoid")
    with pytest.raises(ValueError, match="checkpoints"):
        GPT2(layers=1, width=8, heads=2, vocab=16, context=4, checkpoints="int4")


def test_c_abi_refusals(built_library):
    """Bad arguments come back as SM_ERR_ARG before the library looks for a GPU."""
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096 + 64)
    base = (ctypes.addressof(buf) + 63) // 64 * 64
    arg = 1

    def pack(x=base, dtype=1, rows=2, cols=16, values=base, exponents=base):
        return lib.sm_activation_pack(x, dtype, rows, cols, 16, 1, values, exponents, 0, 0, 0, 0)

    for change in (dict(x=0), dict(dtype=3), dict(dtype=9), dict(rows=-1), dict(cols=-1), dict(rows=1 << 31),
                   dict(cols=1 << 31), dict(values=0), dict(exponents=0), dict(values=base + 8),
                   dict(exponents=base + 2)):
        assert pack(**change) == arg, change
        assert _lib.last_error()
    assert pack(rows=0) == 0 and pack(cols=0) == 0

    def unpack(values=base, exponents=base, rows=2, out=base, dtype=1):
        return lib.sm_activation_unpack(values, exponents, rows, 16, out, dtype, 0)

    for change in (dict(values=0), dict(exponents=base + 1), dict(rows=-1), dict(out=0), dict(dtype=3)):
        assert unpack(**change) == arg, change

    def gelu(x=base, dtype=1, form=0, y=base, in_v=base, in_e=base, out_v=base, out_e=base, sums=0):
        return lib.sm_gelu_forward(x, dtype, 2, 16, 16, 1, form, y, in_v, in_e, out_v, out_e, sums, 0, 0, 0)

    for change in (dict(x=0), dict(dtype=3), dict(form=2), dict(y=0), dict(in_v=base + 1), dict(in_e=0), dict(in_v=0),
                   dict(out_e=0), dict(out_v=0, out_e=0, sums=base)):
        assert gelu(**change) == arg, change

    def back(d=base, dtype=1, form=0, values=base, exponents=base, dx=base):
        return lib.sm_gelu_backward(d, dtype, 2, 16, 16, 1, values, exponents, form, dx, 0)

    for change in (dict(d=0), dict(dtype=3), dict(form=-1), dict(values=0), dict(exponents=0), dict(dx=0)):
        assert back(**change) == arg, change

    def wgrad(d=base, dtype=1, rows=2, d_out=8, values=base, exponents=base, d_in=16, out=base, out_dtype=0):
        return lib.sm_weight_gradient(d, dtype, rows, d_out, 8, 1, values, exponents, d_in, out, out_dtype, 0, 0, 0)

    for change in (dict(d=0), dict(dtype=3), dict(out_dtype=3), dict(rows=-1), dict(d_out=-1), dict(d_in=1 << 31),
                   dict(values=0), dict(exponents=base + 1), dict(out=0)):
        assert wgrad(**change) == arg, change
    assert lib.sm_activation_sums_workspace_bytes(0, 4) == 0
    assert lib.sm_weight_gradient_workspace_bytes(base, 1, 0, 8, 8, 1, 16) == 0


def test_packed_linear_is_selected_and_shares_parameters():
    layer = nn.Linear(40, 5)
    packed = activations.PackedLinear.from_linear(layer)
    assert packed.weight is layer.weight and packed.bias is layer.bias and packed.training
    assert not activations.PackedLinear.from_linear(layer.eval()).training
    assert activations.PackedLinear.from_linear(nn.Linear(4, 3, bias=False)).bias is None
    plain = GPT2(layers=2, width=16, heads=2, vocab=32, context=8)
    model = GPT2(layers=2, width=16, heads=2, vocab=32, context=8, checkpoints="int8")
    assert set(plain.state_dict()) == set(model.state_dict())
    opt = RankOneAWeightedPE(model, lr=1e-2, module_filter=gpt2_matrix_filter)
    attn = model.transformer.h[0].attn
    assert opt.a_sources[id(attn.k_proj.weight)] is attn.q_proj.weight
    assert len(opt.named_matrices) == 12
    opt.close()
    assert not attn.q_proj._forward_hooks and not attn.q_proj._forward_pre_hooks
