"""The 8-bit activation checkpoint operators, case by case: inputs, plain forms and 64-bit values.

A checkpoint holds a layer's input for the backward pass in 8 bits: int8 values in groups of 32
consecutive columns of a row, each group with a power-of-two scale 2^e, e the smallest integer with
max|x| <= 127 * 2^e.  Kinds of cases:

  checkpoint   pack an activation (with the column sums an optimizer's statistics take) and unpack it
  weight       dW = delta^T x_hat, the weight gradient of a linear layer from its packed input
  gelu         GELU with a packed input: forward (packing its output for the next layer) and backward
  linear       forward and backward of linear layers that share one packed input

`run` computes the plain form in 32-bit torch arithmetic, or with `own` calls sandmuon_b200.activations.
"""
import math

import torch

own = False

GROUP = 32
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# smallest and largest e: a scale stays a normal number, values packed from f16 stay f16 numbers, and 127 * 2^e
# stays below the type's largest number
E_RANGE = {"bf16": (-126, 121), "f32": (-126, 121), "f16": (-24, 9)}


def listed():
    return [
        # one row of width 768: what a call costs when there is next to no data
        dict(name="checkpoint-one-row", kind="checkpoint", rows=1, cols=768, dtype="bf16", layout="rows", stats=True),
        # one microbatch of the 9-layer x 768 model: 16 sequences of 1024 tokens
        dict(name="checkpoint-768", kind="checkpoint", rows=16384, cols=768, dtype="bf16", layout="rows", stats=True),
        # the hidden activation of the 24-layer x 2048 model: 8 sequences of 2048 tokens
        dict(name="checkpoint-8192", kind="checkpoint", rows=16384, cols=8192, dtype="bf16", layout="rows", stats=True),
        # FP32 training, columns cut out of a wider tensor, no size a multiple of anything
        dict(name="checkpoint-f32-slice", kind="checkpoint", rows=3001, cols=1111, dtype="f32", layout="slice", stats=False),
        # attention projection of the 9-layer x 768 model: a small output, a long sum over tokens
        dict(name="weight-768", kind="weight", rows=16384, d_in=768, d_out=768, dtype="bf16"),
        # the widest layer of the 24-layer x 2048 model
        dict(name="weight-2048-8192", kind="weight", rows=16384, d_in=2048, d_out=8192, dtype="bf16"),
        # FP32 training: the cotangent in full precision
        dict(name="weight-f32-1024", kind="weight", rows=8192, d_in=1024, d_out=1024, dtype="f32"),
        # FP16 training, ragged in every direction
        dict(name="weight-f16-ragged", kind="weight", rows=4099, d_in=1000, d_out=257, dtype="f16"),
        # between the two layers of an MLP, the packed output going to the second one
        dict(name="gelu-4096", kind="gelu", rows=16384, cols=4096, dtype="bf16", approximate="none", pack_output=True),
        # FP32, odd sizes, the tanh form, no packed output
        dict(name="gelu-f32-odd", kind="gelu", rows=1537, cols=1023, dtype="f32", approximate="tanh",
             pack_output=False),
        # query, key and value projections of one input, FP32 weights, BF16 activations
        dict(name="linear-qkv-768", kind="linear", rows=16384, d_in=768, d_out=768, n=3, bias=False, dtype="bf16"),
        # a short fine-tuning batch through one layer with a bias
        dict(name="linear-short", kind="linear", rows=128, d_in=256, d_out=512, n=1, bias=True, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("checkpoint", "weight", "gelu", "linear"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    rows = _log(rng, 1, 16384)
    if kind == "checkpoint":
        return dict(kind=kind, rows=rows, cols=_log(rng, 8, 8192), dtype=dtype,
                    layout=rng.choice(("rows", "rows", "slice", "columns")), stats=rng.random() < 0.7)
    if kind == "weight":
        return dict(kind=kind, rows=rows, d_in=_log(rng, 8, 4096), d_out=_log(rng, 8, 4096), dtype=dtype)
    if kind == "gelu":
        return dict(kind=kind, rows=rows, cols=_log(rng, 8, 4096), dtype=dtype,
                    approximate=rng.choice(("none", "tanh")), pack_output=dtype != "f32" and rng.random() < 0.6)
    return dict(kind=kind, rows=rows, d_in=_log(rng, 8, 2048), d_out=_log(rng, 8, 2048), n=rng.choice((1, 2, 3)),
                bias=rng.random() < 0.5, dtype=dtype)


# ------------------------------------------------------------------ inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _activation(g, rows, cols, dtype):
    """Channels with means N(0.1, 0.05^2) and standard deviations LogNormal(0, 0.5)."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    std = torch.randn(cols, generator=g, device="cuda").mul_(0.5).exp_()
    mean = torch.randn(cols, generator=g, device="cuda").mul_(0.05).add_(0.1)
    return x.mul_(std).add_(mean).to(DTYPES[dtype])


def _cotangent(g, rows, cols, dtype):
    """Channels with standard deviations LogNormal(0, 0.5) times 1e-3 (times a loss scale of 256 in FP16)."""
    d = torch.randn(rows, cols, generator=g, device="cuda")
    std = torch.randn(cols, generator=g, device="cuda").mul_(0.5).exp_().mul_(0.256 if dtype == "f16" else 1e-3)
    return d.mul_(std).to(DTYPES[dtype])


def prepare(case, seed):
    g = _generator(seed)
    rows, dtype, kind = case["rows"], case["dtype"], case["kind"]
    s = dict(case=case)
    if kind == "checkpoint":
        cols = case["cols"]
        if case["layout"] == "rows":
            s["x"] = _activation(g, rows, cols, dtype)
        elif case["layout"] == "slice":
            s["x"] = _activation(g, rows, cols + 13, dtype)[:, 5:5 + cols]
        else:
            s["x"] = _activation(g, rows, cols, dtype).t().contiguous().t()
    elif kind == "weight":
        s["delta"] = _cotangent(g, rows, case["d_out"], dtype)
        s["values"], s["exponents"] = _stored(_activation(g, rows, case["d_in"], dtype), dtype)
    elif kind == "gelu":
        s["x"] = _activation(g, rows, case["cols"], dtype)
        s["delta"] = _cotangent(g, rows, case["cols"], dtype)
    else:
        s["x"] = _activation(g, rows, case["d_in"], dtype).requires_grad_()
        s["weights"] = [(torch.randn(case["d_out"], case["d_in"], generator=g, device="cuda") * 0.02).requires_grad_()
                        for _ in range(case["n"])]
        s["biases"] = [(torch.randn(case["d_out"], generator=g, device="cuda") * 0.02).requires_grad_()
                       if case["bias"] else None for _ in range(case["n"])]
        s["deltas"] = [_cotangent(g, rows, case["d_out"], dtype) for _ in range(case["n"])]
    return s


# -------------------------------------------------------------- plain forms

def _power(e):
    """2^e in FP32 for integer e in [-126, 127]."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _quantise(x, dtype):
    """(values, e) of a 2-D activation: FP32 integers in [-127, 127] [rows, groups, 32], int32 [rows, groups, 1]."""
    rows, cols = x.shape
    groups = -(-cols // GROUP)
    x = torch.nn.functional.pad(x.float(), (0, groups * GROUP - cols)).view(rows, groups, GROUP)
    low, high = E_RANGE[dtype]
    largest = x.abs().amax(-1, keepdim=True)
    m, k = torch.frexp(largest)
    e = torch.where(largest > 0, k - 7 + (m > 127 / 128).int(), low).clamp(low, high)
    return (x * _power(-e)).round().clamp(-127, 127), e


def _stored(x, dtype):
    """A checkpoint as it is held: int8 [rows, cols rounded up to 16], biased exponents uint8
    [rows, groups rounded up to 4] (padding: values 0, exponents 127)."""
    rows, cols = x.shape
    q, e = _quantise(x, dtype)
    ld, groups = -(-cols // 16) * 16, e.shape[1]
    values = torch.nn.functional.pad(q.view(rows, -1), (0, 16))[:, :ld].to(torch.int8).contiguous()
    codes = torch.nn.functional.pad((e.view(rows, groups) + 127), (0, -groups % 4), value=127)
    return values, codes.to(torch.uint8).contiguous()


def _round_trip(x, dtype):
    """What the checkpoint of x stands for, in FP32."""
    q, e = _quantise(x, dtype)
    return (q * _power(e)).view(x.shape[0], -1)[:, :x.shape[1]]


def _held(values, exponents, cols):
    """What a stored checkpoint stands for, in FP32."""
    scale = _power(exponents.int() - 127).repeat_interleave(GROUP, 1)
    return values[:, :cols].float() * scale[:, :cols]


def _gelu_plain(x, approximate):
    if approximate == "tanh":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))
    return 0.5 * x * torch.erfc(x * -math.sqrt(0.5))


def _gelu_slope_plain(x, approximate):
    if approximate == "tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x))
        return 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * x * x)
    return 0.5 * torch.erfc(x * -math.sqrt(0.5)) + x * torch.exp(-0.5 * x * x) * (1 / math.sqrt(2 * math.pi))


def _plain(s):
    case = s["case"]
    dtype, kind = case["dtype"], case["kind"]
    to = DTYPES[dtype]
    if kind == "checkpoint":
        x = s["x"].float()
        out = [_round_trip(x, dtype).to(to)]
        return out + [torch.stack((x.square().sum(0), x.sum(0)))] if case["stats"] else out
    if kind == "weight":
        return s["delta"].float().t() @ _held(s["values"], s["exponents"], case["d_in"])
    if kind == "gelu":
        y = _gelu_plain(s["x"].float(), case["approximate"]).to(to)
        held = _round_trip(s["x"], dtype)
        out = [y, (s["delta"].float() * _gelu_slope_plain(held, case["approximate"])).to(to)]
        if case["pack_output"]:
            z = y.float()
            out += [_round_trip(z, dtype).to(to), torch.stack((z.square().sum(0), z.sum(0)))]
        return out
    with torch.no_grad():
        x = s["x"].detach().float()
        held = _round_trip(x, dtype)
        weights = [w.detach().to(to).float() for w in s["weights"]]
        deltas = [d.float() for d in s["deltas"]]
        outs = [x @ w.t() if b is None else x @ w.t() + b.detach().to(to).float() for w, b in zip(weights, s["biases"])]
        dx = sum(d @ w for d, w in zip(deltas, weights))
        return [[y.to(to) for y in outs], dx.to(to), [d.t() @ held for d in deltas],
                [d.sum(0) for d, b in zip(deltas, s["biases"]) if b is not None],
                torch.stack((x.square().sum(0), x.sum(0)))]


def _own(s):
    from sandmuon_b200 import activations
    case = s["case"]
    kind = case["kind"]
    if kind == "checkpoint":
        packed = activations.pack(s["x"], stats=case["stats"])
        values = activations.unpack(packed)
        return [values, packed.sums] if case["stats"] else [values]
    if kind == "weight":
        packed = activations.PackedActivation(s["values"], s["exponents"], (case["rows"], case["d_in"]),
                                              DTYPES[case["dtype"]])
        return activations.weight_gradient(s["delta"], packed)
    if kind == "gelu":
        x = s["x"].detach().requires_grad_()
        if case["pack_output"]:
            y, packed = activations.gelu(x, approximate=case["approximate"], pack_output=True, stats=True)
            dx, = torch.autograd.grad(y, x, s["delta"])
            return [y.detach(), dx, activations.unpack(packed), packed.sums]
        y = activations.gelu(x, approximate=case["approximate"])
        dx, = torch.autograd.grad(y, x, s["delta"])
        return [y.detach(), dx]
    packed = activations.pack(s["x"], stats=True)
    outs = [activations.linear(s["x"], w, b, packed=packed) for w, b in zip(s["weights"], s["biases"])]
    biases = [b for b in s["biases"] if b is not None]
    grads = torch.autograd.grad(outs, [s["x"], *s["weights"], *biases], s["deltas"])
    n = len(s["weights"])
    return [[y.detach() for y in outs], grads[0], list(grads[1:1 + n]), list(grads[1 + n:]), packed.sums]


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ---------------------------------------------------------------- the floor

def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    rows, kind = case["rows"], case["kind"]
    held = 1 + 1 / GROUP
    if kind == "checkpoint":
        n = rows * case["cols"]
        return {"bytes": n * (2 * size + 2 * held) + (8 * case["cols"] if case["stats"] else 0), "flops": 0}
    if kind == "weight":
        i, o = case["d_in"], case["d_out"]
        return {"bytes": rows * (i * held + o * size) + 4 * i * o, "flops": 2 * rows * i * o}
    if kind == "gelu":
        n = rows * case["cols"]
        # x, y, delta and dx once each, the packed input written and read, the packed output written, read and unpacked
        bytes_ = n * (4 * size + 2 * held)
        if case["pack_output"]:
            bytes_ += n * (2 * held + size) + 8 * case["cols"]
        return {"bytes": bytes_, "flops": 0}
    i, o, n = case["d_in"], case["d_out"], case["n"]
    # forward, input gradient and weight gradient of each layer; x, dx, outputs, cotangents, the checkpoint once
    # written and read, the FP32 weights and their gradients
    return {"bytes": rows * (2 * i * size + 2 * n * o * size + 2 * held * i) + 8 * n * i * o + 8 * i,
            "flops": 6 * n * rows * i * o}


# ----------------------------------------------------------- 64-bit values

def _power64(e):
    return ((e + 1023) << 52).view(torch.float64)


def _round_trip64(x, dtype):
    """The checkpoint's values from its definition: per 32 columns the smallest e with max|x| <= 127 * 2^e."""
    low, high = E_RANGE[dtype]
    out = torch.empty_like(x)
    for c in range(0, x.shape[1], GROUP):
        part = x[:, c:c + GROUP]
        top = part.abs().max(1, keepdim=True).values
        e = torch.log2(top.clamp(min=1e-300) / 127).ceil().long()
        e += (top > 127 * _power64(e)).long()
        e -= (top <= 127 * _power64(e - 1)).long()
        e = e.clamp(low, high)
        out[:, c:c + GROUP] = torch.round(part / _power64(e)).clamp(-127, 127) * _power64(e)
    return out


def _gelu64(x, approximate):
    """(GELU, its derivative) in FP64."""
    if approximate == "tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (x + 0.044715 * x ** 3))
        return x * (1 + t) / 2, (1 + t) / 2 + x * (1 - t ** 2) / 2 * c * (1 + 0.134145 * x ** 2)
    phi = torch.special.ndtr(x)
    return x * phi, phi + x * torch.exp(-x ** 2 / 2) / math.sqrt(2 * math.pi)


def exact(case, seed):
    s = prepare(case, seed)
    dtype, kind = case["dtype"], case["kind"]
    to = DTYPES[dtype]
    if kind == "checkpoint":
        x = s["x"].double()
        out = [_round_trip64(x, dtype)]
        return out + [torch.stack((x.pow(2).sum(0), x.sum(0)))] if case["stats"] else out
    if kind == "weight":
        scale = _power64(s["exponents"].long() - 127).repeat_interleave(GROUP, 1)[:, :case["d_in"]]
        return s["delta"].double().t() @ (s["values"][:, :case["d_in"]].double() * scale)
    if kind == "gelu":
        x = s["x"].double()
        y, _ = _gelu64(x, case["approximate"])
        _, slope = _gelu64(_round_trip64(x, dtype), case["approximate"])
        out = [y, s["delta"].double() * slope]
        if case["pack_output"]:
            z = y.to(to).double()
            out += [_round_trip64(z, dtype), torch.stack((z.pow(2).sum(0), z.sum(0)))]
        return out
    x = s["x"].detach().double()
    held = _round_trip64(x, dtype)
    weights = [w.detach().to(to).double() for w in s["weights"]]
    deltas = [d.double() for d in s["deltas"]]
    outs = [x @ w.t() + (0 if b is None else b.detach().to(to).double()) for w, b in zip(weights, s["biases"])]
    dx = torch.zeros_like(x)
    for d, w in zip(deltas, weights):
        dx += d @ w
    return [outs, dx, [d.t() @ held for d in deltas],
            [d.sum(0) for d, b in zip(deltas, s["biases"]) if b is not None],
            torch.stack((x.pow(2).sum(0), x.sum(0)))]
