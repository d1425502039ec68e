"""The optimizers' pre-hook on packed layers, without a GPU: it adds the
checkpoint to the call and leaves every other argument as it was."""
import pytest
import torch
from torch import nn

from sandmuon_b200 import DiagonalWeightedPE, activations


class Gated(activations.PackedLinear):
    """A layer with arguments of its own behind the input and its checkpoint."""

    def forward(self, x, packed=None, gate=None, *, scale=1.0):
        self.seen = (packed, gate, scale)
        return nn.functional.linear(x, self.weight)


@pytest.fixture
def model(monkeypatch):
    monkeypatch.setattr(activations, "pack_input", lambda x, *, stats=False: ("packed", stats))
    net = nn.Sequential(Gated(8, 4))
    opt = DiagonalWeightedPE(net, lr=1e-2)
    net[0]._forward_hooks.clear()  # the statistics' own hook needs a GPU
    yield net[0]
    opt.close()


def test_arguments_of_a_subclass_pass_the_hook(model):
    x, gate = torch.randn(3, 8), torch.randn(3, 4)
    ours = ("packed", True)
    for call, want in ((lambda: model(x), (ours, None, 1.0)),
                       (lambda: model(x, gate=gate), (ours, gate, 1.0)),
                       (lambda: model(x, None), (ours, None, 1.0)),
                       (lambda: model(x, None, gate, scale=2.0), (ours, gate, 2.0)),
                       (lambda: model(x, packed=None, scale=3.0), (ours, None, 3.0)),
                       (lambda: model(x, "theirs", gate), ("theirs", gate, 1.0)),
                       (lambda: model(x, packed="theirs", gate=gate), ("theirs", gate, 1.0))):
        call()
        assert model.seen[0] == want[0] and model.seen[1] is want[1] and model.seen[2] == want[2]


def test_no_checkpoint_where_no_statistics_are_taken(model):
    x = torch.randn(3, 8)
    with torch.no_grad():
        model(x, scale=2.0)
    assert model.seen == (None, None, 2.0)
    model.eval()
    model(x)
    assert model.seen == (None, None, 1.0)
    model.train()
    model.weight.requires_grad_(False)
    model(x)
    assert model.seen == (None, None, 1.0)
