"""Optimizer steps between a forward and a backward pass: gradients of dense layers are those of the weights that the forward pass read."""
import pytest
import torch

import difflogic_b200 as D
from difflogic_b200.optim import FlatAdam, FlatMuon

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 8, 9, 32, 33, 100])
@pytest.mark.parametrize("optimizer", [FlatMuon, FlatAdam])
@pytest.mark.parametrize("way", ["native", "python"])
@pytest.mark.parametrize("needs", ["both", "x", "w"])
def test_gradients_are_those_of_the_weights_that_were_read(rows, optimizer, way, needs):
    torch.manual_seed(rows)
    layer = D.DenseLayer(24, 40, activation="silu")
    x = torch.nn.Parameter(torch.randn(rows, 24, device="cuda"))
    opt = optimizer([*layer.parameters(), x], lr=0.1)
    bias = layer.bias if way == "native" else layer.bias[:1].expand(40)     # a bias of other strides goes the other way
    x.requires_grad_(needs != "w")
    layer.weight.requires_grad_(needs != "x")
    y = D.dense(x, layer.weight, bias, activation="silu")
    leaves = [p for p in (x, layer.weight, layer.bias) if p.requires_grad]
    gy = torch.randn_like(y)
    want = torch.autograd.grad(y, leaves, gy, retain_graph=True)
    before = [p.detach().clone() for p in (x, layer.weight)]
    for p in (*layer.parameters(), x):
        p.requires_grad_(True)
        p.grad = torch.randn_like(p)
    opt.step()
    assert all(not torch.equal(p, q) for p, q in zip(before, (x, layer.weight)))
    got = torch.autograd.grad(y, leaves, gy, retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    again = torch.autograd.grad(y, leaves, gy)
    assert all(torch.equal(p, q) for p, q in zip(want, again))
