"""Optimizer steps between a forward and a backward pass: gradients of dense layers are those of the weights that the forward pass read, and
what a step changes in place counts as changed for autograd where it was called on tensors of anybody's graph."""
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


@pytest.mark.parametrize("way", ["native", "python"])
def test_muon_step_is_in_place_for_autograd(way):
    class Weight(torch.nn.Parameter):      # not what the native call takes
        pass

    torch.manual_seed(0)
    w, x = torch.randn(8, 20, device="cuda"), torch.randn(5, 20, device="cuda", requires_grad=True)
    w = torch.nn.Parameter(w) if way == "native" else Weight(w)
    g, m = torch.randn(8, 20, device="cuda"), torch.zeros(8, 20, device="cuda")
    y = torch.nn.functional.linear(x, w)
    versions = w._version, g._version, m._version
    D.ops.muon_step([w], [g], [m], lr=0.1)
    assert (w._version, g._version, m._version) == (versions[0] + 1, versions[1], versions[2] + 1)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    D.dense(x, w).sum().backward()         # the weights as they are now
    assert torch.allclose(x.grad, w.detach().sum(0).expand(5, 20), rtol=1e-5, atol=1e-5)
    with torch.inference_mode():
        state = [torch.randn(8, 20, device="cuda") for _ in range(3)]
        D.ops.muon_step(state[:1], state[1:2], state[2:], lr=0.1)      # these have no counters


def test_an_optimizers_step_leaves_version_counters_alone():
    model = torch.nn.Sequential(D.DenseLayer(20, 30), D.LogicLayer(30, 40), D.GroupSum(4))
    opt = FlatMuon(model.parameters(), lr=0.1)
    versions = [p._version for p in model.parameters()]
    loss = model(torch.randn(40, 20, device="cuda")).sum()
    loss.backward(retain_graph=True)
    opt.step()
    assert versions == [p._version for p in model.parameters()]
    loss.backward()


@pytest.mark.parametrize("rows", [1, 8, 32, 33])
def test_captured_steps_read_the_weights_of_their_replay(rows):
    """What a backward pass reads is laid out anew in every replay."""
    torch.manual_seed(rows)
    x, w, b = (torch.randn(*s, device="cuda", requires_grad=True) for s in ((rows, 24), (40, 24), (40,)))
    gy = torch.randn(rows, 40, device="cuda")
    run = lambda: torch.autograd.grad(D.dense(x, w, b, activation="gelu"), (x, w, b), gy)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graphs, results = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(run())
        graphs.append(graph)
    momenta = [torch.zeros_like(x), torch.zeros_like(w)]
    for _ in range(3):
        D.ops.muon_step([x, w], [torch.randn_like(x), torch.randn_like(w)], momenta, lr=0.1)
        want = run()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for got in results:
            assert all(torch.equal(p, q) for p, q in zip(want, got))
