"""Captures beside a graph that is alive are refused for every form that a dense layer's tensors come in, and run once it is gone."""
import pytest
import torch

import difflogic_b200 as D

pytestmark = pytest.mark.gpu


class Weight(torch.nn.Parameter):
    pass


def tensors(case):
    """The tensors of a call, the leaf that is common to both graphs, and how the call makes its arguments of them."""
    gen = torch.Generator().manual_seed(0)
    make = lambda *s: torch.randn(*s, generator=gen).cuda()  # noqa: E731
    x, w, b, r = make(40, 16), make(24, 16), make(24), make(40, 24)
    same = lambda x, w, b, r: (x, w, b, r)  # noqa: E731
    if case == "x of three dimensions":
        x = make(5, 8, 16).requires_grad_()
        return (x, w, b, None), x, same
    if case == "residual of three dimensions":
        r = make(5, 8, 24).requires_grad_()
        return (x.view(5, 8, 16), w, b, r), r, same
    if case == "expanded leaf":
        b = make(1).expand(24).requires_grad_()
        return (x, w, b, None), b, same
    if case == "leaf that is expanded":
        b = make(1).requires_grad_()
        return (x, w, b, None), b, lambda x, w, b, r: (x, w, b.expand(24), r)
    if case == "weight of other strides":
        w = make(24, 32)[:, ::2].requires_grad_()
        return (x, w, b, None), w, same
    if case == "transposed weight":
        w = make(16, 24).requires_grad_()
        return (x, w, b, None), w, lambda x, w, b, r: (x, w.t(), b, r)
    if case == "subclass":
        w = Weight(w)
        return (x, w, b, r), w, same
    assert case == "x made of the leaf"
    x = make(16, 40).requires_grad_()
    return (x, w, b, r), x, lambda x, w, b, r: (x.t().reshape(5, 8, 16), w, b, r.view(5, 8, 24))


@pytest.mark.parametrize("case", ["x of three dimensions", "residual of three dimensions", "expanded leaf", "leaf that is expanded",
                                  "weight of other strides", "transposed weight", "subclass", "x made of the leaf"])
def test_capture_beside_a_graph_that_is_alive(case):
    given, leaf, arguments = tensors(case)
    call = lambda: D.dense(*arguments(*given), activation="relu")  # noqa: E731
    gy = torch.randn(call().shape, generator=torch.Generator().manual_seed(1)).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            want, = torch.autograd.grad(call(), leaf, gy)
    torch.cuda.current_stream().wait_stream(side)
    alive = call()
    with pytest.raises(RuntimeError, match="alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            call()
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got, = torch.autograd.grad(call(), leaf, gy)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(want, got)
