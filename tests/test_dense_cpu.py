"""Dense layers and orthogonalised updates where no GPU is needed: the pure-torch layer, refusals, the entry points' checks."""
import ctypes

import pytest
import torch

import difflogic_b200 as D
from difflogic_b200 import _native as N
from difflogic_b200 import optim
from difflogic_b200.denselayer import ACTIVATIONS, DenseLayer, dense_python


@pytest.mark.parametrize("activation", [None, "none", "relu", "sigmoid", "silu", "gelu"])
def test_python_layer_is_its_formula(activation):
    torch.manual_seed(0)
    layer = DenseLayer(7, 5, device="cpu", activation=activation)
    assert layer.implementation == "python" and not layer.feature_major
    x, r = torch.randn(3, 7), torch.randn(3, 5)
    z = x.double() @ layer.weight.detach().double().t() + layer.bias.detach().double()
    act = {0: lambda v: v, 1: lambda v: v.clamp(min=0), 2: lambda v: 1 / (1 + (-v).exp()), 3: lambda v: v / (1 + (-v).exp()),
           4: lambda v: v * torch.special.ndtr(v)}[ACTIVATIONS[activation]]
    want = act(z) + r.double()
    assert torch.allclose(layer(x, r).double(), want, rtol=1e-5, atol=1e-6)
    layer(x).sum().backward()
    assert layer.weight.grad.shape == (5, 7) and layer.bias.grad.shape == (5,)


def test_python_layer_gradients_against_differences():
    torch.manual_seed(1)
    x, w, b, r = (torch.randn(*s, dtype=torch.float64, requires_grad=True) for s in [(3, 4), (5, 4), (5,), (3, 5)])
    for activation in ("sigmoid", "silu", "gelu"):
        assert torch.autograd.gradcheck(lambda *t: dense_python(*t, activation=activation), (x, w, b, r))


def test_layer_in_front_of_logic_layers_on_the_cpu():
    torch.manual_seed(2)
    model = torch.nn.Sequential(DenseLayer(6, 12, device="cpu"), D.LogicLayer(12, 20, device="cpu"), D.GroupSum(2, device="cpu"))
    y = model(torch.randn(4, 6))
    assert y.shape == (4, 2)
    y.sum().backward()
    assert model[0].weight.grad.abs().sum() > 0


def test_layer_arguments():
    with pytest.raises(ValueError, match="activation"):
        DenseLayer(3, 4, device="cpu", activation="tanh")
    with pytest.raises(ValueError, match="float32"):
        DenseLayer(3, 4, device="cpu", dtype=torch.float64)
    assert DenseLayer(3, 4, device="cpu", bias=False).bias is None


def test_dense_refuses_what_does_not_fit():
    x, w = torch.randn(3, 4), torch.randn(5, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        D.dense(x, w)
    for bad in [dict(x=torch.randn(3, 5)), dict(weight=torch.randn(4)), dict(weight=torch.randn(0, 4)), dict(bias=torch.randn(4)),
                dict(residual=torch.randn(3, 4)), dict(residual=torch.randn(5)), dict(weight=w.double()), dict(bias=torch.randn(5).half()),
                dict(activation="tanh"), dict(x=torch.tensor(1.0))]:
        with pytest.raises(ValueError):
            D.dense(**{**dict(x=x, weight=w), **bad})


@pytest.mark.parametrize("coefficients, steps", [((3.4445, -4.7750, 2.0315), 0), ((3.4445, -4.7750, 2.0315), 65), ((3.4445, -4.7750, 2.0315), 2.0),
                                                 ((3.4445, -4.7750, 2.0315), True), ((9.0, 9.0, 9.0), 5), ((float("nan"), 0.0, 0.0), 1),
                                                 (((1.5, -0.5, 0.0),) * 2, 3), ((1.5, -0.5), 2), ((70.0, -70.0, 0.0), 1)])
def test_newton_schulz_refuses(coefficients, steps):
    with pytest.raises(ValueError):
        D.ops._newton_schulz(coefficients, steps)


def test_newton_schulz_coefficients_as_the_library_takes_them():
    assert list(D.ops._newton_schulz((1.5, -0.5, 0.0), 2)) == [1.5, -0.5, 0.0] * 2
    table = D.ops._newton_schulz(D.ops._coefficients([[3, -3.5, 1.5], (1.5, -0.5, 0)]), 2)
    assert list(table) == [3.0, -3.5, 1.5, 1.5, -0.5, 0.0]


def test_orthogonalize_and_muon_refuse_on_the_cpu():
    x = torch.randn(4, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        D.ops.orthogonalize(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        D.ops.muon_step([x], [x.clone()], [x.clone()], lr=0.1)
    with pytest.raises(ValueError, match="momenta"):
        D.ops.muon_step([x], [x.clone()], [], lr=0.1)
    for bad in (dict(momentum=1.0), dict(lr=-1.0), dict(weight_decay=-0.1), dict(eps=0.0), dict(momentum=float("nan"))):
        with pytest.raises(ValueError):
            D.ops.muon_step([x], [x.clone()], [x.clone()], **{**dict(lr=0.1), **bad})
    D.ops.muon_step([], [], [], lr=0.1)


def test_flat_muon_arguments():
    p = torch.nn.Parameter(torch.randn(4, 4))
    with pytest.raises(ValueError, match="CUDA"):
        optim.FlatMuon([p])
    for bad in (dict(momentum=1.0), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(ns_steps=0), dict(ns_coefficients=(9, 9, 9))):
        with pytest.raises(ValueError):
            optim.FlatMuon([p], **bad)


def test_entry_points_check_their_arguments():
    """These come back before anything is launched."""
    lib = N.lib()
    coefficients = (ctypes.c_float * 3)(1.5, -0.5, 0.0)
    bad = N.DL_ERR_INVALID_ARG
    assert lib.dl_orthogonalize(None, None, 1, 4, 4, 0, 1, coefficients, 1e-7, None, None) == bad
    assert lib.dl_orthogonalize(None, None, -1, 4, 4, 0, 1, coefficients, 1e-7, None, None) == bad
    assert lib.dl_orthogonalize(None, None, 1, 4, 4, 3, 1, coefficients, 1e-7, None, None) == bad
    assert lib.dl_orthogonalize(None, None, 1, 4, 4, 0, 0, coefficients, 1e-7, None, None) == bad
    assert lib.dl_orthogonalize(None, None, 1, 4, 4, 0, 1, coefficients, 0.0, None, None) == bad
    assert lib.dl_orthogonalize(None, None, 70000, 4, 4, 0, 1, coefficients, 1e-7, None, None) == N.DL_ERR_TOO_LARGE
    assert lib.dl_orthogonalize(None, None, 1, 0, 4, 0, 1, coefficients, 1e-7, None, None) == N.DL_OK
    table = (ctypes.c_int64 * 5)(0, 0, 0, 4, 4)
    assert lib.dl_muon_step_f32(table, 1, 0.1, 0.9, 1, 0.0, 1, coefficients, 1e-7, None, None) == bad
    assert lib.dl_muon_step_f32(None, 0, 0.1, 0.9, 1, 0.0, 1, coefficients, 1e-7, None, None) == N.DL_OK
    assert lib.dl_muon_step_f32(None, 1, 0.1, 0.9, 1, 0.0, 1, coefficients, 1e-7, None, None) == bad
    args = [None, 4, 0, None, None, None, 0, 0, 0, None, 0, None, None, None, None]
    assert lib.dl_dense_forward(*args, 2, 4, 4, 0, None) == bad
    assert lib.dl_dense_forward(*args, 0, 4, 4, 0, None) == N.DL_OK
    assert lib.dl_dense_forward(*args, 2, 0, 4, 0, None) == bad
    assert lib.dl_dense_forward(*args, 2, 4, 4, 7, None) == bad
    assert lib.dl_dense_backward(None, 0, None, None, 4, 0, None, None, None, None, None, None, None, 2, 4, 4, 0, None) == bad
    sizes = (ctypes.c_int64 * 3)()
    for pitch, kind, least in [(8, 1, 0), (7, 1, 100 * 8 * 2), (8, 0, 3 * 100 * 8 * 2)]:     # rows on 16-byte units are read in place
        lib.dl_dense_forward_sizes(16, pitch, 0, 16, 100, 7 if pitch == 7 else 8, 8, 0, kind, sizes)
        assert (sizes[0] == 0) == (least == 0) and sizes[0] >= least
    assert "dl_dense" in N.last_error()


@pytest.mark.parametrize("rows, cols, k, batch, kind", [(1, 1, 1, 1, 0), (128, 4096, 784, 1, 0), (5, 3, 100000, 2, 1), (4096, 4096, 4096, 1, 2)])
def test_workspaces_follow_the_sizes(rows, cols, k, batch, kind):
    lib = N.lib()
    for value in (64, 128, 256, 0):
        with N.tuning(N.TUNE_MATMUL_COLUMNS, value):
            sizes = (ctypes.c_int64 * 3)()
            lib.dl_dense_forward_sizes(16, k, 0, 16, rows, k, cols, value == 64, kind, sizes)
            assert 0 <= sizes[2] <= 64 << 20
            assert lib.dl_orthogonalize_workspace_bytes(batch, rows, cols, kind) > 0
            assert lib.dl_dense_backward_workspace_bytes(16, 0, 1, 16, k, 0, 16, 1, 1, rows, k, cols, kind) > 0


def test_gradients_outside_the_flat_buffer_are_reduced_in_it():
    """A dense layer's gradient is a tensor of its own: before a bucket of the flat buffer is reduced, it moves into its slice."""
    from difflogic_b200.training import TrainStep
    flat = torch.zeros(12)
    inside, outside = torch.nn.Parameter(torch.zeros(4)), torch.nn.Parameter(torch.zeros(2, 4))

    class Optimizer:
        def grad_view(self, p):
            return flat[:4] if p is inside else flat[4:].view(2, 4)

    step = TrainStep.__new__(TrainStep)
    step._on_gpu, step.optimizer = True, Optimizer()
    step._bucket_of, step._bucket_slices, step._pending = {inside: 0, outside: 0}, [flat], [2]
    reduced = []
    step._launch_all_reduce = lambda t: reduced.append(t.clone())
    flat[:4] = 1
    inside.grad, outside.grad = flat[:4], torch.arange(8.).view(2, 4)
    step._reduce_when_ready(outside)
    assert not reduced and outside.grad.data_ptr() == flat[4:].data_ptr()
    step._reduce_when_ready(inside)
    assert inside.grad.data_ptr() == flat.data_ptr()
    assert len(reduced) == 1 and reduced[0].tolist() == [1, 1, 1, 1, 0, 1, 2, 3, 4, 5, 6, 7]
