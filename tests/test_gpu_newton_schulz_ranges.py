"""Newton-Schulz steps whose Gram matrices and polynomials are far from 1: everything that is kept between products has to fit its 16-bit
planes for all coefficients that are accepted, and so have the scales for all eps and sizes of values."""
import math

import pytest
import torch

import difflogic_b200 as D

pytestmark = pytest.mark.gpu

# polynomials with a past 16, with values between 4 and 8 on the way (their squares pass 16), with b s^2 + c s^4 past 16, cubic ones
COEFFICIENTS = [((20.0, -60.0, 48.0),), ((20.0, -60.0, 45.0),), ((20.0, -40.0, 20.0),), ((16.5, -16.5, 0.0),),
                ((6.0, 0.0, 0.0), (0.2, -0.01, 0.0001)), ((5.0, 0.0, 0.0), (0.3, -0.001, 0.00001)), ((8.0, 0.0, 0.0), (1.0, 0.0, 0.0)),
                ((8.0, 0.0, 0.0), (0.5, -0.015, 0.0), (1.5, -0.1, 0.002)), ((24.0, -60.0, 44.0), (0.1, 0.0, 0.0))]


def steps_and_bound(g, coefficients, unit, eps=1e-7):
    """The definition in 64 bits, and how far off (Frobenius norm) iterates may be whose planes are `unit` off, relative to each value.

    With X off by E, p(X) is off by max |p'| E: p acts on the singular values.  A step adds what it rounds itself: S = X X^T from planes that
    are a unit off, summed in 32 bits (2^-23 every 16 values) and stored (a unit, no less than half the smallest 16-bit number over 2^12,
    times the power of two that S and M are kept smaller by, 64 at most); M = a + b S + c S^2 likewise, S^2 of pairs; M X likewise."""
    x = g.double()
    x = x / x.square().sum().sqrt().clamp(min=eps)
    x = x if x.shape[0] <= x.shape[1] else x.mT
    side = x.shape[0]
    F, top = (lambda v: v.norm().item()), (lambda v: torch.linalg.matrix_norm(v, 2).item())
    acc = lambda k: (k / 16 + 8) * 2.0 ** -23  # noqa: E731
    pair = 2.0 ** -22
    least = 2.0 ** -25 / 4096 * 64
    off = unit * F(x) + least * math.sqrt(x.numel())
    for a, b, c in coefficients:
        s = x @ x.mT
        m = a * torch.eye(side, dtype=torch.float64, device=x.device) + b * s + c * s @ s
        s_off = (2 * unit + acc(x.shape[1])) * F(x) ** 2 + pair * F(s) + least * side
        m_off = (abs(b) + 2 * abs(c) * top(s)) * s_off + abs(c) * (2 * pair + acc(side)) * F(s) ** 2 + pair * F(m) + least * side
        own = top(x) * m_off + (2 * unit + acc(side)) * F(m) * F(x) + least * math.sqrt(x.numel())
        reach = top(x) * 1.01
        slopes = torch.linspace(0, reach, 4001, dtype=torch.float64)
        slope = (a + 3 * b * slopes ** 2 + 5 * c * slopes ** 4).abs().max().item()
        x = m @ x
        off = slope * off + own + pair * F(x)
    return (x if g.shape[0] <= g.shape[1] else x.mT), off


def matrix(kind, rows, cols):
    gen = torch.Generator().manual_seed(rows + cols)
    if kind == "one direction":
        return torch.randn(rows, 1, generator=gen) @ torch.randn(1, cols, generator=gen)
    return torch.randn(rows, cols, generator=gen)


@pytest.mark.parametrize("t", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", ["noise", "one direction"])
@pytest.mark.parametrize("coefficients", COEFFICIENTS)
@pytest.mark.parametrize("rows, cols", [(1, 17), (64, 40), (40, 64), (300, 130)])
def test_all_accepted_coefficients_fit(rows, cols, coefficients, kind, t):
    g = matrix(kind, rows, cols).to(t).cuda()
    got = D.ops.orthogonalize(g, steps=len(coefficients), coefficients=coefficients)
    want, off = steps_and_bound(g, coefficients, 2.0 ** -11 if t == torch.bfloat16 else 2.0 ** -22)
    half = torch.finfo(t).eps / 2
    assert bool(torch.isfinite(got).all())
    assert (got.double() - want).norm().item() <= off + half * (want.norm().item() + off) + 2.0 ** -25 * math.sqrt(g.numel())


def test_gate_weights_and_dense_weights_take_the_same_step():
    """The same matrix with columns of zeros behind it: once up to 16 columns, in 64 bits, once in planes."""
    coefficients = ((20.0, -60.0, 48.0),)
    gen = torch.Generator().manual_seed(3)
    narrow = torch.randn(200, 16, generator=gen).cuda()
    wide = torch.cat([narrow, torch.zeros(200, 8, device="cuda")], 1)
    weights, momenta = [torch.zeros_like(narrow), torch.zeros_like(wide)], [torch.zeros_like(narrow), torch.zeros_like(wide)]
    D.ops.muon_step(weights, [narrow, wide], momenta, lr=1.0, steps=1, coefficients=coefficients)
    want, off = steps_and_bound(narrow, coefficients, 2.0 ** -22)
    rate = math.sqrt(200 / 16), math.sqrt(200 / 24)
    for w, r in zip(weights, rate):
        assert bool(torch.isfinite(w).all())
        assert (w[:, :16].double() / -r - want).norm().item() <= 2 * off + 2.0 ** -22 * want.norm().item()


@pytest.mark.parametrize("rows, cols", [(60, 16), (60, 40), (40, 90), (5, 7)])
@pytest.mark.parametrize("eps", [1e-30, 1e-36, 1e-44, 1e-160, 5e-324])
def test_any_eps(rows, cols, eps):
    assert not D.ops.orthogonalize(torch.zeros(rows, cols, device="cuda"), eps=eps).any()
    g = matrix("noise", rows, cols).cuda()
    got = D.ops.orthogonalize(torch.stack([g, torch.zeros_like(g), g]), eps=eps)
    assert not got[1].any() and torch.equal(got[0], got[2])
    want, off = steps_and_bound(g, [D.ops.NEWTON_SCHULZ] * 5, 2.0 ** -22)
    assert (got[0].double() - want).norm().item() <= off + 2.0 ** -23 * want.norm().item()
    w, m = torch.ones(rows, cols, device="cuda"), torch.zeros(rows, cols, device="cuda")
    D.ops.muon_step([w], [torch.zeros_like(w)], [m], lr=0.1, eps=eps)
    assert torch.equal(w, torch.ones_like(w))


@pytest.mark.parametrize("rows, cols", [(60, 16), (60, 40), (40, 90)])
@pytest.mark.parametrize("size", [2.0 ** -140, 2.0 ** -126, 2.0 ** -100, 2.0 ** 100, 2.0 ** 125])
def test_the_smallest_and_the_largest_matrices(rows, cols, size):
    """Brought to norm 1, a matrix is what it was before all its entries were multiplied with a power of two."""
    g = (matrix("noise", rows, cols) * size).cuda()      # rounded to what is left of 24 bits down there
    assert bool(torch.isfinite(g).all())
    got = D.ops.orthogonalize(g, eps=1e-60)
    want, off = steps_and_bound(g, [D.ops.NEWTON_SCHULZ] * 5, 2.0 ** -22, eps=1e-60)
    assert (got.double() - want).norm().item() <= off + 2.0 ** -23 * want.norm().item()


def test_an_optimizer_of_steep_steps():
    """One list of coefficients for gate weights and dense weights: the products of both stay finite, and their sizes are those of the steps."""
    torch.manual_seed(0)
    model = torch.nn.Sequential(D.DenseLayer(30, 50), D.LogicLayer(50, 80), D.GroupSum(4))
    opt = D.optim.FlatMuon(model.parameters(), lr=0.01, weight_decay=0.0, ns_coefficients=(20.0, -60.0, 48.0), ns_steps=1)
    before = [p.detach().clone() for p in model.parameters() if p.dim() == 2]
    model(torch.rand(64, 30, device="cuda")).square().mean().backward()
    grads = [p.grad.clone() for p in model.parameters() if p.dim() == 2]
    opt.step()
    for p, old, g in zip((p for p in model.parameters() if p.dim() == 2), before, grads):
        want, off = steps_and_bound(g * 0.0975, ((20.0, -60.0, 48.0),), 2.0 ** -22)     # (1 - mu) g and nesterov: a multiple of g
        rate = 0.01 * math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
        moved = (old.double() - p.detach().double()) / rate
        assert (moved - want).norm().item() <= 2 * off + 2.0 ** -22 * want.norm().item() + 2 * 2.0 ** -24 * (old.norm() + p.norm()).item() / rate
