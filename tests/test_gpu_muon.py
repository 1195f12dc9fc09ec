"""Orthogonalisation and Muon steps against their definition in 64 bits, and a network of dense and logic layers trained with them."""
import copy
import math

import pytest
import torch

import difflogic_b200 as D
from difflogic_b200 import _native as N
from difflogic_b200.optim import FlatAdam, FlatMuon
from difflogic_b200.training import TrainStep

pytestmark = pytest.mark.gpu

DEFAULT = (3.4445, -4.7750, 2.0315)


def definition(g, steps=5, coefficients=DEFAULT, eps=1e-7):
    x = g.detach().double()
    x = x / x.square().sum((-2, -1), keepdim=True).sqrt().clamp(min=eps)
    sets = [coefficients] * steps if isinstance(coefficients[0], float) else coefficients
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    for a, b, c in sets:
        s = x @ x.mT
        x = a * x + (b * s + c * s @ s) @ x
    return x.mT if tall else x


def bound(t, cols):
    """Relative, in the Frobenius norm.  p(s) = a s + b s^3 + c s^5 has slopes of at most 3.9 where the values go, so what a step rounds
    away grows by that much in every later one, 310 times over five.  Up to 16 columns all of it is done in 64 bits: what is left is the
    result's rounding (fp32: 2^-24, and 2^-24 for the product's).  Else the iterates and products are rounded to 22 bits, half a rounding
    2^-23 on average of four of them a step: 310 * 4 * 2^-23 / sqrt(12).  bf16 works with 11 bits where that is harmless, as far off as
    its own rounding: 2^-9 + 2^-9 / 0.8."""
    half = torch.finfo(t).eps / 2
    if cols <= 16:
        return half + 2.0 ** -22
    return half + (1.25 * 2.0 ** -9 if t == torch.bfloat16 else 310 * 4 * 2.0 ** -23 / math.sqrt(12))


def far(got, want):
    got, want = got.double(), want.double()
    return ((got - want).norm() / want.norm()).item()


def spectrum(kind, rows, cols, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, dtype=torch.float64)
    if kind == "noise":
        return x.float()
    if kind == "few":       # a few strong directions
        r = max(1, min(rows, cols) // 16)
        return (torch.randn(rows, r, generator=g, dtype=torch.float64) @ torch.randn(r, cols, generator=g, dtype=torch.float64) + 1e-3 * x).float()
    u, _, v = torch.linalg.svd(x, full_matrices=False)
    s = torch.logspace(0, -6, min(rows, cols), dtype=torch.float64)
    return ((u * s) @ v).float()


SHAPES = [(1, 1), (1, 16), (16, 1), (3, 4), (16, 16), (5, 16), (33, 16), (1000, 16), (4000, 15), (70, 7), (16, 17), (17, 17), (1, 40), (40, 1), (20, 100),
          (100, 20), (64, 64), (128, 128), (129, 127), (200, 260), (300, 300), (700, 130), (130, 700), (1100, 257)]


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows, cols", SHAPES)
@pytest.mark.parametrize("kind", ["noise", "few", "steep"])
def test_orthogonalize(rows, cols, kind, t):
    g = spectrum(kind, rows, cols).to(t).cuda()
    got = D.ops.orthogonalize(g)
    assert got.dtype == t and got.shape == g.shape
    assert far(got, definition(g)) <= bound(t, cols)


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("columns", [64, 128, 256])
@pytest.mark.parametrize("splits", [0, 3])
@pytest.mark.parametrize("rows, cols", [(40, 300), (300, 40), (260, 390), (513, 258)])
def test_every_tile(rows, cols, splits, columns, t):
    g = torch.stack([spectrum("noise", rows, cols, s) for s in (1, 2)]).to(t).cuda()
    with N.tuning(N.TUNE_MATMUL_COLUMNS, columns), N.tuning(N.TUNE_MATMUL_SPLITS, splits):
        got = D.ops.orthogonalize(g)
    want = definition(g)
    for z in range(2):
        assert far(got[z], want[z]) <= bound(t, cols)


@pytest.mark.parametrize("rows, cols", [(50, 16), (50, 40), (40, 90)])
def test_batches_steps_and_coefficients(rows, cols):
    g = torch.stack([spectrum("noise", rows, cols, s) * 10.0 ** (s - 3) for s in range(6)]).cuda()
    whole = D.ops.orthogonalize(g.view(2, 3, rows, cols))
    assert whole.shape == (2, 3, rows, cols)
    one = D.ops.orthogonalize(g[4])
    assert far(whole.view(6, rows, cols)[4], one) <= 2 * bound(torch.float32, cols)   # other splits, other sums
    for steps, coefficients in [(1, DEFAULT), (2, (1.5, -0.5, 0.0)), (3, [(3.0, -3.2, 1.2), (2.0, -1.5, 0.5), (1.5, -0.5, 0.0)]), (12, (1.5, -0.5, 0.0)), (6, (1.6, -0.7, 0.02))]:
        got = D.ops.orthogonalize(g, steps=steps, coefficients=coefficients)
        want = definition(g, steps, coefficients)
        for z in range(6):
            assert far(got[z], want[z]) <= bound(torch.float32, cols), (steps, z)
    assert D.ops.orthogonalize(g[:0]).shape == (0, rows, cols) and D.ops.orthogonalize(g[:, :0]).shape == (6, 0, cols)
    assert torch.equal(D.ops.orthogonalize(g.transpose(1, 2).contiguous().transpose(1, 2)), D.ops.orthogonalize(g))


@pytest.mark.parametrize("cols", [16, 40])
def test_sizes_of_the_values(cols):
    g = spectrum("noise", 60, cols).cuda()
    want = definition(g)
    for scale in (1e-30, 1e-3, 1e3, 1e30):     # below eps the matrix is no longer brought to norm 1
        got = D.ops.orthogonalize(g * scale, eps=1e-35 if scale < 1e-7 else 1e-7)
        assert far(got, want) <= bound(torch.float32, cols) + 2.0 ** -22, scale
    assert not D.ops.orthogonalize(torch.zeros(60, cols, device="cuda")).any()
    tiny = g / g.norm() * 1e-9
    assert far(D.ops.orthogonalize(tiny), definition(tiny)) <= bound(torch.float32, cols) + 2.0 ** -22
    both = torch.stack([g, g, g])
    both[1, 5, 3] = float("inf")
    got = D.ops.orthogonalize(both)
    assert got[1].isnan().all() and torch.isfinite(got[0]).all() and torch.equal(got[0], got[2])
    both[1, 5, 3] = float("nan")
    assert D.ops.orthogonalize(both)[1].isnan().all()


def test_orthogonalize_refuses():
    g = torch.randn(4, 4, device="cuda")
    for bad in (dict(x=g.double()), dict(x=g[0]), dict(eps=0.0), dict(eps=float("inf")), dict(steps=0), dict(coefficients=(9.0, 9.0, 9.0))):
        with pytest.raises(ValueError):
            D.ops.orthogonalize(**{**dict(x=g), **bad})


def reference_step(w, g, m, lr, momentum, nesterov, decay):
    w, g, m = w.double(), g.double(), m.double()
    m = m + (1 - momentum) * (g - m)
    u = g + momentum * (m - g) if nesterov else m
    return w * (1 - lr * decay) - lr * math.sqrt(max(1.0, w.shape[0] / w.shape[1])) * definition(u), m


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("shapes", [[(500, 16)] * 3, [(100, 16), (0, 16), (33, 16), (7, 5), (64, 5)], [(40, 50), (50, 40), (40, 50), (300, 16), (40, 50)],
                                    [(100, 16)] * 40, [(20, 30)] * 20])
def test_muon_step(shapes, nesterov):
    g = torch.Generator().manual_seed(1)
    make = lambda: [torch.randn(*s, generator=g).cuda() for s in shapes]  # noqa: E731
    weights, momenta = make(), make()
    want = [(w.double(), m.double()) for w, m in zip(weights, momenta)]
    for _ in range(3):
        grads = make()
        D.ops.muon_step(weights, grads, momenta, lr=0.05, momentum=0.9, nesterov=nesterov, weight_decay=0.3)
        want = [reference_step(w, gr, m, 0.05, 0.9, nesterov, 0.3) if w.numel() else (w, m) for (w, m), gr in zip(want, grads)]
    for w, m, (rw, rm) in zip(weights, momenta, want):
        if not w.numel():
            continue
        # momenta: three roundings a step.  weights: those of three updates of norm sqrt(min(rows, cols)), and their own
        assert far(m, rm) <= 9 * 2.0 ** -24
        rate = 0.05 * math.sqrt(max(1.0, w.shape[0] / w.shape[1]))
        off = (w.double() - rw).norm().item()
        assert off <= 3 * rate * math.sqrt(min(w.shape)) * 1.2 * (bound(torch.float32, w.shape[1]) + 2.0 ** -20) + 9 * 2.0 ** -24 * rw.norm().item()


def test_muon_step_off_the_16_byte_units_and_in_a_graph():
    flat = torch.randn(3, 2000 * 16 + 1, generator=torch.Generator().manual_seed(2)).cuda()
    w, g, m = (flat[i, 1:].view(2000, 16) for i in range(3))
    assert w.data_ptr() % 16 == 4
    start = [v.clone() for v in (w, m)]
    want = reference_step(w, g, m, 0.1, 0.95, True, 0.0)
    D.ops.muon_step([w], [g], [m], lr=0.1)
    assert far(w, want[0]) <= 2.0 ** -21 and far(m, want[1]) <= 3 * 2.0 ** -24
    once = [v.clone() for v in (w, m)]
    graph, side = torch.cuda.CUDAGraph(), torch.randn(60, 70, device="cuda")
    buffers = [side.clone(), side * 0.1, side * 0.0]
    with torch.cuda.graph(graph):
        D.ops.muon_step([w, buffers[0]], [g, buffers[1]], [m, buffers[2]], lr=0.1)
    results = []
    for _ in range(2):
        for v, s in zip((w, m), start):
            v.copy_(s)
        for v, s in zip(buffers, (side, side * 0.1, side * 0.0)):
            v.copy_(s)
        graph.replay()
        results.append([v.clone() for v in (w, m, *buffers)])
    assert all(torch.equal(p, q) for p, q in zip(*results)) and torch.equal(results[0][0], once[0]) and torch.equal(results[0][1], once[1])


def test_muon_step_refuses():
    w = torch.randn(4, 4, device="cuda")
    for bad in (dict(grads=[w.half()]), dict(grads=[w[:2]]), dict(weights=[w.t()[:, :3].t()]), dict(momenta=[w]), dict(grads=[])):
        with pytest.raises(ValueError):
            D.ops.muon_step(**{**dict(weights=[w], grads=[w.clone()], momenta=[w.clone()], lr=0.1), **bad})
    with pytest.raises(ValueError, match="twice"):
        D.ops.muon_step([w, w], [w.clone()] * 2, [w.clone(), w.clone()], lr=0.1)


@pytest.mark.parametrize("cols", [4, 40])
def test_muon_step_refuses_shared_memory(cols):
    memory = torch.randn(40, cols, device="cuda")
    a, b, c, d, g = memory[:10], memory[5:15], memory[20:30], memory[30:], torch.randn(10, cols, device="cuda")
    before = memory.clone()
    for weights, grads, momenta in (([a, b], [g, g], [c, d]), ([a, c], [g, g], [d, b]), ([a], [b], [c]), ([a], [a], [c]), ([a], [g], [b]),
                                    ([c], [memory[29:39]], [a])):
        with pytest.raises((ValueError, RuntimeError), match="shares memory"):
            D.ops.muon_step(weights, grads, momenta, lr=0.1)
    assert torch.equal(memory, before)
    D.ops.muon_step([a, c], [g, g], [memory[10:20], d], lr=0.1)     # neighbours, and one gradient for two
    assert not torch.equal(memory[:10], before[:10]) and not torch.equal(memory[20:30], before[20:30])


def test_flat_muon_refuses_before_it_updates():
    model = torch.nn.Sequential(D.DenseLayer(8, 8), D.DenseLayer(8, 8))
    optimizer = FlatMuon(model.parameters(), lr=0.1)
    model(torch.randn(4, 8, device="cuda")).sum().backward()
    model[1].bias.grad = None
    before = optimizer.flat_param.clone(), optimizer.flat_momentum.clone()
    with pytest.raises(RuntimeError, match="vectors"):
        optimizer.step()
    assert torch.equal(optimizer.flat_param, before[0]) and torch.equal(optimizer.flat_momentum, before[1])


def network(seed=0):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Flatten(), D.DenseLayer(48, 120, activation="silu"), D.DenseLayer(120, 200, feature_major=True),
                               D.LogicLayer(200, 400), D.LogicLayer(400, 200), D.GroupSum(10, 5.0))


def batch(seed=0, n=96):
    g = torch.Generator().manual_seed(seed)
    return torch.rand(n, 48, generator=g).cuda(), torch.randint(0, 10, (n,), generator=g).cuda()


def test_network_of_dense_and_logic_layers_takes_the_steps_of_the_definition():
    """One step of every parameter: matrices by Muon from the gradients that the layers give, biases by Adam's first step."""
    model = network()
    x, y = batch()
    before = [p.detach().clone() for p in model.parameters()]
    plain = copy.deepcopy(model)
    torch.nn.functional.cross_entropy(plain(x), y).backward()
    grads = [p.grad.clone() for p in plain.parameters()]
    opt = FlatMuon(model.parameters(), lr=0.02, weight_decay=0.1, adam_lr=0.003)
    step = TrainStep(model, opt)
    step(x, y)
    for p, w, g in zip(model.parameters(), before, grads):
        if p.dim() == 2:
            want = reference_step(w, g, torch.zeros_like(w), 0.02, 0.95, True, 0.1)[0]
            # the same kernels gave both gradients; the loss came another way: 1e-5 of them, 3.9^5 times that at worst in weak directions
            assert (p.detach().double() - want).norm().item() <= 0.02 * math.sqrt(max(1, w.shape[0] / w.shape[1])) * math.sqrt(min(w.shape)) * 1e-2
        else:
            moved = g.abs() > 1e-3 * g.abs().max()
            want = w - 0.003 * g / (g.abs() + 1e-8)
            assert (p.detach() - want)[moved].abs().max().item() <= 2e-3 * 0.003
    step.close()


def test_network_in_a_captured_step_is_the_eager_one():
    x, y = batch()
    results = []
    for captured in (False, True):
        model = network()
        step = TrainStep(model, FlatMuon(model.parameters(), lr=0.02))
        if captured:
            step.capture(x, y, warmup=2)
            for _ in range(3):
                step(x, y)
        else:
            for _ in range(5):
                loss = step(x, y)
            assert math.isfinite(loss.item())
        results.append([p.detach().clone() for p in model.parameters()])
        step.close()
    assert all(torch.equal(p, q) for p, q in zip(*results))


def test_network_with_adam_and_packed_inference_behind_the_encoder():
    model = network()
    x, y = batch()
    step = TrainStep(model, FlatAdam(model.parameters(), lr=0.01))
    first, last = step(x, y).item(), None
    for _ in range(20):
        last = step(x, y).item()
    assert math.isfinite(first) and math.isfinite(last)
    step.close()
    model.eval()
    with torch.no_grad():
        encoded = model[:3](x)
        counts = model[3:](D.PackBitsTensor(encoded > 0.5, bit_count=32))
        assert torch.equal(counts.float(), (model[3:]((encoded > 0.5).float()) * 5.0).round())   # scores are counts over tau
        # weights that a step has changed are what packed inference sees
        model.train()
        opt = FlatMuon(model[3:].parameters(), lr=0.5)
        for p in model[3:].parameters():
            p.grad = torch.randn_like(p)
        model.eval()
        opt.step()
        counts = model[3:](D.PackBitsTensor(encoded > 0.5, bit_count=32))
        assert torch.equal(counts.float(), (model[3:]((encoded > 0.5).float()) * 5.0).round())   # scores are counts over tau


def test_flat_muon_state():
    model = network()
    x, y = batch()
    opt = FlatMuon(model.parameters(), lr=0.02)
    run = lambda m, o: (o.zero_grad(), torch.nn.functional.cross_entropy(m(x), y).backward(), o.step())  # noqa: E731
    for _ in range(2):
        run(model, opt)
    saved = copy.deepcopy((model.state_dict(), opt.state_dict()))
    other = network()
    for i in (3, 4):
        other[i].set_connections(*model[i].indices)
    other_opt = FlatMuon(other.parameters(), lr=0.02)
    other.load_state_dict(saved[0])
    other_opt.load_state_dict(saved[1])
    run(model, opt)
    run(other, other_opt)
    assert all(torch.equal(p, q) for p, q in zip(model.parameters(), other.parameters()))
    with pytest.raises(ValueError, match="dimensions"):
        FlatMuon([torch.nn.Parameter(torch.zeros(2, 2, 2, device="cuda"))])
    with pytest.raises(ValueError, match="float32"):
        FlatMuon([torch.nn.Parameter(torch.zeros(2, 2, device="cuda", dtype=torch.bfloat16))])
    # what has no gradient stays as it is
    frozen = [p.detach().clone() for p in model.parameters()]
    opt.zero_grad()
    opt.step()
    assert all(torch.equal(p, q) for p, q in zip(model.parameters(), frozen))


def test_offsets_behind_32_bits():
    rows, last = 140_000_000, slice(-1000, None)
    torch.manual_seed(6)
    w, g = torch.randn(rows, 16, device="cuda"), torch.randn(rows, 16, device="cuda")
    m, before = torch.zeros_like(g), w[last].double()
    gram = sum(part.double().t() @ part.double() for part in g.split(4_000_000))
    norm = gram.trace().sqrt()
    s, p = gram / norm ** 2, torch.eye(16, dtype=torch.float64, device="cuda")
    for _ in range(5):
        a, b, c = DEFAULT
        step = a * torch.eye(16, dtype=torch.float64, device="cuda") + b * s + c * s @ s
        p, s = p @ step, step @ s @ step
    want = g[last].double() / norm @ p
    assert far(D.ops.orthogonalize(g)[last], want) <= bound(torch.float32, 16)
    lr = 1.0
    D.ops.muon_step([w], [g], [m], lr=lr, momentum=0.5, nesterov=False)
    update = (before - w[last].double()) / (lr * math.sqrt(rows / 16))
    # the difference of two roundings of the weight (2^-24 of up to 6), over a rate of 3000 and entries of 1e-4
    assert far(m[last], 0.5 * g[last].double()) <= 2.0 ** -24 and far(update, want) <= bound(torch.float32, 16) + 2 * 2.0 ** -24 * 6 / 3000 / 8e-5
