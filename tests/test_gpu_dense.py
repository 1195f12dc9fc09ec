"""Dense layers against their definition in 64 bits, forward and backward."""
import math

import pytest
import torch

import difflogic_b200 as D
from difflogic_b200 import _native as N

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = [None, "relu", "sigmoid", "silu", "gelu"]


def definition(x, w, b, r, act):
    z = x @ w.t() if b is None else x @ w.t() + b
    s = torch.sigmoid(z)
    phi = torch.special.ndtr(z)
    y, slope = {None: (z, torch.ones_like(z)), "relu": (z.clamp(min=0), (z > 0).double()), "sigmoid": (s, s * (1 - s)),
                "silu": (z * s, s * (1 + z * (1 - s))),
                "gelu": (z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi))}[act]
    return z, (y if r is None else y + r), slope


def product_error(k):
    """Of a sum of k products, relative to the sum of their absolute values.  Large products are added 16 at a time, cut off at 2^-23 or
    better each time; fp32 planes are exact but for products below 2^-24 of the whole, three of them; what is taken out of tensor memory
    every 64 or 128 values is added up with half a rounding of 2^-23 each.  A product split along k adds up to 64 more."""
    return (k / 16 + k / 64 + 3 + 64) * 2.0 ** -23


def check(x, w, b, r, act, feature_major=False, gy=None, columns=None):
    t = x.dtype
    half = torch.finfo(t).eps / 2
    y = D.dense(x, w, b, residual=r, activation=act, feature_major=feature_major)
    assert y.dtype == t and y.shape == (x.shape[0], w.shape[0])
    X, W = x.detach().double(), w.detach().double()
    B, R = (None if v is None else v.detach().double() for v in (b, r))
    z, want, slope = definition(X, W, B, R, act)
    # sums, with the bias' rounding; activations have slopes of at most 1.13 and cost a few roundings in 32 bits of their own
    z_off = product_error(X.shape[1]) * (X.abs() @ W.abs().t()) + 2.0 ** -24 * z.abs()
    y_off = 1.13 * z_off + 2.0 ** -20 * (want - (0 if R is None else R)).abs() + 2.0 ** -24 * want.abs() + 1e-37
    smallest = {torch.float16: 2.0 ** -25, torch.bfloat16: 1e-38, torch.float32: 1e-38}[t]
    off = (y.detach().double() - want).abs()
    bound = y_off + half * (want.abs() + y_off) + smallest
    assert bool((off <= bound).all()), "y: %.3e over its bound" % (off - bound).max().item()
    if gy is None:
        return y
    leaves = [v for v in (x, w, b, r) if v is not None]
    grads = dict(zip([n for n, v in zip("xwbr", (x, w, b, r)) if v is not None], torch.autograd.grad(y, leaves, gy)))
    G = gy.double()
    gz = G * slope
    # the slope: its own roundings, those of z (second derivatives stay below 1.13), 11 bits where bf16 layers keep it in fp16; gz rounded once
    kept = (2.0 ** -11 if t == torch.bfloat16 else 0) + 2.0 ** -20
    jump = (z.abs() <= 2 * z_off).double() if act == "relu" else 0     # either side of relu's corner
    gz_off = G.abs() * (1.13 * z_off + kept * slope.abs() + (4e-12 if t == torch.bfloat16 else 0) + jump) + 2.0 ** -22 * G.abs() * (act is not None)
    in_product = gz_off + half * (gz.abs() + gz_off) + smallest
    want_g = {"x": gz @ W, "w": gz.t() @ X, "b": gz.sum(0)}
    offs = {"x": in_product @ W.abs() + product_error(W.shape[0]) * (gz.abs() @ W.abs()),
            "w": in_product.t() @ X.abs() + product_error(X.shape[0]) * (gz.abs().t() @ X.abs()),
            "b": gz_off.sum(0) + (X.shape[0] + 8) * 2.0 ** -24 * gz.abs().sum(0)}
    for n, o in offs.items():
        if n not in grads:
            continue
        assert grads[n].dtype == t and grads[n].shape == want_g[n].shape
        off = (grads[n].double() - want_g[n]).abs()
        bound = o + half * (want_g[n].abs() + o) + smallest
        assert bool((off <= bound).all()), "gradient of %s: %.3e over its bound" % (n, (off - bound).max().item())
    if r is not None:
        assert torch.equal(grads["r"], gy)
    return y


def make(rows, inner, cols, t, seed=0, bias=True, residual=False, grad=True):
    g = torch.Generator().manual_seed(seed)
    leaf = lambda v: v.to(t).cuda().requires_grad_(grad)  # noqa: E731
    x, w = leaf(torch.randn(rows, inner, generator=g)), leaf(torch.randn(cols, inner, generator=g) / math.sqrt(inner))
    return (x, w, leaf(torch.randn(cols, generator=g)) if bias else None, leaf(torch.randn(rows, cols, generator=g)) if residual else None,
            torch.randn(rows, cols, generator=g).to(t).cuda())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows, inner, cols", [(1, 1, 1), (1, 64, 64), (2, 17, 3), (3, 784, 100), (7, 100, 1000), (9, 33, 65), (17, 128, 2000), (64, 64, 64),
                                               (65, 63, 129), (128, 256, 128), (129, 257, 127), (255, 72, 513), (257, 130, 258), (300, 1000, 40),
                                               (1000, 24, 8), (513, 4100, 70)])
def test_sizes(rows, inner, cols, t):
    x, w, b, r, gy = make(rows, inner, cols, t, residual=rows % 2 == 0)
    check(x, w, b, r, "silu", gy=gy)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("feature_major", [False, True])
@pytest.mark.parametrize("rows", [6, 300])
def test_activations_and_layouts(act, feature_major, rows, t):
    x, w, b, r, gy = make(rows, 96, 136, t, seed=3, residual=True)
    y = check(x, w, b, r, act, feature_major, gy)
    assert (y.t() if feature_major else y).is_contiguous()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("columns", [64, 128, 256])
@pytest.mark.parametrize("rows, inner, cols", [(70, 200, 90), (260, 500, 300), (600, 130, 520), (5, 3000, 40)])
def test_every_tile(columns, rows, inner, cols, t):
    x, w, b, r, gy = make(rows, inner, cols, t, seed=4, residual=True)
    with N.tuning(N.TUNE_MATMUL_COLUMNS, columns):
        check(x, w, b, r, "gelu", gy=gy)
        with N.tuning(N.TUNE_MATMUL_SPLITS, 5):
            check(x, w, b, r, "sigmoid", feature_major=True, gy=gy)


@pytest.mark.parametrize("t", TYPES)
def test_inputs_as_they_lie(t):
    x, w, b, r, gy = make(40, 50, 70, t, seed=5, residual=True)
    transposed = x.detach().t().contiguous().t().requires_grad_()                       # as a logic layer returns it
    check(transposed, w, b, r, "silu", gy=gy)
    wide = torch.zeros(40, 64, dtype=t, device="cuda")
    wide[:, 3:53] = x.detach()
    check(wide[:, 3:53].requires_grad_(), w, b, r, "silu", gy=gy)                       # rows apart, off the 16-byte units
    check(wide[::2, 8:58].detach().requires_grad_(), w, b, r[::2].detach().requires_grad_(), "silu", gy=gy[::2])
    check(x[:1].detach().expand(40, 50).requires_grad_(), w, b, r, "silu", gy=gy)       # one row for all
    check(x, w, b, r.detach().t().contiguous().t().requires_grad_(), "silu", True, gy)
    check(x, w, b[:1].detach().expand(70).requires_grad_(), None, "silu", gy=gy)
    check(x, w, b, None, "silu", gy=gy.t().contiguous().t())
    check(x, w, b, None, "silu", gy=gy[:1].expand(40, 70))
    check(x, torch.cat([w, w], 1).detach()[:, 25:75].requires_grad_(), None, None, None, gy=gy)
    # more than two dimensions
    y = D.dense(x.detach().view(5, 8, 50), w, b, residual=r.detach().view(5, 8, 70), activation="relu")
    assert torch.equal(y.view(40, 70), D.dense(x, w, b, residual=r, activation="relu"))
    assert D.dense(x[0], w, b).shape == (70,)
    with pytest.raises(ValueError, match="feature_major"):
        D.dense(x.view(5, 8, 50), w, feature_major=True)
    with pytest.raises(ValueError, match="float32"):
        D.dense(x.double(), w.double())


@pytest.mark.parametrize("t", TYPES)
def test_empty_batch(t):
    x, w, b, _, _ = make(0, 5, 6, t)
    y = D.dense(x, w, b, activation="silu")
    assert y.shape == (0, 6)
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], torch.empty_like(y))
    assert gx.shape == (0, 5) and not gw.any() and not gb.any()


@pytest.mark.parametrize("t", TYPES)
def test_only_the_gradients_that_are_asked_for(t):
    x, w, b, r, gy = make(20, 30, 40, t, residual=True)
    whole = torch.autograd.grad(D.dense(x, w, b, residual=r, activation="silu"), [x, w, b, r], gy)
    for i in range(4):
        given = [v.detach().requires_grad_(i == j) for j, v in enumerate((x, w, b, r))]
        got, = torch.autograd.grad(D.dense(given[0], given[1], given[2], residual=given[3], activation="silu"), given[i], gy)
        assert torch.equal(got, whole[i])
    y = D.dense(x, w, b, residual=r, activation="silu")
    with torch.no_grad():
        assert torch.equal(D.dense(x, w, b, residual=r, activation="silu"), y)
    with pytest.raises(RuntimeError):   # differentiable once
        g, = torch.autograd.grad(y, x, gy, create_graph=True)
        g.sum().backward()


@pytest.mark.parametrize("act", ["sigmoid", "silu", "gelu"])
def test_gradients_against_differences(act):
    """Central differences of the fp32 layer along one direction at a time: truncation h^2 / 6 times a third derivative of a few, rounding
    of two sums over 2 h; h = 2^-7 leaves 2e-4 of either for outputs of size one, weighted with gy."""
    x, w, b, r, gy = make(6, 10, 12, torch.float32, seed=7, residual=True)
    grads = torch.autograd.grad(D.dense(x, w, b, residual=r, activation=act), [x, w, b, r], gy)
    h = 2.0 ** -7
    g = torch.Generator().manual_seed(8)
    for i, v in enumerate((x, w, b, r)):
        step = torch.randn(v.shape, generator=g).cuda()
        step /= step.norm()
        at = []
        for sign in (1, -1):
            given = [p.detach() + (sign * h * step if j == i else 0) for j, p in enumerate((x, w, b, r))]
            at.append((D.dense(given[0], given[1], given[2], residual=given[3], activation=act).double() * gy.double()).sum())
        slope = (at[0] - at[1]) / (2 * h)
        assert abs((slope - (grads[i].double() * step.double()).sum()).item()) <= 1e-3 * gy.double().norm().item()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_far_out(act, t):
    """Values where exponentials overflow, and infinities: limits, not undefined values."""
    z = torch.tensor([-3e38 if t != torch.float16 else -6e4, -1e4, -100.0, -20.0, -0.0, 0.0, 20.0, 100.0, 1e4, 3e38 if t != torch.float16 else 6e4])
    x, w = z.to(t).cuda().view(-1, 1).requires_grad_(), torch.ones(1, 1, dtype=t, device="cuda")
    y = D.dense(x, w, activation=act)
    g, = torch.autograd.grad(y, x, torch.ones_like(y))
    _, want, slope = definition(x.detach().double(), w.double(), None, None, act)
    half = torch.finfo(t).eps / 2
    for got, ref in ((y.double(), want), (g.double(), slope)):
        ref = torch.where(ref.isnan(), torch.zeros_like(ref), ref)       # the definition's inf * 0 far out
        assert torch.isfinite(got).all()
        assert torch.allclose(got, ref, rtol=half + 2.0 ** -10, atol=1e-4), (act, t, got, ref)
    if t != torch.float32:
        x = torch.tensor([[float("inf")], [float("-inf")], [float("nan")], [1.0]], dtype=t, device="cuda")
        y = D.dense(x, w, activation=act)
        top = 1.0 if act == "sigmoid" else float("inf")
        bottom = float("-inf") if act is None else 0.0
        assert y[0].item() == top and y[1].item() == bottom and math.isnan(y[2].item()) and math.isfinite(y[3].item())


def test_an_infinite_fp32_operand_reaches_its_own_results_only():
    x, w, b, _, _ = make(300, 40, 50, torch.float32, grad=False)
    clean = D.dense(x, w, b)
    x[7, 3] = float("inf")
    x[9, 0] = float("nan")
    y = D.dense(x, w, b)
    keep = [i for i in range(300) if i not in (7, 9)]
    assert torch.equal(y[keep], clean[keep]) and not torch.isfinite(y[[7, 9]]).any()


def test_large_and_small_fp32_values():
    """The three planes of a value cover fp32's range: products near its ends keep their 24 bits."""
    x = torch.tensor([[3.4e38, 0.0], [1e-30, 0.0], [1.2345678e-38, 0.0], [3.0, 2.9999998]], device="cuda")
    w = torch.tensor([[1.0, 0.0], [0.5, 0.0], [1.0, -1.0]], device="cuda")
    want = x.double() @ w.double().t()
    y = D.dense(x, w).double()
    assert torch.isfinite(y).all()
    assert ((y - want).abs() <= 2.0 ** -22 * (x.double().abs() @ w.double().abs().t()) + 1e-40).all()


def test_a_weight_used_twice():
    x, w, b, _, _ = make(9, 16, 16, torch.float32)
    y = D.dense(D.dense(x, w, b, activation="silu"), w, b, activation="silu")
    y.sum().backward()
    X, W, B = (v.detach().double().requires_grad_() for v in (x, w, b))
    Y = torch.nn.functional.silu(torch.nn.functional.silu(X @ W.t() + B) @ W.t() + B)
    Y.sum().backward()
    for a, ref in ((x, X), (w, W), (b, B)):
        assert torch.allclose(a.grad.double(), ref.grad, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("t", TYPES)
def test_same_result_every_time_and_on_other_streams_and_in_graphs(t):
    x, w, b, r, gy = make(200, 1000, 90, t, residual=True)
    run = lambda: [v.clone() for v in (lambda y: (y.detach(), *torch.autograd.grad(y, [x, w, b], gy)))(D.dense(x, w, b, residual=r, activation="gelu"))]  # noqa: E731
    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(first, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    other = torch.cuda.CUDAGraph()
    with torch.cuda.graph(other):
        more = run()
    with torch.no_grad():
        x.copy_(x * 0.5)
    want = run()
    for _ in range(2):
        graph.replay()
        other.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) and torch.equal(p, s) for p, q, s in zip(want, captured, more))
    assert N.lib().dl_async_error() == 0


def test_layer_feeds_logic_layers_without_a_copy():
    torch.manual_seed(0)
    layer = D.DenseLayer(50, 200, activation="sigmoid", feature_major=True)
    model = torch.nn.Sequential(layer, D.LogicLayer(200, 400), D.LogicLayer(400, 200), D.GroupSum(10, 3.0))
    x = torch.rand(64, 50, device="cuda")
    h = layer(x)
    assert h.t().is_contiguous() and 0 <= h.min().item() and h.max().item() <= 1
    loss = torch.nn.functional.cross_entropy(model(x), torch.arange(64, device="cuda") % 10)
    loss.backward()
    reference = torch.nn.Sequential(D.DenseLayer(50, 200, device="cpu"), D.LogicLayer(200, 400, device="cpu"), D.LogicLayer(400, 200, device="cpu"),
                                    D.GroupSum(10, 3.0, device="cpu")).double()
    with torch.no_grad():
        for mine, ref in zip(model, reference):
            for p, q in zip(mine.parameters(), ref.parameters()):
                q.copy_(p.cpu())
        for i in (1, 2):
            reference[i].set_connections(*(v.cpu() for v in model[i].indices))
    torch.nn.functional.cross_entropy(reference(x.cpu().double()), torch.arange(64) % 10).backward()
    for p, q in zip(model.parameters(), reference.parameters()):
        # the framework's own bound for gradients through logic layers
        assert (p.grad.cpu().double() - q.grad).abs().max().item() <= 1e-4 * q.grad.abs().max().item()


def test_capture_beside_an_eager_graph_is_refused():
    x, w, b = torch.randn(40, 16, device="cuda"), torch.randn(24, 16, device="cuda", requires_grad=True), torch.randn(24, device="cuda", requires_grad=True)
    gy = torch.randn(40, 24, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            want = torch.autograd.grad(D.dense(x, w, b, activation="relu"), (w, b), gy)
    torch.cuda.current_stream().wait_stream(side)
    alive = D.dense(x, w, b, activation="relu")
    with pytest.raises(RuntimeError, match="alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            D.dense(x, w, b, activation="relu")
    with torch.no_grad(), torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
        D.dense(x, w, b)                      # no graph of its own
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = torch.autograd.grad(D.dense(x, w, b, activation="relu"), (w, b), gy)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))


def test_capture_beside_a_warm_up_on_another_stream():
    x, w = torch.randn(40, 16, device="cuda"), torch.randn(24, 16, device="cuda", requires_grad=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            w.grad = None
            loss = D.dense(x, w, activation="silu").sum()
            loss.backward()
    torch.cuda.current_stream().wait_stream(side)
    want = w.grad.clone()
    w.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):        # on a stream of its own, `loss` alive
        D.dense(x, w, activation="silu").sum().backward()
    w.grad.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(w.grad, want) and bool(torch.isfinite(loss.detach()))


def whole_numbers(*size):
    """-1, 0 and 1: sums of products are exact, and so is what they round to."""
    return torch.empty(*size, dtype=torch.bfloat16, device="cuda").random_(-1, 2).requires_grad_()


@pytest.mark.parametrize("rows, inner, cols", [(70000, 16, 33000), (66000, 33000, 24), (3, 33000, 66000)])
def test_offsets_behind_32_bits(rows, inner, cols):
    torch.manual_seed(5)
    x, w, b, r = whole_numbers(rows, inner), whole_numbers(cols, inner), whole_numbers(cols), whole_numbers(rows, cols)
    gy = whole_numbers(rows, cols).detach()
    y = D.dense(x, w, b, residual=r, activation="relu")
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), gy)
    last = slice(-min(rows, 300), None), slice(-40, None)
    with torch.no_grad():
        z = x[last[0]].double() @ w.double().t() + b.double()
        assert torch.equal(y[last[0]], (z.clamp(min=0) + r[last[0]].double()).bfloat16())
        gz = gy[last[0]].double() * (z > 0)
        assert torch.equal(gx[last[0]], (gz @ w.double()).bfloat16())
        del z, gz
        z = torch.cat([part.double() @ w[last[1]].double().t() for part in x.split(4096)]) + b[last[1]].double()
        gz = gy[:, last[1]].double() * (z > 0)
        assert torch.equal(gw[last[1], -40:], (gz.t() @ x[:, -40:].double()).bfloat16()) and torch.equal(gb[last[1]], gz.sum(0).bfloat16())
