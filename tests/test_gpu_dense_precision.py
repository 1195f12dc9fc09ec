"""What the products of fp32 dense layers keep of their 24 bits, on the tensor cores (33 samples and more) and without them.

Operands are made so that one of the planes' products alone carries the answer, or errors are compared in the mean over many results, where
one-sided ones stay and others do not."""
import math

import pytest
import torch

import difflogic_b200 as D

pytestmark = pytest.mark.gpu


def grads(x, w, gy):
    """y and the gradients of a dense layer without an activation: y = x w^T, gx = gy w, gw = gy^T x."""
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    y = D.dense(x, w)
    return (y.detach(), *torch.autograd.grad(y, (x, w), gy))


# (left operand, right operand) along the sum: their product is exact, of a few bits, and comes from one product of planes: of hi = 8 bits,
# mid = the next 8, lo = the last 8.  m = 2^-9 lies in mid, l = 2^-18 beside a mid in lo.
M, L = 2.0 ** -9, 2.0 ** -18
CARRIERS = {"hi hi": ([1.5, 0.0], [1.25, 0.0]), "mid hi": ([1 + M, 1.0], [1.0, -1.0]), "hi mid": ([1.0, -1.0], [1 + M, 1.0]),
            "lo hi": ([1 + M + L, 1 + M], [1.0, -1.0]), "hi lo": ([1.0, -1.0], [1 + M + L, 1 + M]),
            "mid mid": ([1 + M, 1 + M, 1.0, 1.0], [1 + M, -1.0, -(1 + M), 1.0])}


@pytest.mark.parametrize("carrier", sorted(CARRIERS))
@pytest.mark.parametrize("batch, inner, outer", [(40, 4, 8), (40, 64, 64), (130, 70, 300), (300, 520, 136)])
def test_every_product_of_planes_is_there(batch, inner, outer, carrier):
    left, right = CARRIERS[carrier]
    want = sum(a * b for a, b in zip(left, right))      # exact in 64 bits
    assert want != 0 and all(torch.tensor(v).item() == v for v in left + right)

    def matrices(k, n, m):
        a, b = torch.zeros(n, k), torch.zeros(m, k)
        at = [(7 * j) % k for j in range(len(left))] if k > 21 else list(range(len(left)))
        for j, p in enumerate(at):
            a[:, p], b[:, p] = left[j], right[j]
        # rows of their own power of two each
        return a * 2.0 ** (torch.arange(n) % 7 - 3.0)[:, None], b * 2.0 ** (torch.arange(m) % 5 - 2.0)[:, None]

    # forward: summed over the inputs
    a, b = matrices(inner, batch, outer)
    y = D.dense(a.cuda(), b.cuda())
    assert torch.equal(y.cpu().double(), want * (2.0 ** (torch.arange(batch) % 7 - 3.0)[:, None] * 2.0 ** (torch.arange(outer) % 5 - 2.0)[None]).double())
    # the input's gradient: gy [batch][outer] times w [outer][inner], summed over the outputs
    a, b = matrices(outer, batch, inner)
    gx = grads(torch.zeros(batch, inner, device="cuda"), b.t().contiguous().cuda(), a.cuda())[1]
    assert torch.equal(gx.cpu().double(), want * (2.0 ** (torch.arange(batch) % 7 - 3.0)[:, None] * 2.0 ** (torch.arange(inner) % 5 - 2.0)[None]).double())
    # the weight's: gy^T [outer][batch] times x [batch][inner], summed over the batch
    a, b = matrices(batch, outer, inner)
    gw = grads(b.t().contiguous().cuda(), torch.zeros(outer, inner, device="cuda"), a.t().contiguous().cuda())[2]
    assert torch.equal(gw.cpu().double(), want * (2.0 ** (torch.arange(outer) % 7 - 3.0)[:, None] * 2.0 ** (torch.arange(inner) % 5 - 2.0)[None]).double())


@pytest.mark.parametrize("batch, inner, outer", [(33, 64, 64), (65, 63, 129), (128, 784, 400), (300, 1000, 140), (1000, 130, 257)])
def test_mean_error_of_the_planes(batch, inner, outer):
    """Random signs.  Over blocks of 128 products the tensor cores' sums cut off less than 2^-23 of the sum's size, 8 times at most; a
    block's sum of 128 random products is sqrt(128 / k) of the whole, and k / 128 blocks add up like that again: 8 * 2^-23 of the
    result's root mean square, all of it in one direction.  Beside that, 3 products below 2^-24 left out, of random signs; up to 64 roundings
    of the blocks' sums to 24 bits, of random signs.  Leaving out a product of planes that counts would be 2^-18 and more."""
    gen = torch.Generator().manual_seed(batch)
    x, w, gy = (torch.randn(*s, generator=gen).cuda() for s in ((batch, inner), (outer, inner), (batch, outer)))
    got = grads(x, w, gy)
    X, W, G = x.double(), w.double(), gy.double()
    for g, want in zip(got, (X @ W.t(), G @ W, G.t() @ X)):
        rms = lambda v: v.double().square().mean().sqrt().item()  # noqa: E731
        assert rms(g.double() - want) <= (8 * 2.0 ** -23 + 8 * 2.0 ** -24) * rms(want)


@pytest.mark.parametrize("rows", [4, 40])
def test_values_of_any_size(rows):
    """From the largest number to the smallest ones: 2^-21 of each product (without the tensor cores' planes; below) and as much again for
    three sums that are cut off, or what planes of 2^-133, the smallest bf16 number, leave of it.  Values are not cut off at the largest
    bf16, a number smaller than fp32's largest."""
    top = torch.finfo(torch.float32).max
    x = torch.zeros(rows, 3)
    values = [top, -top, 3.4e38, 3.4027e38, 1e-30, 1.2345678e-38, -2.0 ** -110 * 1.2345678, 2.0 ** -126, 7e-39, 1e-41, 2.0 ** -149, 1.2345678]
    for i in range(rows):
        x[i, i % 3] = values[i % len(values)]
        x[i, (i + 1) % 3] = values[i % len(values)] * -0.37
    x, w = x.cuda(), torch.tensor([[1.0, 0.0, 0.0], [0.0, 0.5, 0.25], [1.0, 1.0, 1.0], [0.1234567, -0.7654321, 0.3333333]], device="cuda")
    want = x.double() @ w.double().t()
    got = D.dense(x, w).double()
    assert bool(torch.isfinite(got).all())
    sizes = x.double().abs() @ w.double().abs().t()
    assert bool(((got - want).abs() <= 2.0 ** -20 * sizes + 3 * 2.0 ** -134 * w.double().abs().sum(1) + 2.0 ** -149).all())


@pytest.mark.parametrize("rows", [8, 16, 32, 40])
def test_single_products(rows):
    """One input: y = x w, with nothing added up.  Without the tensor cores' planes a value is 11 bits, rounded to nearest, and a rest of
    which 11 bits count, so that half of the last bit is lost of a quarter of the values: 2^-23 of an operand at most and of either sign,
    and 2^-24 of the product for the two rests' product, 2^-22 at its worst, of either sign.  The sum of the three products is cut off
    at its last bit, three times, 2^-23 each at most; all but the last time that is of a sum 2^-11 as large."""
    gen = torch.Generator().manual_seed(rows)
    x, w = 1 + torch.rand(rows, 1, generator=gen), 1 + torch.rand(8192, 1, generator=gen)
    worst = torch.tensor([0x3f801fff, 0x3f800fff, 0x3f801000, 0x3f801001, 0x3fffffff, 0x3f99a000, 0x3f99999a, 0x3f99afff], dtype=torch.int32)
    x[:8, 0] = worst.view(torch.float32)
    w[:8, 0] = worst.view(torch.float32)
    x, w = x.cuda(), w.cuda()
    want = x.double() @ w.double().t()
    off = (D.dense(x, w).double() - want) / want
    assert off.abs().max().item() <= 2 * 2.0 ** -23 + 2.0 ** -22 + 2 * 2.0 ** -23
    # one-sided is the last cut alone, half of 2^-23 on average
    assert abs(off.mean().item()) <= 2.0 ** -24 + 2.0 ** -23 / math.sqrt(off.numel() / 1000)


@pytest.mark.parametrize("rows", [8, 32])
def test_inputs_that_are_not_finite(rows):
    """Results that a NaN or an infinity enters are not finite, others are what they were."""
    gen = torch.Generator().manual_seed(rows)
    x, w = torch.randn(rows, 50, generator=gen).cuda(), torch.randn(24, 50, generator=gen).cuda()
    clean = D.dense(x, w)
    nans = torch.tensor([0x7fc00000, 0x7f800001, 0x7fffffff, -1, 0x7fbfffff, 0x7f800000, -0x00800000], dtype=torch.int32).view(torch.float32)
    for i, v in enumerate(nans):
        bad = x.clone()
        bad[i, 3 * i] = v.item() if math.isinf(v) else 0
        bad.view(torch.int32)[i, 3 * i] = nans.view(torch.int32)[i].item()
        y = D.dense(bad, w)
        keep = [j for j in range(rows) if j != i]
        assert not torch.isfinite(y[i]).any() and torch.equal(y[keep], clean[keep])
        bad = w.clone()
        bad.view(torch.int32)[i, 3 * i] = nans.view(torch.int32)[i].item()
        y = D.dense(x, bad)
        keep = [j for j in range(24) if j != i]
        assert not torch.isfinite(y[:, i]).any() and torch.equal(y[:, keep], clean[:, keep])


@pytest.mark.parametrize("act", [None, "relu", "sigmoid", "silu", "gelu"])
@pytest.mark.parametrize("rows", [10, 40])
def test_activations_far_out_of_planes(act, rows):
    """Pre-activations where exponentials overflow and planes are cut off, one input and a weight of 1: limits, not undefined values.  An
    activation and its derivative cost a few roundings in 32 bits, relative to values of at most 1.13 |z|; sigmoids' derivatives s (1 - s) lose
    what 1 - s rounds away, 2^-24."""
    z = torch.tensor([torch.finfo(torch.float32).max, torch.finfo(torch.float32).min, 3e38, -3e38, -1e4, -100.0, -20.0, -0.0, 20.0, 1e4])
    x, w = z.repeat(rows // 10).cuda().view(-1, 1).requires_grad_(), torch.ones(1, 1, device="cuda")
    y = D.dense(x, w, activation=act)
    g, = torch.autograd.grad(y, x, torch.ones_like(y))
    v = x.detach().double()
    s, phi = torch.sigmoid(v), torch.special.ndtr(v)
    density = torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    far = v.abs() > 1e3                       # infinity times zero
    want, slope = {None: (v, torch.ones_like(v)), "relu": (v.clamp(min=0), (v > 0).double()), "sigmoid": (s, s * (1 - s)),
                   "silu": (v * s, s + torch.where(far, 0, v * s * (1 - s))), "gelu": (v * phi, phi + torch.where(far, 0, v * density))}[act]
    assert bool(torch.isfinite(y).all() & torch.isfinite(g).all())
    assert bool(((y.double() - want).abs() <= 2.0 ** -19 * want.abs() + 1e-6).all()) and bool(((g.double() - slope).abs() <= 2.0 ** -19 * slope + 2e-6).all())
