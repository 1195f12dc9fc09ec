"""Operators for dense layers beside logic layers and for training both with orthogonalised updates, as cases to be timed.

Three operators, each in a plain form (elementary torch operations in 32 bits, `own` false) and as the package's calls (`own` true):

dense  y = act(x w^T + b) + residual, the product with bias, activation and residual in its epilogue; with "train" also the gradients of
       x, w, b and the residual for a given gradient of y.
ns     X <- G / |G|_F, then `steps` times X <- a X + b (X X^T) X + c (X X^T)^2 X: the orthogonalised update of a matrix.
muon   One optimizer step of all matrices of a network: momentum, orthogonalisation, decayed and scaled update, in place.
"""
import math

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one sample through a dense layer while serving: latency, the weights are read once
        dict(name="dense_one_row_bf16", op="dense", rows=1, inner=2048, cols=2048, type="bf16", act="relu", residual=False, train=False),
        # a handful of images through an encoder in front of a logic network, in the layout that the logic layers read
        dict(name="dense_few_rows_fp32", op="dense", rows=5, inner=784, cols=16000, type="fp32", act="sigmoid", residual=False, train=False),
        # training step of that encoder at the training batch of the logic networks
        dict(name="dense_train_encoder_fp32", op="dense", rows=128, inner=784, cols=8000, type="fp32", act="sigmoid", residual=False, train=True),
        # odd sizes: images without one pixel, a number of classes and a batch that are no multiple of anything
        dict(name="dense_train_odd_fp16", op="dense", rows=1001, inner=783, cols=2001, type="fp16", act="gelu", residual=False, train=True),
        # a residual block of a wide network at a large batch: the largest dense step
        dict(name="dense_train_residual_bf16", op="dense", rows=8192, inner=4096, cols=4096, type="bf16", act="silu", residual=True, train=True),
        # the gradient of one logic layer's weights: many rows of 16 gates
        dict(name="ns_logic_16000", op="ns", batch=1, rows=16000, cols=16, type="fp32"),
        # the two matrices of an encoder, odd sizes, wide
        dict(name="ns_wide_odd_bf16", op="ns", batch=2, rows=783, cols=2001, type="bf16"),
        # matrices of a small dense network, together
        dict(name="ns_square_1024_bf16", op="ns", batch=4, rows=1024, cols=1024, type="bf16"),
        # one matrix of a wide dense network
        dict(name="ns_square_4096_fp32", op="ns", batch=1, rows=4096, cols=4096, type="fp32"),
        # one step of a logic network of 784 -> 5 x 16000
        dict(name="muon_logic_5x16000", op="muon", logic=5, width=16000, dense=0, inner=0, cols=0),
        # one step of a wide logic network, 9216 -> 4 x 128000
        dict(name="muon_logic_4x128000", op="muon", logic=4, width=128000, dense=0, inner=0, cols=0),
        # a network of two dense matrices and logic layers behind them
        dict(name="muon_encoder_logic", op="muon", logic=4, width=8000, dense=2, inner=784, cols=2000),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["dense", "dense", "ns", "ns", "muon"])
    if op == "dense":
        train = rng.random() < 0.6
        type_ = rng.choice(["fp32", "bf16", "fp16"])
        inner, cols = _spread(rng, 16, 4096), _spread(rng, 16, 16000)
        rows = _spread(rng, 1, min(8192, max(1, 3 * 10 ** 10 // (inner * cols))))
        # the gradient of relu jumps at zero, where 32 bits of two orders of summation do not agree: not among the trained ones of that type
        act = rng.choice(["none", "sigmoid", "silu", "gelu"] + ([] if train and type_ == "fp32" else ["relu"]))
        return dict(op=op, rows=rows, inner=inner, cols=cols, type=type_, act=act, residual=rng.random() < 0.4, train=train)
    if op == "ns":
        if rng.random() < 0.4:
            return dict(op=op, batch=rng.choice([1, 1, 2, 5]), rows=_spread(rng, 500, 128000), cols=16, type=rng.choice(["fp32", "fp32", "bf16"]))
        rows, cols = _spread(rng, 20, 4096), _spread(rng, 20, 4096)
        batch = max(1, min(rng.choice([1, 1, 2, 4, 7]), 4096 * 4096 // (rows * cols)))
        return dict(op=op, batch=batch, rows=rows, cols=cols, type=rng.choice(["fp32", "bf16", "fp16"]))
    dense = rng.choice([0, 0, 1, 2, 3])
    return dict(op=op, logic=rng.randint(1, 6), width=_spread(rng, 500, 64000), dense=dense, inner=_spread(rng, 50, 1500) if dense else 0,
                cols=_spread(rng, 50, 2000) if dense else 0)


def _matrix(gen, *shape):
    """What a layer's gradient looks like: a few strong directions under noise of about the same weight."""
    *batch, rows, cols = shape
    rank = max(1, min(rows, cols) // 8)
    left = torch.randn(*batch, rows, rank, generator=gen, device="cuda")
    right = torch.randn(*batch, rank, cols, generator=gen, device="cuda")
    fall = torch.arange(1, rank + 1, device="cuda", dtype=torch.float32) ** -0.5
    strong = (left * fall) @ right
    noise = torch.randn(*shape, generator=gen, device="cuda")
    return (strong * (noise.norm() / strong.norm()) + noise) * 1e-3


def _logic(gen, *shape):
    """The gradient of a logic layer's weights: 16 gates that a softmax ties together, neurons of very different weight."""
    g = torch.randn(*shape, generator=gen, device="cuda") * torch.exp(torch.randn(*shape[:-1], 1, generator=gen, device="cuda"))
    p = torch.softmax(torch.randn(*shape, generator=gen, device="cuda"), -1)
    return p * (g - (p * g).sum(-1, keepdim=True)) * 1e-3


def _shapes(case):
    return ([(case["cols"], case["inner"] if i == 0 else case["cols"]) for i in range(case["dense"])]
            + [(case["width"], 16) for _ in range(case["logic"])])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    if case["op"] == "dense":
        t, rows, inner, cols = TYPES[case["type"]], case["rows"], case["inner"], case["cols"]
        leaf = lambda v: v.to(t).requires_grad_(case["train"])  # noqa: E731
        return dict(case=case, x=leaf(rand(rows, inner)), w=leaf(rand(cols, inner) / math.sqrt(inner)), b=leaf(0.1 * rand(cols)),
                    residual=leaf(rand(rows, cols)) if case["residual"] else None, gy=rand(rows, cols).to(t) if case["train"] else None)
    if case["op"] == "ns":
        make = _logic if case["cols"] == 16 else _matrix
        return dict(case=case, g=make(gen, case["batch"], case["rows"], case["cols"]).to(TYPES[case["type"]]))
    grads, momenta, weights = [], [], []
    for rows, cols in _shapes(case):
        make = _logic if cols == 16 else _matrix
        grads.append(make(gen, rows, cols))
        momenta.append(make(gen, rows, cols) * 0.5 + grads[-1] * 0.5)
        weights.append(rand(rows, cols) if cols == 16 else rand(rows, cols) / math.sqrt(cols))
    return dict(case=case, weights=weights, grads=grads, momenta=momenta)


# -- the plain forms --------------------------------------------------------------------------------------------------------------

def _activation(z, act):
    """act(z) and its derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z * (z > 0), (z > 0).to(z.dtype)
    if act == "gelu":
        phi = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    s = 1 / (1 + torch.exp(-z))
    if act == "sigmoid":
        return s, s * (1 - s)
    return z * s, s * (1 + z * (1 - s))


@torch.no_grad()
def _dense_plain(state):
    case, t = state["case"], state["x"].dtype
    x, w, b = state["x"].float(), state["w"].float(), state["b"].float()
    y, slope = _activation(x @ w.t() + b, case["act"])
    if state["residual"] is not None:
        y = y + state["residual"].float()
    if not case["train"]:
        return y.to(t)
    gz = state["gy"].float() * slope
    grads = [gz @ w, gz.t() @ x, gz.sum(0)]
    return [y.to(t)] + [g.to(t) for g in grads] + ([state["gy"]] if state["residual"] is not None else [])


def _orthogonal_plain(g):
    a, b, c = COEFFICIENTS
    x = g.float()
    if x.shape[-2] > x.shape[-1]:
        x = x.transpose(-2, -1)
    x = x / x.square().sum((-2, -1), keepdim=True).sqrt().clamp(min=1e-7)
    for _ in range(STEPS):
        gram = x @ x.transpose(-2, -1)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x if g.shape[-2] <= g.shape[-1] else x.transpose(-2, -1)


@torch.no_grad()
def _muon_plain(state):
    for w, g, m in zip(state["weights"], state["grads"], state["momenta"]):
        m.copy_(m + (1 - MOMENTUM) * (g - m))
        update = _orthogonal_plain(g + MOMENTUM * (m - g))
        w.copy_(w * (1 - LR * DECAY) - (LR * math.sqrt(max(1.0, w.shape[0] / w.shape[1]))) * update)
    return state["weights"] + state["momenta"]


def run(state):
    case = state["case"]
    if not own:
        if case["op"] == "dense":
            return _dense_plain(state)
        if case["op"] == "ns":
            return _orthogonal_plain(state["g"]).to(state["g"].dtype).contiguous()
        return _muon_plain(state)
    import difflogic_b200 as D
    if case["op"] == "dense":
        x, w, b, residual = state["x"], state["w"], state["b"], state["residual"]
        y = D.dense(x, w, b, residual=residual, activation=case["act"])
        if not case["train"]:
            return y
        leaves = [x, w, b] + ([residual] if residual is not None else [])
        return [y.detach()] + list(torch.autograd.grad(y, leaves, state["gy"]))
    if case["op"] == "ns":
        return D.ops.orthogonalize(state["g"], steps=STEPS, coefficients=COEFFICIENTS)
    D.ops.muon_step(state["weights"], state["grads"], state["momenta"], lr=LR, momentum=MOMENTUM, weight_decay=DECAY, steps=STEPS,
                    coefficients=COEFFICIENTS)
    return state["weights"] + state["momenta"]


# -- what a pass cannot do without ------------------------------------------------------------------------------------------------

def _orthogonal_flops(rows, cols):
    """The Gram matrix and its square are symmetric: half their products.  Either the matrix itself is iterated, or its Gram matrix,
    which the matrix is multiplied with at the end."""
    r, m = min(rows, cols), max(rows, cols)
    return min(STEPS * (m * r * (r + 1) + r * r * (r + 1) + 2 * m * r * r), m * r * (r + 1) + STEPS * 4 * r * r * (r + 1) + 2 * m * r * r)


def work(case):
    if case["op"] == "dense":
        rows, inner, cols, size = case["rows"], case["inner"], case["cols"], 4 if case["type"] == "fp32" else 2
        values = rows * inner + cols * inner + cols + rows * cols * (2 if case["residual"] else 1)
        if case["train"]:
            values += rows * cols + rows * inner + cols * inner + cols
        return dict(bytes=values * size, flops=2 * rows * inner * cols * (3 if case["train"] else 1))
    if case["op"] == "ns":
        size = 4 if case["type"] == "fp32" else 2
        return dict(bytes=2 * size * case["batch"] * case["rows"] * case["cols"], flops=case["batch"] * _orthogonal_flops(case["rows"], case["cols"]))
    shapes = _shapes(case)
    return dict(bytes=sum(5 * 4 * r * c for r, c in shapes), flops=sum(_orthogonal_flops(r, c) for r, c in shapes))


# -- the definitions in 64 bits ---------------------------------------------------------------------------------------------------

def _orthogonal_exact(g):
    """The iteration is X <- X q(X^T X) with a polynomial q, so that X stays G times a polynomial of G^T G: here that one is iterated."""
    a, b, c = COEFFICIENTS
    g = g.double()
    tall = g.shape[-2] >= g.shape[-1]
    x = g if tall else g.mT
    x = x / torch.linalg.matrix_norm(x, keepdim=True).clamp(min=1e-7)
    gram = x.mT @ x
    eye = torch.eye(gram.shape[-1], dtype=torch.float64, device=g.device)
    product = eye.expand_as(gram)
    for _ in range(STEPS):
        q = a * eye + gram @ (b * eye + c * gram)
        product = product @ q
        gram = q @ gram @ q
    x = x @ product
    return x if tall else x.mT


@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "ns":
        return _orthogonal_exact(state["g"]).contiguous()
    if case["op"] == "muon":
        weights, momenta = [], []
        for w, g, m in zip(state["weights"], state["grads"], state["momenta"]):
            w, g, m = w.double(), g.double(), m.double()
            m = MOMENTUM * m + (1 - MOMENTUM) * g
            o = _orthogonal_exact((1 - MOMENTUM) * g + MOMENTUM * m)
            momenta.append(m)
            weights.append(w - LR * DECAY * w - LR * max(1.0, w.shape[0] / w.shape[1]) ** 0.5 * o)
        return weights + momenta
    x, w, b = (state[k].double() for k in ("x", "w", "b"))
    z = torch.addmm(b, x, w.t())
    act = case["act"]
    logistic = torch.special.expit(z)
    y = {"none": lambda: z, "relu": lambda: z.clamp(min=0), "sigmoid": lambda: logistic, "silu": lambda: z * logistic,
         "gelu": lambda: z * torch.special.ndtr(z)}[act]()
    if state["residual"] is not None:
        y = y + state["residual"].double()
    if not case["train"]:
        return y
    slope = {"none": lambda: torch.ones_like(z), "relu": lambda: torch.heaviside(z, torch.zeros_like(z)), "sigmoid": lambda: logistic - logistic ** 2,
             "silu": lambda: logistic + z * logistic - z * logistic ** 2,
             "gelu": lambda: torch.special.ndtr(z) + z / math.sqrt(2 * math.pi) * torch.exp(-z * z / 2)}[act]()
    gz = slope * state["gy"].double()
    return [y, gz @ w, gz.t() @ x, gz.sum(0)] + ([state["gy"].double()] if state["residual"] is not None else [])
