"""Dense layers beside logic layers: y = act(x w^T + bias) + residual on the tensor cores, one kernel for the product and all of that.

A logic network reads values between 0 and 1.  `DenseLayer` learns them -- an encoder whose sigmoid feeds the first LogicLayer, in the
feature-major layout that logic layers read -- or makes the fully connected networks that the reference compares with
(experiments/main_baseline.py).  With `implementation='cuda'` it runs on csrc/dense.cu:

* bf16 and fp16 layers multiply their values as they are, fp32 layers three bf16 planes of each value, all 24 bits, or in the forward pass
  of up to 32 samples two parts of 11 bits (a product is then up to 2^-21 off, of either sign): results are no further off than those of
  32-bit arithmetic; all sums are 32-bit, results are rounded once;
* the backward pass multiplies the incoming gradient with the kept derivative of the activation (fp32, or for bf16
  layers fp16 times 2^14) and rounds the product to the layer's type before the two matrix products.

`implementation='python'` is the pure-torch definition of the same layer and runs anywhere.
"""
import ctypes
import math

import torch

from . import _native as N

ACTIVATIONS = {None: 0, 'none': 0, 'relu': 1, 'sigmoid': 2, 'silu': 3, 'gelu': 4}
TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _layout(t):
    """(tensor, pitch, feature_major): how the kernels read a 2-D tensor; copied where its rows are neither in one piece nor its
    columns."""
    rows, cols = t.shape
    s0, s1 = t.stride()
    if (s1 == 1 or cols == 1) and (s0 >= cols or rows == 1):
        return t, (s0 if rows > 1 else cols), False
    if (s0 == 1 or rows == 1) and (s1 >= rows or cols == 1):
        return t, (s1 if cols > 1 else rows), True
    return t.contiguous(), cols, False


def _bytes(n, like):
    return torch.empty(n, dtype=torch.uint8, device=like.device) if n else None


def _forward(x, w, bias, residual, act, feature_major, want_slope):
    """(y [batch, outer], slope, x, x_planes, w_planes); x as it was read."""
    batch, inner = x.shape
    outer = w.shape[0]
    kind = TYPES[x.dtype]
    y = torch.empty_strided((batch, outer), (1, batch) if feature_major else (outer, 1), dtype=x.dtype, device=x.device)
    slope = None
    if want_slope and act:
        slope = torch.empty(batch * outer, dtype=torch.float16 if x.dtype == torch.bfloat16 else torch.float32, device=x.device)
    if batch == 0:
        return y, slope, x, None, None
    x, pitch, x_feature = _layout(x)
    lib = N.lib()
    kind |= lib.dl_matmul_choice()
    with N.on_device(x):
        px, pw = x.data_ptr(), w.data_ptr()
        sizes = (ctypes.c_int64 * 3)()
        lib.dl_dense_forward_sizes(px, pitch, x_feature, pw, batch, inner, outer, feature_major, kind, sizes)
        x_planes, w_planes, work = (_bytes(n, x) for n in sizes)
        N.check(lib.dl_dense_forward(px, pitch, x_feature, pw, N.ptr(bias), N.ptr(residual), 0 if residual is None else residual.stride(0),
                                     0 if residual is None else residual.stride(1), act, y.data_ptr(), feature_major, N.ptr(slope),
                                     N.ptr(x_planes), N.ptr(w_planes), N.ptr(work), batch, inner, outer, kind, N.stream_of(x)))
    return y, slope, x, x_planes, w_planes


def _lay_out(t, pitch, feature_major):
    """The planes of an operand, as its products read them."""
    rows, cols = reversed(t.shape) if feature_major else t.shape
    lib, kind = N.lib(), TYPES[t.dtype]
    with N.on_device(t):
        planes = _bytes(lib.dl_dense_planes_bytes(rows, cols, kind), t)
        N.check(lib.dl_dense_lay_out(t.data_ptr(), rows, cols, pitch, kind, planes.data_ptr(), N.stream_of(t)))
    return planes


class DenseFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, residual, act, feature_major):
        ctx.set_materialize_grads(False)
        y, slope, read, x_planes, w_planes = _forward(x, w, bias, residual, act, feature_major, True)
        _, ctx.pitch, ctx.x_feature = _layout(read)
        keep_x, keep_w = x_planes is None, w_planes is None
        if x.dtype == torch.float32 and keep_w and x.shape[0] > 0:
            # Few samples.  An optimizer's kernels may change fp32 parameters before the backward pass, without autograd's version counters:
            # it gets the values that were read here, laid out now as it would do itself.
            x_planes = _lay_out(read, ctx.pitch, ctx.x_feature) if ctx.needs_input_grad[1] else None
            w_planes = _lay_out(w, w.shape[1], False) if ctx.needs_input_grad[0] else None
            keep_x = keep_w = False
        # what was laid out for the product serves the backward pass too, in place of the tensor itself
        ctx.save_for_backward(read if keep_x else None, w if keep_w else None, x_planes, w_planes, slope)
        ctx.x_ptr, ctx.w_ptr = read.data_ptr(), w.data_ptr()     # their alignment decided what was laid out
        ctx.sizes = (x.shape[0], x.shape[1], w.shape[0])
        ctx.has_bias, ctx.feature_major, ctx.act = bias is not None, feature_major, act
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy):
        if gy is None:
            return None, None, None, None, None, None
        x, w, x_planes, w_planes, slope = ctx.saved_tensors
        batch, inner, outer = ctx.sizes
        want_x, want_w, want_b = ctx.needs_input_grad[0], ctx.needs_input_grad[1], ctx.has_bias and ctx.needs_input_grad[2]
        gx = gw = gb = None
        if want_x or want_w or want_b:
            make = torch.zeros if batch == 0 else torch.empty
            opts = dict(dtype=gy.dtype, device=gy.device)
            gx = make((batch, inner), **opts) if want_x else None
            gw = make((outer, inner), **opts) if want_w else None
            gb = make((outer,), **opts) if want_b else None
            if batch > 0:
                if gy.is_contiguous():
                    g, feature = gy, False
                elif gy.t().is_contiguous():
                    g, feature = gy, True
                else:
                    g, feature = gy.contiguous(), False
                if slope is not None and feature != ctx.feature_major and batch > 1 and outer > 1:
                    feature = ctx.feature_major
                    g = gy.t().contiguous().t() if feature else gy.contiguous()
                lib = N.lib()
                kind = TYPES[gy.dtype] | lib.dl_matmul_choice()
                with N.on_device(gy):
                    px, pw = x.data_ptr() if x is not None else ctx.x_ptr, w.data_ptr() if w is not None else ctx.w_ptr
                    work = _bytes(lib.dl_dense_backward_workspace_bytes(g.data_ptr(), feature, slope is not None, px, ctx.pitch, ctx.x_feature, pw,
                                                                        want_w and x_planes is None, want_x and w_planes is None, batch, inner,
                                                                        outer, kind), gy)
                    N.check(lib.dl_dense_backward(g.data_ptr(), feature, N.ptr(slope), px, ctx.pitch, ctx.x_feature, pw, N.ptr(x_planes), N.ptr(w_planes),
                                                  N.ptr(gx), N.ptr(gw), N.ptr(gb), work.data_ptr(), batch, inner, outer, kind, N.stream_of(gy)))
        return gx, gw, gb, gy if ctx.needs_input_grad[3] else None, None, None


def _check(x, weight, bias, residual, activation):
    if activation not in ACTIVATIONS:
        raise ValueError("dense: unknown activation %r (one of %s)" % (activation, ", ".join(sorted(a for a in ACTIVATIONS if a))))
    if x.dim() < 1 or weight.dim() != 2:
        raise ValueError("dense: x must have at least one dimension and weight two, got %s and %s" % (tuple(x.shape), tuple(weight.shape)))
    outer, inner = weight.shape
    if x.shape[-1] != inner or inner == 0 or outer == 0:
        raise ValueError("dense: x %s does not fit weight %s" % (tuple(x.shape), tuple(weight.shape)))
    if bias is not None and tuple(bias.shape) != (outer,):
        raise ValueError("dense: bias must be [%d], got %s" % (outer, tuple(bias.shape)))
    if residual is not None and tuple(residual.shape) != tuple(x.shape[:-1]) + (outer,):
        raise ValueError("dense: residual must be %s, got %s" % (tuple(x.shape[:-1]) + (outer,), tuple(residual.shape)))
    for t in (weight, bias, residual):
        if t is not None and (t.dtype != x.dtype or t.device != x.device):
            raise ValueError("dense: all tensors must have one type and device, got %s on %s beside %s on %s" % (t.dtype, t.device, x.dtype, x.device))


def dense(x, weight, bias=None, residual=None, activation=None, feature_major=False):
    """act(x weight^T + bias) + residual, differentiable once and not in forward mode.

    x `[..., in]`, weight `[out, in]`, bias `[out]`, residual `[..., out]`, all of one type (float32, bfloat16 or float16) on one CUDA
    device; activation: None, 'relu', 'sigmoid', 'silu' or 'gelu' (the exact one).  x may be a transposed view, as logic layers return
    them.  An infinite float32 operand makes the results it enters infinite or undefined.  A call that a CUDA graph captures is refused
    while an earlier graph, made on the default stream, is alive that has one of these tensors as a leaf, or the leaf that one of them is a
    view, reshape or copy of.  feature_major: a 2-D result lies in memory as `[out, batch]` (same values, other strides), which a LogicLayer
    reads without a copy."""
    act = ACTIVATIONS.get(activation, -1)
    if act >= 0 and x.is_cuda:
        # the native node; None for a call that is not of the ordinary form
        y = N.nodes().dense(x, weight, bias, residual, act, feature_major)
        if y is not None:
            return y
    _check(x, weight, bias, residual, activation)
    N.require_cuda(x)
    if x.dtype not in TYPES:
        raise ValueError("dense: float32, bfloat16 or float16, got %s" % x.dtype)
    if feature_major and x.dim() != 2:
        raise ValueError("dense: feature_major needs a 2-D x, got %d dimensions" % x.dim())
    lead, outer = x.shape[:-1], weight.shape[0]
    graph = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual))
    if graph:
        N.nodes().refuse_older_graphs(x, weight, bias, residual)
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
        residual = None if residual is None else residual.reshape(-1, outer)
    weight = weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    # apply() refuses forward mode, which there is no derivative for
    if graph or any(t is not None and torch.autograd.forward_ad.unpack_dual(t).tangent is not None for t in (x, weight, bias, residual)):
        y = DenseFunction.apply(x, weight, bias, residual, act, bool(feature_major))
    else:
        y = _forward(x, weight, bias, residual, act, bool(feature_major), False)[0]
    return y if len(lead) == 1 else y.reshape(*lead, outer)


def dense_python(x, weight, bias=None, residual=None, activation=None):
    """The definition of `dense` in torch's operations."""
    _check(x, weight, bias, residual, activation)
    z = torch.nn.functional.linear(x, weight, bias)
    act = {0: lambda v: v, 1: torch.relu, 2: torch.sigmoid, 3: torch.nn.functional.silu, 4: torch.nn.functional.gelu}[ACTIVATIONS[activation]]
    y = act(z)
    return y if residual is None else y + residual


class DenseLayer(torch.nn.Module):
    """A fully connected layer with its activation, in front of, between or instead of logic layers."""

    def __init__(self, in_dim: int, out_dim: int, device: str = 'cuda', activation: str = 'sigmoid', bias: bool = True,
                 implementation: str = None, feature_major: bool = False, dtype: torch.dtype = torch.float32):
        """
        :param in_dim:         number of input features
        :param out_dim:        number of output features
        :param device:         'cuda' or 'cpu'
        :param activation:     None, 'relu', 'sigmoid' (what a logic layer can read), 'silu' or 'gelu'
        :param bias:           whether a learned bias is added
        :param implementation: 'cuda' (the kernels; default on a CUDA device) or 'python' (pure torch; default on CPU)
        :param feature_major:  results of 2-D inputs lie in memory as the next LogicLayer reads them
        :param dtype:          float32, bfloat16 or float16
        """
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError("DenseLayer: unknown activation %r" % (activation,))
        if dtype not in TYPES:
            raise ValueError("DenseLayer: float32, bfloat16 or float16, got %s" % dtype)
        self.in_dim, self.out_dim, self.device, self.activation, self.feature_major = in_dim, out_dim, device, activation, feature_major
        self.implementation = implementation
        if self.implementation is None:
            self.implementation = 'cuda' if torch.device(device).type == 'cuda' else 'python'
        assert self.implementation in ['cuda', 'python'], self.implementation
        bound = 1 / math.sqrt(in_dim)
        self.weight = torch.nn.Parameter(torch.empty(out_dim, in_dim, device=device, dtype=dtype).uniform_(-bound, bound))
        self.bias = torch.nn.Parameter(torch.empty(out_dim, device=device, dtype=dtype).uniform_(-bound, bound)) if bias else None

    def forward(self, x, residual=None):
        if self.implementation == 'python':
            return dense_python(x, self.weight, self.bias, residual, self.activation)
        return dense(x, self.weight, self.bias, residual, self.activation, feature_major=self.feature_major and x.dim() == 2)

    def extra_repr(self):
        return '{}, {}, {}'.format(self.in_dim, self.out_dim, self.activation)
