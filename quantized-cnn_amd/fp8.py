"""Linear layers and row norms in 8-bit floating point: e4m3 codes with a power-of-two scale per block of 128.

    y = fp8.linear(x, weight, bias)                              # weight (in, out) as in MyLinear, fp32 / bf16 / fp16
    y, h = fp8.norm_linear(x, norm_weight, weight, bias, residual=r)   # RMS norm of x + r, its codes straight into the product
    layer = fp8.Fp8Linear(512, 1000); norm = fp8.RMSNorm(512)
    layer.pack()                                                 # serving: the codes of the weights are kept

Forward and both gradients are products of codes (ops.fp8_matmul): activations and gradients in 1 x 128 blocks along the
product's contraction, weights in 128 x 128 tiles.  The weight gradient of fp32 weights is an fp32 product.  Gradients pass the
roundings unchanged (straight through).  The reference has no such layer: parity unpinned.
"""
import math
import weakref

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import ops


def _flat(t):
    """(..., n) -> (rows, n), a view where the strides allow it (rows that share memory, as a broadcast gradient's do, are copied)."""
    if t.dim() == 2 and (t.stride(1) == 1 or t.shape[1] <= 1) and (t.stride(0) >= t.shape[1] or t.shape[0] <= 1):
        return t
    return t.reshape(-1, t.shape[-1]).contiguous()


def _weight_forms(weight, need_dx):
    """-> (codes of weight^T for the forward product, codes of weight for the input gradient or None)."""
    if weight.stride(1) != 1 and weight.stride(0) == 1:  # a transposed view: tiles are square, so its transpose has the same codes
        got = ops.fp8_quantize(_flat(weight.t()), forms="both" if need_dx else "rows", block_rows=ops.FP8_BLOCK)
        return got if need_dx else (got, None)
    if need_dx:
        rows, cols = ops.fp8_quantize(_flat(weight), forms="both", block_rows=ops.FP8_BLOCK)
        return cols, rows
    return ops.fp8_quantize(_flat(weight), forms="cols", block_rows=ops.FP8_BLOCK), None


def _leaf_nodes(fn, weights):
    """The AccumulateGrad nodes of the leaves behind fn's operands: through views, casts and other operators of one operand, behind the operands
    at the places `weights` through any operators; not through nodes of this module, whose own call has looked behind them."""
    found = []
    for i, (node, _) in enumerate(fn.next_functions):
        if type(node).__name__ == "AccumulateGrad":
            found.append(node)
            continue
        stack = [node]
        while stack:
            node = stack.pop()
            if type(node).__name__ == "AccumulateGrad":
                found.append(node)
            elif node is not None and "fp8_checked" not in node.metadata:
                behind = [n for n, _ in node.next_functions if n is not None]
                if len(behind) == 1 or i in weights:
                    stack += behind
    return found


def _checked(out, weights):
    """out, the result of a Function's apply, after a check of the leaves behind its operands (`weights`: places of the weights among them).  A leaf's
    gradient is accumulated on the stream that was current when its first graph was made.  If that graph lives on and was made on the
    default stream, a backward pass in a capture would make that stream wait for the capture, which ends the process: it is refused here,
    where nothing is lost yet."""
    first = out[0] if isinstance(out, tuple) else out
    fn = first.grad_fn
    if fn is not None:
        fn.metadata["fp8_checked"] = True
        capturing = torch.cuda.is_current_stream_capturing()
        if capturing or ops._current_stream(first.device.index) == 0:
            for node in _leaf_nodes(fn, weights):
                if not capturing:
                    node.metadata.setdefault("fp8_default_stream", True)
                elif node.metadata.get("fp8_default_stream"):
                    raise RuntimeError("fp8: a graph of the same parameters, made on the default stream, is still alive (a loss or an output is kept): "
                                       "its gradients cannot be captured; delete or detach it before the capture")
    return out


def _grad_forms(dy, need_dx, need_dw, need_db):
    """Codes of dy along its rows and along its columns, and its column sums, from one read; None where not needed."""
    if need_dw or need_db:
        got = ops.fp8_quantize(dy, forms="both" if need_dx else "cols", colsum=need_db)
        got = got if isinstance(got, tuple) else (got,)
        return got[0] if need_dx else None, got[1 if need_dx else 0], got[-1] if need_db else None
    return ops.fp8_quantize(dy) if need_dx else None, None, None


def _save(ctx, blocks, *tensors):
    """The buffers of two matrices of codes (None: not needed) and tensors as saved tensors, which are freed with the graph, seen by hooks and
    recomputed under checkpointing; the matrices themselves, not used any more, stay without them."""
    a, b = ctx.blocks = blocks
    ctx.save_for_backward(a and a._buf, b and b._buf, *tensors)
    if a is not None:
        a._buf = None
    if b is not None:
        b._buf = None


def _saved(ctx):
    a, b = ctx.blocks
    p, q, *tensors = ctx.saved_tensors
    return a and a._on(p), b and b._on(q), *tensors


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, out_dtype):
        need_dx, need_dw = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        xq, xt = ops.fp8_quantize(x, forms="both") if need_dw else (ops.fp8_quantize(x), None)
        wt, w = _weight_forms(weight, need_dx)
        _save(ctx, (xt, w))
        ctx.types = x.dtype, weight.dtype, bias.dtype if bias is not None else None
        return ops.fp8_matmul(xq, wt, bias=bias.float() if bias is not None else None, out_dtype=out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need_dx, need_dw, need_db = ctx.needs_input_grad[:3]
        xt, w = _saved(ctx)
        xtype, wtype, btype = ctx.types
        dq, dt, db = _grad_forms(_flat(dy), need_dx, need_dw, need_db)
        dx = ops.fp8_matmul(dq, w, out_dtype=xtype) if need_dx else None
        dw = ops.fp8_matmul(xt, dt, out_dtype=wtype) if need_dw else None
        return dx, dw, db.to(btype) if need_db else None, None


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, h, rstd = ops.rms_norm_forward(x, weight, residual=residual, eps=eps)
        ctx.save_for_backward(h, weight, rstd)
        ctx.both = residual is not None
        ctx.set_materialize_grads(False)
        return (y, h) if ctx.both else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight, rstd = ctx.saved_tensors
        if dy is None:  # only h was used
            return dh, None, dh, None
        dx, dw = ops.rms_norm_backward(_flat(dy), h, weight, rstd, dh=_flat(dh) if dh is not None else None,
                                       need_dx=ctx.needs_input_grad[0] or ctx.needs_input_grad[2], need_dweight=ctx.needs_input_grad[1])
        return dx, dw, dx if ctx.both else None, None


class _NormLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, norm_weight, weight, bias, residual, eps, out_dtype):
        need_dn = ctx.needs_input_grad[0] or ctx.needs_input_grad[1] or ctx.needs_input_grad[4]
        xq, h, rstd = ops.rms_norm_forward(x, norm_weight, residual=residual, eps=eps, quantize=True)
        wt, w = _weight_forms(weight, need_dn)
        ctx.types = x.dtype, weight.dtype, bias.dtype if bias is not None else None
        ctx.both = residual is not None
        ctx.set_materialize_grads(False)
        y = ops.fp8_matmul(xq, wt, bias=bias.float() if bias is not None else None, out_dtype=out_dtype)
        _save(ctx, (xq if ctx.needs_input_grad[2] else None, w), h, norm_weight, rstd)
        return (y, h) if ctx.both else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        xq, w, h, norm_weight, rstd = _saved(ctx)
        need_x, need_nw, need_dw, need_db, need_r = ctx.needs_input_grad[:5]
        if dy is None:
            return dh, None, None, None, dh if ctx.both else None, None, None
        need_dn = need_x or need_nw or need_r
        xtype, wtype, btype = ctx.types
        dq, dt, db = _grad_forms(_flat(dy), need_dn, need_dw, need_db)
        dw = ops.fp8_matmul(ops.fp8_transpose(xq), dt, out_dtype=wtype) if need_dw else None
        dx = dnw = None
        if need_dn:
            dn = ops.fp8_matmul(dq, w, out_dtype=xtype)
            dx, dnw = ops.rms_norm_backward(dn, h, norm_weight, rstd, dh=_flat(dh) if dh is not None else None, need_dx=need_x or need_r,
                                            need_dweight=need_nw)
        return dx, dnw, dw, db.to(btype) if need_db else None, dx if ctx.both else None, None, None


def _check_residual(name, x, residual):
    if residual is not None and residual.shape != x.shape:
        raise ValueError("fp8.%s: residual %s, expected x's shape %s" % (name, tuple(residual.shape), tuple(x.shape)))


def linear(x, weight, bias=None, out_dtype=None):
    """x (..., in) @ weight + bias in 8-bit floating point; out_dtype defaults to x's.  weight: (in, out) tensor, quantised in
    this call, or Fp8Blocks (out, in) made before (no gradient of the weight then, and none of x)."""
    out_dtype = out_dtype or x.dtype
    x2 = _flat(x)
    if isinstance(weight, ops.Fp8Blocks):
        if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)):
            raise RuntimeError("fp8.linear: packed weights serve without gradients: call it under torch.no_grad(), or with the weight tensor")
        y = ops.fp8_matmul(ops.fp8_quantize(x2), weight, bias=bias.detach().float() if bias is not None else None, out_dtype=out_dtype)
    else:
        if weight.dim() != 2 or weight.shape[0] != x.shape[-1]:
            raise ValueError("fp8.linear: x %s / weight %s: need (..., in) and (in, out)" % (tuple(x.shape), tuple(weight.shape)))
        y = _checked(_Linear.apply(x2, weight, bias, out_dtype), (1, 2))
    return y if x.dim() == 2 else y.view(x.shape[:-1] + (y.shape[1],))


def rms_norm(x, weight, residual=None, eps=1e-6):
    """h = x + residual; y = h / sqrt(mean(h^2) + eps) * weight over the last axis -> (y, h), or y alone without residual."""
    _check_residual("rms_norm", x, residual)
    out = _checked(_RmsNorm.apply(_flat(x), weight.float(), _flat(residual) if residual is not None else None, eps), (1,))
    if residual is None:
        return out.view(x.shape)
    return out[0].view(x.shape), out[1].view(x.shape)


def norm_linear(x, norm_weight, weight, bias=None, residual=None, eps=1e-6, out_dtype=None):
    """linear(rms_norm(x, norm_weight, residual), weight, bias) with the norm's output kept as codes only (made from
    its fp32 values, without a rounding to x's type between) -> (y, h), or y alone
    without residual."""
    if weight.dim() != 2 or weight.shape[0] != x.shape[-1]:
        raise ValueError("fp8.norm_linear: x %s / weight %s: need (..., in) and (in, out)" % (tuple(x.shape), tuple(weight.shape)))
    _check_residual("norm_linear", x, residual)
    out = _checked(_NormLinear.apply(_flat(x), norm_weight.float(), weight, bias, _flat(residual) if residual is not None else None, eps,
                                     out_dtype or x.dtype), (1, 2, 3) if bias is not None else (1, 2))
    y, h = out if residual is not None else (out, None)
    y = y.view(x.shape[:-1] + (y.shape[1],))
    return y if residual is None else (y, h.view(x.shape))


class Fp8Linear(nn.Module):
    """Linear layer with weight (in_feature, out_feature) like MyLinear's, computed in 8-bit floating point."""

    def __init__(self, in_feature, out_feature, bias=True):
        super().__init__()
        self.weight = nn.Parameter(torch.empty(in_feature, out_feature))
        bound = 1 / math.sqrt(in_feature)
        nn.init.uniform_(self.weight, -bound, bound)
        self.bias = nn.Parameter(torch.empty(out_feature).uniform_(-bound, bound)) if bias else None
        self._packed = self._packed_of = None

    def pack(self):
        """Quantises the weight once, for serving: forward() under no_grad in eval mode then reads the codes.  train(), load_state_dict(),
        moving the module, another parameter in the weight's place, the training steps and torch's writes to it drop them; only a write
        through `weight.data` or from outside torch (a graph of one's own) goes unnoticed: call pack() again after it."""
        with torch.no_grad():
            self._packed, self._packed_of = _weight_forms(self.weight, False)[0], (weakref.ref(self.weight), self._writes())
        return self

    def _writes(self):
        """How often the weight has been written (tensors made in inference mode do not count that)."""
        return None if self.weight.is_inference() else self.weight._version

    def _packed_codes(self):
        """The kept codes; None, for good, if the weight is not the one that they were made of any more."""
        if self._packed is not None:
            (of, writes), w = self._packed_of, self.weight
            if of() is not w or (writes is not None and writes != w._version):
                self._packed = None
        return self._packed

    def __getstate__(self):  # (copies and pickles: the codes go along if they are the weight's)
        self._packed_codes()
        return dict(self.__dict__, _packed_of=None)

    def __setstate__(self, state):
        super().__setstate__(state)
        if self._packed is not None:
            self._packed_of = weakref.ref(self.weight), self._writes()

    def train(self, mode=True):
        if mode:
            self._packed = None
        return super().train(mode)

    def _apply(self, fn, *args, **kw):
        self._packed = None
        return super()._apply(fn, *args, **kw)

    def _load_from_state_dict(self, *args, **kw):
        self._packed = None
        return super()._load_from_state_dict(*args, **kw)

    def buffers_changed(self):
        """Called where a data-parallel wrapper or a captured or fused step has written the parameters in place."""
        self._packed = None

    def forward(self, x):
        if self._packed is not None and not self.training and not torch.is_grad_enabled() and self._packed_codes() is not None:
            return linear(x, self._packed, self.bias)
        return linear(x, self.weight, self.bias)


class RMSNorm(nn.Module):
    """y = x / sqrt(mean(x^2) + eps) * weight over the last axis; forward(x, residual) -> (y, x + residual)."""

    def __init__(self, features, eps=1e-6):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(features))
        self.eps = eps

    def forward(self, x, residual=None):
        return rms_norm(x, self.weight, residual, self.eps)
