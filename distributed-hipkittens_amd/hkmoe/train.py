"""What a training step runs around the experts' products: layer norm, the router's
choice, tokens sorted by expert and back, each with its gradient.

Every operator comes in two forms.  ``layer_norm``, ``route_topk``, ``moe_permute`` and
``moe_combine`` record gradients where an input asks for them (first derivatives, backward only:
dual tensors of forward mode are refused, by autograd, for want of a jvp).  The ``*_forward`` /
``*_backward`` functions are the plain calls that those make, on the current stream, for
programs that run their own backward pass or capture it into a graph.
"""
from typing import NamedTuple

import torch

import tk_kernel

from .layer import _dual, _no_gradient, _written


def _rows(g):
    """A gradient from autograd as the kernels read rows: contiguous and 16-byte aligned, which a slice of a
    flattened concatenation's gradient, for one, is not."""
    g = g.contiguous()
    return g if g.data_ptr() % 16 == 0 else g.clone()


# ----------------------------------------------------------------------------
# layer norm
# ----------------------------------------------------------------------------
def layer_norm_forward(x, weight, bias=None, residual=None, eps=1e-5, residual_out=None):
    """Layer norm of ``x`` (+ ``residual``): returns ``(y, r, stats)``.

    x [R, C] bf16 or fp32, residual like x, weight and bias [C] both bf16 or both fp32.  r is the new
    stream x + residual in x's dtype (x itself without a residual; ``residual_out`` where given, which
    may be x or residual), y the norm of r in x's dtype, stats what
    :func:`layer_norm_backward` wants back (fp32 [R, 4]).  Records no gradient; a ``residual_out`` that
    asks for one is refused."""
    if x.dim() != 2:
        raise RuntimeError("layer_norm: x must be [R, C]")
    y = torch.empty_like(x)
    stats = x.new_empty(x.shape[0], 4, dtype=torch.float32)
    given = residual_out
    if residual is None:
        if residual_out is not None:
            raise RuntimeError("layer_norm: residual_out needs a residual")
        r = x
    else:
        if residual_out is not None:
            _no_gradient(residual_out, "residual_out")
        r = residual_out = torch.empty_like(x) if residual_out is None else residual_out
    tk_kernel.dispatch_layer_norm(x, residual, weight, bias, eps, y, residual_out, stats)
    _written(given)
    return y, r, stats


def layer_norm_backward(dy, r, weight, stats, dr=None, with_bias=True):
    """``(dx, dweight, dbias)`` for the gradient ``dy`` of y and, where given, ``dr`` of the new
    stream r.  dx is the gradient of both x and the residual; dbias is None without ``with_bias``."""
    dx, dw = torch.empty_like(r), torch.empty_like(weight)
    db = torch.empty_like(weight) if with_bias else None
    need = tk_kernel.layer_norm_backward_workspace_size(*r.shape)
    ws = r.new_empty(need, dtype=torch.uint8) if need else None
    tk_kernel.dispatch_layer_norm_backward(dy, r, weight, dr, stats, dx, dw, db, ws)
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps):
        y, r, stats = layer_norm_forward(x, weight, bias, residual, eps)
        ctx.save_for_backward(r, weight, stats)
        ctx.has_bias, ctx.has_residual = bias is not None, residual is not None
        ctx.set_materialize_grads(False)  # of y and r, where one has no use: no zeros to read
        return (y, r) if residual is not None else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dr=None):
        if dy is None:  # the norm has no use: the stream's own gradient is all there is
            return dr, None, None, dr if ctx.has_residual else None, None
        r, weight, stats = ctx.saved_tensors
        dx, dw, db = layer_norm_backward(_rows(dy), r, weight, stats, None if dr is None else _rows(dr), ctx.has_bias)
        return dx, dw, db, dx if ctx.has_residual else None, None


def layer_norm(x, weight, bias=None, residual=None, eps=1e-5):
    """``(y, r)``: the layer norm y of the new stream r = x + residual (x itself without one), both
    in x's dtype; gradients of x, weight, bias and residual are recorded.  Arguments as in
    :func:`layer_norm_forward`."""
    if (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual))
            or _dual(x, weight, bias, residual)):
        out = _LayerNorm.apply(x, weight, bias, residual, eps)
        return out if residual is not None else (out, x)
    return layer_norm_forward(x, weight, bias, residual, eps)[:2]


# ----------------------------------------------------------------------------
# the router's choice
# ----------------------------------------------------------------------------
def route_topk_forward(logits, top_k):
    """``(idx, w)``: the ``top_k`` largest logits of fp32 [T, E] in descending order (int32 [T, k];
    ties to the lower expert) and their softmax (fp32 [T, k])."""
    if logits.dim() != 2:
        raise RuntimeError("route_topk: logits must be [T, E]")
    t, e = logits.shape
    idx = logits.new_empty(t, top_k, dtype=torch.int32)
    w = logits.new_empty(t, top_k)
    counts = logits.new_empty(tk_kernel.route_blocks(t), e, dtype=torch.int32)
    tk_kernel.dispatch_route_topk(logits, idx, w, counts)
    return idx, w


def route_topk_backward(dw, w, idx, num_experts):
    """Gradient of the logits (fp32 [T, E]) for the gradient ``dw`` of the weights ``w``."""
    dlogits = dw.new_empty(dw.shape[0], num_experts)
    tk_kernel.dispatch_route_topk_backward(dw, w, idx, dlogits)
    return dlogits


class _RouteTopk(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_k):
        idx, w = route_topk_forward(logits, top_k)
        ctx.save_for_backward(idx, w)
        ctx.num_experts = logits.shape[1]
        ctx.mark_non_differentiable(idx)
        ctx.set_materialize_grads(False)  # no zeros in idx's place
        return idx, w

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, _, dw):
        if dw is None:
            return None, None
        idx, w = ctx.saved_tensors
        return route_topk_backward(dw.contiguous(), w, idx, ctx.num_experts), None


def route_topk(logits, top_k):
    """:func:`route_topk_forward` with the gradient of w to the logits recorded."""
    if logits.requires_grad and torch.is_grad_enabled() or _dual(logits):
        return _RouteTopk.apply(logits, top_k)
    return route_topk_forward(logits, top_k)


# ----------------------------------------------------------------------------
# tokens by expert and back
# ----------------------------------------------------------------------------
class MoEOrder(NamedTuple):
    """Slots f = t*k + j in expert order: expert e has places offsets[e] .. offsets[e + 1] - 1
    (int32 [E + 1]), place p holds slot perm[p] (int32 [T*k]) and slot (t, j) is at
    inv_perm[t, j] (int32 [T, k]).  Slots without an expert here are at offsets[E] and behind."""
    offsets: torch.Tensor
    perm: torch.Tensor
    inv_perm: torch.Tensor


def moe_permute_forward(x, ids, num_experts):
    """``(xp, order)``: the rows of x [T, H] (bf16, fp32 or e4m3) copied to their slots'
    places [T*k, H], zeros behind the last expert's.  ids int32 [T, k]: each slot's expert; a
    value outside [0, num_experts), for instance -1, has none here."""
    if x.dim() != 2 or ids.dim() != 2 or ids.shape[0] != x.shape[0]:
        raise RuntimeError("moe_permute: x must be [T, H] and ids [T, k]")
    if num_experts < 1:
        raise RuntimeError("moe_permute: num_experts must be positive")
    t, k = ids.shape
    xp = x.new_empty(t * k, x.shape[1])
    order = MoEOrder(ids.new_empty(num_experts + 1), ids.new_empty(t * k), torch.empty_like(ids))
    need = tk_kernel.permute_workspace_size(t, num_experts, k)
    ws = x.new_empty(need, dtype=torch.uint8) if need else None
    tk_kernel.dispatch_permute(x, ids, xp, *order, ws)
    return xp, order


def moe_permute_backward(dxp, order):
    """Gradient of x [T, H]: the sum of its slots' rows of ``dxp`` [T*k, H]."""
    dx = dxp.new_empty(order.inv_perm.shape[0], dxp.shape[1])
    tk_kernel.dispatch_combine_rows(dxp, None, order.offsets, order.inv_perm, dx)
    return dx


def moe_combine_forward(y, w, order):
    """out[t] = sum_j w[t, j] y[inv_perm[t, j]] over the slots that have an expert here: y [T*k, H]
    bf16 or fp32, w fp32 [T, k]; summed in fp32, rounded to y's dtype."""
    out = y.new_empty(order.inv_perm.shape[0], y.shape[1])
    tk_kernel.dispatch_combine_rows(y, w, order.offsets, order.inv_perm, out)
    return out


def moe_combine_backward(dout, y, w, order):
    """``(dy, dw)``: gradients of y (zeros behind the last expert's rows) and w."""
    dy, dw = torch.empty_like(y), torch.empty_like(w)
    tk_kernel.dispatch_combine_rows_backward(dout, y, w, order.offsets, order.inv_perm, dy, dw)
    return dy, dw


class _Permute(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, ids, num_experts):
        xp, order = moe_permute_forward(x, ids, num_experts)
        ctx.save_for_backward(*order)
        ctx.mark_non_differentiable(*order)
        ctx.set_materialize_grads(False)  # no zeros in the order's place
        return (xp, *order)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dxp, *_):
        if dxp is None:
            return None, None, None
        return moe_permute_backward(_rows(dxp), MoEOrder(*ctx.saved_tensors)), None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, w, *order):
        ctx.save_for_backward(y, w, *order)
        return moe_combine_forward(y, w, MoEOrder(*order))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        y, w, *order = ctx.saved_tensors
        return (*moe_combine_backward(_rows(dout), y, w, MoEOrder(*order)), None, None, None)


def moe_permute(x, ids, num_experts):
    """:func:`moe_permute_forward` with the gradient of x recorded (not for e4m3 rows)."""
    if x.requires_grad and torch.is_grad_enabled() or _dual(x):
        xp, *order = _Permute.apply(x, ids, num_experts)
        return xp, MoEOrder(*order)
    return moe_permute_forward(x, ids, num_experts)


def moe_combine(y, w, order):
    """:func:`moe_combine_forward` with the gradients of y and w recorded."""
    if (y.requires_grad or w.requires_grad) and torch.is_grad_enabled() or _dual(y, w):
        return _Combine.apply(y, w, *order)
    return moe_combine_forward(y, w, order)
