"""Plain 64-bit implementations of the dense products' epilogue, layer norm, the router's
choice, tokens by expert and back, and their gradients (torch, any device), with bounds of
how far the kernels may be off.

u = 2^-24 is half a step of fp32.  A sum of n fp32 terms, in whatever order, is off by at
most (depth) u sum |terms|, depth the additions that a term passes through."""
import math

import torch

U = 2.0 ** -24


def half(dtype):
    """Half a step of the type, relative."""
    return torch.finfo(dtype).eps / 2


# ---------------------------------------------------------------------------
# epilogue
# ---------------------------------------------------------------------------
ACTIVATIONS = ["none", "relu", "silu", "gelu", "gelu_tanh"]


def phi(z):
    return 0.5 * torch.special.erfc(-z * 0.5 ** 0.5)


def activate(z, name):
    """(value, bound) of the activation of 64-bit z that is exact in fp32.  The bounds count the
    kernel's roundings: the exponent's (relative to it), an ulp each of exp2 and reciprocal, and
    a half for every other operation; results below the smallest normal number may be 0."""
    tiny = 2.0 ** -126
    if name == "relu":
        return z.clamp_min(0.0), torch.zeros_like(z)
    if name == "silu":
        # exponent |z| (constant, product: 2 u), exp2 2 u, sum u, reciprocal 2 u, product u
        v = z / (1.0 + torch.exp(-z))
        return v, (2 * z.abs() + 8) * U * v.abs() + z.abs() * tiny
    if name == "gelu":
        # max(z, 0) - t Q, Q = Phi(-t): the fit 1.8e-7 = 3 u; s = 1 / (1 + 0.31 t) to 3 u, and Q depends
        # on s with a power of at most 3 at a given t; eight FMAs of P over terms that add up to at most
        # twice P: 16 u; the exponent t^2/2 to 3 u of itself; exp2 2 u; two products 2 u; the last
        # FMA rounds the result
        v = z * phi(z)
        tail = z.abs() * phi(-z.abs())
        return v, (32 + 1.5 * z * z) * U * tail + U * v.abs() + z.abs() * tiny
    if name == "gelu_tanh":
        # exponent 2 u(z): constants, square, FMA and product: 5 u of itself; then as silu
        e = math.sqrt(8.0 / math.pi) * (z + 0.044715 * z ** 3)
        v = z / (1.0 + torch.exp(-e))
        return v, (5 * e.abs() + 8) * U * v.abs() + z.abs() * tiny
    return z, torch.zeros_like(z)


def activation_slope(z, name):
    """Largest slope of the activation, by which an error of z grows."""
    return 1.2 if name in ("silu", "gelu", "gelu_tanh") else 1.0


def epilogue(z, bias, name, residual, dtype):
    """(value, bound) for a product z that is exact in fp32: the additions round once each."""
    if bias is not None:
        z = z + bias.double()
    v, b = activate(z, name)
    if bias is not None:
        b = b + activation_slope(z, name) * U * z.abs()
    if residual is not None:
        v = v + residual.double()
        b = b + U * v.abs()
    return v, (b * (1 + 2 * half(dtype)) + half(dtype) * v.abs() + 2.0 ** -133)


# ---------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------
def layer_norm(r, w, b, eps):
    """(y, mean, rstd) of the 64-bit stream r."""
    m = r.mean(1, keepdim=True)
    c = r - m
    rstd = (c.square().mean(1, keepdim=True) + eps) ** -0.5
    y = c * rstd * w
    return (y if b is None else y + b), m, rstd


def layer_norm_bound(y, r, w, m, rstd, dtype):
    """n: r - m in two fp32 subtractions (each half a step of what it yields; the mean's first term is
    within |m| u), rstd and its product half a step each; y's FMA one, the output's own."""
    n = (r - m).abs() * rstd
    return 5 * U * n * w.abs() + U * U * 4 * m.abs() * rstd * w.abs() + (U + half(dtype)) * y.abs() + 2.0 ** -133


def layer_norm_grad(dy, r, w, eps, dr):
    """(dx, dw, db)."""
    _, m, rstd = layer_norm(r, w, None, eps)
    n = (r - m) * rstd
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - n * (g * n).mean(1, keepdim=True))
    return (dx if dr is None else dx + dr), (dy * n).sum(0), dy.sum(0)


def layer_norm_grad_bound(dy, r, w, eps, dr, dtype, wdtype, rows_each):
    """rows_each: rows that a thread adds up for dw and db in fp32.  A row's sums pass through at most
    32 additions of a thread, 6 of a wave and 16 of a workgroup; n is off by 5 u."""
    rows, cols = r.shape
    _, m, rstd = layer_norm(r, w, None, eps)
    n, g = (r - m) * rstd, dy * w
    ng = 5 * U * n.abs() + 4 * U * U * m.abs() * rstd  # how far n is off
    depth = 56 * U
    e1 = depth * g.abs().mean(1, keepdim=True)
    e2 = (depth + U) * (g * n).abs().mean(1, keepdim=True) + (g.abs() * ng).mean(1, keepdim=True)
    m1, m2 = g.mean(1, keepdim=True), (g * n).mean(1, keepdim=True)
    dx, dw, db = layer_norm_grad(dy, r, w, eps, dr)
    t = (g - m1).abs() + (n * m2).abs()
    bx = rstd * (e1 + n.abs() * e2 + ng * m2.abs() + 2 * U * (g.abs() + m1.abs()) + 4 * U * t) + U * dx.abs()
    long = (rows_each + 20) * U
    bw = (long * (dy * n).abs().sum(0) + (dy.abs() * ng).sum(0))
    bb = long * dy.abs().sum(0)
    return [b * (1 + 2 * half(t)) + half(t) * v.abs() + 2.0 ** -133
            for b, v, t in ((bx, dx, dtype), (bw, dw, wdtype), (bb, db, wdtype))]


# ---------------------------------------------------------------------------
# routing
# ---------------------------------------------------------------------------
def order(ids, experts):
    """(offsets, perm, inv) by Python's stable sort."""
    flat = [e if 0 <= e < experts else experts for e in ids.flatten().tolist()]
    perm = sorted(range(len(flat)), key=lambda f: flat[f])
    inv = [0] * len(flat)
    for p, f in enumerate(perm):
        inv[f] = p
    offsets, n = [], 0
    for e in range(experts + 1):
        offsets.append(n)
        n += flat.count(e) if len(flat) < 4096 else 0
    if len(flat) >= 4096:
        counts = torch.bincount(torch.tensor(flat), minlength=experts + 1)
        offsets = [0] + counts[:experts].cumsum(0).tolist()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return i32(offsets), i32(perm), i32(inv).view(ids.shape)


def in_use(ids, experts):
    return (ids >= 0) & (ids < experts)


def slots(y, inv, here):
    """The slots' rows [T, k, H] in 64 bits, zeros where the slot has no expert."""
    rows = y.double()[inv.long()]
    return torch.where(here[..., None], rows, torch.zeros_like(rows))


def combine(y, w, inv, here):
    rows = slots(y, inv, here)
    return (rows if w is None else rows * w.double()[..., None]).sum(1)


def combine_bound(y, w, inv, here, dtype):
    rows = slots(y, inv, here).abs()
    s = (rows if w is None else rows * w.double().abs()[..., None]).sum(1)
    k = inv.shape[1]
    return (k + 1) * U * s * (1 + 2 * half(dtype)) + half(dtype) * combine(y, w, inv, here).abs() + 2.0 ** -133


def combine_grad(dout, y, w, inv, here):
    """(dy, dw)."""
    rows = slots(y, inv, here)
    d = dout.double()
    dy = torch.zeros_like(y, dtype=torch.float64)
    t, j = here.nonzero(as_tuple=True)
    dy[inv[t, j].long()] = d[t] * w.double()[t, j, None]
    return dy, (rows * d[:, None]).sum(2)


def combine_grad_bound(dout, y, inv, here):
    """dw: 8 values a chunk, a row of up to 4096 values one chunk a thread; 6 additions of a wave, 8 of
    a workgroup."""
    depth = 8 * math.ceil(y.shape[1] / 4096) + 16
    return depth * U * (slots(y, inv, here) * dout.double()[:, None]).abs().sum(2) + 2.0 ** -140


def route_grad(dw, w, idx, experts):
    dw, w = dw.double(), w.double()
    dl = w * (dw - (w * dw).sum(1, keepdim=True))
    out = torch.zeros((dw.shape[0], experts), dtype=torch.float64, device=dw.device)
    here = in_use(idx, experts)
    return out.scatter_add_(1, torch.where(here, idx, torch.zeros_like(idx)).long(), torch.where(here, dl, torch.zeros_like(dl)))


def route_grad_bound(dw, w, idx, experts):
    """The sum over k passes through a product and 6 additions; difference and product half a step
    each, and again where an expert stands in several slots."""
    dw, w = dw.double(), w.double()
    s = (w * dw).abs().sum(1, keepdim=True)
    b = w.abs() * (8 * U * s + U * (dw.abs() + s)) + U * (w * dw).abs() + U * w.abs() * s
    out = torch.zeros((dw.shape[0], experts), dtype=torch.float64, device=dw.device)
    here = in_use(idx, experts)
    out.scatter_add_(1, torch.where(here, idx, torch.zeros_like(idx)).long(), torch.where(here, b, torch.zeros_like(b)))
    return (1 + idx.shape[1]) * out + 2.0 ** -140


def route(logits, k):
    """(idx, w): descending, ties to the lower expert."""
    v, idx = torch.sort(logits.double(), dim=1, descending=True, stable=True)
    return idx[:, :k].to(torch.int32), torch.softmax(v[:, :k], 1)
