"""Cases of the dense product's epilogue and of what a training step runs around
the experts: layer norm, tokens sorted by expert and back, and their gradients.

Each case is what a program does per layer with tensors already on the GPU:

  op "linear"   hkmoe.gemm_fp8 / gemm_mx with a bias, an activation and a residual:
                act(A . B^T + bias) + residual
  op "norm"     hkmoe.layer_norm_forward: the residual's addition and the layer norm;
                with ``grad`` hkmoe.layer_norm_backward after it
  op "permute"  hkmoe.moe_permute: slots sorted by expert and the tokens' rows copied
                in that order; with ``grad`` hkmoe.moe_permute_backward after it
  op "combine"  hkmoe.moe_combine: the experts' rows back in token order, weighted
                and summed, then hkmoe.moe_combine_backward and the gradient of the
                router's logits, hkmoe.route_topk_backward

``own`` chooses between the framework's calls and the plain forms below (the
same formulas in elementary fp32 operations).
"""
import math
import os
import sys

import torch

own = False  # True: the framework's calls

F8 = torch.float8_e4m3fn
DEV = "cuda"
EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _linear(M, N, K, mx, act, out="bf16", bias=True, residual=False):
    return dict(op="linear", M=M, N=N, K=K, mx=mx, act=act, out=out, bias=bias, residual=residual)


def _norm(T, C, dtype="bf16", residual=True, grad=False, weight="bf16"):
    return dict(op="norm", T=T, C=C, dtype=dtype, residual=residual, grad=grad, weight=weight)


def _permute(T, H, E, k, dtype="bf16", drop=0.0, grad=False):
    return dict(op="permute", T=T, H=H, E=E, k=k, dtype=dtype, drop=drop, grad=grad)


def _combine(T, H, E, k, dtype="bf16", drop=0.0):
    return dict(op="combine", T=T, H=H, E=E, k=k, dtype=dtype, drop=drop)


def listed():
    return [
        # one token through the first half of a dense feed-forward: launch latency and B's stream
        dict(name="linear_1", **_linear(1, 4096, 4096, False, "gelu")),
        # a decode batch, microscaled operands
        dict(name="linear_mx_64", **_linear(64, 14336, 4096, True, "silu")),
        # the second half over an odd prefill chunk, added to an fp32 residual stream
        dict(name="linear_1777", **_linear(1777, 4096, 2048, False, "none", out="f32", residual=True)),
        # a large prefill with everything on
        dict(name="linear_8192", **_linear(8192, 4096, 7168, False, "gelu", residual=True)),
        # the norm in front of a decoded token
        dict(name="norm_1", **_norm(1, 4096)),
        # a training step's norm: an odd batch of an fp32 stream without a residual; the flagship width
        dict(name="norm_train_1999", **_norm(1999, 2560, dtype="f32", residual=False, grad=True, weight="f32")),
        dict(name="norm_train_8192", **_norm(8192, 7168, grad=True)),
        # a decode batch in front of the experts
        dict(name="permute_64", **_permute(64, 4096, 128, 8)),
        # an odd fp32 training batch of which a third goes to experts elsewhere
        dict(name="permute_train_777", **_permute(777, 2048, 60, 4, dtype="f32", drop=0.3, grad=True)),
        # the flagship layer's tokens, forward and backward
        dict(name="permute_train_8192", **_permute(8192, 7168, 256, 8, grad=True)),
        # the way back: an odd batch with experts elsewhere, the flagship layer
        dict(name="combine_train_333", **_combine(333, 2048, 60, 6, drop=0.25)),
        dict(name="combine_train_8192", **_combine(8192, 7168, 256, 8)),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "norm", "permute", "combine"])
    if op == "linear":
        N, K = 256 * _log_int(rng, 1, 56), 128 * _log_int(rng, 1, 112)
        M = _log_int(rng, 1, max(1, min(16384, 8192 * 4096 * 7168 // (N * K), 8192 * 14336 // max(N, K))))
        out = rng.choice(["bf16", "bf16", "f32"])
        return _linear(M, N, K, rng.random() < 0.5, rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]), out,
                       rng.random() < 0.8, rng.random() < 0.5)
    dtype = rng.choice(["bf16", "bf16", "f32"])
    half = 1 if dtype == "bf16" else 2
    if op == "norm":
        C = 8 * _log_int(rng, 16, 2048)
        T = _log_int(rng, 1, max(1, min(16384, 8192 * 7168 // (C * half))))
        return _norm(T, C, dtype, rng.random() < 0.6, rng.random() < 0.7, rng.choice(["bf16", "f32"]))
    H, E = 8 * _log_int(rng, 16, 1024), _log_int(rng, 1, 512)
    k = _log_int(rng, 1, min(E, 16))
    T = _log_int(rng, 1, max(1, min(16384, 8192 * 7168 * 8 // (H * k * half))))
    drop = rng.choice([0.0, 0.0, 0.1, 0.5, 0.9])
    if op == "permute":
        return _permute(T, H, E, k, dtype, drop, rng.random() < 0.6)
    return _combine(T, H, E, k, dtype, drop)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)


def _mx_operand(v):
    """(e4m3, e8m0 uint8 [R, C/32]): the exponent of each 1x32 block's largest magnitude."""
    b = v.view(v.shape[0], -1, 32)
    e = (b.abs().amax(2).view(torch.int32) >> 23).clamp_max(254)
    q = torch.ldexp(b, (127 - e)[..., None]).clamp(-448, 448).to(F8).view(v.shape)
    return q, e.to(torch.uint8)


def _words(e):
    """The exponents as the scaled products take them, int32 [C/128, R]: word
    64 i + 16 b + r of a K step holds in byte g the exponent of row 64 i + 16 g + r
    and K block b (R a multiple of 64).  A program does this once, to its weights."""
    rows, kb = e.shape
    v = e.view(rows // 64, 4, 16, kb // 4, 4).permute(3, 0, 4, 2, 1).contiguous()
    return v.view(torch.int32).reshape(kb // 4, rows)


def _linear_inputs(case, seed):
    g = _gen(seed)
    M, N, K, out = case["M"], case["N"], case["K"], DTYPES[case["out"]]
    # activations with a few large channels, weights of unit gain
    a, b = _randn(g, M, K), _randn(g, N, K) * K ** -0.5
    a[:, torch.randperm(K, generator=g, device=DEV)[: max(1, K // 256)]] *= 8.0
    d = dict(case=case, bias=None, residual=None)
    if case["mx"]:
        (d["a"], d["sa"]), (d["b"], d["sb"]) = _mx_operand(a), _mx_operand(b)
        d["b_words"] = _words(d["sb"])
    else:
        d["sa"], d["sb"] = (a.abs().amax() / 448.0).reshape(1), (b.abs().amax() / 448.0).reshape(1)
        d["a"], d["b"] = (a / d["sa"]).clamp(-448, 448).to(F8), (b / d["sb"]).clamp(-448, 448).to(F8)
    if case["bias"]:
        d["bias"] = (0.5 * _randn(g, N)).to(out)
    if case["residual"]:
        d["residual"] = (3.0 * _randn(g, M, N)).to(out)
    return d


def _norm_inputs(case, seed):
    g = _gen(seed)
    T, C, dtype, wt = case["T"], case["C"], DTYPES[case["dtype"]], DTYPES[case["weight"]]
    # a residual stream: a few channels are many times larger than the others, rows off centre
    gain = torch.ones(C, device=DEV)
    gain[torch.randperm(C, generator=g, device=DEV)[: max(1, C // 256)]] = 20.0
    stream = (2.0 * _randn(g, T, C) * gain + _randn(g, T, 1)).to(dtype)
    d = dict(case=case, residual=None, dr=None)
    if case["residual"]:
        d["residual"], d["x"] = stream, _randn(g, T, C).to(dtype)
    else:
        d["x"] = stream
    d["weight"], d["bias"] = (1.0 + 0.2 * _randn(g, C)).to(wt), (0.1 * _randn(g, C)).to(wt)
    if case["grad"]:
        d["dy"] = _randn(g, T, C).to(dtype)
        if case["residual"]:  # what comes back along the stream
            d["dr"] = _randn(g, T, C).to(dtype)
    return d


def _route_inputs(case, g):
    """Routing of T tokens with popular and rare experts; ``ids`` are the experts of
    this device's slots, -1 where the slot's expert is elsewhere."""
    T, E, k = case["T"], case["E"], case["k"]
    logits = _randn(g, T, E) + 1.5 * _randn(g, E)
    top, idx = logits.topk(k, dim=1)
    ids = idx.to(torch.int32)
    if case["drop"]:
        away = torch.rand((T, k), generator=g, device=DEV) < case["drop"]
        ids = torch.where(away, torch.full_like(ids, -1), ids)
    return dict(idx=idx.to(torch.int32), ids=ids, w=torch.softmax(top, 1))


def _permute_inputs(case, seed):
    g = _gen(seed)
    dtype = DTYPES[case["dtype"]]
    d = dict(case=case, **_route_inputs(case, g))
    d["x"] = _randn(g, case["T"], case["H"]).to(dtype)
    if case["grad"]:
        d["dxp"] = _randn(g, case["T"] * case["k"], case["H"]).to(dtype)
    return d


def _order(ids, experts):
    """(offsets [E + 1], perm [T k], inv [T, k]): slots in expert order, equal ones in
    their own order, the slots of no expert here behind the last."""
    key = torch.where((ids >= 0) & (ids < experts), ids, torch.full_like(ids, experts)).flatten()
    by, perm = key.sort(stable=True)
    offsets = torch.searchsorted(by, torch.arange(experts + 1, device=ids.device, dtype=by.dtype))
    inv = torch.empty_like(perm)
    inv[perm] = torch.arange(perm.numel(), device=ids.device)
    return tuple(v.to(torch.int32) for v in (offsets, perm, inv.view(ids.shape)))


def _combine_inputs(case, seed):
    g = _gen(seed)
    dtype, rows = DTYPES[case["dtype"]], case["T"] * case["k"]
    d = dict(case=case, **_route_inputs(case, g))
    d["order"] = _order(d["ids"], case["E"])  # of the way to the experts, kept for the way back
    d["y"] = _randn(g, rows, case["H"]).to(dtype)
    d["dout"] = _randn(g, case["T"], case["H"]).to(dtype)
    return d


INPUTS = {"linear": _linear_inputs, "norm": _norm_inputs, "permute": _permute_inputs, "combine": _combine_inputs}


def prepare(case, seed):
    return INPUTS[case["op"]](case, seed)


# ---------------------------------------------------------------------------
# plain forms: fp32, rounded once at the end
# ---------------------------------------------------------------------------
def _act(z, name):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * 0.5 ** 0.5))
    if name == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh((2.0 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z)))
    return z


def _powers(e):
    return torch.exp2(e.double() - 127.0).repeat_interleave(32, 1)


def _plain_linear(d):
    case = d["case"]
    a, b = d["a"].float(), d["b"].float()
    if case["mx"]:
        z = (a * _powers(d["sa"]).float()) @ (b * _powers(d["sb"]).float()).T
    else:
        z = (a @ b.T) * (d["sa"] * d["sb"])
    if d["bias"] is not None:
        z = z + d["bias"].float()
    z = _act(z, case["act"])
    if d["residual"] is not None:
        z = z + d["residual"].float()
    return z.to(DTYPES[case["out"]])


def _plain_norm(d):
    case, x, w = d["case"], d["x"], d["weight"].float()
    r = x if d["residual"] is None else (x.float() + d["residual"].float()).to(x.dtype)
    v = r.float()
    v = v - v.mean(1, keepdim=True)
    rstd = 1.0 / (v.square().mean(1, keepdim=True) + EPS).sqrt()
    n = v * rstd
    out = dict(y=(n * w + d["bias"].float()).to(x.dtype), r=None if d["residual"] is None else r)
    if not case["grad"]:
        return out
    dy = d["dy"].float()
    gw = dy * w
    dx = (gw - gw.mean(1, keepdim=True) - n * (gw * n).mean(1, keepdim=True)) * rstd
    if d["dr"] is not None:
        dx = dx + d["dr"].float()
    return dict(out, dx=dx.to(x.dtype), dw=(dy * n).sum(0).to(d["weight"].dtype), db=dy.sum(0).to(d["weight"].dtype))


def _plain_permute(d):
    case, x = d["case"], d["x"]
    k, here = case["k"], (d["ids"] >= 0) & (d["ids"] < case["E"])
    offsets, perm, inv = _order(d["ids"], case["E"])
    live = torch.arange(perm.numel(), device=perm.device) < offsets[-1]
    out = dict(xp=torch.where(live[:, None], x[(perm // k).long()], torch.zeros_like(x[:1])), offsets=offsets, perm=perm)
    if case["grad"]:
        rows = d["dxp"].float()[inv.long()]
        out["dx"] = torch.where(here[..., None], rows, torch.zeros_like(rows)).sum(1).to(x.dtype)
    return out


def _plain_combine(d):
    case, w, y, (offsets, perm, inv) = d["case"], d["w"], d["y"], d["order"]
    here = (d["ids"] >= 0) & (d["ids"] < case["E"])
    rows = y.float()[inv.long()]
    rows = torch.where(here[..., None], rows, torch.zeros_like(rows))
    out = (rows * w[..., None]).sum(1).to(y.dtype)
    dout = d["dout"].float()
    dw = (rows * dout[:, None]).sum(2)
    live = torch.arange(perm.numel(), device=perm.device) < offsets[-1]
    dy = dout[(perm // case["k"]).long()] * torch.where(live, w.flatten()[perm.long()], torch.zeros_like(w.flatten()))[:, None]
    dlogits = torch.zeros((case["T"], case["E"]), device=w.device)
    dlogits.scatter_(1, d["idx"].long(), w * (dw - (w * dw).sum(1, keepdim=True)))
    return dict(out=out, dy=dy.to(y.dtype), dw=dw, dlogits=dlogits)


PLAIN = {"linear": _plain_linear, "norm": _plain_norm, "permute": _plain_permute, "combine": _plain_combine}


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _own_linear(hkmoe, d):
    case = d["case"]
    more = dict(out_dtype=DTYPES[case["out"]], bias=d["bias"], activation=case["act"], residual=d["residual"])
    if case["mx"]:
        return hkmoe.gemm_mx(d["a"], hkmoe.mx_pack_scales(d["sa"]), d["b"], d["b_words"], **more)
    return hkmoe.gemm_fp8(d["a"], d["b"], d["sa"], d["sb"], **more)


def _own_norm(hkmoe, d):
    y, r, stats = hkmoe.layer_norm_forward(d["x"], d["weight"], d["bias"], d["residual"], eps=EPS)
    out = dict(y=y, r=None if d["residual"] is None else r)
    if not d["case"]["grad"]:
        return out
    dx, dw, db = hkmoe.layer_norm_backward(d["dy"], r, d["weight"], stats, dr=d["dr"])
    return dict(out, dx=dx, dw=dw, db=db)


def _own_permute(hkmoe, d):
    xp, order = hkmoe.moe_permute(d["x"], d["ids"], d["case"]["E"])
    out = dict(xp=xp, offsets=order.offsets, perm=order.perm)
    if d["case"]["grad"]:
        out["dx"] = hkmoe.moe_permute_backward(d["dxp"], order)
    return out


def _own_combine(hkmoe, d):
    order = hkmoe.MoEOrder(*d["order"])
    out = hkmoe.moe_combine(d["y"], d["w"], order)
    dy, dw = hkmoe.moe_combine_backward(d["dout"], d["y"], d["w"], order)
    return dict(out=out, dy=dy, dw=dw, dlogits=hkmoe.route_topk_backward(dw, d["w"], d["idx"], d["case"]["E"]))


OWN = {"linear": _own_linear, "norm": _own_norm, "permute": _own_permute, "combine": _own_combine}


def run(state):
    if own:
        return OWN[state["case"]["op"]](_framework(), state)
    return PLAIN[state["case"]["op"]](state)


def _framework():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "distributed-hipkittens_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import hkmoe
    return hkmoe


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_linear(case, seed):
    d = _linear_inputs(case, seed)
    a, b = d["a"].double(), d["b"].double()
    if case["mx"]:
        a, b = a * _powers(d["sa"]), b * _powers(d["sb"])
    else:
        a = a * (d["sa"].double() * d["sb"].double())
    z = torch.mm(a, b.t())
    if case["bias"]:
        z += d["bias"].double()
    act = case["act"]
    if act == "relu":
        z = z.clamp_min(0.0)
    elif act == "silu":
        z = z * torch.sigmoid(z)
    elif act == "gelu":
        z = z * torch.special.ndtr(z)
    elif act == "gelu_tanh":  # (1 + tanh u) / 2 is the logistic function of 2 u
        z = z * torch.sigmoid(math.sqrt(8.0 / math.pi) * z * (1.0 + 0.044715 * z ** 2))
    return z if d["residual"] is None else z + d["residual"].double()


def _exact_norm(case, seed):
    d = _norm_inputs(case, seed)
    C = case["C"]
    r = d["x"].double()
    if case["residual"]:  # the stream is kept in its own type, and the norm reads what is kept
        r = (r + d["residual"].double()).to(d["x"].dtype).double()
    c = r - r.sum(1, keepdim=True) / C
    rstd = ((c * c).sum(1, keepdim=True) / C + EPS) ** -0.5
    w = d["weight"].double()
    out = dict(y=c * rstd * w + d["bias"].double(), r=r if case["residual"] else None)
    if not case["grad"]:
        return out
    dy = d["dy"].double()
    g = dy * w
    # through n = c rstd: dc = rstd g - rstd^3 c (g . c) / C; through the mean: less its own mean
    dc = rstd * g - rstd ** 3 * c * (g * c).sum(1, keepdim=True) / C
    dx = dc - dc.sum(1, keepdim=True) / C
    if d["dr"] is not None:
        dx += d["dr"].double()
    return dict(out, dx=dx, dw=(dy * c * rstd).sum(0), db=dy.sum(0))


def _exact_permute(case, seed):
    d = _permute_inputs(case, seed)
    T, k, H, ids = case["T"], case["k"], case["H"], d["ids"].flatten()
    slots = [(ids == e).nonzero()[:, 0] for e in range(case["E"])]
    p = torch.cat(slots)
    xp = torch.zeros((T * k, H), dtype=torch.float64, device=DEV)
    xp[: p.numel()] = d["x"].double()[p // k]
    out = dict(xp=xp, offsets=None, perm=None)
    if case["grad"]:
        out["dx"] = torch.zeros((T, H), dtype=torch.float64, device=DEV)
        out["dx"].index_add_(0, p // k, d["dxp"][: p.numel()].double())
    return out


def _exact_combine(case, seed):
    d = _combine_inputs(case, seed)
    T, k, H, ids = case["T"], case["k"], case["H"], d["ids"].flatten()
    p = torch.cat([(ids == e).nonzero()[:, 0] for e in range(case["E"])])
    y, dout, w = d["y"][: p.numel()].double(), d["dout"].double(), d["w"].double().flatten()
    out = torch.zeros((T, H), dtype=torch.float64, device=DEV)
    out.index_add_(0, p // k, y * w[p, None])
    dw = torch.zeros(T * k, dtype=torch.float64, device=DEV)
    dw[p] = (y * dout[p // k]).sum(1)
    dy = torch.zeros((T * k, H), dtype=torch.float64, device=DEV)
    dy[: p.numel()] = dout[p // k] * w[p, None]
    w, dw = w.view(T, k), dw.view(T, k)
    dlogits = torch.zeros((T, case["E"]), dtype=torch.float64, device=DEV)
    # softmax over the chosen k: dl_j = sum_i dw_i w_i (delta_ij - w_j)
    jac = torch.diag_embed(w) - w[:, :, None] * w[:, None, :]
    dlogits.scatter_(1, d["idx"].long(), (jac * dw[:, :, None]).sum(1))
    return dict(out=out, dy=dy, dw=dw, dlogits=dlogits)


EXACT = {"linear": _exact_linear, "norm": _exact_norm, "permute": _exact_permute, "combine": _exact_combine}


def exact(case, seed):
    return EXACT[case["op"]](case, seed)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        b = 2 if case["out"] == "bf16" else 4
        scales = (M + N) * K // 32 if case["mx"] else 8
        return {"bytes": (M + N) * K + scales + b * M * N * (2 if case["residual"] else 1) + (b * N if case["bias"] else 0),
                "flops": 2 * M * N * K}
    b = 2 if case["dtype"] == "bf16" else 4
    if op == "norm":
        T, C = case["T"], case["C"]
        wb = 2 if case["weight"] == "bf16" else 4
        each = (4 if case["residual"] else 2) + ((3 if case["residual"] else 2) if case["grad"] else 0)
        return {"bytes": b * T * C * each + wb * C * (4 if case["grad"] else 2), "flops": T * C * (18 if case["grad"] else 8)}
    T, H, k = case["T"], case["H"], case["k"]
    live = int(T * k * (1.0 - case["drop"]))  # slots with an expert here
    if op == "permute":
        rows = T + T * k + (live + T if case["grad"] else 0)
        return {"bytes": b * H * rows + 4 * (2 * T * k + case["E"] + 1), "flops": H * live if case["grad"] else T * k}
    rows = live + T + T + T * k  # y and dout in, out and dy out
    return {"bytes": b * H * rows + 4 * (5 * T * k + T * case["E"]), "flops": 5 * H * live}
