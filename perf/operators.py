"""Cases of the operators around the FP8 products: what turns a residual stream
into their operands, and what is added beside them.

Each case is one call that a serving program makes per layer on tensors already
on the GPU:

  op "norm"    hkmoe.rms_norm_quant: the residual's addition, the root-mean-square
               norm and the e4m3 operand with its scales (1x128 groups, 1x32 e8m0
               or one per tensor), beside the new residual and the bf16 norm
  op "router"  hkmoe.router_logits: the bf16 norm times the router's weight, fp32
  op "lora"    hkmoe.lora_add: the low-rank adapters of many requests, added to
               the output of a shared projection

``own`` chooses between the framework's calls and the plain forms below (the
same formulas in elementary fp32 operations).
"""
import math
import os
import sys

import torch

own = False  # True: the framework's calls

F8 = torch.float8_e4m3fn
E8 = torch.float8_e8m0fnu
DEV = "cuda"
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _norm(T, H, scales, dtype="bf16", residual=True, norm=False, static=False):
    return dict(op="norm", T=T, H=H, scales=scales, dtype=dtype, residual=residual, norm=norm, static=static)


def _router(T, H, E):
    return dict(op="router", T=T, H=H, E=E)


def _lora(T, H, N, R, L, used, bare=0, out="bf16", segments=True, wide=0):
    """T rows of which ``bare`` have no adapter and the others share ``used`` of
    L resident ones, in one segment per adapter or shuffled; the projection's
    output is a slice of a buffer that is ``wide`` columns wider."""
    return dict(op="lora", T=T, H=H, N=N, R=R, L=L, used=used, bare=bare, out=out, segments=segments, wide=wide)


def listed():
    return [
        # one token in front of the benchmark's decode layer: launch latency
        dict(name="norm_group_1", **_norm(1, 4096, "group", norm=True)),
        # an odd decode batch in front of an MX linear layer, no residual yet
        dict(name="norm_mx_61", **_norm(61, 2560, "mx", residual=False)),
        # a ragged prefill chunk from an fp32 stream, one scale for the tensor
        dict(name="norm_tensor_1777", **_norm(1777, 4096, "tensor", dtype="f32")),
        # the benchmark's flagship prefill: the layer's operands and the router's
        dict(name="norm_group_8192", **_norm(8192, 7168, "group", norm=True)),
        # the routers of the same layers: one token, the decode batch, a small
        # router over an odd chunk, the flagship prefill
        dict(name="router_1", **_router(1, 4096, 128)),
        dict(name="router_64", **_router(64, 4096, 128)),
        dict(name="router_1999", **_router(1999, 2048, 60)),
        dict(name="router_8192", **_router(8192, 7168, 256)),
        # adapters: one interactive request; a decode batch in which most
        # requests have their own; an odd chunk into a slice of a fused
        # projection, fp32; a prefill of eight ragged requests, one without
        dict(name="lora_1", **_lora(1, 4096, 4096, 16, 8, 1)),
        dict(name="lora_decode_64", **_lora(64, 4096, 4096, 16, 64, 40, bare=3, segments=False)),
        dict(name="lora_slice_777", **_lora(777, 2560, 1024, 24, 16, 5, bare=100, out="f32", wide=512)),
        dict(name="lora_prefill_8192", **_lora(8192, 7168, 4096, 64, 8, 7, bare=900)),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "router", "lora"])
    if op == "norm":
        scales = rng.choice(["group", "mx", "tensor"])
        H = 128 * _log_int(rng, 4, 128)
        dtype = rng.choice(["bf16", "bf16", "f32"])
        T = _log_int(rng, 1, max(1, min(16384, 8192 * 7168 // H // (1 if dtype == "bf16" else 2))))
        return _norm(T, H, scales, dtype, rng.random() < 0.8, rng.random() < 0.5,
                     scales == "tensor" and rng.random() < 0.5)
    if op == "router":
        H, E = 8 * _log_int(rng, 64, 1024), _log_int(rng, 4, 512)
        return _router(_log_int(rng, 1, max(1, min(16384, 8192 * 7168 * 256 // (H * E)))), H, E)
    H, N, R = 8 * _log_int(rng, 64, 1024), 8 * _log_int(rng, 32, 1024), 8 * _log_int(rng, 1, 16)
    T = _log_int(rng, 1, min(8192, 8192 * 11264 // (H + N)))
    bare = rng.randrange(T // 8 + 1)
    most = max(1, min(64, T - bare, 8192 * 512 * 11264 // (T * R * (H + N))))
    used = _log_int(rng, 1, most)
    return _lora(T, H, N, R, used + rng.randrange(max(1, most - used + 1)), used, bare, rng.choice(["bf16", "bf16", "f32"]),
                 rng.random() < 0.6, rng.choice([0, 0, 256]))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)


def _norm_inputs(case, seed):
    g = _gen(seed)
    T, H, dtype = case["T"], case["H"], DTYPES[case["dtype"]]
    # a residual stream: a few channels are many times larger than the others
    gain = torch.ones(H, device=DEV)
    gain[torch.randperm(H, generator=g, device=DEV)[: max(1, H // 256)]] = 20.0
    d = dict(case=case, x=_randn(g, T, H).to(dtype), residual=None, scale=None)
    if case["residual"]:
        d["residual"] = (3.0 * _randn(g, T, H) * gain).to(dtype)
    else:
        d["x"] = (d["x"].float() * gain).to(dtype)
    d["weight"] = (1.0 + 0.2 * _randn(g, H)).to(dtype)
    if case["static"]:
        d["scale"] = torch.full((1,), 0.02, device=DEV)
    return d


def _router_inputs(case, seed):
    g = _gen(seed)
    return dict(case=case, x=_randn(g, case["T"], case["H"]).to(torch.bfloat16),
                w=(_randn(g, case["E"], case["H"]) * case["H"] ** -0.5).to(torch.bfloat16))


def _lora_ids(case, g):
    """Adapter of each row: ``used`` distinct ones, of ragged sizes, -1 for ``bare`` rows."""
    T, L, used, bare = case["T"], case["L"], case["used"], case["bare"]
    which = torch.randperm(L, generator=g, device=DEV)[:used]
    more = (used * torch.rand(T - bare - used, generator=g, device=DEV) ** 2).long().clamp_max(used - 1)
    ids = torch.cat([which, which[more], torch.full((bare,), -1, dtype=torch.long, device=DEV)])
    ids = ids.sort()[0] if case["segments"] else ids[torch.randperm(T, generator=g, device=DEV)]
    return ids.to(torch.int32)


def _lora_inputs(case, seed):
    g = _gen(seed)
    T, H, N, R, L = (case[k] for k in ("T", "H", "N", "R", "L"))
    d = dict(case=case, x=_randn(g, T, H).to(torch.bfloat16), ids=_lora_ids(case, g))
    d["a"] = (_randn(g, L, R, H) * H ** -0.5).to(torch.bfloat16)
    d["b"] = (_randn(g, L, N, R) * R ** -0.5).to(torch.bfloat16)
    d["scaling"] = 0.5 + torch.rand(L, generator=g, device=DEV)
    d["y"] = _randn(g, T, N + case["wide"]).to(DTYPES[case["out"]])[:, case["wide"]:]
    return d


INPUTS = {"norm": _norm_inputs, "router": _router_inputs, "lora": _lora_inputs}


def prepare(case, seed):
    return INPUTS[case["op"]](case, seed)


# ---------------------------------------------------------------------------
# plain forms: fp32, rounded once at the end; a row's mean in 64 bits
# ---------------------------------------------------------------------------
def _scale_of(amax):
    # a tensor divisor: torch multiplies by the reciprocal of a scalar one
    s = (amax / torch.full_like(amax, 448.0)).clamp_min(2.0 ** -126)
    return torch.where(amax > 0, s, torch.ones_like(s))


def _quant(n, scales, scale):
    if scales == "group":
        v = n.view(n.shape[0], -1, 128)
        s = _scale_of(v.abs().amax(2))
        return (v / s[..., None]).clamp(-448, 448).to(F8).view(n.shape), s
    if scales == "mx":
        v = n.view(n.shape[0], -1, 32)
        e = ((v.abs().amax(2).view(torch.int32) >> 23) & 0xFF).clamp_max(254)
        return torch.ldexp(v, (127 - e)[..., None]).to(F8).view(n.shape), e.to(torch.uint8).view(E8)
    s = _scale_of(n.abs().amax().reshape(1)) if scale is None else scale
    return (n / s).clamp(-448, 448).to(F8), s


def _plain_norm(d):
    case, x = d["case"], d["x"]
    r = x if d["residual"] is None else (x.float() + d["residual"].float()).to(x.dtype)
    v = r.float()
    # the mean of a long row in 64 bits: q and the exponents change where n crosses a border
    rstd = (1.0 / (v.double().square().mean(1, keepdim=True) + EPS).sqrt()).float()
    n = v * rstd * d["weight"].float()
    q, s = _quant(n, case["scales"], d["scale"])
    return dict(q=q, s=s, residual=r if case["residual"] else None, norm=n.to(torch.bfloat16) if case["norm"] else None)


def _plain_lora(d):
    a, b, ids, y = d["a"].float(), d["b"].float(), d["ids"], d["y"]
    L, R, H = a.shape
    # every adapter's product, then only the row's own one
    v = (d["x"].float() @ a.view(L * R, H).T).view(-1, L, R)
    mine = ids[:, None] == torch.arange(L, device=ids.device, dtype=ids.dtype)
    v = torch.where(mine[..., None], v * d["scaling"][:, None], torch.zeros_like(v))
    return (y.float() + v.view(-1, L * R) @ b.transpose(1, 2).reshape(L * R, -1)).to(y.dtype)


def run(state):
    case = state["case"]
    if own:
        hkmoe = _framework()
        if case["op"] == "norm":
            q, s, r, n = hkmoe.rms_norm_quant(state["x"], state["weight"], state["residual"], scales=case["scales"],
                                              scale=state["scale"], eps=EPS, with_norm=case["norm"])
            return dict(q=q, s=s.view(E8) if case["scales"] == "mx" else s, residual=r if case["residual"] else None, norm=n)
        if case["op"] == "router":
            return hkmoe.router_logits(state["x"], state["w"])
        return hkmoe.lora_add(state["y"], state["x"], state["a"], state["b"], state["ids"], state["scaling"])
    if case["op"] == "norm":
        return _plain_norm(state)
    if case["op"] == "router":
        return state["x"].float() @ state["w"].float().T
    return _plain_lora(state)


def _framework():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "distributed-hipkittens_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import hkmoe
    return hkmoe


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _e4m3_64(v):
    """Nearest e4m3 value (ties to even, saturating) of 64-bit values."""
    e = torch.frexp(v)[1] - 1
    step = torch.exp2((e.clamp_min(-6) - 3).double())
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def _exact_norm(case, seed):
    d = _norm_inputs(case, seed)
    r = d["x"].double()
    if case["residual"]:  # the stream is kept in its own type, and the norm reads what is kept
        r = (r + d["residual"].double()).to(d["x"].dtype).double()
    n = d["weight"].double() * r / ((r * r).sum(1, keepdim=True) / case["H"] + EPS).sqrt()
    if case["scales"] == "tensor":
        s = d["scale"].double() if case["static"] else (n.abs().max() / 448.0).reshape(1)
        q = _e4m3_64(n / s)
    else:
        width = 128 if case["scales"] == "group" else 32
        blocks = n.reshape(case["T"], case["H"] // width, width)
        top = blocks.abs().amax(2)
        s = top / 448.0 if width == 128 else torch.exp2((torch.frexp(top)[1] - 1).double())
        q = _e4m3_64(blocks / s[..., None]).reshape(n.shape)
    return dict(q=q, s=s, residual=r if case["residual"] else None, norm=n if case["norm"] else None)


def _exact_lora(case, seed):
    d = _lora_inputs(case, seed)
    out = d["y"].double()
    for l in d["ids"].unique().tolist():
        if l < 0:
            continue
        t = (d["ids"] == l).nonzero()[:, 0]
        out[t] += d["scaling"][l].double() * ((d["x"][t].double() @ d["a"][l].double().T) @ d["b"][l].double().T)
    return out


def exact(case, seed):
    if case["op"] == "norm":
        return _exact_norm(case, seed)
    if case["op"] == "lora":
        return _exact_lora(case, seed)
    d = _router_inputs(case, seed)
    return d["x"].double() @ d["w"].double().T


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    T, H = case["T"], case["H"]
    if case["op"] == "norm":
        b = 2 if case["dtype"] == "bf16" else 4
        each = b * (3 if case["residual"] else 1) + 1 + (2 if case["norm"] else 0)
        scales = {"group": T * H // 128 * 4, "mx": T * H // 32, "tensor": 4}[case["scales"]]
        return {"bytes": T * H * each + H * b + scales, "flops": 7 * T * H}
    if case["op"] == "router":
        return {"bytes": 2 * T * H + 2 * case["E"] * H + 4 * T * case["E"], "flops": 2 * T * H * case["E"]}
    N, R, rows = case["N"], case["R"], T - case["bare"]
    b = 2 if case["out"] == "bf16" else 4
    return {"bytes": 2 * rows * H + 2 * case["used"] * R * (H + N) + 2 * b * T * N + 4 * T,
            "flops": 2 * rows * R * (H + N)}
