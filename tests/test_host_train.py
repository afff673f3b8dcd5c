"""Dense products with an epilogue, layer norm, tokens by expert and their gradients: what the
host refuses and launches, and the formulas against differences (no GPU)."""
import ctypes
import os
import re

import numpy as np
import pytest
import torch

import hip_host
import test_gpu_epilogue
import test_host_block
import train_ref as ref

P = ctypes.c_void_p(0x1000)  # never dereferenced: validation fails first
Q = ctypes.c_void_p(0x2000)
ODD = ctypes.c_void_p(0x1008)
i64, i32, dbl, size = ctypes.c_int64, ctypes.c_int32, ctypes.c_double, ctypes.c_size_t


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(os.environ.get("HKMOE_LIB") or hip_host.LIB)
    lib.hkmoe_last_error.restype = ctypes.c_char_p
    lib.hkmoe_layer_norm_backward_workspace_size.restype = size
    lib.hkmoe_permute_workspace_size.restype = size
    return lib


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    return hip_host.build_fake(str(tmp_path_factory.mktemp("fake_hip")))


def _refused(lib, call, bad, says):
    assert call(lib, **bad) == 1, bad
    assert says in lib.hkmoe_last_error().decode(), lib.hkmoe_last_error()


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
def _fp8(lib, a=P, b=P, c=P, m=4, n=256, k=128, out=0, bias=None, bt=0, act=1, res=None):
    return lib.hkmoe_gemm_fp8_epilogue(a, b, c, i64(m), i64(n), i64(k), None, None, out, bias, bt, act, res, None)


def _mx(lib, a=P, b=P, c=P, m=4, n=256, k=128, out=0, bias=None, bt=0, act=1, res=None, sa=P, sb=P):
    return lib.hkmoe_gemm_mx_epilogue(a, sa, b, sb, c, i64(m), i64(n), i64(k), out, bias, bt, act, res, None)


@pytest.mark.parametrize("call", [_fp8, _mx])
@pytest.mark.parametrize("bad,says", [
    (dict(a=None), "null"), (dict(b=None), "null"), (dict(c=None), "null"), (dict(m=-1), "shape"), (dict(n=0), "shape"),
    (dict(k=130), "multiple of 128"), (dict(n=128), "multiple of 256"), (dict(n=(1 << 21) + 256), "2^21"), (dict(out=2), "out_dtype"),
    (dict(m=1 << 26), "too large"), (dict(act=5), "activation"), (dict(act=-1), "activation"), (dict(bias=P, bt=2), "bias_dtype"),
    (dict(bias=ODD), "aligned"), (dict(res=ODD), "aligned"), (dict(c=ODD), "aligned")])
def test_epilogue_refusals(lib, call, bad, says):
    _refused(lib, call, bad, says)


def test_epilogue_no_rows(lib):
    assert _fp8(lib, a=None, c=None, m=0, bias=P) == 0 and _mx(lib, a=None, c=None, sa=None, m=0, res=P) == 0
    _refused(lib, _mx, dict(sa=None), "null")
    _refused(lib, _mx, dict(sb=None, m=0), "null")


def _norm(lib, x=P, residual=None, weight=P, bias=None, rows=4, cols=256, xt=0, wt=0, eps=1e-5, y=P, residual_out=None, stats=P):
    return lib.hkmoe_layer_norm(x, residual, weight, bias, i64(rows), i64(cols), xt, wt, dbl(eps), y, residual_out, stats, None)


def _norm_grad(lib, dy=P, r=P, weight=P, dr=None, stats=P, rows=4, cols=256, xt=0, wt=0, dx=Q, dw=P, db=None, ws=P, ws_bytes=1 << 40):
    return lib.hkmoe_layer_norm_backward(dy, r, weight, dr, stats, i64(rows), i64(cols), xt, wt, dx, dw, db, ws, size(ws_bytes), None)


@pytest.mark.parametrize("bad,says", [
    (dict(x=None), "null"), (dict(weight=None), "null"), (dict(y=None), "null"), (dict(stats=None), "null"), (dict(rows=-1), "shape"),
    (dict(rows=(1 << 24) + 1), "shape"), (dict(cols=0), "multiple of 8"), (dict(cols=12), "multiple of 8"), (dict(cols=16392), "16384"),
    (dict(xt=2), "dtype"), (dict(wt=5), "dtype"), (dict(eps=0.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"),
    (dict(residual=P), "together"), (dict(residual_out=P), "together"), (dict(x=ODD), "aligned"), (dict(y=ODD), "aligned"),
    (dict(bias=ODD), "aligned"), (dict(stats=ODD), "aligned"), (dict(weight=ODD), "aligned")])
def test_norm_refusals(lib, bad, says):
    _refused(lib, _norm, bad, says)


@pytest.mark.parametrize("bad,says", [
    (dict(dy=None), "null"), (dict(r=None), "null"), (dict(weight=None), "null"), (dict(stats=None), "null"), (dict(dx=None), "null"),
    (dict(dw=None), "null"), (dict(rows=-1), "shape"), (dict(cols=4), "multiple of 8"), (dict(cols=16392), "16384"), (dict(xt=3), "dtype"),
    (dict(wt=-1), "dtype"), (dict(dy=ODD), "aligned"), (dict(dr=ODD), "aligned"), (dict(dx=ODD), "aligned"), (dict(dw=ODD), "aligned"),
    (dict(db=ODD), "aligned"), (dict(dx=P), "neither dy nor r"), (dict(dx=P, dy=Q), "neither dy nor r"), (dict(dx=P, r=Q), "neither dy nor r")])
def test_norm_gradient_refusals(lib, bad, says):
    _refused(lib, _norm_grad, bad, says)


def test_norm_workspace(lib):
    need = lib.hkmoe_layer_norm_backward_workspace_size(i64(600), i64(256))
    assert need > 0 and lib.hkmoe_layer_norm_backward_workspace_size(i64(4), i64(256)) == 0  # one launch
    for bad in (dict(ws=None), dict(ws_bytes=need - 1), dict(ws=ODD)):
        assert _norm_grad(lib, rows=600, **bad) == 4
    for rows, cols in ((0, 256), (-1, 256), (2 ** 62, 256), (4, 0), (4, 2 ** 62), (4, 16392)):
        assert lib.hkmoe_layer_norm_backward_workspace_size(i64(rows), i64(cols)) == 0
    assert lib.hkmoe_layer_norm_backward_workspace_size(i64(1 << 24), i64(16384)) >= 2 * 16384 * 4
    assert _norm(lib, rows=0, x=None, y=None, stats=None) == 0


def _permute(lib, x=P, ids=P, t=4, e=8, k=2, h=64, dt=0, xp=P, offsets=P, perm=P, inv=P, ws=P, ws_bytes=1 << 40):
    return lib.hkmoe_permute(x, ids, i64(t), i32(e), i32(k), i64(h), dt, xp, offsets, perm, inv, ws, size(ws_bytes), None)


def _combine(lib, y=P, w=None, offsets=P, inv=P, t=4, e=8, k=2, h=64, dt=0, out=P):
    return lib.hkmoe_combine_rows(y, w, offsets, inv, i64(t), i32(e), i32(k), i64(h), dt, out, None)


def _combine_grad(lib, dout=P, y=P, w=P, offsets=P, inv=P, t=4, e=8, k=2, h=64, dt=0, dy=P, dw=P):
    return lib.hkmoe_combine_rows_backward(dout, y, w, offsets, inv, i64(t), i32(e), i32(k), i64(h), dt, dy, dw, None)


def _route_grad(lib, dw=P, w=P, idx=P, t=4, e=8, k=2, out=P):
    return lib.hkmoe_route_topk_backward(dw, w, idx, i64(t), i32(e), i32(k), out, None)


SLOTS = [(dict(t=-1), "shape"), (dict(t=(1 << 24) + 1), "shape"), (dict(k=0), "shape"), (dict(k=33), "shape"), (dict(e=0), "E=0"),
         (dict(e=1025), "E=1025")]
ROWS = SLOTS + [(dict(h=12), "multiple of 8"), (dict(h=0), "multiple of 8"), (dict(h=(1 << 24) + 8), "2^24"), (dict(dt=3), "dtype")]


@pytest.mark.parametrize("bad,says", ROWS + [
    (dict(x=None), "null"), (dict(ids=None), "null"), (dict(xp=None), "null"), (dict(offsets=None), "null"), (dict(perm=None), "null"),
    (dict(inv=None), "null"), (dict(x=ODD), "aligned"), (dict(xp=ODD), "aligned"), (dict(dt=2, h=24), "multiple of 16")])
def test_permute_refusals(lib, bad, says):
    _refused(lib, _permute, bad, says)


@pytest.mark.parametrize("bad,says", ROWS + [
    (dict(y=None), "null"), (dict(offsets=None), "null"), (dict(inv=None), "null"), (dict(out=None), "null"), (dict(y=ODD), "aligned"),
    (dict(out=ODD), "aligned"), (dict(dt=2), "dtype")])
def test_combine_refusals(lib, bad, says):
    _refused(lib, _combine, bad, says)


@pytest.mark.parametrize("bad,says", ROWS + [
    (dict(dout=None), "null"), (dict(y=None), "null"), (dict(w=None), "null"), (dict(offsets=None), "null"), (dict(inv=None), "null"),
    (dict(dy=None), "null"), (dict(dw=None), "null"), (dict(dout=ODD), "aligned"), (dict(y=ODD), "aligned"), (dict(dy=ODD), "aligned"),
    (dict(dt=2), "dtype")])
def test_combine_gradient_refusals(lib, bad, says):
    _refused(lib, _combine_grad, bad, says)


@pytest.mark.parametrize("bad,says", SLOTS + [
    (dict(dw=None), "null"), (dict(w=None), "null"), (dict(idx=None), "null"), (dict(out=None), "null"), (dict(e=1), "E=1 outside")])
def test_route_gradient_refusals(lib, bad, says):
    _refused(lib, _route_grad, bad, says)


def test_permute_workspace(lib):
    f = lambda t, e, k: lib.hkmoe_permute_workspace_size(i64(t), i32(e), i32(k))  # noqa: E731
    assert f(4, 8, 2) == 0 and f(2048, 8, 2) == 0 and _permute(lib, t=0, x=None, ids=None, xp=None, perm=None, inv=None, e=0) == 1
    for t, e, k in ((0, 8, 2), (-1, 8, 2), (2 ** 62, 8, 2), (1 << 20, 0, 2), (1 << 20, 1025, 2), (1 << 20, 8, 0), (1 << 20, 8, 33)):
        assert f(t, e, k) == 0
    need = f(4096, 8, 2)
    assert need > 0
    assert _permute(lib, t=4096, ws=None) == 4 and _permute(lib, t=4096, ws_bytes=need - 1) == 4 and _permute(lib, t=4096, ws=ODD) == 4
    assert f(1 << 24, 1024, 32) < 1 << 22  # the sorting workgroups are few, however many slots there are


STAND_IN = test_host_block.STAND_IN + """
class There(T):
    def data_ptr(self): return 0x2000
f8, bf = "torch.float8_e4m3fn", "torch.bfloat16"
def gemm(a=T([4, 128], f8), b=T([256, 128], f8), c=T([4, 256]), bias=None, res=None):
    tk_kernel.dispatch_gemm_fp8_epilogue(a, b, c, None, None, bias, 1, res)
def norm(x=T([4, 64]), w=T([64]), b=None, y=T([4, 64]), st=T([4, 4], f32), r=None, ro=None):
    tk_kernel.dispatch_layer_norm(x, r, w, b, 1e-5, y, ro, st)
def norm_grad(dy=T([600, 64]), r=T([600, 64]), w=T([64]), dr=None, st=T([600, 4], f32), dx=There([600, 64]), dw=T([64]), ws=T([1 << 20], u8)):
    tk_kernel.dispatch_layer_norm_backward(dy, r, w, dr, st, dx, dw, None, ws)
def permute(x=T([4, 64]), ids=T([4, 2], i32), xp=T([8, 64]), off=T([9], i32), perm=T([8], i32), inv=T([4, 2], i32)):
    tk_kernel.dispatch_permute(x, ids, xp, off, perm, inv, None)
def combine(y=T([8, 64]), w=T([4, 2], f32), off=T([9], i32), inv=T([4, 2], i32), out=T([4, 64])):
    tk_kernel.dispatch_combine_rows(y, w, off, inv, out)
def combine_grad(dout=T([4, 64]), y=T([8, 64]), w=T([4, 2], f32), off=T([9], i32), inv=T([4, 2], i32), dy=T([8, 64]), dw=T([4, 2], f32)):
    tk_kernel.dispatch_combine_rows_backward(dout, y, w, off, inv, dy, dw)
def route_grad(dw=T([4, 2], f32), w=T([4, 2], f32), idx=T([4, 2], i32), out=T([4, 8], f32)):
    tk_kernel.dispatch_route_topk_backward(dw, w, idx, out)
"""


def test_tensors_of_another_device_and_shape(fake):
    """What the binding asks of each tensor, and the stream that every launch goes to."""
    out = hip_host.run(fake, STAND_IN + """
for f in (gemm, norm, norm_grad, permute, combine, combine_grad, route_grad): f()
for line in log(): print(line)
other = dict(dev=1)
refused(lambda: gemm(res=T([4, 256], **other)))
refused(lambda: gemm(bias=T([256], dev=-1)))
refused(lambda: gemm(bias=T([2, 128])))
refused(lambda: gemm(c=T([4, 256], strides=(512, 1))))
refused(lambda: norm(x=T([4, 64], **other)))
refused(lambda: norm(st=T([4, 4])))
refused(lambda: norm(r=T([4, 64])))
refused(lambda: norm_grad(dy=T([400, 64], f32)))
refused(lambda: norm_grad(ws=T([1 << 20], i32)))
refused(lambda: permute(ids=T([4, 2], i32, **other)))
refused(lambda: permute(xp=T([7, 64])))
refused(lambda: permute(perm=T([8], f32)))
refused(lambda: permute(inv=T([2, 4], i32)))
refused(lambda: combine(w=T([4, 2])))
refused(lambda: combine(off=T([9, 1], i32)))
refused(lambda: combine_grad(dy=T([8, 64], strides=(128, 1))))
refused(lambda: combine_grad(dw=T([4, 3], f32)))
refused(lambda: route_grad(idx=T([4, 2], f32)))
refused(lambda: route_grad(out=T([5, 8], f32)))
""")
    launches = [l for l in out if l.startswith("launch")]
    assert len(launches) == 8 and all(l.endswith("stream=7") for l in launches), out
    said = [l.split(": ", 1)[1] for l in out if l.startswith("refused")]
    wanted = ["residual: tensor must be on the current device", "bias: tensor must be on a GPU device", "bias must be [N]",
              "C: tensor must be contiguous", "x: tensor must be on the current device", "stats must be [R, 4] float32",
              "residual and residual_out come together", "dy must have r's shape and dtype",
              "workspace: expected dtype torch.uint8, got torch.int32", "ids: tensor must be on the current device",
              "xp: expected [8, 64] torch.bfloat16", "perm: expected 8 int32 values", "ids must be [T, k] int32",
              "topk_w: expected [4, 2] torch.float32", "offsets: expected 1-D tensor", "dy: tensor must be contiguous",
              "dw: expected [4, 2] torch.float32", "topk_idx: expected dtype torch.int32", "dlogits: expected [4, 8] torch.float32"]
    assert said == wanted and "taken" not in out, said


# ---------------------------------------------------------------------------
# launches
# ---------------------------------------------------------------------------
LAUNCH = """
Q = ctypes.c_void_p(0x2000)
size, dbl = ctypes.c_size_t, ctypes.c_double
def norm(rows, cols, xt=0):
    assert lib.hkmoe_layer_norm(P, P, P, P, i64(rows), i64(cols), xt, 0, dbl(1e-5), P, P, P, None) == 0, lib.hkmoe_last_error()
    assert lib.hkmoe_layer_norm_backward(P, P, P, P, P, i64(rows), i64(cols), xt, 0, Q, P, P, P, size(1 << 50), None) == 0
def tokens(t, e, k, h, dt=0):
    assert lib.hkmoe_permute(P, P, i64(t), i32(e), i32(k), i64(h), dt, P, P, P, P, P, size(1 << 50), None) == 0
    assert lib.hkmoe_combine_rows(P, P, P, P, i64(t), i32(e), i32(k), i64(h), dt, P, None) == 0
    assert lib.hkmoe_combine_rows_backward(P, P, P, P, P, i64(t), i32(e), i32(k), i64(h), dt, P, P, None) == 0
    if k <= e:
        assert lib.hkmoe_route_topk_backward(P, P, P, i64(t), i32(e), i32(k), P, None) == 0
def act(m, n, k, f32, mx):
    if mx:
        assert lib.hkmoe_gemm_mx_epilogue(P, P, P, P, P, i64(m), i64(n), i64(k), int(f32), P, 1, 3, P, None) == 0
    else:
        assert lib.hkmoe_gemm_fp8_epilogue(P, P, P, i64(m), i64(n), i64(k), P, P, int(f32), P, 0, 2, P, None) == 0
"""


def test_every_grid_dimension_in_range(fake):
    """The sizes where launches change, and the largest that are taken: below 2^32 work-items."""
    out = hip_host.run(fake, LAUNCH + """
for rows in (1, 255, 256, 257, 4096, 1 << 20, (1 << 20) + 1, 1 << 24):
    for cols in (8, 128, 136, 256, 512, 520, 1024, 1032, 8192, 8200, 16384):
        norm(rows, cols)
        norm(rows, cols, 1)
    for e, k in ((1, 1), (1, 32), (1024, 1), (1024, 32)):
        for h in (8, 4096, 4104, 1 << 24):
            tokens(rows, e, k, h)
            tokens(rows, e, k, h, 1)
for line in log(): print(line)
""")
    launches = [l for l in out if l.startswith("launch")]
    names = {l.split()[1] for l in launches}
    assert len([n for n in names if "layer_norm_kernel" in n]) == 12 and len([n for n in names if "layer_norm_grad_kernel" in n]) == 24
    for l in launches:
        v = {k: int(n) for k, n in (f.split("=") for f in l.split()[2:])}
        assert 1 <= v["grid"] and v["grid"] * v["threads"] < 1 << 32 and v["y"] == v["z"] == 1 and 64 <= v["threads"] <= 1024, l


def test_epilogue_shapes_reach_every_kernel(fake):
    """The GPU test's shapes run on every strip, with bf16 C on 128x128 and 256x256 tiles of the FP8
    instructions, with fp32 C on both tiles that widen the operands.  (strips: MX, fp32 output, epilogue)"""
    for mx in (0, 1):
        for f32 in (0, 1):
            out = hip_host.run(fake, LAUNCH + f"""
for s in {test_gpu_epilogue.SHAPES!r}: act(*s, {f32}, {mx})
for line in log(): print(line)
""")
            got = set()
            for line in out:
                m = re.match(r"launch hkmoe::gemm_fp8_(skinny<(\d), *_?(\d), *_?(\d), *_?(\w+), *_?(\w+), *_?(\w+)>|small_act|wide256|wide|persistent)", line)
                if m.group(2):
                    assert m.group(5, 6, 7) == tuple("true" if v else "false" for v in (mx, f32, 1)), line
                got.add(f"strip {m.group(2)}x{m.group(3)}" if m.group(2) else m.group(1))
            want = {"strip 1x1", "strip 2x1", "strip 1x2", "strip 2x2", "strip 2x4", "strip 4x4"}
            assert got == want | ({"wide", "wide256"} if f32 else {"small_act", "persistent"}), (mx, f32, got)


def test_few_rows_need_one_launch_for_the_gradient(fake):
    """Workgroups for the columns beside the rows', and past some rows partial sums and a second launch."""
    out = hip_host.run(fake, LAUNCH + """
for rows, cols in ((1, 4096), (512, 4096), (512, 128), (1024, 4104), (1024, 16384), (513, 4096), (513, 128), (1025, 16384), (0, 128)):
    assert lib.hkmoe_layer_norm_backward(P, P, P, P, P, i64(rows), i64(cols), 0, 0, Q, P, P, P, size(1 << 50), None) == 0
    print(len(log()))
""")
    assert [int(v) for v in out] == [1, 1, 1, 1, 1, 2, 2, 2, 1]


def test_small_batches_sort_in_one_launch(fake):
    out = hip_host.run(fake, LAUNCH + """
for t, k in ((1, 1), (256, 8), (2048, 2), (724, 8), (2049, 2), (725, 8), (1 << 24, 1)):
    assert lib.hkmoe_permute(P, P, i64(t), i32(64), i32(k), i64(64), 0, P, P, P, P, P, size(1 << 50), None) == 0
    print(len(log()))
""")
    assert [int(v) for v in out] == [1, 1, 1, 1, 3, 3, 3]


# ---------------------------------------------------------------------------
# formulas
# ---------------------------------------------------------------------------
def _differences(f, x, h=1e-5):
    """Central differences of the scalar f at x (64 bits)."""
    g = torch.zeros_like(x)
    flat, out = x.view(-1), g.view(-1)
    for i in range(flat.numel()):
        keep = flat[i].item()
        flat[i] = keep + h
        up = f()
        flat[i] = keep - h
        out[i] = (up - f()) / (2 * h)
        flat[i] = keep
    return g


def _near(a, b):
    assert float((a - b).abs().max()) < 1e-7 * (1 + float(b.abs().max())), (a, b)


def test_norm_gradient_formula():
    gen = torch.Generator().manual_seed(0)
    rnd = lambda *s: torch.randn(s, generator=gen, dtype=torch.float64)  # noqa: E731
    r, w, b, dy, dr = rnd(3, 16) + 2, rnd(16), rnd(16), rnd(3, 16), rnd(3, 16)
    loss = lambda: float((ref.layer_norm(r, w, b, 1e-2)[0] * dy).sum() + (r * dr).sum())  # noqa: E731
    dx, dw, db = ref.layer_norm_grad(dy, r, w, 1e-2, dr)
    for v, g in ((r, dx), (w, dw), (b, db)):
        _near(_differences(loss, v), g)


def test_routing_gradient_formulas():
    gen = torch.Generator().manual_seed(1)
    rnd = lambda *s: torch.randn(s, generator=gen, dtype=torch.float64)  # noqa: E731
    t, k, e, h = 5, 3, 6, 4
    logits = rnd(t, e)
    idx, w = ref.route(logits, k)
    ids = torch.where(torch.rand((t, k), generator=gen) < 0.3, torch.full_like(idx, -1), idx)
    offsets, perm, inv = ref.order(ids, e)
    here = ref.in_use(ids, e)
    y, dout = rnd(t * k, h), rnd(t, h)
    dy, dw = ref.combine_grad(dout, y, w, inv, here)
    loss = lambda: float((ref.combine(y, w, inv, here) * dout).sum())  # noqa: E731
    _near(_differences(loss, y), dy)
    _near(_differences(loss, w), dw)
    full = lambda: float((ref.route(logits, k)[1] * dw).sum())  # noqa: E731
    _near(_differences(full, logits, 1e-6), ref.route_grad(dw, w, idx, e))
    # the rows' copies: x[perm / k], whose gradient is the sum over a token's slots
    x, dxp = rnd(t, h), rnd(t * k, h)
    n = int(offsets[-1])
    copies = lambda: float((x[(perm[:n] // k).long()] * dxp[:n]).sum())  # noqa: E731
    _near(_differences(copies, x), ref.combine(dxp, None, inv, here))


def test_gelu_fit():
    """The kernel's form of Phi(-t), operation by operation in fp32 (exp2 and reciprocal rounded where the
    hardware's are an ulp off): within the header's bound of the 64-bit function."""
    f = np.float32
    t = np.concatenate([np.linspace(0, 1, 20001), np.linspace(1, 13, 120001)]).astype(f)
    s = (f(1) / (f(0.31) * t + f(1)).astype(f)).astype(f)
    p = np.full_like(t, f(0.035773511))
    for c in (-0.14138612, 0.15481046, -0.014781747, 0.11010987, 0.10775089, 0.12406693, 0.12365626):
        p = (p.astype(np.float64) * s + np.float64(f(c))).astype(f)
    e = np.exp2((t * t * f(-0.72134752)).astype(np.float64)).astype(f)
    q = (p * (e * s)).astype(f)
    want = ref.phi(torch.from_numpy(-t.astype(np.float64))).numpy()
    assert (np.abs(q - want) <= (16 + t.astype(np.float64) ** 2) * 2.0 ** -23 * want).all()
    near = t < 4
    assert (np.abs(q - want)[near] / want[near]).max() < 4e-6


def test_activation_bounds_hold_a_wrong_constant(monkeypatch):
    """The bounds of the GPU tests would see the tanh form in place of the erf form, and 0.044 in place of
    0.044715 (the mistakes planted here)."""
    z = torch.arange(-256, 257, dtype=torch.float64) / 64
    v, b = ref.activate(z, "gelu")
    u, _ = ref.activate(z, "gelu_tanh")
    assert float(((v - u).abs() > b).double().mean()) > 0.9
    e = (8 / np.pi) ** 0.5 * (z + 0.044 * z ** 3)
    assert float(((z / (1 + torch.exp(-e)) - u).abs() > ref.activate(z, "gelu_tanh")[1]).double().mean()) > 0.9


@pytest.mark.parametrize("name", ["layer_norm", "route_topk", "moe_permute", "moe_combine"])
def test_tensors_on_the_cpu_are_refused(name):
    hkmoe = pytest.importorskip("hkmoe")
    x, ids, w = torch.zeros((4, 64)), torch.zeros((4, 2), dtype=torch.int32), torch.ones((4, 2))
    order = hkmoe.MoEOrder(torch.zeros(9, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), ids)
    args = dict(layer_norm=(x, torch.ones(64)), route_topk=(x, 2), moe_permute=(x, ids, 8), moe_combine=(torch.zeros((8, 64)), w, order))
    with pytest.raises(RuntimeError, match="GPU"):
        getattr(hkmoe, name)(*args[name])


def _plain(lib, a=P, b=P):
    return lib.hkmoe_gemm_fp8(a, b, P, i64(4), i64(256), i64(128), None, None, 0, None)


def _plain_mx(lib, a=P, b=P, sa=P, sb=P):
    return lib.hkmoe_gemm_mx(a, sa, b, sb, P, i64(4), i64(256), i64(128), 0, None)


@pytest.mark.parametrize("call,name", [(c, n) for c in (_plain, _plain_mx, _fp8, _mx) for n in ("a", "b")] +
                         [(c, n) for c in (_plain_mx, _mx) for n in ("sa", "sb")])
def test_operands_of_odd_addresses_are_refused(lib, call, name):
    """The operands, and the MX words, are fetched 16 bytes a lane."""
    _refused(lib, call, {name: ODD}, "aligned")


def test_tails_of_silu_and_gelu_tanh():
    """The kernel's form of z / (1 + 2^x), operation by operation in fp32 (exp2 and reciprocal rounded where the
    hardware's are an ulp off, 0 below the normal numbers): within the header's bounds down to 2^-119, and no
    further off than that below."""
    f = np.float32
    z = np.arange(-105, 40, 1 / 64, dtype=f)
    t = np.arange(-11, 11, 1 / 512, dtype=f)
    slope = ((t * t).astype(np.float64) * f(-0.10294324) + np.float64(f(-2.3022082))).astype(f)  # one FMA
    for v, x, name in ((z, z * f(-1.44269504), "silu"), (t, t * slope, "gelu_tanh")):
        with np.errstate(over="ignore", under="ignore"):
            r = 1 / (f(1) + np.exp2(x.astype(np.float64)).astype(f)).astype(np.float64)
            got = v * np.where(r < 2.0 ** -126, 0, r).astype(f)
        v = torch.from_numpy(v.astype(np.float64))
        e = v if name == "silu" else (8 / np.pi) ** 0.5 * (v + 0.044715 * v ** 3)
        want = v / (1 + torch.exp(-e))
        bound = (4 + (1.0 if name == "silu" else 2.5) * e.abs()) * 2.0 ** -23 * want.abs()
        off = (torch.from_numpy(got.astype(np.float64)) - want).abs()
        far = want.abs() >= 2.0 ** -119
        assert bool((off <= bound)[far].all()) and bool((off[~far] <= 2.0 ** -119).all()), name
        assert not bool(far.all()) and float(want[far & (v < -1)].abs().min()) < 2.0 ** -118  # the grid passes the limit
