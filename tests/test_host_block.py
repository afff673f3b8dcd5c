"""Norm, router and adapters: what the host refuses, and what it launches (no GPU)."""
import ctypes
import os

import pytest

import hip_host

P = ctypes.c_void_p(0x1000)  # never dereferenced: validation fails first
ODD = ctypes.c_void_p(0x1008)
i64, i32, dbl, size = ctypes.c_int64, ctypes.c_int32, ctypes.c_double, ctypes.c_size_t


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(os.environ.get("HKMOE_LIB") or hip_host.LIB)
    lib.hkmoe_last_error.restype = ctypes.c_char_p
    lib.hkmoe_lora_workspace_size.restype = size
    lib.hkmoe_rms_norm_quant_workspace_size.restype = size
    return lib


def _norm(lib, x=P, residual=None, weight=P, rows=4, cols=256, xt=0, wt=0, eps=1e-6, mode=1, scale=None, q=P, s=P,
          residual_out=None, norm=None, ws=None, ws_bytes=0):
    return lib.hkmoe_rms_norm_quant(x, residual, weight, i64(rows), i64(cols), xt, wt, dbl(eps), mode, scale, q, s,
                                    residual_out, norm, ws, size(ws_bytes), None)


@pytest.mark.parametrize("bad,says", [
    (dict(x=None), "null"), (dict(weight=None), "null"), (dict(q=None), "null"), (dict(s=None), "null"),
    (dict(rows=-1), "shape"), (dict(cols=0), "shape"), (dict(rows=1 << 27), "shape"), (dict(cols=200), "multiple of 128"),
    (dict(cols=40, mode=2), "multiple of 32"), (dict(cols=4, mode=0), "multiple of 8"), (dict(cols=65664), "65536"),
    (dict(xt=2), "dtype"), (dict(wt=5), "dtype"), (dict(eps=0.0), "eps"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(mode=3), "scale_mode"),
    (dict(scale=P), "given scale"), (dict(residual=P), "together"), (dict(residual_out=P), "together"),
    (dict(x=ODD), "aligned"), (dict(q=ODD), "aligned"), (dict(norm=ODD), "aligned"), (dict(weight=ODD), "aligned")])
def test_norm_refusals(lib, bad, says):
    assert _norm(lib, **bad) == 1
    assert says in lib.hkmoe_last_error().decode()


def test_norm_workspace(lib):
    need = lib.hkmoe_rms_norm_quant_workspace_size(i64(4), 0, 0)
    assert need >= 4 * 4 and lib.hkmoe_rms_norm_quant_workspace_size(i64(4), 0, 1) == 0
    assert lib.hkmoe_rms_norm_quant_workspace_size(i64(4), 1, 0) == 0
    assert _norm(lib, mode=0) == 4 and _norm(lib, mode=0, ws=P, ws_bytes=need - 1) == 4
    assert _norm(lib, mode=0, ws=ODD, ws_bytes=need) == 4


def test_norm_no_rows_takes_null_buffers(lib):
    assert _norm(lib, rows=0, x=None, q=None, s=None) == 0
    assert _norm(lib, rows=0, x=None, q=None, s=None, mode=0, scale=P) == 0
    assert _norm(lib, rows=0, x=None, q=None, s=None, mode=0) == 1  # its scale is still an output


@pytest.mark.parametrize("bad,says", [
    (dict(x=None), "null"), (dict(w=None), "null"), (dict(logits=None), "null"), (dict(t=-1), "shape"),
    (dict(e=0), "shape"), (dict(e=1025), "shape"), (dict(h=0), "multiple of 8"), (dict(h=12), "multiple of 8"),
    (dict(h=(1 << 20) + 8), "2^20"), (dict(x=ODD), "aligned"), (dict(w=ODD), "aligned"), (dict(t=1 << 27), "shape")])
def test_router_refusals(lib, bad, says):
    a = dict(x=P, w=P, t=4, e=8, h=64, logits=P)
    a.update(bad)
    assert lib.hkmoe_router_logits(a["x"], a["w"], i64(a["t"]), i32(a["e"]), i64(a["h"]), a["logits"], None) == 1
    assert says in lib.hkmoe_last_error().decode()


def _lora(lib, y=P, ys=64, x=P, xs=256, a=P, b=P, ids=P, scaling=None, rows=4, adapters=2, h=256, n=64, r=8, yt=0, out=P,
          os_=64, ws=P, ws_bytes=1 << 40):
    return lib.hkmoe_lora_add(y, i64(ys), x, i64(xs), a, b, ids, scaling, i64(rows), i32(adapters), i64(h), i64(n), i32(r), yt,
                              out, i64(os_), ws, size(ws_bytes), None)


@pytest.mark.parametrize("bad,says", [
    (dict(y=None), "null"), (dict(x=None), "null"), (dict(a=None), "null"), (dict(b=None), "null"), (dict(ids=None), "null"),
    (dict(out=None), "null"), (dict(rows=-1), "shape"), (dict(rows=1 << 27), "shape"), (dict(adapters=0), "shape"),
    (dict(h=12), "multiples of 8"), (dict(n=60), "multiples of 8"), (dict(n=0), "multiples of 8"), (dict(n=(1 << 23) + 8, ys=1 << 24, os_=1 << 24), "2^23"), (dict(xs=(1 << 25) + 8), "2^25"), (dict(r=12), "rank"),
    (dict(r=0), "rank"), (dict(r=264), "rank"), (dict(yt=2), "y_dtype"), (dict(xs=248), "strides"), (dict(xs=260), "strides"),
    (dict(ys=56), "strides"), (dict(ys=68), "strides"), (dict(os_=60), "strides"), (dict(yt=1, ys=66), "strides"),
    (dict(os_=72), "row stride"), (dict(y=ODD), "aligned"), (dict(x=ODD), "aligned"), (dict(out=ODD), "aligned"),
    (dict(a=ODD), "aligned"), (dict(b=ODD), "aligned"), (dict(ids=ctypes.c_void_p(0x1002)), "aligned")])
def test_lora_refusals(lib, bad, says):
    assert _lora(lib, **bad) == 1
    assert says in lib.hkmoe_last_error().decode()


def test_lora_workspace(lib):
    need = lib.hkmoe_lora_workspace_size(i64(4), i64(256), i32(8))
    assert need >= 4 * 8 * 4 and lib.hkmoe_lora_workspace_size(i64(0), i64(256), i32(8)) == 0
    assert _lora(lib, ws=None) == 4 and _lora(lib, ws_bytes=need - 1) == 4 and _lora(lib, ws=ODD) == 4
    assert _lora(lib, rows=0, y=None, x=None, ids=None, out=None, ws=None, ws_bytes=0) == 0


def test_python_refuses_cpu_tensors():
    import torch
    hkmoe = pytest.importorskip("hkmoe")
    x = torch.zeros((4, 256), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        hkmoe.rms_norm_quant(x, x[0])
    with pytest.raises(RuntimeError):
        hkmoe.router_logits(x, x)
    with pytest.raises(RuntimeError):
        hkmoe.lora_add(x, x, x[None], x[None], torch.zeros(4, dtype=torch.int32))


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    return hip_host.build_fake(str(tmp_path_factory.mktemp("hip")))


def test_grids_stay_in_range(fake):
    """The largest sizes that are taken launch with every dimension below 2^32 work-items."""
    out = hip_host.run(fake, """
        size, dbl = ctypes.c_size_t, ctypes.c_double
        big, st = 1 << 24, vp(5)
        lib.hkmoe_lora_workspace_size.restype = size
        for rows in (1, 64, 5000, big):
            for cols in (8, 128, 65536):
                for mode in (0, 1, 2):
                    if mode and cols == 8: continue
                    assert lib.hkmoe_rms_norm_quant(P, None, P, i64(rows), i64(cols), 0, 0, dbl(1e-6), mode, None, P, P, None,
                                                    None, P, size(1 << 50), st) == 0
            for e in (1, 256, 1024):
                assert lib.hkmoe_router_logits(P, P, i64(rows), i32(e), i64(4096), P, st) == 0
            for n in (8, 4096, 1 << 23):
                for yt in (0, 1):
                    assert lib.hkmoe_lora_add(P, i64(n), P, i64(256), P, P, P, None, i64(rows), i32(1000), i64(256), i64(n),
                                              i32(16), yt, P, i64(n), P, size(1 << 50), st) == 0
        for line in log(): print(line)
    """)
    launches = [l for l in out if l.startswith("launch")]
    assert launches and all(l.endswith("stream=5") for l in launches)
    for l in launches:
        grid = int(l.split("grid=")[1].split()[0])
        assert 1 <= grid and grid * (1024 if "norm" in l else 512) < 1 << 32, l


STAND_IN = hip_host.BINDING + """
torch.cuda.current_device = lambda: 0
class T(Tensor):
    def __init__(self, shape, dtype="torch.bfloat16", dev=0, strides=None):
        Tensor.__init__(self, shape, dtype)
        flat, n = [], 1
        for s in reversed(self.shape):
            flat.insert(0, n)
            n *= s
        self.dev, self.flat, self.strides = dev, tuple(flat), strides or tuple(flat)
    def is_contiguous(self): return self.strides == self.flat
    def stride(self): return self.strides
    def get_device(self): return self.dev
f32, u8, i32 = "torch.float32", "torch.uint8", "torch.int32"
def lora(y=T([4, 64]), x=T([4, 256]), a=T([2, 8, 256]), b=T([2, 64, 8]), ids=T([4], i32), scaling=None, out=T([4, 64]),
         ws=T([1 << 20], u8)):
    tk_kernel.dispatch_lora_add(y, x, a, b, ids, scaling, out, ws)
def refused(fn):
    try:
        fn()
    except RuntimeError as e:
        print("refused:", e)
    else:
        print("taken")
"""


def test_tensors_through_their_attributes(fake):
    """A torch without the exchange interface: the same checks, on the attributes."""
    out = hip_host.run(fake, STAND_IN + """
lora()
lora(y=T([4, 64], strides=(192, 1)), out=T([4, 64], strides=(192, 1)), x=T([4, 256], strides=(512, 1)))
tk_kernel.dispatch_router_logits(T([4, 64]), T([8, 64]), T([4, 8], f32))
tk_kernel.dispatch_rms_norm_quant(T([4, 256]), None, T([256]), 1e-6, 1, T([4, 256], "torch.float8_e4m3fn"), T([4, 2], f32))
for line in log(): print(line)
refused(lambda: lora(x=T([4, 256], dev=1)))
refused(lambda: lora(x=T([4, 256], dev=-1)))
refused(lambda: lora(y=T([4, 64], strides=(1, 4))))
refused(lambda: lora(a=T([2, 8, 256], strides=(1, 2, 16))))
refused(lambda: lora(ids=T([4], f32)))
refused(lambda: lora(y=[1, 2]))
refused(lambda: tk_kernel.dispatch_router_logits(T([4, 64], strides=(128, 1)), T([8, 64]), T([4, 8], f32)))
""")
    launches = [l for l in out if l.startswith("launch")]
    assert len(launches) == 6 and all(l.endswith("stream=7") for l in launches), out
    said = [l for l in out if l.startswith("refused")]
    wanted = ["x: tensor must be on the current device", "x: tensor must be on a GPU device", "y: rows must be contiguous",
              "a: tensor must be contiguous", "ids: expected dtype torch.int32", "y: expected a torch.Tensor",
              "x: tensor must be contiguous"]
    assert [s.split(": ", 1)[1] for s in said] == wanted and "taken" not in out


# ---------------------------------------------------------------------------
# workspaces of the layers and of the block in front of them: CPU tensors, and
# dispatches that only note what they were given
# ---------------------------------------------------------------------------
def _bare_layer(hkmoe, torch, mx):
    f8, e, h, i = torch.float8_e4m3fn, 8, 256, 256
    layer = object.__new__(hkmoe.MoELayerMX if mx else hkmoe.MoELayer)
    layer.packed, layer.top_k, layer.num_experts, layer.hidden, layer.inter = True, 2, e, h, i
    layer.block, layer._ws = True, None
    layer.w13_q, layer.w2_q = torch.empty((e, 2 * i, h), dtype=f8), torch.empty((e, h, i), dtype=f8)
    layer.w13_scale = layer.w2_scale = layer.w13_words = layer.w2_words = torch.empty(0)
    return layer


@pytest.mark.parametrize("mx", [False, True])
def test_block_calls_share_no_workspace(monkeypatch, mx):
    """Two calls of one block may overlap in time, on two streams or in two graphs: each has a
    workspace of its own, large enough, and neither is the layer's."""
    import torch
    hkmoe = pytest.importorskip("hkmoe")
    tk, given = hkmoe.tk_kernel, []
    monkeypatch.setattr("hkmoe.layer._check_dev", lambda *ts: None)
    monkeypatch.setattr(tk, "dispatch_rms_norm_quant", lambda *a, **k: None)
    monkeypatch.setattr(tk, "dispatch_router_logits", lambda *a, **k: None)
    monkeypatch.setattr(tk, "dispatch_moe_mx" if mx else "dispatch_moe", lambda *a, **k: given.append(a[9]))
    layer = _bare_layer(hkmoe, torch, mx)
    block = hkmoe.MoEBlock(torch.ones(256), torch.zeros((8, 256), dtype=torch.bfloat16), layer)
    x = torch.zeros((5, 256), dtype=torch.bfloat16)
    for _ in range(2):
        out, r = block(x)
        assert out.shape == (5, 256) and r is x
    need = tk.moe_workspace_size(5, 8, 2, 256, 256, tk.SCALE_MX if mx else tk.SCALE_BLOCK)
    assert len(given) == 2 and all(w.dtype == torch.uint8 and w.numel() >= need for w in given)
    assert given[0].data_ptr() != given[1].data_ptr() and all(w is not layer._ws for w in given)


@pytest.mark.parametrize("mx", [False, True])
def test_layer_keeps_the_workspace_of_a_captured_graph(monkeypatch, mx):
    """A layer's workspace that a capture has used outlives a larger one: the graph writes to it
    whenever it is replayed.  One that only eager calls used does not."""
    import weakref

    import torch
    hkmoe = pytest.importorskip("hkmoe")
    layer, capturing = _bare_layer(hkmoe, torch, mx), []
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: bool(capturing))
    eager = weakref.ref(layer.workspace(4, "cpu"))
    layer.workspace(40, "cpu")
    assert eager() is None
    capturing.append(1)
    held = weakref.ref(layer.workspace(4, "cpu"))  # a graph over fewer tokens: the same workspace
    assert held() is layer._ws
    capturing.clear()
    layer.workspace(400, "cpu")
    assert held() is not None and held() is not layer._ws
    later = weakref.ref(layer._ws)
    layer.workspace(4000, "cpu")
    assert later() is None and held() is not None


def test_adapters_of_many_columns_take_the_matrix_instruction(fake):
    """The shapes on which a row's own workgroup was measured slower in each order of the rows."""
    out = hip_host.run(fake, """
        lib.hkmoe_lora_workspace_size.restype = ctypes.c_size_t
        for rows, h, r, n in ((2048, 4096, 16, 4096), (512, 4096, 32, 4096), (2048, 2048, 16, 8192), (1024, 4096, 24, 4096),
                              (1024, 4096, 16, 4096), (256, 4096, 32, 4096), (2048, 4096, 16, 1024), (200, 4096, 40, 4096)):
            assert lib.hkmoe_lora_add(P, i64(n), P, i64(h), P, P, P, None, i64(rows), i32(64), i64(h), i64(n), i32(r), 0, P, i64(n),
                                      P, ctypes.c_size_t(1 << 40), None) == 0
        for line in log(): print(line)
    """)
    second = [l for l in out if l.startswith("launch") and "lora_expand" in l]
    assert len(second) == 8 and ["small" in l for l in second] == [False] * 4 + [True] * 4, second


@pytest.mark.parametrize("bf16", [True, False])
def test_exact_adapter_inputs_need_every_term(bf16):
    """The inputs of the adapters' equality test: every sum exact in fp32, and one bf16 term of v less
    (the mistake planted here) moves most outputs."""
    import numpy as np

    import block_ref
    rng = np.random.default_rng(0)
    x, a, b, c, v = block_ref.lora_exact_inputs(rng, 50, 264, 136, 40, 3, bf16)
    for part in (x, a, b):
        assert (block_ref.fp8.bf16_round(part) == part).all()
    assert np.abs(v).max() < 1 << 24  # so is every partial sum: x's terms of a row have one sign, A's of a rank too
    terms = 2 if bf16 else 3
    ids = np.arange(50) % 3
    mine = v[ids, np.arange(50)]
    assert (block_ref.split_terms(mine, terms) == mine).all()
    ref, _ = block_ref.lora(np.zeros((50, 136), np.float32), x, a, b, ids, c)
    if bf16:
        assert (block_ref.fp8.bf16_round(ref.astype(np.float32)) == ref).all()
    else:
        assert (ref.astype(np.float32) == ref).all()
    for k in range(1, terms + 1):
        lost = c[ids][:, None] * np.einsum("tr,tnr->tn", block_ref.split_terms(mine, k), b.astype(np.float64)[ids])
        assert (lost == ref).all() if k == terms else (lost != ref).mean() > 0.8


def test_every_grid_dimension_in_range(fake):
    """The largest sizes that are taken: x below 2^32 work-items, y and z at most 65535."""
    out = hip_host.run(fake, """
        size, dbl = ctypes.c_size_t, ctypes.c_double
        for rows in (1, 63, 64, 65, 2048, 4096, 65536, 65537, 1 << 24):
            for cols in (8, 65536):
                for mode in (0, 1, 2):
                    if mode and cols == 8: continue
                    assert lib.hkmoe_rms_norm_quant(P, None, P, i64(rows), i64(cols), 0, 0, dbl(1e-6), mode, None, P, P, None,
                                                    None, P, size(1 << 50), None) == 0
            for e in (1, 1024):
                for h in (8, 1 << 20):
                    assert lib.hkmoe_router_logits(P, P, i64(rows), i32(e), i64(h), P, None) == 0
            for n in (8, 1 << 23):
                for h, r, adapters in ((8, 8, 1), (1 << 20, 8, 1535), (4096, 16, 1 << 20), (4096, 40, 64), (1 << 20, 256, 64)):
                    for yt in (0, 1):
                        assert lib.hkmoe_lora_add(P, i64(n), P, i64(h), P, P, P, None, i64(rows), i32(adapters), i64(h), i64(n),
                                                  i32(r), yt, P, i64(n), P, size(1 << 50), None) == 0
        for line in log(): print(line)
    """)
    launches = [l for l in out if l.startswith("launch")]
    assert len({l.split()[1] for l in launches}) > 15
    for l in launches:
        v = {k: int(n) for k, n in (f.split("=") for f in l.split()[2:])}
        assert 1 <= v["grid"] and v["grid"] * v["threads"] < 1 << 32 and 1 <= v["y"] <= 65535 and 1 <= v["z"] <= 65535, l
        assert v["threads"] <= 1024, l


def test_lora_workspace_of_refused_sizes(lib):
    """Sizes that lora_add refuses have no workspace: no sum of theirs leaves 64 bits."""
    top = 2 ** 63 - 1
    for rows, hidden, rank in ((top, 256, 8), (4, top, 8), (top, top, 2 ** 31 - 1), (4, 256, 2 ** 31 - 1), ((1 << 24) + 1, 256, 8),
                               (4, (1 << 20) + 8, 8), (4, 256, 264)):
        assert lib.hkmoe_lora_workspace_size(i64(rows), i64(hidden), i32(rank)) == 0, (rows, hidden, rank)
    assert lib.hkmoe_lora_workspace_size(i64(1 << 24), i64(1 << 20), i32(256)) >= (1 << 24) * 256 * 4
