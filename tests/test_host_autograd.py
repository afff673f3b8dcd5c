"""What the Python layer tells autograd, on the CPU: the kernels are stand-ins that compute the
formulas with torch and, like them, write through a pointer that autograd does not see."""

import pytest
import torch

import train_ref as ref

hkmoe = pytest.importorskip("hkmoe")
BF16, F32, F8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def _put(to, value):
    to.data.copy_(value)  # .data: the version stays


def _layer_norm(x, residual, w, b, eps, y, residual_out, stats):
    x = x.detach()
    r = x if residual is None else x + residual.detach()
    out, m, rstd = ref.layer_norm(r.double(), w.detach().double(), None if b is None else b.detach().double(), eps)
    if residual is not None:
        _put(residual_out, r)
    _put(y, out)
    _put(stats, torch.cat([m, torch.zeros_like(m), rstd, torch.zeros_like(m)], 1))


def _layer_norm_backward(dy, r, w, dr, stats, dx, dw, db, ws):
    got = ref.layer_norm_grad(dy.double(), r.double(), w.double(), 1e-5, None if dr is None else dr.double())
    for to, v in zip((dx, dw, db), got):
        if to is not None:
            _put(to, v)


def _gemm(a, b, c, sa, sb, bias=None, act=0, residual=None):
    z = a.float() @ b.float().T
    z = z if bias is None else z + bias.detach()
    _put(c, z if residual is None else z + residual.detach())


def _fill(*places):
    """A kernel that writes to these of its arguments."""
    return lambda *args, **kw: [_put(args[i], torch.ones(args[i].shape)) for i in places if args[i] is not None]


@pytest.fixture
def hk(monkeypatch):
    tk = hkmoe.tk_kernel
    monkeypatch.setattr(hkmoe.layer, "_check_dev", lambda *ts: None)
    for name, kernel in dict(
            layer_norm=_layer_norm, layer_norm_backward=_layer_norm_backward, gemm_fp8=_gemm, gemm_fp8_epilogue=_gemm,
            gemm_mx=lambda a, sa, b, sb, c: _gemm(a, b, c, None, None),
            gemm_mx_epilogue=lambda a, sa, b, sb, c, bias, act, res: _gemm(a, b, c, None, None, bias, act, res),
            rms_norm_quant=_fill(5, 8), router_logits=_fill(2), lora_add=_fill(6), moe=_fill(8), moe_mx=_fill(8)).items():
        monkeypatch.setattr(tk, "dispatch_" + name, kernel)
    return hkmoe


def _f8(*shape):
    return torch.ones(shape).to(F8)


def _mx_layer():
    layer = object.__new__(hkmoe.MoELayerMX)
    layer.__dict__.update(w13_q=None, w13_words=None, w2_q=None, w2_words=None, top_k=2, hidden=256, packed=True)
    return layer


# every call that writes into a tensor of the caller's: (shape and dtype of it, the call)
TARGETS = {
    "gemm_fp8": ((4, 256), BF16, lambda hk, o: hk.gemm_fp8(_f8(4, 128), _f8(256, 128), out=o)),
    "gemm_fp8 epilogue": ((4, 256), BF16, lambda hk, o: hk.gemm_fp8(_f8(4, 128), _f8(256, 128), activation="none", out=o)),
    "gemm_mx": ((4, 256), F32, lambda hk, o: hk.gemm_mx(_f8(4, 128), None, _f8(256, 128), None, out=o)),
    "gemm_mx epilogue": ((4, 256), F32, lambda hk, o: hk.gemm_mx(_f8(4, 128), None, _f8(256, 128), None, residual=o, out=o)),
    "layer_norm_forward": ((4, 64), F32, lambda hk, o: hk.layer_norm_forward(torch.ones(4, 64), torch.ones(64), residual=o, residual_out=o)),
    "rms_norm_quant": ((4, 128), F32, lambda hk, o: hk.rms_norm_quant(torch.ones(4, 128), torch.ones(128), residual=o, residual_out=o)),
    "router_logits": ((4, 8), F32, lambda hk, o: hk.router_logits(torch.ones(4, 64), torch.ones(8, 64), out=o)),
    "lora_add": ((4, 64), F32, lambda hk, o: hk.lora_add(o, torch.ones(4, 64), torch.ones(1, 8, 64), torch.ones(1, 64, 8),
                                                         torch.zeros(4, dtype=torch.int32), out=o)),
    "moe_forward": ((4, 256), BF16, lambda hk, o: hk.moe_forward(_f8(4, 256), torch.ones(1), torch.ones(4, 8), _f8(8, 512, 256), None,
                                                                 _f8(8, 256, 256), None, 2, out=o)),
    "MoELayerMX": ((4, 256), BF16, lambda hk, o: _mx_layer()(_f8(4, 256), None, torch.ones(4, 8), out=o, workspace=torch.empty(8))),
}


@pytest.mark.parametrize("name", TARGETS)
def test_given_outputs_count_as_written(hk, name):
    """Their version rises, that of a tensor they are a view of with it, also without gradients being recorded."""
    shape, dtype, call = TARGETS[name]
    buf = torch.zeros((2, *shape), dtype=dtype)
    for ctx in (torch.enable_grad(), torch.no_grad()):
        with ctx:
            before = buf._version
            call(hk, buf[1])
            assert buf._version > before


@pytest.mark.parametrize("name", TARGETS)
def test_given_outputs_made_for_inference(hk, name):
    """Tensors of torch.inference_mode() have no version: the calls take them."""
    shape, dtype, call = TARGETS[name]
    with torch.inference_mode():
        call(hk, torch.zeros(shape, dtype=dtype))


def test_refused_calls_leave_the_version(hk, monkeypatch):
    def refuse(*args):
        raise RuntimeError("refused")
    monkeypatch.setattr(hk.tk_kernel, "dispatch_gemm_fp8", refuse)
    out = torch.zeros((4, 256), dtype=BF16)
    with pytest.raises(RuntimeError, match="refused"):
        hk.gemm_fp8(_f8(4, 128), _f8(256, 128), out=out)
    assert out._version == 0


def _overwrites(hk, r):
    return {
        "gemm_fp8": lambda: hk.gemm_fp8(_f8(4, 128), _f8(256, 128), residual=r, out=r),
        "layer_norm_forward": lambda: hk.layer_norm_forward(torch.ones(4, 256), torch.ones(256), residual=r, residual_out=r),
    }


@pytest.mark.parametrize("name", ["gemm_fp8", "layer_norm_forward"])
def test_an_overwritten_stream_has_no_gradient(hk, name):
    """The norm's gradient reads the stream: once a later call has overwritten it in place, the backward
    pass raises, as torch's own in-place calls make it, and does not use the new values."""
    x, w, s = torch.randn(4, 256), torch.ones(256, requires_grad=True), torch.randn(4, 256)
    y, r = hk.layer_norm(x, w, residual=s)
    with torch.no_grad():
        _overwrites(hk, r)[name]()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_a_stream_that_is_left_alone_has_one(hk):
    x, w, s = torch.randn(4, 256), torch.ones(256, requires_grad=True), torch.randn(4, 256)
    y, r = hk.layer_norm(x, w, residual=s)
    kept = r.detach().clone()
    with torch.no_grad():
        _overwrites(hk, kept)["gemm_fp8"]()
    y.backward(torch.ones_like(y))
    assert torch.allclose(w.grad, ref.layer_norm_grad(torch.ones(4, 256).double(), r.detach().double(), w.detach().double(), 1e-5, None)[1].float())


PRODUCTS = {"gemm_fp8": lambda hk, **e: hk.gemm_fp8(_f8(4, 128), _f8(256, 128), **e),
            "gemm_mx": lambda hk, **e: hk.gemm_mx(_f8(4, 128), None, _f8(256, 128), None, **{"out_dtype": BF16, **e})}


@pytest.mark.parametrize("call", PRODUCTS.values(), ids=PRODUCTS)
@pytest.mark.parametrize("name", ["bias", "residual", "out"])
def test_products_refuse_tensors_that_ask_for_a_gradient(hk, call, name):
    """The products record none: without an error, C would carry no gradient of the bias or the residual, and
    the old history of a given tensor.  Detached, or without gradients being recorded, they are taken."""
    t = torch.zeros(256 if name == "bias" else (4, 256), dtype=BF16, requires_grad=True)
    for given in (t, t * 1):
        with pytest.raises(RuntimeError, match=f"{name} asks for a gradient"):
            call(hk, **{name: given})
        assert not call(hk, **{name: given.detach()}).requires_grad
        with torch.no_grad():
            call(hk, **{name: given})
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(t.detach(), torch.ones_like(t))
        with torch.no_grad(), pytest.raises(RuntimeError, match=f"{name} asks for a gradient"):
            call(hk, **{name: dual})
        call(hk, **{name: t.detach()})


def test_the_stream_in_place_refuses_a_gradient(hk):
    """layer_norm_forward records none; a new stream written into a tensor that has a history would keep it."""
    r = torch.zeros((4, 64), requires_grad=True) * 1
    with pytest.raises(RuntimeError, match="residual_out asks for a gradient"):
        hk.layer_norm_forward(torch.ones(4, 64), torch.ones(64), residual=r, residual_out=r)
    with torch.no_grad():
        hk.layer_norm_forward(torch.ones(4, 64), torch.ones(64), residual=r, residual_out=r)


def _recorded(hk):
    """The recorded calls: name -> (the tensors that may ask for a gradient, the call on them)."""
    order = hk.MoEOrder(torch.tensor([0, 4, 8], dtype=torch.int32), torch.arange(8, dtype=torch.int32),
                        torch.arange(8, dtype=torch.int32).view(4, 2))
    rows, w = torch.randn(8, 64), torch.rand(4, 2)
    return {
        "layer_norm": ([torch.randn(4, 64), torch.ones(64), torch.zeros(64), torch.randn(4, 64)],
                       lambda x, w, b, s: hk.layer_norm(x, w, b, s)),
        "layer_norm alone": ([torch.randn(4, 64), torch.ones(64)], lambda x, w: hk.layer_norm(x, w)),
        "route_topk": ([torch.randn(4, 8)], lambda x: hk.route_topk(x, 2)),
        "moe_permute": ([torch.randn(4, 64)], lambda x: hk.moe_permute(x, torch.zeros((4, 2), dtype=torch.int32), 2)),
        "moe_combine": ([rows, w], lambda y, w: hk.moe_combine(y, w, order)),
    }


@pytest.mark.parametrize("name", ["layer_norm", "layer_norm alone", "route_topk", "moe_permute", "moe_combine"])
def test_forward_mode_is_refused(hk, monkeypatch, name):
    """Only backward gradients are recorded: a dual tensor's tangent is never dropped without an error, whether or
    not gradients are on, and calls without one run inside a dual level."""
    for kernel, places in dict(route_topk=(1, 2), permute=(2, 3, 4, 5), combine_rows=(4,)).items():
        monkeypatch.setattr(hk.tk_kernel, "dispatch_" + kernel, _fill(*places))
    tensors, call = _recorded(hk)[name]
    with torch.autograd.forward_ad.dual_level():
        call(*tensors)
        for i, t in enumerate(tensors):
            dual = tensors[:i] + [torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))] + tensors[i + 1:]
            for ctx in (torch.enable_grad(), torch.no_grad()):
                with ctx, pytest.raises(RuntimeError, match="jvp"):
                    call(*dual)


def _needs_aligned(kernel, *places):
    """A kernel that refuses what the library refuses: these of its arguments at other than 16-byte addresses."""
    def run(*args):
        for i in places:
            if args[i] is not None and (args[i].data_ptr() % 16 or not args[i].is_contiguous()):
                raise RuntimeError("tensors must be contiguous and 16-byte aligned")
        kernel(*args)
    return run


def _odd_gradient(t):
    """A scalar whose gradient comes back to t as a slice at an odd address: t behind one value, flattened together."""
    flat = torch.cat([torch.zeros(1, dtype=t.dtype), t.reshape(-1)])
    return (flat * torch.arange(flat.numel()).to(t.dtype)).sum()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gradients_at_odd_addresses(hk, monkeypatch, dtype):
    """Where autograd lays out a gradient is not the caller's choice: one that is contiguous but not 16-byte
    aligned (a slice of a flattened concatenation) is taken."""
    tk = hk.tk_kernel
    monkeypatch.setattr(tk, "dispatch_layer_norm_backward", _needs_aligned(_layer_norm_backward, 0, 1, 3))
    monkeypatch.setattr(tk, "dispatch_permute", _fill(2, 3, 4, 5))
    monkeypatch.setattr(tk, "dispatch_combine_rows", _needs_aligned(_fill(4), 0))
    monkeypatch.setattr(tk, "dispatch_combine_rows_backward", _needs_aligned(_fill(5, 6), 0, 1))
    leaf = lambda *s: torch.randn(s).to(dtype).requires_grad_()  # noqa: E731
    x, s, w = leaf(4, 64), leaf(4, 64), torch.ones(64, dtype=dtype, requires_grad=True)
    y, r = hk.layer_norm(x, w, residual=s)
    (_odd_gradient(y) + _odd_gradient(r)).backward()
    dy = torch.arange(1, 257).to(dtype).view(4, 64).double()
    want = ref.layer_norm_grad(dy, r.detach().double(), w.detach().double(), 1e-5, dy)[0].to(dtype)
    assert torch.allclose(x.grad, want) and torch.equal(x.grad, s.grad) and x.grad.data_ptr() != s.grad.data_ptr()
    x = leaf(4, 64)
    xp, order = hk.moe_permute(x, torch.zeros((4, 2), dtype=torch.int32), 2)
    _odd_gradient(xp).backward()
    tw = torch.rand((4, 2), requires_grad=True)
    _odd_gradient(hk.moe_combine(leaf(8, 64), tw, order)).backward()
    assert x.grad is not None and tw.grad is not None
