"""Dense FP8 and MX products with bias, activation and residual against the formulas in 64
bits: operands of +-1 (MX: exponents around a common one) make every product exact in fp32, so
what is off is the epilogue's own rounding, which the bounds count.  The shapes reach every
kernel, with row remainders of every tile (test_host_train.py states which)."""
import math

import pytest
import torch

import train_ref as ref

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
SHAPES = [(1, 256, 128), (16, 256, 256), (17, 512, 1152), (31, 8192, 384), (33, 512, 384), (48, 256, 16384),
          (64, 2048, 4224), (65, 2048, 1024), (129, 256, 2048), (300, 1024, 1152), (257, 4096, 4096), (63, 768, 640),
          (1000, 4096, 256), (2001, 2048, 384), (1, 4352, 128), (16, 7168, 2048), (65, 32768, 1152), (4095, 4096, 384),
          (1000, 1024, 2176), (50, 16384, 256), (2000, 768, 128), (3000, 1024, 512), (2049, 1024, 640),
          (1777, 4096, 1152), (2047, 4096, 128), (1537, 8192, 256), (4097, 3840, 896)]


def _operands(m, n, k, mx, seed):
    """(call, z): call(hk, **epilogue) runs the product whose exact value is z (64 bits)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    pm1 = lambda *s: (torch.randint(0, 2, s, generator=gen, device="cuda") * 2 - 1).float()  # noqa: E731
    a, b = pm1(m, k), pm1(n, k)
    aq, bq = a.to(torch.float8_e4m3fn), b.to(torch.float8_e4m3fn)
    a, b = a.double(), b.double()
    down = round(math.log2(4.0 / math.sqrt(k)))  # z has a spread of about 4
    if mx:
        lo = 127 + down // 2
        ea = torch.randint(lo - 1, lo + 2, (m, k // 32), generator=gen, device="cuda", dtype=torch.uint8)
        eb = torch.randint(lo - 1, lo + 2, (n, k // 32), generator=gen, device="cuda", dtype=torch.uint8)
        z = (a.view(m, -1, 32) * torch.exp2(ea.double() - 127)[..., None]).view(m, k) @ \
            (b.view(n, -1, 32) * torch.exp2(eb.double() - 127)[..., None]).view(n, k).T
        return lambda hk, **e: hk.gemm_mx(aq, hk.mx_pack_scales(ea), bq, hk.mx_pack_scales(eb), **e), z
    sa, sb = torch.full((1,), 4.0, device="cuda"), torch.full((1,), 2.0 ** (down - 2), device="cuda")
    return lambda hk, **e: hk.gemm_fp8(aq, bq, sa, sb, **e), (a @ b.T) * 2.0 ** down


def _check(got, want, bound):
    off = (got.double() - want).abs() - bound
    assert not bool((off > 0).any()) and not bool(torch.isnan(off).any()), float(off.max())


def _bias(n, dtype, seed):
    return torch.randn(n, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_shapes(hk, m, n, k, mx):
    """Every kernel, both outputs, everything on; rows behind the last one stay untouched."""
    call, z = _operands(m, n, k, mx, m * 7 + n + k)
    for i, dtype in enumerate((BF16, F32)):
        act = ref.ACTIVATIONS[(m + n // 256 + k // 128 + i) % 5]
        bias = _bias(n, (F32, BF16)[(m + i) % 2], m)
        buf = torch.full((m + 1, n), 7.0, dtype=dtype, device="cuda")
        res = torch.randn(m, n, device="cuda").to(dtype)
        kept = res.clone()
        got = call(hk, bias=bias, activation=act, residual=res, out=buf[:m])
        torch.cuda.synchronize()
        _check(got, *ref.epilogue(z, bias, act, res, dtype))
        assert bool((buf[m] == 7.0).all()) and torch.equal(res, kept)


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("m,n,k", [(5, 512, 256), (200, 4096, 4096), (2500, 4096, 512)])
@pytest.mark.parametrize("act", ref.ACTIVATIONS)
def test_parts(hk, m, n, k, mx, act):
    """Each part alone and left out, in strips, 128x128 and 256x256 tiles."""
    call, z = _operands(m, n, k, mx, n + k)
    for dtype in (BF16, F32):
        for bias, residual in ((None, False), (BF16, False), (None, True)):
            b = None if bias is None else _bias(n, bias, 1)
            res = (4 * torch.randn(m, n, device="cuda")).to(dtype) if residual else None
            got = call(hk, bias=b, activation=act, residual=res, out_dtype=dtype)
            assert got.dtype == dtype
            _check(got, *ref.epilogue(z, b, act, res, dtype))


@pytest.mark.parametrize("m,n,k", [(3, 512, 256), (200, 4096, 4096), (2500, 4096, 512)])
def test_residual_in_place(hk, m, n, k):
    call, z = _operands(m, n, k, False, 3)
    for dtype in (BF16, F32):
        stream = torch.randn(m, n, device="cuda").to(dtype)
        first = stream.clone()
        assert call(hk, activation="gelu", residual=stream, out=stream) is stream
        _check(stream, *ref.epilogue(z, None, "gelu", first, dtype))


@pytest.mark.parametrize("act", ref.ACTIVATIONS)
def test_whole_range(hk, act):
    """z over [-40, 40) in steps of 2^-5 and at large magnitudes, through the bias: the fp32 results
    keep their relative size in the tails."""
    n = 2560
    aq = torch.zeros((1, 128), device="cuda").to(torch.float8_e4m3fn)
    bq = torch.zeros((n, 128), device="cuda").to(torch.float8_e4m3fn)
    z = torch.arange(n, device="cuda", dtype=F32) / 32 - 40
    big = torch.cat([z, torch.tensor([1e4, -1e4, 1e30, -1e30, 0.0, -0.0] + [2.0 ** -i for i in range(250)], device="cuda")])
    for bias in (z, big[-256:]):
        b = bias.contiguous()
        got = hk.gemm_fp8(aq, bq[: b.numel()].contiguous(), bias=b, activation=act, out_dtype=F32)[0]
        want, bound = ref.activate(b.double(), act)
        _check(got, want, bound + ref.U * want.abs() + 2.0 ** -149)  # a step below the normal numbers


@pytest.mark.parametrize("act", ref.ACTIVATIONS)
def test_not_finite(hk, act):
    """Infinities and NaN reach only their own column; +inf stays, -inf ends at the activation's limit
    or NaN, a NaN stays NaN."""
    n = 256
    aq = torch.ones((2, 128), device="cuda").to(torch.float8_e4m3fn)
    bq = torch.zeros((n, 128), device="cuda").to(torch.float8_e4m3fn)
    bias = torch.zeros(n, device="cuda")
    bias[3], bias[5], bias[7] = math.inf, -math.inf, math.nan
    got = hk.gemm_fp8(aq, bq, bias=bias, activation=act, out_dtype=F32)
    assert bool((got[:, 3] == math.inf).all()) and bool(torch.isnan(got[:, 7]).all())
    if act == "none":
        assert bool((got[:, 5] == -math.inf).all())
    else:
        assert bool(((got[:, 5] == 0) | torch.isnan(got[:, 5])).all())
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[[3, 5, 7]] = False
    assert bool((got[:, rest] == 0).all())


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("m,n,k", [(16, 256, 256), (40, 512, 1152), (300, 1024, 640), (2500, 4096, 256)])
def test_fp32_keeps_small_products(hk, m, n, k, mx):
    """One product of 2^16 and one of 2^-7 to 2^8 at every distance in K: their sum needs at most 24 bits, so
    fp32 C is exact; the FP8 matrix instructions alone would drop the small one where the two are neighbours."""
    gen = torch.Generator(device="cuda").manual_seed(m)
    a, b = torch.zeros((m, k), device="cuda"), torch.zeros((n, k), device="cuda")
    t = torch.arange(m, device="cuda")
    at = torch.randint(0, k, (m,), generator=gen, device="cuda")
    near = torch.where(t % 2 == 0, at ^ (1 + t // 2 % 7), (at + 1 + t) % k)  # neighbours, and anywhere
    a[t, at], a[t, near] = 256.0, 2.0 ** (t % 8 - 3).float()
    # every column has 2^8 where one row's large value is and 2^-4 elsewhere
    b += 2.0 ** -4
    pick = at[torch.arange(n, device="cuda") % m]
    b[torch.arange(n, device="cuda"), pick] = 256.0
    aq, bq = a.to(torch.float8_e4m3fn), b.to(torch.float8_e4m3fn)
    want = aq.double() @ bq.double().T
    if mx:
        ea = torch.full((m, k // 32), 120, dtype=torch.uint8, device="cuda")
        eb = torch.full((n, k // 32), 137, dtype=torch.uint8, device="cuda")
        got = hk.gemm_mx(aq, hk.mx_pack_scales(ea), bq, hk.mx_pack_scales(eb), activation="none", out_dtype=F32)
        want = want * 8
    else:
        got = hk.gemm_fp8(aq, bq, activation="none", out_dtype=F32)
    assert torch.equal(got.double(), want)


def test_fp32_extreme_exponents(hk):
    """Exponents whose sum is ordinary although each is far from it, to the stated limits."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    for m in (5, 400):
        aq = (torch.randint(0, 2, (m, 256), generator=gen, device="cuda") * 2 - 1).to(torch.float8_e4m3fn)
        bq = (torch.randint(0, 2, (256, 256), generator=gen, device="cuda") * 2 - 1).to(torch.float8_e4m3fn)
        for x, y in ((3, 246), (246, 3), (0, 127), (60, 190)):
            ea = torch.full((m, 8), x, dtype=torch.uint8, device="cuda")
            eb = torch.full((256, 8), y, dtype=torch.uint8, device="cuda")
            got = hk.gemm_mx(aq, hk.mx_pack_scales(ea), bq, hk.mx_pack_scales(eb), activation="none", out_dtype=F32)
            want = (aq.double() @ bq.double().T) * 2.0 ** (x + y - 254)
            assert torch.equal(got.double(), want), (x, y)


def test_no_epilogue_is_the_product(hk):
    """activation "none" without the rest is the plain product, bit for bit."""
    call, z = _operands(70, 512, 512, False, 4)
    assert torch.equal(call(hk, activation="none"), call(hk))
    assert torch.equal(call(hk), z.to(F32).to(BF16))


def test_no_rows(hk):
    aq = torch.empty((0, 128), device="cuda").to(torch.float8_e4m3fn)
    bq = torch.ones((256, 128), device="cuda").to(torch.float8_e4m3fn)
    res = torch.empty((0, 256), device="cuda", dtype=BF16)
    assert hk.gemm_fp8(aq, bq, activation="silu", bias=torch.ones(256, device="cuda"), residual=res).shape == (0, 256)


def test_far_rows(hk):
    """Outputs past 2^31 bytes and 2^31 elements: the last rows are those of a short call."""
    n, k = 65536, 128
    m = (1 << 31) // n + 300
    aq = (torch.randint(0, 2, (m, k), device="cuda") * 2 - 1).to(torch.float8_e4m3fn)
    bq = (torch.randint(0, 2, (n, k), device="cuda") * 2 - 1).to(torch.float8_e4m3fn)
    bias = torch.randn(n, device="cuda")
    res = torch.zeros((m, n), device="cuda", dtype=BF16)
    res[-256:] = torch.randn((256, n), device="cuda").to(BF16)
    got = hk.gemm_fp8(aq, bq, bias=bias, activation="relu", residual=res)
    few = hk.gemm_fp8(aq[-256:].contiguous(), bq, bias=bias, activation="relu", residual=res[-256:].contiguous())
    assert torch.equal(got[-256:], few)  # sums of +-1 are exact in every kernel


def test_refusals(hk):
    aq = torch.ones((4, 128), device="cuda").to(torch.float8_e4m3fn)
    bq = torch.ones((256, 128), device="cuda").to(torch.float8_e4m3fn)
    ok = torch.zeros(256, device="cuda")
    res = torch.zeros((4, 256), device="cuda", dtype=BF16)
    wide = torch.zeros((4, 512), device="cuda", dtype=BF16)
    for bad, says in ((dict(activation="swish"), "activation must be one of"), (dict(bias=ok[:128]), "bias must be"),
                      (dict(bias=ok.double()), "bias: expected"), (dict(bias=ok.cpu()), "GPU"),
                      (dict(bias=torch.zeros(260, device="cuda")[1:257]), "aligned"), (dict(residual=res.float()), "residual must have"),
                      (dict(residual=res[:3]), "residual must be"), (dict(residual=wide[:, :256]), "contiguous"),
                      (dict(activation="relu", out=res.float()[:3]), "C must be"), (dict(bias=torch.zeros(512, device="cuda")[::2]), "contiguous")):
        with pytest.raises(RuntimeError, match=says):
            hk.gemm_fp8(aq, bq, **bad)
    with pytest.raises(RuntimeError, match="packed"):
        hk.gemm_mx(aq, torch.zeros((1, 32), dtype=torch.int32, device="cuda"), bq,
                   torch.zeros((1, 256), dtype=torch.int32, device="cuda"), activation="relu")


def test_out_of_the_plain_products(hk):
    """C in a given tensor, without an epilogue as well; one that the stores would not fit is refused."""
    aq = torch.ones((4, 128), device="cuda").to(torch.float8_e4m3fn)
    bq = torch.ones((256, 128), device="cuda").to(torch.float8_e4m3fn)
    sa = hk.mx_pack_scales(torch.full((4, 4), 127, dtype=torch.uint8, device="cuda"))
    sb = hk.mx_pack_scales(torch.full((256, 4), 127, dtype=torch.uint8, device="cuda"))
    for call in (lambda out: hk.gemm_fp8(aq, bq, out=out), lambda out: hk.gemm_mx(aq, sa, bq, sb, out=out)):
        for dtype in (BF16, F32):
            buf = torch.zeros((6, 256), device="cuda", dtype=dtype)
            assert call(buf[1:5]).data_ptr() == buf[1:5].data_ptr()
            assert bool((buf[1:5] == 128).all()) and not buf[0].any() and not buf[5].any()
            with pytest.raises(RuntimeError, match="aligned"):
                call(buf.view(-1)[1:1025].view(4, 256))
            with pytest.raises(RuntimeError, match="device"):
                call(torch.zeros((4, 256), dtype=dtype))
        with pytest.raises(RuntimeError):
            call(torch.zeros((3, 256), device="cuda"))
        with pytest.raises(RuntimeError):
            call(torch.zeros((4, 256), device="cuda", dtype=torch.float16))


def test_streams_and_graph(hk):
    """Calls on two streams at once, and replays of a captured call with changing inputs, next to
    eager work."""
    (c1, z1), (c2, z2) = _operands(300, 1024, 512, False, 8), _operands(64, 1024, 512, True, 9)
    bias = _bias(1024, F32, 2)
    res = torch.randn(300, 1024, device="cuda").to(BF16)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(8):
        with torch.cuda.stream(s1):
            outs.append((c1(hk, bias=bias, activation="gelu", residual=res), z1, res, BF16, "gelu"))
        with torch.cuda.stream(s2):
            outs.append((c2(hk, bias=bias, activation="silu", out_dtype=F32), z2, None, F32, "silu"))
    torch.cuda.synchronize()
    for got, z, r, dtype, act in outs:
        _check(got, *ref.epilogue(z, bias, act, r, dtype))
    out = torch.empty((300, 1024), dtype=BF16, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c1(hk, bias=bias, activation="gelu", residual=res, out=out)
    for i in range(4):
        res.copy_(torch.randn(300, 1024, device="cuda"))
        bias.copy_(torch.randn(1024, device="cuda"))
        g.replay()
        eager = c1(hk, bias=bias, activation="gelu", residual=res)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_tensors_that_ask_for_a_gradient_are_refused(hk):
    aq, bq = torch.ones((4, 128), device="cuda").to(torch.float8_e4m3fn), torch.ones((256, 128), device="cuda").to(torch.float8_e4m3fn)
    bias, r = torch.zeros(256, device="cuda", requires_grad=True), torch.zeros((4, 256), device="cuda", dtype=BF16, requires_grad=True) * 1
    for bad in (dict(bias=bias), dict(residual=r), dict(out=r), dict(residual=r, out=r)):
        with pytest.raises(RuntimeError, match="asks for a gradient"):
            hk.gemm_fp8(aq, bq, **bad)
        assert not r.any()  # nothing ran
    assert bool((hk.gemm_fp8(aq, bq, bias=bias.detach(), residual=r.detach()) == 128).all())
    with torch.no_grad():
        assert bool((hk.gemm_fp8(aq, bq, bias=bias, residual=r, out=r) == 128).all())


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_tails(hk, act):
    """Small negative results keep the header's relative bounds down to 2^-119, rounded to bf16 as well, in strips
    and on every tile."""
    lo, hi = {"silu": (-105.0, -75.0), "gelu": (-14.0, -11.0), "gelu_tanh": (-11.0, -8.0)}[act]
    n = 1024
    z = torch.linspace(lo, hi, n, device="cuda")
    v = z.double()
    if act == "gelu":
        want, bound = v * ref.phi(v), (16 + v * v) * 2.0 ** -23
    else:
        e = v if act == "silu" else math.sqrt(8 / math.pi) * (v + 0.044715 * v ** 3)
        want, bound = v / (1 + torch.exp(-e)), (4 + (1.0 if act == "silu" else 2.5) * e.abs()) * 2.0 ** -23
    far = want.abs() >= 2.0 ** -119
    assert bool(far.any()) and not bool(far.all())
    bq = torch.zeros((n, 128), device="cuda").to(torch.float8_e4m3fn)
    for m in (1, 300, 2000, 5000, 20000):
        aq = torch.zeros((m, 128), device="cuda").to(torch.float8_e4m3fn)
        for dtype in (F32, BF16):
            got = hk.gemm_fp8(aq, bq, bias=z, activation=act, out_dtype=dtype)
            assert torch.equal(got, got[:1].expand_as(got))
            off = (got[0].double() - want).abs()
            allow = (bound + (0 if dtype == F32 else ref.half(dtype)) * (1 + bound)) * want.abs()
            assert bool((off <= allow)[far].all()), (m, dtype, float((off / want.abs())[far].max()))
            assert bool((off[~far] <= 2.0 ** -119).all())


@pytest.mark.parametrize("m,n,k", [(5, 256, 256), (40, 512, 1152), (2000, 1024, 256), (5000, 1024, 256)])
def test_nan_exponents(hk, m, n, k):
    """Exponent byte 255, e8m0's NaN, in blocks of A, of B and of zeros: NaN in the row or the column that the
    block is part of and nowhere else, on the widened operands (fp32 C), the FP8 instructions (bf16 C), and in
    the plain product alike."""
    gen = torch.Generator(device="cuda").manual_seed(m)
    pm1 = lambda *s: (torch.randint(0, 2, s, generator=gen, device="cuda") * 2 - 1).float()  # noqa: E731
    a, b = pm1(m, k), pm1(n, k)
    ea = torch.full((m, k // 32), 127, dtype=torch.uint8, device="cuda")
    eb = torch.full((n, k // 32), 127, dtype=torch.uint8, device="cuda")
    rows, cols = [0, m // 2, m - 1], [1, n // 2 + 3, n - 1]
    for i, (r, c) in enumerate(zip(rows, cols)):
        ea[r, (3 * i) % (k // 32)] = 255
        eb[c, (5 * i + 1) % (k // 32)] = 255
    z = ((3 * 2) % (k // 32)) * 32
    a[m - 1, z:z + 32] = 0.0
    aq, bq = a.to(torch.float8_e4m3fn), b.to(torch.float8_e4m3fn)
    want = aq.double() @ bq.double().T
    want[rows, :] = math.nan
    want[:, cols] = math.nan
    pa, pb = hk.mx_pack_scales(ea), hk.mx_pack_scales(eb)
    for dtype in (F32, BF16):
        for act in ("none", None):
            got = hk.gemm_mx(aq, pa, bq, pb, activation=act, out_dtype=dtype)
            assert torch.equal(got.double().nan_to_num(nan=1e9), want.float().to(dtype).double().nan_to_num(nan=1e9)), (dtype, act)
