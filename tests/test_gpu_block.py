"""Norm with 8-bit output, router product and adapters against plain 64-bit
implementations, at the sizes and masks where their tilings end, and the run of
them together in front of the layers, eager and from captured graphs."""
import numpy as np
import pytest
import torch

import block_ref
from helpers import bf16_np, f8_np
from oracle import fp8

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _bf16(a):
    return fp8.bf16_round(np.asarray(a, np.float32))


def _dev(a, dtype):
    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(dtype).cuda()


def _stream(rng, rows, cols, bf16):
    """A residual stream: a few large channels, rows of very different sizes."""
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    x[:, rng.integers(0, cols, max(1, cols // 100))] *= 20
    x *= np.float32(2.0) ** rng.integers(-8, 9, (rows, 1)).astype(np.float32)
    return _bf16(x) if bf16 else x


# ---------------------------------------------------------------------------
# norm
# ---------------------------------------------------------------------------
def _norm_case(hk, rows, cols, scales, x_bf16, w_bf16, residual, given=None, in_place=False, seed=0):
    rng = np.random.default_rng(rows * 31 + cols + seed)
    x = _stream(rng, rows, cols, x_bf16)
    res = _stream(rng, rows, cols, x_bf16) if residual else None
    w = (1.0 + 0.2 * rng.standard_normal(cols)).astype(np.float32)
    w = _bf16(w) if w_bf16 else w
    r_ref, n_ref = block_ref.rms_norm(x, res, w, 1e-6, x_bf16)
    q_ref, s_ref = block_ref.quantise(n_ref, scales, given)
    xt = BF16 if x_bf16 else F32
    xg, rg = _dev(x, xt), _dev(res, xt) if residual else None
    sg = None if given is None else torch.tensor([given], device="cuda")
    q, s, r, n = hk.rms_norm_quant(xg, _dev(w, BF16 if w_bf16 else F32), rg, scales=scales, scale=sg, with_norm=True,
                                   residual_out=rg if in_place else None)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(f8_np(q), q_ref)
    np.testing.assert_array_equal(s.cpu().numpy(), s_ref)
    np.testing.assert_array_equal(bf16_np(n), _bf16(n_ref))
    np.testing.assert_array_equal(bf16_np(r), r_ref)
    assert (r is xg) if not residual else (r is rg) if in_place else True
    if not in_place:
        np.testing.assert_array_equal(bf16_np(xg), x)
        if residual:
            np.testing.assert_array_equal(bf16_np(rg), res)


@pytest.mark.parametrize("scales,cols", [("group", 128), ("group", 640), ("group", 2560), ("group", 7168), ("group", 8192),
                                         ("group", 8320), ("group", 16384), ("group", 16512), ("group", 65536),
                                         ("mx", 32), ("mx", 160), ("mx", 4096), ("mx", 8224), ("mx", 33024),
                                         ("tensor", 8), ("tensor", 520), ("tensor", 4096), ("tensor", 20488)])
@pytest.mark.parametrize("rows", [1, 5])
@pytest.mark.parametrize("x_bf16", [True, False])
def test_norm_widths(hk, scales, cols, rows, x_bf16):
    _norm_case(hk, rows, cols, scales, x_bf16, x_bf16, True)


@pytest.mark.parametrize("scales", ["group", "mx", "tensor"])
@pytest.mark.parametrize("rows", [1, 2, 63, 300, 1023, 1025, 2500])
def test_norm_rows(hk, scales, rows):
    _norm_case(hk, rows, 256, scales, True, False, rows % 2 == 0, in_place=rows % 4 == 0)


@pytest.mark.parametrize("given", [0.01, 3.0, 1e-30])
@pytest.mark.parametrize("x_bf16", [True, False])
def test_norm_given_scale(hk, given, x_bf16):
    """A given scale: values past 448 scale saturate."""
    _norm_case(hk, 37, 520, "tensor", x_bf16, True, True, given=given)


@pytest.mark.parametrize("scales", ["group", "mx", "tensor"])
def test_norm_no_rows(hk, scales):
    x = torch.empty((0, 256), dtype=BF16, device="cuda")
    w = torch.ones(256, dtype=BF16, device="cuda")
    q, s, r, n = hk.rms_norm_quant(x, w, x.clone(), scales=scales, with_norm=True)
    assert q.shape == (0, 256) and r.shape == (0, 256) and n.shape == (0, 256)
    if scales == "tensor":
        assert s.item() == 1.0


@pytest.mark.parametrize("scales", ["group", "mx", "tensor"])
def test_norm_rows_of_zeros_and_non_finite(hk, scales):
    """Padding rows, and rows with a NaN or an infinity: the bytes and scales of the
    quantisers for the same n (a NaN's sign apart)."""
    rng = np.random.default_rng(5)
    x = _stream(rng, 6, 256, True)
    x[1] = 0
    x[2, 7] = np.nan
    x[3, 130] = np.inf
    x[4] = 1e30
    w = np.ones(256, np.float32)
    with np.errstate(all="ignore"):
        _, n = block_ref.rms_norm(x, None, w, 1e-6, True)
    ng = torch.from_numpy(n).cuda()
    q0, s0 = {"group": hk.quant_group, "mx": hk.quant_mx, "tensor": hk.quant_tensor}[scales](ng)
    q, s, _, norm = hk.rms_norm_quant(_dev(x, BF16), _dev(w, F32), scales=scales, with_norm=True)
    torch.cuda.synchronize()
    nan = np.isnan(n)
    got, want = f8_np(q), f8_np(q0)
    np.testing.assert_array_equal(np.where(nan, got & 0x7F, got), np.where(nan, want & 0x7F, want))
    np.testing.assert_array_equal(s.cpu().numpy(), s0.cpu().numpy())
    np.testing.assert_array_equal(np.isnan(bf16_np(norm)), nan)
    assert not f8_np(q)[1].any()


def test_norm_far_rows(hk):
    """Offsets past 2^31 values: the last rows of a long stream are those of a short one."""
    rows, cols = (1 << 31) // 8192 + 70, 8192
    x = torch.zeros((rows, cols), dtype=BF16, device="cuda")
    x[-64:] = torch.randn((64, cols), device="cuda").to(BF16)
    w = torch.rand(cols, device="cuda")
    for scales in ("group", "mx", "tensor"):
        q, s, _, n = hk.rms_norm_quant(x, w, scales=scales, with_norm=True)
        q1, s1, _, n1 = hk.rms_norm_quant(x[-64:], w, scales=scales, with_norm=True)
        assert torch.equal(q[-64:].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(n[-64:], n1)
        assert torch.equal(s[-64:] if scales != "tensor" else s, s1)
        del q, s, n


# ---------------------------------------------------------------------------
# router
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("t,e,h", [(1, 1, 8), (1, 128, 4096), (3, 60, 264), (15, 17, 128), (16, 16, 64), (17, 64, 72),
                                   (33, 256, 1000), (64, 128, 4096), (65, 130, 520), (129, 8, 2048), (300, 1024, 256),
                                   (1000, 60, 2048), (2050, 256, 1032), (4100, 129, 512)])
def test_router(hk, t, e, h):
    """Off by one rounding of 2^-24 of the terms' magnitudes per step of a sum at most."""
    rng = np.random.default_rng(t + e + h)
    x, w = _bf16(rng.standard_normal((t, h))), _bf16(rng.standard_normal((e, h)))
    buf = torch.full((t * e + 64,), 7.0, device="cuda")
    out = hk.router_logits(_dev(x, BF16), _dev(w, BF16), out=buf[: t * e].view(t, e))
    torch.cuda.synchronize()
    ref = x.astype(np.float64) @ w.astype(np.float64).T
    mag = np.abs(x).astype(np.float64) @ np.abs(w).astype(np.float64).T
    assert (np.abs(out.cpu().numpy() - ref) <= (h + 8) * 2.0 ** -24 * mag).all()
    assert bool((buf[t * e:] == 7.0).all())


def test_router_exact_integers(hk):
    """Small whole numbers: every product and sum is exact, so every logit is."""
    rng = np.random.default_rng(0)
    for t, e, h in [(7, 60, 1000), (130, 256, 4096), (3000, 200, 640)]:
        x, w = rng.integers(-3, 4, (t, h)).astype(np.float32), rng.integers(-3, 4, (e, h)).astype(np.float32)
        out = hk.router_logits(_dev(x, BF16), _dev(w, BF16))
        np.testing.assert_array_equal(out.cpu().numpy(), x @ w.T)


def test_router_non_finite_stays_in_its_row(hk):
    x = torch.randn((70, 256), device="cuda").to(BF16)
    w = torch.randn((33, 256), device="cuda").to(BF16)
    clean = hk.router_logits(x, w)
    x[5, 9] = float("nan")
    x[66, 0] = float("inf")
    out = hk.router_logits(x, w)
    rows = torch.ones(70, dtype=torch.bool, device="cuda")
    rows[5] = rows[66] = False
    assert torch.equal(out[rows], clean[rows]) and bool(out[5].isnan().all()) and not bool(out[66].isfinite().any())


def test_router_no_tokens(hk):
    x = torch.empty((0, 64), dtype=BF16, device="cuda")
    assert hk.router_logits(x, torch.ones((4, 64), dtype=BF16, device="cuda")).shape == (0, 4)


# ---------------------------------------------------------------------------
# adapters
# ---------------------------------------------------------------------------
def _ids(rng, t, adapters, how):
    if how == "none":
        return np.full(t, -1, np.int32)
    if how == "one":
        return np.full(t, adapters - 1, np.int32)
    ids = rng.integers(-1, adapters, t).astype(np.int32)
    if how == "segments":
        return np.sort(ids)[::-1].copy()
    if how == "out of range":
        ids[rng.integers(0, t, (t + 3) // 4)] = rng.choice([adapters, adapters + 1, -2, -2 ** 31, 2 ** 31 - 1], (t + 3) // 4)
    return ids


def _lora_data(rng, t, h, n, r, adapters, bf16):
    y = rng.standard_normal((t, n)).astype(np.float32)
    return (_bf16(y) if bf16 else y, _bf16(rng.standard_normal((t, h))),
            _bf16(rng.standard_normal((adapters, r, h)) * h ** -0.5),
            _bf16(rng.standard_normal((adapters, n, r)) * r ** -0.5), rng.uniform(-2, 2, adapters).astype(np.float32))


def _lora_case(hk, t, h, n, r, adapters, how, bf16=True, wide=0, in_place=False, scaled=True):
    rng = np.random.default_rng(t * 7 + h + n + r)
    y, x, a, b, c = _lora_data(rng, t, h, n, r, adapters, bf16)
    ids = _ids(rng, t, adapters, how)
    dt = BF16 if bf16 else F32
    # y and out as slices: what lies beside and behind them must stay untouched
    ybuf = torch.full((t + 2, n + 2 * wide), 3.0, dtype=dt, device="cuda")
    yg = ybuf[:t, wide:wide + n]
    yg.copy_(_dev(y, dt))
    xbuf = torch.full((t + 1, h + wide), float("nan"), dtype=BF16, device="cuda")
    xg = xbuf[:t, :h]
    xg.copy_(_dev(x, BF16))
    obuf = ybuf if in_place else torch.full((t + 2, n + 2 * wide), 3.0, dtype=dt, device="cuda")
    og = obuf[:t, wide:wide + n]
    out = hk.lora_add(yg, xg, _dev(a, BF16), _dev(b, BF16), torch.from_numpy(ids).cuda(),
                      torch.from_numpy(c).cuda() if scaled else None, out=og)
    torch.cuda.synchronize()
    assert out is og
    ref, mag = block_ref.lora(y, x, a, b, ids, c if scaled else None)
    bound = block_ref.lora_bound(ref, mag, h, r, bf16)
    got = bf16_np(out).astype(np.float64)
    off = np.abs(got - ref) - bound
    assert (off <= 0).all(), (np.argwhere(off > 0)[:5], off.max())
    bare = ~((ids >= 0) & (ids < adapters))
    np.testing.assert_array_equal(got[bare], y[bare])
    assert bool((obuf[t:] == 3.0).all()) and bool((obuf[:, :wide] == 3.0).all()) and bool((obuf[:, wide + n:] == 3.0).all())
    if not in_place:
        np.testing.assert_array_equal(bf16_np(yg), y)


@pytest.mark.parametrize("t", [1, 2, 15, 16, 17, 63, 64, 65, 129, 300])
@pytest.mark.parametrize("how", ["none", "one", "mixed", "segments", "out of range"])
def test_lora_rows(hk, t, how):
    _lora_case(hk, t, 264, 264, 16, 5, how, bf16=t % 2 == 0, wide=0 if t % 3 else 8, in_place=t % 4 == 1)


@pytest.mark.parametrize("h", [8, 24, 64, 72, 1000, 4096, 8200])
@pytest.mark.parametrize("bf16", [True, False])
def test_lora_hidden(hk, h, bf16):
    _lora_case(hk, 33, h, 256, 8, 3, "mixed", bf16=bf16)


@pytest.mark.parametrize("n", [8, 16, 56, 64, 72, 248, 256, 264, 1000, 4104])
@pytest.mark.parametrize("bf16", [True, False])
def test_lora_columns(hk, n, bf16):
    _lora_case(hk, 70, 128, n, 24, 4, "mixed", bf16=bf16, wide=16, in_place=bf16)


@pytest.mark.parametrize("r", [8, 16, 24, 32, 40, 64, 72, 128, 136, 256])
@pytest.mark.parametrize("bf16", [True, False])
def test_lora_ranks(hk, r, bf16):
    _lora_case(hk, 40, 512, 136, r, 4, "mixed", bf16=bf16, scaled=r % 16 == 0)


@pytest.mark.parametrize("h", [8, 72, 120, 1000, 4096])
@pytest.mark.parametrize("r", [8, 16, 24, 32, 40, 64, 72, 200])
def test_lora_panels(hk, h, r):
    """More than 16 rows of an adapter: every rank tile, ragged and whole K."""
    _lora_case(hk, 90, h, 72, r, 2, "one", bf16=r % 16 == 0)


@pytest.mark.parametrize("t,adapters,how", [(64, 70, "mixed"), (256, 300, "mixed"), (2000, 3, "segments"),
                                            (5000, 64, "segments"), (1500, 200, "mixed")])
def test_lora_many(hk, t, adapters, how):
    """Blocks with a different adapter in every row, and more rows than one round of workgroups."""
    _lora_case(hk, t, 128, 320, 16, adapters, how)


@pytest.mark.parametrize("t,r", [(1, 72), (15, 136), (16, 72), (17, 72), (33, 256), (63, 72), (64, 136), (65, 72), (130, 72),
                                 (204, 40), (205, 40), (257, 64), (1024, 32), (1025, 32), (2049, 16)])
@pytest.mark.parametrize("how", ["none", "one", "mixed", "segments", "out of range"])
def test_lora_matrix_rows(hk, t, r, how):
    """Ranks and row counts on both sides of the matrix instruction's share."""
    _lora_case(hk, t, 72, 264, r, 5, how, bf16=(t + r) % 2 == 0, wide=8 if t % 3 else 0, in_place=t % 4 == 1)


@pytest.mark.parametrize("n", [8, 56, 64, 72, 248, 256, 264, 520, 1032, 4104])
@pytest.mark.parametrize("bf16", [True, False])
def test_lora_matrix_columns(hk, n, bf16):
    _lora_case(hk, 70, 64, n, 72, 4, "mixed", bf16=bf16, wide=16, in_place=bf16)


@pytest.mark.parametrize("t,n,r,bf16", [(2100, 4104, 16, True), (2100, 2056, 24, False), (1100, 8200, 72, True)])
def test_lora_large_outputs(hk, t, n, r, bf16):
    """Outputs past what the caches hold."""
    _lora_case(hk, t, 64, n, r, 6, "segments", bf16=bf16)
    _lora_case(hk, t, 64, n, r, 6, "mixed", bf16=bf16, in_place=True)


@pytest.mark.parametrize("how", ["none", "one", "mixed", "segments", "out of range"])
@pytest.mark.parametrize("t,adapters,r,h", [(65, 200, 128, 2048), (130, 64, 64, 2048), (1000, 20, 72, 1032), (1029, 64, 16, 1048),
                                            (2500, 1535, 8, 1024), (2500, 1536, 8, 1024), (9000, 20, 72, 264), (66, 65, 256, 2056)])
def test_lora_sorted_first(hk, t, adapters, r, h, how):
    """Batches whose rows are sorted by adapter first (and, at 1536 adapters, just not)."""
    _lora_case(hk, t, h, 72, r, adapters, how, bf16=t % 2 == 0, in_place=t % 4 == 2)


def test_lora_sorted_first_same_bits(hk):
    """The groups, and with them the order of each row's sums, are the same every time."""
    rng = np.random.default_rng(11)
    y, x, a, b, c = _lora_data(rng, 1500, 2048, 264, 64, 40, False)
    args = [_dev(y, F32), _dev(x, BF16), _dev(a, BF16), _dev(b, BF16),
            torch.from_numpy(rng.integers(-1, 40, 1500).astype(np.int32)).cuda(), torch.from_numpy(c).cuda()]
    first = hk.lora_add(*args)
    for _ in range(20):
        assert torch.equal(hk.lora_add(*args), first)


def test_lora_sorted_first_from_graphs(hk):
    """Two graphs of one sorted batch on a stream of their own, replayed in turn with other ids
    each time and eager calls between."""
    rng = np.random.default_rng(12)
    y, x, a, b, c = _lora_data(rng, 1500, 2048, 264, 64, 40, True)
    ids = torch.zeros(1500, dtype=torch.int32, device="cuda")
    args = [_dev(y, BF16), _dev(x, BF16), _dev(a, BF16), _dev(b, BF16), ids, torch.from_numpy(c).cuda()]
    hk.lora_add(*args)
    side = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = hk.lora_add(*args)
        graphs.append((g, out))
    for k, how in enumerate(["mixed", "none", "segments", "one", "out of range", "mixed"]):
        ids.copy_(torch.from_numpy(_ids(rng, 1500, 40, how)))
        eager = hk.lora_add(*args)
        g, out = graphs[k % 2]
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), how
        assert torch.equal(hk.lora_add(*args), eager), how


def test_lora_far_offsets(hk):
    """An adapter whose weights lie past 2^31 values, and far rows of strided x, y and out."""
    l, r, h, n = 140, 256, 65536, 512
    a = torch.zeros((l, r, h), dtype=BF16, device="cuda")
    a[-1] = torch.randn((r, h), device="cuda").to(BF16) * h ** -0.5
    b = torch.randn((l, n, r), device="cuda").to(BF16)
    t, step = 70, 32_000_000  # 70 rows, 2.2e9 values apart in all
    xbuf = torch.zeros(t * step, dtype=BF16, device="cuda")
    x = xbuf.as_strided((t, h), (step, 1))
    x.copy_(torch.randn((t, h), device="cuda").to(BF16))
    y = torch.zeros((t, n), device="cuda")
    ids = torch.full((t,), l - 1, dtype=torch.int32, device="cuda")
    out = hk.lora_add(y, x, a, b, ids)
    ref = hk.lora_add(y, x.contiguous(), a[-1:].clone(), b[-1:].clone(), torch.zeros_like(ids))
    assert torch.equal(out, ref) and bool(out.abs().max() > 0)
    ybuf = torch.zeros(t * step, dtype=F32, device="cuda")
    yo = ybuf.as_strided((t, n), (step, 1))
    hk.lora_add(yo, x, a, b, ids, out=yo)
    assert torch.equal(yo, ref)


def test_lora_no_rows(hk):
    y = torch.empty((0, 64), dtype=BF16, device="cuda")
    x = torch.empty((0, 32), dtype=BF16, device="cuda")
    a, b = torch.ones((2, 8, 32), dtype=BF16, device="cuda"), torch.ones((2, 64, 8), dtype=BF16, device="cuda")
    assert hk.lora_add(y, x, a, b, torch.empty(0, dtype=torch.int32, device="cuda")).shape == (0, 64)


def test_lora_non_finite_stays_in_its_row(hk):
    rng = np.random.default_rng(3)
    y, x, a, b, c = (torch.from_numpy(v).cuda() for v in _lora_data(rng, 70, 256, 264, 16, 3, True))
    y, x, a, b = y.to(BF16), x.to(BF16), a.to(BF16), b.to(BF16)
    ids = torch.arange(70, device="cuda", dtype=torch.int32) % 3
    clean = hk.lora_add(y, x, a, b, ids, c)
    x[5, 9] = float("nan")
    x[66, 0] = float("inf")
    y[9, 3] = float("nan")
    a2 = torch.cat([a, torch.full_like(a[:1], float("nan"))])  # an adapter that no row uses
    b2 = torch.cat([b, torch.full_like(b[:1], float("inf"))])
    out = hk.lora_add(y, x, a2, b2, ids, torch.cat([c, c[:1]]))
    rows = torch.ones(70, dtype=torch.bool, device="cuda")
    rows[5] = rows[66] = rows[9] = False
    assert torch.equal(out[rows], clean[rows])
    assert bool(out[5].isnan().all()) and not bool(out[66].isfinite().any())
    assert bool(out[9, 3].isnan()) and torch.equal(out[9, 4:], clean[9, 4:])


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
T, H, I, E, K, N, R, L = 150, 512, 256, 16, 4, 512, 16, 5


def _weights(hk, seed, scales):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def rand(*s):
        return torch.randn(s, generator=g, device="cuda") * s[-1] ** -0.5
    w13, w2 = rand(E, 2 * I, H), rand(E, H, I)
    if scales == "mx":
        q13, s13 = hk.quant_mx(w13.view(-1, H))
        q2, s2 = hk.quant_mx(w2.view(-1, I))
        layer = hk.MoELayerMX(q13.view(E, 2 * I, H), s13.view(E, 2 * I, -1), q2.view(E, H, I), s2.view(E, H, -1), K)
        wq, ws = hk.quant_mx(rand(N, H))
    else:
        if scales == "group":
            layer = hk.MoELayer(*hk.quant_block(w13), *hk.quant_block(w2), K)
        else:
            q13, s13 = zip(*[hk.quant_tensor(w) for w in w13])
            q2, s2 = zip(*[hk.quant_tensor(w) for w in w2])
            f8 = torch.float8_e4m3fn
            stack = lambda q: torch.stack([v.view(torch.uint8) for v in q]).view(f8)  # noqa: E731
            layer = hk.MoELayer(stack(q13), torch.cat(s13), stack(q2), torch.cat(s2), K)
        wq, ws = hk.quant_tensor(rand(N, H))
    return dict(layer=layer, norm=1 + 0.1 * rand(1, H)[0] * H ** 0.5, router=rand(E, H).to(BF16), wq=wq, ws=ws,
                a=rand(L, R, H).to(BF16), b=rand(L, N, R).to(BF16), c=torch.rand(L, generator=g, device="cuda"))


class _Chain:
    """One decoder layer's worth: projection with adapters from the stream, then the MoE block."""

    def __init__(self, hk, scales):
        d = _weights(hk, 1, scales)
        self.hk, self.d, self.scales = hk, d, "mx" if scales == "mx" else "tensor"
        self.proj = hk.LoraLinear(d["wq"], d["ws"], d["a"], d["b"], d["c"])
        self.block = hk.MoEBlock(d["norm"], d["router"], d["layer"])

    def __call__(self, x, residual, ids):
        q, s, r, n = self.hk.rms_norm_quant(x, self.d["norm"], residual, scales=self.scales, with_norm=True)
        y = self.proj(q, s, n, ids)
        out, r2 = self.block(y, r)
        return out, r2, y


def _inputs(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn((T, H), generator=g, device="cuda").to(BF16), torch.randn((T, H), generator=g, device="cuda").to(BF16),
            torch.randint(-1, L, (T,), generator=g, device="cuda", dtype=torch.int32))


@pytest.mark.parametrize("scales", ["group", "mx", "tensor"])
def test_together(hk, scales):
    """The classes against the single calls, and those against fp32 of the same operands."""
    chain = _Chain(hk, scales)
    d = chain.d
    x, res, ids = _inputs(2)
    out, r2, y = chain(x, res, ids)
    q, s, r, n = hk.rms_norm_quant(x, d["norm"], res, scales=chain.scales, with_norm=True)
    base = (hk.gemm_mx(q, hk.mx_pack_scales(s), d["wq"], hk.mx_pack_scales(d["ws"]), out_dtype=BF16) if scales == "mx"
            else hk.gemm_fp8(q, d["wq"], s, d["ws"]))
    assert torch.equal(y, hk.lora_add(base, n, d["a"], d["b"], ids, d["c"]))
    assert torch.equal(r, (x.float() + res.float()).to(BF16))
    q2, s2, r3, n2 = hk.rms_norm_quant(y, d["norm"], r, scales=chain.block.scales, with_norm=True)
    logits = hk.router_logits(n2, d["router"])
    assert torch.equal(r2, r3) and torch.equal(out, d["layer"](q2, s2, logits))
    # 512 products: 2^-24 of the magnitudes for each
    ref = n2.cpu().double() @ d["router"].cpu().double().T
    mag = n2.cpu().double().abs() @ d["router"].cpu().double().abs().T
    assert bool(((logits.cpu().double() - ref).abs() <= (H + 8) * 2.0 ** -24 * mag).all())
    assert bool(out.isfinite().all())


@pytest.mark.parametrize("scales", ["group", "mx", "tensor"])
def test_together_from_a_graph(hk, scales):
    """Two graphs of the run, replayed in turn with eager calls and new inputs between."""
    chain = _Chain(hk, scales)
    sets = [_inputs(s) for s in (3, 4, 5)]
    eager = [[v.clone() for v in chain(*s)] for s in sets]
    torch.cuda.synchronize()
    graphs = []
    for s in sets[:2]:
        static = [v.clone() for v in s]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = chain(*static)
        graphs.append((g, static, out))
    for k in range(6):
        g, static, out = graphs[k % 2]
        want = eager[k % 3]
        for a, b in zip(static, sets[k % 3]):
            a.copy_(b)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k
        again = chain(*sets[(k + 1) % 3])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(again, eager[(k + 1) % 3])), k


def test_on_another_stream(hk):
    """On a side stream, with the inputs still being written there when the call is made."""
    chain = _Chain(hk, "group")
    x, res, ids = _inputs(6)
    want = [v.clone() for v in chain(x, res, ids)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = torch.zeros_like(x)
        for _ in range(20):
            late.copy_(x)
        got = chain(late, res, ids)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_streams_at_once(hk):
    """Calls that overlap in time: each takes its workspace from the allocator."""
    chains, sets = [_Chain(hk, "mx"), _Chain(hk, "tensor")], [_inputs(8), _inputs(9)]
    want = [[v.clone() for v in c(*s)] for c, s in zip(chains, sets)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in chains]
    got = [[], []]
    for _ in range(10):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(chains[k](*sets[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for g in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[k]))


def test_same_bits_every_time(hk):
    x, res, ids = _inputs(7)
    chain = _Chain(hk, "tensor")
    first = [v.clone() for v in chain(x, res, ids)]
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(chain(x, res, ids), first))


def test_refusals_on_the_device(hk):
    """Checked on the host, with real tensors: nothing is launched."""
    x = torch.zeros((4, 256), dtype=BF16, device="cuda")
    w = torch.ones(256, dtype=BF16, device="cuda")
    for bad in (dict(x=x[:, ::2]), dict(x=x.half()), dict(x=x[0]), dict(residual=x.float()), dict(residual=x[:2]),
                dict(scales="row"), dict(scale=torch.ones(1, device="cuda")), dict(eps=0.0), dict(residual_out=x.clone()),
                dict(weight=w[:128]), dict(x=x[:, :200].contiguous(), weight=w[:200].contiguous()), dict(x=x.cpu())):
        args = dict(x=x, weight=w)
        args.update(bad)
        with pytest.raises(RuntimeError):
            hk.rms_norm_quant(**args)
    r = torch.zeros((8, 256), dtype=BF16, device="cuda")
    for a, b in ((x.float(), r), (x, r.float()), (x, r[:, :128].contiguous()), (x[:, :100].contiguous(), r[:, :100].contiguous()),
                 (x, torch.zeros((1025, 256), dtype=BF16, device="cuda"))):
        with pytest.raises(RuntimeError):
            hk.router_logits(a, b)
    y = torch.zeros((4, 64), dtype=BF16, device="cuda")
    a, b = torch.zeros((2, 8, 256), dtype=BF16, device="cuda"), torch.zeros((2, 64, 8), dtype=BF16, device="cuda")
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    ok = dict(y=y, x=x, a=a, b=b, ids=ids)
    for bad in (dict(y=y.half()), dict(x=x.float()), dict(x=x[:3]), dict(ids=ids.long()), dict(ids=ids[:3]), dict(b=b[:1]),
                dict(a=a[:, :4].contiguous(), b=b[:, :, :4].contiguous()), dict(scaling=torch.ones(3, device="cuda")),
                dict(out=y.float()), dict(out=y[:, :32]), dict(y=y.t()), dict(y=y.t().contiguous().t()),
                dict(y=torch.zeros((4, 65), dtype=BF16, device="cuda")[:, 1:]), dict(a=a.transpose(1, 2)),
                dict(workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))):
        args = dict(ok)
        args.update(bad)
        with pytest.raises(RuntimeError):
            hk.lora_add(**args)
    hk.lora_add(**ok)


@pytest.mark.parametrize("scales", ["group", "mx", "tensor"])
def test_one_block_on_two_streams(hk, scales):
    """Calls of one block that overlap in time, on inputs of their own."""
    d = _weights(hk, 1, scales)
    block = hk.MoEBlock(d["norm"], d["router"], d["layer"])
    sets = [_inputs(s)[:2] for s in (10, 11)]
    want = [[v.clone() for v in block(*s)] for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(10):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(block(*sets[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for g in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[k]))


def test_block_graph_beside_larger_calls(hk):
    """A graph of the block replayed after eager calls of more tokens, which need a larger workspace."""
    d = _weights(hk, 1, "group")
    block = hk.MoEBlock(d["norm"], d["router"], d["layer"])
    x, res, _ = _inputs(12)
    want = [v.clone() for v in block(x, res)]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = block(x, res)
    for k in (2, 5, 9):
        big = block(x.repeat(k, 1), res.repeat(k, 1))
        held = torch.zeros(1 << 22, device="cuda")  # takes whatever memory is free now
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k
        assert not held.any() and all(bool(v.isfinite().all()) for v in big)


@pytest.mark.parametrize("scales", ["group", "mx"])
def test_layer_graph_beside_larger_calls(hk, scales):
    """The same for a layer called by itself, whose workspace is cached."""
    layer = _weights(hk, 1, scales)["layer"]
    quant = hk.quant_mx if scales == "mx" else hk.quant_group
    g = torch.Generator(device="cuda").manual_seed(13)
    x_q, x_s = quant(torch.randn((T, H), generator=g, device="cuda"))
    logits = torch.randn((T, E), generator=g, device="cuda")
    want = layer(x_q, x_s, logits).clone()
    out = torch.empty_like(want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(x_q, x_s, logits, out=out)
    seen = layer._ws
    size = seen.numel()
    del seen
    for k in (2, 5, 9):
        big = layer(*(v.view(torch.uint8).repeat(k, 1).view(v.dtype) for v in (x_q, x_s, logits)))
        held = torch.zeros(size, dtype=torch.uint8, device="cuda")  # would take the first workspace's place
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(big[:T], big[-T:]) and not held.any(), k


# ---------------------------------------------------------------------------
# norm: scales and epsilons at the ends of their range
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("given", [1e-44, 2e-38, 1e30, 1e36, 3e38])
def test_norm_given_scale_at_the_ends(hk, given):
    """Subnormal scales, and scales of which 448 is past fp32: values past 448 scale saturate, an
    infinite one too."""
    rng = np.random.default_rng(17)
    x = rng.standard_normal((6, 520)).astype(np.float32)
    x[2:4] = 0
    x[2, 3], x[3, 3] = -5, 5  # n = -sqrt(520) w and sqrt(520) w there
    w = (rng.standard_normal(520).astype(np.float32) * np.float32(30 * min(given, 1e36))).astype(np.float32)
    w[3] = np.float32(min(3e37, 100 * given))
    with np.errstate(all="ignore"):
        _, n = block_ref.rms_norm(x, None, w, 1e-6, False)
        q_ref, _ = block_ref.quantise(n, "tensor", given)
    assert given < 1e36 or np.isinf(n[2, 3])
    assert q_ref[2, 3] == 0xFE and q_ref[3, 3] == 0x7E
    q = hk.rms_norm_quant(_dev(x, F32), _dev(w, F32), scales="tensor", scale=torch.tensor([given], device="cuda"))[0]
    torch.cuda.synchronize()
    np.testing.assert_array_equal(f8_np(q), q_ref)


@pytest.mark.parametrize("scales", ["group", "mx", "tensor", "given"])
@pytest.mark.parametrize("eps", [1e-80, 1e-300])
def test_norm_rows_of_zeros_tiny_eps(hk, scales, eps):
    """1 / sqrt(eps) past fp32: rows of zeros stay zeros, the others do not notice."""
    rng = np.random.default_rng(18)
    x = rng.standard_normal((5, 256)).astype(np.float32)
    x[1] = x[4] = 0
    w = np.ones(256, np.float32)
    _, n_ref = block_ref.rms_norm(x, None, w, 1e-30, False)  # far below the other rows' last bit
    given = 0.01 if scales == "given" else None
    q_ref, s_ref = block_ref.quantise(n_ref, "tensor" if given else scales, given)
    q, s, _, n = hk.rms_norm_quant(_dev(x, F32), _dev(w, F32), scales="tensor" if given else scales, eps=eps, with_norm=True,
                                   scale=torch.tensor([given], device="cuda") if given else None)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(bf16_np(n), _bf16(n_ref))
    np.testing.assert_array_equal(f8_np(q), q_ref)
    np.testing.assert_array_equal(s.cpu().numpy(), s_ref)


@pytest.mark.parametrize("t,r,n", [(1023, 16, 8192), (1024, 16, 8192), (127, 64, 4096), (128, 64, 4096), (511, 32, 4096), (512, 32, 4096)])
@pytest.mark.parametrize("how", ["mixed", "segments"])
@pytest.mark.parametrize("bf16", [True, False])
def test_lora_rows_at_the_small_kernels_end(hk, t, r, n, how, bf16):
    """The last shapes in which a row reads its own B, and the first after them."""
    _lora_case(hk, t, 72, n, r, 9, how, bf16=bf16, in_place=bf16)


# ---------------------------------------------------------------------------
# adapters: v's terms, held to equality
# ---------------------------------------------------------------------------
def _exact_lora(hk, t, h, n, r, adapters, how, bf16):
    rng = np.random.default_rng(t + h + r)
    x, a, b, c, v = block_ref.lora_exact_inputs(rng, t, h, n, r, adapters, bf16)
    ids = _ids(rng, t, adapters, how)
    y = np.zeros((t, n), np.float32)
    ref = block_ref.lora(y, x, a, b, ids, c)[0]
    out = hk.lora_add(_dev(y, BF16 if bf16 else F32), _dev(x, BF16), _dev(a, BF16), _dev(b, BF16), torch.from_numpy(ids).cuda(),
                      torch.from_numpy(c).cuda())
    torch.cuda.synchronize()
    np.testing.assert_array_equal(bf16_np(out).astype(np.float64), ref)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("how", ["one", "mixed", "segments"])
@pytest.mark.parametrize("t,adapters,r,h", [(40, 2, 72, 4096), (40, 12, 72, 4096), (20, 3, 256, 264), (300, 4, 64, 1024),
                                            (1100, 6, 32, 2048), (1000, 20, 72, 1032), (2500, 40, 16, 1048), (150, 3, 200, 8200),
                                            (33, 5, 16, 4096)])
def test_lora_exact_terms(hk, t, adapters, r, h, how, bf16):
    """Whole numbers whose every product and sum is exact, with a v that needs all of its terms: the
    matrix instruction's two (three for an fp32 output), split and unsplit sums, few and many rows
    of an adapter, sorted or not, and the small kernel's plain products."""
    _exact_lora(hk, t, h, 136, r, adapters, how, bf16)


# ---------------------------------------------------------------------------
# more rows than one pass of the grid, or than are sorted
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("scales", ["group", "mx", "tensor"])
def test_norm_more_rows_than_workgroups(hk, scales):
    rows, cols = (1 << 20) + 70, 128
    g = torch.Generator(device="cuda").manual_seed(19)
    x, res = (torch.randn((rows, cols), generator=g, device="cuda").to(BF16) for _ in range(2))
    w = torch.rand(cols, generator=g, device="cuda")
    scale = torch.full((1,), 0.01, device="cuda") if scales == "tensor" else None  # given: independent of the other rows
    q, s, r, n = hk.rms_norm_quant(x, w, res, scales=scales, scale=scale, with_norm=True)
    for part in (slice(0, 200), slice((1 << 20) - 60, rows)):
        q1, s1, r1, n1 = hk.rms_norm_quant(x[part], w, res[part], scales=scales, scale=scale, with_norm=True)
        assert torch.equal(q[part].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(n[part], n1)
        assert torch.equal(r[part], r1) and (scale is not None or torch.equal(s[part], s1))


@pytest.mark.parametrize("t,e,h", [(70001, 8, 64), (100003, 60, 72)])
def test_router_many_rows(hk, t, e, h):
    rng = np.random.default_rng(t)
    x, w = rng.integers(-3, 4, (t, h)).astype(np.float32), rng.integers(-3, 4, (e, h)).astype(np.float32)
    np.testing.assert_array_equal(hk.router_logits(_dev(x, BF16), _dev(w, BF16)).cpu().numpy(), x @ w.T)


@pytest.mark.parametrize("how", ["mixed", "segments"])
@pytest.mark.parametrize("r,bf16", [(8, True), (72, False)])
def test_lora_more_rows_than_are_sorted(hk, r, bf16, how):
    _lora_case(hk, 65536 + 70, 72, 72, r, 5, how, bf16=bf16, in_place=bf16)
