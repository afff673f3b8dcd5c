"""Layer norm, the router's choice, tokens by expert and back, and their gradients against
the formulas in 64 bits, at the sizes and masks where their launches change, and a block of them
together, eager, on several streams and from captured graphs."""
import math

import pytest
import torch

import train_ref as ref

pytestmark = pytest.mark.gpu

BF16, F32, F8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
PARTS = 256  # workgroups that dweight's rows are spread over


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _check(got, want, bound, what=""):
    assert got.shape == want.shape, what
    off = (got.double() - want).abs() - bound
    assert not bool((off > 0).any()) and not bool(torch.isnan(off).any()), (what, float(off.max()))


# ---------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------
def _norm_inputs(rows, cols, dtype, wdtype, seed, centre=2.0):
    gen = _gen(seed)
    x = _randn(gen, rows, cols)
    x[:, torch.randint(0, cols, (max(1, cols // 100),), generator=gen, device="cuda")] *= 20
    x = x * torch.exp2(torch.randint(-8, 9, (rows, 1), generator=gen, device="cuda").float()) + centre * _randn(gen, rows, 1)
    return (x.to(dtype), (1 + 0.2 * _randn(gen, cols)).to(wdtype), (0.3 * _randn(gen, cols)).to(wdtype), gen)


def _norm_case(hk, rows, cols, dtype, wdtype, residual=True, bias=True, dr=True, in_place=False, eps=1e-5, centre=2.0):
    x, w, b, gen = _norm_inputs(rows, cols, dtype, wdtype, rows * 31 + cols, centre)
    b = b if bias else None
    res = (2 * _randn(gen, rows, cols)).to(dtype) if residual else None
    want_r = x if res is None else (x.float() + res.float()).to(dtype)
    y, r, stats = hk.layer_norm_forward(x, w, b, res, eps=eps, residual_out=res if in_place and residual else None)
    torch.cuda.synchronize()
    assert torch.equal(r, want_r) and (r is res) == (in_place and residual)
    r64, w64 = want_r.double(), w.double()
    want, m, rstd = ref.layer_norm(r64, w64, None if b is None else b.double(), eps)
    _check(y, want, ref.layer_norm_bound(want, r64, w64, m, rstd, dtype), "y")
    dy = _randn(gen, rows, cols).to(dtype)
    back = _randn(gen, rows, cols).to(dtype) if dr else None
    got = hk.layer_norm_backward(dy, r, w, stats, dr=back, with_bias=bias)
    torch.cuda.synchronize()
    args = (dy.double(), r64, w64, eps, None if back is None else back.double())
    # additions behind each other: a part's rows, or a lane's share of up to 512 rows in 24 or 1024 in 72 (22,
    # 15); and then 8 to 16 parts or lanes and waves
    each = max(22, math.ceil(rows / PARTS)) + 16
    for name, g, v, bd in zip(("dx", "dw", "db"), got, ref.layer_norm_grad(*args), ref.layer_norm_grad_bound(*args, dtype, wdtype, each)):
        if name == "db" and not bias:
            assert g is None
        else:
            _check(g, v, bd, name)


@pytest.mark.parametrize("cols", [8, 120, 128, 136, 256, 264, 512, 520, 1024, 1032, 2560, 4096, 7168, 8192, 8200, 16384])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [1, 5])
def test_norm_widths(hk, cols, dtype, rows):
    _norm_case(hk, rows, cols, dtype, (BF16, F32)[cols // 8 % 2], residual=rows == 5)


@pytest.mark.parametrize("rows", [2, 4, 16, 17, 32, 33, 63, 64, 255, 256, 257, 1000, 4099])
@pytest.mark.parametrize("cols", [64, 200, 384, 1000, 1400])
def test_norm_rows(hk, rows, cols):
    _norm_case(hk, rows, cols, (BF16, F32)[rows % 2], F32, residual=rows % 3 != 0, bias=rows % 5 != 0, dr=rows % 2 == 0,
               in_place=rows % 2 == 1)


@pytest.mark.parametrize("rows", [511, 512, 513, 1023, 1024, 1025])
@pytest.mark.parametrize("cols", [72, 520, 1160, 4096, 4104, 8200])
def test_norm_rows_where_launches_change(hk, rows, cols):
    _norm_case(hk, rows, cols, (BF16, F32)[cols // 8 % 2], (BF16, F32)[rows % 2], residual=False, bias=rows % 2 == 0)


@pytest.mark.parametrize("cols", [64, 1000, 4096, 10000])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_norm_stream_in_place(hk, cols, dtype):
    """The new stream over x, and over the residual, with more rows than workgroups."""
    x, w, b, gen = _norm_inputs(1500, cols, dtype, dtype, 8)
    res = _randn(gen, 1500, cols).to(dtype)
    y, r, stats = hk.layer_norm_forward(x, w, b, res)
    for which in (0, 1):
        t = [x.clone(), res.clone()]
        y1, r1, stats1 = hk.layer_norm_forward(t[0], w, b, t[1], residual_out=t[which])
        assert r1 is t[which] and torch.equal(r1, r) and torch.equal(y1, y) and torch.equal(stats1, stats)
        assert torch.equal(t[1 - which], (x, res)[1 - which])


def test_norm_far_from_zero(hk):
    """A mean of 2^12 times the spread (the stream is what it is rounded to): the bits of r - mean stay."""
    for cols in (128, 1000, 4096):
        _norm_case(hk, 37, cols, F32, F32, residual=False, centre=4096.0)


def test_norm_constant_rows(hk):
    """Rows of one value, zeros among them, are the bias, whatever eps is; their gradients are finite."""
    for cols in (128, 2048):
        x = torch.tensor([0.0, 1.0, -3.5, 1e30], device="cuda")[:, None].expand(4, cols).contiguous()
        w, b = torch.rand(cols, device="cuda"), torch.rand(cols, device="cuda")
        for eps in (1e-5, 1e-300):
            y, r, stats = hk.layer_norm_forward(x, w, b, eps=eps)
            assert torch.equal(y, b.expand(4, cols))
        y, r, stats = hk.layer_norm_forward(x, w, b)
        dx, dw, db = hk.layer_norm_backward(torch.ones_like(x), r, w, stats)
        assert bool(torch.isfinite(dx).all()) and not bool(dw.any()) and bool((db == 4).all())


def test_norm_large_and_not_finite(hk):
    """Squares past fp32 are no trouble; a NaN or an infinity stays in its own row, and in the
    weight's gradients."""
    for cols in (256, 4096):
        x, w, b, gen = _norm_inputs(6, cols, F32, F32, 3)
        x[1] *= 1e25
        x[2, 7], x[3, 9] = math.nan, math.inf
        y, r, stats = hk.layer_norm_forward(x, w, b)
        fine = torch.tensor([0, 1, 4, 5], device="cuda")
        want, m, rstd = ref.layer_norm(x.double()[fine], w.double(), b.double(), 1e-5)
        _check(y[fine], want, ref.layer_norm_bound(want, x.double()[fine], w.double(), m, rstd, F32))
        assert bool(torch.isnan(y[2]).all()) and bool(torch.isnan(y[3]).any())
        dy = _randn(gen, 6, cols)
        dx, dw, db = hk.layer_norm_backward(dy, r, w, stats)
        d4 = dy.double()[fine]
        args = (d4, x.double()[fine], w.double(), 1e-5, None)
        _check(dx[fine], ref.layer_norm_grad(*args)[0], ref.layer_norm_grad_bound(*args, F32, F32, 20)[0])


def test_norm_no_rows(hk):
    x, w = torch.empty((0, 256), device="cuda", dtype=BF16), torch.ones(256, device="cuda")
    y, r, stats = hk.layer_norm_forward(x, w, w, x.clone())
    assert y.shape == r.shape == (0, 256) and stats.shape == (0, 4)
    dx, dw, db = hk.layer_norm_backward(x, r, w, stats)
    assert dx.shape == (0, 256) and not bool(dw.any()) and not bool(db.any())


def test_norm_gradient_in_place(hk):
    """dx over dr, as the C entry point allows; over dy and r, which others still read, it is refused."""
    for rows in (300, 3000):
        for cols in (256, 4096, 9000):
            x, w, b, gen = _norm_inputs(rows, cols, BF16, BF16, 5)
            y, r, stats = hk.layer_norm_forward(x, w, b)
            dy, dr = _randn(gen, rows, cols).to(BF16), _randn(gen, rows, cols).to(BF16)
            want = hk.layer_norm_backward(dy, r, w, stats, dr=dr)
            need = hk.tk_kernel.layer_norm_backward_workspace_size(rows, cols)
            dw, db, ws = torch.empty_like(w), torch.empty_like(w), torch.empty(need, dtype=torch.uint8, device="cuda")
            dx = dr.clone()
            hk.tk_kernel.dispatch_layer_norm_backward(dy, r, w, dx, stats, dx, dw, db, ws)
            assert torch.equal(dx, want[0]) and torch.equal(dw, want[1]) and torch.equal(db, want[2])
            for bad in (dy, r):
                with pytest.raises(RuntimeError, match="neither dy nor r"):
                    hk.tk_kernel.dispatch_layer_norm_backward(dy, r, w, dr, stats, bad, dw, db, ws)


def test_norm_far_rows(hk):
    """Offsets past 2^31 values, more rows than workgroups: the last rows are those of a short call."""
    for rows, cols in (((1 << 31) // 2048 + 70, 2048), ((1 << 24), 128)):
        x = torch.zeros((rows, cols), dtype=BF16, device="cuda")
        x[-64:] = torch.randn((64, cols), device="cuda").to(BF16)
        w = torch.rand(cols, device="cuda")
        y, r, stats = hk.layer_norm_forward(x, w)
        y1, r1, stats1 = hk.layer_norm_forward(x[-64:], w)
        assert torch.equal(y[-64:], y1) and torch.equal(stats[-64:], stats1)
        del y
        dx, dw, _ = hk.layer_norm_backward(x, r, w, stats)
        dx1, dw1, _ = hk.layer_norm_backward(x[-64:], r1, w, stats1)
        assert torch.equal(dx[-64:], dx1)
        # the other rows add zeros; only the order of the sums differs
        n = (x[-64:].double() - x[-64:].double().mean(1, keepdim=True)) * stats1[:, 2:3].double()
        assert bool(((dw - dw1).abs() <= 2 * 100 * ref.U * (x[-64:].double() * n).abs().sum(0)).all())
        del x, r, dx


def test_norm_refusals(hk):
    x = torch.zeros((4, 64), device="cuda", dtype=BF16)
    w = torch.ones(64, device="cuda")
    for args, says in (((x[0], w), r"must be \[R, C\]"), ((x, w[:32]), "weight must be"), ((x.half(), w), "bfloat16 or float32"),
                       ((x, w, w.to(BF16)), "bias must have"), ((x, w, None, x.float()), "residual must have"),
                       ((x, w, None, x[:2]), "residual must have"), ((x.cpu(), w), "GPU"), ((x[:, :32], w[:32]), "contiguous"),
                       ((x[:, :60].contiguous(), w[:60]), "multiple of 8")):
        with pytest.raises(RuntimeError, match=says):
            hk.layer_norm_forward(*args)
    for eps in (0.0, -1.0, math.nan):
        with pytest.raises(RuntimeError, match="eps"):
            hk.layer_norm_forward(x, w, eps=eps)
    with pytest.raises(RuntimeError, match="16384"):
        hk.layer_norm_forward(torch.zeros((1, 16392), device="cuda"), torch.zeros(16392, device="cuda"))
    with pytest.raises(RuntimeError, match="needs a residual"):
        hk.layer_norm_forward(x, w, residual_out=x)
    y, r, stats = hk.layer_norm_forward(x, w)
    for args, says in (((x.float(), r, w, stats), "dy must have"), ((x, r, w, stats[:3]), "stats must be"),
                       ((x, r, w, stats, x[:3]), "dr must have"), ((x, r, w[:32], stats), "weight must be")):
        with pytest.raises(RuntimeError, match=says):
            hk.layer_norm_backward(*args)


# ---------------------------------------------------------------------------
# tokens by expert and back
# ---------------------------------------------------------------------------
def _ids(gen, t, k, experts, away):
    """Ids with popular and rare experts; a part ``away``: -1, E, and other values outside."""
    p = torch.rand(experts, generator=gen, device="cuda") ** 3 + 1e-3
    ids = torch.multinomial(p, t * k, replacement=True, generator=gen).to(torch.int32).view(t, k)
    if away:
        out = torch.tensor([-1, experts, experts + 1, -(2 ** 31), 2 ** 31 - 1], dtype=torch.int32, device="cuda")
        pick = out[torch.randint(0, 5, (t, k), generator=gen, device="cuda")]
        ids = torch.where(torch.rand((t, k), generator=gen, device="cuda") < away, pick, ids)
    return ids


def _permute_case(hk, t, k, experts, hidden, dtype, away, seed=0):
    gen = _gen(t * 7 + k + experts + hidden + seed)
    ids = _ids(gen, t, k, experts, away)
    offsets, perm, inv = (v.cuda() for v in ref.order(ids.cpu(), experts))
    here = ref.in_use(ids, experts)
    x = _randn(gen, t, hidden).to(dtype)
    xp, order = hk.moe_permute(x, ids, experts)
    torch.cuda.synchronize()
    assert torch.equal(order.offsets, offsets) and torch.equal(order.perm, perm) and torch.equal(order.inv_perm, inv)
    bits = xp.view(torch.uint8) if dtype == F8 else xp
    rows = (x.view(torch.uint8) if dtype == F8 else x)[(perm // k).long()]
    rows[int(offsets[-1]):] = 0
    assert torch.equal(bits, rows)
    if dtype == F8:
        return
    # rows behind the last expert's are never read
    n = int(offsets[-1])
    dxp = _randn(gen, t * k, hidden).to(dtype)
    dxp[n:] = math.nan
    _check(hk.moe_permute_backward(dxp, order), ref.combine(dxp, None, inv, here), ref.combine_bound(dxp, None, inv, here, dtype), "dx")
    y = _randn(gen, t * k, hidden).to(dtype)
    y[n:] = math.inf
    w = torch.softmax(2 * _randn(gen, t, k), 1)
    w[~here] = math.nan
    clean = torch.where(here, w, torch.zeros_like(w))
    _check(hk.moe_combine(y, w, order), ref.combine(y, clean, inv, here), ref.combine_bound(y, clean, inv, here, dtype), "out")
    dout = _randn(gen, t, hidden).to(dtype)
    dy, dw = hk.moe_combine_backward(dout, y, w, order)
    want_y, want_w = ref.combine_grad(dout, y, clean, inv, here)
    _check(dy, want_y, (ref.U + ref.half(dtype)) * 1.01 * want_y.abs() + 2.0 ** -133, "dy")
    _check(dw, want_w, ref.combine_grad_bound(dout, y, inv, here), "dw")


@pytest.mark.parametrize("t,k,experts,hidden", [
    (1, 1, 1, 8), (1, 8, 128, 4096), (3, 2, 5, 520), (64, 8, 128, 256), (255, 8, 256, 64), (256, 8, 60, 64), (257, 8, 60, 72),
    (2048, 1, 1024, 16), (2049, 1, 1024, 16), (2048, 2, 1000, 16), (2049, 2, 1000, 16), (724, 8, 40, 24), (725, 8, 40, 24), (500, 6, 1, 128), (40, 32, 1024, 4104), (700, 32, 33, 32), (5000, 5, 7, 24),
    (33000, 8, 255, 16), (50, 3, 2, 9000)])
@pytest.mark.parametrize("away", [0.0, 0.4])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_permute(hk, t, k, experts, hidden, away, dtype):
    _permute_case(hk, t, k, experts, hidden, dtype, away)


@pytest.mark.parametrize("t,k", [(5, 3), (3000, 4)])
def test_permute_bytes(hk, t, k):
    _permute_case(hk, t, k, 40, 272, F8, 0.2)


@pytest.mark.parametrize("t,k", [(7, 4), (3000, 4)])
def test_permute_nothing_here(hk, t, k):
    """No slot has an expert here: zeros everywhere, and no row is read back."""
    _permute_case(hk, t, k, 16, 64, BF16, 1.1)


@pytest.mark.parametrize("t,k", [(7, 4), (3000, 4)])
def test_permute_one_expert(hk, t, k):
    """Every slot at one expert, the same twice in a row: their own order."""
    ids = torch.full((t, k), 3, dtype=torch.int32, device="cuda")
    x = torch.randn((t, 64), device="cuda")
    xp, order = hk.moe_permute(x, ids, 9)
    assert torch.equal(order.perm, torch.arange(t * k, dtype=torch.int32, device="cuda"))
    assert order.offsets.tolist() == [0] * 4 + [t * k] * 6 and torch.equal(xp, x.repeat_interleave(k, 0))


def test_permute_many_slots(hk):
    """More slots than the sorting workgroups take at a time, and more tokens than workgroups."""
    t, k, experts = (1 << 20) + 77, 2, 300
    gen = _gen(1)
    ids = _ids(gen, t, k, experts, 0.1)
    x = _randn(gen, t, 8)
    xp, order = hk.moe_permute(x, ids, experts)
    key = torch.where(ref.in_use(ids, experts), ids, torch.full_like(ids, experts)).flatten()
    by, perm = key.sort(stable=True)
    assert torch.equal(order.perm.long(), perm)
    assert torch.equal(order.offsets.long(), torch.searchsorted(by, torch.arange(experts + 1, device="cuda", dtype=torch.int32)))
    n = int(order.offsets[-1])
    assert torch.equal(xp[:n], x[perm[:n] // k]) and not bool(xp[n:].any())
    here = ref.in_use(ids, experts)
    y, dout, w = _randn(gen, t * k, 8), _randn(gen, t, 8), torch.rand((t, k), generator=gen, device="cuda")
    _check(hk.moe_combine(y, w, order), ref.combine(y, w, order.inv_perm, here), ref.combine_bound(y, w, order.inv_perm, here, F32))
    dy, dw = hk.moe_combine_backward(dout, y, w, order)
    want_y, want_w = ref.combine_grad(dout, y, w, order.inv_perm, here)
    _check(dy, want_y, 2 * ref.U * want_y.abs())
    _check(dw, want_w, ref.combine_grad_bound(dout, y, order.inv_perm, here))


def test_permute_far_rows(hk):
    """Places past 2^32 bytes."""
    t, k, hidden = 40000, 4, 16384
    x = torch.randn((t, hidden), device="cuda").to(BF16)
    ids = torch.randint(0, 8, (t, k), dtype=torch.int32, device="cuda")
    xp, order = hk.moe_permute(x, ids, 8)
    for p in torch.randint(0, t * k, (20,)).tolist() + [0, t * k - 1]:
        assert torch.equal(xp[p], x[int(order.perm[p]) // k])
    out = hk.moe_combine(xp, torch.full((t, k), 0.25, device="cuda"), order)
    assert torch.equal(out, x)
    del out
    dy, dw = hk.moe_combine_backward(x, xp, torch.full((t, k), 0.5, device="cuda"), order)
    for p in torch.randint(0, t * k, (20,)).tolist() + [t * k - 1]:
        assert torch.equal(dy[p], x[int(order.perm[p]) // k] * 0.5)


def test_permute_no_tokens(hk):
    x, ids = torch.empty((0, 64), device="cuda"), torch.empty((0, 2), dtype=torch.int32, device="cuda")
    xp, order = hk.moe_permute(x, ids, 5)
    assert xp.shape == (0, 64) and order.offsets.tolist() == [0] * 6
    assert hk.moe_permute_backward(xp, order).shape == (0, 64)
    w = torch.empty((0, 2), device="cuda")
    assert hk.moe_combine(xp, w, order).shape == (0, 64)
    dy, dw = hk.moe_combine_backward(x, xp, w, order)
    assert dy.shape == (0, 64) and dw.shape == (0, 2)


def test_order_of_another_batch_stays_inside(hk):
    """Places outside the buffers are skipped, not followed."""
    t, k = 20, 3
    x = torch.randn((t, 64), device="cuda")
    _, order = hk.moe_permute(x, torch.zeros((t, k), dtype=torch.int32, device="cuda"), 2)
    wild = order._replace(inv_perm=torch.full((t, k), 2 ** 30, dtype=torch.int32, device="cuda"))
    below = order._replace(inv_perm=torch.full((t, k), -5, dtype=torch.int32, device="cuda"))
    high = order._replace(offsets=torch.full((3,), 2 ** 30, dtype=torch.int32, device="cuda"))
    y, w = torch.randn((t * k, 64), device="cuda"), torch.rand((t, k), device="cuda")
    for o in (wild, below):
        assert not bool(hk.moe_combine(y, w, o).any())
        dy, dw = hk.moe_combine_backward(x, y, w, o)
        assert not bool(dw.any())
    here = torch.ones((t, k), dtype=torch.bool, device="cuda")
    _check(hk.moe_combine(y, w, high), ref.combine(y, w, order.inv_perm, here), ref.combine_bound(y, w, order.inv_perm, here, F32))


def test_permute_refusals(hk):
    x = torch.zeros((4, 64), device="cuda")
    ids = torch.zeros((4, 2), dtype=torch.int32, device="cuda")
    for args, says in (((x, ids[:3], 2), "ids"), ((x, ids.long(), 2), "int32"), ((x, ids, 0), "positive"), ((x, ids, 1025), "1024"),
                       ((x.half(), ids, 2), "bfloat16 or float32"), ((x.cpu(), ids, 2), "GPU"),
                       ((x, torch.zeros((4, 33), dtype=torch.int32, device="cuda"), 2), "k=33"),
                       ((x[:, :60].contiguous(), ids, 2), "multiple of 8"), ((x[:, :8].contiguous().to(F8), ids, 2), "multiple of 16"),
                       ((x[:, :32], ids, 2), "contiguous"), ((x[0], ids, 2), r"\[T, H\]")):
        with pytest.raises(RuntimeError, match=says):
            hk.moe_permute(*args)
    xp, order = hk.moe_permute(x, ids, 2)
    w = torch.ones((4, 2), device="cuda")
    for args, says in (((xp[:7], w, order), "y: expected"), ((xp, w[:3], order), "topk_w: expected"),
                       ((xp, w.double(), order), "topk_w: expected"), ((xp.half(), w, order), "bfloat16 or float32")):
        with pytest.raises(RuntimeError, match=says):
            hk.moe_combine(*args)
    with pytest.raises(RuntimeError, match="dout: expected"):
        hk.moe_combine_backward(x.to(BF16), xp, w, order)


# ---------------------------------------------------------------------------
# the router's choice
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("t,experts,k", [(1, 1, 1), (1, 128, 8), (5, 60, 6), (63, 64, 2), (64, 65, 32), (1000, 256, 8), (33, 1024, 32)])
def test_route(hk, t, experts, k):
    gen = _gen(t + experts + k)
    logits = 3 * _randn(gen, t, experts)
    idx, w = hk.route_topk(logits, k)
    want_idx, want_w = ref.route(logits, k)
    assert torch.equal(idx, want_idx)
    # expf to 2 ulp of arguments that are half a step of up to 30 off, a sum of k, a quotient
    _check(w, want_w, (64 + k) * ref.U * want_w)
    dw = _randn(gen, t, k)
    _check(hk.route_topk_backward(dw, w, idx, experts), ref.route_grad(dw, w, idx, experts), ref.route_grad_bound(dw, w, idx, experts))


def test_route_gradient_of_any_indexes(hk):
    """An expert in several slots adds up; indexes outside are skipped."""
    idx = torch.tensor([[3, 3, 1], [-1, 70, 64], [2 ** 31 - 1, 0, -(2 ** 31)]], dtype=torch.int32, device="cuda")
    dw, w = torch.randn((3, 3), device="cuda"), torch.rand((3, 3), device="cuda")
    for experts in (65, 71):
        _check(hk.route_topk_backward(dw, w, idx, experts), ref.route_grad(dw, w, idx, experts),
               ref.route_grad_bound(dw, w, idx, experts))


def test_route_refusals(hk):
    logits = torch.zeros((4, 8), device="cuda")
    idx, w = hk.route_topk(logits, 2)
    with pytest.raises(RuntimeError, match="dw: expected"):
        hk.route_topk_backward(w[:3], w, idx, 8)
    with pytest.raises(RuntimeError, match="E=1 outside"):
        hk.route_topk_backward(w, w, idx, 1)
    with pytest.raises(RuntimeError):
        hk.route_topk(logits, 9)
    with pytest.raises(RuntimeError, match=r"\[T, E\]"):
        hk.route_topk(logits[0], 1)
    e = hk.route_topk(torch.empty((0, 8), device="cuda"), 2)
    assert e[0].shape == (0, 2) and hk.route_topk_backward(e[1], e[1], e[0], 8).shape == (0, 8)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
class Block:
    """A mixture-of-experts block in plain products with these operators around them."""

    def __init__(self, hidden, inter, experts, k, dtype, seed=0):
        gen = _gen(seed)
        p = lambda *s: (_randn(gen, *s) * s[-1] ** -0.5).to(dtype)  # noqa: E731
        self.k, self.experts = k, experts
        self.norm_w, self.norm_b = (1 + 0.1 * _randn(gen, hidden)).to(dtype), (0.1 * _randn(gen, hidden)).to(dtype)
        self.router, self.w1, self.w2 = p(experts, hidden).float(), p(experts, inter, hidden), p(experts, hidden, inter)

    def params(self):
        return [self.norm_w, self.norm_b, self.router, self.w1, self.w2]

    def experts_of(self, xp, offsets):
        rows, at = [], offsets.tolist()
        for e in range(self.experts):
            h = torch.tanh(xp[at[e]:at[e + 1]] @ self.w1[e].T)
            rows.append(h @ self.w2[e].T)
        rows.append(xp[at[-1]:] * 0)
        return torch.cat(rows)

    def __call__(self, hk, x, stream):
        n, r = hk.layer_norm(x, self.norm_w, self.norm_b, stream)
        idx, w = hk.route_topk(n.float() @ self.router.T, self.k)
        xp, order = hk.moe_permute(n, torch.where(idx == 1, torch.full_like(idx, -1), idx), self.experts)  # expert 1 is elsewhere
        return hk.moe_combine(self.experts_of(xp, order.offsets), w, order), r

    def plain(self, x, stream):
        """The same in torch's own 64-bit operations, dense over the experts."""
        nw, nb, router, w1, w2 = self.params()
        r = x + stream
        n = ref.layer_norm(r, nw, nb, 1e-5)[0]
        top, idx = (n @ router.T).topk(self.k, 1)
        w = torch.softmax(top, 1)
        out = 0
        for e in range(self.experts):
            if e != 1:
                out = out + (w * (idx == e)).sum(1, keepdim=True) * (torch.tanh(n @ w1[e].T) @ w2[e].T)
        return out, r


def test_block_gradients(hk):
    """Forward and backward of the whole block through the recorded gradients, against 64 bits.  fp32
    products of K terms are off by K u of their magnitudes; the chain of five of them (K 64 and less)
    stays far below 1e-4 of the gradients' norms."""
    t, hidden = 130, 64
    b = Block(hidden, 48, 10, 3, F32)
    gen = _gen(7)
    x, s = _randn(gen, t, hidden), _randn(gen, t, hidden)
    dout, dr = _randn(gen, t, hidden), _randn(gen, t, hidden)
    leaves = [v.requires_grad_() for v in (x, s, *b.params())]
    out, r = b(hk, x, s)
    grads = torch.autograd.grad((out, r), leaves, (dout, dr))
    b64 = Block(hidden, 48, 10, 3, F32)
    for name in ("norm_w", "norm_b", "router", "w1", "w2"):
        setattr(b64, name, getattr(b, name).detach().double().requires_grad_())
    x64, s64 = x.detach().double().requires_grad_(), s.detach().double().requires_grad_()
    out64, r64 = b64.plain(x64, s64)
    want = torch.autograd.grad((out64, r64), [x64, s64, *b64.params()], (dout.double(), dr.double()))
    for got, v in zip((out, r, *grads), (out64, r64, *want)):
        assert float((got.detach().double() - v).norm() / v.norm()) < 1e-4


class _Undefined(torch.autograd.Function):
    """Passes a value on and no gradient back."""

    @staticmethod
    def forward(ctx, t):
        return t.clone()

    @staticmethod
    def backward(ctx, _):
        return None


def test_gradients_only_where_asked(hk):
    """Frozen inputs get none; without a graph nothing is recorded; dbias without a bias is none; a
    broadcast or strided output gradient is taken as it is."""
    x = torch.randn((6, 64), device="cuda")
    w = torch.rand(64, device="cuda", requires_grad=True)
    y, r = hk.layer_norm(x, w)
    assert r is x and y.requires_grad
    y.sum().backward()  # an expanded gradient
    n = ref.layer_norm(x.double(), torch.ones(64, device="cuda").double(), None, 1e-5)[0]
    _check(w.grad, n.sum(0), 60 * ref.U * n.abs().sum(0))
    with torch.no_grad():
        assert not hk.layer_norm(x, w)[0].requires_grad
    y, r = hk.layer_norm(x, w, residual=x)
    (g,) = torch.autograd.grad(r.sum() + y[:, ::2].sum(), [w])  # r's own gradient does not reach w
    sel = torch.zeros(64, device="cuda", dtype=torch.float64)
    sel[::2] = 1
    n = ref.layer_norm(r.double(), torch.ones(64, device="cuda").double(), None, 1e-5)[0] * sel
    _check(g, n.sum(0), 60 * ref.U * n.abs().sum(0))
    xr = x.clone().requires_grad_()
    y, r = hk.layer_norm(xr, w, residual=x)  # the norm, and then the stream, without a use
    gx, gw = torch.autograd.grad(r.sum(), [xr, w], allow_unused=True, retain_graph=True)
    assert bool((gx == 1).all()) and gw is None
    gx, _ = torch.autograd.grad((y * y).sum(), [xr, w])
    y2, r2, stats2 = hk.layer_norm_forward(x, w.detach(), None, x)
    assert torch.equal(gx, hk.layer_norm_backward(2 * y2, r2, w.detach(), stats2)[0])
    ids = torch.zeros((6, 2), device="cuda", dtype=torch.int32)
    logits = torch.randn((6, 9), device="cuda", requires_grad=True)
    xs = x.clone().requires_grad_()
    for leaf, out in ((xs, hk.moe_permute(xs, ids, 9)[0]), (logits, hk.route_topk(logits, 2)[1])):
        assert torch.autograd.grad(_Undefined.apply(out).sum(), leaf, allow_unused=True) == (None,)
    idx, tw = hk.route_topk(torch.randn((6, 9), device="cuda", requires_grad=True), 2)
    assert tw.requires_grad and not idx.requires_grad
    xp, order = hk.moe_permute(x, idx, 9)
    assert not xp.requires_grad
    out = hk.moe_combine(xp, tw, order)
    assert out.requires_grad


def _step(hk, b, x, s, dout, dr, w_all):
    """The block's operators forward and backward by their plain calls, without the experts."""
    y, r, stats = hk.layer_norm_forward(x, b.norm_w, b.norm_b, s)
    idx, w = hk.route_topk_forward(w_all, b.k)
    xp, order = hk.moe_permute_forward(y, idx, b.experts)
    out = hk.moe_combine_forward(xp, w, order)
    dxp, dw = hk.moe_combine_backward(dout, xp, w, order)
    dlogits = hk.route_topk_backward(dw, w, idx, b.experts)
    dx, dnw, dnb = hk.layer_norm_backward(hk.moe_permute_backward(dxp, order), r, b.norm_w, stats, dr=dr)
    return out, dlogits, dx, dnw, dnb


@pytest.mark.parametrize("t", [50, 2500])
def test_step_captured(hk, t):
    """Two captured steps that share no workspace, replayed with changing inputs between eager work."""
    b = Block(256, 32, 24, 4, BF16)
    gen = _gen(3)
    new = lambda: [_randn(gen, t, 256).to(BF16) for _ in range(4)] + [_randn(gen, t, 24)]  # noqa: E731
    sets = [new(), new()]
    for a in sets:
        _step(hk, b, *a)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for a in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_step(hk, b, *a))
        graphs.append(g)
    for i in range(4):
        for a in sets:
            for v, n in zip(a, new()):
                v.copy_(n)
        for g in graphs:
            g.replay()
        for a, o in zip(sets, outs):
            for got, want in zip(o, _step(hk, b, *a)):
                assert torch.equal(got, want), i
        torch.cuda.synchronize()


def test_step_on_streams(hk):
    """Steps that overlap on two streams give the bits of one alone."""
    b = Block(512, 32, 24, 4, BF16)
    gen = _gen(4)
    sets = [[_randn(gen, t, 512).to(BF16) for _ in range(4)] + [_randn(gen, t, 24)] for t in (3000, 70)]
    want = [_step(hk, b, *a) for a in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(6):
        for s, a, w in zip(streams, sets, want):
            with torch.cuda.stream(s):
                got.append((_step(hk, b, *a), w))
    torch.cuda.synchronize()
    for g, w in got:
        assert all(torch.equal(u, v) for u, v in zip(g, w))


def test_dense_half_of_a_block(hk):
    """Layer norm, both halves of a dense feed-forward with its epilogues, in place on the stream: the
    operands are what the quantiser made, so the formulas are those of the dequantised values."""
    t, hidden, inter = 77, 512, 1024
    gen = _gen(6)
    x = _randn(gen, t, hidden)
    w1, w2 = _randn(gen, inter, hidden) * hidden ** -0.5, _randn(gen, hidden, inter) * inter ** -0.5
    b1, b2 = _randn(gen, inter), _randn(gen, hidden)
    nw, nb = 1 + 0.1 * _randn(gen, hidden), 0.1 * _randn(gen, hidden)
    q1, s1 = hk.quant_tensor(w1)
    q2, s2 = hk.quant_tensor(w2)
    n, r = hk.layer_norm(x, nw, nb)
    a, sa = hk.quant_tensor(n)
    h = hk.gemm_fp8(a, q1, sa, s1, bias=b1, activation="gelu", out_dtype=F32)
    c, sc = hk.quant_tensor(h)
    stream = r.clone()
    hk.gemm_fp8(c, q2, sc, s2, bias=b2, residual=stream, out=stream)
    d = torch.float64
    z = (a.to(d) @ q1.to(d).T) * (sa.to(d) * s1.to(d)) + b1.to(d)
    want_h = z * ref.phi(z)
    want = (c.to(d) @ q2.to(d).T) * (sc.to(d) * s2.to(d)) + b2.to(d) + r.to(d)
    # sums of K products in fp32: K u (and a few operations) of the terms' magnitudes
    mag_h = (a.to(d).abs() @ q1.to(d).abs().T) * (sa.to(d) * s1.to(d)) + b1.to(d).abs()
    mag = (c.to(d).abs() @ q2.to(d).abs().T) * (sc.to(d) * s2.to(d)) + b2.to(d).abs() + r.to(d).abs()
    _check(h, want_h, 1.2 * (hidden + 64) * ref.U * mag_h)
    _check(stream, want, (inter + 64) * ref.U * mag)


def test_an_overwritten_stream_has_no_gradient(hk):
    """The norm's gradient reads the stream: after a product into it, or another norm's new stream, the backward
    pass raises; without one it runs."""
    aq, bq = torch.ones((4, 128), device="cuda").to(F8), torch.ones((256, 128), device="cuda").to(F8)
    w = torch.ones(256, device="cuda", dtype=BF16, requires_grad=True)
    x = torch.randn((4, 256), device="cuda").to(BF16)
    for write in (lambda r: hk.gemm_fp8(aq, bq, residual=r, out=r), lambda r: hk.gemm_fp8(aq, bq, out=r),
                  lambda r: hk.layer_norm_forward(x, w, residual=r, residual_out=r)):
        y, r = hk.layer_norm(x, w, residual=torch.randn_like(x))
        y.sum().backward(retain_graph=True)
        with torch.no_grad():
            write(r)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gradients_at_odd_addresses(hk, dtype):
    """A gradient that autograd hands back as a slice at an odd address: the same bits as from an aligned one."""
    gen = _gen(17)
    t, h, k, e = 6, 264, 2, 4
    leaf = lambda *s: _randn(gen, *s).to(dtype).requires_grad_()  # noqa: E731
    x, s, w, b, y = leaf(t, h), leaf(t, h), leaf(h), leaf(h), leaf(t * k, h)
    tw = torch.rand((t, k), generator=gen, device="cuda").requires_grad_()
    ids = torch.randint(-1, e, (t, k), generator=gen, device="cuda", dtype=torch.int32)
    weights = _randn(gen, 4 * t * k * h + 1).to(dtype)

    def gradients(odd):
        n, r = hk.layer_norm(x, w, b, s)
        xp, order = hk.moe_permute(n, ids, e)
        flat = lambda v: torch.cat([torch.zeros(odd, device="cuda", dtype=dtype), v.reshape(-1)]) if odd else v.reshape(-1)  # noqa: E731
        loss = 0.0
        for v in (n, r, xp, hk.moe_combine(y, tw, order)):
            f = flat(v)
            loss = loss + (f.float() * weights[1 - odd:][: f.numel()].float()).sum()
        return torch.autograd.grad(loss, (x, s, w, b, y, tw))

    for got, want in zip(gradients(1), gradients(0)):
        assert torch.equal(got, want)
