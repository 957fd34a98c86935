"""The 8-bit linear layer against its definition in 64 bits.

Quantisation is defined exactly (nearest integer to 127 x / max, ties to even) and compared for equality.  The
product's sum is exact, so only the float32 epilogue rounds: the sum to float32, two products, one addition
(5 half-steps of 2^-24 on what they act on), then half a step of the result's type.  The gradients sum float32 terms: at
most one step 2^-23 for each addition of the terms' magnitudes, and where every term is an integer below 2^24 the
result must be equal."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0 ** -24


def _half(dt):
    return torch.finfo(dt).eps / 2


def _floor(dt):
    """Half the spacing of dt's subnormal numbers: what a rounding can be off near zero."""
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps


def quantised(x):
    """(q, scale) of rows in 64 bits on the CPU; scale rounded to float32 as it is stored."""
    xd = x.detach().cpu().double()
    a = xd.abs().amax(-1, keepdim=True)
    q = torch.where(a > 0, torch.round(127 * xd / torch.where(a > 0, a, 1.0)), 0.0)
    return q, (a.float() / 127).squeeze(-1)


def _product_close(y, qa, sa, qb, sb, bias, dt):
    prod = (qa.double() @ qb.double().t()) * sa.double()[:, None] * sb.double()
    want = prod + (bias.detach().cpu().double() if bias is not None else 0.0)
    tol = 4 * U * prod.abs() + U * want.abs() + _half(dt) * want.abs() * (1 + 2 ** -8) + _floor(dt) + 2.0 ** -126
    err = (y.detach().cpu().double() - want).abs()
    assert y.dtype == dt and (err <= tol).all(), "max error %g of its bound" % (err / tol).max()


def _close_or_over(y, prod, want, dt):
    """_product_close's bound on the device; what half a step of the type beyond its largest number reaches is rounded to
    infinity."""
    tol = 4 * U * prod.abs() + U * want.abs() + _half(dt) * want.abs() * (1 + 2 ** -8) + _floor(dt) + 2.0 ** -126
    limit = torch.finfo(dt).max * (1 + _half(dt) / 2)
    over = want.abs() - tol >= limit
    assert torch.equal(y[over].double(), want[over].sign() * torch.inf)
    assert (((y.double() - want).abs() <= tol) | (want.abs() + tol >= limit)).all()


# ---- rows to 8 bits ------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 7), (5, 64), (17, 1000), (4, 4096), (2, 4099), (3, 8192), (2, 16384),
                                    (2, 16392), (1, 40001)])
def test_quantize_rows_is_exact(dt, rows, k):
    import sc_functional as F
    print("quantize", dt, rows, k, flush=True)
    g = torch.Generator().manual_seed(rows * 1000 + k)
    x = torch.randn(rows, k, generator=g).to(dt)
    if rows > 2:
        x[1] = 0
    q, s = F.quantize_rows(x.cuda())
    qe, se = quantised(x)
    assert q.dtype == torch.int8 and q.shape == x.shape and s.shape == (rows,)
    assert torch.equal(q.cpu().double(), qe) and torch.equal(s.cpu(), se)
    assert q.stride(0) % 128 == 0
    pad = q.as_strided((rows, q.stride(0)), (q.stride(0), 1))[:, k:]
    assert not pad.any(), "the rows' padding is not zero"


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("k", [4, 8, 31, 255, 256, 257, 264, 520, 1101, 1536, 1537, 1544, 2001, 3060, 3080, 4098, 5001, 6144, 6145,
                               6152, 8193, 9001, 12288, 12289, 12296, 16383])
def test_quantize_rows_around_the_numbers_of_threads(dt, k):
    """Also of a matrix inside another one: rows that begin anywhere, beside elements that must not be read as theirs."""
    import sc_functional as F
    print("quantize", dt, k, flush=True)
    g = torch.Generator().manual_seed(k)
    whole = torch.randn(19, k + 11, generator=g).to(dt)
    whole[:, :3] = 1e4
    whole[:, k + 3:] = -1e4
    gpu = whole.cuda()
    for x, y in ((whole[:, 3:k + 3], gpu[:, 3:k + 3]), (whole[:, 8:].contiguous(), gpu[:, 8:].contiguous())):
        q, s = F.quantize_rows(y)
        qe, se = quantised(x)
        assert torch.equal(q.cpu().double(), qe) and torch.equal(s.cpu(), se)
        pad = q.as_strided((19, q.stride(0)), (q.stride(0), 1))[:, y.shape[1]:]
        assert not pad.any(), "the rows' padding is not zero"


def test_quantize_rows_ties_and_extremes():
    import sc_functional as F
    # max 127: 127 x / max = x, so every half-integer is a tie
    x = torch.arange(-253, 255, 2, dtype=torch.float32)[None] / 2
    x = torch.cat([x, torch.tensor([[127.0]])], 1)
    for scale in (1.0, 2.0 ** 100, 2.0 ** -140, 2.0 ** -100, 2.0 ** 120):
        v = (x.double() * scale).float()
        q, s = F.quantize_rows(v.cuda())
        qe, se = quantised(v)
        assert torch.equal(q.cpu().double(), qe) and torch.equal(s.cpu(), se), scale
    # one step of float32 beside a tie
    for m in (1.0, 1.3, 0.7531, 3.1e-38, 2.9e38):
        a = torch.tensor(m).float()
        half = (torch.arange(-126, 127, dtype=torch.float64) + 0.5) * a.double() / 127
        near = half.float()
        up, down = torch.nextafter(near, torch.tensor(float("inf"))), torch.nextafter(near, torch.tensor(float("-inf")))
        v = torch.cat([near, up, down, a[None]])[None]
        q, _ = F.quantize_rows(v.cuda())
        assert torch.equal(q.cpu().double(), quantised(v)[0]), m
    # bfloat16 patterns over a maximum whose mantissa makes exact ties
    v = torch.arange(0, 0x3F7F, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)[None]
    v = torch.cat([v, torch.tensor([[1.984375]], dtype=torch.bfloat16)], 1)
    q, _ = F.quantize_rows(v.cuda())
    assert torch.equal(q.cpu().double(), quantised(v)[0])


def test_quantize_rows_nan_inf_and_layouts():
    import sc_functional as F
    x = torch.randn(6, 300)
    x[1, 7], x[2, 299], x[3, 0] = float("nan"), float("inf"), float("-inf")
    q, s = F.quantize_rows(x.cuda())
    bad = torch.tensor([0, 1, 1, 1, 0, 0], dtype=torch.bool)
    assert torch.equal(s.cpu().isnan(), bad) and not q.cpu()[bad].any()
    assert torch.equal(q.cpu()[~bad].double(), quantised(x)[0][~bad])
    base = torch.randn(9, 411)
    for v in (base[::2], base[:, 3:200], base[1:, 1:2], base.t(), base[:, ::3], base.view(3, 3, 411), base[0],
              base.view(3, 3, 411)[:, 1], base[:0]):
        q, s = F.quantize_rows(v.cuda())  # .cuda() makes some dense: the strided ones are built on the device below
        assert q.shape == v.shape and s.shape == v.shape[:-1]
    dev = base.cuda()
    for name, v in (("rows", dev[::2]), ("columns", dev[:, 3:200]), ("one", dev[1:, 1:2]), ("t", dev.t()), ("step", dev[:, ::3]),
                    ("3d", dev.view(3, 3, 411)), ("3d slice", dev.view(3, 3, 411)[:, 1]), ("expanded", dev[:1].expand(5, 411))):
        q, s = F.quantize_rows(v)
        qe, se = quantised(v)
        assert torch.equal(q.cpu().double(), qe) and torch.equal(s.cpu(), se), name


# ---- the product ---------------------------------------------------------------------------------
SHAPES = [(1, 1, 1), (1, 10, 16), (2, 3, 5), (1, 257, 129), (5, 64, 64), (16, 16, 128), (17, 100, 127), (33, 129, 200),
          (64, 1000, 512), (65, 67, 1000), (100, 300, 77), (129, 255, 384), (200, 130, 2050), (257, 513, 640), (1, 512, 4099),
          (7, 1100, 4096), (300, 40, 3001)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matmul_int8(m, n, k):
    import sc_functional as F
    print("matmul_int8", m, n, k, flush=True)
    g = torch.Generator().manual_seed(m * 7 + n * 3 + k)
    qa = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int8)
    qb = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8)
    sa, sb = torch.rand(m, generator=g) + 0.01, torch.rand(n, generator=g) + 0.01
    bias = torch.randn(n, generator=g) * k
    for dt, b in ((torch.float32, None), (torch.float32, bias), (torch.bfloat16, bias.bfloat16()), (torch.float16, bias)):
        if dt == torch.float16:
            sa, sb = sa / k, sb / 128
        y = F.matmul_int8(qa.cuda(), sa.cuda(), qb.cuda(), sb.cuda(), None if b is None else b.cuda(), dt)
        _product_close(y, qa, sa, qb, sb, b, dt)


@pytest.mark.parametrize("m,n,k", [(4, 9, 131071), (70, 5, 100001)])
def test_longest_reduction_does_not_overflow(m, n, k):
    import sc_functional as F
    qa, qb = torch.full((m, k), -128, dtype=torch.int8), torch.full((n, k), -128, dtype=torch.int8)
    one = lambda c: torch.ones(c, device="cuda")
    y = F.matmul_int8(qa.cuda(), one(m), qb.cuda(), one(n))
    want = torch.tensor(float(16384 * k), dtype=torch.float64).float()  # one rounding: the sum to float32
    assert (y.cpu() == want).all()


@pytest.mark.parametrize("m", [1, 3, 20, 70, 150])
@pytest.mark.parametrize("k", [5, 100, 129, 1000])
def test_bytes_behind_a_row_do_not_matter(m, k):
    """Operands cut out of larger tensors: what lies behind a row's end, or behind the last row, is not taken in."""
    import sc_functional as F
    g = torch.Generator().manual_seed(m + k)
    n, wide = 37, -(-k // 16) * 16 + 48
    A = torch.randint(-128, 128, (m + 5, wide), generator=g, dtype=torch.int8).cuda()
    B = torch.randint(-128, 128, (n + 5, wide), generator=g, dtype=torch.int8).cuda()
    for off in (0, 16, 5):  # 5: not aligned, taken to an aligned copy
        a, b = A[2:2 + m, off:off + k], B[1:1 + n, off:off + k]
        sa, sb = torch.rand(m, generator=g), torch.rand(n, generator=g)
        y = F.matmul_int8(a, sa.cuda(), b, sb.cuda())
        _product_close(y, a.cpu(), sa, b.cpu(), sb, None, torch.float32)
    at = torch.randint(-128, 128, (k, m), generator=g, dtype=torch.int8).cuda().t()
    y = F.matmul_int8(at, sa.cuda(), b, sb.cuda())
    _product_close(y, at.cpu(), sa, b.cpu(), sb, None, torch.float32)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("m,n,k", [(1, 10, 4096), (1, 4096, 512), (2, 33, 17), (9, 40, 1000), (16, 70, 4099), (37, 515, 1025),
                                   (64, 1000, 512), (130, 65, 300), (1, 7, 131071)])
def test_linear_int8_serving(dt, m, n, k):
    import sc_functional as F
    print("linear_int8", dt, m, n, k, flush=True)
    g = torch.Generator().manual_seed(m + n + k)
    x = (torch.randn(m, k, generator=g) * 3).to(dt)
    x[:, ::61] *= 8
    if m > 2:
        x[m // 2] = 0
    w, bias = torch.randn(n, k, generator=g) * k ** -0.5, torch.randn(n, generator=g)
    wq, ws = F.quantize_rows(w.cuda())
    for b in (None, bias, bias.to(dt)):
        y = F.linear_int8(x.cuda(), wq, None if b is None else b.cuda(), weight_scale=ws)
        qx, sx = quantised(x)
        _product_close(y, qx, sx, wq.cpu(), ws.cpu(), b, dt)


def test_linear_int8_shapes_layouts_and_empties():
    import sc_functional as F
    w, b = torch.randn(30, 70).cuda(), torch.randn(30).cuda()
    wq, ws = F.quantize_rows(w)
    base = torch.randn(4, 6, 70, device="cuda")
    want = F.linear_int8(base, wq, b, weight_scale=ws)
    assert want.shape == (4, 6, 30)
    assert torch.equal(F.linear_int8(base.transpose(0, 1), wq, b, weight_scale=ws), want.transpose(0, 1))
    wide = torch.zeros(4, 6, 99, device="cuda")
    wide[..., 11:81] = base
    assert torch.equal(F.linear_int8(wide[..., 11:81], wq, b, weight_scale=ws), want)
    assert torch.equal(F.linear_int8(base[2, 3], wq, b, weight_scale=ws), want[2, 3])
    assert torch.equal(F.linear_int8(base[::2, 1::2], wq, b, weight_scale=ws), want[::2, 1::2])
    assert torch.equal(F.linear_int8(base[:1, :1].expand(3, 2, 70), wq, b, weight_scale=ws), want[:1, :1].expand(3, 2, 30))
    assert F.linear_int8(base[:0], wq, b, weight_scale=ws).shape == (0, 6, 30)
    assert F.linear_int8(base, wq[:0], None, weight_scale=ws[:0]).shape == (4, 6, 0)
    assert torch.equal(F.linear_int8(base, w, b), want)
    # a row with a NaN gives a row of NaN and leaves the others alone
    bad = base.clone()
    bad[1, 2, 5] = float("nan")
    y = F.linear_int8(bad, wq, b, weight_scale=ws)
    assert y[1, 2].isnan().all()
    y[1, 2] = want[1, 2]
    assert torch.equal(y, want)


# ---- gradients -----------------------------------------------------------------------------------
GRADS = [(1, 1, 1), (1, 10, 16), (5, 3, 7), (64, 64, 64), (70, 33, 129), (129, 200, 66), (300, 17, 500), (256, 10, 1024)]


@pytest.mark.parametrize("m,n,k", GRADS)
@pytest.mark.parametrize("dt", DTYPES)
def test_gradients_of_integers_are_exact(dt, m, n, k):
    """Integer gradients and rows whose scale is a power of two (largest value 127): every term is an integer multiple
    of that power and the sums stay below 2^24, so float32 results have no rounding at all."""
    import sc_functional as F
    print("exact gradients", dt, m, n, k, flush=True)
    g = torch.Generator().manual_seed(m + 31 * n + k)
    x = torch.randint(-60, 61, (m, k), generator=g).float()
    w = torch.randint(-60, 61, (n, k), generator=g).float()
    x[:, 0], w[:, k - 1] = 127, -127
    go = torch.randint(-8, 9, (m, n), generator=g).float()
    wt, bt = w.cuda().requires_grad_(True), torch.zeros(n, device="cuda", requires_grad=True)
    xt = x.to(dt).cuda().requires_grad_(True)
    y = F.linear_int8(xt, wt, bt)
    dx, dw, db = torch.autograd.grad(y, [xt, wt, bt], go.to(dt).cuda())
    assert dx.dtype == dt and dw.dtype == torch.float32 and db.dtype == torch.float32
    assert torch.equal(dw.cpu().double(), go.double().t() @ x.double())
    assert torch.equal(db.cpu().double(), go.double().sum(0))
    want = go.double() @ w.double()
    assert torch.equal(dx.cpu(), want.float().to(dt))


@pytest.mark.parametrize("dt,wdt", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                    (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32),
                                    (torch.float16, torch.float16)])
@pytest.mark.parametrize("m,n,k", GRADS)
def test_gradients(dt, wdt, m, n, k):
    import sc_functional as F
    print("gradients", dt, wdt, m, n, k, flush=True)
    g = torch.Generator().manual_seed(m + n * 5 + k)
    x, w = torch.randn(m, k, generator=g).to(dt), (torch.randn(n, k, generator=g) * k ** -0.5).to(wdt)
    b, go = torch.randn(n, generator=g).to(wdt), torch.randn(m, n, generator=g).to(dt)
    if m > 3:
        x[2] = 0
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    y = F.linear_int8(*leaves)
    qx, sx = quantised(x)
    qw, sw = quantised(w)
    _product_close(y, qx, sx, qw, sw, b, dt)
    dx, dw, db = torch.autograd.grad(y, leaves, go.cuda())
    xd, wd, gd = qx * sx.double()[:, None], qw * sw.double()[:, None], go.double()

    def close(got, want, size, terms, out):
        # the factor g * scale is taken apart into binary16 pieces, each off by half a step of that type, eps / 2 = 2^-11:
        # one, for bfloat16 results, leaves 2^-11 of a term, two, for the others, 2^-11 * 2^-11 = 2^-22.  Terms below
        # 2^-28 of the row's largest: 2^-40 of that, nothing beside the additions' share of `size`.
        pieces = 1 if out == torch.bfloat16 else 2
        tol = size * ((terms * pieces + 4) * 2.0 ** -23 + 2.0 ** (-11 * pieces))
        tol = tol + _half(out) * (want.abs() + tol) + _floor(out)
        err = (got.cpu().double() - want).abs()
        assert got.dtype == out and (err <= tol).all(), "max error %g of its bound" % (err / tol).max()

    close(dx, gd @ wd, gd.abs() @ wd.abs(), n, dt)
    close(dw, gd.t() @ xd, gd.abs().t() @ xd.abs(), m, wdt)
    want = gd.sum(0)
    tol = gd.abs().sum(0) * (m + 4) * U + _half(wdt) * want.abs() * (1 + 2 ** -8) + _floor(wdt)
    assert ((db.cpu().double() - want).abs() <= tol).all() and db.dtype == wdt


def test_gradient_against_differences():
    """y is linear in the dequantised operands: a step of a whole quantisation unit moves y by the gradient times it."""
    import sc_functional as F
    w = torch.randint(-50, 51, (6, 40)).float()
    x = torch.randint(-50, 51, (5, 40)).float()
    w[:, 0], x[:, 1] = 127, 127
    go = torch.randint(-4, 5, (5, 6)).float().cuda()
    f = lambda a, c: (F.linear_int8(a.cuda(), c.cuda()) * go).sum().item()
    xt, wt = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    dx, dw = torch.autograd.grad((F.linear_int8(xt, wt) * go).sum(), [xt, wt])
    for i, j in ((0, 0), (3, 17), (4, 39)):
        p = x.clone()
        p[i, j] += 1
        assert f(p, w) - f(x, w) == dx[i, j].item()
        p = w.clone()
        p[i, j + (j == 0)] += 1
        assert f(x, p) - f(x, w) == dw[i, j + (j == 0)].item()


def test_gradient_forms():
    """Which gradients are asked for, expanded (broadcast) gradients, no tokens, and a frozen weight."""
    import sc_functional as F
    x0, w0, b0 = torch.randn(12, 50, device="cuda"), torch.randn(20, 50, device="cuda"), torch.randn(20, device="cuda")
    leaf = lambda t, r: t.clone().requires_grad_(r)
    full = None
    for rx, rw, rb in itertools.product((True, False), repeat=3):
        if not (rx or rw or rb):
            continue
        x, w, b = leaf(x0, rx), leaf(w0, rw), leaf(b0, rb)
        y = F.linear_int8(x, w, b)
        wanted = [t for t in (x, w, b) if t.requires_grad]
        got = dict(zip([n for n, r in zip("xwb", (rx, rw, rb)) if r], torch.autograd.grad(y.sum(), wanted)))
        full = full or got
        for name, t in got.items():
            tol = 40 * U * 12 if name == "b" else 0
            assert (t - full[name]).abs().max() <= tol, (name, rx, rw, rb)
    x, w, b = leaf(x0[:0], True), leaf(w0, True), leaf(b0, True)
    dx, dw, db = torch.autograd.grad(F.linear_int8(x, w, b).sum(), [x, w, b])
    assert dx.shape == (0, 50) and not dw.any() and not db.any()
    wq, ws = F.quantize_rows(w0)
    x, b = leaf(x0, True), leaf(b0, True)
    dx, db = torch.autograd.grad(F.linear_int8(x, wq, b, weight_scale=ws).sum(), [x, b])
    assert torch.equal(dx, full["x"])
    with pytest.raises(RuntimeError):
        y = F.linear_int8(leaf(x0, True), w0)
        gx, = torch.autograd.grad(y.sum(), [y.grad_fn.next_functions[0][0].variable], create_graph=True)
        gx.sum().backward()


def test_gradient_of_an_infinite_and_a_nan_output_gradient():
    import sc_functional as F
    x, w = torch.randn(3, 16, device="cuda").requires_grad_(True), torch.randn(4, 16, device="cuda").requires_grad_(True)
    go = torch.ones(3, 4, device="cuda")
    go[1, 2], go[2, 0] = float("inf"), float("nan")
    dx, dw = torch.autograd.grad(F.linear_int8(x, w), [x, w], go)
    clean = torch.autograd.grad(F.linear_int8(x, w), [x], torch.ones_like(go))[0]
    assert torch.equal(dx[0], clean[0]) and not dx[1].isfinite().any() and dx[2].isnan().all()
    assert dw[[1, 3]].isfinite().all() and not dw[2].isfinite().any() and dw[0].isnan().all()


# ---- every tile and share of the reduction ---------------------------------------------------------
@pytest.mark.parametrize("tile", ["32", "64", "128", "256"])
@pytest.mark.parametrize("splits", ["1", "3", "16"])
def test_forced_tiles_and_splits(tile, splits, monkeypatch):
    """Integer sums do not depend on the plan; the gradients' float32 sums are exact here (integers, see above)."""
    import sc_functional as F
    monkeypatch.setenv("REXSC_TUNE_INT8_TILE", tile)
    monkeypatch.setenv("REXSC_TUNE_INT8_SPLITS", splits)
    g = torch.Generator().manual_seed(5)
    for m, n, k in ((1, 1, 1), (3, 70, 129), (130, 259, 500), (257, 65, 2100), (300, 513, 127)):
        print("forced", tile, splits, m, n, k, flush=True)
        qa = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int8)
        qb = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8)
        sa, sb, bias = torch.rand(m, generator=g), torch.rand(n, generator=g), torch.randn(n, generator=g)
        for dt in (torch.float32, torch.bfloat16):
            y = F.matmul_int8(qa.cuda(), sa.cuda(), qb.cuda(), sb.cuda(), bias.cuda(), dt)
            _product_close(y, qa, sa, qb, sb, bias, dt)
        x, w = torch.randint(-60, 61, (m, k), generator=g).float(), torch.randint(-60, 61, (n, k), generator=g).float()
        x[:, 0], w[:, k - 1] = 127, -127
        go = torch.randint(-8, 9, (m, n), generator=g).float()
        xt, wt = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
        dx, dw = torch.autograd.grad(F.linear_int8(xt, wt), [xt, wt], go.cuda())
        assert torch.equal(dx.cpu().double(), go.double() @ w.double())
        assert torch.equal(dw.cpu().double(), go.double().t() @ x.double())


def test_offsets_behind_32_bits():
    """A result and an operand of more than 2^31 elements: the last rows are as right as the first."""
    import sc_functional as F
    m, n, k = 70001, 32776, 48
    a = torch.randint(-128, 128, (m, k), device="cuda", dtype=torch.int8)
    b = torch.randint(-128, 128, (n, k), device="cuda", dtype=torch.int8)
    one = torch.ones(max(m, n), device="cuda")
    y = F.matmul_int8(a, one[:m], b, one[:n], None, torch.bfloat16)
    for r in (0, 40000, 65535, 65536, m - 1):
        want = (a[r].cpu().double() @ b.cpu().double().t()).float().bfloat16()
        assert torch.equal(y[r].cpu(), want), r
    del y
    x = torch.randn(1 << 19, 4100, device="cuda", dtype=torch.bfloat16)
    q, s = F.quantize_rows(x)
    for r in (0, 300000, (1 << 19) - 1):
        qe, se = quantised(x[r])
        assert torch.equal(q[r].cpu().double(), qe) and torch.equal(s[r].cpu(), se), r


def test_result_of_more_tiles_than_a_launch_of_small_ones():
    """131072 x 131104 (34 GB): more 64 x 32 tiles than a launch of them could have."""
    import sc_functional as F
    m, n, k = 1 << 17, (1 << 17) + 32, 16
    a = torch.randint(-128, 128, (m, k), device="cuda", dtype=torch.int8)
    b = torch.randint(-128, 128, (n, k), device="cuda", dtype=torch.int8)
    one = torch.ones(n, device="cuda")
    y = F.matmul_int8(a, one[:m], b, one, None, torch.bfloat16)
    for r in (0, 255, 256, 65535, 100000, m - 1):
        want = (a[r].cpu().double() @ b.cpu().double().t()).float().bfloat16()
        assert torch.equal(y[r].cpu(), want), r


@pytest.mark.parametrize("dt,n", [(torch.bfloat16, 4104), (torch.float16, 4101), (torch.float32, 4100), (torch.float32, 4099)])
@pytest.mark.parametrize("k", [1, 100, 128, 129, 300, 513])
def test_more_large_tiles_than_blocks(dt, n, k, monkeypatch):
    """A block goes on from tile to tile: each tile's rows, columns and factors must be its own, whatever the number of
    steps (one, two, an odd number) and wherever the last tiles end."""
    import sc_functional as F
    m = 4353
    print("tiles", dt, m, n, k, flush=True)
    gen = torch.Generator(device="cuda").manual_seed(n + k)
    pitch = max(128, -(-k // 128) * 128)
    a, b = (torch.randint(-127, 128, (r, pitch), device="cuda", dtype=torch.int8, generator=gen)[:, :k] for r in (m, n))
    sa, sb = (torch.rand(r, device="cuda", generator=gen) + 0.5 for r in (m, n))
    bias = torch.randn(n, device="cuda", generator=gen).to(dt)
    monkeypatch.setenv("REXSC_TUNE_INT8_TILE", "256")
    y = F.matmul_int8(a, sa, b, sb, bias, out_dtype=dt)
    prod = (a.double() @ b.double().t().contiguous()) * sa.double()[:, None] * sb.double()
    want = prod + bias.double()
    _close_or_over(y, prod, want, dt)


@pytest.mark.parametrize("dt,n", [(torch.bfloat16, 4104), (torch.float16, 4101), (torch.float32, 4099)])
@pytest.mark.parametrize("k", [8192, 8205])
def test_last_tiles_split_over_the_reduction(dt, n, k, monkeypatch):
    """4353 x 4100 is one round of 256 tiles and 50 more, which are summed in shares."""
    import sc_functional as F
    m = 4353
    gen = torch.Generator(device="cuda").manual_seed(n + k)
    pitch = -(-k // 128) * 128
    a, b = (torch.randint(-127, 128, (r, pitch), device="cuda", dtype=torch.int8, generator=gen)[:, :k] for r in (m, n))
    sa, sb = ((torch.rand(r, device="cuda", generator=gen) + 0.5) / 100 for r in (m, n))
    bias = torch.randn(n, device="cuda", generator=gen).to(dt)
    monkeypatch.setenv("REXSC_TUNE_INT8_TILE", "256")
    y = F.matmul_int8(a, sa, b, sb, bias, out_dtype=dt)
    prod = (a.double() @ b.double().t().contiguous()) * sa.double()[:, None] * sb.double()
    _close_or_over(y, prod, prod + bias.double(), dt)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_gradients_whose_last_tiles_are_split(dt, monkeypatch):
    """As test_gradients_of_integers_are_exact, dx of 306 tiles and 66 or 33 steps."""
    import sc_functional as F
    m, n, k = 4353, 2100, 4100
    monkeypatch.setenv("REXSC_TUNE_INT8_TILE", "256")
    g = torch.Generator(device="cuda").manual_seed(5)
    ints = lambda top, *shape: torch.randint(-top, top + 1, shape, device="cuda", generator=g).float()
    x, w, go = ints(60, m, k), ints(60, n, k), ints(8, m, n)
    x[:, 0], w[:, k - 1] = 127, -127
    xt, wt = x.to(dt).requires_grad_(True), w.clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(F.linear_int8(xt, wt), [xt, wt], go.to(dt))
    assert torch.equal(dx, (go.double() @ w.double()).float().to(dt))
    assert torch.equal(dw.double(), go.double().t().contiguous() @ x.double())


@pytest.mark.parametrize("m,n", [(4353, 4100), (1100, 900)])
@pytest.mark.parametrize("k", [100, 385, 1100])
def test_tiles_of_128_alone_on_a_cu_and_not(m, n, k, monkeypatch):
    import sc_functional as F
    gen = torch.Generator(device="cuda").manual_seed(m + k)
    pitch = -(-k // 128) * 128
    a, b = (torch.randint(-127, 128, (r, pitch), device="cuda", dtype=torch.int8, generator=gen)[:, :k] for r in (m, n))
    sa, sb = (torch.rand(r, device="cuda", generator=gen) + 0.5 for r in (m, n))
    monkeypatch.setenv("REXSC_TUNE_INT8_TILE", "128")
    y = F.matmul_int8(a, sa, b, sb, None)
    want = (a.double() @ b.double().t().contiguous()) * sa.double()[:, None] * sb.double()
    assert ((y.double() - want).abs() <= 5 * U * want.abs() + 2.0 ** -126).all()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("m,n,k", [(1, 24, 8192), (2, 24, 4096), (2, 24, 4104), (2, 24, 8192), (16, 24, 1024), (16, 40, 520), (16, 40, 512),
                                   (3, 24, 5000), (1, 24, 8200), (2, 4096, 600), (2, 4104, 600), (2, 8200, 600), (2, 16392, 600),
                                   (4, 4104, 2056), (4, 8200, 2056)])
def test_serving_around_the_fused_sizes(dt, m, n, k):
    test_linear_int8_serving(dt, m, n, k)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("m,n", [(3, 33), (70, 65), (70, 1001), (130, 1002), (300, 130), (700, 5003)])
def test_nothing_is_written_behind_a_result(dt, m, n, monkeypatch):
    """The result lies inside a larger buffer whose rest must stay as it was, from the kernel's own entry."""
    import _lib
    import _ops
    gen = torch.Generator(device="cuda").manual_seed(m * n)
    a, b = (torch.randint(-127, 128, (r, 128), device="cuda", dtype=torch.int8, generator=gen) for r in (m, n))
    sa, sb = (torch.rand(r, device="cuda", generator=gen) + 0.5 for r in (m, n))
    # (a kernel may round the last multiply-add to the type at once or by way of float32, so two of them are a step of the
    # type apart where the value lies within a float32 rounding of a tie: each is held to the bound, not to another)
    want = (a.double() @ b.double().t().contiguous()) * sa.double()[:, None] * sb.double()
    for tile in ("", "32", "64", "128", "256"):
        monkeypatch.setenv("REXSC_TUNE_INT8_TILE", tile) if tile else monkeypatch.delenv("REXSC_TUNE_INT8_TILE", raising=False)
        for before in (8, 5, 2):  # elements in front of the result: aligned to 16 bytes, or to an element only
            whole = torch.full((before + m * n + 512,), 7.0, device="cuda", dtype=dt)
            d = _lib.Int8Desc.packed(m, n, 128, _ops._dtype_code(dt, ""), 0, 0, 0, 0, 128, 128)
            ws, nbytes = _ops._int8_space(_lib.lib(), d, _lib.INT8_PRODUCT, a.device)
            rc = _lib.lib().rexsc_int8_product(d, a.data_ptr(), sa.data_ptr(), b.data_ptr(), sb.data_ptr(), None,
                                               whole.data_ptr() + before * whole.element_size(), _ops._addr(ws), nbytes,
                                               _ops._raw_stream(0))
            _lib.check(rc, "rexsc_int8_product")
            _close_or_over(whole[before:before + m * n].view(m, n), want, want, dt)
            assert (whole[:before] == 7).all() and (whole[before + m * n:] == 7).all(), (tile, before)


def test_more_rows_than_blocks():
    import sc_functional as F
    x = torch.randn((1 << 23) + 9, 3, device="cuda", dtype=torch.float16)
    q, s = F.quantize_rows(x)
    for sl in (slice(0, 1000), slice((1 << 23) - 500, None)):
        qe, se = quantised(x[sl])
        assert torch.equal(q[sl].cpu().double(), qe) and torch.equal(s[sl].cpu(), se)


# ---- streams, graphs, threads --------------------------------------------------------------------
def test_two_streams_at_once():
    import sc_functional as F
    x = [torch.randn(m, 1000, device="cuda") for m in (3, 200)]
    w = torch.randn(300, 1000, device="cuda")
    wq, ws = F.quantize_rows(w)
    want = [F.linear_int8(v, wq, None, weight_scale=ws) for v in x]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(F.linear_int8(x[i], wq, None, weight_scale=ws))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


@pytest.mark.parametrize("m", [1, 24, 150])
def test_captured_forward_and_backward(m):
    import sc_functional as F
    print("graph", m, flush=True)
    x0, w0, g0 = torch.zeros(m, 520, device="cuda"), torch.zeros(90, 520, device="cuda"), torch.zeros(m, 90, device="cuda")
    b0 = torch.zeros(90, device="cuda")
    wq, ws = F.quantize_rows(torch.randn(90, 520, device="cuda"))

    def step():
        x, w, b = (t.detach().requires_grad_(True) for t in (x0, w0, b0))
        y = F.linear_int8(x, w, b)
        return (y.detach(),) + torch.autograd.grad(y, [x, w, b], g0) + (F.linear_int8(x0, wq, b0, weight_scale=ws),)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for r in range(3):
        for t in (x0, w0, b0, g0):
            t.normal_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, b in zip(got, step()):
            assert torch.equal(a, b), "replay %d" % r


# ---- layers --------------------------------------------------------------------------------------
def test_layer_trains_freezes_and_reloads():
    import sc_functional as F
    from sc_layers import Linear_Int8
    torch.manual_seed(1)
    layer = Linear_Int8(70, 33).cuda()
    x = torch.randn(5, 70, device="cuda")
    y = layer(x)
    y.square().sum().backward()
    assert layer.weight.grad.shape == (33, 70) and layer.bias.grad.abs().sum() > 0
    other = Linear_Int8.from_linear(torch.nn.Linear(70, 33, bias=False)).cuda()
    assert other.bias is None and torch.equal(other(x), F.linear_int8(x, other.weight))
    with torch.no_grad():
        want = layer(x)
    layer.freeze()
    assert layer.frozen and layer.weight is None
    assert torch.equal(layer(x), want)
    assert layer.freeze() is layer
    state = layer.state_dict()
    assert set(state) == {"bias", "weight_q", "weight_scale"}
    fresh = Linear_Int8(70, 33).cuda()
    fresh.load_state_dict(state)
    assert torch.equal(fresh(x), want)
    moved = layer.cpu().cuda()
    assert torch.equal(moved(x), want)
    xg = x.clone().requires_grad_(True)
    layer(xg).sum().backward()
    assert xg.grad.shape == x.shape


def test_frozen_layer_in_half_precision():
    from sc_layers import Linear_Int8
    layer = Linear_Int8(70, 33, bias=False).cuda().freeze()
    x = torch.randn(5, 70, device="cuda").half()
    with torch.no_grad():
        want = layer(x)
        scale = layer.weight_scale.clone()
        assert torch.equal(layer.half()(x), want) and torch.equal(layer.weight_scale, scale)
        assert layer.weight_scale.dtype == torch.float32


def test_autocast_region():
    import sc_functional as F
    x, w = torch.randn(6, 64, device="cuda"), torch.randn(9, 64, device="cuda").requires_grad_(True)
    for dt in (torch.float16, torch.bfloat16):
        with torch.autocast("cuda", dtype=dt):
            y = F.linear_int8(x, w)
        assert y.dtype == dt and torch.equal(y.detach(), F.linear_int8(x.to(dt), w.detach()))
        dw, = torch.autograd.grad(y.float().sum(), [w])
        assert dw.dtype == torch.float32


@pytest.mark.parametrize("wdt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(4, 2, 16), (70, 34, 129), (256, 10, 1024)])
def test_bfloat16_gradients_are_sums_of_float32_factors(wdt, m, n, k):
    """Terms that cancel to a part in 256 of their size: what the factor g * scale is held in shows there.  Two binary16
    pieces are off by 2^-22 of a term, each of the additions of both by at most 2^-23 of the terms' magnitudes, and the
    sum is rounded once."""
    import sc_functional as F
    g = torch.Generator().manual_seed(m + n + k)
    pairs = lambda r, c: (torch.randn(r // 2, c, generator=g) * 3).repeat_interleave(2, 0)
    x, w = pairs(m, k).bfloat16(), pairs(n, k).to(wdt)
    go = torch.randn(m // 2, n // 2, generator=g).bfloat16().float()
    near = (go * (1 + 2.0 ** -7)).bfloat16().float()
    # rows and columns in pairs of opposite sign, one of four a step of bfloat16 beside the others
    go = torch.stack([torch.stack([near, -go], -1), torch.stack([-go, go], -1)], 1).reshape(m, n).bfloat16()
    xt, wt = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    dx, dw = torch.autograd.grad(F.linear_int8(xt, wt), [xt, wt], go.cuda())
    (qx, sx), (qw, sw) = quantised(x), quantised(w)
    xd, wd, gd = qx * sx.double()[:, None], qw * sw.double()[:, None], go.double()
    for got, want, size, terms, out in ((dx, gd @ wd, gd.abs() @ wd.abs(), n, torch.bfloat16), (dw, gd.t() @ xd, gd.abs().t() @ xd.abs(), m, wdt)):
        tol = size * ((terms * 2 + 4) * 2.0 ** -23 + 2.0 ** -22)
        tol = tol + _half(out) * (want.abs() + tol) + _floor(out)
        err = (got.cpu().double() - want).abs()
        assert (err <= tol).all(), "max error %g of its bound" % (err / tol).max()


@pytest.mark.parametrize("n", [30, 64, 1000])
def test_gradient_with_scales_of_any_layout(n):
    """Scales out of a table of several per channel, and one for all channels expanded: as their dense copies."""
    import sc_functional as F
    x0, wq = torch.randn(20, 70, device="cuda"), F.quantize_rows(torch.randn(n, 70, device="cuda"))[0]
    table, go = torch.rand(n, 3, device="cuda") + 0.1, torch.randn(20, n, device="cuda")

    def both(scale):
        x = x0.clone().requires_grad_(True)
        y = F.linear_int8(x, wq, None, weight_scale=scale)
        return y.detach(), torch.autograd.grad(y, [x], go)[0]

    for scale in (table[:, 1], table[:, :1], table[:1, 0].expand(n), table[0, 2].expand(n), table[:, 0].flip(0)):
        assert all(torch.equal(a, b) for a, b in zip(both(scale), both(scale.contiguous())))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("m,n,k", [(6, 8, 40), (70, 33, 129), (300, 10, 2048)])
def test_infinite_and_nan_gradients_go_where_the_product_takes_them(dt, m, n, k):
    """inf times a nonzero value is an infinity of its sign, times 0 a NaN; the finite results are as without them."""
    import sc_functional as F
    g = torch.Generator().manual_seed(m + n)
    x, w = torch.randint(-3, 4, (m, k), generator=g).to(dt), torch.randint(-3, 4, (n, k), generator=g).float()
    x[:, 0], w[:, 0] = 3, -3
    go = torch.randint(-8, 9, (m, n), generator=g).to(dt)
    inf = float("inf")
    go[1, 2], go[2, 0], go[3, 1], go[3, 4], go[4, 5], go[4, 6] = inf, float("nan"), -inf, inf, inf, inf
    xt, wt = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    dx, dw = torch.autograd.grad(F.linear_int8(xt, wt), [xt, wt], go.cuda())
    (qx, sx), (qw, sw) = quantised(x), quantised(w)
    for got, a, b, s in ((dx, go.double() * sw.double(), qw, "dx"), (dw, (go.double() * sx.double()[:, None]).t(), qx, "dw")):
        want = (a[:, :, None] * b[None]).sum(1) if a.shape[0] * b.numel() < 1 << 25 else torch.stack([(r[:, None] * b).sum(0) for r in a])
        got = got.cpu().double()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf()), s
        assert torch.equal(got[got.isinf()], want[want.isinf()])
        ok = want.isfinite()
        size = (a.abs().nan_to_num(0, 0, 0) @ b.abs())
        tol = size * ((2 * a.shape[1] + 4) * 2.0 ** -23 + 2.0 ** -11) + _half(dt) * want.abs() * (1 + 2.0 ** -8) + _floor(dt)
        assert ((got - want).abs() <= tol)[ok].all()
    assert dx[1].isinf().any() and dx[4].isinf().any() and dw[2].isinf().any()


@pytest.mark.parametrize("m", [3, 60])
def test_weights_whose_rows_are_far_apart(m):
    import sc_functional as F
    store = torch.randint(-127, 128, ((16 << 20) + 64,), device="cuda", dtype=torch.int8)
    x, s = torch.randn(m, 48, device="cuda"), torch.rand(3, device="cuda")
    far = store.as_strided((3, 48), (8 << 20, 1))
    xg = x.clone().requires_grad_(True)
    y = F.linear_int8(xg, far, None, weight_scale=s)
    want = F.linear_int8(xg, far.contiguous(), None, weight_scale=s)
    assert torch.equal(y, want)
    assert torch.equal(*(torch.autograd.grad(t.sum(), [xg])[0] for t in (y, want)))


def test_gradient_of_the_input_for_more_tokens_than_the_weights_sums_over():
    """A frozen weight has no gradient to sum over the tokens: their number is not held to that sum's limit."""
    import sc_functional as F
    m, n, k = (1 << 22) + 5, 10, 24
    gen = torch.Generator(device="cuda").manual_seed(1)
    wq = torch.randint(-127, 128, (n, k), device="cuda", generator=gen).to(torch.int8)
    x = torch.zeros(m, k, device="cuda", dtype=torch.float16).requires_grad_(True)
    go = torch.randint(-8, 9, (m, n), device="cuda", generator=gen).half()
    b = torch.zeros(n, device="cuda", requires_grad=True)
    y = F.linear_int8(x, wq, b, weight_scale=torch.ones(n, device="cuda"))
    dx, db = torch.autograd.grad(y, [x, b], go)
    assert torch.equal(dx, (go.float() @ wq.float()).half())  # integers below 2^24: exact, then rounded once
    assert torch.equal(db.double(), go.double().sum(0))
    w = wq.float().requires_grad_(True)
    with pytest.raises(RuntimeError, match="at most"):
        torch.autograd.grad(F.linear_int8(x.detach(), w), [w], go)
