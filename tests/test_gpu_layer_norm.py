"""Layer norm against its definition in 64 bits.

Bounds, with u = 2^-24 and `depth` the longest chain of additions in a row's sum (a thread's elements, six steps over
the lanes, the waves): the mean is off by at most depth u mean|x|, so (x - mu) r by E = u r (|x| + |mu| + depth mean|x|)
plus (depth + 8) u |h| for the variance and the reciprocal root; y adds two roundings and half a step of its type.
dx = r (gw - m0 - h m1) carries E through both sums."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0 ** -24
SIZES = [(1, 1), (2, 3), (5, 64), (3, 255), (7, 1000), (9, 1024), (4, 1003), (3, 1032), (6, 2048), (2, 4096), (3, 4097),
         (2, 8192), (2, 8200), (3, 16384), (2, 16385), (1, 40000), (1000, 40), (515, 512), (4100, 16), (0, 8)]


def _half(dt):
    return torch.finfo(dt).eps / 2


def _floor(dt):
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps


def reference(x, w, b, g, eps=1e-5):
    x, D = x.double(), x.shape[1]
    w = torch.ones(D, dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(D, dtype=torch.float64) if b is None else b.double()
    depth = max(16, -(-D // 1024)) + 6 + 16
    mu = x.mean(1, keepdim=True)
    r = (x - mu).square().mean(1, keepdim=True).add(eps).rsqrt()
    h = (x - mu) * r
    e = U * (r * (x.abs() + mu.abs() + depth * x.abs().mean(1, keepdim=True)) + (depth + 8) * h.abs())
    y = h * w + b
    ty = e * w.abs() + 2 * U * (y.abs() + (h * w).abs())
    out = {"y": (y, ty)}
    if g is not None:
        g = g.double()
        gw = g * w
        m0, m1 = gw.mean(1, keepdim=True), (gw * h).mean(1, keepdim=True)
        dx = r * (gw - m0 - h * m1)
        s0, s1 = gw.abs().mean(1, keepdim=True), (gw * h).abs().mean(1, keepdim=True)
        # errors of m0 and m1, of h times m1, and of r (depth + 8 half-steps), on the magnitudes they act on
        t1 = (depth + 4) * U * s1 + (gw.abs() * e).mean(1, keepdim=True)
        tdx = r * ((depth + 4) * U * s0 + h.abs() * t1 + e * m1.abs() + 4 * U * (gw.abs() + m0.abs() + (h * m1).abs()))
        tdx = tdx + (depth + 8) * U * r * (gw.abs() + m0.abs() + (h * m1).abs())
        n = x.shape[0]
        out["dx"] = (dx, tdx)
        out["dw"] = ((g * h).sum(0), (g.abs() * e).sum(0) + (n + 8) * U * (g * h).abs().sum(0))
        out["db"] = (g.sum(0), (n + 8) * U * g.abs().sum(0))
    return out


def close(got, ref, dt, what):
    want, tol = ref
    tol = tol + _half(dt) * (want.abs() + tol) + _floor(dt)
    err = (got.detach().cpu().double() - want).abs()
    assert got.dtype == dt and got.shape == want.shape, what
    assert (err <= tol).all(), "%s: max error %g of its bound" % (what, (err / tol).max())


@pytest.mark.parametrize("rows,d", SIZES)
@pytest.mark.parametrize("dt,wdt", [(torch.float32, torch.float32), (torch.float16, torch.float32),
                                    (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16),
                                    (torch.float16, torch.float16)])
def test_forward_and_gradients(dt, wdt, rows, d):
    import sc_functional as F
    print("layer norm", dt, wdt, rows, d, flush=True)
    gen = torch.Generator().manual_seed(rows * 17 + d)
    x = (torch.randn(rows, d, generator=gen) * 2 + 0.7).to(dt)
    x[:, ::13] *= 6
    w, b = (1 + 0.2 * torch.randn(d, generator=gen)).to(wdt), torch.randn(d, generator=gen).to(wdt)
    g = torch.randn(rows, d, generator=gen).to(dt)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    y = F.layer_norm(*leaves)
    ref = reference(x, w, b, g)
    close(y, ref["y"], dt, "y")
    dx, dw, db = torch.autograd.grad(y, leaves, g.cuda())
    close(dx, ref["dx"], dt, "dx")
    close(dw, ref["dw"], wdt, "dw")
    close(db, ref["db"], wdt, "db")
    assert torch.equal(F.layer_norm(x.cuda(), w.cuda(), b.cuda()), y.detach())


@pytest.mark.parametrize("dt,wdt", [(torch.float32, torch.float32), (torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("d", [256, 257, 264, 1032, 1101, 1280, 1281, 1288, 1536, 1537, 2001, 2560, 2561, 2568, 3060, 3080, 4104,
                               5120, 5121, 5128, 6144, 6145, 8193, 8200, 9001, 10240, 10241, 12001, 12288, 12289, 16383])
def test_widths_around_the_numbers_of_threads(dt, wdt, d):
    test_forward_and_gradients(dt, wdt, 3, d)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("d", [37, 250, 1101, 1536, 2001, 5001, 8200, 9001, 12288, 16383])
def test_rows_inside_another_matrix(dt, d):
    """Rows that begin anywhere, beside elements that must neither be read as theirs nor written."""
    import sc_functional as F
    gen = torch.Generator().manual_seed(d)
    whole = torch.randn(5, d + 11, generator=gen).to(dt)
    whole[:, :3], whole[:, d + 3:] = 1e4, -1e4
    w, b = 1 + 0.2 * torch.randn(d, generator=gen), torch.randn(d, generator=gen)
    g = torch.randn(5, d, generator=gen).to(dt)
    x = whole.cuda()[:, 3:d + 3].requires_grad_()
    leaves = [x, w.cuda().requires_grad_(), b.cuda().requires_grad_()]
    y = F.layer_norm(*leaves)
    ref = reference(whole[:, 3:d + 3], w, b, g)
    close(y, ref["y"], dt, "y")
    for name, got, t in zip(("dx", "dw", "db"), torch.autograd.grad(y, leaves, g.cuda()), (dt, torch.float32, torch.float32)):
        close(got, ref[name], t, name)


@pytest.mark.parametrize("dt,wdt", [(torch.float32, torch.float32), (torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("rows,d", [(511, 33), (512, 2048), (513, 33), (512, 2049), (4, 2047), (15, 16), (17, 17), (100, 1), (1, 2048)])
def test_around_the_backward_pass_in_one_launch(dt, wdt, rows, d):
    test_forward_and_gradients(dt, wdt, rows, d)


@pytest.mark.parametrize("d", [48, 1003, 5000])
def test_without_weight_or_bias_and_partial_gradients(d):
    import sc_functional as F
    gen = torch.Generator().manual_seed(d)
    x, w, b = torch.randn(21, d, generator=gen), torch.randn(d, generator=gen), torch.randn(d, generator=gen)
    g = torch.randn(21, d, generator=gen)
    for hw, hb in ((True, False), (False, True), (False, False), (True, True)):
        wt, bt = w if hw else None, b if hb else None
        ref = reference(x, wt, bt, g)
        for mask in range(1, 8):
            xs = x.cuda().requires_grad_(bool(mask & 1))
            ws = wt.cuda().requires_grad_(bool(mask & 2)) if hw else None
            bs = bt.cuda().requires_grad_(bool(mask & 4)) if hb else None
            named = [(n, t) for n, t in (("dx", xs), ("dw", ws), ("db", bs)) if t is not None and t.requires_grad]
            y = F.layer_norm(xs, ws, bs)
            close(y, ref["y"], torch.float32, "y")
            if named:
                for (n, _), got in zip(named, torch.autograd.grad(y, [t for _, t in named], g.cuda())):
                    close(got, ref[n], torch.float32, n)


def test_layouts_and_constant_rows():
    import sc_functional as F
    w, b = torch.randn(96, device="cuda"), torch.randn(96, device="cuda")
    base = torch.randn(6, 5, 120, device="cuda")
    for v in (base[..., :96], base[..., 7:103], base[::2, 1:, 8:104], base.transpose(0, 1)[..., 24:], base[0, 0, :96],
              base[:1, :1, :96].expand(3, 4, 96), torch.randn(96, 40, device="cuda").t()):
        # rows that do not start on 16 bytes are summed in another order than a dense copy's (single elements in place of
        # vectors per thread), so the two agree within the bounds above and not bit for bit
        y = F.layer_norm(v, w, b)
        ref = reference(v.cpu().reshape(-1, 96), w.cpu(), b.cpu(), None)["y"]
        assert y.shape == v.shape
        close(y.reshape(-1, 96), ref, torch.float32, "strided")
        leaf = v.detach().clone(memory_format=torch.preserve_format).requires_grad_(True)
        y = F.layer_norm(leaf, w, b)
        gx, = torch.autograd.grad(y, [leaf], torch.ones(1, device="cuda").expand(y.shape))
        assert gx.shape == v.shape
    # a row of equal values has variance 0: y is the bias exactly where the mean is exact
    const = torch.full((3, 96), 5.0, device="cuda")
    assert torch.equal(F.layer_norm(const, w, b), b.expand(3, 96))
    # a far mean: the variance is taken around it, not as a difference of squares
    x = torch.randn(4, 96) + 4096.0
    close(F.layer_norm(x.cuda(), w, b), reference(x, w.cpu(), b.cpu(), None)["y"], torch.float32, "far mean")
    # a NaN stays in its row
    bad = base[0, :, :96].clone()
    bad[2, 5] = float("nan")
    y = F.layer_norm(bad, w, b)
    assert y[2].isnan().all() and y[[0, 1, 3, 4]].isfinite().all()


def test_gradient_against_differences():
    import sc_functional as F
    x, w, b = torch.randn(3, 20), torch.randn(20), torch.randn(20)
    g = torch.randn(3, 20)
    f = lambda *t: (reference(t[0], t[1], t[2], None)["y"][0] * g.double()).sum()
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    got = torch.autograd.grad(F.layer_norm(*leaves), leaves, g.cuda())
    for i, t in enumerate((x, w, b)):
        for at in (0, t.numel() // 2, t.numel() - 1):
            plus, minus = t.double().clone(), t.double().clone()
            plus.view(-1)[at] += 1e-4
            minus.view(-1)[at] -= 1e-4
            args = [x, w, b]
            d = (f(*args[:i], plus, *args[i + 1:]) - f(*args[:i], minus, *args[i + 1:])) / 2e-4
            # central differences of a smooth function: third derivative times h^2 (1e-8, with factors up to 1e2 here),
            # and float32's own error of some 1e-6
            assert abs(d - got[i].view(-1)[at].cpu().double()) <= 2e-5 * (1 + abs(d)), (i, at)


def test_captured_and_two_streams():
    import sc_functional as F
    x0, w0, g0 = torch.zeros(33, 700, device="cuda"), torch.ones(700, device="cuda"), torch.zeros(33, 700, device="cuda")

    def step():
        x, w = x0.detach().requires_grad_(True), w0.detach().requires_grad_(True)
        y = F.layer_norm(x, w, None)
        return (y.detach(),) + torch.autograd.grad(y, [x, w], g0)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        for t in (x0, w0, g0):
            t.normal_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
    want, streams, got = step(), [torch.cuda.Stream(), torch.cuda.Stream()], []
    torch.cuda.synchronize()
    for _ in range(6):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(step())
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, want))  # no atomics: the same bits every time


def test_offsets_behind_32_bits():
    import sc_functional as F
    x = torch.randn((1 << 21) + 3, 1032, device="cuda", dtype=torch.bfloat16)
    w, b = torch.randn(1032, device="cuda"), torch.randn(1032, device="cuda")
    xl = x.requires_grad_(True)
    y = F.layer_norm(xl, w, b)
    g = torch.zeros_like(y)
    rows = [0, 5, 1 << 20, (1 << 21) + 2]
    g[rows] = torch.randn(4, 1032, device="cuda").bfloat16()
    dx, = torch.autograd.grad(y, [xl], g)
    ref = reference(x.detach()[rows].cpu(), w.cpu(), b.cpu(), g[rows].cpu())
    close(y.detach()[rows], ref["y"], torch.bfloat16, "y")
    close(dx[rows], ref["dx"], torch.bfloat16, "dx")
    assert not dx[6:1000].any()


def test_rows_longer_than_a_launch_of_column_sums():
    """More columns than a launch has 16-column blocks, and so many that the rows' shares of the weight gradients are
    fewer than the rows."""
    import sc_functional as F
    for rows, d in ((2, (1 << 25) + 17), (70, (1 << 25) + 3)):
        print("rows", rows, d, flush=True)
        gen = torch.Generator(device="cuda").manual_seed(rows)
        dt = torch.float32 if rows == 2 else torch.bfloat16
        x, g = (torch.randn(rows, d, device="cuda", generator=gen).to(dt) for _ in range(2))
        w, b = (torch.randn(d, device="cuda", generator=gen).requires_grad_() for _ in range(2))
        x.requires_grad_()
        y = F.layer_norm(x, w, b)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), g)
        with torch.no_grad():
            mu = torch.stack([r.double().mean() for r in x])[:, None]
            var = torch.stack([(r.double() - m).square().mean() for r, m in zip(x, mu)])[:, None]
            r = (var + 1e-5).rsqrt()
            depth = d // 1024 + 22
            for part in (slice(0, 3000), slice(d - 3000, d)):
                xs, gs, ws = x[:, part].double(), g[:, part].double(), w[part].double()
                h = (xs - mu) * r
                e = U * (r * (xs.abs() + mu.abs() + depth) + (depth + 8) * h.abs())  # mean|x| of a normal row is below 1
                ref = {"y": (h * ws + b[part].double(), e * ws.abs() + 2 * U * (2 * (h * ws).abs() + b[part].double().abs())),
                       "dw": ((gs * h).sum(0), (gs.abs() * e).sum(0) + (rows + 8) * U * (gs * h).abs().sum(0)),
                       "db": (gs.sum(0), (rows + 8) * U * gs.abs().sum(0))}
                for name, got in (("y", y[:, part]), ("dw", dw[part]), ("db", db[part])):
                    close(got, tuple(t.cpu() for t in ref[name]), got.dtype, "%s %d" % (name, rows))
        del x, g, y, dx


def test_layer():
    from sc_layers import LayerNorm
    import sc_functional as F
    layer = LayerNorm((4, 10)).cuda()
    with torch.no_grad():
        layer.weight.normal_()
        layer.bias.normal_()
    x = torch.randn(3, 2, 4, 10, device="cuda", requires_grad=True)
    y = layer(x)
    assert torch.equal(y.detach(), F.layer_norm(x.detach().view(3, 2, 40), layer.weight.detach().view(-1),
                                                layer.bias.detach().view(-1)).view(3, 2, 4, 10))
    y.sum().backward()
    assert layer.weight.grad.shape == (4, 10) and x.grad.shape == x.shape
    assert LayerNorm(10, elementwise_affine=False).cuda()(x).shape == x.shape
    with torch.autocast("cuda", dtype=torch.float16):
        assert layer(x).dtype == torch.float32
    with pytest.raises(RuntimeError, match="shape"):
        LayerNorm(9).cuda()(x)


@pytest.mark.parametrize("rows,d", [(5, 100), (600, 264), (3, 4096), (2, 17000)])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_partial_gradients_of_mixed_types(dt, rows, d):
    """A float32 weight is used as it is whichever gradients are asked for, also where only those of 16 bits are."""
    import sc_functional as F
    gen = torch.Generator().manual_seed(d)
    x, w, b = torch.randn(rows, d, generator=gen).to(dt), 1 + 0.3 * torch.randn(d, generator=gen), torch.randn(d, generator=gen).to(dt)
    g = torch.randn(rows, d, generator=gen).to(dt)
    ref = reference(x, w, b, g)
    for mask in range(1, 8):
        leaves = [t.cuda().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w, b))]
        named = [(n, t) for n, t in zip(("dx", "dw", "db"), leaves) if t.requires_grad]
        for (n, t), got in zip(named, torch.autograd.grad(F.layer_norm(*leaves), [t for _, t in named], g.cuda())):
            close(got, ref[n], t.dtype, "%s %d" % (n, mask))
