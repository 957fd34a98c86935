"""The AdamW step against its definition in 64 bits.

Bounds with u = 2^-24: m and v carry their constants' rounding and three operations (6 u of the two terms'
magnitudes), the root half of v's, the quotient and the subtraction a few more, p half a step of its type.  8-bit states
are e4m3 values: half a step of that grid (2^-4 relative, 2^-10 below 2^-6) and the roundings before it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0 ** -24
E4M3 = torch.float8_e4m3fn
H = dict(lr=3e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.05)


def _half(dt):
    return torch.finfo(dt).eps / 2


def _floor(dt):
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps


def blocks(t):
    """t in rows of 256, padded with zeros."""
    pad = -t.numel() % 256
    return torch.nn.functional.pad(t.reshape(-1), (0, pad)).view(-1, 256)


def decode(values, scale):
    n = values.numel()
    return (blocks(values.reshape(-1).float().cpu()).double() * scale.cpu().double()[:, None]).reshape(-1)[:n]


def reference(p, g, m, v, step, h=H, clamp=None):
    """(p, its bound, m, its bound, root of v, its bound) in 64 bits."""
    p, g = p.double().reshape(-1), g.double().reshape(-1)
    a, c = h["beta1"] * m, (1 - h["beta1"]) * g
    m = a + c
    tm = 6 * U * (a.abs() + c.abs())
    v = h["beta2"] * v + (1 - h["beta2"]) * g * g
    root = v.sqrt()
    troot = 6 * U * root + 2.0 ** -75  # v below the smallest normal number
    size, b2 = h["lr"] / (1 - h["beta1"] ** step), 1 / math.sqrt(1 - h["beta2"] ** step)
    den = root * b2 + h["eps"]
    move = size * m / den
    q = p * (1 - h["lr"] * h["weight_decay"]) - move
    tq = size * tm / den + move.abs() * (8 * U + (b2 * troot / den)) + 4 * U * (p.abs() + move.abs())
    if clamp is not None:
        q = q.clamp(float(torch.tensor(clamp[0])), float(torch.tensor(clamp[1])))
    return q, tq, m, tm, root, troot


def check(got, want, tol, dt, what):
    tol = tol + _half(dt) * (want.abs() + tol) + _floor(dt)
    err = (got.detach().reshape(-1).cpu().double() - want).abs()
    assert (err <= tol).all(), "%s: max error %g of its bound" % (what, (err / tol).max())


def check8(values, scale, want, tol, what, positive):
    """e4m3 values and scales of `want`, which is known to within tol."""
    w, n = blocks(want), want.numel()
    top = w.abs().amax(1)
    s = scale.cpu().double()
    lost = blocks(tol).amax(1)
    assert ((s - top / 448).abs() <= lost / 448 + 2 * U * top / 448 + 2.0 ** -140).all(), what + ": scale"
    q = blocks(values.reshape(-1).float().cpu()).double()
    # the smallest block magnitude that is kept is 2^-100
    exact = torch.where((s > 0)[:, None], w / torch.where(s > 0, s, 1.0)[:, None], 0.0)
    if positive:
        exact = torch.where(exact > 0, exact.clamp(min=2.0 ** -9), exact)
    slack = blocks(tol) / torch.where(s > 0, s, 1.0)[:, None] + 4 * U * exact.abs()
    half = torch.maximum(exact.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10, dtype=torch.float64))
    err = ((q - exact).abs() - slack).reshape(-1)[:n]
    assert (err <= half.reshape(-1)[:n]).all(), "%s: off by %g of half a step" % (what, (err / half.reshape(-1)[:n]).max())
    if positive:
        assert ((q > 0) | (w <= 0) | (top < 2.0 ** -100)[:, None]).all(), what + ": a positive root became 0"


def tensors(shapes, dt, seed, size=1e-3):
    gen = torch.Generator().manual_seed(seed)
    out = []
    for s in shapes:
        p, g = torch.randn(s, generator=gen) * 0.1, torch.randn(s, generator=gen) * size
        m = torch.randn(s, generator=gen) * size * 0.3
        v = (torch.randn(s, generator=gen) * size).square()
        out.append((p.to(dt), g.to(dt), m, v))
    return out


SHAPES = [(1,), (3,), (255,), (256,), (257,), (64, 3, 7, 7), (1000, 512), (4096,), (4097,), (10, 4096), (5, 819, 3), (0,), (1, 1)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("step", [1, 2, 1000])
@pytest.mark.parametrize("clamp", [None, (-0.05, 0.049)])
def test_32_bit_states(dt, step, clamp):
    import sc_optim
    print("adamw 32", dt, step, clamp, flush=True)
    sets = tensors(SHAPES, dt, step)
    dev = [[t.cuda() for t in s] for s in sets]
    sc_optim.adamw_step(*[list(c) for c in zip(*dev)], step=step, clamp=clamp, **H)
    for (p, g, m, v), (dp, dg, dm, dv) in zip(sets, dev):
        q, tq, me, tm, root, troot = reference(p, g, m.double().reshape(-1), v.double().reshape(-1), step, clamp=clamp)
        check(dp, q, tq, dt, "p %s" % (tuple(p.shape),))
        check(dm, me, tm, torch.float32, "m")
        check(dv, root.square(), 12 * U * root.square() + 2.0 ** -149, torch.float32, "v")
        assert torch.equal(dg.cpu(), g)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("size", [1e-3, 1e-12, 1e3])
def test_8_bit_states(dt, size):
    import sc_optim
    if dt == torch.float16:
        size = min(max(size, 1e-3), 1.0)
    print("adamw 8", dt, size, flush=True)
    sets = tensors(SHAPES, dt, 5, size)
    P, G, M, V, MS, VS, old = [], [], [], [], [], [], []
    for p, g, m, v in sets:
        P.append(p.cuda()), G.append(g.cuda())
        n = p.numel()
        state = []
        for t in (m, v.sqrt()):
            b = blocks(t)
            s = b.abs().amax(1) / 448
            q = (b / torch.where(s > 0, s, 1.0)[:, None]).clamp(-448, 448)
            state.append((q.reshape(-1)[:n].to(E4M3), s))
        (mq, ms), (vq, vs) = state
        old.append((decode(mq, ms), decode(vq, vs).square()))
        M.append(mq.cuda()), MS.append(ms.cuda()), V.append(vq.cuda()), VS.append(vs.cuda())
    for step in (7, 8):
        sc_optim.adamw_step(P, G, M, V, MS, VS, step=step, **H)
        for i, (p, g, _, _) in enumerate(sets):
            if p.numel() == 0:
                continue
            before = p if step == 7 else after[i]
            q, tq, me, tm, root, troot = reference(before, g, *old[i], step)
            check(P[i], q, tq, dt, "p %s" % (tuple(p.shape),))
            check8(M[i], MS[i], me, tm, "m", False)
            check8(V[i], VS[i], root, troot, "root of v", True)
        after = [t.cpu() for t in P]
        old = [(decode(a, b), decode(c, d).square()) for a, b, c, d in zip(M, MS, V, VS)]


def test_8_bit_start_from_nothing_and_wide_range():
    """Zero states, zero gradients, and elements twelve orders of magnitude apart in one block."""
    import sc_optim
    n = 700
    g = torch.logspace(-13, 0, n, dtype=torch.float64).float()
    g[::50] = 0
    p = torch.randn(n).cuda()
    before = p.cpu().clone()
    u8 = lambda: torch.zeros(n, dtype=torch.uint8, device="cuda").view(E4M3)
    M, V, MS, VS = u8(), u8(), torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda")
    sc_optim.adamw_step([p], [g.cuda()], [M], [V], [MS], [VS], step=1, **H)
    zero = torch.zeros(n, dtype=torch.float64)
    q, tq, me, tm, root, troot = reference(before, g, zero, zero, 1)
    check(p, q, tq, torch.float32, "p")
    check8(M, MS, me, tm, "m", False)
    check8(V, VS, root, troot, "root", True)
    mid = p.clone()
    sc_optim.adamw_step([p], [torch.zeros(n, device="cuda")], [M], [V], [MS], [VS], step=2, **H)
    q, tq, *_ = reference(mid.cpu(), torch.zeros(n), decode(M, MS) * 0, zero, 2)
    assert p.isfinite().all() and (p - mid).abs().max() < 20 * H["lr"]  # no element was divided by eps alone


def test_a_lost_block_stays_within_its_block():
    import sc_optim
    n = 1024
    p, g = torch.randn(n, device="cuda"), torch.randn(n, device="cuda")
    g[300], g[600] = float("nan"), float("inf")
    u8 = lambda: torch.zeros(n, dtype=torch.uint8, device="cuda").view(E4M3)
    M, V, MS, VS = u8(), u8(), torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda")
    sc_optim.adamw_step([p], [g], [M], [V], [MS], [VS], step=1, **H)
    assert MS.isnan().tolist() == [False, True, True, False] and VS.isnan().tolist() == [False, True, True, False]
    assert p[:256].isfinite().all() and p[768:].isfinite().all() and p[300].isnan()


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_and_unaligned_ones(bits):
    """More tensors than one launch takes, of every length around a chunk, at offsets that rule out vector loads."""
    import sc_optim
    shapes = [((i * 37) % 600 + 1,) for i in range(150)] + [(4095,), (4096,), (4098,), (12289,)]
    dt = torch.bfloat16
    sets = tensors(shapes, dt, 3)
    flat = lambda i, t, off: torch.cat([torch.zeros(off, dtype=t.dtype), t]).cuda()[off:]
    P = [flat(i, s[0], i % 5) for i, s in enumerate(sets)]
    G = [flat(i, s[1], i % 3) for i, s in enumerate(sets)]
    if bits == 32:
        M, V = ([flat(i, s[k], i % 2) for i, s in enumerate(sets)] for k in (2, 3))
        sc_optim.adamw_step(P, G, M, V, step=3, **H)
        old = [(s[2].double(), s[3].double()) for s in sets]
    else:
        zeros = lambda: [torch.zeros(s[0].numel() + i % 3, dtype=torch.uint8, device="cuda")[i % 3:].view(E4M3)
                         for i, s in enumerate(sets)]
        scales = lambda: [torch.zeros(-(-s[0].numel() // 256), device="cuda") for s in sets]
        M, V, MS, VS = zeros(), zeros(), scales(), scales()
        sc_optim.adamw_step(P, G, M, V, MS, VS, step=3, **H)
        old = [(torch.zeros(s[0].numel(), dtype=torch.float64),) * 2 for s in sets]
    for i, s in enumerate(sets):
        q, tq, me, tm, root, troot = reference(s[0], s[1], *old[i], 3)
        check(P[i], q, tq, dt, "p %d" % i)
        if bits == 8:
            check8(M[i], MS[i], me, tm, "m", False)
            check8(V[i], VS[i], root, troot, "root", True)
        else:
            check(M[i], me, tm, torch.float32, "m")


@pytest.mark.parametrize("bits", [32, 8])
def test_a_tensor_of_more_than_a_table_entry(bits):
    """2^30 elements are one entry of a launch's table: the next ones are as right as the first."""
    import sc_optim
    n = (1 << 30) + 5000
    p, g = torch.full((n,), 0.5, device="cuda", dtype=torch.bfloat16), torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    at = [0, 4097, (1 << 30) - 1, 1 << 30, (1 << 30) + 256, n - 1]
    g[at] = 0.25
    if bits == 32:
        m, v, s = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda"), ()
    else:
        m, v = (torch.zeros(n, device="cuda", dtype=torch.uint8).view(E4M3) for _ in range(2))
        s = tuple([torch.zeros(-(-n // 256), device="cuda")] for _ in range(2))
    sc_optim.adamw_step([p], [g], [m], [v], *s, step=1, lr=0.125, weight_decay=0.0)
    moved = p != 0.5
    assert moved.sum().item() == len(at) and moved[at].all()
    assert torch.equal(p[at].cpu(), torch.full((len(at),), 0.375, dtype=torch.bfloat16))  # the first move is lr
    if bits == 8:
        assert s[0][0].count_nonzero().item() == len({i // 256 for i in at})


def test_a_step_between_forward_and_backward_is_noticed():
    import sc_optim
    p = torch.nn.Parameter(torch.ones(8, device="cuda"))
    opt = sc_optim.AdamW([p], lr=0.1)
    y = (p * p).sum()
    p.grad = torch.ones_like(p)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_a_parameter_given_twice_is_refused():
    import sc_optim
    t = lambda: torch.zeros(300, device="cuda")
    p, e = t(), torch.zeros(0, device="cuda")
    with pytest.raises(RuntimeError, match="twice"):
        sc_optim.adamw_step([p, p], [t(), t()], [t(), t()], [t(), t()], step=1, lr=0.1)
    sc_optim.adamw_step([e, e, p], [e, e, t()], [e, e, t()], [e, e, t()], step=1, lr=0.1)


def test_step_on_the_device_scaler_and_capture():
    import sc_optim
    p0, g0, m0, v0 = tensors([(3000,)], torch.float32, 1)[0]
    mk = lambda: [t.clone().cuda() for t in (p0, m0, v0)]
    g = g0.cuda()
    (p, m, v), (pa, ma, va) = mk(), mk()
    step = torch.tensor([4], dtype=torch.int64, device="cuda")
    for t in (5, 6, 7):
        sc_optim.adamw_step([p], [g], [m], [v], step=step, **H)
        sc_optim.adamw_step([pa], [g], [ma], [va], step=t, **H)
        assert torch.equal(p, pa) and torch.equal(m, ma) and torch.equal(v, va) and step.item() == t
    # a gradient scaler's factor, and a step that is left out
    scale, inf = torch.tensor(1024.0, device="cuda"), torch.zeros(1, device="cuda")
    sc_optim.adamw_step([p], [g * 1024], [m], [v], step=step, grad_scale=scale, found_inf=inf, **H)
    sc_optim.adamw_step([pa], [g], [ma], [va], step=8, **H)
    assert torch.equal(p, pa) and torch.equal(v, va) and step.item() == 8
    inf.fill_(1.0)
    sc_optim.adamw_step([p], [g * float("inf")], [m], [v], step=step, grad_scale=scale, found_inf=inf, **H)
    assert torch.equal(p, pa) and torch.equal(m, ma) and step.item() == 8
    # captured: each replay is the next step
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        sc_optim.adamw_step([p], [g], [m], [v], step=step, **H)
    for t in (9, 10, 11):
        g.normal_().mul_(1e-3)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        sc_optim.adamw_step([pa], [g], [ma], [va], step=t, **H)
        assert torch.equal(p, pa) and torch.equal(m, ma) and torch.equal(v, va) and step.item() == t


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_class_follows_the_function(bits):
    import sc_optim
    torch.manual_seed(0)
    params = [torch.nn.Parameter(torch.randn(s, device="cuda") * 0.1) for s in ((40, 30), (40,), (16, 8, 3, 3))]
    params[2].data = params[2].data.contiguous(memory_format=torch.channels_last)
    twin = [p.detach().clone(memory_format=torch.preserve_format) for p in params]
    opt = sc_optim.AdamW(params, lr=1e-2, weight_decay=0.1, state_bits=bits, clamp=(-1, 0.999))
    if bits == 32:
        M, V, S = [torch.zeros_like(p) for p in twin], [torch.zeros_like(p) for p in twin], ()
    else:
        M, V = ([torch.zeros(p.numel(), dtype=torch.uint8, device="cuda").view(E4M3) for p in twin] for _ in range(2))
        S = tuple([torch.zeros(-(-p.numel() // 256), device="cuda") for p in twin] for _ in range(2))
    for t in range(1, 4):
        for p in params:
            p.grad = torch.randn_like(p)
        sc_optim.adamw_step(twin, [p.grad for p in params], M, V, *S, step=t, lr=1e-2, weight_decay=0.1, clamp=(-1, 0.999))
        opt.step()
        assert all(torch.equal(a.detach(), b) for a, b in zip(params, twin))
    # a reloaded optimiser goes on where the first one was
    copies = [torch.nn.Parameter(p.detach().clone(memory_format=torch.preserve_format)) for p in params]
    again = sc_optim.AdamW(copies, lr=1e-2, weight_decay=0.1, state_bits=bits, clamp=(-1, 0.999))
    again.load_state_dict(opt.state_dict())
    for p, c in zip(params, copies):
        p.grad = torch.randn_like(p)
        c.grad = p.grad.contiguous()  # another layout than a channels-last parameter's
    params[1].grad = copies[1].grad = None  # and one without a gradient
    opt.step(), again.step()
    assert all(torch.equal(a, b) for a, b in zip(params, copies))
    if bits == 8:
        assert opt.state[params[0]]["exp_avg"].dtype == E4M3 and opt.state[params[0]]["exp_avg_scale"].dtype == torch.float32
        assert again.state[copies[0]]["exp_avg"].dtype == E4M3


@pytest.mark.parametrize("bits", [32, 8])
def test_a_group_that_becomes_capturable_and_back_keeps_its_count(bits):
    import sc_optim
    torch.manual_seed(1)
    ps, qs = ([torch.nn.Parameter(torch.ones(n, device="cuda")) for n in (300, 7)] for _ in range(2))
    a, b = (sc_optim.AdamW(v, lr=0.1, state_bits=bits) for v in (ps, qs))
    for capturable in (False, False, True, True, False, False, True):
        a.param_groups[0]["capturable"] = capturable
        for p, q in zip(ps, qs):
            p.grad = torch.randn_like(p)
            q.grad = p.grad.clone()
        a.step(), b.step()
        assert all(torch.equal(p, q) for p, q in zip(ps, qs)), capturable
    assert all(int(a.state[p]["step"]) == 7 for p in ps)


def test_gradient_scaler_leaves_out_a_step_without_a_synchronisation():
    import sc_optim
    p, q = (torch.nn.Parameter(torch.ones(300, device="cuda")) for _ in range(2))
    a, b = sc_optim.AdamW([p], lr=0.1, capturable=True), sc_optim.AdamW([q], lr=0.1, capturable=True)
    scaler = torch.amp.GradScaler("cuda", init_scale=256.0)
    for bad in (False, True, False):
        g = torch.linspace(0.1, 1, 300, device="cuda")
        p.grad = g * scaler.scale(torch.ones(1, device="cuda"))
        if bad:
            p.grad[7] = float("inf")
        else:
            q.grad = g
            b.step()
        scaler.step(a)
        scaler.update()
        assert torch.equal(p, q)
    assert a.state[p]["step"].item() == 2


def test_agrees_with_torch_adamw():
    """Twenty steps beside torch's: both round in float32, some 10 half-steps of each element's move (below lr) a step."""
    import sc_optim
    torch.manual_seed(2)
    p = torch.nn.Parameter(torch.randn(5000, device="cuda") * 0.2)
    q = torch.nn.Parameter(p.detach().clone())
    a, b = sc_optim.AdamW([p], lr=1e-2), torch.optim.AdamW([q], lr=1e-2)
    for _ in range(20):
        p.grad = torch.randn_like(p)
        q.grad = p.grad.clone()
        a.step(), b.step()
    assert (p - q).abs().max().item() <= 20 * (16 * U * 1.0 + 64 * U * 1e-2 * 10)


# ---- stored states, bit for bit -------------------------------------------------------------------
def stored8(t, least):
    """(values, scales) of a float32 tensor of whole blocks as the header defines them: scale = the block's largest
    magnitude times the float32 nearest to 1 / 448, value = the e4m3 number nearest to the float32 quotient.  Quotients
    are taken in 64 bits and rounded to float32, which is the float32 quotient (53 bits are more than 2 x 24 + 2)."""
    b = t.view(-1, 256)
    scale = b.abs().amax(1) * torch.tensor(1.0 / 448, dtype=torch.float32, device=t.device)
    q = (b.double() / torch.where(scale > 0, scale, 1.0).double()[:, None]).float()
    if least:
        q = torch.where(q > 0, q.clamp(min=2.0 ** -9), q)
    return q.clamp(-448, 448).to(E4M3).view(-1), scale


@pytest.mark.parametrize("dt,n,far", [(torch.bfloat16, 1 << 26, 1.0), (torch.float32, (1 << 24) + 256, 1.0), (torch.float32, 1 << 20, 8.0)])
def test_stored_8_bit_states_are_the_definitions(dt, n, far):
    """Two steps in a row: each operation of m = b1 m + (1 - b1) g and v = b2 v + (1 - b2) g^2 is rounded to float32, and
    values and scales are then decided as defined, next to a midpoint of the e4m3 grid too.  A value that went the other
    way there would be its block's largest a step later and take the scale of 256 elements with it."""
    import sc_optim
    print("stored", dt, n, far, flush=True)
    gen = torch.Generator(device="cuda").manual_seed(n)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    size = torch.exp(far * rand(n // 256))
    size[::97] = 0  # blocks that nothing has reached yet
    size = size.repeat_interleave(256)
    f = lambda v: torch.tensor(v, dtype=torch.float32, device="cuda")
    b1, a1, b2, a2 = f(H["beta1"]), f(1 - H["beta1"]), f(H["beta2"]), f(1 - H["beta2"])
    p = (rand(n) * 0.05).to(dt)
    (M, MS), (V, VS) = stored8(rand(n) * 3e-4 * size, False), stored8((rand(n) * 1e-3 * size).abs(), True)
    m, ms, v, vs = M.clone(), MS.clone(), V.clone(), VS.clone()
    for step in (42, 43):
        g = (rand(n) * 1e-3 * size).to(dt)
        sc_optim.adamw_step([p], [g], [M], [V], [MS], [VS], step=step, **H)
        back = lambda q, s: (q.float().view(-1, 256) * s[:, None]).view(-1)
        gf, u = g.float(), back(v, vs)
        m, ms = stored8(back(m, ms) * b1 + gf * a1, False)
        v, vs = stored8(((u * u * b2 + gf * gf * a2).double().sqrt()).float(), True)
        wrong = {name: int((a.float() != b.float()).sum()) for name, a, b in (("m", M, m), ("its scale", MS, ms), ("root", V, v), ("its scale ", VS, vs))}
        assert not any(wrong.values()), (step, wrong)
        assert p.isfinite().all()


@pytest.mark.parametrize("n", [1 << 20, 1001])
def test_32_bit_states_root_and_quotient_are_correctly_rounded(n):
    """With betas, eps and decay 0 and lr 1 a parameter of 0 becomes -g / sqrt(g^2), a handful of operations that are each
    rounded to nearest: 64 bits rounded to float32 are the float32 root and quotient."""
    import sc_optim
    gen = torch.Generator(device="cuda").manual_seed(n)
    m0 = torch.randn(n, generator=gen, device="cuda")
    g = torch.randn(n, generator=gen, device="cuda") * torch.exp(6 * torch.randn(n, generator=gen, device="cuda"))
    p, m, v = torch.zeros(n, device="cuda"), m0.clone(), torch.zeros(n, device="cuda")
    sc_optim.adamw_step([p], [g], [m], [v], step=1, lr=1.0, beta1=0.5, beta2=0.0, eps=0.0, weight_decay=0.0)
    half = torch.tensor(0.5, device="cuda")
    m1, v1 = m0 * half + g * half, g * g
    assert torch.equal(m, m1) and torch.equal(v, v1)
    q = (m1.double() / v1.double().sqrt().float().double()).float()
    assert torch.equal(p, -(q * 2))  # lr / (1 - 1/2)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_reloaded_capturable_optimiser_goes_on_as_the_first_one(bits):
    import sc_optim
    torch.manual_seed(4)
    make = lambda: [torch.nn.Parameter(torch.ones(n, device="cuda")) for n in (300, 7)]
    a, b = (sc_optim.AdamW(make(), lr=0.1, state_bits=bits, capturable=True) for _ in range(2))
    step = lambda which: [opt.step() for opt in (a, b) if set_gradients(opt, which)]

    def set_gradients(opt, which):
        for i, p in enumerate(opt.param_groups[0]["params"]):
            p.grad = grads[i].clone() if i in which else None
        return True

    for which in ((0, 1), (0, 1), (1,), (1,), (0, 1), (0,), (0, 1)):
        grads = [torch.randn(n, device="cuda") for n in (300, 7)]
        step(which)
        fresh = sc_optim.AdamW([torch.nn.Parameter(p.detach().clone()) for p in b.param_groups[0]["params"]], lr=0.1,
                               state_bits=bits, capturable=True)
        if which != (1,):  # else the next step is one of the reloaded optimiser too
            fresh.load_state_dict(b.state_dict())
            b = fresh
        for p, q in zip(a.param_groups[0]["params"], b.param_groups[0]["params"]):
            assert torch.equal(p, q) and a.state[p]["step"].item() == b.state[q]["step"].item(), which


@pytest.mark.parametrize("dt", DTYPES)
def test_stored_8_bit_states_of_odd_lengths_and_a_scaled_gradient(dt):
    """The same behind the last whole chunk, where elements go one by one, and with a gradient scaler's factor, a power of
    two that the gradient takes exactly."""
    import sc_optim
    gen = torch.Generator(device="cuda").manual_seed(9)
    n = 300 * 4096 + 1001
    pad = lambda t: torch.nn.functional.pad(t, (0, -n % 256))
    g = torch.randn(n, generator=gen, device="cuda") * 0.1
    p, g = torch.zeros(n + 1, device="cuda", dtype=dt)[1:], torch.cat([g[:1], g]).to(dt)[1:]
    u8 = lambda: torch.zeros(n + 1, dtype=torch.uint8, device="cuda")[1:].view(E4M3)
    (M, V), (MS, VS) = (u8(), u8()), (torch.zeros(-(-n // 256), device="cuda") for _ in range(2))
    step, scale = torch.tensor([6], dtype=torch.int64, device="cuda"), torch.tensor(64.0, device="cuda")
    sc_optim.adamw_step([p], [g * 64], [M], [V], [MS], [VS], step=step, grad_scale=scale, **H)
    f = lambda v: torch.tensor(v, dtype=torch.float32, device="cuda")
    gf = pad(g.float())
    m, ms = stored8(gf * f(1 - H["beta1"]), False)
    v, vs = stored8((gf * gf * f(1 - H["beta2"])).double().sqrt().float(), True)
    assert torch.equal(M.float(), m[:n].float()) and torch.equal(V.float(), v[:n].float())
    assert torch.equal(MS, ms) and torch.equal(VS, vs) and step.item() == 7
