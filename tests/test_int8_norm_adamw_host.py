"""What the 8-bit linear layer, layer norm and AdamW refuse, and their planning: host code, no GPU."""
import ctypes
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = ctypes.c_void_p(1 << 20)  # an aligned address that is never read: every call below is refused before a launch
ODD = ctypes.c_void_p((1 << 20) + 8)


def _int8(M=4, N=4, K=32, dtype=0, bias=0, weight=0, reserved=0, xs=None, a=32, b=32):
    import _lib
    return _lib.Int8Desc(M, N, K, dtype, bias, weight, reserved, K if xs is None else xs, a, b)


def _error(L):
    return L.rexsc_last_error().decode()


def test_descriptors_mirror_the_header():
    import _lib
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "rexsc.h")).read(), flags=re.S)
    kinds = {"int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "float": ctypes.c_float, "double": ctypes.c_double}
    for name, cls in (("rexsc_int8_desc", _lib.Int8Desc), ("rexsc_norm_desc", _lib.NormDesc), ("rexsc_adamw_desc", _lib.AdamwDesc)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1)
        fields = [(f.strip(), kinds[k]) for k, decl in re.findall(r"(int32_t|int64_t|float|double)([^;]*);", body) for f in decl.split(",")]
        assert fields == list(cls._fields_), name
    body = re.search(r"typedef struct rexsc_adamw_tensor \{(.*?)\} rexsc_adamw_tensor;", text, flags=re.S).group(1)
    assert len(re.findall(r";", body)) == _lib.ADAMW_TENSOR_FIELDS
    assert int(re.search(r"#define REXSC_ADAMW_COEF_BYTES (\d+)", text).group(1)) == _lib.ADAMW_COEF_BYTES


def test_int8_workspace_and_refusals():
    import _lib
    L = _lib.lib()
    none = ctypes.c_size_t(-1).value
    ws = lambda d, what: L.rexsc_int8_workspace_bytes(ctypes.byref(d), what)
    assert ws(_int8(M=1000, K=4096), _lib.INT8_LINEAR) >= 1000 * 4096 + 4000
    # both pieces of g for either gradient, and the transposed operands, in binary16
    assert ws(_int8(M=100, N=50, K=70), _lib.INT8_BACKWARD) >= 2 * (2 * 100 * 64 + 70 * 64 + 2 * 50 * 128 + 70 * 128)
    assert ws(_int8(M=0), _lib.INT8_BACKWARD) == ws(_int8(N=0), _lib.INT8_BACKWARD) == 0
    for d, text in ((_int8(K=0), "K must be"), (_int8(K=131072), "K must be"), (_int8(M=-1), "M -1"), (_int8(dtype=3), "dtypes"),
                    (_int8(bias=-1), "dtypes"), (_int8(weight=9), "dtypes"), (_int8(reserved=1), "reserved")):
        for what in range(3):
            assert ws(d, what) == none and text in _error(L)
    assert ws(_int8(), 3) == none and "number 3" in _error(L)
    d = _int8()
    d.struct_size -= 8
    assert ws(d, 0) == none and "struct_size" in _error(L)


def test_int8_calls_refuse():
    import _lib
    L = _lib.lib()
    product = lambda d, a=FAKE, b=FAKE, sa=FAKE, y=FAKE: L.rexsc_int8_product(ctypes.byref(d), a, sa, b, FAKE, None, y, None, 0, None)
    for d, kw, text in ((_int8(a=24), {}, "tokens"), (_int8(a=16), {}, "tokens"), (_int8(b=40), {}, "channels"),
                        (_int8(), {"a": ODD}, "tokens"), (_int8(), {"b": ODD}, "channels"), (_int8(), {"a": None}, "null"),
                        (_int8(), {"sa": None}, "null"), (_int8(), {"y": None}, "null")):
        assert product(d, **kw) == -1 and text in _error(L), text
    assert product(_int8(M=0), a=None, b=None) == 0 and product(_int8(N=0), a=None) == 0  # nothing to do
    linear = lambda d, x=FAKE, ws=None, n=0: L.rexsc_int8_linear(ctypes.byref(d), x, FAKE, FAKE, None, FAKE, ws, n, None)
    big = _int8(M=1000, K=32)
    need = L.rexsc_int8_workspace_bytes(ctypes.byref(big), _lib.INT8_LINEAR)
    assert linear(big) == -2 and "workspace" in _error(L)
    assert linear(big, ws=FAKE, n=need - 1) == -2
    assert linear(big, ws=ODD, n=need) == -1 and "16-byte" in _error(L)
    assert linear(_int8(xs=31)) == -1 and "overlap" in _error(L)
    assert linear(_int8(), x=ctypes.c_void_p(3)) == -1 and "aligned" in _error(L)
    back = lambda d, g=FAKE, a=FAKE, b=FAKE, dx=FAKE, dw=FAKE, db=FAKE, ws=None, n=0: L.rexsc_int8_backward(
        ctypes.byref(d), g, a, FAKE, b, FAKE, dx, dw, db, ws, n, None)
    assert back(_int8()) == -2 and "workspace" in _error(L)
    for d, kw, text in ((_int8(a=40), {}, "tokens"), (_int8(b=16), {}, "channels"), (_int8(), {"a": ODD}, "tokens"),
                        (_int8(), {"b": None}, "null"), (_int8(), {"g": None}, "null"), (_int8(), {"g": ctypes.c_void_p(2)}, "aligned"),
                        (_int8(M=4194304, N=1), {}, "at most")):
        need = L.rexsc_int8_workspace_bytes(ctypes.byref(d), _lib.INT8_BACKWARD)
        assert back(d, ws=FAKE, n=need, **kw) == -1 and text in _error(L), text
    # what a gradient does not read is not checked; none wanted, or empty: nothing to do
    assert back(_int8(a=40), dw=None) == -2 and back(_int8(b=16), dx=None) == -2
    assert back(_int8(), dx=None, dw=None, db=None) == 0 and back(_int8(M=0, N=0)) == 0
    q = lambda rows, cols, stride, out=FAKE, x=FAKE, dt=0: L.rexsc_quantize_rows(x, dt, rows, cols, cols, out, stride, FAKE, None)
    assert q(0, 4, 16) == 0
    for args, text in (((2, 0, 16), "elements"), ((2, 20, 16), "int8 rows"), ((2, 20, 24), "int8 rows"), ((2, 4, 16, ODD), "int8 rows"),
                       ((2, 4, 16, None), "null"), ((2, 4, 16, FAKE, ctypes.c_void_p(2)), "aligned"),
                       ((2, 4, 16, FAKE, FAKE, 5), "dtype")):
        assert q(*args) == -1 and text in _error(L), text


def test_layer_norm_refusals():
    import _lib
    L = _lib.lib()
    D = lambda dt=0, wdt=0, eps=1e-5, rows=4, cols=8, xs=8: _lib.NormDesc(dt, wdt, eps, rows, cols, xs)
    fwd = lambda d, x=FAKE, y=FAKE, m=FAKE, r=FAKE: L.rexsc_layer_norm_forward(ctypes.byref(d), x, FAKE, FAKE, y, m, r, None)
    for d, kw, text in ((D(dt=3), {}, "dtype"), (D(dt=1, wdt=2), {}, "weight and bias"), (D(eps=-1.0), {}, "eps"),
                        (D(eps=float("nan")), {}, "eps"), (D(rows=-1), {}, "rows"), (D(cols=0), {}, "rows"),
                        (D(xs=7), {}, "distance"), (D(), {"x": None}, "null"), (D(), {"r": None}, "together"),
                        (D(), {"x": ctypes.c_void_p(6)}, "aligned")):
        assert fwd(d, **kw) == -1 and text in _error(L), text
    assert fwd(D(rows=0), x=None, y=None) == 0
    bytes_ = L.rexsc_layer_norm_backward_workspace_bytes
    many = D(rows=513)  # up to 512 short rows need no partial sums
    assert bytes_(ctypes.byref(many)) >= 2 * 8 * 4 and bytes_(ctypes.byref(D())) == 0
    assert bytes_(ctypes.byref(D(cols=2049, xs=2049))) >= 2 * 2049 * 4
    assert bytes_(ctypes.byref(D(cols=0))) == ctypes.c_size_t(-1).value
    bwd = lambda d, g=FAKE, dx=FAKE, dw=FAKE, ws=None, n=0: L.rexsc_layer_norm_backward(
        ctypes.byref(d), g, FAKE, FAKE, FAKE, FAKE, dx, dw, None, ws, n, None)
    assert bwd(many) == -2 and "workspace" in _error(L)
    assert bwd(D(), g=None) == -1 and "null" in _error(L)
    assert bwd(D(), dx=None, dw=None) == 0


def test_adamw_refusals():
    import _lib
    L = _lib.lib()
    T = lambda p=1 << 20, g=1 << 20, m=1 << 20, v=1 << 20, ms=0, vs=0, n=10: (p, g, m, v, ms, vs, n)
    D = lambda dt=0, bits=32, clamp=0, lr=1e-3, b1=0.9, b2=0.99, eps=1e-8, wd=0.0, lo=0.0, hi=0.0, step=1: _lib.AdamwDesc(
        dt, bits, clamp, lr, b1, b2, eps, wd, lo, hi, step)

    def call(d, t, step=None, scale=None, inf=None, coef=None):
        arr = (ctypes.c_int64 * 7)(*t)
        return L.rexsc_adamw_step(ctypes.byref(d), ctypes.cast(arr, ctypes.c_void_p), 1, step, scale, inf, coef, None)

    for d, t, kw, text in ((D(dt=4), T(), {}, "dtype"), (D(bits=16), T(), {}, "32 or 8"), (D(b1=1.0), T(), {}, "betas"),
                           (D(b2=-0.1), T(), {}, "betas"), (D(lr=-1.0), T(), {}, "negative"), (D(eps=float("nan")), T(), {}, "negative"),
                           (D(clamp=1, lo=1.0, hi=0.0), T(), {}, "clamp"), (D(step=0), T(), {}, "counts from 1"),
                           (D(), T(), {"step": FAKE}, "workspace"), (D(), T(), {"scale": FAKE}, "need the step"),
                           (D(), T(), {"inf": FAKE}, "need the step"), (D(), T(n=-1), {}, "elements"), (D(), T(g=0), {}, "null"),
                           (D(), T(m=0), {}, "null"), (D(bits=8), T(), {}, "scales"), (D(), T(p=(1 << 20) + 2), {}, "aligned"),
                           (D(), T(v=(1 << 20) + 1), {}, "aligned")):
        assert call(d, t, **kw) == -1 and text in _error(L), text
    assert call(D(), T(p=0, g=0, m=0, v=0, n=0)) == 0  # a tensor without elements


def test_python_checks_need_no_gpu():
    import _ops
    import sc_functional as F
    import sc_layers
    import sc_optim
    x, w = torch.randn(3, 8), torch.randn(4, 8)
    with pytest.raises(RuntimeError, match="HIP device"):
        F.linear_int8(x, w)
    with pytest.raises(RuntimeError, match="HIP device"):
        F.layer_norm(x)
    with pytest.raises(RuntimeError, match="HIP device"):
        F.quantize_rows(x)
    with pytest.raises(RuntimeError, match="HIP device"):
        sc_optim.adamw_step([x], [x], [x], [x], step=1, lr=1e-3)
    with pytest.raises(ValueError, match="weight_scale"):
        F.linear_int8(x, w.to(torch.int8))
    with pytest.raises(ValueError, match="weight_scale"):
        F.linear_int8(x, w, weight_scale=torch.ones(4))
    with pytest.raises(ValueError, match="expected input"):
        F.linear_int8(x, torch.randn(4, 9))
    for t in (torch.zeros(2, 3), torch.zeros(2, 0, dtype=torch.int8), torch.zeros(6, dtype=torch.int8),
              torch.zeros(1, 131072, dtype=torch.int8)):
        with pytest.raises(RuntimeError, match="int8 matrix"):
            _ops._operand8(t, "matmul_int8")
    with pytest.raises(RuntimeError, match="scales"):
        _ops._scale_vector(torch.ones(3), 4, torch.device("cpu"), "x")
    with pytest.raises(RuntimeError, match="bias"):
        _ops._bias_vector(torch.ones(3, 1), 3, "x")
    for kw in ({"state_bits": 16}, {"lr": -1}, {"betas": (1.0, 0.9)}, {"clamp": (1, 0)}, {"eps": float("nan")}):
        with pytest.raises(ValueError):
            sc_optim.AdamW([torch.nn.Parameter(x)], **kw)
    with pytest.raises(RuntimeError, match="lengths"):
        sc_optim.adamw_step([x], [], [x], [x], step=1, lr=1e-3)
    with pytest.raises(RuntimeError, match="both lists"):
        sc_optim.adamw_step([x], [x], [x], [x], [x], step=1, lr=1e-3)
    layer = sc_layers.Linear_Int8(8, 4)
    assert not layer.frozen and set(layer.state_dict()) == {"weight", "bias"}


def test_operand_layouts():
    """Which int8 tensors are read in place: rows 16-byte aligned and readable to the next multiple of 16."""
    import _ops
    whole = torch.zeros(10, 64, dtype=torch.int8)
    for t, kept in ((whole, True), (whole[:, :50], True), (whole[:, 16:40], True), (whole[2:, 5:30], False), (whole[::2], True),
                    (whole.t(), False), (torch.zeros(4, 30, dtype=torch.int8), False), (whole[:1, :30], True),
                    (torch.zeros(1, 30, dtype=torch.int8), False), (torch.zeros(46, dtype=torch.int8).as_strided((3, 14), (16, 1)), False)):
        got, stride = _ops._operand8(t, "x")
        assert (got.data_ptr() == t.data_ptr()) == kept and torch.equal(got, t) and stride % 16 == 0 and stride >= t.shape[1]
    import sc_optim
    d = sc_optim._dense
    assert d(torch.zeros(3, 4)) and d(torch.zeros(3, 4).t()) and d(torch.zeros(2, 3, 4, 5).contiguous(memory_format=torch.channels_last))
    assert not d(torch.zeros(3, 8)[:, :4]) and not d(torch.zeros(1, 4).expand(3, 4)) and d(torch.zeros(0, 4))


def test_a_reloaded_capturable_optimiser_has_one_step_count(monkeypatch):
    """Every parameter of a capturable group, with a gradient at the moment or without, counts the same steps after a
    reload, after a change of `capturable`, and when it joins late.  (The kernel's part, advancing a device count, is
    done by the test.)"""
    import sc_optim

    def advance(params, *lists, step, **rest):
        if isinstance(step, torch.Tensor):
            step += 1
        seen.append(int(step))

    seen = []
    monkeypatch.setattr(sc_optim, "adamw_step", advance)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    make = lambda: [torch.nn.Parameter(torch.ones(3)) for _ in range(3)]

    def step(opt, which):
        for i, p in enumerate(opt.param_groups[0]["params"]):
            p.grad = torch.ones(3) if i in which else None
        opt.step()

    first = sc_optim.AdamW(make(), capturable=True)
    for _ in range(5):
        step(first, (0, 1))
    again = sc_optim.AdamW(make(), capturable=True)
    again.load_state_dict(first.state_dict())
    for which in ((1,), (1,), (1,), (0, 1), (0, 1, 2), (2,), (0,)):
        step(again, which)
    assert seen == [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12]
    counts = [again.state[p]["step"] for p in again.param_groups[0]["params"]]
    assert all(c is counts[0] for c in counts) and int(first.state[first.param_groups[0]["params"][0]]["step"]) == 5
    # a count on the host becomes the group's: parameters without a gradient at that moment count on too
    seen.clear()
    late = sc_optim.AdamW(make(), capturable=False)
    for _ in range(4):
        step(late, (0, 1, 2))
    late.param_groups[0]["capturable"] = True
    for which in ((1,), (1,), (0, 1, 2)):
        step(late, which)
    assert seen == [1, 2, 3, 4, 5, 6, 7]


def test_forward_mode_derivatives_are_refused():
    """A dual tensor need not require a gradient: its tangent must not be dropped without a word, whichever argument it
    is and whether or not another one requires a gradient.  Tensors without a tangent go on to the kernel (refused here
    for want of a device)."""
    import torch.autograd.forward_ad as fw
    import sc_functional as F
    import sc_layers
    x, v, w = torch.randn(3, 8), torch.randn(8), torch.randn(4, 8)
    q, s = torch.zeros(4, 8, dtype=torch.int8), torch.ones(4)
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))
        frozen = sc_layers.Linear_Int8(8, 4)
        frozen.weight_q, frozen.weight_scale, frozen.weight = torch.zeros(4, 128, dtype=torch.int8), s, None
        for leaf in (False, True):
            g = v.clone().requires_grad_(leaf)
            for call in (lambda: F.layer_norm(dual(x), g), lambda: F.layer_norm(x, g, dual(v)), lambda: F.layer_norm(x, dual(v), g),
                         lambda: F.linear_int8(dual(x), w), lambda: F.linear_int8(x, dual(w)), lambda: F.linear_int8(x, w, dual(s)),
                         lambda: F.linear_int8(dual(x), q, weight_scale=s), lambda: F.linear_int8(x, q, weight_scale=dual(s)),
                         lambda: sc_layers.LayerNorm(8)(dual(x)), lambda: frozen(dual(x))):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call()
        for call in (lambda: F.layer_norm(x), lambda: F.linear_int8(x, q, weight_scale=s)):
            with pytest.raises(RuntimeError, match="HIP device"):
                call()


def test_rows_far_apart_are_copied():
    """The tiled product reaches rows less than 8 MiB apart: whether a layout works must not depend on the tokens' number."""
    import _ops
    far = torch.arange((8 << 20) + 64, dtype=torch.int64).to(torch.int8).as_strided((2, 48), (8 << 20, 1))
    got, stride = _ops._operand8(far, "x")
    assert torch.equal(got, far) and stride == 128 and got.data_ptr() != far.data_ptr()
    near = torch.zeros((8 << 20) + 64, dtype=torch.int8).as_strided((2, 48), ((8 << 20) - 16, 1))
    assert _ops._operand8(near, "x")[0].data_ptr() == near.data_ptr()


def test_backward_workspace_holds_what_is_wanted():
    import _lib
    L = _lib.lib()
    none = ctypes.c_size_t(-1).value
    ws = lambda d, wanted: L.rexsc_int8_backward_workspace_bytes(ctypes.byref(d), wanted)
    DX, DW, DB = _lib.INT8_DX, _lib.INT8_DW, _lib.INT8_DB
    d = _int8(M=8192, N=4096, K=4096, a=4096, b=4096)
    # both pieces of g for a gradient, and its other operand transposed, in binary16, and little beside them
    dx, dw = 2 * (2 * 8192 * 4096 + 4096 * 4096), 2 * (2 * 4096 * 8192 + 4096 * 8192)
    assert dx <= ws(d, DX) <= dx + (1 << 17) and dw <= ws(d, DW) <= dw + (1 << 20) and ws(d, DB) <= 1 << 20
    assert ws(d, DX | DW | DB) == L.rexsc_int8_workspace_bytes(ctypes.byref(d), _lib.INT8_BACKWARD) >= dx + dw
    assert ws(d, 0) == ws(_int8(M=0), DX) == ws(_int8(N=0), DW | DB) == 0 and ws(d, 8) == none and "flags 8" in _error(L)
    # a workspace of that size is enough for such a call, and one byte less is not
    back = lambda d, n, dx, dw, db: L.rexsc_int8_backward(ctypes.byref(d), FAKE, FAKE, FAKE, FAKE, FAKE, dx, dw, db, FAKE, n, None)
    for wanted in range(1, 8):
        assert back(d, ws(d, wanted) - 1, *(FAKE if wanted & f else None for f in (DX, DW, DB))) == -2, wanted
    # more tokens than the weight's gradient sums over, and more channels than the input's: refused for that one alone
    for d, no, yes in ((_int8(M=5000000, N=10), DW, DX | DB), (_int8(M=10, N=5000000), DX, DW | DB)):
        assert ws(d, no) == none and "at most" in _error(L)
        assert 0 < ws(d, yes) < none


def test_sizes_at_the_end_of_32_bits():
    import _lib
    L = _lib.lib()
    none = ctypes.c_size_t(-1).value
    for kw in ({"M": 2 ** 31 - 1}, {"N": 2 ** 31 - 1}, {"M": 2 ** 31 - 255}):
        for what in range(3):
            assert L.rexsc_int8_workspace_bytes(ctypes.byref(_int8(**kw)), what) == none and "int8 linear: M " in _error(L)
    assert L.rexsc_int8_workspace_bytes(ctypes.byref(_int8(M=2 ** 31 - 256)), _lib.INT8_LINEAR) >= (2 ** 31 - 256) * 132
    with pytest.raises(RuntimeError, match="does not fit"):
        _lib.Int8Desc.packed(2 ** 31, 4, 32, 0, 0, 0, 0, 32, 32, 32)


def test_states_of_another_layout(monkeypatch):
    """A parameter whose memory order changes after its states were made, or that loads those of another order: 32-bit
    states follow it, 8-bit ones, whose blocks run along the memory, cannot and are refused."""
    import sc_optim
    seen = []
    monkeypatch.setattr(sc_optim, "adamw_step", lambda params, grads, m, v, *rest, **kw: seen.append((params, m, v)))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    shape = (6, 5, 3, 3)
    last = lambda t: t.contiguous(memory_format=torch.channels_last)

    def optimiser(bits, make):
        p = torch.nn.Parameter(make(torch.randn(shape)))
        p.grad = torch.randn_like(p)
        return p, sc_optim.AdamW([p], state_bits=bits)

    for bits in (32, 8):
        for a, b in ((last, torch.Tensor.contiguous), (torch.Tensor.contiguous, last)):
            p, first = optimiser(bits, a)
            first.step()
            q, again = optimiser(bits, b)
            if bits == 32:
                first.state[p]["exp_avg"].copy_(torch.randn(shape))
                again.load_state_dict(first.state_dict())
                again.step()
                state = again.state[q]["exp_avg"]
                assert state.stride() == q.stride() and torch.equal(state, first.state[p]["exp_avg"])
                p.data = b(p.data)  # and without a reload
                before = first.state[p]["exp_avg"].clone()
                first.step()
                assert first.state[p]["exp_avg"].stride() == p.stride() and torch.equal(first.state[p]["exp_avg"], before)
            else:
                again.load_state_dict(first.state_dict())
                for opt, t in ((again, q), (first, p)):
                    t.data = b(t.data)
                    with pytest.raises(RuntimeError, match="layout"):
                        opt.step()
                q.data = a(q.data)
                again.step()
    # dimensions of one element have no layout
    p = torch.nn.Parameter(last(torch.randn(8, 4, 1, 1)))
    p.grad = torch.randn_like(p)
    opt = sc_optim.AdamW([p], state_bits=8)
    opt.step()
    p.data = p.data.contiguous()
    opt.step()


def test_a_capturable_state_loads_without_a_device():
    import sc_optim
    make = lambda: sc_optim.AdamW([torch.nn.Parameter(torch.ones(n)) for n in (3, 4)], capturable=True)
    opt = make()
    step = torch.tensor([7])
    for p in opt.param_groups[0]["params"]:
        opt.state[p] = {**opt._new_state(p, opt.param_groups[0]), "step": step}
    again = make()
    again.load_state_dict(opt.state_dict())
    a, b = (again.state[p]["step"] for p in again.param_groups[0]["params"])
    assert a is b and a is not step and a.item() == 7 and a.dtype == torch.int64


def test_a_captured_step_after_loading_states_that_differ_in_dimensions_of_one_element(monkeypatch):
    import sc_optim
    seen = []
    monkeypatch.setattr(sc_optim, "adamw_step", lambda params, *rest, **kw: seen.append(params))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    p = torch.nn.Parameter(torch.randn(8, 4, 1, 1))
    p.grad = torch.randn_like(p)
    opt = sc_optim.AdamW([p], capturable=True)
    last = lambda: torch.zeros(8, 4, 1, 1).as_strided((8, 4, 1, 1), (4, 1, 4, 4))
    opt.state[p] = {"exp_avg": last(), "exp_avg_sq": last(), "step": torch.tensor([1])}
    opt.step()
    assert len(seen) == 1
