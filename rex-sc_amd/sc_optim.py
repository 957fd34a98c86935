"""AdamW over many tensors at once on the HIP kernels, with 32-bit or 8-bit states and the clamp of the weights that SC
training applies after every step (utils_own.py:187-190) folded into it."""
import array
import itertools
import operator

import torch

import _lib
import _ops

BLOCK = 256  # elements of an 8-bit state that share a scale
E4M3 = torch.float8_e4m3fn


def _dense(t):
    """Whether t's elements fill one block of memory, in whatever order of the dimensions."""
    if t.is_contiguous():
        return True
    at = 1
    for n, s in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n > 1), key=lambda v: v[1]):
        if s != at:
            return False
        at *= n
    return True


def _memory_order(shape, stride):
    """What tells two orders of a dense tensor's elements in memory apart: its dimensions with their strides, or None for
    row by row, however the shape is cut."""
    kept = [(n, s) for n, s in zip(shape, stride) if n > 1]
    at = 1
    for n, s in reversed(kept):
        if s != at:
            return kept
        at *= n
    return None


_T = torch.Tensor
_PTR, _NUMEL, _DENSE, _DEV = _T.data_ptr, _T.numel, _T.is_contiguous, _T.get_device
_DTYPE = operator.attrgetter("dtype")


def _check_list(tensors, what, params, dtype, device, numels):
    """All of one type, on one device and as long as the parameters (one pass in C per property: a step of a network
    with many small tensors is bound by this)."""
    if not (set(map(_DTYPE, tensors)) == {dtype} and set(map(_DEV, tensors)) == {device} and list(map(_NUMEL, tensors)) == numels):
        for p, t, n in zip(params, tensors, numels):
            if t.dtype != dtype or t.get_device() != device or t.numel() != n:
                raise RuntimeError("adamw_step: %s of a %s %s parameter on %s must be %s, of %d elements and beside it (got %s %s "
                                   "on %s)" % (what, tuple(p.shape), p.dtype, p.device, dtype, n, t.dtype, tuple(t.shape), t.device))


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales=None, exp_avg_sq_scales=None, *, step, lr, beta1=0.9,
               beta2=0.999, eps=1e-8, weight_decay=1e-2, clamp=None, grad_scale=None, found_inf=None):
    """One AdamW step of all `params` in place: one launch for up to 96 tensors (64 with 8-bit states).

    params, grads: lists of tensors of one type (float32, float16, bfloat16) on one device, each dense in memory and the
    gradient laid out like its parameter.  exp_avgs, exp_avg_sqs: float32 states laid out likewise, or, with the two
    lists of scales, 8-bit ones: float8_e4m3fn tensors of m / scale and sqrt(v) / scale, one float32 scale for each 256
    elements in memory order.  The tensors of a call do not overlap, and a captured call keeps to theirs.  step: the
    number of this step, from 1 on; or a device int64 tensor that holds the steps taken, which the call advances on the
    stream (a captured call needs that).  clamp: (lo, hi) of the updated parameter.  grad_scale, found_inf: float32
    device tensors of a gradient scaler, with a device step: gradients are divided by the one, and where the other is
    not 0 the step is left out."""
    eight = exp_avg_scales is not None
    lists = [params, grads, exp_avgs, exp_avg_sqs]
    if eight != (exp_avg_sq_scales is not None):
        raise RuntimeError("adamw_step: 8-bit states come with both lists of scales")
    if eight:
        lists += [exp_avg_scales, exp_avg_sq_scales]
    if any(len(v) != len(params) for v in lists):
        raise RuntimeError("adamw_step: lists of different lengths (%s)" % ", ".join(str(len(v)) for v in lists))
    if not params:
        return
    first = params[0]
    if not first.is_cuda:
        _ops._require_cuda(first)
    code = _ops._dtype_code(first, "adamw_step")
    state, dev = E4M3 if eight else torch.float32, first.get_device()
    numels = list(map(_NUMEL, params))
    _check_list(params, "each parameter, as the first", params, first.dtype, dev, numels)
    _check_list(grads, "the gradient", params, first.dtype, dev, numels)
    _check_list(exp_avgs, "exp_avg", params, state, dev, numels)
    _check_list(exp_avg_sqs, "exp_avg_sq", params, state, dev, numels)
    if not (all(map(_DENSE, params)) and all(map(_DENSE, grads)) and all(map(_DENSE, exp_avgs)) and all(map(_DENSE, exp_avg_sqs))):
        for p, g, m, v in zip(params, grads, exp_avgs, exp_avg_sqs):
            if p.is_contiguous() and g.is_contiguous() and m.is_contiguous() and v.is_contiguous():
                continue
            same = p.stride() == g.stride() and (m.is_contiguous() and v.is_contiguous() if eight else
                                                 p.stride() == m.stride() == v.stride())
            if not (same and _dense(p)):
                raise RuntimeError("adamw_step: a parameter, its gradient and its states must be dense and laid out alike "
                                   "(strides %s, %s, %s, %s)" % (p.stride(), g.stride(), m.stride(), v.stride()))
    where = list(map(_PTR, params))
    if len(set(where)) != len(where) and len({a for a, n in zip(where, numels) if n}) != sum(map(bool, numels)):
        raise RuntimeError("adamw_step: a parameter is given twice")
    columns = [where, map(_PTR, grads), map(_PTR, exp_avgs), map(_PTR, exp_avg_sqs)]
    if eight:
        blocks = [-(-n // BLOCK) for n in numels]
        for scales, what in ((exp_avg_scales, "exp_avg_scale"), (exp_avg_sq_scales, "exp_avg_sq_scale")):
            _check_list(scales, what, params, torch.float32, dev, blocks)
            if not all(map(_DENSE, scales)):
                raise RuntimeError("adamw_step: the scales of a state must be contiguous")
        columns += [map(_PTR, exp_avg_scales), map(_PTR, exp_avg_sq_scales)]
    else:
        columns += [itertools.repeat(0), itertools.repeat(0)]
    table = array.array("q", itertools.chain.from_iterable(zip(*columns, numels)))
    on_device = isinstance(step, torch.Tensor)
    if on_device and (step.dtype != torch.int64 or step.numel() != 1 or step.device != first.device):
        raise RuntimeError("adamw_step: a step held in a tensor is one int64 beside the parameters")
    if not on_device and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("adamw_step: a captured step needs its number in a device tensor (a number would be frozen)")
    for name, t in (("grad_scale", grad_scale), ("found_inf", found_inf)):
        if t is not None and (not on_device or t.dtype != torch.float32 or t.numel() != 1 or t.device != first.device):
            raise RuntimeError("adamw_step: %s is one float32 beside the parameters, and needs the step in a tensor" % name)
    lo, hi = (0.0, 0.0) if clamp is None else (float(clamp[0]), float(clamp[1]))
    d = _lib.AdamwDesc.packed(code, 8 if eight else 32, int(clamp is not None), float(lr), float(beta1), float(beta2), float(eps),
                       float(weight_decay), lo, hi, 0 if on_device else int(step))
    with _ops._on(dev):
        coef = torch.empty(_lib.ADAMW_COEF_BYTES, dtype=torch.uint8, device=first.device) if on_device else None
        rc = _lib.lib().rexsc_adamw_step(d, table.buffer_info()[0], len(params),
                                         _ops._addr(step if on_device else None), _ops._addr(grad_scale),
                                         _ops._addr(found_inf), _ops._addr(coef), _ops._raw_stream(dev))
        if rc:
            _lib.check(rc, "rexsc_adamw_step")
    # for autograd's check of tensors changed between a forward and its backward pass
    torch.autograd.graph.increment_version(params)


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's update on adamw_step: parameters may be float32, float16 or bfloat16, dense in memory.

    state_bits: 32, or 8 for float8_e4m3fn states with a scale for each 256 elements (2 bytes of state per parameter in
    place of 8).  clamp: (lo, hi) that every parameter of the group is held to, (-1, 0.999) for SC weights.
    capturable: the step number lives on the device, one for all parameters of a group that have a gradient; needed
    under graph capture, and what torch.amp.GradScaler needs to leave out a step without a host synchronisation (its
    scale is then applied inside the step).  Hyperparameters are frozen into a captured step."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, clamp=None,
                 capturable=False):
        if state_bits not in (8, 32):
            raise ValueError("AdamW: state_bits must be 32 or 8 (got %r)" % (state_bits,))
        if not (lr >= 0 and eps >= 0 and weight_decay >= 0 and all(0 <= b < 1 for b in betas)):
            raise ValueError("AdamW: lr, eps and weight_decay must not be negative and betas in [0, 1) (got %r, %r, %r, %r)"
                             % (lr, eps, weight_decay, betas))
        if clamp is not None and not clamp[0] <= clamp[1]:
            raise ValueError("AdamW: clamp to (%r, %r)" % tuple(clamp))
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      clamp=clamp, capturable=capturable))

    @property
    def _step_supports_amp_scaling(self):  # torch.amp.GradScaler asks for it and then sets grad_scale and found_inf
        return all(g["capturable"] for g in self.param_groups)

    def _new_state(self, p, group):
        if not _dense(p):
            raise RuntimeError("AdamW: a parameter of strides %s is not dense in memory" % (p.stride(),))
        if group["state_bits"] == 32:
            zeros = lambda: torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
            return {"exp_avg": zeros(), "exp_avg_sq": zeros()}
        zeros = lambda: torch.zeros(p.numel(), dtype=torch.uint8, device=p.device).view(E4M3)
        scale = lambda: torch.zeros(-(-p.numel() // BLOCK), dtype=torch.float32, device=p.device)
        return {"exp_avg": zeros(), "exp_avg_sq": zeros(), "exp_avg_scale": scale(), "exp_avg_sq_scale": scale(),
                "layout": (tuple(p.shape), p.stride())}

    def _follow(self, p, state):
        """Brings the states of a parameter that lies otherwise in memory than when they were made, or than the one whose
        states were loaded, into its order."""
        if "exp_avg_scale" in state:
            now = (tuple(p.shape), p.stride())
            if "layout" in state and _memory_order(*state["layout"]) != _memory_order(*now):
                raise RuntimeError("AdamW: 8-bit states lie in blocks along the memory of a parameter of layout %s, this one's is "
                                   "%s (shape, strides)" % (state["layout"], now))
            state["layout"] = now
        elif state["exp_avg"].shape == p.shape and _dense(p):  # (else adamw_step refuses them)
            if torch.cuda.is_current_stream_capturing():
                if p.is_contiguous() and state["exp_avg"].is_contiguous():  # dimensions of one element apart
                    return
                raise RuntimeError("AdamW: a parameter whose layout has changed needs an eager step before a captured one")
            for k in ("exp_avg", "exp_avg_sq"):
                state[k] = torch.empty_like(p, dtype=torch.float32, memory_format=torch.preserve_format).copy_(state[k])

    def load_state_dict(self, state_dict):
        # torch casts a state to its parameter's type on loading: 8-bit states and their scales keep their own
        super().load_state_dict(state_dict)
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        ours = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(ids, ours):
            for k, v in state_dict["state"].get(i, {}).items():
                if isinstance(v, torch.Tensor):
                    self.state[p][k] = v.to(device=p.device, copy=True)
        for group in self.param_groups:  # each parameter has a copy of the count now: one for all again
            if group["capturable"]:
                for key in {(p.dtype, p.device) for p in group["params"]}:
                    self._share_step(group, key)

    def _share_step(self, group, key):
        """The step count that the parameters of `group` with this type and device share on the device, held by every
        state there is from now on, also of those that have no gradient at the moment."""
        states = [self.state[p] for p in group["params"] if (p.dtype, p.device) == key and self.state.get(p)]
        held = [s["step"] for s in states if "step" in s]
        if held and isinstance(held[0], torch.Tensor) and all(t is held[0] for t in held):
            step = held[0]
        else:  # the first step, a loaded state, or a group that was not capturable before
            if held and key[1].type == "cuda" and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AdamW: a group that becomes capturable needs an eager step before a captured one")
            step = torch.full((1,), max(map(int, held), default=0), dtype=torch.int64, device=key[1])
        for s in states:
            s["step"] = step
        return step

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        grad_scale, found_inf = getattr(self, "grad_scale", None), getattr(self, "found_inf", None)
        for group in self.param_groups:
            sets = {}  # tensors that go into one call: one type, device and step number
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("AdamW: sparse gradients are not supported")
                state = self.state[p]
                if not state:
                    if torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("AdamW: every parameter needs one eager step before a step is captured (its "
                                           "state would be cleared on every replay)")
                    state.update(self._new_state(p, group))
                    if not group["capturable"]:
                        state["step"] = 0
                elif p.stride() != (state["layout"][1] if "layout" in state else state["exp_avg"].stride()):
                    self._follow(p, state)
                if group["capturable"]:
                    key = (p.dtype, p.device)
                else:
                    state["step"] = int(state["step"]) + 1  # (a tensor's where the group was capturable before)
                    key = (p.dtype, p.device, state["step"])
                sets.setdefault(key, []).append((p, state))
            for key, members in sets.items():
                if group["capturable"]:
                    step = members[0][1].get("step")
                    if not isinstance(step, torch.Tensor) or any(s.get("step") is not step for _, s in members):
                        step = self._share_step(group, key)
                else:
                    step = key[2]
                grads = [p.grad if p.grad.stride() == p.stride() else torch.empty_like(p).copy_(p.grad) for p, _ in members]
                col = lambda name: [s[name] for _, s in members]
                eight = group["state_bits"] == 8
                adamw_step([p for p, _ in members], grads, col("exp_avg"), col("exp_avg_sq"),
                           col("exp_avg_scale") if eight else None, col("exp_avg_sq_scale") if eight else None, step=step,
                           lr=group["lr"], beta1=group["betas"][0], beta2=group["betas"][1], eps=group["eps"],
                           weight_decay=group["weight_decay"], clamp=group["clamp"],
                           grad_scale=grad_scale if group["capturable"] else None,
                           found_inf=found_inf if group["capturable"] else None)
        return loss
