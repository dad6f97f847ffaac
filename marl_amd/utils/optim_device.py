"""Host side of the optimiser kernels (include/marl_amd.h).

ec_adam_clip_step: `clip_grad_norm_` + `Adam.step()` of up to four small networks in one launch.  The optimiser objects stay
the owners of their state (exp_avg, exp_avg_sq, step), so state_dicts and checkpoints are torch's; the kernel updates those
tensors in place.

ec_grad_clip_coef, ec_adamw_step: AdamW over any number of tensors of any size, moments in 32 or 8 bits (`AdamW`, and
`clip_coef` / `adamw_step` on lists of tensors)."""
import array
import ctypes as C
import operator

import torch as th

from marl_amd import _abi
from marl_amd.utils.norm_device import DTYPES, launch, ptr

MAX_NETS, MAX_TENSORS = 4, 16


def _eligible(opt):
    if type(opt) is not th.optim.Adam or len(opt.param_groups) != 1:
        return False
    g = opt.param_groups[0]
    if g.get("weight_decay", 0) != 0 or g.get("amsgrad", False) or g.get("maximize", False) or g.get("differentiable", False):
        return False
    ps = g["params"]
    if not 1 <= len(ps) <= MAX_TENSORS:
        return False
    for p in ps:
        if (not p.is_cuda or p.dtype != th.float32 or not p.is_contiguous() or p.grad is None or not p.grad.is_contiguous()
                or p.grad.dtype != th.float32 or p.grad.is_sparse):
            return False
    return True


def _state(opt, p):
    st = opt.state[p]
    if len(st) == 0:  # as Adam._init_group does
        capturable = opt.param_groups[0].get("capturable", False)
        st["step"] = (th.zeros((), dtype=th.float32, device=p.device) if capturable else th.tensor(0.0, dtype=th.float32))
        st["exp_avg"] = th.zeros_like(p, memory_format=th.preserve_format)
        st["exp_avg_sq"] = th.zeros_like(p, memory_format=th.preserve_format)
    return st


def clip_adam_step(optimizers, max_norm):
    """clip_grad_norm_(params of optimizers[i], max_norm) and optimizers[i].step() for every i, in one launch.
    max_norm: one number for all, or one per optimiser (None / <= 0: no clipping).  Returns False — having done nothing —
    when an optimiser is not a plain fp32 torch.optim.Adam on the device (the caller then takes the torch path)."""
    optimizers = list(optimizers)
    if not 1 <= len(optimizers) <= MAX_NETS or not all(_eligible(o) for o in optimizers):
        return False
    if not isinstance(max_norm, (list, tuple)):
        max_norm = [max_norm] * len(optimizers)
    dev = optimizers[0].param_groups[0]["params"][0].device
    n_t, P, G, M, V, S, numel, step_host, hyper, host_counted = [], [], [], [], [], [], [], [], [], []
    # every optimiser is checked before any state is touched: a refusal leaves all of them as they were
    for opt in optimizers:
        ps = opt.param_groups[0]["params"]
        on_dev = [("step" in opt.state[p] and opt.state[p]["step"].is_cuda) or
                  ("step" not in opt.state[p] and opt.param_groups[0].get("capturable", False)) for p in ps]
        if any(on_dev) != all(on_dev) or any(p.device != dev for p in ps):
            return False
    for opt, mn in zip(optimizers, max_norm):
        g = opt.param_groups[0]
        ps = g["params"]
        n_t.append(len(ps))
        sts = [_state(opt, p) for p in ps]
        if not sts[0]["step"].is_cuda:  # the host keeps the count (non-capturable Adam): advanced once the launch is made
            step_host.append(float(sts[0]["step"]) + 1.0)
            host_counted.append(sts)
        else:
            step_host.append(0.0)
        for p, st in zip(ps, sts):
            P.append(p.data_ptr())
            G.append(p.grad.data_ptr())
            M.append(st["exp_avg"].data_ptr())
            V.append(st["exp_avg_sq"].data_ptr())
            S.append(st["step"].data_ptr() if st["step"].is_cuda else 0)
            numel.append(p.numel())
        b1, b2 = g["betas"]
        hyper.append((float(g["lr"]), float(b1), float(b2), float(g["eps"]), float(mn) if mn else 0.0))
    n = len(P)
    vps = lambda xs: (C.c_void_p * n)(*xs)
    f32s = lambda xs: (C.c_double * len(xs))(*xs)
    with th.cuda.device(dev):
        _abi.check(_abi.lib().ec_adam_clip_step(
            len(optimizers), (C.c_int32 * len(n_t))(*n_t), vps(P), vps(G), vps(M), vps(V), vps(S), (C.c_int64 * n)(*numel),
            f32s(step_host), f32s([h[0] for h in hyper]), f32s([h[1] for h in hyper]), f32s([h[2] for h in hyper]),
            f32s([h[3] for h in hyper]), f32s([h[4] for h in hyper]),
            C.c_void_p(th.cuda.current_stream(dev).cuda_stream)), "ec_adam_clip_step")
    for sts in host_counted:  # (after the launch's return code: a failed call has advanced nothing)
        for st in sts:
            st["step"] += 1
    for opt in optimizers:
        opt._opt_called = True  # (what an lr_scheduler looks at to tell that step() came first)
    return True


# ---- AdamW over many tensors of any size (ec_grad_clip_coef, ec_adamw_step) ----
QBLOCK = 256                      # elements that share a scale of the 8-bit states
STATE8 = th.float8_e4m3fn
_FLOATS = set(DTYPES)


def scale_count(p):
    """scales of one 8-bit state of p"""
    return -(-p.numel() // QBLOCK)


_DTYPE, _NUMEL, _DEVICE, _PTR, _PACKED = (operator.attrgetter("dtype"), th.Tensor.numel, th.Tensor.get_device, th.Tensor.data_ptr,
                                          th.Tensor.is_contiguous)


def _pointers(who, name, tensors, at, numel, dtypes):
    """addresses (array of 64-bit words) of contiguous tensors on device `at`, with `numel` elements each and types in `dtypes`
    (a set for all of them, or a list, one each).  Whole lists at a time: at hundreds of tensors these checks are the call's
    longest part on the host"""
    kinds = list(map(_DTYPE, tensors))
    if (list(map(_NUMEL, tensors)) == numel and set(map(_DEVICE, tensors)) == {at} and set(map(_PACKED, tensors)) == {True}
            and (kinds == dtypes if isinstance(dtypes, list) else dtypes.issuperset(kinds))):
        return array.array("Q", map(_PTR, tensors))
    if len(tensors) != len(numel):
        raise ValueError("%s: %d %s for %d tensors" % (who, len(tensors), name, len(numel)))
    for i, t in enumerate(tensors):
        want = {dtypes[i]} if isinstance(dtypes, list) else dtypes
        if t.get_device() != at or t.numel() != numel[i] or not t.is_contiguous() or t.dtype not in want:
            raise ValueError("%s: %s[%d] is %s %s on %s%s; %d contiguous elements of %s on cuda:%d are needed"
                             % (who, name, i, t.dtype, tuple(t.shape), t.device, "" if t.is_contiguous() else ", not contiguous",
                                numel[i], "/".join(map(str, want)), at))


def _address(a):
    """of an array's words (None: NULL)"""
    return a.buffer_info()[0] if a is not None else None


def _device_of(who, tensors):
    if not tensors:
        raise ValueError("%s: no tensors" % who)
    dev = tensors[0].device
    if dev.type != "cuda":
        raise RuntimeError("%s needs device tensors: marl_amd has no CPU fallback" % who)
    return dev


def clip_coef(grads, max_norm):
    """(norm, coef) of the gradients in the list (float32, bfloat16, float16): their total 2-norm and clip_grad_norm_'s factor
    min(1, max_norm / (norm + 1e-6)), as float32 scalars on the device.  The gradients are only read: hand coef to
    adamw_step.  The sums are double and in a fixed order."""
    grads = list(grads)
    dev = _device_of("clip_coef", grads)
    if not max_norm > 0:
        raise ValueError("clip_coef: max_norm %r" % (max_norm,))
    numel = list(map(_NUMEL, grads))
    G = _pointers("clip_coef", "grads", grads, dev.index, numel, _FLOATS)
    return _clip_coef(dev, G, array.array("q", numel), array.array("i", map(DTYPES.get, map(_DTYPE, grads))), max_norm)


def _clip_coef(dev, G, numel, codes, max_norm):
    n, counts = len(numel), numel.buffer_info()[0]
    nbytes = _abi.lib().ec_grad_clip_workspace(n, counts)
    work = th.empty(nbytes // 8 + 1, dtype=th.float64, device=dev)
    norm, coef = work[-1:].view(th.float32).unbind(0)
    launch("ec_grad_clip_coef", dev, n, _address(G), counts, _address(codes), max_norm, norm.data_ptr(), coef.data_ptr(), work.data_ptr(),
           nbytes)
    return norm, coef


def adamw_step(params, grads, exp_avg, exp_avg_sq, exp_avg_scale=None, exp_avg_sq_scale=None, *, step, lr, betas=(0.9, 0.999),
               eps=1e-8, weight_decay=1e-2, max_norm=None, coef=None):
    """One AdamW step over lists of contiguous tensors on one device, in place:
      m = m + (g - m)(1 - b1);  v = v b2 + (1 - b2) g^2
      p = p (1 - lr weight_decay) - lr / (1 - b1^step) m / (sqrt(v) / sqrt(1 - b2^step) + eps)
    params, grads: float32, bfloat16 or float16 (grads[i] as params[i]); the arithmetic is float32, rounded once to a
    parameter's type.
    States in 32 bits: exp_avg, exp_avg_sq float32.  In 8 bits: exp_avg, exp_avg_sq float8_e4m3fn with exp_avg_scale,
    exp_avg_sq_scale [scale_count(p)] float32, where exp_avg * scale is m and exp_avg_sq * scale is sqrt(v), one scale for each
    256 consecutive elements (an infinite gradient is lost to all of them, a NaN only to its own).
    step: this step's count, from 1 on; or a float32 scalar on the device (what a HIP graph needs), which the call advances
    first, and with which lr may be such a scalar too.
    max_norm: the gradients enter scaled by clip_coef(grads, max_norm)'s coef, and its norm is returned; coef: scaled by that
    device scalar (one clip over several calls).  The gradients are only read."""
    work = _checked_step(params, grads, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, step, lr, betas, eps, weight_decay, coef)
    norm = None
    if max_norm is not None:
        if coef is not None:
            raise ValueError("adamw_step: max_norm and coef")
        if not max_norm > 0:
            raise ValueError("adamw_step: max_norm %r" % (max_norm,))
        dev, _, (_, G, _, _, _, _, counts, codes) = work[:3]
        norm, coef = _clip_coef(dev, G, counts, codes, max_norm)
    _launch_step(coef, *work)
    return norm


def _checked_step(params, grads, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, step, lr, betas, eps, weight_decay, coef=None):
    """all that adamw_step refuses, ahead of all that it launches; what _launch_step takes behind coef"""
    who = "adamw_step"
    dev = _device_of(who, params)
    n, at = len(params), dev.index
    numel = list(map(_NUMEL, params))
    kinds = list(map(_DTYPE, params))
    P = _pointers(who, "params", params, at, numel, _FLOATS)
    G = _pointers(who, "grads", grads, at, numel, kinds)
    bits = 8 if exp_avg_scale is not None else 32
    st = {STATE8} if bits == 8 else {th.float32}
    M = _pointers(who, "exp_avg", exp_avg, at, numel, st)
    V = _pointers(who, "exp_avg_sq", exp_avg_sq, at, numel, st)
    MS = VS = None
    if bits == 8:
        if exp_avg_sq_scale is None:
            raise ValueError("adamw_step: exp_avg_scale without exp_avg_sq_scale")
        blocks = [-(-k // QBLOCK) for k in numel]
        MS = _pointers(who, "exp_avg_scale", exp_avg_scale, at, blocks, {th.float32})
        VS = _pointers(who, "exp_avg_sq_scale", exp_avg_sq_scale, at, blocks, {th.float32})
    elif exp_avg_sq_scale is not None:
        raise ValueError("adamw_step: exp_avg_sq_scale without exp_avg_scale")
    for name, a in (("parameter", P), ("exp_avg", M), ("exp_avg_sq", V), ("exp_avg_scale", MS), ("exp_avg_sq_scale", VS)):
        if a is not None and len(set(a)) != n and len({x for x, k in zip(a, numel) if k}) != sum(map(bool, numel)):
            raise ValueError("adamw_step: the same %s twice" % name)
    for name, t in (("step", step), ("lr", lr), ("coef", coef)):
        if isinstance(t, th.Tensor) and (t.device != dev or t.dtype != th.float32 or t.numel() != 1):
            raise ValueError("adamw_step: %s on the device is one float32 value on %s" % (name, dev))
    if isinstance(step, th.Tensor):
        pass
    elif isinstance(lr, th.Tensor):
        raise ValueError("adamw_step: a learning rate on the device needs a step count there")
    elif not step >= 1:
        raise ValueError("adamw_step: step %r (from 1 on)" % (step,))
    elif th.cuda.is_current_stream_capturing():
        raise RuntimeError("adamw_step: a recorded HIP graph would repeat step %r; pass a step count on the device" % (step,))
    b1, b2 = (float(b) for b in betas)
    if not (0 <= b1 < 1 and 0 <= b2 < 1 and eps >= 0 and weight_decay >= 0 and (isinstance(lr, th.Tensor) or lr >= 0)):
        raise ValueError("adamw_step: lr %r, betas %r, eps %r, weight_decay %r" % (lr, betas, eps, weight_decay))
    counts, codes = array.array("q", numel), array.array("i", map(DTYPES.get, kinds))
    return dev, params, (P, G, M, V, MS, VS, counts, codes), bits, step, lr, b1, b2, eps, weight_decay


def _launch_step(coef, dev, params, pointers, bits, step, lr, b1, b2, eps, weight_decay):
    """pointers: addresses of parameters, gradients and states, sizes and types, an array (or None) each"""
    on_dev, lr_dev = isinstance(step, th.Tensor), isinstance(lr, th.Tensor)
    dyn = th.empty(3, dtype=th.float32, device=dev) if on_dev else None
    launch("ec_adamw_step", dev, len(params), *map(_address, pointers), bits, ptr(coef), 0.0 if on_dev else step,
           ptr(step if on_dev else None), ptr(dyn), 0.0 if lr_dev else lr, ptr(lr if lr_dev else None), b1, b2, eps, weight_decay)
    # (written through raw pointers: autograd has to know; what was made in inference mode counts no versions)
    th.autograd.graph.increment_version([p for p in params if not p.is_inference()] if params[0].is_inference() else params)


def _need_options(group):
    """torch's optimisers share their group's options by state_dict: one under which the update is another is refused"""
    get = group.get
    if get("maximize") or get("amsgrad") or get("differentiable"):
        raise ValueError("AdamW: %s (only False)" % ", ".join("%s=%r" % (k, get(k)) for k in ("maximize", "amsgrad", "differentiable")))
    if not get("decoupled_weight_decay", True) and group["weight_decay"]:
        raise ValueError("AdamW: weight_decay %r with decoupled_weight_decay=False" % (group["weight_decay"],))


def _need_state(i, p, st, bits):
    """a saved state of parameter p, the i-th: its names, shapes and types"""
    float_of = lambda t: t.is_floating_point() and t.dtype != STATE8
    moment = lambda t: t.shape == p.shape and (t.dtype == STATE8 if bits == 8 else float_of(t))
    want = dict(exp_avg=moment, exp_avg_sq=moment)
    if bits == 8:
        want["exp_avg_scale"] = want["exp_avg_sq_scale"] = lambda t: t.shape == (scale_count(p),) and float_of(t)
    bad = sorted(set(st) ^ set(want) ^ {"step"}) or [k for k, ok in want.items() if not isinstance(st[k], th.Tensor) or not ok(st[k])]
    if not bad and not (st["step"].numel() == 1 if isinstance(st["step"], th.Tensor) else isinstance(st["step"], (int, float))):
        bad = ["step"]
    if bad:
        is_ = lambda v: "%s %s" % (v.dtype, tuple(v.shape)) if isinstance(v, th.Tensor) else repr(v)
        raise ValueError("AdamW.load_state_dict: parameter %s %s has %s for states of %d bits"
                         % (i, tuple(p.shape), ", ".join("%s %s" % (k, is_(st[k]) if k in st else "missing") for k in bad), bits))


class AdamW(th.optim.Optimizer):
    """torch.optim.AdamW's update (decoupled weight decay, no amsgrad) over all tensors in a few launches, with moments in 32
    bits or in 8 (state_bits, per group), and clip_grad_norm_ over all groups on the way (max_norm; the gradients stay as
    they are; `last_norm` holds the norm).  Parameters: contiguous, on one device, float32, bfloat16 or float16.

    State: state[p] = {"step", "exp_avg", "exp_avg_sq"} and, with 8 bits, {"exp_avg_scale", "exp_avg_sq_scale"} (see
    adamw_step); state_dict / load_state_dict keep their types.  capturable: step counts live on the device, and lr may be a
    device scalar -- for steps recorded into a HIP graph.  Parameters of a group that have taken the same steps share one
    count; where a gradient is missing for some of them they get one of their own.  Not while a graph is recorded, and not
    once a graph has recorded the shared one, which it would go on advancing for all (RuntimeError)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, max_norm=None, state_bits=32,
                 capturable=False):
        if max_norm is not None and not max_norm > 0:
            raise ValueError("AdamW: max_norm %r" % (max_norm,))
        self.max_norm, self.last_norm, self._recorded = max_norm, None, []
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      capturable=capturable))

    def __getstate__(self):  # (torch's names three attributes: what a copy or a pickle keeps)
        return dict(super().__getstate__(), max_norm=self.max_norm, last_norm=None, _recorded=[])

    def __setstate__(self, state):  # (a pickle may be older than the list)
        super().__setstate__(state)
        self.__dict__.setdefault("_recorded", [])

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        g = self.param_groups[-1]
        try:
            _need_options(g)
            if g["state_bits"] not in (8, 32):
                raise ValueError("AdamW: state_bits %r (8 or 32)" % (g["state_bits"],))
            if isinstance(g["lr"], th.Tensor) and not g["capturable"]:
                raise ValueError("AdamW: a learning rate on the device needs capturable=True")
            b1, b2 = g["betas"]
            if not (0 <= b1 < 1 and 0 <= b2 < 1 and g["eps"] >= 0 and g["weight_decay"] >= 0
                    and (isinstance(g["lr"], th.Tensor) or g["lr"] >= 0)):
                raise ValueError("AdamW: lr %r, betas %r, eps %r, weight_decay %r" % (g["lr"], g["betas"], g["eps"], g["weight_decay"]))
            dev = next((p.device for group in self.param_groups for p in group["params"]), None)
            for p in g["params"]:
                if p.dtype not in DTYPES or not p.is_contiguous() or p.device != dev:
                    raise ValueError("AdamW: a parameter of type %s, strides %s on %s (contiguous float32, bfloat16 or float16 on one "
                                     "device)" % (p.dtype, p.stride(), p.device))
        except ValueError:
            self.param_groups.pop()
            raise

    def _init(self, group, p, count):
        """p's state; count: the step count of a capturable group's parameters that take their first step together"""
        if th.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: the first step of a parameter makes its state; take it before a HIP graph is recorded")
        st = self.state[p]
        kw = dict(device=p.device)
        if group["state_bits"] == 8:
            for k in ("exp_avg", "exp_avg_sq"):
                st[k] = th.zeros(p.shape, dtype=th.uint8, **kw).view(STATE8)
                st[k + "_scale"] = th.zeros(scale_count(p), dtype=th.float32, **kw)
        else:
            st["exp_avg"] = th.zeros(p.shape, dtype=th.float32, **kw)
            st["exp_avg_sq"] = th.zeros(p.shape, dtype=th.float32, **kw)
        if not group["capturable"]:
            st["step"] = 0
        else:
            st["step"] = count if count is not None else th.zeros((), dtype=th.float32, **kw)
        return st

    def _split(self, calls, idle):
        """a count of their own, as it stands, for parameters without a gradient (`idle`: their states) that share one which
        this step advances"""
        live = {id(step): step for _, step, _ in calls if isinstance(step, th.Tensor)}
        apart = {}
        for st in idle:
            if id(st["step"]) in live:
                apart.setdefault(id(st["step"]), []).append(st)
        if apart and (th.cuda.is_current_stream_capturing() or any(id(t) in apart for t in self._recorded)):
            raise RuntimeError("AdamW: parameters with and without a gradient share a step count that a HIP graph records; take a "
                               "step with the same gradients missing before it is recorded")
        for at, sts in apart.items():
            own = live[at].clone()
            for st in sts:
                st["step"] = own

    @th.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with th.enable_grad():
                loss = closure()
        calls, every, idle, state = [], [], [], self.state
        for group in self.param_groups:
            _need_options(group)
            by_step, count, last = {}, None, None
            for p in group["params"]:
                g = p.grad
                if g is None:
                    if p in state:
                        idle.append(state[p])
                    continue
                if g.is_sparse:
                    raise RuntimeError("AdamW: sparse gradients are not supported")
                if not g.is_contiguous():
                    g = g.contiguous()
                st = state.get(p)
                if st is None:
                    st = self._init(group, p, count)
                    count = st["step"]
                step = st["step"]
                if step is not last:  # (tensors by identity)
                    last, ts = step, by_step.setdefault((id(step),) if isinstance(step, th.Tensor) else step, [])
                ts.append((p, g, st))
                every.append(g)
            calls += [(group, ts[0][2]["step"], ts) for ts in by_step.values()]
        if not every:
            return loss
        # (all calls are checked before the first is launched: what is refused has changed nothing)
        checked = []
        for group, step, ts in calls:
            cols = lambda k: [st[k] for _, _, st in ts]
            scales = [cols("exp_avg_scale"), cols("exp_avg_sq_scale")] if group["state_bits"] == 8 else [None, None]
            checked.append(_checked_step([p for p, _, _ in ts], [g for _, g, _ in ts], cols("exp_avg"), cols("exp_avg_sq"), *scales,
                                         step if isinstance(step, th.Tensor) else step + 1, group["lr"], group["betas"], group["eps"],
                                         group["weight_decay"]))
        if idle:
            self._split(calls, idle)
        coef = None
        if self.max_norm is not None:
            self.last_norm, coef = clip_coef(every, self.max_norm)
        for (_, step, ts), work in zip(calls, checked):
            _launch_step(coef, *work)
            if not isinstance(step, th.Tensor):
                step += 1
                for _, _, st in ts:
                    st["step"] = step
            elif th.cuda.is_current_stream_capturing():
                self._recorded.append(step)
        return loss

    def load_state_dict(self, state_dict):
        """torch's load casts states to their parameter's type: here they keep their own.  Takes torch.optim.AdamW's state_dict
        too (states in 32 bits, no amsgrad, not maximize).  What does not fit is refused before anything is replaced."""
        own = []

        def check(_, saved):
            self._need_state_dict(saved)
            own[:] = saved, self._options()

        # (behind the last of the user's hooks in front of a load, and ahead of the first behind it)
        hooks = [self.register_load_state_dict_pre_hook(check),
                 self.register_load_state_dict_post_hook(lambda _: self._take_states(*own), prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for h in hooks:
                h.remove()

    def _options(self):
        return [{k: group[k] for k in self.defaults if k in group} for group in self.param_groups]

    def _need_state_dict(self, state_dict):
        for saved, group, own in zip(state_dict["param_groups"], self.param_groups, self._options()):
            saved = {**own, **saved}
            _need_options(saved)
            bits = saved["state_bits"]
            if bits not in (8, 32):
                raise ValueError("AdamW.load_state_dict: state_bits %r (8 or 32)" % (bits,))
            if isinstance(saved["lr"], th.Tensor) and not saved["capturable"]:
                raise ValueError("AdamW.load_state_dict: a learning rate on the device needs capturable=True")
            for i, p in zip(saved["params"], group["params"]):
                if i in state_dict["state"]:
                    _need_state(i, p, state_dict["state"][i], bits)

    def _take_states(self, state_dict, own):
        """what torch's load has cast, as it was saved; own: each group's options before"""
        for saved, group, options in zip(state_dict["param_groups"], self.param_groups, own):
            for k, v in options.items():  # (what the state_dict does not name stays as it was)
                group.setdefault(k, v)
            group["capturable"] = bool(group["capturable"])
            if isinstance(group["lr"], th.Tensor) and group["params"]:  # (a checkpoint's may have come by the host)
                group["lr"] = group["lr"].detach().to(group["params"][0].device, th.float32)
            counts = {}  # (of a capturable group: one for each value)
            for i, p in zip(saved["params"], group["params"]):
                if i not in state_dict["state"]:
                    continue
                st = self.state[p] = {}
                for k, v in state_dict["state"][i].items():
                    if k != "step":
                        st[k] = v.detach().to(p.device, STATE8 if v.dtype == STATE8 else th.float32, copy=True).contiguous()
                    elif group["capturable"]:
                        if float(v) not in counts:
                            counts[float(v)] = th.tensor(float(v), dtype=th.float32, device=p.device)
                        st[k] = counts[float(v)]
                    else:
                        st[k] = int(v)
