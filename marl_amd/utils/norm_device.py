"""Host side of ec_layer_norm_fwd / _bwd (include/marl_amd.h): layer norm over the last dimension, for rows of any width.

`layer_norm` is the autograd form; `layer_norm_fwd` and `layer_norm_bwd` are the two passes by hand, for update steps that
keep no autograd graph and for recording into a HIP graph."""
import torch as th
from torch.autograd import forward_ad

from marl_amd import _abi

DTYPES = {th.float32: 0, th.bfloat16: 1, th.float16: 2}  # EC_F32, EC_BF16, EC_F16


def need_device(who, *tensors):
    """one ROCm device for all of them (None: not given)"""
    at = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != at or at < 0:
            if not t.is_cuda or at < 0:
                raise RuntimeError("%s needs device tensors: marl_amd has no CPU fallback" % who)
            raise ValueError("%s: tensors on %s and %s" % (who, tensors[0].device, t.device))
    return tensors[0].device


def ptr(t):
    return t.data_ptr() if t is not None else None


def launch(name, dev, *args):
    """the C entry point `name` on dev's current stream (the last argument of each).  Calls of a few microseconds are
    what these operators' small sizes cost, so the device is only switched when it is another, and pointers go in as ints"""
    fn, at = getattr(_abi.lib(), name), dev.index
    stream = th._C._cuda_getCurrentRawStream(at)
    if th._C._cuda_getDevice() == at:
        rc = fn(*args, stream)
    else:
        with th.cuda.device(dev):
            rc = fn(*args, stream)
    if rc:
        _abi.check(rc, name)


def need_dtype(who, t):
    code = DTYPES.get(t.dtype)
    if code is None:
        raise TypeError("%s: %s (float32, bfloat16 or float16)" % (who, t.dtype))
    return code


def refuse_capture(who, instead):
    """autograd while a HIP graph is recorded: a gradient accumulator that an earlier eager graph of the same leaf keeps
    alive belongs to that graph's stream, and the backward pass would draw that stream into the recording, which ends the
    process -- refused before anything is recorded"""
    if th.cuda.is_current_stream_capturing():
        raise RuntimeError("%s: no autograd while a HIP graph is recorded; record %s" % (who, instead))


def refuse_tangent(who, *tensors):
    """a forward-mode tangent would be dropped and the result pass for a constant: such a tensor has requires_grad False"""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("%s: no forward-mode derivative" % who)


def _rows(t, cols):
    """[rows, cols] with contiguous columns and rows that do not overlap; a view where the strides allow one"""
    if t.dim() != 2:
        t = t.reshape(-1, cols)
    return t if (cols == 1 or t.stride(1) == 1) and (t.stride(0) >= cols or t.shape[0] <= 1) else t.contiguous()


def _check(who, x, weight, bias, eps):
    dev = need_device(who, x, weight, bias)
    code = need_dtype(who, x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("%s: shape %s has no last dimension to normalise over" % (who, tuple(x.shape)))
    if not eps >= 0:
        raise ValueError("%s: eps %r" % (who, eps))
    wcode = code
    for t in (weight, bias):
        if t is None:
            continue
        if t.dim() != 1 or t.shape[0] != x.shape[-1]:
            raise ValueError("%s: weight / bias of shape %s for %d columns" % (who, tuple(t.shape), x.shape[-1]))
        wcode = need_dtype(who, t)
        if t.dtype not in (x.dtype, th.float32) or (weight is not None and bias is not None and weight.dtype != bias.dtype):
            raise TypeError("%s: weight and bias are both of the rows' type (%s) or both float32" % (who, x.dtype))
    return dev, code, wcode


def layer_norm_fwd(x, weight=None, bias=None, eps=1e-5, want_stats=True):
    """(y, mean, rstd): y = (x - mean) * rstd * weight + bias over the last dimension of x (float32, bfloat16, float16),
    of x's shape and type; mean, rstd [x.shape[:-1]] float32, what layer_norm_bwd takes (None without want_stats).
    weight, bias [x.shape[-1]]: of x's type or float32, or None (1 and 0).  All sums are float32."""
    dev, code, wcode = _check("layer_norm_fwd", x, weight, bias, eps)
    cols = x.shape[-1]
    x2 = _rows(x, cols)
    rows = x2.shape[0]
    y = th.empty_like(x, memory_format=th.contiguous_format)
    mean = rstd = None
    if want_stats:
        mean = th.empty(x.shape[:-1], dtype=th.float32, device=dev)
        rstd = th.empty_like(mean)
    weight = weight.contiguous() if weight is not None else None
    bias = bias.contiguous() if bias is not None else None
    launch("ec_layer_norm_fwd", dev, x2.data_ptr(), x2.stride(0), ptr(weight), ptr(bias), code, wcode, rows, cols, eps, y.data_ptr(),
           ptr(mean), ptr(rstd))
    return y, mean, rstd


def layer_norm_bwd(dy, x, mean, rstd, weight=None, want_dx=True, want_dweight=True, want_dbias=True, param_dtype=None):
    """(dx, dweight, dbias) for dy = d loss / d y of layer_norm_fwd, with its x, mean, rstd and weight; None for what is not
    wanted.  dx has x's type; dweight and dbias have weight's (without a weight: param_dtype, or x's type).  The sums over
    the rows are added in a fixed order: the same bits every run."""
    dev, code, wcode = _check("layer_norm_bwd", x, weight, None, 0.0)
    need_device("layer_norm_bwd", x, dy, mean, rstd)
    if weight is None and param_dtype is not None:
        if param_dtype not in (x.dtype, th.float32):
            raise TypeError("layer_norm_bwd: param_dtype %s for rows of %s" % (param_dtype, x.dtype))
        wcode = DTYPES[param_dtype]
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError("layer_norm_bwd: dy is %s %s, x is %s %s" % (tuple(dy.shape), dy.dtype, tuple(x.shape), x.dtype))
    for t in (mean, rstd):
        if t.shape != x.shape[:-1] or t.dtype != th.float32:
            raise ValueError("layer_norm_bwd: mean and rstd are layer_norm_fwd's, float32 of shape %s" % (tuple(x.shape[:-1]),))
    cols = x.shape[-1]
    ptype = weight.dtype if weight is not None else (param_dtype or x.dtype)
    x2, dy2 = _rows(x, cols), _rows(dy, cols)
    rows = x2.shape[0]
    dx = th.empty_like(x, memory_format=th.contiguous_format) if want_dx else None
    if rows == 0:
        zeros = lambda want: th.zeros(cols, dtype=ptype, device=dev) if want else None
        return dx, zeros(want_dweight), zeros(want_dbias)
    dw = th.empty(cols, dtype=ptype, device=dev) if want_dweight else None
    db = th.empty(cols, dtype=ptype, device=dev) if want_dbias else None
    n_part = _abi.lib().ec_layer_norm_bwd_partials(rows, cols, code) if want_dweight or want_dbias else 0
    partials = th.empty(n_part, 2, cols, dtype=th.float32, device=dev) if n_part else None
    weight = weight.contiguous() if weight is not None else None
    mean, rstd = mean.contiguous(), rstd.contiguous()
    launch("ec_layer_norm_bwd", dev, dy2.data_ptr(), dy2.stride(0), x2.data_ptr(), x2.stride(0), mean.data_ptr(), rstd.data_ptr(),
           ptr(weight), code, wcode, rows, cols, ptr(dx), ptr(partials), n_part, ptr(dw), ptr(db))
    return dx, dw, db


class _LayerNormFn(th.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_fwd(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.param_dtype = bias.dtype if weight is None and bias is not None else None
        return y

    @staticmethod
    @th.autograd.function.once_differentiable
    def backward(ctx, dy):
        refuse_capture("layer_norm", "layer_norm_fwd and layer_norm_bwd")
        x, weight, mean, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, db = layer_norm_bwd(dy, x, mean, rstd, weight, need[0], need[1], need[2], ctx.param_dtype)
        return dx, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """layer_norm_fwd's y, with gradients for x, weight and bias.  Not while a HIP graph is recorded (RuntimeError, unless
    nothing needs a gradient): record layer_norm_fwd and layer_norm_bwd there.  No forward-mode derivative (RuntimeError)."""
    refuse_tangent("layer_norm", x, weight, bias)
    if th.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        refuse_capture("layer_norm", "layer_norm_fwd and layer_norm_bwd")
        return _LayerNormFn.apply(x, weight, bias, eps)
    return layer_norm_fwd(x, weight, bias, eps, want_stats=False)[0]
