"""Host side of ec_token_logprobs_fwd / _bwd (include/marl_amd.h): log-probs of given tokens (or actions) under
softmax(logits), the entropy, and the likeliest alternatives, for any number of tokens.

`token_logprobs` is the autograd form; `token_logprobs_fwd` and `token_logprobs_bwd` are the two passes by hand, for update
steps that keep no autograd graph and for recording into a HIP graph."""
from collections import namedtuple

import torch as th

from marl_amd import _abi
from marl_amd.utils.norm_device import launch, need_device, need_dtype, ptr, refuse_capture, refuse_tangent

MAX_TOP = 64  # EC_TOKEN_LOGPROBS_MAX_TOP

TokenLogprobs = namedtuple("TokenLogprobs", "logp entropy top_logp top_index lse")


def _breaks(t):
    """leading dimensions of t [..., vocab] that do not continue the one behind them (by stride): where its rows stop lying one
    stride apart.  Each as the number of dimensions up to and with it"""
    shape, stride = t.shape, t.stride()
    dims = [d for d in range(len(shape) - 1) if shape[d] != 1]
    return {a + 1 for a, b in zip(dims, dims[1:]) if stride[a] != stride[b] * shape[b]}


def _steps(t, at):
    """(outer, inner) stride of t's rows as [shape[:at], shape[at:-1]] (a part of one row: any)"""
    shape, stride = t.shape, t.stride()
    last = lambda lo, hi: next((stride[d] for d in range(hi - 1, lo - 1, -1) if shape[d] != 1), 0)
    return last(0, at), last(at, len(shape) - 1)


def _layout(logits, avail):
    """(logits, avail, inner, logits' outer and inner stride, avail's): rows as [outer, inner] of them, of both tensors alike,
    and in place wherever their strides allow one such split (a slice of steps out of [batch, steps, agents, vocab] does)"""
    vocab = logits.shape[-1]
    if vocab > 1 and logits.stride(-1) != 1:
        logits = logits.contiguous()
    if avail is not None and vocab > 1 and avail.stride(-1) != 1:
        avail = avail.contiguous()
    if logits.dim() == 2:
        return logits, avail, 1, logits.stride(0), 0, avail.stride(0) if avail is not None else 0, 0
    at = _breaks(logits)
    if avail is not None:
        both = at | _breaks(avail)
        if len(both) > 1:
            avail = avail.contiguous()
        else:
            at = both
    if len(at) > 1:
        logits, at = logits.contiguous(), set()
    at = at.pop() if at else logits.dim() - 1
    return (logits, avail, max(1, logits.shape[at:-1].numel()), *_steps(logits, at), *(_steps(avail, at) if avail is not None else (0, 0)))


def _inputs(who, logits, tokens, avail):
    """checked arguments, as both passes of the C entry points take them first"""
    dev = need_device(who, logits, tokens, avail)
    code = need_dtype(who, logits)
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError("%s: logits of shape %s" % (who, tuple(logits.shape)))
    if tokens.shape != logits.shape[:-1]:
        raise ValueError("%s: tokens of shape %s for logits of shape %s" % (who, tuple(tokens.shape), tuple(logits.shape)))
    if tokens.dtype not in (th.int64, th.int32):
        raise TypeError("%s: tokens of type %s" % (who, tokens.dtype))
    vocab = logits.shape[-1]
    kind = 0
    if avail is not None:
        if avail.is_floating_point() or avail.is_complex():
            raise TypeError("%s: avail of type %s (bool or integers)" % (who, avail.dtype))
        try:
            avail = avail if avail.shape == logits.shape else avail.expand(logits.shape)
        except RuntimeError:
            raise ValueError("%s: avail of shape %s for logits of shape %s" % (who, tuple(avail.shape), tuple(logits.shape))) from None
        if avail.dtype not in (th.bool, th.uint8, th.int8, th.int32):
            avail = avail != 0
        kind = 2 if avail.dtype == th.int32 else 1
    logits, avail, inner, so, si, ao, ai = _layout(logits, avail)
    tokens = tokens.to(th.int64).contiguous()
    # (the tensors are kept by the caller until the launch is made)
    head = (logits.data_ptr(), inner, so, si, tokens.data_ptr(), ptr(avail), kind, ao, ai, code, tokens.numel(), vocab)
    return dev, head, (logits, tokens, avail)


def token_logprobs_fwd(logits, tokens, avail=None, top_k=0):
    """TokenLogprobs(logp, entropy, top_logp, top_index, lse) for logits [..., V] (float32, bfloat16, float16; any V) and
    tokens [...] (int64 or int32).  avail (bool or integers, broadcastable to logits; the env's avail_actions): entries
    with 0 are excluded, whatever their logit holds; so are logits of -inf.
      logp [...]: log-prob of the token; 0 for a token below 0 (a padded row), NaN for one >= V, -inf for an excluded one
      entropy [...] of the distribution
      top_logp, top_index [..., top_k] (top_k <= 64; None for 0): the likeliest entries, equal ones by index; -inf and -1
        where there are fewer
      lse [..., 2]: largest logit and log-sum-exp above it, for token_logprobs_bwd
    all float32 (top_index int64).  A row with everything excluded has logp -inf, entropy 0 and gradient 0."""
    dev, head, keep = _inputs("token_logprobs_fwd", logits, tokens, avail)
    top_k = int(top_k)
    if not 0 <= top_k <= MAX_TOP:
        raise ValueError("token_logprobs_fwd: top_k %d (0 .. %d)" % (top_k, MAX_TOP))
    lead = tuple(tokens.shape)
    rows, vocab, code = head[-2], head[-1], head[-3]
    # (memory of its own for each: views of one tensor could not be changed in place under autograd)
    logp = th.empty_like(tokens, dtype=th.float32, memory_format=th.contiguous_format)
    entropy = th.empty_like(logp)
    lse = th.empty(lead + (2,), dtype=th.float32, device=dev)
    top_logp = th.empty(lead + (top_k,), dtype=th.float32, device=dev) if top_k else None
    top_index = th.empty(lead + (top_k,), dtype=th.int64, device=dev) if top_k else None
    nbytes = _abi.lib().ec_token_logprobs_workspace(rows, vocab, code, top_k)
    work = th.empty(nbytes, dtype=th.uint8, device=dev) if nbytes else None
    launch("ec_token_logprobs_fwd", dev, *head, top_k, logp.data_ptr(), entropy.data_ptr(), lse.data_ptr(), ptr(top_logp),
           ptr(top_index), ptr(work), nbytes)
    del keep
    return TokenLogprobs(logp, entropy, top_logp, top_index, lse)


def token_logprobs_bwd(logits, tokens, lse, entropy, dlogp=None, dentropy=None, avail=None):
    """d loss / d logits [..., V], contiguous and of logits' type, for dlogp = d loss / d logp and dentropy = d loss / d
    entropy [...] (None: 0), with token_logprobs_fwd's inputs and its lse and entropy:
      dlogp (1[v = token] - p_v) - dentropy p_v (log p_v + entropy),
    0 at excluded entries; a token below 0 takes no dlogp."""
    dev, head, keep = _inputs("token_logprobs_bwd", logits, tokens, avail)
    need_device("token_logprobs_bwd", logits, lse, entropy, dlogp, dentropy)
    small = []
    for name, t, shape in (("lse", lse, tokens.shape + (2,)), ("entropy", entropy, tokens.shape), ("dlogp", dlogp, tokens.shape),
                           ("dentropy", dentropy, tokens.shape)):
        if t is not None and (t.shape != shape or t.dtype != th.float32):
            raise ValueError("token_logprobs_bwd: %s is float32 of shape %s, not %s %s" % (name, tuple(shape), t.dtype, tuple(t.shape)))
        small.append(t.contiguous() if t is not None else None)
    out = th.empty_like(logits, memory_format=th.contiguous_format)
    launch("ec_token_logprobs_bwd", dev, *head, *map(ptr, small), out.data_ptr())
    del keep
    return out


class _TokenLogprobsFn(th.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, avail, top_k):
        f = token_logprobs_fwd(logits, tokens, avail, top_k)
        ctx.save_for_backward(logits, tokens, avail, f.lse, f.entropy)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*[t for t in (f.top_logp, f.top_index, f.lse) if t is not None])
        return tuple(f)

    @staticmethod
    @th.autograd.function.once_differentiable
    def backward(ctx, dlogp, dentropy, *_):
        refuse_capture("token_logprobs", "token_logprobs_fwd and token_logprobs_bwd")
        logits, tokens, avail, lse, entropy = ctx.saved_tensors
        if dlogp is None and dentropy is None:
            return None, None, None, None
        return token_logprobs_bwd(logits, tokens, lse, entropy, dlogp, dentropy, avail), None, None, None


def token_logprobs(logits, tokens, avail=None, top_k=0):
    """token_logprobs_fwd with gradients of logp and entropy for logits (the alternatives and lse carry none).  Not while a
    HIP graph is recorded (RuntimeError, unless logits need no gradient): record token_logprobs_fwd and token_logprobs_bwd
    there.  No forward-mode derivative (RuntimeError)."""
    refuse_tangent("token_logprobs", logits)
    if th.is_grad_enabled() and logits.requires_grad:
        refuse_capture("token_logprobs", "token_logprobs_fwd and token_logprobs_bwd")
        return TokenLogprobs(*_TokenLogprobsFn.apply(logits, tokens, avail, top_k))
    return token_logprobs_fwd(logits, tokens, avail, top_k)
