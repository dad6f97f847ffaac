"""The operators of a policy's training step without a GPU: what their C entry points and host code refuse before anything
is launched, and the sizes of their scratch."""
import ctypes as C

import pytest
import torch as th

EINVAL = -1
PTR = C.c_void_p(4096)   # never read: every call here is refused on the host
NUL = C.c_void_p(0)


def _lib():
    from marl_amd import _abi
    return _abi.lib()


def _message():
    return _lib().ec_last_error().decode()


def test_layer_norm_refuses_bad_arguments():
    L = _lib()
    fwd = lambda x=PTR, xs=8, dt=0, wdt=0, rows=4, cols=8, eps=1e-5, y=PTR: L.ec_layer_norm_fwd(
        x, xs, PTR, PTR, dt, wdt, rows, cols, eps, y, PTR, PTR, NUL)
    for kw in (dict(dt=3), dict(dt=-1), dict(wdt=1), dict(dt=1, wdt=2), dict(rows=-1), dict(cols=0), dict(cols=(1 << 24) + 1),
               dict(x=NUL), dict(xs=-1), dict(xs=7), dict(eps=-1.0), dict(eps=float("nan")), dict(y=NUL)):
        assert fwd(**kw) == EINVAL and "ec_layer_norm_fwd" in _message(), kw
    assert fwd(rows=0, x=NUL, y=NUL) == 0
    n = L.ec_layer_norm_bwd_partials(1000, 64, 0)
    bwd = lambda dy=PTR, dys=64, mean=PTR, rows=1000, part=PTR, n_part=n, dw=PTR, dx=PTR: L.ec_layer_norm_bwd(
        dy, dys, PTR, 64, mean, PTR, PTR, 0, 0, rows, 64, dx, part, n_part, dw, NUL, NUL)
    for kw in (dict(dy=NUL), dict(dys=-2), dict(dys=63), dict(mean=NUL), dict(rows=0), dict(part=NUL), dict(n_part=n - 1), dict(n_part=n + 1)):
        assert bwd(**kw) == EINVAL and "ec_layer_norm_bwd" in _message(), kw
    assert bwd(part=NUL, n_part=0, dw=NUL, dx=NUL) == 0            # nothing asked for
    assert L.ec_layer_norm_bwd_partials(0, 64, 0) == 0 and L.ec_layer_norm_bwd_partials(5, 0, 0) == 0
    for rows, cols in ((1, 1), (7, 64), (10 ** 6, 64), (3, 10 ** 6), (10 ** 6, 4096)):
        for dt in (0, 1, 2):
            assert 1 <= L.ec_layer_norm_bwd_partials(rows, cols, dt) <= min(rows, 4096)


def test_token_logprobs_refuse_bad_arguments():
    L = _lib()
    def fwd(logits=PTR, inner=1, so=9, si=0, tok=PTR, av=NUL, kind=0, ao=0, ai=0, dt=0, rows=4, vocab=9, k=0, tl=NUL, ti=NUL, work=NUL, nb=0):
        return L.ec_token_logprobs_fwd(logits, inner, so, si, tok, av, kind, ao, ai, dt, rows, vocab, k, PTR, PTR, PTR, tl, ti, work, nb, NUL)
    need = L.ec_token_logprobs_workspace(1, 10 ** 6, 0, 5)
    assert need > 0 and need % 8 == 0 and L.ec_token_logprobs_workspace(10 ** 6, 11, 0, 5) == 0
    for kw in (dict(dt=5), dict(kind=3, av=PTR), dict(kind=1), dict(av=PTR), dict(rows=-1), dict(inner=0), dict(vocab=0), dict(vocab=1 << 31),
               dict(so=-1), dict(si=-1), dict(ao=-1), dict(ai=-9), dict(logits=NUL), dict(tok=NUL), dict(k=-1), dict(k=65, tl=PTR, ti=PTR),
               dict(k=3), dict(k=3, tl=PTR), dict(rows=1, vocab=10 ** 6, k=5, tl=PTR, ti=PTR),
               dict(rows=1, vocab=10 ** 6, k=5, tl=PTR, ti=PTR, work=PTR, nb=need - 1),
               dict(rows=1, vocab=10 ** 6, k=5, tl=PTR, ti=PTR, work=C.c_void_p(4100), nb=need)):
        assert fwd(**kw) == EINVAL and "ec_token_logprobs_fwd" in _message(), kw
    assert fwd(rows=0, logits=NUL, tok=NUL) == 0
    def bwd(lse=PTR, ent=PTR, out=PTR, rows=4, dt=0):
        return L.ec_token_logprobs_bwd(PTR, 1, 9, 0, PTR, NUL, 0, 0, 0, dt, rows, 9, lse, ent, NUL, NUL, out, NUL)
    for kw in (dict(lse=NUL), dict(ent=NUL), dict(out=NUL), dict(dt=9)):
        assert bwd(**kw) == EINVAL and "ec_token_logprobs_bwd" in _message(), kw
    assert bwd(rows=0, lse=NUL) == 0


def test_adamw_refuses_bad_arguments():
    L = _lib()
    arr = lambda *xs: (C.c_void_p * len(xs))(*xs)
    one, none = arr(4096), arr(None)

    def step(n=1, p=one, g=one, m=one, v=one, ms=None, vs=None, numel=100, dt=0, bits=32, t=1.0, tdev=NUL, dyn=NUL, lr=1e-3, lrdev=NUL,
             b1=0.9, b2=0.99, eps=1e-8, wd=0.0):
        return L.ec_adamw_step(n, p, g, m, v, ms, vs, (C.c_int64 * 1)(numel), (C.c_int32 * 1)(dt), bits, NUL, t, tdev, dyn, lr, lrdev, b1,
                               b2, eps, wd, NUL)
    nan = float("nan")
    for kw in (dict(n=-1), dict(p=None), dict(g=None), dict(p=none), dict(g=none), dict(m=none), dict(v=none), dict(numel=-1),
               dict(numel=1 << 41), dict(dt=3), dict(bits=16), dict(bits=8), dict(bits=8, ms=one, vs=none), dict(t=0.0), dict(t=nan),
               dict(tdev=PTR), dict(lrdev=PTR), dict(lr=-1.0), dict(lr=nan), dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0), dict(wd=nan)):
        assert step(**kw) == EINVAL and "ec_adamw_step" in _message(), kw
    assert step(numel=0, p=none, g=none, m=none, v=none) == 0
    clip = lambda n=1, g=one, numel=100, dt=0, mx=1.0, coef=PTR, work=PTR, nb=1 << 20: L.ec_grad_clip_coef(
        n, g, (C.c_int64 * 1)(numel), (C.c_int32 * 1)(dt), mx, PTR, coef, work, nb, NUL)
    for kw in (dict(n=-1), dict(g=none), dict(numel=-5), dict(dt=7), dict(mx=0.0), dict(mx=nan), dict(coef=NUL), dict(work=NUL), dict(nb=7),
               dict(work=C.c_void_p(4100))):
        assert clip(**kw) == EINVAL and "ec_grad_clip_coef" in _message(), kw
    sizes = (C.c_int64 * 3)(0, 5, 10 ** 9)
    assert 8 * 2 <= L.ec_grad_clip_workspace(3, sizes) <= 8 * 5000


def test_host_code_refuses_cpu_tensors():
    from marl_amd.utils import logprob_device, norm_device, optim_device
    x, t = th.randn(3, 5), th.zeros(3, dtype=th.int64)
    for f in (lambda: norm_device.layer_norm(x), lambda: norm_device.layer_norm_fwd(x), lambda: logprob_device.token_logprobs(x, t),
              lambda: logprob_device.token_logprobs_bwd(x, t, x, x), lambda: optim_device.clip_coef([x], 1.0),
              lambda: optim_device.adamw_step([x], [x], [x], [x], step=1, lr=1e-3)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            f()
