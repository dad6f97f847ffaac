"""layer_norm_fwd / _bwd / layer_norm (csrc/ec_norm.hip) against the formulas in float64.

Tolerances.  u = 2^-24 is half a step of fp32.  A row's sum is added by threads of at most 16 elements each (64 for rows
beyond 16384 columns, per 65536 of them) and a tree of 10 levels: under 128 roundings, so mean and variance carry at most
128 u of their absolute terms, and xhat at most E = 128 u (rstd max|x| + |xhat|).  What follows from E is propagated through
the formulas; the last term of each bound is the output's own rounding, half a step of its type (finfo.eps / 2)."""
import pytest
import torch as th

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
SHAPES = [(1, 1), (3, 2), (5, 3), (1, 4096), (7, 11), (33, 41), (257, 64), (64, 65), (130, 128), (19, 255), (9, 1023), (21, 1024),
          (6, 2053), (5, 4097), (3, 8200), (2, 16384), (3, 16391), (2, 40003), (1000, 24), (4100, 64)]


def _half(t):
    return th.finfo(t).eps / 2


def _inputs(rows, cols, dtype, wdtype, seed=0, pad=0):
    g = th.Generator(device="cuda").manual_seed(seed + rows * 131 + cols)
    r = lambda *s: th.randn(*s, device="cuda", generator=g)
    x = (r(rows, cols + pad) * (0.5 + r(rows, 1).abs()) + 2 * r(rows, 1)).to(dtype)[:, :cols]
    return x, (1 + 0.3 * r(cols)).to(wdtype), (0.3 * r(cols)).to(wdtype), r(rows, cols).to(dtype)


def _reference(x, w, b, dy, eps):
    x, dy = x.double(), dy.double()
    w = w.double() if w is not None else th.ones_like(x[0])
    b = b.double() if b is not None else th.zeros_like(x[0])
    mean = x.mean(1, keepdim=True)
    rstd = ((x - mean).square().mean(1, keepdim=True) + eps) ** -0.5
    h = (x - mean) * rstd
    a = dy * w
    dx = rstd * (a - a.mean(1, keepdim=True) - h * (a * h).mean(1, keepdim=True))
    e = 128 * U * (rstd * x.abs().amax(1, keepdim=True) + h.abs())            # of xhat
    s1 = a.abs().mean(1, keepdim=True)
    s2 = (a * h).abs().mean(1, keepdim=True)
    e2 = (a.abs() * e).mean(1, keepdim=True) + 128 * U * s2                   # of mean(a xhat)
    tol_y = e * w.abs() + 4 * U * (h * w).abs() + 4 * U * b.abs()
    tol_dx = rstd * (128 * U * s1 + h.abs() * e2 + e * s2 + 8 * U * (a.abs() + s1 + h.abs() * s2)) + 128 * U * dx.abs()
    depth = 64 + x.shape[0] / 256
    tol_dw = (dy.abs() * e).sum(0) + depth * U * (dy * h).abs().sum(0)
    tol_db = depth * U * dy.abs().sum(0)
    return (h * w + b, dx, (dy * h).sum(0), dy.sum(0)), (tol_y, tol_dx, tol_dw, tol_db)


def _within(got, want, tol, what):
    tol = tol + _half(got.dtype) * want.abs() + th.finfo(got.dtype).smallest_normal * th.finfo(got.dtype).eps
    off = (got.double() - want).abs() - tol
    assert got.shape == want.shape and bool((off <= 0).all()), (what, float(off.max()))


@pytest.mark.parametrize("dtype,wdtype", [(th.float32, th.float32), (th.bfloat16, th.bfloat16), (th.bfloat16, th.float32),
                                          (th.float16, th.float16), (th.float16, th.float32)])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_both_passes_match_the_formulas(rows, cols, dtype, wdtype):
    from marl_amd.utils import norm_device
    x, w, b, dy = _inputs(rows, cols, dtype, wdtype)
    want, tol = _reference(x, w, b, dy, 1e-5)
    y, mean, rstd = norm_device.layer_norm_fwd(x, w, b, 1e-5)
    dx, dw, db = norm_device.layer_norm_bwd(dy, x, mean, rstd, w)
    assert dw.dtype == db.dtype == wdtype and y.dtype == dx.dtype == dtype
    for got, a, t, name in zip((y, dx, dw, db), want, tol, ("y", "dx", "dw", "db")):
        _within(got, a, t, name)
    again = norm_device.layer_norm_bwd(dy, x, mean, rstd, w)
    assert all(th.equal(p, q) for p, q in zip((dx, dw, db), again))        # the same bits every run


@pytest.mark.parametrize("what", ["padded", "offset", "transposed", "broadcast", "batched_slice"])
@pytest.mark.parametrize("dtype", [th.float32, th.bfloat16])
def test_views(what, dtype):
    """rows that are not packed: every stride and alignment gives what the packed copy gives, bit for bit"""
    from marl_amd.utils import norm_device
    g = th.Generator(device="cuda").manual_seed(3)
    r = lambda *s: th.randn(*s, device="cuda", generator=g).to(dtype)
    cols = 203
    x, dy = {"padded": lambda: (r(37, cols + 9)[:, :cols], r(37, cols + 1)[:, 1:]),
             "offset": lambda: (r(37 * cols + 3)[3:].view(37, cols), r(37 * cols + 1)[1:].view(37, cols)),
             "transposed": lambda: (r(cols, 37).t(), r(cols, 37).t()),
             "broadcast": lambda: (r(1, cols).expand(37, cols), r(cols).expand(37, cols)),
             "batched_slice": lambda: (r(4, 9, cols)[:, 1:], r(4, 8, 2 * cols)[..., ::2])}[what]()
    w, b = r(2 * cols)[1:cols + 1], r(2 * cols)[::2]
    got = norm_device.layer_norm_fwd(x, w, b)
    want = norm_device.layer_norm_fwd(x.contiguous(), w.clone(), b.contiguous())
    assert all(th.equal(p, q) for p, q in zip(got, want)) and got[0].is_contiguous() and got[0].shape == x.shape
    got = norm_device.layer_norm_bwd(dy, x, got[1], got[2], w)
    want = norm_device.layer_norm_bwd(dy.contiguous(), x.contiguous(), want[1], want[2], w.clone())
    assert all(th.equal(p, q) for p, q in zip(got, want))


def test_without_weight_or_bias_and_partial_gradients():
    from marl_amd.utils import norm_device
    x, w, b, dy = _inputs(70, 300, th.bfloat16, th.float32, seed=1)
    for ww, bb in ((None, None), (w, None), (None, b)):
        want, tol = _reference(x, ww, bb, dy, 1e-3)
        y, mean, rstd = norm_device.layer_norm_fwd(x, ww, bb, 1e-3)
        _within(y, want[0], tol[0], "y")
        full = norm_device.layer_norm_bwd(dy, x, mean, rstd, ww, param_dtype=th.float32)
        for got, a, t, name in zip(full, want[1:], tol[1:], ("dx", "dw", "db")):
            _within(got, a, t, name)
        assert full[1].dtype == full[2].dtype == th.float32
        for wants in ((True, False, False), (False, True, False), (False, False, True), (False, False, False)):
            part = norm_device.layer_norm_bwd(dy, x, mean, rstd, ww, *wants, param_dtype=th.float32)
            assert all((p is None) if not on else th.equal(p, f) for p, f, on in zip(part, full, wants))


def test_edges():
    """no rows; one column (xhat is 0); constant rows (rstd = 1 / sqrt(eps)); a NaN and an inf stay in their row; a mean far
    from 0 costs only its own rounding"""
    from marl_amd.utils import norm_device
    dev = "cuda"
    w = th.full((8,), 2.0, device=dev)
    y, mean, rstd = norm_device.layer_norm_fwd(th.empty(0, 8, device=dev), w, w)
    assert y.shape == (0, 8) and mean.shape == (0,)
    dx, dw, db = norm_device.layer_norm_bwd(y, y, mean, rstd, w)
    assert dx.shape == (0, 8) and not dw.any() and not db.any()
    x = th.full((3, 8), 5.0, device=dev)
    y, mean, rstd = norm_device.layer_norm_fwd(x, w, w, 1e-2)
    assert th.equal(y, x.new_full((3, 8), 2.0)) and th.equal(mean, x[:, 0]) and bool(((rstd - 10).abs() <= 10 * 4 * U).all())
    x, w, b, dy = _inputs(6, 700, th.float32, th.float32, seed=5)
    clean = norm_device.layer_norm_fwd(x, w, b)[0]
    x[2, 699], x[4, 0] = float("nan"), float("inf")
    y, mean, rstd = norm_device.layer_norm_fwd(x, w, b)
    dx, dw, db = norm_device.layer_norm_bwd(dy, x, mean, rstd, w)
    for r in range(6):
        assert bool(th.isnan(y[r]).any()) == (r in (2, 4)) and bool(th.isnan(dx[r]).any()) == (r in (2, 4))
        assert r in (2, 4) or th.equal(y[r], clean[r])
    assert bool(th.isnan(dw).all()) and not bool(th.isnan(db).any())
    for cols in (64, 700, 5000, 20000):
        x = th.randn(3, cols, device=dev) + 4096.0
        want, tol = _reference(x, th.ones(cols, device=dev), None, x, 1e-5)
        _within(norm_device.layer_norm_fwd(x)[0], want[0], tol[0], cols)


def test_an_outlier_in_the_first_column_costs_nothing():
    """(what squares about the first element, or a sum of squares, would lose)"""
    from marl_amd.utils import norm_device
    x = th.randn(4, 3000, device="cuda")
    x[:, 0] = 3e4
    want, tol = _reference(x, th.ones(3000, device="cuda"), None, x, 1e-5)
    _within(norm_device.layer_norm_fwd(x)[0], want[0], tol[0], "y")


def test_autograd_and_differences():
    """layer_norm's gradients are layer_norm_bwd's, for leaves of any shape; and they are the slopes of the loss: central
    differences of the float64 formula at the same point agree with them"""
    from marl_amd.utils import norm_device
    x, w, b, dy = _inputs(12, 50, th.float32, th.float32, seed=9)
    xs, ws, bs = (t.clone().requires_grad_(True) for t in (x.view(3, 4, 50), w, b))
    out = norm_device.layer_norm(xs, ws, bs, 1e-5)
    out.backward(dy.view(3, 4, 50))
    y, mean, rstd = norm_device.layer_norm_fwd(x, w, b)
    dx, dw, db = norm_device.layer_norm_bwd(dy, x, mean, rstd, w)
    assert th.equal(out.detach().view_as(y), y) and th.equal(xs.grad.view_as(dx), dx) and th.equal(ws.grad, dw) and th.equal(bs.grad, db)
    f = lambda x_, w_, b_: (dy.double() * _reference(x_, w_, b_, dy, 1e-5)[0][0]).sum()
    g = th.Generator(device="cuda").manual_seed(1)
    for k, (t, grad) in enumerate(((x, dx), (w, dw), (b, db))):
        v = th.randn(t.shape, device="cuda", generator=g, dtype=th.float64)
        at = [x.double(), w.double(), b.double()]
        step = 1e-4
        hi, lo = ([a + s * step * v if i == k else a for i, a in enumerate(at)] for s in (1, -1))
        slope = float((f(*hi) - f(*lo)) / (2 * step))
        # (third derivatives of O(sum |dy| v^3 / sigma^3) times step^2, and fp32 gradients)
        assert abs(slope - float((grad.double() * v).sum())) <= 1e-5 * float((grad.double() * v).abs().sum()) + 1e-4, k
    frozen = norm_device.layer_norm(xs.detach(), ws.detach(), bs, 1e-5)
    frozen.sum().backward()
    assert ws.grad is not None and not norm_device.layer_norm(x, w, b).requires_grad


def test_outputs_changed_in_place():
    from marl_amd.utils.norm_device import layer_norm, layer_norm_fwd
    x, w, b, dy = _inputs(21, 64, th.float32, th.float32)
    grads = []
    for in_place in (False, True):
        a = x.clone().requires_grad_()
        y = layer_norm(a, w, b)
        (y.relu_() if in_place else y.relu()).backward(dy)
        grads.append(a.grad)
    assert th.equal(*grads)
    _, mean, rstd = layer_norm_fwd(x, w, b)
    s = rstd.clone().requires_grad_()
    mean.mul_(s).sum().backward()
    assert s.grad is not None


def test_refusals():
    from marl_amd.utils import norm_device
    x, w, b, dy = _inputs(4, 32, th.bfloat16, th.float32)
    y, mean, rstd = norm_device.layer_norm_fwd(x, w, b)
    for bad in (lambda: norm_device.layer_norm_fwd(x.double()), lambda: norm_device.layer_norm_fwd(x, w.half()),
                lambda: norm_device.layer_norm_fwd(x, w, b.bfloat16()), lambda: norm_device.layer_norm_bwd(dy, x, mean, rstd, None, param_dtype=th.float16)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: norm_device.layer_norm_fwd(x, w[:31]), lambda: norm_device.layer_norm_fwd(x, w, b, -1.0),
                lambda: norm_device.layer_norm_fwd(x, w, b, float("nan")), lambda: norm_device.layer_norm_fwd(x[:, :0]),
                lambda: norm_device.layer_norm_bwd(dy.float(), x, mean, rstd, w), lambda: norm_device.layer_norm_bwd(dy[:3], x, mean, rstd, w),
                lambda: norm_device.layer_norm_bwd(dy, x, mean[:3], rstd, w), lambda: norm_device.layer_norm_bwd(dy, x, mean, rstd.double(), w)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        norm_device.layer_norm_fwd(x, w.cpu())


def test_captured_and_replayed():
    """both passes in a HIP graph: every replay on new inputs equals the eager passes; autograd in a capture is refused"""
    from marl_amd.utils import norm_device
    x, w, b, dy = _inputs(300, 96, th.float32, th.float32)
    w.requires_grad_(True)
    side = th.cuda.Stream()
    side.wait_stream(th.cuda.current_stream())
    with th.cuda.stream(side):
        norm_device.layer_norm_fwd(x, w, b)
    th.cuda.current_stream().wait_stream(side)
    graph = th.cuda.CUDAGraph()
    with th.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="recorded"):
            norm_device.layer_norm(x, w, b)
        y, mean, rstd = norm_device.layer_norm_fwd(x, w.detach(), b)
        grads = norm_device.layer_norm_bwd(dy, x, mean, rstd, w.detach())
    for k in range(4):
        x.copy_(_inputs(300, 96, th.float32, th.float32, seed=k + 1)[0])
        graph.replay()
        th.cuda.synchronize()
        e = norm_device.layer_norm_fwd(x, w.detach(), b)
        eg = norm_device.layer_norm_bwd(dy, x, e[1], e[2], w.detach())
        assert all(th.equal(p, q) for p, q in zip((y, mean, rstd) + tuple(grads), e + eg)), k


def test_many_rows_and_offsets_past_32_bits():
    """a view whose last rows lie beyond 2^31 elements (8.6 GB of bf16, of which 40 rows are touched), and a tall batch"""
    from marl_amd.utils import norm_device
    cols, stride = 130, 110_000_003
    flat = th.empty(39 * stride + cols, dtype=th.bfloat16, device="cuda")
    x = flat.as_strided((40, cols), (stride, 1))
    src = th.randn(40, cols, device="cuda").bfloat16()
    x.copy_(src)
    got, want = norm_device.layer_norm_fwd(x), norm_device.layer_norm_fwd(src)
    assert all(th.equal(p, q) for p, q in zip(got, want))
    dy = th.randn(40, cols, device="cuda").bfloat16()
    assert all(th.equal(p, q) for p, q in zip(norm_device.layer_norm_bwd(dy, x, got[1], got[2]),
                                              norm_device.layer_norm_bwd(dy, src, want[1], want[2])))
    del flat, x
    x, w, b, dy = _inputs(200003, 64, th.float32, th.float32, seed=2)
    want, tol = _reference(x, w, b, dy, 1e-5)
    y, mean, rstd = norm_device.layer_norm_fwd(x, w, b)
    for got, a, t, name in zip((y,) + norm_device.layer_norm_bwd(dy, x, mean, rstd, w), want, tol, ("y", "dx", "dw", "db")):
        _within(got, a, t, name)
