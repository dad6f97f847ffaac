"""token_logprobs_fwd / _bwd / token_logprobs (csrc/ec_logprob.hip) against softmax in float64.

Tolerances.  u = 2^-24 is half a step of fp32.  A thread adds at most vocab / 256 + 32 terms one after the other, then come a
tree and the joins of waves and splits: D = vocab / 256 + 128 roundings.  Each term e^(l - m) carries the rounding of
(l - m) log2(e) and the exponential's own step: (4 + 4 |l - m|) u of itself, and e^-t t <= 0.37, so S1 is off by at most (D + 8) u
of itself and log S1 by that plus 4 u of its size.  The entropy is log S1 - S2 / S1 with |S2| / S1 <= log S1 + ..., taken with
2 + 2 log(vocab).  A gradient entry has p off by (D + 8 + 8 |log p|) u of itself.  Outputs in 16 bits add half a step
(finfo.eps / 2) and half of the smallest step near 0."""
import math

import pytest
import torch as th

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
INF = float("inf")
SHAPES = [(1, 1), (5, 2), (300, 11), (257, 41), (64, 64), (33, 65), (9, 127), (130, 1000), (3, 4096), (2, 8192), (7, 8201), (1, 50021),
          (600, 5003), (3, 131072)]


def _entropy_tol(vocab):
    return (vocab / 256 + 136) * U * (2 + 2 * math.log(vocab + 1))


def _inputs(rows, vocab, dtype, mask, seed=0):
    g = th.Generator(device="cuda").manual_seed(seed + 7 * rows + vocab)
    l = (3 * th.randn(rows, vocab, device="cuda", generator=g)).to(dtype)
    t = th.randint(0, vocab, (rows,), device="cuda", generator=g)
    avail = None
    if mask is not None:
        on = th.rand(rows, vocab, device="cuda", generator=g) < 0.5
        on[th.arange(rows), t] = True
        if rows > 2:
            on[1] = False                                     # a row with nothing
            on[2] = False
            on[2, t[2]] = True                                # a row with one entry
        junk = th.tensor([float("nan"), INF, th.finfo(dtype).min, -INF], device="cuda", dtype=dtype)
        l = th.where(on, l, junk[th.arange(rows * vocab, device="cuda") % 4].view(rows, vocab))
        avail = on.to(mask)
    if rows > 4:
        t[3] = -1
        t[4] = -100
    g1, g2 = (th.randn(rows, device="cuda", generator=g) for _ in range(2))
    return l, t, avail, g1, g2


def _reference(l, t, avail, g, h):
    l = l.double()
    if avail is not None:
        l = l.masked_fill(avail == 0, -INF)
    rows, vocab = l.shape
    dead = (l == -INF).all(1)
    lp = th.log_softmax(l, 1)
    lp[dead] = -INF
    p = lp.exp()
    fin = lp.masked_fill(lp == -INF, 0.0)
    ent = -(p * fin).sum(1)
    i = th.arange(rows, device=l.device)
    skip = t < 0
    logp = lp[i, t.clamp(min=0)]
    hit = ~skip & (logp > -INF)
    logp = logp.masked_fill(skip, 0.0)
    g = g.double().masked_fill(skip, 0.0)
    h = h.double()
    d = -p * (g[:, None] + h[:, None] * (fin + ent[:, None]))
    d[i[hit], t[hit]] += g[hit]
    m = l.amax(1).masked_fill(dead, 0.0)
    ls = (th.logsumexp(l, 1) - m).masked_fill(dead, 0.0)
    depth = vocab / 256 + 136
    e_ls = depth * U + 4 * U * ls
    e_ent = _entropy_tol(vocab)
    tol = (e_ls + 4 * U * (logp.masked_fill(logp == -INF, 0.0).abs() + ls), e_ent + 0 * ent,
           p * (depth + 8 * fin.abs()) * U * (g.abs() + h.abs() * (1 + ent))[:, None] + (p * h.abs()[:, None]) * (
               8 * U * (fin.abs() + ent[:, None]) + e_ent) + 4 * U * g.abs()[:, None] * (p > 0) + 2.0 ** -140)
    return lp, (logp, ent, d), tol


def _within(got, want, tol, what):
    f = th.finfo(got.dtype)
    live = th.isfinite(want)
    assert th.equal(got.double()[~live], want[~live]), what
    off = (got.double() - want)[live].abs() - (tol + (f.eps / 2 * want.abs() + f.smallest_normal * f.eps / 2 if got.dtype != th.float32
                                                    else 2.0 ** -126))[live]
    assert got.shape == want.shape and (not off.numel() or float(off.max()) <= 0), (what, float(off.max()))


def _top(l, avail, lp, k):
    """indices and log-probs of the k largest, ties by index, by a stable sort"""
    l = l.double() if avail is None else l.double().masked_fill(avail == 0, -INF)
    at = th.sort(-l, dim=1, stable=True)[1][:, :k]
    val = lp.gather(1, at)
    at = at.masked_fill(val == -INF, -1)
    more = k - at.shape[1]
    return th.nn.functional.pad(val, (0, more), value=-INF), th.nn.functional.pad(at, (0, more), value=-1)


@pytest.mark.parametrize("mask", [None, th.bool, th.int32])
@pytest.mark.parametrize("dtype", [th.float32, th.bfloat16, th.float16])
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_both_passes_match_the_formulas(rows, vocab, dtype, mask):
    from marl_amd.utils import logprob_device
    l, t, avail, g, h = _inputs(rows, vocab, dtype, mask)
    lp, want, tol = _reference(l, t, avail, g, h)
    for k in (0, 1, 20):
        f = logprob_device.token_logprobs_fwd(l, t, avail, top_k=k)
        _within(f.logp, want[0], tol[0], "logp")
        _within(f.entropy, want[1], tol[1], "entropy")
        if k:
            val, at = _top(l, avail, lp, k)
            assert th.equal(f.top_index, at), k
            _within(f.top_logp, val, (tol[0].max() + 4 * U * val.abs()), "top_logp")
    d = logprob_device.token_logprobs_bwd(l, t, f.lse, f.entropy, g, h, avail)
    assert d.dtype == dtype
    _within(d, want[2], tol[2], "dlogits")


@pytest.mark.parametrize("dtype", [th.float32, th.bfloat16])
@pytest.mark.parametrize("vocab", [7, 40, 300, 9000, 70001])
def test_ties_go_to_the_lowest_index(vocab, dtype):
    """equal logits, few distinct values, rising and falling rows, signed zeros: what a stable sort gives"""
    from marl_amd.utils import logprob_device
    g = th.Generator(device="cuda").manual_seed(vocab)
    ramp = th.arange(vocab, device="cuda") % 1024 / 8.0
    zeros = th.where(th.arange(vocab, device="cuda") % 2 == 0, -0.0, 0.0)
    l = th.stack([th.zeros(vocab, device="cuda"), th.randint(0, 3, (vocab,), device="cuda", generator=g).float(), ramp, -ramp, zeros,
                  th.full((vocab,), th.finfo(dtype).min, device="cuda")]).to(dtype)
    t = th.zeros(6, dtype=th.int64, device="cuda")
    for k in (1, 5, 64):
        f = logprob_device.token_logprobs_fwd(l, t, top_k=k)
        val, at = _top(l + 0.0, None, th.log_softmax(l.double(), 1), k)
        assert th.equal(f.top_index, at)
        assert bool(th.isfinite(f.logp[[0, 5]]).all()) and bool(((f.entropy[[0, 5]] - math.log(vocab)).abs() <= _entropy_tol(vocab)).all())


def test_edges():
    """no rows, one entry, rows of -inf, huge and far logits, NaN and +inf rows, tokens outside"""
    from marl_amd.utils import logprob_device
    F = logprob_device.token_logprobs_fwd
    dev = "cuda"
    f = F(th.empty(0, 5, device=dev), th.empty(0, dtype=th.int64, device=dev), top_k=2)
    assert f.logp.shape == (0,) and f.top_index.shape == (0, 2) and f.lse.shape == (0, 2)
    assert logprob_device.token_logprobs_bwd(th.empty(0, 5, device=dev), f.logp.long(), f.lse, f.entropy).shape == (0, 5)
    one = F(th.tensor([7.0], device=dev), th.tensor(0, device=dev), top_k=2)   # no leading dimension
    assert one.logp.shape == () and float(one.logp) == 0 and float(one.entropy) == 0 and one.top_index.tolist() == [0, -1]
    big = th.finfo(th.float32).max
    for vocab in (5, 200, 9000):
        l = th.zeros(9, vocab, device=dev)
        l[0] = -INF
        l[1] = -big
        l[1, 3] = big                     # differences beyond the type's range
        l[2] = 1e30
        l[3, 1] = float("nan")
        l[4, 2] = INF
        l[5], l[5, 4] = -INF, -3.0        # one entry
        l[6] = 3e4 + th.arange(vocab, device=dev) % 3
        t = th.full((9,), 3, dtype=th.int32, device=dev)
        t[5], t[7], t[8] = 4, vocab, -7
        f = F(l, t, top_k=3)
        assert float(f.logp[0]) == -INF and float(f.entropy[0]) == 0 and f.top_index[0].tolist() == [-1] * 3 and f.lse[0].tolist() == [-INF, 0]
        assert float(f.logp[1]) == 0 and float(f.entropy[1]) == 0 and f.top_index[1].tolist() == [3, 0, 1]
        assert abs(float(f.logp[2]) + math.log(vocab)) <= _entropy_tol(vocab)
        for r in (3, 4):
            assert math.isnan(float(f.logp[r])) and math.isnan(float(f.entropy[r])) and f.top_index[r].tolist() == [-1] * 3
            assert bool(th.isnan(f.top_logp[r]).all())
        assert float(f.logp[5]) == 0 and float(f.entropy[5]) == 0 and f.top_index[5].tolist() == [4, -1, -1]
        want = th.log_softmax(l[6].double(), 0)[3]
        assert abs(float(f.logp[6]) - float(want)) <= _entropy_tol(vocab)   # (fp32 cannot hold this row's log-sum-exp to 1e-3)
        assert math.isnan(float(f.logp[7])) and float(f.logp[8]) == 0
        d = logprob_device.token_logprobs_bwd(l, t, f.lse, f.entropy, th.ones(9, device=dev), th.ones(9, device=dev))
        assert not d[0].any() and not d[5].any() and bool(th.isnan(d[3]).any()) and bool(th.isnan(d[4]).any()) and bool(th.isnan(d[7]).all())
        p = th.softmax(l[6].double(), 0)
        ent = th.special.entr(p).sum()
        dd = -p * (1 + p.log() + ent)
        dd[3] += 1
        assert bool(((d[6].double() - dd).abs() <= 2 * _entropy_tol(vocab) * dd.abs().max()).all())
        assert bool(th.isfinite(d[[1, 2, 6, 8]]).all())


@pytest.mark.parametrize("vocab", [11, 500, 9001])
def test_views_and_broadcast_masks(vocab):
    """steps sliced out of [batch, steps, vocab], padded and transposed rows, masks of every integer type and broadcast shape"""
    from marl_amd.utils import logprob_device
    F, B = logprob_device.token_logprobs_fwd, logprob_device.token_logprobs_bwd
    g = th.Generator(device="cuda").manual_seed(vocab)
    base = th.randn(3, 6, vocab + 3, device="cuda", generator=g)
    t = th.randint(0, vocab, (3, 5), device="cuda", generator=g)
    on = th.rand(3, 5, vocab, device="cuda", generator=g) < 0.7
    gl = th.randn(3, 5, device="cuda", generator=g)

    def same(l, av, av_plain):
        a, b = F(l, t, av, top_k=4), F(l.contiguous(), t, av_plain, top_k=4)
        assert all(th.equal(p, q) for p, q in zip(a, b))
        assert th.equal(B(l, t, a.lse, a.entropy, gl, gl, av), B(l.contiguous(), t, b.lse, b.entropy, gl, gl, av_plain))
    same(base[:, :-1, :vocab], None, None)
    same(base[:, 1:, 3:], on, on.int())
    same(base.transpose(0, 1)[:5, :, :vocab].transpose(0, 1), on.long(), on)
    same(th.randn(vocab, 5, 3, device="cuda", generator=g).permute(2, 1, 0), on.to(th.uint8), on)
    same(base[:, :5, 1:vocab + 1], on[:, :1], on[:, :1].expand(3, 5, vocab).contiguous())
    same(base[:, :5, 1:vocab + 1], on[0, 0].int(), on[0, 0].expand(3, 5, vocab).contiguous())
    same(base[:, :5, 2:vocab + 2], on[:1] * 8, on[:1].expand(3, 5, vocab).contiguous())
    four = base[:, :-1, :vocab].unsqueeze(0)
    a = F(four, t.unsqueeze(0), on)
    assert th.equal(a.logp[0], F(base[:, :-1, :vocab], t, on).logp) and a.logp.shape == (1, 3, 5)


@pytest.mark.parametrize("dtype", [th.float32, th.bfloat16])
@pytest.mark.parametrize("vocab", [1, 3, 8, 11, 30, 40, 130])
def test_rows_with_gaps(vocab, dtype):
    """logits and masks as views of wider buffers, in one order and in different ones: the bits of the packed call"""
    from marl_amd.utils import logprob_device
    gen = th.Generator(device="cuda").manual_seed(vocab)
    big = th.randn(9, 8, 7, vocab + 3, device="cuda", generator=gen).to(dtype)
    on = th.rand(9, 8, 7, vocab + 3, device="cuda", generator=gen) < 0.6
    views = [lambda x: x[:, :-1, :, :vocab], lambda x: x[:8, 1:, :, 3:], lambda x: x[:8, :7, :, 1:vocab + 1].contiguous(),
             lambda x: x[..., :vocab].contiguous()[:, :-1], lambda x: x[..., :vocab].contiguous()[1:, 1:],
             lambda x: x[..., :vocab].contiguous()[:, :, 1:], lambda x: x[:7, :8, :, :vocab].transpose(0, 1),
             lambda x: x[:1, :1, :, 2:vocab + 2].expand(8, 7, 7, vocab), lambda x: x[:1, :7, :1, 2:vocab + 2].expand(8, 7, 7, vocab)]
    for i, lv in enumerate(views):
        for k, mv in enumerate([None, views[i], *views[:5], *views[7:]]):
            l = lv(big)
            a = mv(on) if mv else None
            if a is not None:                                # (what both have)
                n, m, o = (min(x, y) for x, y in zip(l.shape[:3], a.shape[:3]))
                l, a = l[:n, :m, :o], a[:n, :m, :o]
            a = a.to((th.int32, th.bool, th.int64)[(i + k) % 3]) if a is not None and k % 2 else a
            t = th.randint(0, vocab, l.shape[:-1], device="cuda", generator=gen)
            g = th.randn(l.shape[:-1], device="cuda", generator=gen)
            plain = a.contiguous() if a is not None else None
            f = logprob_device.token_logprobs_fwd(l, t, a, min(3, vocab))
            e = logprob_device.token_logprobs_fwd(l.contiguous(), t, plain, min(3, vocab))
            assert all(th.equal(p, q) for p, q in zip(f, e)), (i, k)
            assert th.equal(logprob_device.token_logprobs_bwd(l, t, f.lse, f.entropy, g, g, a),
                            logprob_device.token_logprobs_bwd(l.contiguous(), t, e.lse, e.entropy, g, g, plain)), (i, k)
    for shape in ((2, 0, vocab), (0, 3, vocab), (0, vocab)):
        f = logprob_device.token_logprobs_fwd(big.new_empty(shape), th.zeros(shape[:-1], dtype=th.int64, device="cuda"))
        assert f.logp.shape == shape[:-1]


def test_autograd_and_differences():
    """token_logprobs' gradient is token_logprobs_bwd's, also through either output alone, and the slope of the loss"""
    from marl_amd.utils import logprob_device
    l, t, avail, g, h = _inputs(40, 23, th.float32, th.bool, seed=3)
    avail[1] = True                        # (a row of NaN: its gradient is NaN, and it has no slope to compare)
    l = th.where(avail, l, 0.0)
    same = lambda a, b: th.allclose(a, b, rtol=0, atol=0, equal_nan=True)
    leaf = l.clone().requires_grad_(True)
    f = logprob_device.token_logprobs(leaf, t, avail, top_k=3)
    assert not f.top_logp.requires_grad and not f.lse.requires_grad
    ((f.logp * g).sum() + (f.entropy * h).sum()).backward()
    e = logprob_device.token_logprobs_fwd(l, t, avail)
    both = logprob_device.token_logprobs_bwd(l, t, e.lse, e.entropy, g, h, avail)
    assert same(leaf.grad, both) and bool(th.isnan(both[1]).any())
    for k, (gg, hh) in enumerate(((g, None), (None, h))):
        leaf.grad = None
        f = logprob_device.token_logprobs(leaf, t, avail)
        (f[k] * (g, h)[k]).sum().backward()
        assert same(leaf.grad, logprob_device.token_logprobs_bwd(l, t, e.lse, e.entropy, gg, hh, avail))
    v = th.randn(l.shape, device="cuda", dtype=th.float64, generator=th.Generator(device="cuda").manual_seed(1)) * avail
    keep = th.arange(40, device="cuda") != 1
    l, t, avail, g, h, v, both = (x[keep] for x in (l, t, avail, g, h, v, both))
    loss = lambda x: (lambda w: (w[0] * g).sum() + (w[1] * h).sum())(_reference(x, t, avail, g, h)[1])
    step = 1e-4
    slope = float((loss(l.double() + step * v) - loss(l.double() - step * v)) / (2 * step))
    assert abs(slope - float((both.double() * v).sum())) <= 1e-5 * float((both.double() * v).abs().sum())
    assert not logprob_device.token_logprobs(l, t).logp.requires_grad


def test_outputs_changed_in_place():
    from marl_amd.utils.logprob_device import token_logprobs
    l, t, _, g1, g2 = _inputs(40, 9, th.float32, None)
    grads = []
    for in_place in (False, True):
        x = l.clone().requires_grad_()
        f = token_logprobs(x, t)
        (f.logp.mul_(g1) if in_place else f.logp * g1).sum().backward()
        grads.append(x.grad)
    assert th.equal(*grads)
    with th.no_grad():
        f = token_logprobs(l, t)
    w = g1.clone().requires_grad_()
    f.logp.mul_(w).add_(f.entropy.mul_(g2)).sum().backward()   # (no gradient of logits: plain tensors)
    assert w.grad is not None


def test_matches_the_learners_own_evaluation():
    """PPOAgent.evaluate_actions' formulas (masked_fill, softmax, Categorical) on the env's int32 masks"""
    from torch.distributions import Categorical
    from marl_amd.utils import logprob_device
    g = th.Generator(device="cuda").manual_seed(0)
    outs = th.randn(6, 20, 10, 11, device="cuda", generator=g)
    avail = (th.rand(6, 20, 10, 11, device="cuda", generator=g) < 0.5).int()
    avail[..., -1] = 1
    dist = Categorical(th.softmax(outs.double().masked_fill(avail == 0, -1e10), -1))
    acts = dist.sample()
    f = logprob_device.token_logprobs_fwd(outs, acts, avail)
    assert float((f.logp - dist.log_prob(acts)).abs().max()) <= 200 * U * (1 + float(dist.log_prob(acts).abs().max()))
    assert float((f.entropy - th.special.entr(dist.probs).sum(-1)).abs().max()) <= 200 * U * (2 + 2 * math.log(11))


def test_refusals():
    from marl_amd.utils import logprob_device
    F, B = logprob_device.token_logprobs_fwd, logprob_device.token_logprobs_bwd
    l, t, avail, g, h = _inputs(6, 9, th.float32, th.bool)
    f = F(l, t, avail)
    for bad in (lambda: F(l.double(), t), lambda: F(l, t.float()), lambda: F(l, t, avail.float())):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: F(l, t[:5]), lambda: F(l, t[:, None]), lambda: F(l, t, avail[:, :8]), lambda: F(l, t, top_k=65),
                lambda: F(l, t, top_k=-1), lambda: F(l[:, :0], t), lambda: F(l[0, 0], t[0]), lambda: B(l, t, f.lse[:, 0], f.entropy, g),
                lambda: B(l, t, f.lse, f.entropy[:5], g), lambda: B(l, t, f.lse, f.entropy, g.double()),
                lambda: B(l, t, f.lse, f.entropy, g, h[:1])):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: F(l.cpu(), t), lambda: F(l, t.cpu()), lambda: F(l, t, avail.cpu())):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            bad()


@pytest.mark.parametrize("rows,vocab", [(200, 11), (40, 700), (2, 60000)])
def test_captured_and_replayed(rows, vocab):
    from marl_amd.utils import logprob_device
    F, B = logprob_device.token_logprobs_fwd, logprob_device.token_logprobs_bwd
    l, t, avail, g, h = _inputs(rows, vocab, th.float32, th.int32)
    F(l, t, avail, 5)
    graphs = []
    for _ in range(2):                      # two graphs, replayed in turn: neither uses the other's scratch
        graph = th.cuda.CUDAGraph()
        with th.cuda.graph(graph):
            with pytest.raises(RuntimeError, match="recorded"):
                logprob_device.token_logprobs(l.detach().requires_grad_(True), t)
            f = F(l, t, avail, 5)
            graphs.append((graph, f, B(l, t, f.lse, f.entropy, g, h, avail)))
    for k in range(4):
        l.copy_(_inputs(rows, vocab, th.float32, None, seed=k + 1)[0])
        graphs[k % 2][0].replay()
        graphs[1 - k % 2][0].replay()
        th.cuda.synchronize()
        e = F(l, t, avail, 5)
        d = B(l, t, e.lse, e.entropy, g, h, avail)
        for _, f, dl in graphs:
            assert all(th.equal(p, q) for p, q in zip(f, e)) and th.equal(dl, d), k


def test_offsets_past_32_bits():
    """rows of a view that lie beyond 2^31 elements, logits and mask"""
    from marl_amd.utils import logprob_device
    for vocab in (13, 6000):
        stride = 1_100_000_003
        flat = th.empty(2 * stride + vocab, dtype=th.bfloat16, device="cuda")
        mask = th.empty(2 * stride + vocab, dtype=th.uint8, device="cuda")
        l, av = flat.as_strided((3, vocab), (stride, 1)), mask.as_strided((3, vocab), (stride, 1))
        src, t, _, g, h = _inputs(3, vocab, th.bfloat16, None)
        on = th.rand(3, vocab, device="cuda") < 0.8
        l.copy_(src)
        av.copy_(on)
        a, b = (logprob_device.token_logprobs_fwd(x, t, m, 3) for x, m in ((l, av), (src, on)))
        assert all(th.equal(p, q) for p, q in zip(a, b))
        assert th.equal(logprob_device.token_logprobs_bwd(l, t, a.lse, a.entropy, g, h, av),
                        logprob_device.token_logprobs_bwd(src, t, b.lse, b.entropy, g, h, on))
        del flat, mask, l, av


def test_more_rows_than_a_launch_has_threads_along_x():
    """2^26 + 3 rows with alternatives take a wave each: 2^32 + 192 threads.  All rows hold the same 64 logits, so each has
    what a call of 64 rows, one per token, gives (the same kernel: the same bits)"""
    from marl_amd.utils.logprob_device import token_logprobs_bwd, token_logprobs_fwd
    rows, vocab = 2 ** 26 + 3, 64
    one = th.randn(1, vocab, device="cuda").bfloat16()
    each = th.arange(vocab, device="cuda")
    few = token_logprobs_fwd(one.expand(vocab, vocab), each, top_k=1)
    tokens = th.randint(0, vocab, (rows,), device="cuda")
    all_rows = one.expand(rows, vocab)
    f = token_logprobs_fwd(all_rows, tokens, top_k=1)
    assert th.equal(f.logp, few.logp[tokens])
    for name in ("entropy", "lse", "top_logp", "top_index"):
        got, want = getattr(f, name), getattr(few, name)
        assert bool((got == want[0]).all()), name
    g = th.ones(rows, device="cuda")
    d = token_logprobs_bwd(all_rows, tokens, f.lse, f.entropy, g)
    few_d = token_logprobs_bwd(one.expand(vocab, vocab), each, few.lse, few.entropy, g[:vocab])
    for a in range(0, rows, 2 ** 22):
        assert th.equal(d[a:a + 2 ** 22], few_d[tokens[a:a + 2 ** 22]]), a
