"""adamw_step, clip_coef and AdamW (csrc/ec_adamw.hip) against the formulas in float64.

Tolerances.  u = 2^-24 is half a step of fp32; every operation of the kernel is rounded once (no contraction), and 1 - beta,
lr / (1 - beta1^t) and the like once each.  m: three operations on |m| + |g|, 6 u of that.  v: all terms positive, 8 u of v;
its root 5 u.  The step lr' m / (root / bc + eps): 8 u (|m| + |g|) / denominator + 12 u of itself; the parameter: 3 u of
itself.  A parameter in 16 bits and an 8-bit state add half a step of their type (finfo.eps / 2; e4m3: 2^-4 of the value, and
half of the smallest step, 2^-10 scales, near 0; ROOT0 below); v's root is held as no less than 2^-9 scales."""
import copy
import math

import pytest
import torch as th

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
# fp32's smallest step is 2^-149: v' = v b2 + (1 - b2) g g is off by up to 2^-149 where its products underflow (three of half a
# step each, and less), and its root, near v = 0, by up to the root of that
ROOT0 = 2.0 ** -74
Q = 256
HYPER = dict(lr=1e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05)
SIZES = [1, 3, 4, 5, 255, 256, 257, 1000, 4095, 4096, 4097, 70001, 0, 12345]


def _state(sizes, dtype, bits, seed=0, scale=1e-2):
    g = th.Generator(device="cuda").manual_seed(seed)
    r = lambda n: th.randn(n, device="cuda", generator=g)
    out = [[(0.1 * r(n)).to(dtype) for n in sizes], [(scale * r(n)).to(dtype) for n in sizes]]
    if bits == 32:
        return out + [[0.3 * scale * r(n) for n in sizes], [scale ** 2 * r(n).square() for n in sizes]]
    k = [-(-n // Q) for n in sizes]
    q = lambda n, lo: (448 * th.rand(n, device="cuda", generator=g) * (1 if lo else th.sign(r(n)))).to(th.float8_e4m3fn)
    return out + [[q(n, False) for n in sizes], [q(n, True) for n in sizes]] + [
        [scale * (0.5 + th.rand(n, device="cuda", generator=g)) / 448 for n in k] for _ in range(2)]


def _values(q, s):
    return q.double().view(-1) * s.double().repeat_interleave(Q)[:q.numel()]


def _copy(lists):
    return [[t.clone() for t in ts] for ts in lists]


def _reference(lists, i, step, coef, lr, betas, eps, weight_decay):
    """float64 (p, m, v) after the step, and their tolerances before rounding to a type"""
    p, g = lists[0][i].double().view(-1), lists[1][i].double().view(-1) * coef
    if len(lists) == 4:
        m, v = lists[2][i].double().view(-1), lists[3][i].double().view(-1)
    else:
        m, v = _values(lists[2][i], lists[4][i]), _values(lists[3][i], lists[5][i]).square()
    mag = m.abs() + g.abs()
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    den = v.sqrt() / math.sqrt(1 - betas[1] ** step) + eps
    s = lr / (1 - betas[0] ** step)
    p = p * (1 - lr * weight_decay)
    tol_p = 3 * U * p.abs() + s * (8 * U * mag / den + 12 * U * m.abs() / den)
    p = p - s * m / den
    tol_p = tol_p + U * p.abs()
    return (p, m, v), (tol_p, 6 * U * mag, 8 * U * v)


def _check(got, before, step, coef=1.0, **hyper):
    for i in range(len(got[0])):
        (p, m, v), (tp, tm, tv) = _reference(before, i, step, coef, **hyper)
        n = p.numel()
        if n == 0:
            continue
        f = th.finfo(got[0][i].dtype)
        if f.bits == 16:
            tp = tp + f.eps / 2 * p.abs() + f.smallest_normal * f.eps / 2
        assert bool(((got[0][i].double().view(-1) - p).abs() <= tp + 1e-40).all()), ("p", i)
        assert th.equal(got[1][i], before[1][i])                                    # gradients are only read
        if len(got) == 4:
            assert bool(((got[2][i].double().view(-1) - m).abs() <= tm + 1e-40).all()), ("m", i)
            assert bool(((got[3][i].double().view(-1) - v).abs() <= tv + 1e-44).all()), ("v", i)
            continue
        for q, s, want, off in ((got[2][i], got[4][i], m, tm), (got[3][i], got[5][i], v.sqrt(), 5 * U * v.sqrt() + ROOT0)):
            k = s.numel()
            full = th.nn.functional.pad(want.abs(), (0, k * Q - n)).view(k, Q)
            slack = th.nn.functional.pad(off, (0, k * Q - n)).view(k, Q).amax(1)
            assert bool(((s.double() - full.amax(1) / 448).abs() <= 4 * U * s.double() + slack / 448 + 2.0 ** -126).all()), ("scale", i)
            each = s.double().repeat_interleave(Q)[:n]
            least = 2.0 ** -9 if q is got[3][i] else 2.0 ** -10
            room = th.maximum(2.0 ** -4 * want.abs(), least * each) * (1 + 1e-5) + off + 2.0 ** -126
            assert bool(((_values(q, s) - want).abs() <= room).all()), ("state", i)
            if q is got[3][i]:
                live = want > ROOT0
                assert bool((q.view(-1).float() > 0)[live].all()) and not bool(q.view(-1).float()[want == 0].any()), ("a root became 0", i)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [th.float32, th.bfloat16, th.float16])
@pytest.mark.parametrize("step", [1, 77])
def test_step_matches_the_formulas(dtype, bits, step):
    from marl_amd.utils import optim_device
    lists = _state(SIZES, dtype, bits)
    before = _copy(lists)
    assert optim_device.adamw_step(*lists, step=step, **HYPER) is None
    _check(lists, before, step, **HYPER)


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_of_mixed_types_with_clip(bits):
    """200 tensors of three types, in several launches; the norm is over all of them; twice the same bits"""
    from marl_amd.utils import optim_device
    sizes = [(37 * i * i) % 5003 + 1 for i in range(200)]
    lists = _state(sizes, th.float32, bits, seed=4)
    for k in (0, 1):
        lists[k] = [t.to((th.float32, th.bfloat16, th.float16)[i % 3]) for i, t in enumerate(lists[k])]
    before, twin = _copy(lists), _copy(lists)
    for max_norm in (1e-3, 1e6):
        norm = optim_device.adamw_step(*lists, step=5, max_norm=max_norm, **HYPER)
        want = math.sqrt(sum(float(g.double().square().sum()) for g in before[1]))
        assert abs(float(norm) - want) <= 2 * U * want
        coef = min(1.0, max_norm / (want + 1e-6))
        # (the factor is off by 4 u: of the gradient's part of every bound, which 8 u more of it covers)
        _check(lists, before, 5, coef=float(optim_device.clip_coef(before[1], max_norm)[1]), **HYPER)
        assert abs(float(optim_device.clip_coef(before[1], max_norm)[1]) - coef) <= 4 * U * coef
        optim_device.adamw_step(*twin, step=5, max_norm=max_norm, **HYPER)
        assert all(th.equal(a.view(th.uint8), b.view(th.uint8)) for x, y in zip(lists, twin) for a, b in zip(x, y))
        before, twin = _copy(lists), _copy(lists)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [th.float32, th.bfloat16])
def test_packed_tensors_at_any_alignment(dtype, bits):
    """tensors one behind the other in flat buffers, as FlatGrads lays gradients out: the bits of aligned ones; the element
    before the first and the one after the last stay as they were"""
    from marl_amd.utils import optim_device
    sizes = [1, 7, 19 * 64, 64, 4099, 256, 11 * 64, 11, 513]
    lists = _state(sizes, dtype, bits, seed=2)
    packed = []
    for ts in lists:
        ns = [t.numel() for t in ts]
        flat = th.zeros(sum(ns) + 2, dtype=ts[0].dtype, device="cuda")
        flat[0], flat[-1] = 3.0, 3.0
        cut, at = [], 1
        for t in ts:
            cut.append(flat[at:at + t.numel()])
            cut[-1].copy_(t)
            at += t.numel()
        packed.append((flat, cut))
    optim_device.adamw_step(*lists, step=3, **HYPER)
    optim_device.adamw_step(*[c for _, c in packed], step=3, **HYPER)
    for ts, (flat, cut) in zip(lists, packed):
        assert all(th.equal(a.view(th.uint8), b.contiguous().view(th.uint8)) for a, b in zip(ts, cut))
        assert float(flat[0]) == 3 and float(flat[-1]) == 3


def test_edges_of_values():
    """a gradient of zeros, a fresh state, gradients so small that squares vanish, and a NaN or inf: only its element's
    states in 32 bits, its block of 256 in 8"""
    from marl_amd.utils import optim_device
    for bits in (32, 8):
        lists = _state([1024, 1024, 1024, 1024], th.float32, bits)
        for ts in lists[2:]:
            for t in ts:
                t.copy_(th.zeros_like(t, dtype=th.float32))
        lists[1][0].zero_()
        lists[1][1].mul_(1e-25)
        lists[1][2][300], lists[1][3][301] = float("nan"), float("inf")
        before = _copy(lists)
        optim_device.adamw_step(*lists, step=1, **HYPER)
        _check([x[:2] for x in lists], [x[:2] for x in before], 1, **HYPER)
        assert th.equal(lists[0][0], before[0][0] * (1 - HYPER["lr"] * HYPER["weight_decay"]))
        for i in (2, 3):
            bad = th.isnan(lists[0][i])
            assert bool(bad[300 + i - 2]) and int(bad.sum()) == 1, (bits, i)
            if bits == 8:
                hurt = ~th.isfinite(lists[2][i].float() * lists[4][i].repeat_interleave(Q))
                assert bool(hurt[300 + i - 2]) and not bool(hurt[:256].any()) and not bool(hurt[512:].any())


def test_non_finite_norm_reaches_every_gradient():
    """as clip_grad_norm_: a NaN norm makes every parameter NaN; an infinite one scales finite gradients to 0"""
    from marl_amd.utils import optim_device
    for bad in (float("nan"), float("inf")):
        lists = _state([500, 300], th.float32, 32)
        lists[1][0][7] = bad
        before = _copy(lists)
        norm = optim_device.adamw_step(*lists, step=1, max_norm=1.0, **HYPER)
        assert not math.isfinite(float(norm))
        assert bool(th.isnan(lists[0][0][7])) and bool(th.isnan(lists[0][1]).all()) == math.isnan(bad)
        if math.isinf(bad):
            before[1] = [th.zeros_like(g) for g in before[1]]
            before[1][0][7], lists[0][0][7] = 0.0, 0.0
            (p, _, _), (tp, _, _) = _reference(before, 1, 1, 1.0, **HYPER)
            assert bool(((lists[0][1].double() - p).abs() <= tp).all())


def _net(seed=0):
    th.manual_seed(seed)
    return th.nn.Sequential(th.nn.Linear(19, 64), th.nn.LayerNorm(64), th.nn.ReLU(), th.nn.Linear(64, 11)).cuda()


@pytest.mark.parametrize("capturable", [False, True])
def test_optimiser_follows_torch(capturable):
    """eight steps of two groups against torch.optim.AdamW and clip_grad_norm_ in float64, one parameter without a gradient
    in the first three (with its own step count, unless capturable), a StepLR, a tensor of zeros elements"""
    from marl_amd.utils import optim_device
    a, b = _net(), _net().double()
    b.load_state_dict({k: v.double() for k, v in a.state_dict().items()})

    def groups(net):
        ps = list(net.parameters())
        return [dict(params=ps[:4], weight_decay=0.1), dict(params=ps[4:], lr=3e-3, weight_decay=0.0)]
    oa = optim_device.AdamW(groups(a), lr=1e-3, betas=(0.9, 0.99), max_norm=0.5, capturable=capturable)
    ob = th.optim.AdamW(groups(b), lr=1e-3, betas=(0.9, 0.99))
    sa, sb = (th.optim.lr_scheduler.StepLR(o, step_size=3, gamma=0.5) for o in (oa, ob))
    g = th.Generator(device="cuda").manual_seed(5)
    lag = list(a.parameters())[1]
    for step in range(8):
        for pa, pb in zip(a.parameters(), b.parameters()):
            pa.grad = th.randn(pa.shape, device="cuda", generator=g)
            pb.grad = pa.grad.double()
            if pa is lag and step < 3 and not capturable:
                pa.grad = pb.grad = None
        norm = th.nn.utils.clip_grad_norm_(b.parameters(), 0.5)
        oa.step()
        ob.step()
        sa.step()
        sb.step()
        assert abs(float(oa.last_norm) - float(norm)) <= 4 * U * float(norm)
        for pa, pb in zip(a.parameters(), b.parameters()):
            # each step adds (20 + 6) u of a step of at most 10 lr and 4 u of the parameter (see the module's bounds; the
            # moments' own errors enter through m / root, 8 steps of 14 u)
            tol = (step + 1) * (4 * U * pb.abs() + 10 * 3e-3 * 140 * U)
            assert bool(((pa.double() - pb).abs() <= tol).all()), step
            if pa in oa.state:
                assert float(oa.state[pa]["step"]) == float(ob.state[pb]["step"])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("capturable", [False, True])
def test_state_dict_round_trip(bits, capturable, tmp_path):
    """saved, loaded with weights_only, and continued: the same bits as the optimiser that went on; bf16 parameters keep
    their float32 states"""
    from marl_amd.utils import optim_device
    nets = [_net().bfloat16() for _ in range(2)]
    make = lambda n: optim_device.AdamW(n.parameters(), lr=1e-2, state_bits=bits, capturable=capturable, max_norm=1.0)
    opts = [make(n) for n in nets]
    g = th.Generator(device="cuda").manual_seed(5)

    def step(n, o, seed):
        g.manual_seed(seed)
        for p in n.parameters():
            p.grad = th.randn(p.shape, device="cuda", generator=g).bfloat16()
        o.step()
    for k in range(3):
        step(nets[0], opts[0], k)
    th.save([nets[0].state_dict(), opts[0].state_dict()], tmp_path / "o.th")
    net_sd, opt_sd = th.load(tmp_path / "o.th", map_location="cpu", weights_only=True)
    nets[1].load_state_dict(net_sd)
    opts[1].load_state_dict(opt_sd)
    for k in range(3, 6):
        step(nets[0], opts[0], k)
        step(nets[1], opts[1], k)
    for pa, pb in zip(nets[0].parameters(), nets[1].parameters()):
        assert th.equal(pa, pb)
        assert set(opts[0].state[pa]) == set(opts[1].state[pb])
        for k, v in opts[0].state[pa].items():
            w = opts[1].state[pb][k]
            assert (v == w) if not isinstance(v, th.Tensor) else (v.dtype == w.dtype and th.equal(v.reshape(-1).view(th.uint8), w.reshape(-1).view(th.uint8))), k
    if capturable:
        counts = {id(opts[1].state[p]["step"]) for p in nets[1].parameters()}
        assert len(counts) == 1 and float(opts[1].state[next(nets[1].parameters())]["step"]) == 6
    clone = copy.deepcopy(opts[0])
    assert clone.max_norm == 1.0


def test_loads_the_state_of_torch_adamw():
    """a checkpoint of torch.optim.AdamW, and the next step equals torch's; 32-bit states are refused by an 8-bit optimiser"""
    from marl_amd.utils import optim_device
    a, b = _net(), _net()
    ob = th.optim.AdamW(b.parameters(), lr=1e-3)
    g = th.Generator(device="cuda").manual_seed(5)

    def grads():
        for pa, pb in zip(a.parameters(), b.parameters()):
            pa.grad = th.randn(pa.shape, device="cuda", generator=g)
            pb.grad = pa.grad.clone()
    grads()
    ob.step()
    a.load_state_dict(b.state_dict())
    oa = optim_device.AdamW(a.parameters(), lr=5.0)
    oa.load_state_dict(ob.state_dict())
    grads()
    oa.step()
    ob.step()
    for pa, pb in zip(a.parameters(), b.parameters()):
        # the step (at most 10 lr) to 40 u on either side, and 4 u of the parameter
        assert bool(((pa - pb).abs() <= 80 * U * 1e-2 + 8 * U * pb.abs()).all())
        assert oa.state[pa]["step"] == 2 and th.equal(oa.state[pa]["exp_avg_sq"] > 0, ob.state[pb]["exp_avg_sq"] > 0)
    q = optim_device.AdamW(a.parameters(), state_bits=8)
    with pytest.raises(ValueError, match="8 bits"):
        q.load_state_dict(ob.state_dict())


def test_200_steps_stay_finite():
    """a least-squares problem of 4096 unknowns with either kind of state: everything stays finite, the types and the count hold"""
    from marl_amd.utils import optim_device
    g = th.Generator(device="cuda").manual_seed(0)
    want = th.randn(4096, device="cuda", generator=g)
    for bits in (32, 8):
        w = th.zeros(4096, device="cuda", requires_grad=True)
        opt = optim_device.AdamW([w], lr=2e-2, weight_decay=0.0, state_bits=bits)
        for _ in range(200):
            opt.zero_grad()
            (w - want).square().mean().backward()
            opt.step()
        assert bool(th.isfinite(w.detach()).all()) and opt.state[w]["exp_avg"].dtype == (th.float32 if bits == 32 else th.float8_e4m3fn)
        assert opt.state[w]["step"] == 200


def test_captured_and_replayed():
    """steps in two HIP graphs with device step counts and a device learning rate: every replay equals the eager step"""
    from marl_amd.utils import optim_device
    for bits in (32, 8):
        nets = [_net() for _ in range(2)]
        lrs = [th.full((), 1e-2, device="cuda") for _ in nets]
        opts = [optim_device.AdamW(n.parameters(), lr=lr, state_bits=bits, capturable=True, max_norm=1.0) for n, lr in zip(nets, lrs)]
        for n in nets:
            for p in n.parameters():
                p.grad = th.zeros_like(p)
        graph = th.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="first step"):
            with th.cuda.graph(graph):
                opts[0].step()
        for o in opts:
            o.step()
        graphs = [th.cuda.CUDAGraph() for _ in range(2)]
        for gr in graphs:
            with th.cuda.graph(gr):
                opts[0].step()
        g = th.Generator(device="cuda").manual_seed(5)
        for k in range(5):
            for pa, pb in zip(nets[0].parameters(), nets[1].parameters()):
                pa.grad.copy_(th.randn(pa.shape, device="cuda", generator=g))
                pb.grad.copy_(pa.grad)
            for lr in lrs:
                lr.fill_(1e-2 / (k + 1))
            graphs[k % 2].replay()
            opts[1].step()
            th.cuda.synchronize()
            for pa, pb in zip(nets[0].parameters(), nets[1].parameters()):
                assert th.equal(pa, pb), k
                assert float(opts[0].state[pa]["step"]) == k + 2
        with pytest.raises(RuntimeError, match="step count on the device"):
            with th.cuda.graph(th.cuda.CUDAGraph()):
                ps = [p.data for p in nets[1].parameters()]
                optim_device.adamw_step(ps, ps, ps, ps, step=1, lr=1e-3)


@pytest.mark.parametrize("sizes,dtypes", [
    ([1], [th.float32]), ([32768], [th.float32]), ([32769], [th.float32]), ([1023, 0, 1025, 7, 5000], [th.float32]),
    ([5, 2049, 4097], [th.bfloat16]), ([300, 4001], [th.float16]), ([300, 4001], [th.float32, th.bfloat16]), ([17] * 48, [th.float32]),
    ([17] * 49, [th.bfloat16]), ([8191, 8193, 70001], [th.float16])])
def test_the_norm_of_few_and_of_many(sizes, dtypes):
    """one block's sum (few elements of one type) and the joined ones; gradients at odd addresses.  The squares are exact in
    double, their sum is off by less than 2^-36 of itself: what is left are the rounding of the norm to fp32, and for the
    coefficient those of the sum and the quotient too"""
    from marl_amd.utils.optim_device import clip_coef
    gen = th.Generator(device="cuda").manual_seed(sum(sizes))
    grads = [th.randn(n + 1, device="cuda", generator=gen).to(dtypes[i % len(dtypes)])[1:] for i, n in enumerate(sizes)]
    want = float(th.cat([g.double() for g in grads]).norm())
    for max_norm in (0.5 * want, 2 * want + 1):
        norm, coef = (float(t) for t in clip_coef(grads, max_norm))
        assert abs(norm - want) <= 1.01 * U * want
        exact = min(1.0, max_norm / (want + 1e-6))
        assert abs(coef - exact) <= 5 * U * exact, (coef, exact)
        assert (norm, coef) == tuple(float(t) for t in clip_coef(grads, max_norm))
    grads[-1][-1] = float("nan")
    norm, coef = clip_coef(grads, 1.0)
    assert norm.isnan() and coef.isnan()



def test_refusals():
    from marl_amd.utils import optim_device
    S = optim_device.adamw_step
    P, G, M, V = _state([10, 300], th.float32, 32)
    before = _copy([P, G, M, V])
    one = th.ones((), device="cuda")
    bad = [lambda: S(P, G[:1], M, V, step=1, lr=1e-3), lambda: S(P, [g.bfloat16() for g in G], M, V, step=1, lr=1e-3),
           lambda: S(P, G, [m.half() for m in M], V, step=1, lr=1e-3), lambda: S(P, [g[:5] for g in G], M, V, step=1, lr=1e-3),
           lambda: S([P[0], P[0]], [G[0], G[0]], [M[0], M[0]], [V[0], V[0]], step=1, lr=1e-3),
           lambda: S(P, G, [M[1][:10], M[1]], V, step=1, lr=1e-3), lambda: S(P, G, M, [V[1][:10], V[1]], step=1, lr=1e-3),
           lambda: S([p.double() for p in P], G, M, V, step=1, lr=1e-3), lambda: S(P, G, M, V, step=0, lr=1e-3),
           lambda: S(P, G, M, V, step=1, lr=-1e-3), lambda: S(P, G, M, V, step=1, lr=1e-3, betas=(1.0, 0.9)),
           lambda: S(P, G, M, V, step=1, lr=1e-3, eps=-1.0), lambda: S(P, G, M, V, step=1, lr=1e-3, weight_decay=-1.0),
           lambda: S(P, G, M, V, step=1, lr=float("nan")), lambda: S(P, G, M, V, step=1, lr=one),
           lambda: S(P, G, M, V, step=one.double(), lr=1e-3), lambda: S(P, G, M, V, step=1, lr=1e-3, max_norm=0.0),
           lambda: S(P, G, M, V, step=1, lr=1e-3, max_norm=1.0, coef=one), lambda: S(P, G, M, V, step=1, lr=1e-3, coef=th.ones(2, device="cuda")),
           lambda: S(P, G, M, V, M, None, step=1, lr=1e-3), lambda: S(P, G, M, V, None, M, step=1, lr=1e-3),
           lambda: S(P, G, M, V, M, V, step=1, lr=1e-3), lambda: S([], [], [], [], step=1, lr=1e-3),
           lambda: S([th.zeros(4, 6, device="cuda").t()], [th.zeros(6, 4, device="cuda")], [th.zeros(6, 4, device="cuda")],
                     [th.zeros(6, 4, device="cuda")], step=1, lr=1e-3), lambda: optim_device.clip_coef(G, float("nan"))]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail("not refused: %d" % i)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        S([p.cpu() for p in P], G, M, V, step=1, lr=1e-3)
    assert all(th.equal(a, b) for x, y in zip([P, G, M, V], before) for a, b in zip(x, y))
    w = th.zeros(4, 6, device="cuda", requires_grad=True)
    for kw in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(max_norm=-1.0), dict(lr=one)):
        with pytest.raises(ValueError):
            optim_device.AdamW([w], **kw)
    for p in (th.zeros(4, 6, device="cuda").t().requires_grad_(True), w.detach().double().requires_grad_(True)):
        with pytest.raises(ValueError):
            optim_device.AdamW([p])
    opt = optim_device.AdamW([w])
    opt.step()                               # no gradients: nothing to do
    w.grad = th.zeros(6, 4, device="cuda").t()
    opt.step()                               # a gradient of other strides
    assert opt.state[w]["step"] == 1 and w._version > 0
