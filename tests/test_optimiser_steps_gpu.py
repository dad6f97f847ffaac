"""optim_device.AdamW's steps where parameters have gradients at different times, where a call is refused half way, and where
loaded states are continued: against torch.optim.AdamW in float64, or against itself bit for bit.

Tolerance of a parameter after k steps, u = 2^-24: each step adds 4 u of the parameter and 26 u of a step of at most 10 lr,
and the moments carry at most 14 u of themselves from each of the steps before into it: k (4 u |p| + 10 lr (26 + 14 k) u)."""
import copy

import pytest
import torch as th

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
SHAPES = [(19, 64), (64,), (64, 11), (11,), (300,)]


def _params(seed=0, dtype=th.float32):
    g = th.Generator(device="cuda").manual_seed(seed)
    return [th.nn.Parameter((0.1 * th.randn(s, device="cuda", generator=g)).to(dtype)) for s in SHAPES]


def _grads(ps, seed, live=None):
    g = th.Generator(device="cuda").manual_seed(seed)
    for i, p in enumerate(ps):
        x = th.randn(p.shape, device="cuda", generator=g)
        p.grad = x.to(p.dtype) if live is None or i in live else None


def _follows(a, b, steps, lr):
    for pa, pb in zip(a, b):
        tol = steps * (4 * U * pb.abs() + 10 * lr * (26 + 14 * steps) * U)
        assert bool(((pa.double() - pb).abs() <= tol).all()), steps


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("capturable", [False, True])
def test_gradients_that_come_and_go(capturable, bits):
    """parameters that get their first gradient late, or none for some steps: each follows its own count, as torch's do"""
    from marl_amd.utils.optim_device import AdamW
    a = _params()
    b = [th.nn.Parameter(p.detach().double()) for p in a]
    kw = dict(lr=1e-3, betas=(0.9, 0.99), weight_decay=0.1)
    oa, ob = AdamW(a, **kw, capturable=capturable, state_bits=bits), th.optim.AdamW(b, **kw)
    for step, live in enumerate(([0, 1], [0, 1], [0, 1, 2, 3], [1, 2], [0, 1, 2, 3, 4], [4], [0, 1, 2, 3, 4], [0, 1, 2, 3, 4])):
        _grads(a, step, live)
        for pa, pb in zip(a, b):
            pb.grad = pa.grad.double() if pa.grad is not None else None
        oa.step()
        ob.step()
        assert [float(oa.state[p]["step"]) for p in a if p in oa.state] == [float(ob.state[p]["step"]) for p in b if p in ob.state]
        if bits == 32:
            _follows(a, b, step + 1, 1e-3)
        else:
            # a first step's moments are those of its gradient, not yet rounded: lr (1 +- the rounding), as torch's
            for pa, pb in zip(a, b):
                if pb in ob.state and float(ob.state[pb]["step"]) == 1 and pb.grad is not None:
                    _follows([pa], [pb], 1, 1e-3)


def test_a_count_that_a_graph_advances_is_not_split():
    """parameters that share a count go on together once a HIP graph has recorded it: a step of some of them alone is refused
    (and leaves everything as it was), as it is while a graph is recorded; a graph of a part has its own count"""
    from marl_amd.utils.optim_device import AdamW
    a, b = _params(), _params()
    oa, ob = (AdamW(ps, lr=1e-2, capturable=True, max_norm=1.0) for ps in (a, b))
    for ps, o in ((a, oa), (b, ob)):
        _grads(ps, 1)
        o.step()
        _grads(ps, 2, [0, 1, 2])        # from here on 3 and 4 have a count of their own
        o.step()
        _grads(ps, 3)
    with pytest.raises(RuntimeError, match="share a step count"):
        a[0].grad, kept = None, a[0].grad
        with th.cuda.graph(th.cuda.CUDAGraph()):
            oa.step()
    a[0].grad = kept
    graph = th.cuda.CUDAGraph()
    with th.cuda.graph(graph):
        oa.step()
    for k in range(3):
        _grads(b, 3)
        graph.replay()
        ob.step()
        th.cuda.synchronize()
        assert all(th.equal(x, y) for x, y in zip(a, b)), k
        assert [float(oa.state[p]["step"]) for p in a] == [float(ob.state[p]["step"]) for p in b] == [3 + k] * 3 + [2 + k] * 2
    before = copy.deepcopy(oa.state_dict()), [p.detach().clone() for p in a]
    a[4].grad = None
    with pytest.raises(RuntimeError, match="share a step count"):
        oa.step()
    after = oa.state_dict()["state"]
    assert all(th.equal(x, y) for x, y in zip(a, before[1]))
    assert all(th.equal(after[i][k], v) for i, st in before[0]["state"].items() for k, v in st.items())
    a[3].grad = None                    # neither of those two: nothing is split
    oa.step()
    assert [float(oa.state[p]["step"]) for p in a] == [6] * 3 + [4] * 2


def test_a_checkpoint_on_the_host_continues_with_a_learning_rate_on_the_device(tmp_path):
    """saved, loaded with map_location="cpu" and continued, recorded into a HIP graph: the bits of the optimiser that went on"""
    from marl_amd.utils.optim_device import AdamW
    a, b = _params(), _params()
    oa, ob = (AdamW(ps, lr=th.full((), 1e-2, device="cuda"), capturable=True) for ps in (a, b))
    _grads(a, 0)
    oa.step()
    th.save([[p.detach() for p in a], oa.state_dict()], tmp_path / "o.th")
    ps, saved = th.load(tmp_path / "o.th", map_location="cpu", weights_only=True)
    for p, q in zip(b, ps):
        p.data.copy_(q)
    ob.load_state_dict(saved)
    lr = ob.param_groups[0]["lr"]
    assert lr.device == b[0].device and lr.dtype == th.float32
    _grads(b, 1)
    graph = th.cuda.CUDAGraph()
    with th.cuda.graph(graph):
        ob.step()
    for k in range(1, 5):
        _grads(a, k)
        for p, q in zip(a, b):
            q.grad.copy_(p.grad)
        oa.param_groups[0]["lr"].fill_(1e-2 / k)
        lr.fill_(1e-2 / k)
        graph.replay()
        oa.step()
        th.cuda.synchronize()
        assert all(th.equal(p, q) for p, q in zip(a, b)), k


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("what", ["lr", "betas", "state", "parameter", "gradient", "option"])
def test_a_step_that_is_refused_has_done_nothing(what, bits):
    """something wrong in the last of two groups: no parameter, state, count or norm changes in either; put right, the step is
    the one of an optimiser that met no refusal"""
    from marl_amd.utils.optim_device import AdamW
    a, b = _params(), _params()
    oa, ob = (AdamW([dict(params=ps[:2]), dict(params=ps[2:])], max_norm=1.0, state_bits=bits) for ps in (a, b))
    for ps, o in ((a, oa), (b, ob)):
        _grads(ps, 0)
        o.step()
        _grads(ps, 1)
    before = copy.deepcopy(oa.state_dict()), [p.detach().clone() for p in a], oa.last_norm
    group, st = oa.param_groups[1], oa.state[a[4]]
    kept = dict(group), dict(st), a[4].data, a[4].grad
    if what == "lr":
        group["lr"] = -1.0
    elif what == "betas":
        group["betas"] = (0.9, 1.0)
    elif what == "state":
        st["exp_avg_sq"] = st["exp_avg_sq"][:-1].clone()
    elif what == "parameter":
        a[4].data = th.zeros(600, device="cuda")[::2]
    elif what == "gradient":
        a[4].grad = None
        a[4].grad_dtype = None
        a[4].grad = kept[3].bfloat16()
    else:
        group["maximize"] = True
    with pytest.raises(ValueError):
        oa.step()
    a[4].data = kept[2]
    a[4].grad = kept[3]
    st.update(kept[1])
    group.update(kept[0])
    group.pop("maximize", None) if what == "option" else None
    assert oa.last_norm is before[2] and all(th.equal(p, q) for p, q in zip(a, before[1]))
    for i, s in oa.state_dict()["state"].items():
        assert all(th.equal(v.view(-1).view(th.uint8), w.view(-1).view(th.uint8)) if isinstance(v, th.Tensor) else v == w
                   for v, w in zip(s.values(), before[0]["state"][i].values()))
    oa.step()
    ob.step()
    assert all(th.equal(p, q) for p, q in zip(a, b)) and th.equal(oa.last_norm, ob.last_norm)
