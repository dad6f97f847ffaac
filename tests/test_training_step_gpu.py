"""Layer norm, token log-probs and AdamW together, as an update step of a policy of any width uses them: against the same step
in float64 torch, and recorded into a HIP graph."""
import copy

import pytest
import torch as th

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


class _Policy(th.nn.Module):
    """rows -> width -> layer norm -> actions; `hip`: with the framework's layer norm"""

    def __init__(self, n_in, width, n_out):
        super().__init__()
        self.fc1, self.ln, self.fc2 = th.nn.Linear(n_in, width), th.nn.LayerNorm(width), th.nn.Linear(width, n_out)

    def forward(self, x, hip):
        h = self.fc1(x)
        if hip:
            from marl_amd.utils import norm_device
            h = norm_device.layer_norm(h, self.ln.weight, self.ln.bias, self.ln.eps)
        else:
            h = self.ln(h)
        return self.fc2(th.relu(h))


def _batch(rows, n_out, seed):
    g = th.Generator().manual_seed(seed)
    x = th.randn(rows, 19, generator=g)
    avail = (th.rand(rows, n_out, generator=g) < 0.6).int()
    avail[:, -1] = 1
    act = th.multinomial(avail.float(), 1, generator=g)[:, 0]
    return x, avail, act, 0.1 * th.randn(rows, generator=g) - 2.0, th.randn(rows, generator=g)


def _objective(logp, entropy, old, adv):
    ratio = th.exp(logp - old)
    return -(th.min(ratio * adv, ratio.clamp(0.8, 1.2) * adv) + 0.01 * entropy).mean()


@pytest.mark.parametrize("width,n_out", [(100, 41), (256, 1000)])
def test_ppo_steps_follow_float64(width, n_out):
    from marl_amd.utils import logprob_device, optim_device
    th.manual_seed(1)
    ref = _Policy(19, width, n_out).double()
    net = copy.deepcopy(ref).float().cuda()
    opt = optim_device.AdamW(net.parameters(), lr=1e-3, eps=1e-5, max_norm=0.5)
    opt_ref = th.optim.AdamW(ref.parameters(), lr=1e-3, eps=1e-5)
    for step in range(3):
        # (a unit on relu's kink or a ratio on a clip border would have no gradient to compare: with these seeds the nearest
        # is 1e-6 away, ten times what fp32 rounds here)
        x, avail, act, old, adv = _batch(64, n_out, seed=10 + step)
        lp = th.log_softmax(ref(x.double(), False).masked_fill(avail == 0, -1e6), -1)
        want = _objective(lp.gather(1, act[:, None])[:, 0], -(lp.exp() * lp).sum(-1), old.double(), adv.double())
        opt_ref.zero_grad()
        want.backward()
        dev = [t.cuda() for t in (x, avail, act, old, adv)]
        f = logprob_device.token_logprobs(net(dev[0], True), dev[2], dev[1])
        got = _objective(f.logp, f.entropy, dev[3], dev[4])
        opt.zero_grad()
        got.backward()
        assert abs(float(got) - float(want)) <= 1e-4 * (1 + abs(float(want)))
        for (name, p), q in zip(net.named_parameters(), ref.parameters()):
            # a few hundred roundings of terms that add up to at most a few times the largest entry
            assert float((p.grad.cpu().double() - q.grad).abs().max()) <= 4096 * U * float(q.grad.abs().max()) + 1e-9, (step, name)
        th.nn.utils.clip_grad_norm_(ref.parameters(), 0.5)
        opt.step()
        opt_ref.step()
        for p, q in zip(net.parameters(), ref.parameters()):
            # a step moves an entry by at most a few lr; where a gradient is rounding noise around 0 the two may differ by it
            assert float((p.detach().cpu().double() - q).abs().max()) <= (step + 1) * 4e-3
            assert float((p.detach().cpu().double() - q).abs().mean()) <= (step + 1) * 2e-5


def test_on_another_stream_than_the_default():
    """inputs made, used and read on a side stream behind a long kernel there, from a thread of its own: nothing of a call runs
    on the default stream"""
    import threading

    from marl_amd.utils import logprob_device, norm_device, optim_device
    out = {}

    def work(key, stream):
        with th.cuda.stream(stream):
            g = th.Generator(device="cuda").manual_seed(3)
            a = th.randn(4096, 4096, device="cuda", generator=g)
            x = th.zeros(500, 700, device="cuda")
            busy = a
            for _ in range(4):
                busy = busy @ a * 1e-3
            x.copy_(th.randn(500, 700, device="cuda", generator=g))        # (behind the products)
            w = th.ones(700, device="cuda").requires_grad_(True)
            tok = th.arange(500, device="cuda")
            f = logprob_device.token_logprobs(norm_device.layer_norm(x, w), tok, top_k=3)
            f.logp.sum().backward()
            opt = optim_device.AdamW([w], lr=0.1, max_norm=1.0)
            opt.step()
            out[key] = [t.detach().cpu() for t in (f.logp, f.entropy, f.top_logp, f.top_index, w.grad, w, opt.last_norm)]
    threads = [threading.Thread(target=work, args=(k, th.cuda.Stream())) for k in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    work("default", th.cuda.default_stream())
    for k in range(2):
        assert all(th.equal(p, q) for p, q in zip(out[k], out["default"]))


def test_an_update_step_in_a_graph():
    """the passes by hand, with clip and AdamW, recorded once and replayed on new batches: the bits of the eager steps"""
    from marl_amd.utils import logprob_device, norm_device, optim_device
    rows, width, vocab = 96, 128, 300
    g = th.Generator(device="cuda").manual_seed(0)
    r = lambda *s: th.randn(*s, device="cuda", generator=g)
    data = dict(h=r(rows, width), tok=th.randint(0, vocab, (rows,), device="cuda", generator=g), adv=r(rows))

    def make():
        g2 = th.Generator(device="cuda").manual_seed(7)
        ps = [(th.ones(width, device="cuda")), th.zeros(width, device="cuda"), 0.1 * th.randn(vocab, width, device="cuda", generator=g2)]
        return ps, [th.zeros_like(p) for p in ps], [th.zeros_like(p) for p in ps], th.zeros((), device="cuda")

    def update(ps, m, v, count):
        y, mean, rstd = norm_device.layer_norm_fwd(data["h"], ps[0], ps[1])
        logits = y @ ps[2].t()
        f = logprob_device.token_logprobs_fwd(logits, data["tok"])
        dl = logprob_device.token_logprobs_bwd(logits, data["tok"], f.lse, f.entropy, -data["adv"] / rows, None)
        dw2 = dl.t() @ y
        _, dw, db = norm_device.layer_norm_bwd(dl @ ps[2], data["h"], mean, rstd, ps[0])
        norm = optim_device.adamw_step(ps, [dw, db, dw2], m, v, step=count, lr=1e-2, max_norm=1.0)
        return f.logp, norm
    a, b = make(), make()
    for _ in range(2):                       # warm: the GEMM library's workspaces
        update(*make())
    graph = th.cuda.CUDAGraph()
    with th.cuda.graph(graph):
        logp, norm = update(*a)
    for k in range(5):
        data["h"].copy_(r(rows, width))
        data["adv"].copy_(r(rows))
        graph.replay()
        want_logp, want_norm = update(*b)
        th.cuda.synchronize()
        assert th.equal(logp, want_logp) and th.equal(norm, want_norm), k
        assert all(th.equal(p, q) for x, y in zip(a[:3], b[:3]) for p, q in zip(x, y)) and float(a[3]) == k + 1, k
