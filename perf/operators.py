"""The operators of a policy's training step, as they are measured: layer norm, log-probs of given tokens (actions) with
entropy and top alternatives, and AdamW over many tensors.  `run` computes them in plain torch operations, or (own = True)
through marl_amd's entry points, on the same inputs."""
import math
import random

import torch as th

own = False  # set by whoever imports this file

DT = {"float32": th.float32, "bfloat16": th.bfloat16, "float16": th.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}
QBLOCK = 256      # elements that share a scale in the 8-bit optimiser states
QMAX = 448.0      # e4m3's largest value
QMIN = 2.0 ** -9  # and its smallest positive one
F8 = th.float8_e4m3fn
BETAS, EPS, DECAY, LR = (0.9, 0.999), 1e-8, 1e-2, 1e-4
NORM_EPS = 1e-5


# ---- the cases ---------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token of a policy that answers step by step: latency
        dict(name="norm_one_row", op="norm", train=False, rows=1, cols=4096, dtype="bfloat16", wdtype="bfloat16", pad=0),
        # an update over a whole rollout of 4096 envs x 100 steps x 10 agents, hidden width 64
        dict(name="norm_rollout_64", op="norm", train=True, rows=4096000, cols=64, dtype="float32", wdtype="float32", pad=0),
        # a training batch of a wide sequence policy
        dict(name="norm_wide_batch", op="norm", train=True, rows=16384, cols=4096, dtype="bfloat16", wdtype="float32", pad=0),
        # odd width, rows that are a view of a wider buffer
        dict(name="norm_odd_view", op="norm", train=True, rows=4999, cols=2053, dtype="float16", wdtype="float16", pad=10),
        # an update over a whole rollout: 11 actions (10 nodes), the env's int32 action masks
        dict(name="logp_rollout_11", op="logp", train=True, rows=4096000, vocab=11, dtype="float32", mask="int32", top_k=0),
        # answers with their alternatives for a few requests: latency of long rows
        dict(name="logp_answer", op="logp", train=False, rows=4, vocab=131072, dtype="bfloat16", mask="", top_k=20),
        # a training batch with a large vocabulary, padded rows among it
        dict(name="logp_wide_batch", op="logp", train=True, rows=8192, vocab=65536, dtype="bfloat16", mask="", top_k=0),
        # odd vocabulary under a mask, alternatives for the log
        dict(name="logp_odd_masked", op="logp", train=True, rows=1009, vocab=50021, dtype="float32", mask="bool", top_k=5),
        # the six tensors of a 64-wide policy network: latency
        dict(name="adamw_policy", op="adamw", net="policy", width=64, dtype="float32", bits=32, max_norm=10.0),
        # a network of 12 blocks, 1024 wide, states in 32 bits
        dict(name="adamw_blocks_32", op="adamw", net="blocks", width=1024, layers=12, dtype="float32", bits=32, max_norm=0.0),
        # 4 blocks, 2048 wide, weights in bf16, states in 8 bits, clipped
        dict(name="adamw_blocks_8", op="adamw", net="blocks", width=2048, layers=4, dtype="bfloat16", bits=8, max_norm=1.0),
        # ninety tensors of odd sizes, packed one behind the other in one buffer
        dict(name="adamw_packed_8", op="adamw", net="packed", tensors=90, total=8_000_001, dtype="float32", bits=8, max_norm=0.0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "logp", "adamw"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if op == "norm":
        cols = _log_int(rng, 4, 16384)
        if rng.random() < 0.5 and cols > 8:
            cols -= cols % 8
        rows = _log_int(rng, 1, max(1, min(4000000, (1 << 27) // cols)))
        return dict(op=op, train=rng.random() < 0.7, rows=rows, cols=cols, dtype=dtype,
                    wdtype=rng.choice([dtype, "float32"]), pad=rng.choice([0, 0, 3, 16]))
    if op == "logp":
        vocab = _log_int(rng, 2, 262144)
        if rng.random() < 0.5 and vocab > 8:
            vocab -= vocab % 8
        rows = _log_int(rng, 1, max(1, min(4000000, (1 << 26) // vocab)))
        return dict(op=op, train=rng.random() < 0.6, rows=rows, vocab=vocab, dtype=dtype,
                    mask=rng.choice(["", "", "int32", "bool"]), top_k=rng.choice([0, 0, 1, 5, 20]))
    return dict(op=op, net="packed", tensors=_log_int(rng, 1, 200), total=_log_int(rng, 4000, 1 << 26),
                dtype=dtype, bits=rng.choice([32, 8]), max_norm=rng.choice([0.0, 1.0]))


def _shapes(case):
    w = case.get("width")
    if case["net"] == "policy":    # 9 observations + 10 agent ids -> w -> w -> 11 actions
        return [(w, 19), (w,), (w, w), (w,), (11, w), (11,)]
    if case["net"] == "blocks":
        one = [(w,), (w,), (w, w), (w, w), (w, w), (w, w), (w,), (w,), (4 * w, w), (4 * w,), (w, 4 * w), (w,)]
        return one * case["layers"]
    r = random.Random(case["total"] * 1000 + case["tensors"])
    share = [math.exp(r.uniform(0.0, 4.0)) for _ in range(case["tensors"])]
    return [(max(1, int(case["total"] * s / sum(share))),) for s in share]


def _places(case):
    """offset of every tensor in the flat buffers, offset of its scales, and both totals"""
    step = 1 if case["net"] == "packed" else 64
    at, blk, places = 0, 0, []
    for s in _shapes(case):
        n = math.prod(s)
        places.append((s, n, at, blk))
        at += -(-n // step) * step
        blk += -(-n // QBLOCK)
    return places, at, blk


def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "norm":
        n, c = case["rows"] * case["cols"], case["cols"] * SIZE[case["wdtype"]]
        if case["train"]:
            return {"bytes": 5.0 * n * e + 4 * c, "flops": 22.0 * n}
        return {"bytes": 2.0 * n * e + 2 * c, "flops": 8.0 * n}
    if case["op"] == "logp":
        n, r = float(case["rows"] * case["vocab"]), case["rows"]
        once = n * (e + {"": 0, "int32": 4, "bool": 1}[case["mask"]])
        small = r * (8.0 + 8 + 12 * case["top_k"])
        if case["train"]:   # each input once, though the gradient needs what the whole forward pass leaves
            return {"bytes": once + n * e + small + 8 * r, "flops": 14.0 * n}
        return {"bytes": once + small, "flops": 7.0 * n}
    n = float(sum(math.prod(s) for s in _shapes(case)))
    if case["bits"] == 32:
        return {"bytes": n * (3 * e + 16), "flops": 16.0 * n}
    return {"bytes": n * (3 * e + 4 + 16.0 / QBLOCK), "flops": 26.0 * n}


# ---- their inputs ------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = th.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: th.rand(*s, device="cuda", generator=g)      # noqa: E731
    randn = lambda *s: th.randn(*s, device="cuda", generator=g)    # noqa: E731
    dt = DT[case["dtype"]]
    if case["op"] == "norm":
        r, c, wt = case["rows"], case["cols"], DT[case["wdtype"]]
        x = randn(r, c + case["pad"])
        x.mul_(0.5 + rand(r, 1)).add_(randn(r, 1))
        s = dict(case=case, x=x.to(dt)[:, :c], w=(1 + 0.2 * randn(c)).to(wt), b=(0.2 * randn(c)).to(wt))
        if case["train"]:
            s["dy"] = randn(r, c).to(dt)
        return s
    if case["op"] == "logp":
        r, v = case["rows"], case["vocab"]
        s = dict(case=case, logits=randn(r, v).mul_(3).to(dt), avail=None)
        s["tokens"] = th.randint(0, v, (r,), device="cuda", generator=g)
        if case["mask"]:
            s["tokens"][: r // 2] = s["logits"][: r // 2].argmax(-1)   # (half of them likely ones)
            on = rand(r, v) < 0.6
            on[th.arange(r, device="cuda"), s["tokens"]] = True        # what was taken was available
            on[::97] &= rand(on[::97].shape[0], 1) < 0.5               # and a few rows with nothing available
            low = th.tensor([float("nan"), float("inf"), th.finfo(dt).min], device="cuda", dtype=dt)
            k = th.arange(0, r * v, 1013, device="cuda")               # masked places hold anything
            flat, off = s["logits"].view(-1), ~on.view(-1)
            flat[k] = th.where(off[k], low[k % 3], flat[k])
            s["avail"] = on if case["mask"] == "bool" else on.to(th.int32)
        else:
            s["tokens"][::10] = -100                                   # padded rows
        if case["train"]:
            s["dlogp"], s["dent"] = randn(r), 0.01 * randn(r)           # (a loss scaled up, as fp16 needs it)
        return s
    places, n, blocks = _places(case)
    pad = th.ones(n, dtype=th.bool, device="cuda")
    for _, m, at, _ in places:
        pad[at:at + m] = False
    flat = lambda t: t.masked_fill_(pad, 0)   # noqa: E731
    s = dict(case=case, step=100, p=flat(0.05 * randn(n)).to(dt), g=flat(1e-3 * randn(n)).to(dt))
    if case["bits"] == 32:
        s["m"], s["v"] = flat(3e-4 * randn(n)), flat(1e-6 * (0.1 + rand(n)))
    else:
        s["m"] = flat((120 * randn(n)).clamp_(-QMAX, QMAX)).to(F8)
        s["v"] = flat(150 + 250 * rand(n)).to(F8)
        s["ms"], s["vs"] = 2e-6 + 1e-6 * rand(blocks), 2e-6 + 1e-6 * rand(blocks)
    cut = lambda name: [s[name][at:at + m].view(sh) for sh, m, at, _ in places]   # noqa: E731
    s["lists"] = [cut("p"), cut("g"), cut("m"), cut("v")]
    if case["bits"] == 8:
        s["lists"] += [[s[k][b:b - (-m // QBLOCK)] for _, m, _, b in places] for k in ("ms", "vs")]
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    if case["op"] == "norm":
        return _run_norm(s, case)
    if case["op"] == "logp":
        return _run_logp(s, case)
    return _run_adamw(s, case)


def _run_norm(s, case):
    if own:
        from marl_amd.utils import norm_device
        if not case["train"]:
            return {"y": norm_device.layer_norm_fwd(s["x"], s["w"], s["b"], NORM_EPS, want_stats=False)[0]}
        y, mean, rstd = norm_device.layer_norm_fwd(s["x"], s["w"], s["b"], NORM_EPS)
        dx, dw, db = norm_device.layer_norm_bwd(s["dy"], s["x"], mean, rstd, s["w"])
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    x, w, b = s["x"].float(), s["w"].float(), s["b"].float()
    d = x - x.mean(-1, keepdim=True)
    rstd = 1.0 / th.sqrt((d * d).mean(-1, keepdim=True) + NORM_EPS)
    xhat = d * rstd
    out = {"y": (xhat * w + b).to(s["x"].dtype)}
    if case["train"]:
        dy = s["dy"].float()
        a = dy * w
        dx = rstd * (a - a.mean(-1, keepdim=True) - xhat * (a * xhat).mean(-1, keepdim=True))
        out.update(dx=dx.to(s["x"].dtype), dw=(dy * xhat).sum(0).to(s["w"].dtype), db=dy.sum(0).to(s["b"].dtype))
    return out


def _run_logp(s, case):
    if own:
        from marl_amd.utils import logprob_device
        f = logprob_device.token_logprobs_fwd(s["logits"], s["tokens"], s["avail"], top_k=case["top_k"])
        out = {"logp": f.logp, "entropy": f.entropy}
        if case["top_k"]:
            out.update(top_logp=f.top_logp, top_index=f.top_index)
        if case["train"]:
            out["dlogits"] = logprob_device.token_logprobs_bwd(s["logits"], s["tokens"], f.lse, f.entropy, s["dlogp"], s["dent"],
                                                               s["avail"])
        return out
    inf = float("inf")
    l = s["logits"].float()
    if s["avail"] is not None:
        l = l.masked_fill(s["avail"] == 0, -inf)
    top = l.max(-1, keepdim=True)[0]
    e = th.exp(l - th.where(top > -inf, top, 0.0))
    total = e.sum(-1, keepdim=True)
    lse = top + th.log(total)
    lp = th.where(l > -inf, l - lse, -inf)
    p = th.where(top > -inf, e / total, 0.0)
    finite = th.where(lp > -inf, lp, 0.0)
    ent = -(p * finite).sum(-1, keepdim=True)
    t = s["tokens"]
    taken = lp.gather(-1, t.clamp(min=0)[:, None])[:, 0]
    out = {"logp": th.where(t < 0, 0.0, taken), "entropy": ent[:, 0]}
    if case["top_k"]:
        k, v = min(case["top_k"], case["vocab"]), case["vocab"]
        bits = (l + 0.0).view(th.int32)                            # (-0 counts as 0)
        key = th.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * (1 << 32) + (v - 1 - th.arange(v, device=l.device))
        at = v - 1 - (th.topk(key, k, dim=-1)[0] & 0xFFFFFFFF)     # ties: the lowest index
        val = lp.gather(-1, at)
        at = th.where(val > -inf, at, -1)
        fill = case["top_k"] - k
        out["top_logp"] = th.cat([val, val.new_full((val.shape[0], fill), -inf)], 1)
        out["top_index"] = th.cat([at, at.new_full((at.shape[0], fill), -1)], 1)
    if case["train"]:
        g = th.where(t < 0, 0.0, s["dlogp"])[:, None]
        d = -p * (g + s["dent"][:, None] * (finite + ent))
        one = th.zeros_like(d).scatter_(1, t.clamp(min=0)[:, None], th.where(taken > -inf, g[:, 0], 0.0)[:, None])
        out["dlogits"] = (d + one).to(s["logits"].dtype)
    return out


def _run_adamw(s, case):
    s["step"] += 1
    out = {k: s[k] for k in ("p", "m", "v", "ms", "vs") if k in s}
    if own:
        from marl_amd.utils import optim_device
        norm = optim_device.adamw_step(*s["lists"], step=s["step"], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY,
                                       max_norm=case["max_norm"] or None)
    else:
        coef, norm = None, None
        if case["max_norm"]:
            norm = th.sqrt(sum(g.double().square().sum() for g in s["lists"][1])).float()
            coef = (case["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
        [_plain_adamw(s["step"], coef, *ts) for ts in zip(*s["lists"])]
    return dict(out, norm=norm) if case["max_norm"] else out


def _blocks(t, n):
    """a flat tensor as [blocks, QBLOCK], the last block filled up with zeros"""
    full = th.zeros(-(-n // QBLOCK) * QBLOCK, device=t.device)
    full[:n] = t.reshape(-1)
    return full.view(-1, QBLOCK)


def _plain_adamw(step, coef, p, g, m, v, ms=None, vs=None):
    b1, b2 = BETAS
    n = p.numel()
    grad = g.float() if coef is None else g.float() * coef
    if ms is None:
        m0, v0 = m, v
    else:
        m0 = (_blocks(m.float(), n) * ms[:, None]).view(-1)[:n].view(p.shape)
        v0 = (_blocks(v.float(), n) * vs[:, None]).view(-1)[:n].view(p.shape).square()
    m1 = m0 + (grad - m0) * (1 - b1)
    v1 = v0 * b2 + (1 - b2) * grad * grad
    root = th.sqrt(v1)
    p.copy_(p.float() * (1 - LR * DECAY) - LR / (1 - b1 ** step) * m1 / (root / math.sqrt(1 - b2 ** step) + EPS))
    if ms is None:
        m.copy_(m1)
        v.copy_(v1)
        return
    for q, scale, full in ((m, ms, m1), (v, vs, root)):
        full = _blocks(full, n)
        new = full.abs().amax(-1) / QMAX
        new = th.where(new < 2.0 ** -126, 0.0, new)
        code = (full * th.where(new > 0, 1.0 / new, 0.0)[:, None]).to(F8).float()
        if scale is vs:
            code = th.where((full > 0) & (new > 0)[:, None], code.clamp(min=QMIN), code)
        q.copy_(code.view(-1)[:n].view(q.shape).to(F8))
        scale.copy_(new)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x, w, b = s["x"].double(), s["w"].double(), s["b"].double()
        var, mean = th.var_mean(x, dim=1, unbiased=False, keepdim=True)
        sd = (var + NORM_EPS).sqrt()
        y = (x - mean) / sd * w + b
        if not case["train"]:
            return {"y": y}
        dy = s["dy"].double()
        c = case["cols"]
        inner, cov = (dy * w).sum(1, keepdim=True), (dy * w * (x - mean)).sum(1, keepdim=True)
        dx = (dy * w - inner / c - (x - mean) * cov / (c * (var + NORM_EPS))) / sd
        return {"y": y, "dx": dx, "dw": ((x - mean) / sd).mul_(dy).sum(0), "db": dy.sum(0)}
    if case["op"] == "logp":
        l = s["logits"].double()
        if s["avail"] is not None:
            l[s["avail"] == 0] = -math.inf
        dead = (l == -math.inf).all(1)
        lp = th.log_softmax(l, 1)
        lp[dead] = -math.inf
        p = lp.exp()
        ent = th.special.entr(p).sum(1)
        rows = th.arange(case["rows"], device=l.device)
        t = s["tokens"]
        skip = t < 0
        logp = lp[rows, t.clamp(min=0)]
        gone = th.isinf(logp)
        logp[skip] = 0.0
        out = {"logp": logp, "entropy": ent}
        if case["top_k"]:
            k = min(case["top_k"], case["vocab"])
            val = lp.topk(k, dim=1)[0]
            out["top_logp"] = th.nn.functional.pad(val, (0, case["top_k"] - k), value=-math.inf)
            out["top_index"] = None
        if case["train"]:
            g, h = s["dlogp"].double().masked_fill(skip, 0.0), s["dent"].double()
            d = -p * g[:, None] + h[:, None] * (th.special.entr(p) - p * ent[:, None])
            live = ~(skip | gone)
            d[rows[live], t[live]] += g[live]
            out["dlogits"] = d
        return out
    step, (b1, b2) = s["step"] + 1, BETAS
    norm = s["g"].double().norm()
    g = s["g"].double()
    if case["max_norm"]:
        g *= min(1.0, case["max_norm"] / (float(norm) + 1e-6))
    places, n, blocks = _places(case)
    if case["bits"] == 32:
        m, v = s["m"].double(), s["v"].double()
    else:
        of = th.zeros(n, dtype=th.long, device="cuda")
        for _, k, at, blk in places:
            of[at:at + k] = blk + th.arange(k, device="cuda") // QBLOCK
        m = s["m"].double() * s["ms"].double()[of]
        v = (s["v"].double() * s["vs"].double()[of]) ** 2
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = s["p"].double()
    p = p - LR * DECAY * p - LR * (m / (1 - b1 ** step)) / ((v / (1 - b2 ** step)).sqrt() + EPS)
    out = {"p": p}
    if case["max_norm"]:
        out["norm"] = norm
    if case["bits"] == 32:
        return dict(out, m=m, v=v)
    r = v.sqrt()
    for name, t in (("m", m), ("v", r)):
        scale = th.zeros(blocks, dtype=th.float64, device="cuda").scatter_reduce_(0, of, t.abs(), "amax") / QMAX
        q = (t / scale.clamp(min=1e-300)[of]).to(F8).double()
        out[name] = th.where((q == 0) & (t > 0), QMIN, q) if name == "v" else q
        out[name + "s"] = scale
    return out
