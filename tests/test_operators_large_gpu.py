"""Layer norm, token log-probs and AdamW at the sizes that batches have: blocks that take several rows or batches of a row, the
kernels with the streaming hint, tall grids.  Against the formulas in float64, with the bounds that stand at the functions
imported here; and against the same rows (or tensors) in calls of their own, bit for bit, where those add in the same order.

The bound of a weight gradient's sum holds for these row counts too: a thread adds rows / (blocks rows-a-block) terms, at most
rows / 256 + 1, a block's threads 10 more, and the partial rows of at most 1024 blocks 64 + 16."""
import math

import pytest
import torch as th

from tests import test_adamw_gpu as A
from tests import test_logprob_gpu as L
from tests import test_norm_gpu as N

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


# rows: past one round of all blocks and no multiple of it (waves a CU times 256 CUs, as blocks_for has them)
NORM = [(270001, 11), (70003, 29), (20011, 61), (10007, 125), (9001, 250), (9001, 300), (5003, 1003), (2503, 1601), (2503, 2048),
        (1100, 4093), (700, 8191), (300, 16384), (1027, 16391), (40, 40003)]
# past 2^25 elements: the streaming hint
NORM_FAR = [(4800001, 7), (3100001, 11), (1200001, 29), (600001, 61), (280001, 125), (140001, 250), (70001, 500), (34001, 1003),
            (16501, 2047), (8301, 4093), (8301, 4099), (2053, 16384)]


@pytest.mark.parametrize("dtype,wdtype", [(th.float32, th.float32), (th.bfloat16, th.float32), (th.float16, th.float16)])
@pytest.mark.parametrize("rows,cols", NORM + NORM_FAR)
def test_layer_norm(rows, cols, dtype, wdtype):
    from marl_amd.utils import norm_device
    x, w, b, dy = N._inputs(rows, cols, dtype, wdtype)
    y, mean, rstd = norm_device.layer_norm_fwd(x, w, b, 1e-5)
    dx, dw, db = norm_device.layer_norm_bwd(dy, x, mean, rstd, w)
    for at in (0, rows // 3, rows - 37):                     # rows of later rounds as those of a first one
        s = slice(at, at + 37)
        part = norm_device.layer_norm_fwd(x[s], w, b, 1e-5)
        assert all(th.equal(p, q[s]) for p, q in zip(part, (y, mean, rstd))), at
        assert th.equal(norm_device.layer_norm_bwd(dy[s], x[s], mean[s], rstd[s], w)[0], dx[s]), at
    want, tol = N._reference(x, w, b, dy, 1e-5)
    for got, a, t, name in zip((y, dx, dw, db), want, tol, ("y", "dx", "dw", "db")):
        N._within(got, a, t, name)


@pytest.mark.parametrize("mask", [None, th.bool, th.int32])
@pytest.mark.parametrize("rows,vocab,dtype", [
    (4099, 1203, th.float32), (4099, 4001, th.float32), (4099, 2100, th.bfloat16), (4099, 8001, th.float16),  # a wave a row, batch by batch
    (4099, 4101, th.float32), (1009, 50021, th.float32), (601, 100003, th.bfloat16), (601, 100003, th.float16),  # a block; the last three far
    (307, 200, th.bfloat16), (307, 400, th.bfloat16), (307, 200, th.float16), (307, 400, th.float16), (307, 120, th.float32),  # 16
    (307, 200, th.float32), (307, 400, th.float32)])                          # lanes a row, and a wave
def test_token_logprobs_of_middle_and_wide_rows(rows, vocab, dtype, mask):
    from marl_amd.utils import logprob_device
    l, t, avail, g, h = L._inputs(rows, vocab, dtype, mask)
    lp, want, tol = L._reference(l, t, avail, g, h)
    for k in (0, 1, 20, 64):
        f = logprob_device.token_logprobs_fwd(l, t, avail, top_k=k)
        L._within(f.logp, want[0], tol[0], "logp")
        L._within(f.entropy, want[1], tol[1], "entropy")
        if k:
            val, at = L._top(l, avail, lp, k)
            assert th.equal(f.top_index, at), k
            L._within(f.top_logp, val, (tol[0].max() + 4 * U * val.abs()), "top_logp")
    L._within(logprob_device.token_logprobs_bwd(l, t, f.lse, f.entropy, g, h, avail), want[2], tol[2], "dlogits")


@pytest.mark.parametrize("vocab,dtype", [(2500, th.float32), (5003, th.bfloat16)])
def test_ties_over_the_batches_of_a_wave(vocab, dtype):
    """rows of equal logits, of few values, rising, falling, and with equal largest ones in every batch: what a stable sort gives"""
    from marl_amd.utils import logprob_device
    gen = th.Generator(device="cuda").manual_seed(vocab)
    rows = 4200
    l = th.randint(-2, 3, (rows, vocab), device="cuda", generator=gen).float()
    ramp = th.arange(vocab, device="cuda") / 64.0
    l[0], l[1], l[2], l[3] = 0.0, ramp, -ramp, -float("inf")
    l[4] = th.where(th.arange(vocab, device="cuda") % 700 == 699, 5.0, l[4])
    l[5, :-1] = -float("inf")
    l = l.to(dtype)
    t = th.zeros(rows, dtype=th.int64, device="cuda")
    lp = th.log_softmax(l.double(), 1)
    lp[3] = -float("inf")
    for k in (1, 20, 64):
        assert th.equal(logprob_device.token_logprobs_fwd(l, t, top_k=k).top_index, L._top(l + 0.0, None, lp, k)[1]), k


@pytest.mark.parametrize("gaps", [False, True])
@pytest.mark.parametrize("mask", [None, th.bool, th.int32])
@pytest.mark.parametrize("dtype", [th.float32, th.bfloat16, th.float16])
@pytest.mark.parametrize("vocab", [11, 20, 26])
def test_token_logprobs_of_few_entries_with_the_streaming_hint(vocab, dtype, mask, gaps):
    """more than 96 MiB of logits and mask: the bits of calls on parts of the rows, which have no hint, and the formulas there"""
    from marl_amd.utils import logprob_device
    F, B = logprob_device.token_logprobs_fwd, logprob_device.token_logprobs_bwd
    rows = (100 << 20) // (vocab * (th.finfo(dtype).bits // 8 + {None: 0, th.bool: 1, th.int32: 4}[mask])) + 3
    l, t, avail, g, h = L._inputs(rows, vocab, dtype, mask)
    if gaps:
        wide = lambda x: th.nn.functional.pad(x.view(th.uint8) if x.dtype == th.bool else x, (1, 2))[:, 1:vocab + 1]
        l, avail = wide(l), wide(avail) if avail is not None else None
    f = F(l, t, avail, 3)
    d = B(l, t, f.lse, f.entropy, g, h, avail)
    for at in range(0, rows, 128 * 2500):                   # (a block takes 128 rows, each lane one: the same sums)
        s = slice(at, at + 128 * 2500)
        a = avail[s] if avail is not None else None
        e = F(l[s], t[s], a, 3)
        assert all(th.equal(p, q[s]) if p.dtype == th.int64 else th.equal(p.view(th.int32), q[s].view(th.int32)) for p, q in zip(e, f)), at
        assert th.equal(B(l[s], t[s], e.lse, e.entropy, g[s], h[s], a), d[s]), at
    lp, want, tol = L._reference(l[-30001:], t[-30001:], avail[-30001:] if avail is not None else None, g[-30001:], h[-30001:])
    for got, a, b, name in zip((f.logp, f.entropy, d), want, tol, ("logp", "entropy", "dlogits")):
        L._within(got[-30001:], a, b, name)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [th.float32, th.bfloat16, th.float16])
def test_adamw_with_the_streaming_hint(dtype, bits):
    """9.5 M elements in one call against the formulas, and tensor by tensor (under the 8 M of the hint): the same bits"""
    from marl_amd.utils import optim_device
    lists = A._state([5_000_003, 3_500_001, 77, 0, 1_000_000], dtype, bits, seed=3)
    before, alone = A._copy(lists), A._copy(lists)
    optim_device.adamw_step(*lists, step=9, **A.HYPER)
    A._check(lists, before, 9, **A.HYPER)
    for i in range(5):
        optim_device.adamw_step(*[[x[i]] for x in alone], step=9, **A.HYPER)
    assert all(th.equal(a.view(th.uint8), b.view(th.uint8)) for x, y in zip(lists, alone) for a, b in zip(x, y))


@pytest.mark.parametrize("dtype", [th.float32, th.bfloat16, th.float16])
def test_the_norm_of_more_than_a_chunk_a_block(dtype):
    """35 M elements: blocks of 16384, several batches each, and ragged last ones; squares in double, so the bound of the norm's
    own rounding"""
    from marl_amd.utils.optim_device import clip_coef
    gen = th.Generator(device="cuda").manual_seed(0)
    grads = [th.randn(n + 1, device="cuda", generator=gen).to(dtype)[1:] for n in (30_000_001, 5_000_000, 12_289, 1000, 3)]
    want = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    norm, coef = (float(x) for x in clip_coef(grads, 1.0))
    assert abs(norm - want) <= 1.01 * U * want and abs(coef - 1 / (want + 1e-6)) <= 5 * U * coef
    assert (norm, coef) == tuple(float(x) for x in clip_coef(grads, 1.0))


def test_adamw_with_more_blocks_than_a_launch_takes_along_x():
    """2^32 + 1027 elements in one tensor (52 GB with its gradient and states), all alike: each as in a small call"""
    from marl_amd.utils.optim_device import adamw_step
    n = 2 ** 32 + 1027
    values = ((0.5, th.bfloat16), (0.25, th.bfloat16), (0.125, th.float32), (0.0625, th.float32))
    few, many = ([[th.full((k,), v, dtype=t, device="cuda")] for v, t in values] for k in (5, n))
    for x in (few, many):
        adamw_step(*x, step=3, **A.HYPER)
    for a, b in zip(few, many):
        want = a[0][0]
        assert bool((a[0] == want).all())
        for at in range(0, n, 2 ** 29):
            assert bool((b[0][at:at + 2 ** 29] == want).all()), at
