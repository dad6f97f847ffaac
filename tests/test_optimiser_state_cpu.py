"""What optim_device.AdamW takes into its state and its groups: nothing is launched, so all of it is checked without a GPU."""
import copy

import pytest
import torch as th


def _params(*shapes):
    g = th.Generator().manual_seed(0)
    return [th.nn.Parameter(th.randn(s, generator=g)) for s in shapes or ((3, 4), (7,))]


def _stepped(opt, steps=1):
    """a torch optimiser after `steps` steps"""
    for _ in range(steps):
        for g in opt.param_groups:
            for p in g["params"]:
                p.grad = th.ones_like(p)
        opt.step()
    return opt


def _snapshot(opt):
    return copy.deepcopy(opt.state_dict())


def _same(a, b):
    if isinstance(a, dict):
        return a.keys() == b.keys() and all(_same(a[k], b[k]) for k in a)
    if isinstance(a, (list, tuple)):
        return len(a) == len(b) and all(map(_same, a, b))
    if isinstance(a, th.Tensor):
        return a.dtype == b.dtype and a.shape == b.shape and th.equal(a.reshape(-1).view(th.uint8), b.reshape(-1).view(th.uint8))
    return a == b


@pytest.mark.parametrize("option", ["maximize", "amsgrad", "differentiable"])
@pytest.mark.parametrize("steps", [0, 1])
def test_options_of_another_update_are_refused(option, steps):
    """torch's AdamW with an option that changes the step: its state_dict, a group made with it, and a group that got it later
    are refused; the optimiser stays as it was"""
    from marl_amd.utils.optim_device import AdamW
    ps = _params()
    if option == "differentiable" and steps:
        pytest.skip("torch steps a leaf in place under this option only where no gradient is recorded")
    saved = _stepped(th.optim.AdamW(ps, **{option: True}), steps).state_dict()
    opt = AdamW(_params())
    before = _snapshot(opt)
    with pytest.raises(ValueError, match=option if option != "amsgrad" or not steps else "amsgrad|max_exp_avg_sq"):
        opt.load_state_dict(saved)
    assert _same(opt.state_dict(), before)
    with pytest.raises(ValueError, match=option):
        AdamW([{"params": _params(), option: True}])
    with pytest.raises(ValueError, match=option):
        opt.add_param_group({"params": _params(), option: True})
    assert len(opt.param_groups) == 1
    opt.param_groups[0][option] = True
    with pytest.raises(ValueError, match=option):
        opt.step()


def test_a_decay_that_is_part_of_the_gradient_is_refused():
    """torch.optim.Adam's weight decay enters the moments; without one its states continue here, as does its group"""
    from marl_amd.utils.optim_device import AdamW
    opt = AdamW(_params())
    with pytest.raises(ValueError, match="decoupled_weight_decay"):
        opt.load_state_dict(_stepped(th.optim.Adam(_params(), weight_decay=0.1)).state_dict())
    assert not opt.state and opt.param_groups[0]["weight_decay"] == 1e-2
    opt.load_state_dict(_stepped(th.optim.Adam(_params()), 3).state_dict())
    assert [st["step"] for st in opt.state.values()] == [3, 3]
    opt.param_groups[0]["weight_decay"] = 0.1
    with pytest.raises(ValueError, match="decoupled_weight_decay"):
        opt.step()


def test_a_capturable_group_keeps_each_parameters_count():
    """torch's states hold a count per parameter: loaded, each parameter has its own back, equal ones share one tensor"""
    from marl_amd.utils.optim_device import AdamW
    src = th.optim.AdamW(_params((4,), (5,), (6,)))
    ps = src.param_groups[0]["params"]
    for step in range(3):
        for i, p in enumerate(ps):
            p.grad = th.ones_like(p) if i != 1 or step == 2 else None
        src.step()
    saved = src.state_dict()
    saved["param_groups"][0]["capturable"] = True
    opt = AdamW(_params((4,), (5,), (6,)), capturable=True)
    opt.load_state_dict(saved)
    steps = [opt.state[p]["step"] for p in opt.param_groups[0]["params"]]
    assert [float(s) for s in steps] == [3, 1, 3] and steps[0] is steps[2] and steps[0] is not steps[1]
    again = AdamW(_params((4,), (5,), (6,)), capturable=True)
    again.load_state_dict(opt.state_dict())
    assert _same(again.state_dict(), opt.state_dict())


def _saved(bits, opt=None):
    """a state_dict of one step, of parameters (3, 4) and (7,)"""
    from marl_amd.utils.optim_device import STATE8, AdamW
    opt = opt or AdamW(_params(), state_bits=bits)
    for p in opt.param_groups[0]["params"]:
        n = p.numel()
        st = opt.state[p] = dict(step=1, exp_avg=th.ones(p.shape), exp_avg_sq=th.ones(p.shape))
        if bits == 8:
            st.update(exp_avg=th.ones(p.shape).to(STATE8), exp_avg_sq=th.ones(p.shape).to(STATE8))
            st.update(exp_avg_scale=th.ones(-(-n // 256)), exp_avg_sq_scale=th.ones(-(-n // 256)))
    return opt.state_dict()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("key", ["exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "step"])
def test_states_of_other_sizes_and_types_are_refused(key, bits):
    """before anything of the optimiser is replaced"""
    from marl_amd.utils.optim_device import AdamW
    if bits == 32 and key.endswith("_scale"):
        pytest.skip("no scales")
    good = _saved(bits)
    opt = AdamW(_params(), state_bits=bits, lr=0.25)
    opt.load_state_dict(_saved(bits, AdamW(_params(), state_bits=bits, lr=0.25)))
    before = _snapshot(opt)
    old = good["state"][1][key]
    bad = [th.ones(3), "1"] if key == "step" else [th.ones(8).to(old.dtype), th.ones(1, 7).to(old.dtype), [1.0] * 7]
    if key in ("exp_avg", "exp_avg_sq"):
        bad += [old.to(th.float32 if bits == 8 else th.float8_e4m3fn), old.to(th.int32)]
    for value in bad:
        saved = copy.deepcopy(good)
        saved["state"][1][key] = value
        with pytest.raises(ValueError, match="parameter 1"):
            opt.load_state_dict(saved)
        assert _same(opt.state_dict(), before)
    del good["state"][1][key]
    with pytest.raises(ValueError, match="parameter 1"):
        opt.load_state_dict(good)
    assert _same(opt.state_dict(), before)


@pytest.mark.parametrize("default", [32, 8])
def test_a_groups_own_bits_outlast_a_load_that_names_none(default):
    """torch's state_dict names no state_bits: each group keeps its own, whatever the constructor's default was"""
    from marl_amd.utils.optim_device import AdamW
    make = lambda: AdamW([dict(params=_params(), state_bits=40 - default), dict(params=_params((5,)))], state_bits=default)
    torchs = lambda: th.optim.AdamW([dict(params=_params()), dict(params=_params((5,)))])
    opt = make()
    opt.load_state_dict(torchs().state_dict())
    assert [g["state_bits"] for g in opt.param_groups] == [40 - default, default]
    # states only for the group of 32 bits: taken; for that of 8: refused
    wide, narrow = (0, 1) if default == 8 else (1, 0)
    for k in (wide, narrow):
        src = torchs()
        for p in src.param_groups[k]["params"]:
            p.grad = th.ones_like(p)
        src.step()
        opt = make()
        if k == wide:
            opt.load_state_dict(src.state_dict())
            assert all(opt.state[p]["exp_avg"].dtype == th.float32 for p in opt.param_groups[k]["params"])
            assert [g["state_bits"] for g in opt.param_groups] == [40 - default, default]
        else:
            with pytest.raises(ValueError, match="8 bits"):
                opt.load_state_dict(src.state_dict())
    with pytest.raises(ValueError, match="state_bits"):
        saved = make().state_dict()
        saved["param_groups"][1]["state_bits"] = 16
        make().load_state_dict(saved)


def test_options_that_a_state_dict_lacks_are_the_groups_own():
    from marl_amd.utils.optim_device import AdamW
    opt = AdamW([dict(params=_params(), capturable=True, eps=1e-5)])
    saved = opt.state_dict()
    for k in ("capturable", "eps"):
        del saved["param_groups"][0][k]
    opt.load_state_dict(saved)
    assert opt.param_groups[0]["capturable"] is True and opt.param_groups[0]["eps"] == 1e-5


def test_a_learning_rate_on_the_device_needs_capturable_at_load_too():
    from marl_amd.utils.optim_device import AdamW
    opt = AdamW(_params(), lr=0.5)
    before = _snapshot(opt)
    with pytest.raises(ValueError, match="capturable"):
        opt.load_state_dict(th.optim.AdamW(_params(), lr=th.tensor(1e-3), foreach=False).state_dict())
    assert _same(opt.state_dict(), before)


def test_groups_without_parameters():
    """as torch takes them (a net without biases, say): first, last and filled by none"""
    from marl_amd.utils.optim_device import AdamW
    opt = AdamW([dict(params=[]), dict(params=_params()), dict(params=[], lr=1.0)])
    assert [len(g["params"]) for g in opt.param_groups] == [0, 2, 0]
    AdamW([dict(params=[]), dict(params=_params()), dict(params=[], lr=1.0)]).load_state_dict(opt.state_dict())
    with pytest.raises(ValueError, match="on one device"):
        opt.add_param_group(dict(params=[th.nn.Parameter(th.zeros(3, device="meta"))]))
    assert len(opt.param_groups) == 3


def test_load_state_dict_hooks():
    """a pre-hook's state_dict is the one that is checked and loaded; a post-hook sees, and may change, the loaded states"""
    from marl_amd.utils.optim_device import AdamW
    ps = [p.bfloat16() for p in _params()]
    opt = AdamW([th.nn.Parameter(p.detach()) for p in ps])

    def pre(o, state_dict):
        return dict(state_dict, state={i: {k: v * 2 if k == "exp_avg" else v for k, v in st.items()}
                                       for i, st in state_dict["state"].items()})
    seen = []

    def post(o):
        seen.extend(st["exp_avg"].dtype for st in o.state.values())
        for st in o.state.values():
            st["step"] = 7
    opt.register_load_state_dict_pre_hook(pre)
    opt.register_load_state_dict_post_hook(post)
    opt.load_state_dict(_saved(32))
    assert seen == [th.float32, th.float32]
    assert all(st["step"] == 7 and bool((st["exp_avg"] == 2).all()) for st in opt.state.values())
    opt.register_load_state_dict_pre_hook(lambda o, s: dict(s, state={0: {"step": 1}}))
    with pytest.raises(ValueError, match="parameter 0"):
        opt.load_state_dict(_saved(32))
    assert all(st["step"] == 7 for st in opt.state.values())
    opt = AdamW(_params())
    for _ in range(2):                                        # (nothing of a load is left behind)
        opt.load_state_dict(_saved(32))
    assert not opt._optimizer_load_state_dict_pre_hooks and not opt._optimizer_load_state_dict_post_hooks


def test_loaded_again_and_copied():
    """a load after a load, and after a copy (torch adds an option to the defaults there that no group has)"""
    from marl_amd.utils.optim_device import AdamW
    opt = AdamW(_params(), state_bits=8)
    saved = _saved(8)
    for o in (opt, copy.deepcopy(opt)):
        for _ in range(3):
            o.load_state_dict(saved)
            assert _same(o.state_dict()["state"], saved["state"])


def test_pickled_before_it_kept_recorded_counts():
    """a pickle without the list of counts that graphs advance: unpickled it has an empty one"""
    from marl_amd.utils.optim_device import AdamW
    old = AdamW(_params(), capturable=True, max_norm=2.0).__getstate__()
    del old["_recorded"]
    opt = AdamW.__new__(AdamW)
    opt.__setstate__(old)
    assert opt._recorded == [] and opt.max_norm == 2.0


@pytest.mark.parametrize("missing", ["lr", "weight_decay", "betas"])
def test_options_that_are_checked_at_load_may_be_missing(missing):
    from marl_amd.utils.optim_device import AdamW
    opt = AdamW(_params(), lr=0.5, weight_decay=0.0)
    saved = th.optim.Adam(_params()).state_dict()
    del saved["param_groups"][0][missing]
    opt.load_state_dict(saved)
    assert opt.param_groups[0]["lr"] == (0.5 if missing == "lr" else 1e-3) and opt.param_groups[0]["betas"] == (0.9, 0.999)
    opt.param_groups[0]["weight_decay"] = 0.1
    del saved["param_groups"][0]["weight_decay" if missing != "weight_decay" else "lr"]
    with pytest.raises(ValueError, match="decoupled"):   # (with the weight decay that the group would then have)
        opt.load_state_dict(saved)
