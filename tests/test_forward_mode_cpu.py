"""layer_norm and token_logprobs have no forward-mode derivative: an input that carries a tangent is refused, where the result
would pass for a constant (checked before anything looks for a device, so without one)."""
import pytest
import torch as th
import torch.autograd.forward_ad as fw


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("leaf", [False, True])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_layer_norm(which, leaf, grad):
    from marl_amd.utils.norm_device import layer_norm
    args = [th.randn(3, 8), th.randn(8), th.randn(8)]
    with fw.dual_level(), th.set_grad_enabled(grad):
        args[which] = fw.make_dual(args[which].requires_grad_(leaf), th.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            layer_norm(*args)
        with pytest.raises(RuntimeError, match="no CPU fallback"):     # (the tangent is its own call's)
            layer_norm(th.randn(3, 8))


@pytest.mark.parametrize("leaf", [False, True])
def test_token_logprobs(leaf):
    from marl_amd.utils.logprob_device import token_logprobs
    logits, tokens = th.randn(3, 8), th.zeros(3, dtype=th.int64)
    with fw.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            token_logprobs(fw.make_dual(logits.requires_grad_(leaf), th.ones(3, 8)), tokens)
    with pytest.raises(RuntimeError, match="forward-mode"):
        th.func.jvp(lambda x: token_logprobs(x, tokens).logp, (logits.detach(),), (th.ones(3, 8),))
