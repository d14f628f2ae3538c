"""Derivatives that the jagged attention does not have are refused."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import torchlib_xpu_b200

pytestmark = pytest.mark.gpu

torchlib_xpu_b200.load_torch_ops()
attention = torch.ops.fbgemm.b200tbe_jagged_attention


def _attention_arguments():
    gen = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(9, h, 16, generator=gen).cuda() for h in (4, 2, 2))
    return [q, k, v, torch.tensor([0, 4, 9], device="cuda")]


@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_jagged_attention_refuses_forward_mode(which, grad_mode):
    args = _attention_arguments()
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            attention(*args)
        args[which].requires_grad_()
        with pytest.raises(NotImplementedError, match="forward-mode"):
            attention(*args)


def test_the_gradients_refuse_forward_mode():
    args = _attention_arguments()
    args[0].requires_grad_()
    out = attention(*args)
    with forward_ad.dual_level():
        g = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(out, args[0], g)
