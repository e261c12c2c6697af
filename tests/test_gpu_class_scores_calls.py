"""Calls of `token_log_probs` and `distillation_loss` at the border of what they take."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import k2_b200 as k2

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def test_forward_mode_is_refused_wherever_it_comes_in():
    """A teacher's tangent is not dropped either: the loss would look constant in it."""
    x, token = torch.randn(2, 3, 8, device=DEV), torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    tt, lp = token[..., None].expand(2, 3, 4).contiguous(), torch.randn(2, 3, 4, device=DEV)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        teacher = forward_ad.make_dual(lp, torch.ones_like(lp))
        for call in (lambda: k2.token_log_probs(dual, token),
                     lambda: k2.distillation_loss(dual, tt, lp),
                     lambda: k2.distillation_loss(x, tt, teacher)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
