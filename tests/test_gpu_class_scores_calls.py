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


@pytest.mark.parametrize("shape", [(5, 0, 7, 0, 9), (2, 0, 3, 0, 4, 9), (3, 5, 0, 7, 9), (0, 0, 9)])
def test_no_rows_in_several_dimensions(shape):
    x = torch.zeros(shape, device=DEV, requires_grad=True)
    tt = torch.zeros(shape[:-1] + (3,), dtype=torch.int32, device=DEV)
    outs = [k2.distillation_loss(x, tt, tt.float(), reduction=r) for r in ("none", "sum", "mean")]
    got = k2.token_log_probs(x, tt[..., 0], top_k=2, entropy=True)
    for out in outs + [got.log_probs, got.entropy, got.top_log_probs]:
        assert torch.autograd.grad(out.sum(), x, retain_graph=True)[0].shape == shape


@pytest.mark.parametrize("rows,classes", [(300, 5000), (300, 20000), (2, 20000), (700, 5000)])
def test_as_many_top_classes_as_a_block_has_threads_or_more(rows, classes):
    """The bound comes from the groups that there are, and from those only: among scores around 0,
    among log-probs, and where all scores are one very low value."""
    g = torch.Generator(device=DEV).manual_seed(classes)
    x = torch.randn(rows, classes, generator=g, device=DEV) * 3
    for values in (x, torch.log_softmax(x, -1), x - 1e30):
        order = torch.sort(values, dim=-1, descending=True, stable=True).indices.int()
        for top_k in (63, 64, 65, 96, 113, 114, 127, 128):
            got = k2.token_log_probs(values, top_k=top_k)
            assert torch.equal(got.top_tokens, order[:, :top_k]), top_k
