"""Token scores and distillation without a GPU: what the C-ABI and the Python layer refuse."""
import ctypes

import pytest
import torch

import k2_b200 as k2
from class_scores_util import distil_reference, tokens_reference
from k2_b200 import _lib

INVALID, TOO_SMALL = 1, 3
FAR = 0x1000  # an address that no refused call looks at


def rows(**kw):
    return _lib.ClassRows(**dict(dict(scores=FAR, type=0, num_classes=8, outer=2, inner=3,
                                      outer_stride=24, inner_stride=8), **kw))


def teacher(**kw):
    return _lib.Teacher(**dict(dict(tokens=FAR, tokens_64=0, scores=FAR, type=0, entries=4,
                                    temperature=1.0, weight=1.0, reduction=1), **kw))


def token_scores(r, tokens=FAR, top_k=2, log_probs=FAR, top=FAR):
    return _lib.lib.k2b200_token_scores(ctypes.byref(r), tokens, 0, top_k, log_probs, None, top,
                                        top, None, None)


def token_backward(r, norm=FAR, grad=FAR, top_k=2, tokens=FAR, given=None, top=None):
    none = _lib.RowGrad()
    a, b = _lib.RowGrad(grad=given), _lib.RowGrad(grad=top)
    return _lib.lib.k2b200_token_scores_backward(
        ctypes.byref(r), tokens, 0, top_k, None, norm, ctypes.byref(a), ctypes.byref(none),
        ctypes.byref(b), grad, 24, 8, None)


def distil(r, t, loss=FAR, grad=None, workspace=FAR, size=1 << 20):
    return _lib.lib.k2b200_distillation(ctypes.byref(r), ctypes.byref(t), loss, None, grad, 24, 8,
                                        workspace, size, None)


def distil_backward(r, t, norm=FAR, up=FAR, grad=FAR, workspace=FAR, size=1 << 20):
    g = _lib.RowGrad(grad=up)
    return _lib.lib.k2b200_distillation_backward(ctypes.byref(r), ctypes.byref(t), norm,
                                                 ctypes.byref(g), 0, grad, 24, 8, workspace, size,
                                                 None)


@pytest.mark.parametrize("bad", [
    dict(type=3), dict(type=-1), dict(num_classes=0), dict(outer=-1), dict(inner=-2),
    dict(outer=1 << 20, inner=1 << 11), dict(outer=1 << 40, inner=0), dict(scores=None)])
def test_rows_that_are_refused(bad):
    r = rows(**bad)
    for status in (token_scores(r), token_backward(r), distil(r, teacher()),
                   distil_backward(r, teacher())):
        assert status == INVALID and _lib.lib.k2b200_last_error()


def test_token_calls_that_are_refused():
    for status in (token_scores(rows(), top_k=-1), token_scores(rows(), top_k=9),
                   token_scores(rows(num_classes=1000), top_k=129),
                   token_scores(rows(), tokens=None), token_scores(rows(), log_probs=None),
                   token_scores(rows(), top=None), token_backward(rows(), norm=None),
                   token_backward(rows(), grad=None), token_backward(rows(), top_k=9),
                   token_backward(rows(), tokens=None, given=FAR),
                   token_backward(rows(), top=FAR)):
        assert status == INVALID and _lib.lib.k2b200_last_error()


@pytest.mark.parametrize("bad", [
    dict(type=3), dict(entries=0), dict(entries=129), dict(temperature=0.0),
    dict(temperature=float("nan")), dict(temperature=float("inf")), dict(reduction=3),
    dict(reduction=-1), dict(tokens=None), dict(scores=None)])
def test_teachers_that_are_refused(bad):
    t = teacher(**bad)
    assert distil(rows(), t) == INVALID and distil_backward(rows(), t) == INVALID


def test_distillation_calls_that_are_refused():
    for status in (distil(rows(), teacher(), loss=None),
                   distil(rows(), teacher(), workspace=None),
                   distil(rows(), teacher(reduction=0), grad=FAR),
                   distil_backward(rows(), teacher(), norm=None),
                   distil_backward(rows(), teacher(), up=None),
                   distil_backward(rows(), teacher(), grad=None),
                   distil_backward(rows(), teacher(), workspace=None)):
        assert status == INVALID
    need = _lib.lib.k2b200_distillation_workspace_bytes(ctypes.byref(rows()))
    assert need > 0
    assert distil(rows(), teacher(), size=need - 1) == TOO_SMALL
    assert distil_backward(rows(), teacher(), size=7) == TOO_SMALL


def test_addresses_that_are_not_aligned_are_refused():
    odd, half = rows(scores=FAR + 1, type=1), rows(scores=FAR + 2)
    for status in (token_scores(odd), token_scores(half), token_backward(odd), distil(odd, teacher()),
                   distil_backward(half, teacher()), token_backward(rows(), norm=FAR + 8),
                   token_backward(rows(), grad=FAR + 2), token_backward(rows(type=2), grad=FAR + 1),
                   distil(rows(), teacher(), grad=FAR + 2),
                   distil_backward(rows(), teacher(), norm=FAR + 8),
                   distil_backward(rows(), teacher(), grad=FAR + 2)):
        assert status == INVALID and b"aligned" in _lib.lib.k2b200_last_error()


def token_call(r, tokens=FAR, tokens_64=0, log_probs=FAR, entropy=None, top_values=FAR,
               top_classes=FAR):
    return _lib.lib.k2b200_token_scores(ctypes.byref(r), tokens, tokens_64, 2, log_probs, entropy,
                                        top_values, top_classes, None, None)


def token_backward_call(r, tokens=FAR, tokens_64=0, classes=FAR, ups=(FAR, FAR, FAR)):
    a, b, c = (_lib.RowGrad(grad=up) for up in ups)
    return _lib.lib.k2b200_token_scores_backward(
        ctypes.byref(r), tokens, tokens_64, 2, classes, FAR, ctypes.byref(a), ctypes.byref(b),
        ctypes.byref(c), FAR, 24, 8, None)


@pytest.mark.parametrize("call", [
    lambda: token_scores(rows(lengths=FAR + 2)),
    lambda: distil(rows(lengths=FAR + 4, lengths_64=1), teacher()),
    lambda: token_call(rows(), tokens=FAR + 2), lambda: token_call(rows(), FAR + 4, 1),
    lambda: token_call(rows(), log_probs=FAR + 2), lambda: token_call(rows(), entropy=FAR + 1),
    lambda: token_call(rows(), top_values=FAR + 2), lambda: token_call(rows(), top_classes=FAR + 2),
    lambda: token_backward_call(rows(), tokens=FAR + 4, tokens_64=1),
    lambda: token_backward_call(rows(), classes=FAR + 2),
    lambda: token_backward_call(rows(), ups=(FAR + 2, FAR, FAR)),
    lambda: token_backward_call(rows(), ups=(FAR, FAR + 2, FAR)),
    lambda: token_backward_call(rows(), ups=(FAR, FAR, FAR + 2)),
    lambda: distil(rows(), teacher(tokens=FAR + 2)),
    lambda: distil(rows(), teacher(tokens=FAR + 4, tokens_64=1)),
    lambda: distil(rows(), teacher(scores=FAR + 2)),
    lambda: distil_backward(rows(), teacher(scores=FAR + 1, type=2)),
    lambda: distil(rows(), teacher(), loss=FAR + 2),
    lambda: distil(rows(), teacher(), workspace=FAR + 4),
    lambda: distil_backward(rows(), teacher(), workspace=FAR + 4),
    lambda: distil_backward(rows(), teacher(), up=FAR + 2)])
def test_arrays_that_are_not_aligned_are_refused(call):
    """The device would stop at such an address."""
    assert call() == INVALID and b"aligned" in _lib.lib.k2b200_last_error()


def test_no_rows_are_no_work():
    empty = rows(outer=0, scores=None)
    assert token_scores(empty) == 0 and token_backward(empty) == 0
    assert distil_backward(empty, teacher()) == 0


def test_a_host_can_ask_whether_they_are_there():
    """A library of the same version that came before them has no minor version."""
    assert (_lib.lib.k2b200_abi_version(), _lib.lib.k2b200_abi_minor_version()) >= (5, 1)


def test_there_is_no_cpu_path():
    x, token = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        k2.token_log_probs(x, token)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        k2.distillation_loss(x, token[:, None], torch.zeros(2, 1))


def test_the_references_agree_with_torch():
    """The definitions that the GPU is held to, against torch's own losses and derivatives."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(5, 30, generator=g, dtype=torch.float64)
    token = torch.randint(0, 30, (5,), generator=g)
    up = {"log_probs": torch.randn(5, generator=g), "entropy": torch.randn(5, generator=g),
          "top_log_probs": torch.randn(5, 4, generator=g)}
    want, _ = tokens_reference(x, token, 4, None, up)
    leaf = x.clone().requires_grad_(True)
    log_p = torch.log_softmax(leaf, -1)
    top = torch.topk(log_p, 4)
    h = torch.distributions.Categorical(logits=leaf).entropy()
    given = -torch.nn.functional.nll_loss(log_p, token, reduction="none")
    torch.autograd.backward([given, h, top.values], [v.double() for v in up.values()])
    assert torch.allclose(want["grad"], leaf.grad, rtol=0, atol=1e-12)
    assert torch.allclose(want["entropy"], h) and torch.allclose(want["log_probs"], given)
    assert torch.equal(want["top_tokens"].long(), top.indices)
    tt = torch.stack([torch.randperm(30, generator=g)[:6] for _ in range(5)])
    lp = torch.randn(5, 6, generator=g, dtype=torch.float64)
    want, _ = distil_reference(x, tt, lp, 2.0, 0.7, "sum")
    leaf = x.clone().requires_grad_(True)
    target = torch.zeros(5, 30, dtype=torch.float64).scatter_(1, tt, torch.softmax(lp / 2, -1))
    loss = 0.7 * 4 * torch.nn.functional.kl_div(torch.log_softmax(leaf / 2, -1), target,
                                                reduction="sum")
    loss.backward()
    assert torch.allclose(want["loss"], loss.detach())
    assert torch.allclose(want["grad"], leaf.grad, rtol=0, atol=1e-12)
