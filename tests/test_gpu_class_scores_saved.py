"""What the backward passes of `token_log_probs` and `distillation_loss` read is what was saved
for them: under hooks that keep tensors elsewhere, and where the caller's tensors have changed
since."""
import pytest
import torch
from torch.autograd.graph import (allow_mutation_on_saved_tensors, save_on_cpu,
                                  saved_tensors_hooks)
from torch.utils.checkpoint import checkpoint

import k2_b200 as k2
from class_scores_util import assert_close, distil_reference, tokens_reference

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
SHAPE = (3, 5)


def inputs(classes, dtype=torch.float32, time_first=False, entries=6):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(*SHAPE, classes, generator=g) * 2
    data = dict(x=x.to(dtype), tokens=torch.randint(0, classes, SHAPE, generator=g),
                teacher_tokens=torch.randint(-1, classes, SHAPE + (entries,), generator=g),
                teacher=torch.randn(*SHAPE, entries, generator=g),
                lengths=torch.tensor([5, 2, 4]))
    data = {k: v.to(DEV) for k, v in data.items()}
    if time_first:
        data["x"] = data["x"].transpose(0, 1).contiguous().transpose(0, 1)
    return data


def live(lengths):
    return torch.arange(SHAPE[1])[None] < lengths.cpu()[:, None]


def call(kind, x, d, lengths):
    """A scalar of all that `kind` gives in the logits x."""
    if kind == "tokens":
        got = k2.token_log_probs(x, d["tokens"], top_k=4, entropy=True, lengths=lengths)
        return got.log_probs.sum() + 2 * got.entropy.sum() + got.top_log_probs.sum()
    reduction, by = {"sum": ("sum", 1), "scaled": ("mean", 3), "rows": ("none", 1)}[kind]
    loss = k2.distillation_loss(x, d["teacher_tokens"], d["teacher"], 2.0, 0.5, reduction,
                                lengths)
    return (loss if by == 1 else by * loss) if reduction != "none" else loss.sum()


def expected(kind, d):
    if kind == "tokens":
        up = dict(log_probs=torch.ones(SHAPE), entropy=2 * torch.ones(SHAPE),
                  top_log_probs=torch.ones(SHAPE + (4,)))
        want, tol = tokens_reference(d["x"], d["tokens"], 4, live(d["lengths"]), up)
    else:
        reduction, up = {"sum": ("sum", None), "scaled": ("mean", torch.tensor(3.0)),
                         "rows": ("none", None)}[kind]
        want, tol = distil_reference(d["x"], d["teacher_tokens"], d["teacher"], 2.0, 0.5,
                                     reduction, live(d["lengths"]), up)
    return want["grad"], tol["grad"]


KINDS = ["tokens", "sum", "scaled", "rows"]


def read_by(kind):
    return ["logits", "lengths"] + (["tokens"] if kind == "tokens"
                                    else ["teacher_tokens", "teacher"])


@pytest.mark.parametrize("classes", [40, 2500])
@pytest.mark.parametrize("kind", KINDS)
def test_changes_that_are_allowed_do_not_reach_the_gradient(kind, classes):
    want, tol = expected(kind, inputs(classes))
    for victim in read_by(kind):
        d = inputs(classes)
        x = d["x"].requires_grad_(True)
        with allow_mutation_on_saved_tensors():
            y = x * 1.0
            out = call(kind, y, d, d["lengths"])
            with torch.no_grad():
                (y if victim == "logits" else d[victim]).fill_(1)
            grad, = torch.autograd.grad(out, x)
        assert_close(grad, want, tol, victim)


@pytest.mark.parametrize("time_first", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", KINDS)
def test_what_was_kept_on_the_cpu_is_what_is_read(kind, dtype, time_first):
    want, tol = expected(kind, inputs(501, dtype))
    for victim in read_by(kind):
        d = inputs(501, dtype, time_first)
        x = d["x"].requires_grad_(True)
        with save_on_cpu():
            y = x * 1.0
            out = call(kind, y, d, d["lengths"])
        with torch.no_grad():
            (y if victim == "logits" else d[victim]).fill_(1)
        grad, = torch.autograd.grad(out, x)
        assert_close(grad, want, tol, victim)


@pytest.mark.parametrize("kind", KINDS)
def test_hooks_may_give_other_strides_and_alignment(kind):
    d = inputs(501, torch.float16)
    want, tol = expected(kind, d)

    def pack(t):
        wide = torch.zeros(t.shape[:-1] + (t.shape[-1] + 3,), dtype=t.dtype, device=t.device)
        wide[..., 1:-2] = t
        return wide

    x = d["x"].requires_grad_(True)
    with saved_tensors_hooks(pack, lambda wide: wide[..., 1:-2]):
        out = call(kind, x, d, d["lengths"])
    grad, = torch.autograd.grad(out, x)
    assert_close(grad, want, tol)


@pytest.mark.parametrize("kind", KINDS)
def test_hooks_that_give_something_else_are_refused(kind):
    def narrow(t):
        return t[..., :-1]

    for pack, unpack in ((lambda t: t, narrow), (torch.Tensor.cpu, lambda t: t),
                         (lambda t: t, lambda t: t.to(torch.float64))):
        d = inputs(40)
        x = d["x"].requires_grad_(True)
        with saved_tensors_hooks(pack, unpack):
            out = call(kind, x, d, d["lengths"])
        with pytest.raises(RuntimeError, match="saved tensor"):
            torch.autograd.grad(out, x)


@pytest.mark.parametrize("kind", KINDS)
def test_hooks_take_all_that_is_large(kind):
    """Between the passes nothing of the logits' size stays on the device."""
    d = inputs(200003)
    size = d["x"].numel() * 4
    x = d["x"].requires_grad_(True)
    torch.cuda.synchronize()
    with save_on_cpu():
        before = torch.cuda.memory_allocated()
        y = x * 1.0
        out = call(kind, y, d, d["lengths"])
        del y
        torch.cuda.synchronize()
        assert torch.cuda.memory_allocated() - before < size / 2
    grad, = torch.autograd.grad(out, x)
    want, tol = expected(kind, d)
    assert_close(grad, want, tol)


@pytest.mark.parametrize("kind", KINDS)
def test_in_a_part_that_is_computed_again(kind):
    d = inputs(501)
    want, tol = expected(kind, d)
    x = d["x"].requires_grad_(True)
    out = checkpoint(lambda t: call(kind, t * 1.0, d, d["lengths"]), x, use_reentrant=False)
    grad, = torch.autograd.grad(out, x)
    assert_close(grad, want, tol)


@pytest.mark.parametrize("kind", ["tokens", "rows"])
def test_copies_are_the_calls_own(kind):
    """Lengths on the CPU are read at the call, and tokens with gaps are copied there: the
    gradient does not care what becomes of them."""
    d = inputs(40)
    want, tol = expected(kind, d)
    lengths = d["lengths"].cpu()
    for name in ("tokens", "teacher_tokens"):
        d[name] = torch.stack([d[name], d[name]], -1)[..., 0]
    x = d["x"].requires_grad_(True)
    out = call(kind, x, d, lengths)
    for t in (lengths, d["tokens"], d["teacher_tokens"]):
        t.zero_()
    grad, = torch.autograd.grad(out, x)
    assert_close(grad, want, tol)


def test_only_what_a_gradient_needs_is_asked_for():
    """Top classes may be changed where no gradient comes back through their log-probs."""
    d = inputs(40)
    x = d["x"].requires_grad_(True)
    got = k2.token_log_probs(x, d["tokens"], top_k=3)
    got.top_tokens.zero_()
    grad, = torch.autograd.grad(got.log_probs.sum(), x)
    want, tol = tokens_reference(x.detach(), d["tokens"], 0, None,
                                 dict(log_probs=torch.ones(SHAPE)))
    assert_close(grad, want["grad"], tol["grad"])


@pytest.mark.parametrize("kind", KINDS)
def test_what_a_hook_raises_arrives(kind):
    class Stop(Exception):
        pass

    def stop(t):
        raise Stop

    d = inputs(40)
    x = d["x"].requires_grad_(True)
    with saved_tensors_hooks(stop, lambda t: t), pytest.raises(Stop):
        call(kind, x, d, d["lengths"])
    with saved_tensors_hooks(lambda t: t, stop):
        out = call(kind, x, d, d["lengths"])
    with pytest.raises(Stop):
        torch.autograd.grad(out, x)


@pytest.mark.parametrize("reduction", ["none", "sum"])
def test_a_teacher_in_inference_mode(reduction):
    """Its tensors have no versions that could be compared: they are copied."""
    g = torch.Generator().manual_seed(0)
    of_teacher = torch.randn(*SHAPE, 60, generator=g).to(DEV)
    x = torch.randn(*SHAPE, 60, generator=g).to(DEV).requires_grad_(True)
    with torch.inference_mode():
        lengths = torch.tensor([5, 2, 4], device=DEV)
        named = k2.token_log_probs(of_teacher, top_k=8, lengths=lengths)
    loss = k2.distillation_loss(x, named.top_tokens, named.top_log_probs, reduction=reduction,
                                lengths=lengths)
    scored = k2.token_log_probs(x, named.top_tokens[..., 0], lengths=lengths)
    want, tol = distil_reference(x.detach(), named.top_tokens, named.top_log_probs, 1.0, 1.0,
                                 reduction, live(lengths))
    up = dict(log_probs=torch.ones(SHAPE))
    given, given_tol = tokens_reference(x.detach(), named.top_tokens[..., 0].clone(), 0,
                                        live(lengths), up)
    with torch.inference_mode():
        named.top_tokens.zero_()
        named.top_log_probs.zero_()
        lengths.zero_()
    grad, = torch.autograd.grad(loss.sum(), x)
    assert_close(grad, want["grad"], tol["grad"])
    grad, = torch.autograd.grad(scored.log_probs.sum(), x)
    assert_close(grad, given["grad"], given_tol["grad"])
