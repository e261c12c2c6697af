"""Rows of class scores whose sums are known to the last bits: a class that is lost, or that
comes twice, at an edge of what a thread, a block or a part of a row has, shows."""
import math

import pytest
import torch

import k2_b200 as k2

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = [torch.float32, torch.float16, torch.bfloat16]
E32 = 2.0 ** -24  # half a step of float32, relative

# rows, classes: a warp's, a block's, few rows over clusters, rows that no cluster holds at once
LONG = [(700, 1500), (700, 5000), (300, 16391), (160, 50021), (300, 32001), (2, 50021),
        (2, 131072), (1, 300007), (1, 1000003)]


def close_log(got, n, what):
    """got against ln n in 64 bits: a logarithm of an exact sum, which is off by one unit of the
    last place at most (2^-23 relative), and one rounding."""
    want = math.log(n)
    off = (got.double() - want).abs().max().item()
    assert off <= 3 * E32 * abs(want), (what, off, want)


def edges(classes, size, shift):
    """Classes at the edges of vectors of 16 bytes, of the slices of 1 to 8 blocks, of the parts
    of a slice that 32 to 512 threads have of at most 24 vectors each, of a thread's turns."""
    per = 16 // size
    vectors = (shift + classes + per - 1) // per
    at = set()
    for cluster in (1, 2, 4, 8):
        width = -(-vectors // cluster)
        for first in range(0, vectors, width):
            last = min(vectors, first + width)
            at.update((first, last - 1))
            for team in (32, 128, 256, 512):
                at.update((min(last - 1, first + team - 1), min(last - 1, first + team)))
                each = -(-(last - first) // team)
                for most in {min(24, each), min(28, each), each}:
                    for tile in range(first, last, team * most):
                        at.update((tile, max(first, tile - 1)))
    classes_at = {v * per - shift + k for v in at for k in (0, 1, per - 1)}
    classes_at.update(range(20))
    classes_at.update(range(classes - 20, classes))
    return sorted(c for c in classes_at if 0 <= c < classes)


def shifted(rows, classes, dtype, shift, value):
    """[rows, classes] that begins `shift` elements behind a vector of 16 bytes."""
    flat = torch.full((rows * classes + 16,), value, dtype=dtype, device=DEV)
    return flat[shift:shift + rows * classes].view(rows, classes)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,classes", LONG)
def test_rows_of_one_value(rows, classes, dtype):
    """Every class adds exactly 1 to the sum, so that the log-probs are -ln C to the last bits: of
    1000003 classes a lost vector of 4 changes them by 4e-6, where 2.5e-6 is the bound."""
    x = shifted(rows, classes, dtype, 1, 2.5).requires_grad_(True)
    token = torch.randint(0, classes, (rows,), device=DEV)
    # (without top classes rows take another way, and so they do without an entropy)
    for top_k, entropy in ((0, False), (0, True), (7, True)):
        got = k2.token_log_probs(x, token, top_k=top_k, entropy=entropy)
        close_log(-got.log_probs.detach(), classes, "log_probs")
        if entropy:
            close_log(got.entropy.detach(), classes, "entropy")
        if top_k:
            close_log(-got.top_log_probs.detach(), classes, "top")
            assert (got.top_tokens.cpu() == torch.arange(top_k)).all()
    loss = k2.distillation_loss(x, token[:, None], torch.zeros(rows, 1, device=DEV),
                                reduction="none")
    close_log(loss.detach(), classes, "loss")


@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,classes", LONG)
def test_rows_with_classes_at_every_edge(rows, classes, dtype, shift):
    """All but n classes have probability 0, and those 1 / n: the sum is n, exactly.  Rows behind
    the first begin at other places of a vector, and have the first row's classes."""
    size = torch.tensor([], dtype=dtype).element_size()
    some = edges(classes, size, shift)
    n = len(some)
    at = torch.tensor(some, device=DEV)
    x = shifted(rows, classes, dtype, shift, -math.inf)
    x[:, at] = -3.0
    x.requires_grad_(True)
    token = at[torch.randint(0, n, (rows,), device=DEV)]
    top_k = min(n, 128)
    for k, entropy in ((0, False), (0, True), (top_k, True)):
        got = k2.token_log_probs(x, token, top_k=k, entropy=entropy)
        close_log(-got.log_probs.detach(), n, "log_probs")
        if entropy:
            close_log(got.entropy.detach(), n, "entropy")
        if k:
            close_log(-got.top_log_probs.detach(), n, "top")
            assert torch.equal(got.top_tokens, at[:k].int().expand(rows, k))
    # gradients: p is 2^0 / n in float32 (two roundings), then rounded to the scores' type; the
    # given class has one rounding of p - 1 more
    given, = torch.autograd.grad(got.log_probs.sum(), x)
    loss = k2.distillation_loss(x, token[:, None], torch.zeros(rows, 1, device=DEV))
    want = rows * math.log(n)
    # (rows' losses in float32, their sum in 64 bits and rounded)
    assert abs(loss.item() - want) <= 4 * E32 * want
    made, = torch.autograd.grad(loss, x, retain_graph=True)
    again, = torch.autograd.grad(loss, x, torch.tensor(2.0, device=DEV))
    p = torch.zeros(rows, classes, dtype=torch.float64, device=DEV)
    p[:, at] = 1.0 / n
    p[torch.arange(rows, device=DEV), token] -= 1.0
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    for grad, by in ((given, -1), (made, 1), (again, 2)):
        off = (grad.double() - by * p).abs()
        assert (off <= (half * (1 + E32) + 3 * E32) * (by * p).abs() + E32 * abs(by) * (p < 0)
                + tiny * (p != 0)).all(), (by, off.max().item())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,classes", LONG)
def test_one_class_in_each_part_of_a_row(rows, classes, dtype):
    """The largest score in one place, and the rest so far below that it does not matter: whatever
    part of a row has it, and whatever the parts before and behind it found as their largest."""
    size = torch.tensor([], dtype=dtype).element_size()
    some = edges(classes, size, 0)
    picks = some[::max(1, len(some) // 12)]
    for c in picks:
        x = shifted(rows, classes, dtype, 0, -200.0)
        x[:, c] = 5.0
        x.requires_grad_(True)
        token = torch.full((rows,), c, device=DEV)
        # ln (1 + (C - 1) e^-205) is 0 in 64 bits too
        for k, entropy in ((0, False), (0, True), (2, True)):
            got = k2.token_log_probs(x, token, top_k=k, entropy=entropy)
            assert (got.log_probs == 0).all() and (not entropy or (got.entropy == 0).all())
            if k:
                assert (got.top_tokens[:, 0] == c).all()
                assert (got.top_tokens[:, 1] == (1 if c == 0 else 0)).all()
        loss = k2.distillation_loss(x, token[:, None], torch.zeros(rows, 1, device=DEV))
        assert loss == 0
        made, = torch.autograd.grad(loss, x)
        assert (made == 0).all()
