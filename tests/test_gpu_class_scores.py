"""`token_log_probs` and `distillation_loss` on the GPU against their definitions in 64 bits."""
import gc
import itertools
import math

import pytest
import torch

import k2_b200 as k2
from class_scores_util import assert_close, distil_reference, tokens_reference

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = [torch.float32, torch.float16, torch.bfloat16]

# rows before the classes: one, a few, odd numbers; classes: fewer than lanes, odd ones, the
# framework's own, a power of two and its neighbours, and what no block holds at once
SHAPES = [((), 1), ((1,), 2), ((3,), 5), ((2, 5), 29), ((7,), 64), ((4, 33), 500), ((2, 7), 501),
          ((3,), 1023), ((2, 3), 1025), ((5,), 2049), ((3, 3), 5000), ((2, 2), 16391),
          ((3,), 32001), ((2,), 131072), ((1,), 300007)]


def scores(shape, dtype, seed=0, sigma=2.0, peak=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * sigma
    if peak:
        at = torch.randint(0, shape[-1], shape[:-1] + (1,), generator=g)
        x.scatter_add_(-1, at, torch.full(at.shape, peak))
    return x.to(dtype)


def ints(low, high, shape, seed=0):
    return torch.randint(low, high, shape, generator=torch.Generator().manual_seed(seed))


def check_tokens(x, token=None, top_k=0, entropy=True, lengths=None, seed=3, backward=True):
    """x: a tensor on the device, as the call gets it."""
    x = x.detach().requires_grad_(backward)
    got = k2.token_log_probs(x, token, top_k=top_k, entropy=entropy, lengths=lengths)
    live = None
    if lengths is not None:
        live = torch.arange(x.shape[1])[None] < lengths.cpu()[:, None]
    names = [n for n in ("log_probs", "entropy", "top_log_probs")
             if getattr(got, n) is not None]
    g = torch.Generator().manual_seed(seed)
    up = {n: torch.randn(getattr(got, n).shape, generator=g) for n in names}
    want, tol = tokens_reference(x.detach(), token, top_k, live, up)
    for n in names:
        assert getattr(got, n).dtype == torch.float32
        assert_close(getattr(got, n), want[n], tol[n], n)
    if top_k:
        assert got.top_tokens.dtype == torch.int32
        assert torch.equal(got.top_tokens.cpu(), want["top_tokens"])
    if backward:
        grad, = torch.autograd.grad([getattr(got, n) for n in names], x,
                                    [up[n].to(DEV) for n in names])
        assert grad.dtype == x.dtype
        assert_close(grad, want["grad"], tol["grad"], "grad")
    return got


def teacher(shape, classes, entries, seed=0, missing=0.0):
    g = torch.Generator().manual_seed(seed)
    rows = math.prod(shape)
    tokens = torch.stack([torch.randperm(classes, generator=g)[:entries]
                          for _ in range(rows)]) if rows else torch.zeros(0, entries)
    tokens = tokens.reshape(*shape, entries).long()
    lp = torch.randn(*shape, entries, generator=g) * 2 - 3
    if missing:
        tokens[torch.rand(tokens.shape, generator=g) < missing] = -1
    return tokens, lp


def check_distil(x, tokens, lp, lengths=None, up=None, **kw):
    x = x.detach().requires_grad_(True)
    loss = k2.distillation_loss(x, tokens, lp, lengths=lengths, **kw)
    live = None
    if lengths is not None:
        live = torch.arange(x.shape[1])[None] < lengths.cpu()[:, None]
    if up is None:
        up = torch.ones(loss.shape) if loss.dim() == 0 else torch.linspace(
            -1, 2, loss.numel()).reshape(loss.shape)
    want, tol = distil_reference(x.detach(), tokens, lp, kw.get("temperature", 1.0),
                                 kw.get("weight", 1.0), kw.get("reduction", "sum"), live, up)
    assert loss.dtype == torch.float32
    assert_close(loss, want["loss"], tol["loss"], "loss")
    grad, = torch.autograd.grad(loss, x, up.to(DEV))
    assert grad.dtype == x.dtype
    assert_close(grad, want["grad"], tol["grad"], "grad")
    with torch.no_grad():  # the same without a gradient
        again = k2.distillation_loss(x, tokens, lp, lengths=lengths, **kw)
    assert torch.equal(again.nan_to_num(7), loss.detach().nan_to_num(7))
    return loss, grad


# --------------------------------------------------------------------------- token_log_probs
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,classes", SHAPES)
def test_tokens_and_entropy(shape, classes, dtype):
    x = scores(shape + (classes,), dtype, seed=classes, peak=4.0).to(DEV)
    check_tokens(x, ints(-1, classes, shape, 5).to(DEV))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,classes", SHAPES)
def test_top_classes(shape, classes, dtype):
    x = scores(shape + (classes,), dtype, seed=classes + 1).to(DEV)
    for top_k in sorted({1, min(3, classes), min(8, classes), min(33, classes),
                         min(128, classes)}):
        check_tokens(x, ints(0, classes, shape, 6).to(DEV, torch.int32), top_k=top_k,
                     entropy=top_k % 2 == 0)


@pytest.mark.parametrize("top_k", [1, 5, 16, 17, 40, 64, 100, 128])
@pytest.mark.parametrize("classes", [128, 500, 1300, 5000, 40000])
def test_top_classes_of_awkward_rows(classes, top_k):
    """Rows whose order is all ties, sorted either way, or has its largest scores side by side or
    at a stride, where a thread, a warp or a vector of loads holds all of them."""
    c = torch.arange(classes, dtype=torch.float32)
    rows = [torch.zeros(classes), c / 16, -c / 16, (c % 2), (c % 7) - 3,
            torch.where(c < 130, 100 - c / 4, -c / 256), torch.where(c >= classes - 130, c, -c),
            torch.full((classes,), -math.inf), torch.where(c % 3 == 0, 0.0, -math.inf),
            torch.where(c % 2 == 0, 0.0, -0.0), torch.where(c == 7, 1.0, -math.inf)]
    for stride in (4, 8, 32, 128, 256, 1024, 2048):
        rows.append(torch.where(c % stride == 3, 50 + c / 1024, -1.0))
    for dtype in TYPES:
        x = torch.stack(rows).to(dtype).to(DEV)
        check_tokens(x, None, top_k=top_k, entropy=False, backward=False)
        check_tokens(x[:, 1:], None, top_k=min(top_k, classes - 1), entropy=False,
                     backward=False)


# rows enough for every way that they are dealt out: a warp each (short rows in registers, longer ones
# in shared memory), blocks of several sizes, clusters, and rows that not even a cluster holds
MANY = [(700, 2100), (600, 5003), (593, 9000), (600, 9300), (160, 20000), (150, 33333),
        (149, 60001), (75, 40000), (2, 1000003)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,classes", MANY)
def test_every_way_that_rows_are_dealt_out(rows, classes, dtype):
    """All rows are computed, some of them looked at."""
    g = torch.Generator(device=DEV).manual_seed(rows)
    wide = torch.randn(rows, classes + 1, device=DEV, generator=g).mul_(2).to(dtype)
    pick = torch.unique(torch.cat([torch.arange(0, rows, max(1, rows // 12)),
                                   torch.tensor([rows - 1])])).to(DEV)
    token = ints(-1, classes, (rows,), 1).to(DEV)
    tt = ints(0, classes, (rows, 40), 2).to(DEV)
    tt[::3, 7:] = -1
    tt[1] = -1
    lp = torch.randn(rows, 40, device=DEV, generator=g)
    live = torch.ones(rows, dtype=torch.bool)
    live[2::7] = False
    # (rows as sequences of one frame)
    lengths = live.to(DEV, torch.int32)
    up = {n: torch.randn(rows, *more, device=DEV, generator=g)
          for n, more in (("log_probs", ()), ("entropy", ()), ("top_log_probs", (20,)))}
    # adjacent rows, and rows of a wider matrix, whose gradient lies otherwise
    for x in (wide.reshape(-1)[:rows * classes].view(rows, classes), wide[:, 1:]):
        for top_k in (0, 20):
            leaf = x[:, None].detach().requires_grad_(True)
            got = k2.token_log_probs(leaf, token[:, None], top_k=top_k, entropy=True,
                                     lengths=lengths)
            names = ["log_probs", "entropy"] + (["top_log_probs"] if top_k else [])
            grad, = torch.autograd.grad([getattr(got, n) for n in names], leaf,
                                        [up[n][:, None] for n in names])
            want, tol = tokens_reference(x[pick], token[pick], top_k, live[pick.cpu()],
                                         {n: up[n][pick] for n in names})
            for n in names:
                assert_close(getattr(got, n)[pick, 0], want[n], tol[n], n)
            if top_k:
                assert torch.equal(got.top_tokens[pick, 0].cpu(), want["top_tokens"])
            assert_close(grad[pick, 0], want["grad"], tol["grad"], "grad")
            assert (grad[~live.to(DEV)] == 0).all()
        for reduction, upstream in (("sum", None), ("none", up["entropy"])):
            leaf = x[:, None].detach().requires_grad_(True)
            loss = k2.distillation_loss(leaf, tt[:, None], lp[:, None], 2.0, 0.5, reduction,
                                        lengths)
            grad, = torch.autograd.grad(loss, leaf, None if upstream is None
                                        else upstream[:, None])
            want, tol = distil_reference(x[pick], tt[pick], lp[pick], 2.0, 0.5, reduction,
                                         live[pick.cpu()],
                                         None if upstream is None else upstream[pick])
            assert_close(grad[pick, 0], want["grad"], tol["grad"], "grad")
            assert (grad[~live.to(DEV)] == 0).all()
            if reduction == "none":
                each = loss.detach()
                assert_close(loss[pick, 0], want["loss"], tol["loss"], "loss")
        # the sum is that of the rows' own, which the same kernel computes (halving them is exact):
        # added in 64 bits and rounded once, by half a step of float32
        with torch.no_grad():
            total = k2.distillation_loss(x[:, None], tt[:, None], lp[:, None], 2.0, 0.5, "sum",
                                         lengths)
        rows_sum = each.double().sum()
        assert abs(float(total - rows_sum)) <= 2.0 ** -23 * float(each.double().abs().sum())


@pytest.mark.parametrize("rows,classes", [(300007, 9), (160001, 33)])
def test_more_rows_than_a_warp_takes_at_once(rows, classes):
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(rows, classes, device=DEV, generator=g)
    token = ints(0, classes, (rows,), 1).to(DEV)
    tt = ints(0, classes, (rows, 3), 2).to(DEV)
    lp = torch.randn(rows, 3, device=DEV, generator=g)
    check_tokens(x, token, top_k=2)
    check_distil(x, tt, lp, reduction="none")
    check_distil(x, tt, lp, reduction="mean")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [40, 500, 501, 1000])
def test_order_of_the_smallest_differences(classes, dtype):
    """Subnormals, zeros of both signs and neighbours of a type are told apart as numbers are."""
    g = torch.Generator().manual_seed(classes)
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # the smallest subnormal
    steps = torch.randint(-5, 6, (8, classes), generator=g).double()
    rows = [steps * tiny, steps.clamp(max=0) * tiny, steps.sign() * 0.0,
            1 + steps * torch.finfo(dtype).eps, -1 - steps * torch.finfo(dtype).eps]
    x = torch.cat(rows).to(dtype)
    assert ((x == 0).any(1) & (x != 0).any(1)).any()
    for top_k in (1, 2, 7, 8, 9, 30):
        check_tokens(x.to(DEV), None, top_k=top_k, entropy=False, backward=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [5, 77, 500, 5000, 33001])
def test_rows_with_infinities_and_lowest_values(classes, dtype):
    low = torch.finfo(dtype).min
    x = scores((9, classes), dtype, seed=3)
    x[0] = -math.inf
    x[1] = low
    x[2, ::2] = -math.inf
    x[3, 1:] = -math.inf
    x[4, 1:] = low
    x[5] = torch.finfo(dtype).max
    x[6, :-1] = -math.inf
    x[7] = 0
    x = x.to(DEV)
    token = torch.tensor([1, 2, 2, 0, 1, 0, classes - 1, classes // 2, 4], device=DEV)
    check_tokens(x, token, top_k=min(4, classes))
    got = k2.token_log_probs(x, token, top_k=1, entropy=True)
    assert got.log_probs[0] == -math.inf and got.entropy[0] == 0 and got.top_tokens[0] == 0
    assert got.log_probs[3] == 0 and got.entropy[3] == 0


@pytest.mark.parametrize("classes", [5, 500, 3000, 50000])
def test_rows_with_nan_and_plus_infinity(classes):
    x = scores((4, classes), torch.float32, seed=4)
    x[0, 3] = math.nan
    x[1, 2] = math.inf
    x[2, classes - 1] = math.nan
    x[2, 1] = -math.nan
    x = x.to(DEV).requires_grad_(True)
    got = k2.token_log_probs(x, torch.zeros(4, dtype=torch.int32, device=DEV), top_k=3,
                             entropy=True)
    grad, = torch.autograd.grad(got.log_probs.sum() + got.entropy.sum(), x)
    for v in (got.log_probs, got.entropy, got.top_log_probs, grad):
        assert torch.isnan(v[:3]).any(-1).all() if v.dim() > 1 else torch.isnan(v[:3]).all()
        assert torch.isfinite(v[3]).all()
    want, _ = tokens_reference(x.detach(), top_k=3)
    assert torch.equal(got.top_tokens.cpu(), want["top_tokens"])


def test_tokens_that_are_no_class():
    x = scores((5, 40), torch.float32).to(DEV).requires_grad_(True)
    token = torch.tensor([-1, -2, 40, 2**31 + 3, 39], device=DEV)
    got = k2.token_log_probs(x, token)
    assert got.log_probs[0] == 0 and torch.isnan(got.log_probs[1:4]).all()
    grad, = torch.autograd.grad(got.log_probs.sum(), x)
    assert (grad[0] == 0).all() and torch.isnan(grad[1:4]).all() and (grad[4] != 0).any()
    # without an upstream for the log-probs, they do not matter
    got = k2.token_log_probs(x, token, entropy=True)
    grad, = torch.autograd.grad(got.entropy.sum(), x)
    assert torch.isfinite(grad).all()


def layouts(x):
    """Tensors that are equal to x and lie otherwise in memory (x: [N, T, C])."""
    n, t, c = x.shape
    yield "time first", x.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.full((n, t, c + 3), 9.0, dtype=x.dtype, device=x.device)
    wide[..., 2:2 + c] = x
    yield "columns of a wider matrix", wide[..., 2:2 + c]
    every = torch.full((n, 2 * t + 1, c), 9.0, dtype=x.dtype, device=x.device)
    every[:, 1::2][:, :t] = x
    yield "every second row", every[:, 1::2][:, :t]
    flat = torch.empty(n * t * c + 5, dtype=x.dtype, device=x.device)
    flat[5:] = x.reshape(-1)
    yield "behind an odd offset", flat[5:].view(n, t, c)
    yield "classes not adjacent", x.transpose(1, 2).contiguous().transpose(1, 2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [29, 500, 501, 5003])
def test_strides_and_alignment(classes, dtype):
    base = scores((3, 6, classes), dtype, seed=9).to(DEV)
    token = ints(-1, classes, (3, 6), 2).to(DEV)
    tt, lp = teacher((3, 6), classes, 7, missing=0.2)
    lengths = torch.tensor([6, 0, 4], device=DEV)
    for what, x in layouts(base):
        assert torch.equal(x, base), what
        for ls in (None, lengths):
            check_tokens(x, token, top_k=5, lengths=ls)
            check_tokens(x, token.t().contiguous().t(), lengths=ls)
            check_distil(x, tt.to(DEV), lp.to(DEV), lengths=ls)
            check_distil(x, tt.to(DEV, torch.int32), lp.to(DEV).transpose(0, 1).contiguous()
                         .transpose(0, 1), lengths=ls, reduction="none", temperature=1.5)
    # one row for all (stride 0), and four dimensions that no two strides describe
    row = base[:1, :1].expand(3, 6, classes)
    check_tokens(row, token, top_k=5)
    check_distil(row, tt.to(DEV), lp.to(DEV))
    four = scores((2, 3, 4, 5, classes), dtype).to(DEV)[:, ::2].transpose(0, 2)
    check_tokens(four, ints(0, classes, four.shape[:-1]).to(DEV), top_k=2)


def test_a_gradient_keeps_the_strides_of_the_logits():
    x = scores((5, 4, 30), torch.bfloat16).to(DEV).transpose(0, 1).requires_grad_(True)
    tt, lp = teacher((4, 5), 30, 3)
    loss = k2.distillation_loss(x, tt.to(DEV), lp.to(DEV))
    assert torch.autograd.grad(loss, x)[0].stride() == x.stride()
    lp = k2.token_log_probs(x, tt[..., 0].to(DEV)).log_probs
    assert torch.autograd.grad(lp.sum(), x)[0].stride() == x.stride()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [29, 500, 2500])
@pytest.mark.parametrize("where", ["cpu", DEV])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_lengths(kind, where, classes, dtype):
    n, t = 6, 9
    x = scores((n, t, classes), dtype).to(DEV)
    lengths = torch.tensor([0, 1, 9, 4, 100, -3]).to(kind).to(where)
    token = ints(0, classes, (n, t)).to(DEV)
    # what lies behind the lengths is not looked at
    x[1, 1:] = math.nan
    token[1, 1:] = 10**6
    got = check_tokens(x, token, top_k=3, lengths=lengths)
    for v in got:
        assert (v[0] == (-1 if v.dtype == torch.int32 else 0)).all()
    tt, lp = teacher((n, t), classes, 4)
    tt[1, 1:] = -7
    lp[1, 1:] = math.nan
    for reduction in ("sum", "mean", "none"):
        check_distil(x, tt.to(DEV), lp.to(DEV), lengths=lengths, reduction=reduction)
        none = torch.zeros(n, dtype=kind, device=where)
        loss, grad = check_distil(x, tt.to(DEV), lp.to(DEV), lengths=none, reduction=reduction)
        assert (loss == 0).all() and (grad == 0).all()


def test_no_rows():
    for shape in ((0, 7), (0, 5, 7), (3, 0, 7)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        token = torch.zeros(shape[:-1], dtype=torch.int64, device=DEV)
        got = k2.token_log_probs(x, token, top_k=2, entropy=True)
        assert got.log_probs.shape == shape[:-1] and got.top_tokens.shape == shape[:-1] + (2,)
        assert torch.autograd.grad(got.entropy.sum(), x)[0].shape == shape
        tt = torch.zeros(shape[:-1] + (3,), dtype=torch.int32, device=DEV)
        for reduction in ("sum", "mean"):
            loss = k2.distillation_loss(x, tt, tt.float(), reduction=reduction)
            assert loss == 0
            assert torch.autograd.grad(loss, x)[0].shape == shape
        loss = k2.distillation_loss(x, tt, tt.float(), reduction="none")
        assert loss.shape == shape[:-1]
        if len(shape) == 3:
            lengths = torch.zeros(shape[0], dtype=torch.int32, device=DEV)
            assert k2.distillation_loss(x, tt, tt.float(), lengths=lengths) == 0


def test_rows_behind_offsets_of_more_than_32_bits():
    # 2.3 G elements of one allocation: rows on both sides of 2^31 and one at its end
    c, pitch = 500, 1 << 20
    rows = 2200
    big = torch.empty(rows * pitch, dtype=torch.bfloat16, device=DEV)
    view = big.view(rows, pitch)[:, :c]
    x = scores((rows, c), torch.bfloat16).to(DEV)
    view.copy_(x)
    # Against the definition, not against the bits of the same rows elsewhere: these rows begin at
    # the start of a vector of 16 bytes, every second one of x 8 bytes behind it, so that its terms
    # are added in another order, and each sum is off by up to sum_error(c) on its own.
    got = k2.token_log_probs(view, None, top_k=6, entropy=True)
    want, tol = tokens_reference(x, None, 6)
    for name in ("entropy", "top_log_probs"):
        assert_close(getattr(got, name), want[name], tol[name], name)
    assert torch.equal(got.top_tokens.cpu(), want["top_tokens"])
    tt, lp = teacher((rows,), c, 3)
    loss = k2.distillation_loss(view, tt.to(DEV), lp.to(DEV), reduction="none")
    want, tol = distil_reference(x, tt, lp, reduction="none")
    assert_close(loss, want["loss"], tol["loss"])


@pytest.mark.parametrize("classes", [29, 500, 5000])
def test_any_of_the_upstreams(classes):
    x = scores((3, 4, classes), torch.float32).to(DEV)
    token = ints(0, classes, (3, 4)).to(DEV)
    for used in itertools.chain.from_iterable(itertools.combinations(
            ["log_probs", "entropy", "top_log_probs"], n) for n in (1, 2)):
        leaf = x.clone().requires_grad_(True)
        got = k2.token_log_probs(leaf, token, top_k=4, entropy=True)
        # a sum's gradient arrives with strides of 0, a transposed weight's transposed
        w = torch.linspace(-1, 1, 12, device=DEV).reshape(4, 3).t()
        up, loss = {}, 0
        for k, name in enumerate(used):
            v = getattr(got, name)
            if k == 0:
                loss = loss + v.sum() * 0.5
                up[name] = torch.full(v.shape, 0.5)
            else:
                weight = w if v.dim() == 2 else w[..., None].expand(3, 4, 4)
                loss = loss + (v * weight).sum()
                up[name] = weight
        loss.backward()
        want, tol = tokens_reference(x, token, 4, None, up)
        assert_close(leaf.grad, want["grad"], tol["grad"], str(used))


# --------------------------------------------------------------------------- distillation_loss
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,classes", SHAPES)
def test_distillation(shape, classes, dtype):
    x = scores(shape + (classes,), dtype, seed=classes, peak=3.0).to(DEV)
    for entries, temperature, reduction in ((1, 1.0, "sum"), (min(8, classes), 2.0, "mean"),
                                            (min(16, classes), 1.0, "none"),
                                            (min(33, classes), 0.5, "sum"),
                                            (min(128, classes), 3.0, "none")):
        tt, lp = teacher(shape, classes, entries, entries, missing=0.1)
        check_distil(x, tt.to(DEV), lp.to(DEV), temperature=temperature, weight=0.7,
                     reduction=reduction)


@pytest.mark.parametrize("kind", TYPES)
def test_types_of_the_teacher(kind):
    x = scores((4, 5, 60), torch.float16).to(DEV)
    tt, lp = teacher((4, 5), 60, 9)
    check_distil(x, tt.to(DEV, torch.int32), lp.to(kind).to(DEV))


@pytest.mark.parametrize("classes", [6, 500, 5000, 40000])
def test_odd_teachers(classes):
    x = scores((9, classes), torch.float32, seed=2)
    x[8] = -math.inf
    x[7, 1] = -math.inf
    tt, lp = teacher((9,), classes, 5, 3)
    tt[0] = -1  # nothing there
    lp[0] = math.nan  # ... whatever its score
    lp[1] = -math.inf  # no mass
    tt[2] = 3  # one class five times
    tt[3, 1], tt[3, 4] = tt[3, 0], tt[3, 0]
    lp[4, 2] = -math.inf
    lp[5] += 1e4
    lp[6] = torch.tensor([0.0, -300.0, 500.0, 0.0, 1.0])
    tt[7] = torch.tensor([1, 0, 2, 3, 4])  # a class that the student rules out
    for reduction in ("none", "sum"):
        rows = 7 if reduction == "sum" else 9
        loss, grad = check_distil(x[:rows].to(DEV), tt[:rows].to(DEV), lp[:rows].to(DEV),
                                  reduction=reduction)
        assert (grad[:2] == 0).all()
    assert (loss[7:] == math.inf).all() if loss.dim() else True
    # a class without mass may be ruled out
    lp[7, 0] = -math.inf
    check_distil(x[:8].to(DEV), tt[:8].to(DEV), lp[:8].to(DEV), reduction="none")


def test_wrong_teachers_are_nan_in_their_row_alone():
    x = scores((6, 50), torch.float32).to(DEV)
    tt, lp = teacher((6,), 50, 4)
    tt[0, 1], tt[1, 2], tt[2, 3] = 50, -2, 2**40
    lp[3, 0], lp[4, 0] = math.nan, math.inf
    x = x.requires_grad_(True)
    loss = k2.distillation_loss(x, tt.to(DEV), lp.to(DEV), reduction="none")
    grad, = torch.autograd.grad(loss.sum(), x)
    assert torch.isnan(loss[:5]).all() and torch.isfinite(loss[5])
    assert torch.isnan(grad[:5]).all() and torch.isfinite(grad[5]).all()
    loss = k2.distillation_loss(x, tt.to(DEV), lp.to(DEV))
    grad, = torch.autograd.grad(loss, x)
    assert torch.isnan(loss) and torch.isnan(grad[:5]).all() and torch.isfinite(grad[5]).all()
    # a student's NaN
    bad = x.detach().clone()
    bad[5, 3], bad[4, 2] = math.nan, math.inf
    lp[4, 0] = 0
    loss = k2.distillation_loss(bad, tt.to(DEV), lp.to(DEV), reduction="none")
    assert torch.isnan(loss[4:]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [29, 500, 5000, 20011])
@pytest.mark.parametrize("reduction", ["sum", "mean"])
def test_an_upstream_other_than_one(reduction, classes, dtype):
    x = scores((3, 4, classes), dtype).to(DEV)
    tt, lp = teacher((3, 4), classes, 6)
    for up in (-3.0, 0.0, 0.37, 1024.0):
        check_distil(x, tt.to(DEV), lp.to(DEV), reduction=reduction, up=torch.tensor(up),
                     temperature=1.7)


def test_differentiated_again():
    x = scores((3, 40), torch.float32).to(DEV).requires_grad_(True)
    tt, lp = teacher((3,), 40, 6)
    loss = k2.distillation_loss(x, tt.to(DEV), lp.to(DEV))
    loss.backward(retain_graph=True)
    first = x.grad.clone()
    loss.backward(retain_graph=True)
    assert torch.equal(x.grad, 2 * first)
    (second,) = torch.autograd.grad(2 * loss, x)
    assert torch.equal(second, 2 * first)
    with pytest.raises(RuntimeError, match="already differentiated"):
        loss.backward()
    lp = k2.token_log_probs(x, tt[:, 0].to(DEV)).log_probs.sum()
    a, = torch.autograd.grad(lp, x, retain_graph=True)
    b, = torch.autograd.grad(lp, x)
    assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="already differentiated"):
        lp.backward()


def test_what_changed_in_between_is_noticed():
    tt, lp = teacher((3,), 40, 6)
    tt, lp = tt.to(DEV), lp.to(DEV)
    for victim in ("x", "tokens", "teacher"):
        x = scores((3, 40), torch.float32).to(DEV).requires_grad_(True)
        y, t, s = x * 1.0, tt.clone(), lp.clone()
        loss = k2.distillation_loss(y, t, s)
        {"x": y, "tokens": t, "teacher": s}[victim].data.add_(0)  # (.data: no version)
        with torch.no_grad():
            {"x": y, "tokens": t, "teacher": s}[victim].add_(0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    x = scores((3, 40), torch.float32).to(DEV).requires_grad_(True)
    got = k2.token_log_probs(x, tt[:, 0], top_k=3)
    got.top_tokens.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        got.top_log_probs.sum().backward()


@pytest.mark.parametrize("classes", [7, 300])
def test_gradients_against_differences(classes):
    """Central differences along random directions.  Along a direction v of |v_c| <= 1 every
    third derivative of log p_c is at most 8 and of the entropy at most 8 (3 + log C), so that a
    step of h leaves at most h^2 / 6 of it; and the difference of two losses of 32 bits is off by
    their errors over 2 h."""
    h = 2.0 ** -6
    x = scores((4, classes), torch.float32, sigma=1.0).to(DEV)
    token = ints(0, classes, (4,)).to(DEV)
    tt, lp = teacher((4,), classes, 5)
    tt, lp = tt.to(DEV), lp.to(DEV)

    def sums(y):
        got = k2.token_log_probs(y, token, top_k=2, entropy=True)
        return got.log_probs.sum() + got.top_log_probs.sum() + got.entropy.sum()

    def loss(y):
        return k2.distillation_loss(y, tt, lp, temperature=1.0)

    # 4 rows: a token, two top classes and an entropy; errors of 2^-20 of values up to 16 each
    for f, third in ((sums, 4 * (3 * 8 + 8 * (3 + math.log(classes)))), (loss, 4 * 8)):
        leaf = x.clone().requires_grad_(True)
        grad, = torch.autograd.grad(f(leaf), leaf)
        for seed in range(4):
            v = torch.rand(x.shape, generator=torch.Generator().manual_seed(seed)) * 2 - 1
            v = v.to(DEV)
            diff = (f(x + h * v).double() - f(x - h * v).double()) / (2 * h)
            want = (grad.double() * v.double()).sum()
            assert abs(float(diff - want)) <= h * h / 6 * third + 16 * 16 * 2 ** -20 / h


# --------------------------------------------------------------------------- around the calls
def test_the_same_bits_every_time():
    x = scores((64, 50, 500), torch.bfloat16).to(DEV)
    tt, lp = teacher((64, 50), 500, 8)
    tt, lp = tt.to(DEV), lp.to(DEV)
    first = None
    for _ in range(3):
        leaf = x.clone().requires_grad_(True)
        loss = k2.distillation_loss(leaf, tt, lp, reduction="mean")
        grad, = torch.autograd.grad(loss, leaf)
        got = k2.token_log_probs(leaf, tt[..., 0], top_k=8, entropy=True)
        g2, = torch.autograd.grad(got.entropy.sum() + got.top_log_probs.sum(), leaf)
        all_of_it = [loss.detach(), grad, got.log_probs.detach(), got.entropy.detach(), g2]
        if first is not None:
            assert all(torch.equal(a, b) for a, b in zip(first, all_of_it))
        first = all_of_it


def test_on_another_stream_and_on_two_at_once():
    x = scores((40, 700), torch.float16).to(DEV)
    tt, lp = teacher((40,), 700, 8)
    tt, lp = tt.to(DEV), lp.to(DEV)

    def step():
        leaf = x.detach().requires_grad_(True)
        loss = k2.distillation_loss(leaf, tt, lp, reduction="mean")
        got = k2.token_log_probs(leaf, tt[..., 0], top_k=8)
        return [loss.detach(), *torch.autograd.grad(loss, leaf), got.log_probs.detach(),
                got.top_tokens]

    want = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(step())
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("shape,classes", [((5, 6), 500), ((2, 3), 5000), ((2, 1), 70001)])
def test_captured_and_replayed(shape, classes):
    """A training step as a graph, with other inputs in its buffers at each replay; two graphs
    replayed in turn."""
    n = shape[0]

    def inputs(seed):
        tt, lp = teacher(shape, classes, 4, seed)
        return [scores(shape + (classes,), torch.float32, seed).to(DEV), tt.to(DEV), lp.to(DEV),
                ints(1, shape[1] + 1, (n,), seed).to(DEV)]

    def step(leaf, tt, lp, lengths):
        loss = k2.distillation_loss(leaf, tt, lp, reduction="mean", lengths=lengths)
        got = k2.token_log_probs(leaf, tt[..., 0], top_k=3, entropy=True, lengths=lengths)
        total = 0.5 * loss + got.log_probs.sum() + got.entropy.sum()
        grad, = torch.autograd.grad(total, leaf)
        return [loss.detach(), grad, got.log_probs.detach(), got.top_tokens]

    def plain(seed):
        x, *rest = inputs(seed)
        return step(x.requires_grad_(True), *rest)

    graphs = []
    for seed in (1, 2):
        held = inputs(seed)
        held[0].requires_grad_(True)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*held)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*held)
        graphs.append((graph, held, out))
    for seed in (5, 6, 7):
        for k, (graph, held, out) in enumerate(graphs):
            with torch.no_grad():
                for a, b in zip(held, inputs(seed + 10 * k)):
                    a.copy_(b)
            graph.replay()
        torch.cuda.synchronize()
        for k, (graph, held, out) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(out, plain(seed + 10 * k)))


@pytest.mark.parametrize("classes", [300, 5000])
def test_a_forward_pass_replayed_by_itself(classes):
    """Its gradients are no part of it: those of one replay stay when the next one runs."""
    tt, lp = teacher((3,), classes, 6)
    tt, lp = tt.to(DEV), lp.to(DEV)
    inputs = [scores((3, classes), torch.float32, seed).to(DEV) for seed in (1, 2)]
    x = inputs[0].clone().requires_grad_(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = k2.distillation_loss(x, tt, lp)
    got = []
    for value in inputs:
        x.data.copy_(value)  # (.data: the buffer of a captured call, no version)
        graph.replay()
        torch.cuda.synchronize()
        got += torch.autograd.grad(loss, x, retain_graph=True)
        torch.cuda.synchronize()
    for grad, value in zip(got, inputs):
        want, tol = distil_reference(value, tt, lp)
        assert_close(grad, want["grad"], tol["grad"])


@pytest.mark.parametrize("classes", [300, 5000])
def test_passes_captured_one_by_one(classes):
    """A backward pass that is replayed twice, with an upstream of 1 behind another one."""
    tt, lp = teacher((3,), classes, 6)
    tt, lp = tt.to(DEV), lp.to(DEV)
    x = scores((3, classes), torch.float32).to(DEV).requires_grad_(True)
    graphed = torch.cuda.make_graphed_callables(k2.DistillationLoss(), (x, tt, lp))
    loss = graphed(x, tt, lp)
    for up in (2.0, 1.0, 1.0):
        got, = torch.autograd.grad(loss, x, torch.tensor(up, device=DEV), retain_graph=True)
        want, tol = distil_reference(x.detach(), tt, lp, up=torch.tensor(up))
        assert_close(got, want["grad"], tol["grad"])
        got.fill_(7.0)


def test_a_captured_backward_pass_beside_a_graph_of_the_same_leaf():
    """Refused where that graph was made on the default stream; the capture goes on, and the other
    graph is what it was."""
    tt, lp = teacher((3,), 300, 6)
    tt, lp = tt.to(DEV), lp.to(DEV)
    x = scores((3, 300), torch.float32).to(DEV).requires_grad_(True)
    for call in (lambda: k2.distillation_loss(x, tt, lp),
                 lambda: k2.token_log_probs(x, tt[:, 0]).log_probs.sum()):
        other = call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            loss = call()
            with pytest.raises(RuntimeError, match="another graph of the same logits"):
                torch.autograd.grad(loss, x)
        want, = torch.autograd.grad(other, x)
        del loss, other, graph
        gc.collect()  # (what was raised refers to them)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            grad, = torch.autograd.grad(call(), x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(grad, want)


def test_refusals():
    x = torch.zeros(2, 3, 8, device=DEV)
    token = torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    tt, lp = token[..., None].expand(2, 3, 4), torch.zeros(2, 3, 4, device=DEV)
    ones = torch.ones(2, dtype=torch.int32)
    for call in (
            lambda: k2.token_log_probs(x),
            lambda: k2.token_log_probs(x.double(), token),
            lambda: k2.token_log_probs(x, token[:, :2]),
            lambda: k2.token_log_probs(x, token.float()),
            lambda: k2.token_log_probs(x, top_k=9),
            lambda: k2.token_log_probs(x, top_k=-1),
            lambda: k2.token_log_probs(torch.zeros(1, 200, device=DEV), top_k=129),
            lambda: k2.token_log_probs(x[..., :0], token),
            lambda: k2.token_log_probs(x, token, lengths=ones[:1]),
            lambda: k2.token_log_probs(x, token, lengths=ones.float()),
            lambda: k2.token_log_probs(x[0], token[0], lengths=ones),
            lambda: k2.distillation_loss(x, tt, lp[..., :2]),
            lambda: k2.distillation_loss(x, tt[..., :0], lp[..., :0]),
            lambda: k2.distillation_loss(x, tt.expand(2, 3, 4).repeat(1, 1, 33),
                                         lp.repeat(1, 1, 33)),
            lambda: k2.distillation_loss(x, tt.float(), lp),
            lambda: k2.distillation_loss(x, tt, lp.double()),
            lambda: k2.distillation_loss(x, tt, lp, temperature=0.0),
            lambda: k2.distillation_loss(x, tt, lp, temperature=-1.0),
            lambda: k2.distillation_loss(x, tt, lp, temperature=math.nan),
            lambda: k2.distillation_loss(x, tt, lp, weight=math.inf),
            lambda: k2.distillation_loss(x, tt, lp, reduction="max"),
            lambda: k2.distillation_loss(x, tt, lp.clone().requires_grad_(True)),
            lambda: k2.DistillationLoss(reduction="max")):
        with pytest.raises(AssertionError):
            call()
    for call in (lambda: k2.token_log_probs(x.cpu(), token.cpu()),
                 lambda: k2.token_log_probs(x, token.cpu()),
                 lambda: k2.distillation_loss(x, tt.cpu(), lp),
                 lambda: k2.distillation_loss(x, tt, lp.cpu())):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()
    leaf = x.clone().requires_grad_(True)
    loss = k2.distillation_loss(leaf, tt, lp)
    with pytest.raises(RuntimeError, match="second order"):
        torch.autograd.grad((loss * leaf.sum()), leaf, create_graph=True)
    loss = k2.distillation_loss(leaf, tt, lp)
    with pytest.raises(RuntimeError, match="second order"):
        loss.backward(create_graph=True)
    with pytest.raises(RuntimeError, match="second order"):
        k2.token_log_probs(leaf, token).log_probs.sum().backward(create_graph=True)


def test_a_module_with_settings():
    x = scores((2, 3, 8), torch.float32).to(DEV)
    tt, lp = teacher((2, 3), 8, 4)
    module = k2.DistillationLoss(temperature=2.0, weight=0.5, reduction="mean")
    lengths = torch.tensor([3, 1])
    got = module(x, tt.to(DEV), lp.to(DEV), lengths)
    want = k2.distillation_loss(x, tt.to(DEV), lp.to(DEV), 2.0, 0.5, "mean", lengths)
    assert torch.equal(got, want)


def test_a_student_learns_from_a_teacher_beside_its_ctc_loss():
    """The operators as they are used together: a teacher writes its top classes, the student is
    trained on the CTC loss and on the teacher, and its alignment is scored."""
    n, t, c = 3, 40, 60
    lengths = torch.tensor([40, 31, 25], dtype=torch.int32)
    teacher_logits = scores((n, t, c), torch.float32, 1, peak=6.0).to(DEV)
    student = scores((n, t, c), torch.float32, 2).to(DEV).requires_grad_(True)
    symbols = [[5, 9, 9, 3], [7, 1], [2, 4, 6, 8, 10]]
    top = k2.token_log_probs(teacher_logits, top_k=8, lengths=lengths)
    segments = torch.tensor([[i, 0, int(lengths[i])] for i in range(n)], dtype=torch.int32)

    def ctc(x):
        graph = k2.ctc_graph(symbols, device=DEV)
        return k2.ctc_loss(graph, k2.DenseFsaVec.from_logits(x, segments[
            torch.argsort(lengths, descending=True)]), output_beam=10.0)

    kd = k2.distillation_loss(student, top.top_tokens, top.top_log_probs, temperature=2.0,
                              weight=0.3, lengths=lengths)
    total = ctc(student) + kd
    total.backward()
    other = student.detach().clone().requires_grad_(True)
    ctc(other).backward()
    live = torch.arange(t)[None] < lengths[:, None]
    want, tol = distil_reference(student.detach(), top.top_tokens, top.top_log_probs, 2.0, 0.3,
                                 "sum", live)
    # the two gradients are added in 32 bits
    sum_tol = 2.0 ** -24 * (other.grad.abs().double().cpu() + want["grad"].abs())
    assert_close(student.grad, want["grad"] + other.grad.double().cpu(), tol["grad"] + sum_tol)
    assert_close(kd, want["loss"], tol["loss"])
    # frames of the best path, scored along the path
    graph = k2.ctc_graph(symbols, device=DEV)
    dense = k2.DenseFsaVec.from_logits(student.detach(), segments)
    lattice = k2.intersect_dense(graph, dense, 1e4)
    best = k2.shortest_path(lattice, use_double_scores=True)
    splits = best.arcs.h_arc_splits
    frames = torch.full((n, t), -1, dtype=torch.int32)
    for i in range(n):
        labels = best.labels[int(splits[i]):int(splits[i + 1]) - 1].cpu()
        assert len(labels) == int(lengths[i])
        frames[i, :len(labels)] = labels
    got = k2.token_log_probs(student.detach(), frames.to(DEV), entropy=True, lengths=lengths)
    path = best.get_tot_scores(log_semiring=False, use_double_scores=True)
    # a path's score adds up to 40 arcs of 32-bit log-probs
    assert_close(got.log_probs.double().sum(1).float(), path.double().cpu(),
                 torch.full((n,), 40 * 2.0 ** -18).double())
