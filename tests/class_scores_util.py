"""Token scores and distillation from their definitions in 64 bits, with bounds of what 32-bit
arithmetic may be off by."""
import math

import torch

E32 = 2.0 ** -24  # half a step of float32, relative


def sum_error(c):
    """Relative error of a sum of `c` terms 2^d >= 0: additions one after the other within 1/32
    of the terms, then a tree; 2^d itself (2 units of the last place) and d (a subtraction, a
    product and a factor of two roundings, on terms that matter, |d| <= 32: 2^-24 * 4 * 32 *
    ln 2)."""
    return (c / 32 + 16) * E32 + 2 ** -22 + 90 * E32


def log_softmax(x):
    """In 64 bits; a row of nothing but -inf has log-probs -inf."""
    none = (x == -math.inf).all(-1, keepdim=True)
    return torch.where(none, torch.full_like(x, -math.inf), torch.log_softmax(x, -1))


def top_order(x, k):
    """The k largest per row: NaN first, then by value (-0 = +0), then the lower class."""
    key = torch.where(torch.isnan(x), torch.full_like(x, math.inf), x + 0.0)
    # (NaN above +inf: a stable sort by two keys, the less important one first)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    nan = torch.isnan(x).gather(-1, order).to(torch.int8)
    return order.gather(-1, torch.sort(nan, dim=-1, descending=True,
                                       stable=True).indices)[..., :k]


def tokens_reference(x, token=None, top_k=0, live=None, up=None):
    """Everything of `token_log_probs`, and its gradient for the upstreams `up` (a dict), in 64
    bits; `tol`: what each may be off by."""
    x = x.double().cpu()
    c = x.shape[-1]
    live = torch.ones(x.shape[:-1], dtype=torch.bool) if live is None else live.cpu()
    x = torch.where(live[..., None], x, 0)  # nobody looks at the others
    up = up or {}
    log_p = log_softmax(x)
    p = log_p.exp()
    rel = sum_error(c)
    # log p = (x - high) - log sum: two roundings, and log sum <= log c
    lp_tol = rel + 3 * E32 * (log_p.abs().nan_to_num(0, posinf=0, neginf=0) + math.log(c) + 1)
    h = torch.special.entr(p).sum(-1)
    # sum e d: errors of e, d and the additions, relative to sum p |d| <= h + log c
    h_tol = 2 * rel * (1 + h + math.log(c)) + 4 * E32 * (1 + math.log(c))
    out, tol, grad = {}, {}, torch.zeros_like(x)
    grad_tol = torch.zeros_like(x)
    # p: |d| beyond 32 belongs to a p below 2^-32
    p_rel = 2 * rel
    if token is not None:
        token = token.cpu().long()
        valid = (token >= 0) & (token < c)
        at = torch.where(valid, token, 0)[..., None]
        lp = torch.where(valid, log_p.gather(-1, at)[..., 0], torch.zeros(()).double())
        lp = torch.where(valid | (token == -1), lp, math.nan)
        out["log_probs"] = torch.where(live, lp, 0)
        tol["log_probs"] = lp_tol.gather(-1, at)[..., 0]
        if "log_probs" in up:
            g = torch.where(live & (token != -1), up["log_probs"].double().cpu(), 0.0)
            g = torch.where(live & ~(valid | (token == -1)), math.nan, g)[..., None]
            grad -= torch.where(p > 0, g * p, torch.where(torch.isnan(g), math.nan, 0.0))
            grad.scatter_add_(-1, at, torch.where(valid[..., None], g, 0.0))
            grad_tol += g.abs() * p * p_rel
            grad_tol.scatter_add_(-1, at, g.abs() * 4 * E32)
    out["entropy"] = torch.where(live, h, 0)
    tol["entropy"] = h_tol
    if "entropy" in up:
        g = torch.where(live, up["entropy"].double().cpu(), 0.0)[..., None]
        inner = torch.where(p > 0, log_p + h[..., None], 0.0)
        grad -= g * p * inner
        grad_tol += g.abs() * p * (p_rel * inner.abs() + lp_tol + h_tol[..., None])
    if top_k:
        at = top_order(x, top_k)
        out["top_tokens"] = torch.where(live[..., None], at, -1).to(torch.int32)
        out["top_log_probs"] = torch.where(live[..., None], log_p.gather(-1, at), 0)
        tol["top_log_probs"] = lp_tol.gather(-1, at)
        if "top_log_probs" in up:
            g = torch.where(live[..., None], up["top_log_probs"].double().cpu(), 0.0)
            grad -= torch.where(p > 0, g.sum(-1, keepdim=True) * p, 0.0)
            grad.scatter_add_(-1, at, g)
            size = g.abs().sum(-1, keepdim=True)
            grad_tol += size * p * (p_rel + top_k * E32)
            grad_tol.scatter_add_(-1, at, g.abs() * 4 * E32)
    out["grad"], tol["grad"] = grad, grad_tol
    return out, tol


def distil_reference(x, tokens, scores, temperature=1.0, weight=1.0, reduction="sum",
                     live=None, up=None):
    """The loss and its gradient for the upstream `up` (1 where None), and `tol` of both."""
    x, scores = x.double().cpu() / temperature, scores.double().cpu()
    tokens = tokens.cpu().long()
    c, k = x.shape[-1], tokens.shape[-1]
    live = torch.ones(x.shape[:-1], dtype=torch.bool) if live is None else live.cpu()
    x, tokens, scores = (torch.where(live[..., None], v, 0) for v in (x, tokens, scores))
    there = (tokens >= 0) & (tokens < c)
    t = torch.where(there, scores / temperature, -math.inf)
    some = (t > -math.inf).any(-1, keepdim=True) | torch.isnan(t).any(-1, keepdim=True)
    q = torch.where(some, torch.softmax(t, -1), 0.0)
    log_q = torch.where(some, torch.log_softmax(t, -1), 0.0)
    log_p = log_softmax(x)
    at = torch.where(there, tokens, 0)
    lp = log_p.gather(-1, at)
    term = torch.where(q == 0, 0.0, q * (log_q - lp))
    row = temperature ** 2 * term.sum(-1)
    wrong = ((tokens < -1) | (tokens >= c)).any(-1)
    row = torch.where(wrong, math.nan, row)
    rel, rel_q = sum_error(c), sum_error(32 * k)
    # of each term: the share's error, those of both logarithms
    size = (log_q.nan_to_num(0, neginf=0).abs() + lp.nan_to_num(0, neginf=0).abs()
            + math.log(c) + 1)
    row_tol = temperature ** 2 * (q.nan_to_num(0) * ((2 * rel_q + (k + 8) * E32) * size
                                                    + rel + rel_q)).sum(-1)
    row, row_tol = torch.where(live, row, 0), torch.where(live, row_tol, 0)
    count = max(1, int(live.sum())) if reduction == "mean" else 1
    up = torch.ones(()).double() if up is None else up.double().cpu()
    up_rows = torch.broadcast_to(up, row.shape) if up.dim() == 0 else up
    p = log_p.exp()
    hit = torch.zeros_like(x).scatter_add_(-1, at, torch.where(there, q, 0.0))
    grad = torch.where(some, p - hit, 0.0)
    grad = torch.where(wrong[..., None], math.nan, grad)
    by = temperature * weight / count * up_rows[..., None]
    hits = torch.zeros_like(x).scatter_add_(-1, at, there.double() * q.nan_to_num(0))
    grad_tol = by.abs() * (p * 2 * rel + hits * (2 * rel_q + k * E32) + 4 * E32 * (p + hits))
    grad = torch.where(live[..., None], grad * by, 0.0)
    out, tol = {"grad": grad}, {"grad": grad_tol}
    if reduction == "none":
        out["loss"], tol["loss"] = row * weight, row_tol * abs(weight) + 2 * E32 * row.abs()
    else:
        out["loss"] = row.sum() * weight / count
        tol["loss"] = ((row_tol + 2 * E32 * row.abs()).sum() * abs(weight) / count
                       + 2 * E32 * out["loss"].abs())
    return out, tol


def assert_close(got, want, tol, what=""):
    """got (of its own type) against want and tol in 64 bits; NaN and infinities where they are
    in want; the rounding to got's type (half a step, with subnormals) comes on top of tol."""
    assert tuple(got.shape) == tuple(want.shape), (what, got.shape, want.shape)
    finfo = torch.finfo(got.dtype)
    g = got.detach().double().cpu()
    odd = ~torch.isfinite(want)
    same = (g == want) | (torch.isnan(g) & torch.isnan(want))
    assert same[odd].all(), (what, "not finite", g[odd][~same[odd]][:5], want[odd][~same[odd]][:5])
    step = finfo.eps / 2 * want.abs() + finfo.smallest_normal * finfo.eps
    # (values below 2^-126 are 0 in the kernels)
    off = (g - want).abs() - (tol * (1 + finfo.eps) + step + 1e-36)
    off = torch.where(odd, torch.full_like(off, -1.0), off)
    assert not torch.isnan(off).any(), (what, "NaN", g[torch.isnan(off)][:5])
    assert (off <= 0).all(), (what, float(off.max()), int(off.argmax()),
                              g.reshape(-1)[off.argmax()], want.reshape(-1)[off.argmax()])
