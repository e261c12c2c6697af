"""Scores of given tokens and distillation from a teacher's top classes, as cases that can be
timed and compared.

Two operators on the class scores that a network gives for N sequences of T frames:

  tokens   `k2.token_log_probs`: log-probs of one given class per frame, the entropy of the
           frame's distribution and its top classes, forward or forward and backward
  distil   `k2.distillation_loss`: the divergence of the scores from a teacher's distribution
           over its own top classes, forward or forward and backward

`run` computes them in a plain form out of elementary torch operations, or, where `own` is
set, through the framework.  `exact` computes them from their definitions in 64 bits."""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _tokens(name=None, **kw):
    """classes: columns of the scores; short: the shortest sequence as a share of the longest
    (1: no lengths are given); tokens, entropy, top_k: what is asked for; backward: gradients
    of all of it; sigma, peak: spread of the scores and what is added at a reference
    alignment (0: an untrained network, 9: a trained one); time_first: the scores are a
    transposed view of a [T, N, C] tensor."""
    case = dict(name=name, kind="tokens", sequences=8, frames=200, classes=500, dtype="fp32",
                short=1.0, tokens=True, entropy=True, top_k=0, backward=False, sigma=1.5,
                peak=6.0, time_first=False)
    return dict(case, **kw)


def _distil(name=None, **kw):
    """entries: classes that the teacher gives per frame; missing: share of the entries that
    are absent (class -1)."""
    case = dict(name=name, kind="distil", sequences=8, frames=200, classes=500, dtype="fp32",
                short=1.0, entries=8, missing=0.0, temperature=1.0, weight=1.0,
                reduction="sum", backward=True, sigma=1.5, peak=6.0, time_first=False)
    return dict(case, **kw)


def listed():
    return [
        # confidences of a chunk of four live streams, beside their decoder
        _tokens("tokens_stream", sequences=4, frames=16, top_k=4),
        # a whole batch of the headline configuration scored along its alignment
        _tokens("tokens_batch", sequences=64, frames=1000, short=0.6, dtype="bf16", top_k=8),
        # a teacher with a large vocabulary writes its top classes for later distillation
        _tokens("tokens_teacher", sequences=32, frames=500, classes=5000, dtype="fp16",
                tokens=False, entropy=False, top_k=32),
        # characters: few classes, an odd number of them, trained on scores and entropy
        _tokens("tokens_chars", sequences=16, frames=1500, classes=29, top_k=3, backward=True),
        # a training step on token scores with an entropy bonus, words as classes
        _tokens("tokens_words", sequences=4, frames=1024, classes=32001, dtype="bf16",
                backward=True, peak=9.0),
        # the next token of three hypotheses out of a large vocabulary
        _tokens("tokens_next", sequences=3, frames=1, classes=131072, top_k=64, peak=9.0),
        # distillation on the small benchmark configuration
        _distil("distil_small"),
        # one utterance scored against a teacher, without gradient
        _distil("distil_eval", sequences=1, frames=80, classes=501, entries=10, reduction="none",
                backward=False),
        # a full batch of long, ragged utterances
        _distil("distil_batch", sequences=64, frames=1000, short=0.6, dtype="bf16", entries=16,
                temperature=2.0, weight=0.5, reduction="mean"),
        # a large vocabulary, teachers of unlike numbers of classes, scores with time first
        _distil("distil_pieces", sequences=32, frames=500, classes=5000, dtype="fp16",
                entries=32, missing=0.3, short=0.5, time_first=True),
        # words as classes
        _distil("distil_words", sequences=4, frames=1024, classes=50021, dtype="bf16",
                entries=64, temperature=2.0, reduction="mean"),
        # a few frames of a very large vocabulary
        _distil("distil_few", sequences=16, frames=1, classes=131072, entries=100,
                temperature=4.0),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    classes = _spread(rng, 20, 131072)
    rows = _spread(rng, 1, max(1, min(64000, 200_000_000 // classes)))
    sequences = min(_spread(rng, 1, 64), rows)
    shape = dict(sequences=sequences, frames=max(1, rows // sequences), classes=classes,
                 dtype=rng.choice(sorted(DTYPES)), short=rng.choice([1.0, 0.7, 0.4]),
                 sigma=rng.choice([1.0, 1.5, 3.0]), peak=rng.choice([0.0, 6.0, 9.0]),
                 time_first=rng.random() < 0.25)
    if shape["dtype"] == "fp32":
        shape["frames"] = max(1, shape["frames"] // 2)
    if rng.random() < 0.5:
        backward = rng.random() < 0.5
        case = _tokens(top_k=rng.choice([0, _spread(rng, 1, min(128, classes))]), tokens=True,
                       entropy=rng.random() < 0.7, backward=backward, **shape)
    else:
        case = _distil(entries=_spread(rng, 1, min(128, classes)),
                       missing=rng.choice([0.0, 0.0, 0.3]),
                       temperature=rng.choice([1.0, 2.0, 3.5]), weight=rng.choice([1.0, 0.3]),
                       reduction=rng.choice(["sum", "mean", "none"]),
                       backward=rng.random() < 0.8, **shape)
        if case["dtype"] == "fp16" and case["reduction"] == "mean":
            case["reduction"] = "sum"  # a mean's gradient is too small for fp16
    del case["name"]
    return case


def prepare(case, seed):
    n, t, c = case["sequences"], case["frames"], case["classes"]
    device = torch.device("cuda:0")
    g = torch.Generator(device=device).manual_seed(int(seed))

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device=device)

    reference = torch.randint(0, c, (n, t), generator=g, device=device)
    first, second = (t, n) if case["time_first"] else (n, t)
    x = torch.randn(first, second, c, generator=g, device=device)
    x.mul_(case["sigma"])
    x = x.transpose(0, 1) if case["time_first"] else x
    x.scatter_add_(2, reference[..., None],
                   torch.full((n, t, 1), float(case["peak"]), device=device))
    state = {"case": case, "lengths": None}
    if case["short"] < 1:
        low = max(1, int(t * case["short"]))
        state["lengths"] = torch.randint(low, t + 1, (n,), generator=g, device=device,
                                         dtype=torch.int32)
    if case["kind"] == "tokens":
        # the alignment is right nine times out of ten, and silent frames have no token
        other = torch.randint(0, c, (n, t), generator=g, device=device)
        chance = uniform(n, t)
        token = torch.where(chance < 0.9, reference, other)
        token = torch.where(chance > 0.95, torch.full_like(token, -1), token)
        state["tokens"] = token.to(torch.int32) if case["tokens"] else None
        if case["backward"]:
            state["upstream"] = {
                "log_probs": torch.randn(n, t, generator=g, device=device),
                "entropy": 0.01 * torch.randn(n, t, generator=g, device=device),
                "top_log_probs": torch.randn(n, t, case["top_k"], generator=g, device=device)}
    else:
        # a teacher of the same kind: what the student scores, and its own view
        teacher = torch.randn(n, t, c, generator=g, device=device).add_(x)
        top, where = teacher.topk(case["entries"], dim=2)
        state["teacher_log_probs"] = top - torch.logsumexp(teacher, 2, keepdim=True)
        absent = uniform(n, t, case["entries"]) < case["missing"]
        state["teacher_tokens"] = torch.where(absent, torch.full_like(where, -1),
                                              where).to(torch.int32)
        del teacher
    x = x.to(DTYPES[case["dtype"]])  # keeps the strides
    state["logits"] = x.requires_grad_(True) if case["backward"] else x
    return state


# --------------------------------------------------------------------------- plain forms
def _inside(s):
    """[N, T] truth values: frames within the lengths."""
    n, t = s["logits"].shape[:2]
    if s["lengths"] is None:
        return torch.ones(n, t, dtype=torch.bool, device=s["logits"].device)
    return torch.arange(t, device=s["logits"].device)[None] < s["lengths"][:, None]


def _plain_top(x, k):
    """The k largest of every row, the lowest class first among equals."""
    c = x.shape[-1]
    bits = (x + 0.0).view(torch.int32)
    ordered = bits ^ ((bits >> 31) & 0x7FFFFFFF)
    rest = torch.arange(c - 1, -1, -1, device=x.device)
    key = (ordered.to(torch.int64) << 32) + rest
    return c - 1 - (torch.topk(key, k, dim=-1).values & 0xFFFFFFFF)


def _plain_tokens(s):
    case, inside = s["case"], _inside(s)
    x = s["logits"].detach().to(torch.float32)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    log_p = x - top - torch.log(total)
    p = e / total
    out = {}
    zero = torch.zeros((), device=x.device)
    grad = torch.zeros_like(x) if case["backward"] else None
    if case["tokens"]:
        there = inside & (s["tokens"] >= 0)
        at = s["tokens"].clamp(min=0).long()[..., None]
        out["log_probs"] = torch.where(there, log_p.gather(2, at)[..., 0], zero)
        if case["backward"]:
            g = torch.where(there, s["upstream"]["log_probs"], zero)[..., None]
            grad -= g * p
            grad.scatter_add_(2, at, g)
    if case["entropy"]:
        h = -(p * log_p).sum(-1)
        out["entropy"] = torch.where(inside, h, zero)
        if case["backward"]:
            g = torch.where(inside, s["upstream"]["entropy"], zero)[..., None]
            grad -= g * p * (log_p + h[..., None])
    if case["top_k"]:
        at = _plain_top(x, case["top_k"])
        out["top_log_probs"] = torch.where(inside[..., None], log_p.gather(2, at), zero)
        out["top_tokens"] = torch.where(inside[..., None], at, torch.full_like(at, -1)).to(
            torch.int32)
        if case["backward"]:
            g = torch.where(inside[..., None], s["upstream"]["top_log_probs"], zero)
            grad -= g.sum(-1, keepdim=True) * p
            grad.scatter_add_(2, at, g)
    if case["backward"]:
        out["grad"] = grad.to(s["logits"].dtype)
    return out


def _plain_distil(s):
    case, inside = s["case"], _inside(s)
    temperature, weight = case["temperature"], case["weight"]
    x = s["logits"].detach().to(torch.float32) / temperature
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    there = (s["teacher_tokens"] >= 0) & inside[..., None]
    teacher = torch.where(there, s["teacher_log_probs"] / temperature, -math.inf)
    some = there.any(-1, keepdim=True)
    highest = torch.where(some, teacher.amax(-1, keepdim=True), 0.0)
    mass = torch.exp(teacher - highest)
    norm = torch.where(some, mass.sum(-1, keepdim=True), 1.0)
    q = mass / norm
    at = s["teacher_tokens"].clamp(min=0).long()
    log_q = teacher - highest - torch.log(norm)
    term = q * (log_q - (x.gather(2, at) - top - torch.log(total)))
    rows = temperature**2 * torch.where(there, term, 0.0).sum(-1, dtype=torch.float64)
    scale = torch.full((), weight, dtype=torch.float64, device=x.device)
    if case["reduction"] == "mean":
        scale = weight / inside.sum().clamp(min=1).to(torch.float64)
    loss = rows * scale
    if case["reduction"] != "none":
        loss = loss.sum()
    out = {"loss": loss.to(torch.float32)}
    if case["backward"]:
        grad = torch.where(some, e / total, 0.0).scatter_add_(2, at, -q)
        out["grad"] = (grad * (temperature * scale).to(torch.float32)).to(s["logits"].dtype)
    return out


# --------------------------------------------------------------------------- the framework
def _own_tokens(s):
    import k2_b200 as k2
    case = s["case"]
    got = k2.token_log_probs(s["logits"], s["tokens"], top_k=case["top_k"],
                             entropy=case["entropy"], lengths=s["lengths"])
    out = {k: v for k, v in got._asdict().items() if v is not None}
    if case["backward"]:
        names = [k for k in out if k in s["upstream"]]
        out["grad"], = torch.autograd.grad([out[k] for k in names], s["logits"],
                                           [s["upstream"][k] for k in names])
    return {k: v.detach() for k, v in out.items()}


def _own_distil(s):
    import k2_b200 as k2
    case = s["case"]
    loss = k2.distillation_loss(s["logits"], s["teacher_tokens"], s["teacher_log_probs"],
                                temperature=case["temperature"], weight=case["weight"],
                                reduction=case["reduction"], lengths=s["lengths"])
    out = {"loss": loss.detach()}
    if case["backward"]:
        upstream = torch.ones_like(loss) if case["reduction"] == "none" else None
        out["grad"], = torch.autograd.grad(loss, s["logits"], upstream)
    return out


def run(state):
    if own:
        return (_own_tokens if state["case"]["kind"] == "tokens" else _own_distil)(state)
    return (_plain_tokens if state["case"]["kind"] == "tokens" else _plain_distil)(state)


def work(case):
    rows = case["sequences"] * case["frames"]
    # frames within the lengths, which are even between the shortest and the longest
    inside = rows * (1 + case["short"]) / 2 if case["short"] < 1 else rows
    size = 4 if case["dtype"] == "fp32" else 2
    scores = inside * case["classes"] * size
    grad = rows * case["classes"] * size if case["backward"] else 0
    if case["kind"] == "tokens":
        small = rows * (8 * case["tokens"] + 4 * case["entropy"] + 8 * case["top_k"])
        if case["backward"]:
            small += rows * 4 * (case["tokens"] + case["entropy"] + case["top_k"])
        flops = 4 + 2 * case["entropy"] + 4 * case["backward"]
    else:
        small = inside * 8 * case["entries"] + (4 * rows if case["reduction"] == "none" else 4)
        flops = 4 + 2 * case["backward"]
    return {"bytes": scores + grad + small, "flops": flops * inside * case["classes"]}


# --------------------------------------------------------------------------- 64 bits
def _exact_tokens_rows(case, x, token, up):
    """Rows of one chunk: the definitions over [R, C] in 64 bits."""
    log_p = torch.log_softmax(x, 1)
    p = torch.exp(log_p)
    out, grad, eye = {}, torch.zeros_like(x), torch.arange(x.shape[0], device=x.device)
    if case["tokens"]:
        some = token >= 0
        column = torch.where(some, token, 0).long()
        out["log_probs"] = log_p[eye, column] * some
        if case["backward"]:
            g = up["log_probs"].double() * some
            grad.addcmul_(p, g[:, None], value=-1)
            grad[eye, column] += g
    if case["entropy"]:
        out["entropy"] = torch.special.entr(p).sum(1)
        if case["backward"]:
            slope = -log_p - out["entropy"][:, None]
            grad += p * slope * up["entropy"].double()[:, None]
    if case["top_k"]:
        order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["top_k"]]
        out["top_log_probs"], out["top_tokens"] = torch.take_along_dim(log_p, order, 1), order
        if case["backward"]:
            g = up["top_log_probs"].double()
            grad.scatter_add_(1, order, g).addcmul_(p, g.sum(1, keepdim=True), value=-1)
    if case["backward"]:
        out["grad"] = grad
    return out


def _exact_distil_rows(case, x, tokens, scores):
    tau = case["temperature"]
    some = tokens >= 0
    target = torch.zeros_like(x)
    share = torch.where(some, scores.double() / tau, -math.inf).softmax(1).nan_to_num(0.0)
    target.scatter_add_(1, torch.where(some, tokens, 0).long(), share)
    log_p = torch.log_softmax(x / tau, 1)
    loss = tau * tau * (torch.xlogy(share, share).sum(1) - (target * log_p).sum(1))
    out = {"loss": loss}
    if case["backward"]:
        out["grad"] = tau * (log_p.exp() * target.sum(1, keepdim=True) - target)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    logits = s["logits"].detach()
    n, t, c = logits.shape
    rows = n * t
    lengths = s["lengths"] if s["lengths"] is not None else torch.full((n,), t, device="cuda:0")
    parts = {}
    chunk = max(1, 30_000_000 // c)
    flat = lambda v: None if v is None else v.reshape(rows, *v.shape[2:])  # noqa: E731
    x = flat(logits)
    ups = {k: flat(v) for k, v in s.get("upstream", {}).items()}
    counted = lengths.clamp(0, t).sum().clamp(min=1).double()
    for first in range(0, rows, chunk):
        part = slice(first, min(rows, first + chunk))
        row = torch.arange(part.start, part.stop, device=x.device)
        live = row % t < lengths[row // t]
        if case["kind"] == "tokens":
            token = flat(s["tokens"])[part] if case["tokens"] else None
            got = _exact_tokens_rows(case, x[part].double(), token,
                                     {k: v[part] for k, v in ups.items()})
        else:
            got = _exact_distil_rows(case, x[part].double(), flat(s["teacher_tokens"])[part],
                                     flat(s["teacher_log_probs"])[part])
            scale = case["weight"] / (counted if case["reduction"] == "mean" else 1.0)
            got = {k: v * scale for k, v in got.items()}
        for k, v in got.items():
            dead = ~live.reshape(-1, *[1] * (v.dim() - 1))
            parts.setdefault(k, []).append(v.masked_fill(dead, -1 if k == "top_tokens" else 0))
    out = {k: torch.cat(v).reshape(n, t, *v[0].shape[1:]) for k, v in parts.items()}
    if "top_tokens" in out:
        out["top_tokens"] = out["top_tokens"].to(torch.int32)
    if case["kind"] == "distil" and case["reduction"] != "none":
        out["loss"] = out["loss"].sum()
    return out
