"""Scores of given classes and distillation, on the class scores of a network: the rows that
`DenseFsaVec.from_logits` normalises and `ctc_loss` trains on.

`token_log_probs` says what a network thinks of given labels (an alignment's, a hypothesis's),
how sure it is, and which classes it would have taken; `distillation_loss` trains a network on
the classes that another one would have taken.  The reference has neither."""
from typing import NamedTuple, Optional

import torch
import torch.nn as nn

from ._lib import _host


class TokenLogProbs(NamedTuple):
    """What `token_log_probs` gives; None for what was not asked for."""
    log_probs: Optional[torch.Tensor]  # [...] float32
    entropy: Optional[torch.Tensor]  # [...] float32, in nats
    top_log_probs: Optional[torch.Tensor]  # [..., top_k] float32, largest first
    top_tokens: Optional[torch.Tensor]  # [..., top_k] int32


def token_log_probs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, top_k: int = 0,
                    entropy: bool = False,
                    lengths: Optional[torch.Tensor] = None) -> TokenLogProbs:
    """Log-probs of given classes under softmax(logits), with the entropy of every row and its
    top classes.  Log-probs, entropy and top log-probs are differentiable in the logits (once).

    Args:
      logits: [..., C] on a GPU, float32, float16 or bfloat16; any strides (rows of adjacent
        classes at one or two strides are read in place, others are copied).  Log-probs will
        do as well: they are their own logits.
      tokens: [...] int32 or int64, the class asked about in each row; -1 for none, whose
        log-prob is 0 and has no gradient.  Any other number that is no class gives NaN, in the
        log-prob and, where that has an upstream gradient, in the row's gradient.
      top_k: so many of the largest log-probs, and their classes (0 to 128); among equal logits
        the lowest class comes first.  A short row's time grows steeply above 32 (64000 rows of
        500 classes: 57 us for 8, 122 for 32, 629 for 64, 858 for 128).
      entropy: whether -sum_c p_c log p_c is wanted.
      lengths: [N] int32 or int64, on the CPU or the device, for logits [N, T, C]: frames from
        `lengths[n]` on are not read; they get 0 everywhere, -1 as top classes, and no
        gradient.  Those on the CPU are read at the call: a captured call keeps them.

    A logit of -inf is a class of probability 0; in a row without any other every log-prob is
    -inf and the entropy 0.  A row with NaN or +inf is NaN (NaN comes first among the top
    classes)."""
    return TokenLogProbs(*_host.token_log_probs(logits, tokens, top_k, entropy, lengths))


def distillation_loss(logits: torch.Tensor, teacher_tokens: torch.Tensor,
                      teacher_log_probs: torch.Tensor, temperature: float = 1.0,
                      weight: float = 1.0, reduction: str = "sum",
                      lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The divergence of softmax(logits / temperature) from a teacher's distribution over its top
    classes.  Per row

        weight * temperature^2 * sum_j q_j (log q_j - log p[teacher_tokens[j]])

    with q = softmax(teacher_log_probs / temperature) over the entries of the row and p over
    all classes.

    Args:
      logits: [..., C], as in `token_log_probs`.
      teacher_tokens: [..., K] int32 or int64, 1 <= K <= 128: the teacher's classes, e.g.
        `top_tokens` of `token_log_probs`; -1 for an entry that is not there.  A class that
        comes twice counts twice; any other number that is no class makes its row NaN.
      teacher_log_probs: [..., K] float32, float16 or bfloat16: their log-probs or logits (what
        is common to a row's entries does not matter).  No gradient goes there.
      reduction: "sum", "mean" over the frames within the lengths (over all rows without any;
        0 where there are none), or "none": [...].
      lengths: as in `token_log_probs`; frames beyond them give no loss and no gradient.

    A row without an entry, or with none above -inf, gives 0 and no gradient; one with NaN or +inf
    among its entries is NaN.

    With "sum" and "mean" the gradient is made beside the loss, while a row is at hand, for an
    upstream of 1, and made again from the logits where the upstream is another: a factor of the
    loss is cheaper as `weight` than as a product.  It takes as much memory as the logits until the
    backward pass; under `torch.autograd.graph.saved_tensors_hooks` (offloading, checkpoints) it
    is made there."""
    return _host.distillation_loss(logits, teacher_tokens, teacher_log_probs, temperature, weight,
                                   reduction, lengths)


class DistillationLoss(nn.Module):
    """`distillation_loss` with its settings, beside `CtcLoss`."""

    def __init__(self, temperature: float = 1.0, weight: float = 1.0,
                 reduction: str = "sum") -> None:
        super().__init__()
        assert reduction in ("none", "mean", "sum")
        self.temperature = temperature
        self.weight = weight
        self.reduction = reduction

    def forward(self, logits: torch.Tensor, teacher_tokens: torch.Tensor,
                teacher_log_probs: torch.Tensor,
                lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
        return distillation_loss(logits, teacher_tokens, teacher_log_probs, self.temperature,
                                 self.weight, self.reduction, lengths)
