"""The operators on a vocabulary's logits restated in float64 on the CPU: log
probabilities of given tokens with entropy and the largest, and the
distillation loss against a teacher's top logits.

TEST INFRASTRUCTURE ONLY (see oracle/__init__.py).

Written from the definitions, in torch operations that autograd differentiates,
so that a parity test takes the gradients from here.
"""

from __future__ import annotations

from typing import Optional

import torch


def log_probs(logits: torch.Tensor, temperature: float = 1.0) -> torch.Tensor:
    """log softmax(logits / T); NaN in a row with a NaN or +inf, or of -inf."""
    return torch.log_softmax(logits.double() / temperature, -1)


def moments(logp: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(entropy, sum p ln^2 p); nothing from p = 0."""
    p = logp.exp()
    lp = torch.where(p > 0, logp, 0.0)
    return -(p * lp).sum(-1), (p * lp * lp).sum(-1)


def logsumexp(logits: torch.Tensor, temperature: float = 1.0) -> torch.Tensor:
    """Moved by the row's largest, whose own gradient cancels: at the types'
    lowest values 64 bits hold no log V beside it, and p = exp(z - lse) would be 1
    in every column of a row of them."""
    z = logits.double() / temperature
    most = z.detach().amax(-1, keepdim=True)
    most = torch.where(most == -torch.inf, 0.0, most)
    return most.squeeze(-1) + torch.logsumexp(z - most, -1)


def largest(logits: torch.Tensor, k: int) -> torch.Tensor:
    """The ids of the k largest of each row, one after the other: the first of
    the largest that is left (NaN as -inf)."""
    left = torch.where(logits.isnan(), -torch.inf, logits.double())
    taken = torch.zeros_like(left, dtype=torch.bool)
    out = []
    for _ in range(k):
        most = torch.where(taken, -torch.inf, left).amax(-1, keepdim=True)
        first = ((left == most) & ~taken).to(torch.uint8).argmax(-1, keepdim=True)
        taken.scatter_(-1, first, True)
        out.append(first)
    return torch.cat(out, -1)


def teacher_probs(teacher_ids, teacher_logits, temperature: float, teacher_lse: Optional[torch.Tensor] = None):
    """(q, log q) of the entries: ids below 0 have q = 0 and log q = -inf, and so
    has every entry of a row without a finite logit."""
    t = (teacher_logits.double() / temperature).masked_fill(teacher_ids < 0, -torch.inf)
    if teacher_lse is None:
        most = t.amax(-1, keepdim=True)  # first, as in logsumexp above
        t = t - torch.where(most == -torch.inf, 0.0, most)
        lse = torch.logsumexp(t, -1, keepdim=True)
        lse = torch.where(lse == -torch.inf, 0.0, lse)
    else:
        lse = teacher_lse.double().unsqueeze(-1)
    return (t - lse).exp(), t - lse


def distillation(logp, teacher_ids, q, log_q, temperature: float) -> torch.Tensor:
    """T^2 sum q (log q - log p[id]), nothing from q = 0."""
    lp = logp.gather(-1, teacher_ids.long().clamp(min=0))
    return temperature**2 * torch.where(q == 0, 0.0, q * (log_q - lp)).sum(-1)
