"""Operators on a vocabulary's logits, on the HIP kernels of libdsa.so
(include/dsa_vocab.h): what a masked language model learns from and answers
with.

  fused_token_logprobs      log probabilities of given tokens, the entropy, the
                            logsumexp and the top alternatives of each row, and
                            their gradient
  fused_distillation_loss   the divergence from a teacher's top logits, and its
                            gradient
  FusedMLMHead              dense, GELU, LayerNorm and the vocabulary's matrix
                            product, then these two: the generator's loss, a
                            student's loss, the best tokens for a mask

One pass over the logits forward and one backward; they are float32 or bfloat16
of any width, row stride and element alignment, arithmetic and results are
float32, and equal calls give equal bits (the order of a row's sums goes by the
shape and type, by whether top alternatives are asked for and by where the row
begins between two 128-byte borders: any of these may change the last bits).  With
z = logits / temperature and lse = log(sum(exp(z))), a logit of -inf has
probability 0 and adds nothing; a row with a NaN or +inf, or without a finite
logit, has NaN results (lse -inf where all are -inf).

In plain eager mode the functions go through the package's extension
(csrc/vocab_ext.h); CPU tensors run the same in torch operations (float64 ones
in float64).  The ops under the functions (``deberta_amd::token_logprobs``,
``distill_loss`` and the backwards) take device tensors only; like the package's
other ops they have fake implementations and autograd, are not twice
differentiable, and refuse a stream that is capturing a HIP graph.
"""

from __future__ import annotations

import math
from typing import Any, NamedTuple, Optional

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch import Tensor

from deberta_amd import _eager
from deberta_amd.blocks import _on_gpu, call_bias_gelu, fused_add_layer_norm
from deberta_amd.hidden import _ext, _wide_dtype

_TAGS = (torch.Tag.cudagraph_unsafe,)  # as the package's other ops
MAX_ENTRIES = 128  # top alternatives, or a teacher's entries, of a row
MAX_TOP_VOCAB = 1 << 19  # columns of a call that asks for top alternatives


class TokenLogprobs(NamedTuple):
    """What :func:`fused_token_logprobs` gives, float32 but for the ids."""

    logprobs: Optional[Tensor]  # (...), with ids
    entropy: Tensor  # (...)
    logsumexp: Tensor  # (...)
    top_logprobs: Optional[Tensor]  # (..., top_k), the largest first
    top_ids: Optional[Tensor]  # (..., top_k) int64


def _check_temperature(what: str, temperature: float) -> float:
    t = float(temperature)
    if not 2.0**-100 <= t <= 2.0**100:
        raise ValueError(f"{what}: temperature must be positive and finite (2^-100 to 2^100), got {temperature}")
    return t


# ---------------------------------------------------------------------------
# log probabilities


def _token_logprobs_impl(
    logits: Tensor, ids: Optional[Tensor], top_k: int, temperature: float, ignore_index: int
) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    """(logprobs, entropy, lse, top_logprobs, top_ids, stats): logprobs empty
    without ids, the top ones of no columns with ``top_k`` 0; stats is the
    backward's."""
    return _ext().logprobs_fwd(logits, ids, top_k, temperature, ignore_index)


def _token_logprobs_bwd_impl(
    dlogprobs: Optional[Tensor],
    dentropy: Optional[Tensor],
    dlse: Optional[Tensor],
    dtop: Optional[Tensor],
    logits: Tensor,
    ids: Optional[Tensor],
    top_ids: Optional[Tensor],
    stats: Tensor,
    temperature: float,
    ignore_index: int,
) -> Tensor:
    """The logits' gradient in their type; None for results without one, not
    for all."""
    return _ext().logprobs_bwd(dlogprobs, dentropy, dlse, dtop, logits, ids, top_ids, stats, temperature, ignore_index)


token_logprobs = torch.library.custom_op(
    "deberta_amd::token_logprobs", _token_logprobs_impl, mutates_args=(), device_types="cuda", tags=_TAGS
)
token_logprobs_bwd = torch.library.custom_op(
    "deberta_amd::token_logprobs_bwd", _token_logprobs_bwd_impl, mutates_args=(), device_types="cuda", tags=_TAGS
)


@token_logprobs.register_fake
def _token_logprobs_fake(logits, ids, top_k, temperature, ignore_index):
    rows = logits.shape[:-1]
    row = lambda *s: logits.new_empty(s, dtype=torch.float32)  # noqa: E731
    return (
        row(*rows) if ids is not None else row(0),
        row(*rows),
        row(*rows),
        row(*rows, top_k),
        logits.new_empty((*rows, top_k), dtype=torch.int64),
        row(logits.numel() // logits.shape[-1], 4),
    )


@token_logprobs_bwd.register_fake
def _token_logprobs_bwd_fake(dlogprobs, dentropy, dlse, dtop, logits, ids, top_ids, stats, temperature, ignore_index):
    return logits.new_empty(logits.shape)


def _token_logprobs_setup(ctx, inputs, output):
    logits, ids, top_k, ctx.temperature, ctx.ignore_index = inputs
    logprobs, _, _, top_logprobs, top_ids, stats = output
    ctx.mark_non_differentiable(
        top_ids, stats, *(() if ids is not None else (logprobs,)), *(() if top_k else (top_logprobs,))
    )
    ctx.save_for_backward(logits, ids, top_ids if top_k else None, stats)
    ctx.set_materialize_grads(False)


def _token_logprobs_backward(ctx, dlogprobs, dentropy, dlse, dtop, dtop_ids, dstats):
    logits, ids, top_ids, stats = ctx.saved_tensors
    if ids is None:
        dlogprobs = None
    if top_ids is None:
        dtop = None
    if dlogprobs is None and dentropy is None and dlse is None and dtop is None:
        return (None,) * 5
    dx = token_logprobs_bwd(
        dlogprobs, dentropy, dlse, dtop, logits, ids, top_ids, stats, ctx.temperature, ctx.ignore_index
    )
    return dx, None, None, None, None


torch.library.register_autograd(
    "deberta_amd::token_logprobs", _token_logprobs_backward, setup_context=_token_logprobs_setup
)


def _cpu_rows(what: str, logits: Tensor) -> None:
    if logits.dim() == 0 or logits.shape[-1] == 0:
        raise ValueError(f"{what}: logits need a last dimension of at least one column, got shape {tuple(logits.shape)}")
    if not logits.dtype.is_floating_point:
        raise TypeError(f"{what}: logits must be floating point, got {logits.dtype}")


def _cpu_scaled(logits: Tensor, out_of: Optional[Tensor], temperature: float) -> tuple[Tensor, Tensor]:
    """((x - m) / T, m / T) in the type that results are computed in, m the row's
    largest: scaled without it a row of the type's lowest value would overflow.
    Rows ``out_of`` are zeros, whatever they hold."""
    x = logits.to(_wide_dtype(logits.dtype))
    if out_of is not None:
        x = torch.where(out_of.unsqueeze(-1), 0.0, x)
    most = x.detach().amax(-1, keepdim=True)
    most = torch.where(most == -math.inf, torch.finfo(x.dtype).min, most)
    return (x - most) / temperature, (most / temperature).squeeze(-1)


def _cpu_whole(what: str, name: str, t: Tensor, shape: tuple, logits: Tensor) -> Tensor:
    if t.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{what}: {name} must be int64 or int32, got {t.dtype}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{what}: {name} must have shape {shape}, got {tuple(t.shape)}")
    if t.device != logits.device:
        raise ValueError(f"{what}: {name} are on {t.device}, the logits on {logits.device}")
    return t.long()


def _cpu_token_logprobs(logits: Tensor, ids: Optional[Tensor], top_k: int, temperature: float, ignore_index: int) -> TokenLogprobs:
    what = "fused_token_logprobs"
    _cpu_rows(what, logits)
    V = logits.shape[-1]
    if not 0 <= top_k <= min(V, MAX_ENTRIES):
        raise ValueError(f"{what}: top_k must be in [0, min(V, {MAX_ENTRIES})], got {top_k} for {V} columns")
    if top_k and V > MAX_TOP_VOCAB:
        raise ValueError(f"{what}: top_k needs a vocabulary of at most {MAX_TOP_VOCAB}, got {V}")
    out_of = None
    if ids is not None:
        ids = _cpu_whole(what, "ids", ids, tuple(logits.shape[:-1]), logits)
        out_of = ids == ignore_index
        ids = ids.masked_fill(out_of, 0)
        if ((ids < 0) | (ids >= V)).any():
            raise IndexError(f"{what}: an id is outside the vocabulary of {V}")
    z, most = _cpu_scaled(logits, out_of, temperature)
    fill = lambda t: t if out_of is None else t.masked_fill(out_of.view(out_of.shape + (1,) * (t.dim() - out_of.dim())), 0.0)  # noqa: E731
    logp = torch.log_softmax(z, -1)
    p = logp.exp()
    entropy = -(p * torch.where(p > 0, logp, 0.0)).sum(-1)
    lse = most + torch.logsumexp(z, -1)
    logprobs = None if ids is None else fill(logp.gather(-1, ids.unsqueeze(-1)).squeeze(-1))
    top_logprobs = top_ids = None
    if top_k:
        order = logits.detach().masked_fill(logits.isnan(), -math.inf)
        top_ids = torch.sort(order, dim=-1, descending=True, stable=True).indices[..., :top_k]
        top_logprobs = fill(logp.gather(-1, top_ids))
        if out_of is not None:
            top_ids = top_ids.masked_fill(out_of.unsqueeze(-1), -1)
    return TokenLogprobs(logprobs, fill(entropy), fill(lse), top_logprobs, top_ids)


def fused_token_logprobs(
    logits: Tensor,
    ids: Optional[Tensor] = None,
    top_k: int = 0,
    temperature: float = 1.0,
    ignore_index: int = -100,
) -> TokenLogprobs:
    """For each row of ``(..., V)`` logits, in one pass over them: the log
    probability of its token in ``ids`` (int64 or int32, ``(...)``), the entropy
    ``-sum(p log p)``, ``logsumexp(z)``, and the ``top_k`` (at most 128) largest
    logits' log probabilities and ids, the largest first, equal ones by the lower
    id.  All of it is of ``softmax(logits / temperature)``, in float32.

    A row whose id is ``ignore_index`` is left out: its logits are not read, its
    results are 0, its top ids -1, its gradient 0.  An id outside the vocabulary
    has the log probability NaN, and its row's gradient is NaN unless that of the
    log probability is 0 (on CPU tensors it raises).

    Every result but the ids is differentiable; the gradient has the logits'
    type and reads them again.  The logits are kept for it: change them in
    place only after the backward.  ``top_k`` needs ``V <= 524288``; NaN counts as
    -inf among the largest."""
    t = _check_temperature("fused_token_logprobs", temperature)
    if not logits.is_cuda:
        return _cpu_token_logprobs(logits, ids, int(top_k), t, int(ignore_index))
    if _eager.eager(logits):
        out = _ext().logprobs(logits, ids, int(top_k), t, int(ignore_index))
        if out is not None:
            return TokenLogprobs(*out)
    lp, entropy, lse, top_lp, top_ids, _ = torch.ops.deberta_amd.token_logprobs(logits, ids, int(top_k), t, int(ignore_index))
    return TokenLogprobs(
        lp if ids is not None else None, entropy, lse, top_lp if top_k else None, top_ids if top_k else None
    )


# ---------------------------------------------------------------------------
# distillation


def _distill_loss_impl(
    logits: Tensor, teacher_ids: Tensor, teacher_logits: Tensor, teacher_lse: Optional[Tensor], temperature: float
) -> tuple[Tensor, Tensor]:
    """(loss per row, the backward's stats)."""
    return _ext().distill_fwd(logits, teacher_ids, teacher_logits, teacher_lse, temperature)


def _distill_loss_bwd_impl(
    dloss: Tensor,
    logits: Tensor,
    teacher_ids: Tensor,
    teacher_logits: Tensor,
    teacher_lse: Optional[Tensor],
    stats: Tensor,
    temperature: float,
) -> Tensor:
    """The logits' gradient in their type."""
    return _ext().distill_bwd(dloss, logits, teacher_ids, teacher_logits, teacher_lse, stats, temperature)


distill_loss = torch.library.custom_op(
    "deberta_amd::distill_loss", _distill_loss_impl, mutates_args=(), device_types="cuda", tags=_TAGS
)
distill_loss_bwd = torch.library.custom_op(
    "deberta_amd::distill_loss_bwd", _distill_loss_bwd_impl, mutates_args=(), device_types="cuda", tags=_TAGS
)


@distill_loss.register_fake
def _distill_loss_fake(logits, teacher_ids, teacher_logits, teacher_lse, temperature):
    rows = logits.shape[:-1]
    stats = logits.new_empty((logits.numel() // logits.shape[-1], 4), dtype=torch.float32)
    return logits.new_empty(rows, dtype=torch.float32), stats


@distill_loss_bwd.register_fake
def _distill_loss_bwd_fake(dloss, logits, teacher_ids, teacher_logits, teacher_lse, stats, temperature):
    return logits.new_empty(logits.shape)


def _distill_loss_setup(ctx, inputs, output):
    *tensors, ctx.temperature = inputs
    _, stats = output
    ctx.mark_non_differentiable(stats)
    ctx.save_for_backward(*tensors, stats)


def _distill_loss_backward(ctx, dloss, dstats):
    return distill_loss_bwd(dloss, *ctx.saved_tensors, ctx.temperature), None, None, None, None


torch.library.register_autograd("deberta_amd::distill_loss", _distill_loss_backward, setup_context=_distill_loss_setup)


def _cpu_distillation(
    logits: Tensor, teacher_ids: Tensor, teacher_logits: Tensor, teacher_lse: Optional[Tensor], temperature: float
) -> Tensor:
    what = "fused_distillation_loss"
    _cpu_rows(what, logits)
    V, rows = logits.shape[-1], tuple(logits.shape[:-1])
    if teacher_ids.dim() != logits.dim() or not 1 <= teacher_ids.shape[-1] <= MAX_ENTRIES:
        raise ValueError(
            f"{what}: teacher_ids must be (..., K) with the logits' rows and K in [1, {MAX_ENTRIES}], got shape "
            f"{tuple(teacher_ids.shape)}"
        )
    ids = _cpu_whole(what, "teacher_ids", teacher_ids, (*rows, teacher_ids.shape[-1]), logits)
    for name, t, shape in (("teacher_logits", teacher_logits, tuple(ids.shape)), ("teacher_lse", teacher_lse, rows)):
        if t is not None and (tuple(t.shape) != shape or t.device != logits.device):
            raise ValueError(f"{what}: {name} must have shape {shape} and be on {logits.device}, got {tuple(t.shape)} on {t.device}")
    wide = _wide_dtype(logits.dtype)  # float64 beside a student in float64 alone
    if teacher_logits.dtype not in (torch.float32, torch.bfloat16, wide):
        raise TypeError(f"{what} teacher_logits: dtype must be float32 or bfloat16, got {teacher_logits.dtype}")
    if teacher_lse is not None and teacher_lse.dtype not in (torch.float32, wide):
        raise TypeError(f"{what}: teacher_lse must be float32, got {teacher_lse.dtype}")
    if (ids >= V).any():
        raise IndexError(f"{what}: a teacher's id is outside the vocabulary of {V}")
    given = ids >= 0
    t = teacher_logits.to(wide).masked_fill(~given, -math.inf)
    if teacher_lse is not None:
        log_q = t / temperature - teacher_lse.to(wide).unsqueeze(-1)
    else:
        # the largest off first, as from the student's: the type's lowest value would overflow
        most = t.amax(-1, keepdim=True)
        some = most != -math.inf
        log_q = torch.log_softmax(torch.where(some, (t - most) / temperature, 0.0), -1).masked_fill(~some, -math.inf)
    log_q = log_q.masked_fill(~given, -math.inf)
    q = log_q.exp()
    z, _ = _cpu_scaled(logits, ~given.any(-1), temperature)
    log_p = torch.log_softmax(z, -1).gather(-1, ids.clamp(min=0))
    return temperature * (temperature * torch.where(q == 0, 0.0, q * (log_q - log_p)).sum(-1))


def fused_distillation_loss(
    logits: Tensor,
    teacher_ids: Tensor,
    teacher_logits: Tensor,
    temperature: float = 1.0,
    teacher_lse: Optional[Tensor] = None,
) -> Tensor:
    """``T^2 sum_t q_t (log q_t - log p[id_t])`` for each row of ``(..., V)``
    logits, float32 ``(...)``, with ``p = softmax(logits / T)`` over the whole
    vocabulary and the teacher's entries ``teacher_ids`` (int64 or int32) and
    ``teacher_logits`` (float32 or bfloat16), both ``(..., K)`` with K at most 128,
    in any order.

    ``q = softmax(teacher_logits / T)`` over the row's entries, to which a constant
    of the row does not matter: for example the ``top_ids`` and ``top_logprobs`` of
    :func:`fused_token_logprobs` at temperature 1, or at any temperature t
    ``t * top_logprobs`` (its results are of ``logits / t``, and this function divides
    by T whatever it is given).

    With ``teacher_lse`` (float32 ``(...)``), the logsumexp of the teacher's whole
    ``logits / T``, ``q = exp(teacher_logits / T - teacher_lse)``, whose sum is
    below one: what the teacher gives to other tokens is then left out.  The two
    have to be of the same logits, and a constant of one alone does matter: of a
    teacher's pass at the temperature T itself ``T * top_logprobs`` with a
    ``teacher_lse`` of zeros (its ``logsumexp`` goes with the raw logits, not with
    its log probabilities).

    A negative id is no entry, and one of probability 0 adds nothing whatever
    the student's is; a row without entries is not read, its loss and gradient are
    0.  An id that occurs twice counts twice.  An id of V or more makes the row's
    loss NaN, and its gradient unless the loss' is 0 (on CPU tensors it raises).
    The loss' rounding is T^2 times that of the sum, which a large T brings near 0.
    The gradient is the student's alone: a teacher that needs one raises."""
    t = _check_temperature("fused_distillation_loss", temperature)
    if torch.is_grad_enabled() and (teacher_logits.requires_grad or (teacher_lse is not None and teacher_lse.requires_grad)):
        raise ValueError("fused_distillation_loss has no gradient for the teacher: detach its logits")
    if not logits.is_cuda:
        return _cpu_distillation(logits, teacher_ids, teacher_logits, teacher_lse, t)
    if _eager.eager(logits):
        loss = _ext().distill(logits, teacher_ids, teacher_logits, teacher_lse, t)
        if loss is not None:
            return loss
    return torch.ops.deberta_amd.distill_loss(logits, teacher_ids, teacher_logits, teacher_lse, t)[0]


# ---------------------------------------------------------------------------
# module


class FusedMLMHead(nn.Module):
    """A masked language model's head: ``LayerNorm(gelu(dense(hidden)))`` (one
    kernel each behind the dense product), the product with the vocabulary's
    ``(V, C)`` matrix given at the call (the embedding's, where they are tied)
    plus ``bias``, and on these logits the operators above.

    ``hidden`` is ``(..., C)``: commonly the masked positions, gathered."""

    def __init__(self, config: Any) -> None:
        super().__init__()
        hidden = int(config.hidden_size)
        act = getattr(config, "hidden_act", "gelu")
        if act != "gelu":
            raise NotImplementedError(f"FusedMLMHead supports hidden_act 'gelu', got {act!r}")
        self.dense = nn.Linear(hidden, hidden)
        self.LayerNorm = nn.LayerNorm(hidden, eps=float(getattr(config, "layer_norm_eps", 1e-7)))
        self.bias = nn.Parameter(torch.zeros(int(config.vocab_size)))

    def forward(self, hidden: Tensor, weight: Tensor) -> Tensor:
        """The logits, ``(..., V)``."""
        if _on_gpu(hidden):
            x = F.linear(hidden, self.dense.weight)
            x = fused_add_layer_norm(call_bias_gelu(x, self.dense.bias.to(x.dtype)), None, None, self.LayerNorm)
        else:
            x = self.LayerNorm(F.gelu(self.dense(hidden)))
        return F.linear(x, weight, self.bias)

    def forward_loss(
        self, hidden: Tensor, weight: Tensor, labels: Tensor, ignore_index: int = -100
    ) -> tuple[Tensor, TokenLogprobs]:
        """The mean of ``-log p[label]`` over the labels that are not
        ``ignore_index`` (0 without any), and the rows' results."""
        rows = fused_token_logprobs(self(hidden, weight), labels, ignore_index=ignore_index)
        count = (labels != ignore_index).sum().clamp(min=1)
        return -rows.logprobs.sum() / count, rows

    def forward_distillation(
        self,
        hidden: Tensor,
        weight: Tensor,
        teacher_ids: Tensor,
        teacher_logits: Tensor,
        temperature: float = 1.0,
        teacher_lse: Optional[Tensor] = None,
    ) -> Tensor:
        """The mean of :func:`fused_distillation_loss` over the rows that have an
        entry (0 without any)."""
        loss = fused_distillation_loss(self(hidden, weight), teacher_ids, teacher_logits, temperature, teacher_lse)
        return loss.sum() / (teacher_ids >= 0).any(-1).sum().clamp(min=1)

    @torch.no_grad()
    def predict(self, hidden: Tensor, weight: Tensor, top_k: int = 5, temperature: float = 1.0) -> TokenLogprobs:
        """The ``top_k`` best tokens for each position with their log
        probabilities, and the entropy."""
        return fused_token_logprobs(self(hidden, weight), top_k=top_k, temperature=temperature)
