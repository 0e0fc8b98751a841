"""Timed cases of the operators on a vocabulary's logits: the log probabilities
of given tokens with the entropy and the top alternatives, and the
distillation loss against a teacher's top logits, each with its gradient.

Each case is one call a user's program makes: a serving or scoring pass, or a
training step's forward and backward of the operator.  ``listed()`` names the
cases, ``draw`` gives more of the same ranges, ``prepare`` builds what the
program holds before the call and ``run`` makes it, in elementary torch
operations (float32, rounded once at the end), or through this package's entry
points where ``own`` is set.  ``exact`` is the operator's definition in float64.

Sizes follow the repository's configurations (vocabulary 128100, 16 x 512
positions of which 15% are masked, 4096 packed positions) and generic ones
around them, odd ones included.

With z = logits / T, lse = log sum_j exp(z_j) and p = exp(z - lse):

    logprob  = z_id - lse                entropy = -sum_j p_j (z_j - lse)
    top      = the k largest z (ties: the lower index), their z - lse
    loss     = T^2 sum_t q_t (log q_t - (z_{id_t} - lse)),  q = softmax(teacher / T)

A row whose id is -100 (or that has no teacher entry: every id -1) gives zeros,
its top ids are -1 and its gradient is zero.
"""

from __future__ import annotations

import math
import random
from types import SimpleNamespace

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp32": 4}
IGNORE = -100
MOST_BYTES = 4096 * 128100 * 2  # of a drawn case's logits, as the largest listed one's


# ---------------------------------------------------------------------------
# the cases


def _logprobs(name, rows, vocab, dtype, top, ids, ignore, banned, temperature, train):
    """top: alternatives a row; ids: with given tokens; ignore: the share of
    rows that are left out; banned: columns at the end that are -inf; train:
    "", "nll" (the gradient of the given tokens' log probabilities) or "all"
    (those of every result)."""
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "dtype": dtype, "top": top, "ids": ids,
            "ignore": ignore, "banned": banned, "temperature": temperature, "train": train}


def _distil(name, rows, vocab, dtype, teacher, entries, pad, temperature):
    """teacher: the type of its logits; entries: how many a row; pad: the share
    of rows that have fewer, some of them none."""
    return {"name": name, "op": "distil", "rows": rows, "vocab": vocab, "dtype": dtype, "teacher": teacher,
            "entries": entries, "pad": pad, "temperature": temperature}


def listed():
    return [
        # serving: the best five tokens for one masked position
        _logprobs("fill_one", 1, 128100, "bf16", 5, False, 0.0, 0, 1.0, ""),
        # serving: eight requests' candidates with their alternatives, float32 logits of an odd vocabulary
        _logprobs("score_few", 8, 50021, "fp32", 20, True, 0.0, 0, 0.7, ""),
        # scoring a sequence of 512 tokens, logits padded to a multiple of 128 columns
        _logprobs("score_sequence", 512, 128128, "bf16", 10, True, 0.0, 28, 1.0, ""),
        # a teacher's pass: its 64 best tokens for each masked position, to distil from
        _logprobs("teacher_top", 2048, 128100, "bf16", 64, False, 0.0, 0, 2.0, ""),
        # a test-sized training step
        _logprobs("mlm_small", 39, 1001, "fp32", 0, True, 0.1, 0, 1.0, "nll"),
        # the generator's loss of a base-sized batch: the masked 15% of 16 x 512 positions, gathered
        _logprobs("mlm_base", 1229, 128100, "bf16", 0, True, 0.0, 0, 1.0, "nll"),
        # the same loss on every position's logits, the unmasked ones left out by their label
        _logprobs("mlm_all_positions", 4096, 128100, "bf16", 0, True, 0.85, 0, 1.0, "nll"),
        # a training step that uses the entropy and the alternatives too
        _logprobs("entropy_odd", 700, 50021, "fp32", 8, True, 0.05, 0, 1.3, "all"),
        # distillation of a few positions
        _distil("distil_few", 16, 128100, "bf16", "bf16", 16, 0.0, 1.0),
        # a base-sized batch's masked positions against 64 stored entries each
        _distil("distil_base", 1229, 128100, "bf16", "fp32", 64, 0.2, 2.0),
        # ragged entries, float32 logits of an odd vocabulary
        _distil("distil_odd", 777, 50021, "fp32", "fp32", 17, 0.5, 3.0),
        # packed positions against 128 entries each
        _distil("distil_packed", 4096, 128100, "bf16", "bf16", 128, 0.1, 2.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    vocab = rng.choice((128100, _log(rng, 1000, 128100)))
    rows = _log(rng, 1, min(4096, MOST_BYTES // (2 * BYTES[dtype] * vocab)))
    temperature = rng.choice((1.0, round(rng.uniform(0.5, 4.0), 2)))
    if rng.random() < 0.4:
        case = _distil("", rows, vocab, dtype, rng.choice(("bf16", "fp32")), _log(rng, 1, 128),
                       rng.choice((0.0, round(rng.uniform(0.1, 0.6), 2))), temperature)
    else:
        train = rng.choice(("", "nll", "nll", "all"))
        ids = bool(train) or rng.random() < 0.6
        top = rng.choice((0, _log(rng, 1, 128))) if ids and train != "all" else _log(rng, 1, 128)
        ignore = round(rng.uniform(0.05, 0.9), 2) if ids and rng.random() < 0.4 else 0.0
        case = _logprobs("", rows, vocab, dtype, top, ids, ignore, rng.choice((0, 0, _log(rng, 1, 200))), temperature, train)
    del case["name"]
    return case


# ---------------------------------------------------------------------------
# what a program holds before the call


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    N, V, dtype = case["rows"], case["vocab"], TYPES[case["dtype"]]
    s = SimpleNamespace(case=dict(case), T=case["temperature"])
    # a model's logits: a spread of two around nothing, and the right token above them
    logits = torch.randn((N, V), generator=g, device=DEV).mul_(2.0)
    uniform = lambda *shape: torch.rand(shape, generator=g, device=DEV, dtype=torch.float64)  # noqa: E731
    rows = torch.arange(N, device=DEV)
    if case["op"] == "logprobs":
        words = V - case["banned"]
        # token frequencies fall as 1 / rank
        s.ids = torch.exp(uniform(N) * math.log(words)).long().clamp_(0, words - 1)
        logits[rows, s.ids] += 12.0 * uniform(N).float()
        if case["banned"]:
            logits[:, words:] = -math.inf
        if case["ignore"]:
            s.ids.masked_fill_(uniform(N) < case["ignore"], IGNORE)
        active = (s.ids != IGNORE).float()
        if not case["ids"]:
            s.ids = None
        if case["train"]:  # the gradient of a mean over the rows that count
            s.g = -active / active.sum().clamp(min=1.0)
        if case["train"] == "all":
            s.g_entropy, s.g_lse, s.g_top = (torch.randn(shape, generator=g, device=DEV) / N for shape in (N, N, (N, case["top"])))
    else:
        K = case["entries"]
        # a teacher's entries: other tokens in each row, the largest first
        step = 1 + (uniform(N, 1) * (V // K - 1)).long()
        s.teacher_ids = ((uniform(N, 1) * V).long() + step * torch.arange(K, device=DEV)) % V
        teacher = (3.0 * torch.randn((N, K), generator=g, device=DEV) + 6.0).sort(-1, descending=True).values
        logits.scatter_(1, s.teacher_ids, 0.7 * teacher + torch.randn((N, K), generator=g, device=DEV))
        s.teacher = teacher.to(TYPES[case["teacher"]])
        if case["pad"]:
            kept = torch.where(uniform(N, 1) < case["pad"], (uniform(N, 1) * (K + 1)).long(), K)
            s.teacher_ids.masked_fill_(torch.arange(K, device=DEV) >= kept, -1)
        s.g = (s.teacher_ids >= 0).any(-1).float()
        s.g /= s.g.sum().clamp(min=1.0)
    s.logits = logits.to(dtype).requires_grad_(case["op"] == "distil" or bool(case["train"]))
    return s


# ---------------------------------------------------------------------------
# one pass


def run(s):
    if s.case["op"] == "logprobs":
        return _own_logprobs(s) if own else _plain_logprobs(s)
    return _own_distil(s) if own else _plain_distil(s)


def _own_logprobs(s):
    from deberta_amd import fused_token_logprobs

    c = s.case
    o = fused_token_logprobs(s.logits, s.ids, top_k=c["top"], temperature=s.T)
    out = [t for t in (o.logprobs, o.entropy, o.logsumexp) if t is not None]
    if c["top"]:
        out += [o.top_logprobs, o.top_ids]
    if c["train"] == "nll":
        out += torch.autograd.grad(o.logprobs, (s.logits,), s.g)
    elif c["train"]:
        out += torch.autograd.grad((o.logprobs, o.entropy, o.logsumexp, o.top_logprobs), (s.logits,),
                                   (s.g, s.g_entropy, s.g_lse, s.g_top))
    return tuple(out)


def _own_distil(s):
    from deberta_amd import fused_distillation_loss

    loss = fused_distillation_loss(s.logits, s.teacher_ids, s.teacher, temperature=s.T)
    return (loss, *torch.autograd.grad(loss, (s.logits,), s.g))


def _log_softmax(s):
    """(z - lse, lse) in float32."""
    z = s.logits.float() / s.T
    most = z.amax(-1, keepdim=True)
    z = z - most
    log_sum = z.exp().sum(-1, keepdim=True).log()
    return z - log_sum, most + log_sum


def _top(logits, k):
    """The indices of the k largest values of each row, equal ones by their
    index: the largest of whole numbers that order as (value, -index)."""
    bits = logits.float().add(0.0).contiguous().view(torch.int32).long()  # -0 counts as 0
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    key = (order << 32) | (0xFFFFFFFF - torch.arange(logits.shape[-1], device=DEV))
    return 0xFFFFFFFF - (key.topk(k, -1).values & 0xFFFFFFFF)


@torch.no_grad()
def _plain_logprobs(s):
    c = s.case
    logp, lse = _log_softmax(s)
    p = logp.exp()
    entropy = -(p * torch.where(p > 0, logp, 0.0)).sum(-1)
    lse = lse.squeeze(-1)
    out = [entropy, lse]
    if s.ids is not None:
        active = s.ids != IGNORE
        at = s.ids.masked_fill(~active, 0).unsqueeze(-1)
        left_out = lambda t: t.masked_fill(~active.view([-1] + [1] * (t.dim() - 1)), 0.0)  # noqa: E731
        out = [left_out(t) for t in (logp.gather(-1, at).squeeze(-1), entropy, lse)]
    if c["top"]:
        top = _top(s.logits, c["top"])
        values = logp.gather(-1, top)
        out += [values, top] if s.ids is None else [left_out(values), top.masked_fill(~active.unsqueeze(-1), -1)]
    if c["train"]:
        # of z: p_j (-g - sum g_top - g_entropy (log p_j + entropy) + g_lse), and g or g_top where j is the token
        weight, per_p = -s.g, 0.0
        if c["train"] == "all":
            weight = weight - s.g_top.sum(-1) - s.g_entropy * entropy + s.g_lse
            per_p = s.g_entropy.unsqueeze(-1)
        d = p * (weight.unsqueeze(-1) - per_p * torch.where(p > 0, logp, 0.0))
        d = d.scatter_add_(-1, at, s.g.unsqueeze(-1))
        if c["train"] == "all":
            d = d.scatter_add_(-1, top, s.g_top)
        out.append(left_out(d / s.T).to(s.logits.dtype))
    return tuple(out)


@torch.no_grad()
def _plain_distil(s):
    logp, _ = _log_softmax(s)
    given = s.teacher_ids >= 0
    at = s.teacher_ids.clamp(min=0)
    t = (s.teacher.float() / s.T).masked_fill(~given, -math.inf)
    most = t.amax(-1, keepdim=True).clamp(min=-3e38)  # a row without entries
    e = (t - most).exp()
    total = e.sum(-1, keepdim=True)
    any_given = total > 0
    total = torch.where(any_given, total, 1.0)
    q = e / total
    log_q = torch.where(q > 0, t - most - total.log(), 0.0)
    log_p = torch.where(q > 0, logp.gather(-1, at), 0.0)
    loss = s.T * s.T * (q * (log_q - log_p)).sum(-1)
    g = s.g.unsqueeze(-1) * s.T
    d = (logp.exp() * torch.where(any_given, g, 0.0)).scatter_add_(-1, at, -g * q)
    return loss, d.to(s.logits.dtype)


# ---------------------------------------------------------------------------
# what a pass cannot do without


def work(case):
    N, V, b = case["rows"], case["vocab"], BYTES[case["dtype"]]
    if case["op"] == "logprobs":
        read = N * (1.0 - case["ignore"])
        per_row = 8 + 8 * case["ids"] + 4 * case["ids"] + 12 * case["top"]
        train = case["train"]
    else:
        read = N * (1.0 - case["pad"] / (case["entries"] + 1))  # the rows that have an entry
        per_row = 4 + 4 + case["entries"] * (8 + BYTES[case["teacher"]])
        train = "nll"
    # a value's: its scaling, maximum, exp, sum and the entropy's product; backward exp, products and rounding
    return {"bytes": read * V * b + N * per_row + (N * V * b if train else 0), "flops": read * V * (6.0 + (5.0 if train else 0.0))}


# ---------------------------------------------------------------------------
# the definitions, in float64


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    N = case["rows"]
    parts = [(_exact_logprobs if case["op"] == "logprobs" else _exact_distil)(s, slice(lo, min(N, lo + 256)))
             for lo in range(0, N, 256)]
    return tuple(torch.cat(column) for column in zip(*parts))


def _exact_logprobs(s, rows):
    c = s.case
    z = s.logits[rows].double() / s.T
    lse = torch.logsumexp(z, -1)
    logp = z - lse[:, None]
    p = logp.exp()
    plogp = torch.special.xlogy(p, p)
    entropy = -plogp.sum(-1)
    ids = s.ids[rows] if s.ids is not None else torch.zeros(len(z), dtype=torch.int64, device=DEV)
    out_of = ids == IGNORE
    mine = torch.arange(len(z), device=DEV)
    ids = torch.where(out_of, 0, ids)
    results = [entropy, lse]
    if s.ids is not None:
        results.insert(0, logp[mine, ids])
    if c["top"]:
        values, top = torch.sort(logp, dim=-1, descending=True, stable=True)
        values, top = values[:, : c["top"]], top[:, : c["top"]]
        results += [values, top]
    if c["train"]:
        g = s.g[rows].double()
        d = -g[:, None] * p
        if c["train"] == "all":
            g_entropy, g_lse, g_top = (t[rows].double() for t in (s.g_entropy, s.g_lse, s.g_top))
            d -= g_entropy[:, None] * (plogp + p * entropy[:, None])
            d += (g_lse - g_top.sum(-1))[:, None] * p
            d[mine[:, None], top] += g_top
        d[mine, ids] += g
        results.append(d / s.T)
    for t in results:
        t[out_of] = -1 if t.dtype is torch.int64 else 0
    return results


def _exact_distil(s, rows):
    logp = torch.log_softmax(s.logits[rows].double() / s.T, -1)
    ids, g = s.teacher_ids[rows], s.g[rows].double()
    none = (ids < 0).all(-1)
    t = (s.teacher[rows].double() / s.T).masked_fill(ids < 0, -math.inf)
    t[none] = 0.0  # any, they are left out below
    q = torch.softmax(t, -1)
    log_q = torch.where(ids < 0, 0.0, torch.log_softmax(t, -1))
    mine = torch.arange(len(ids), device=DEV)[:, None]
    loss = s.T**2 * (q * (log_q - logp[mine, ids.clamp(min=0)])).sum(-1)
    d = logp.exp()
    d.index_put_((mine.expand_as(ids), ids.clamp(min=0)), -q, accumulate=True)
    d *= s.T * g[:, None]
    loss[none], d[none] = 0.0, 0.0
    return [loss, d]
