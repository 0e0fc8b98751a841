"""Calls of the vocabulary operators on the GPU that need care on the way to the
kernels: tensors without memory of their own, wrapped and traced calls, views with
a pending sign, transforms, calls that overlap on streams, rows by the hundred
megabytes and by the million.  Tolerances as in test_gpu_vocab.py."""

from __future__ import annotations

import sys

import pytest
import torch

import deberta_amd as da
from deberta_amd import vocab
from oracle import vocab as ov
from tests._hidden import Wrapper

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float32
U = 2.0**-24


def _say(*a):
    print(*a, file=sys.stderr, flush=True)


def _rand(*shape, seed, dtype=FP, std=2.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def _on_gpu(*shape, seed, gpu, dtype, std=2.0):
    return torch.randn(shape, generator=torch.Generator(device=gpu).manual_seed(seed), device=gpu).mul_(std).to(dtype)


def test_wrapped_arguments_count(gpu):
    x, ids = _rand(5, 24, seed=1).to(gpu), torch.tensor([3, 0, 4, 1, 2], device=gpu)
    t_ids, teacher, lse = ids[:, None].repeat(1, 2), _rand(5, 2, seed=2).to(gpu), torch.ones(5, device=gpu) * 3
    want = da.fused_token_logprobs(x, ids, top_k=3)
    for a, b in ((Wrapper(x), ids), (x, Wrapper(ids)), (Wrapper(x), Wrapper(ids))):
        got = da.fused_token_logprobs(a, b, top_k=3)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    args = [x, t_ids, teacher, 2.0, lse]
    want = da.fused_distillation_loss(*args)
    for k in (0, 1, 2, 4):
        assert torch.equal(da.fused_distillation_loss(*[Wrapper(t) if i == k else t for i, t in enumerate(args)]), want)


def _refusal(call, *given):
    """The error's text, and no tensor without memory in a traceback: printing one
    reads it."""
    try:
        call(*given)
    except Exception as e:
        return f"{type(e).__name__}: {e}"
    return "none"


def _freed(t):
    t = t.clone()
    t.untyped_storage().resize_(0)
    return t


def test_tensors_without_memory_are_refused(gpu):
    x, ids = _rand(5, 24, seed=1).to(gpu), torch.tensor([3, 0, 4, 1, 2], device=gpu)
    t_ids, teacher, lse = ids[:, None].repeat(1, 2), _rand(5, 2, seed=2).to(gpu), torch.ones(5, device=gpu)
    lp, _, _, top, top_ids, stats = vocab._token_logprobs_impl(x, ids, 2, 1.0, -100)
    loss, d_stats = vocab._distill_loss_impl(x, t_ids, teacher, lse, 1.0)
    calls = (
        (da.fused_token_logprobs, [x, ids], (0, 1)),
        (da.fused_distillation_loss, [x, t_ids, teacher, 1.0, lse], (0, 1, 2, 4)),
        (vocab._token_logprobs_bwd_impl, [lp, lp, lp, top, x, ids, top_ids, stats, 1.0, -100], range(8)),
        (vocab._distill_loss_bwd_impl, [loss, x, t_ids, teacher, lse, d_stats, 1.0], range(6)),
    )
    said = [(f.__name__, k, _refusal(f, *[_freed(t) if i == k else t for i, t in enumerate(args)])) for f, args, which in calls for k in which]
    bad = [s for s in said if not (s[2].startswith("ValueError") and "no memory" in s[2])]
    assert not bad


def test_a_pending_sign_counts(gpu):
    x, ids = _rand(5, 24, seed=1).to(gpu), torch.tensor([3, 0, 4, 1, 2], device=gpu)
    t_ids, teacher, lse, g = ids[:, None].repeat(1, 2), _rand(5, 2, seed=2).to(gpu), torch.ones(5, device=gpu), _rand(5, seed=3).to(gpu)
    _, _, _, top, top_ids, stats = vocab._token_logprobs_impl(x, ids, 3, 1.0, -100)
    d_stats = vocab._distill_loss_impl(x, t_ids, teacher, None, 1.0)[1]
    neg = torch._neg_view
    for call in (
        lambda f: da.fused_token_logprobs(f(x), ids, top_k=3).top_logprobs,
        lambda f: da.fused_distillation_loss(f(x), t_ids, f(teacher), 2.0, f(lse)),
        lambda f: vocab._token_logprobs_bwd_impl(f(g), f(g), f(g), f(top), x, ids, top_ids, stats, 1.0, -100),
        lambda f: vocab._distill_loss_bwd_impl(f(g), x, t_ids, teacher, None, d_stats, 1.0),
    ):
        assert torch.equal(call(neg), call(lambda t: -t))


def test_results_are_allocated_as_others(gpu):
    """Results are inference tensors in inference mode, and in the allocator's count."""
    x, ids = _rand(5, 24, seed=1).to(gpu), torch.tensor([3, 0, 4, 1, 2], device=gpu)
    want = da.fused_token_logprobs(x, ids, top_k=3)
    with torch.inference_mode():
        got = da.fused_token_logprobs(x, ids, top_k=3)
        loss = da.fused_distillation_loss(x, ids[:, None], x[:, :1])
    assert all(t.is_inference() for t in (*got, loss)) and not any(t.is_inference() for t in want)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    before = torch.cuda.memory_allocated()
    big = da.fused_token_logprobs(torch.zeros(1 << 20, 2, device=gpu))
    assert torch.cuda.memory_allocated() - before == 2 * 4 << 20  # entropy and lse; the logits are gone
    del big
    assert torch.cuda.memory_allocated() == before


def test_traced_calls_compute(gpu):
    """torch.jit.trace records the ops, not what the extension allocates."""
    x, y = _rand(5, 300, seed=1).to(gpu), _rand(5, 300, seed=2).to(gpu)
    ids = torch.tensor([3, 0, 4, 1, 2], device=gpu)

    def f(v):
        o = da.fused_token_logprobs(v, ids, top_k=3)
        return o.logprobs, o.top_ids, da.fused_distillation_loss(v, ids[:, None], v[:, :1] * 0.0, 2.0)

    traced = torch.jit.trace(f, (x,), check_trace=False)
    assert all(torch.equal(a, b) for a, b in zip(traced(y), f(y)))


def test_transforms_raise(gpu):
    """Forward-mode tangents and torch.func have no rule here: an error, not a
    result without them."""
    import torch.autograd.forward_ad as fwAD

    x, ids = _rand(5, 24, seed=1).to(gpu), torch.tensor([3, 0, 4, 1, 2], device=gpu)
    t_ids, teacher, lse = ids[:, None].repeat(1, 2), _rand(5, 2, seed=2).to(gpu), torch.ones(5, device=gpu)
    for call, t in (
        (lambda v: da.fused_token_logprobs(v, ids).logprobs, x),
        (lambda v: da.fused_distillation_loss(v, t_ids, teacher), x),
        (lambda v: da.fused_distillation_loss(x, t_ids, v), teacher),
        (lambda v: da.fused_distillation_loss(x, t_ids, teacher, 1.0, v), lse),
    ):
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(t.expand(3, *t.shape))
        with pytest.raises((RuntimeError, ValueError)):
            torch.func.grad(lambda v: call(v).sum())(t)
        with fwAD.dual_level(), pytest.raises(RuntimeError):
            call(fwAD.make_dual(t, torch.ones_like(t)))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda i: da.fused_token_logprobs(x, i).logprobs)(ids.expand(3, 5))


def test_logits_changed_in_place_are_noticed(gpu):
    """The backward reads them again."""
    base = _rand(4, 500, seed=1).to(gpu).requires_grad_()
    ids = torch.tensor([3, 0, 4, 1], device=gpu)
    for call in (lambda v: da.fused_token_logprobs(v, ids).logprobs, lambda v: da.fused_distillation_loss(v, ids[:, None], base.detach()[:, :1])):
        x = base * 1.0
        y = call(x).sum()
        x.mul_(2.0)
        with pytest.raises(RuntimeError, match="inplace"):
            y.backward()
    x = base * 1.0
    o = da.fused_token_logprobs(x, ids, top_k=3)
    o.top_ids.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        o.top_logprobs.sum().backward()


def test_a_graph_of_the_gradient_and_a_second_backward(gpu):
    x = _rand(4, 500, seed=1).to(gpu).requires_grad_()
    ids = torch.tensor([3, 0, 4, 1], device=gpu)
    lp = da.fused_token_logprobs(x, ids).logprobs
    (a,) = torch.autograd.grad(lp.sum(), x, retain_graph=True)
    (b,) = torch.autograd.grad(lp.sum(), x, create_graph=True)
    assert torch.equal(a, b) and b.requires_grad
    with pytest.raises(RuntimeError, match="logits are not twice"):
        b.sum().backward()


def test_checkpointed_logits(gpu):
    """Activation checkpointing runs the forward again in the backward."""
    from torch.utils.checkpoint import checkpoint

    w, h = _rand(700, 32, seed=1, std=0.3).to(gpu).requires_grad_(), _rand(6, 32, seed=2).to(gpu).requires_grad_()
    ids = torch.tensor([3, 0, 4, 1, 699, -100], device=gpu)

    def f(h):
        return da.fused_token_logprobs(h @ w.t(), ids).logprobs

    want = torch.autograd.grad(f(h).sum(), (h, w))
    got = torch.autograd.grad(checkpoint(f, h, use_reentrant=False).sum(), (h, w))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_overlapping_calls_keep_their_workspaces(gpu):
    """Calls in parts on several streams at once: each has a workspace of its own."""
    V, N = 128100, 24
    xs = [_on_gpu(N, V, seed=k, gpu=gpu, dtype=BF) for k in range(4)]
    ids = torch.randint(0, V, (N,), generator=torch.Generator().manual_seed(1)).to(gpu)
    t_ids, teacher = torch.randint(0, V, (N, 20), generator=torch.Generator().manual_seed(2)).to(gpu), _rand(N, 20, seed=3).to(gpu)

    def call(x):
        o = da.fused_token_logprobs(x, ids, top_k=30)
        return [*o, da.fused_distillation_loss(x, t_ids, teacher, 2.0)]

    want = [call(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[] for _ in xs]
    for _ in range(4):
        for k, (x, s) in enumerate(zip(xs, streams)):
            with torch.cuda.stream(s):
                got[k].append(call(x))
    torch.cuda.synchronize()
    for k, w in enumerate(want):
        assert all(torch.equal(a, b) for o in got[k] for a, b in zip(o, w))


def test_rows_by_the_hundred_megabytes(gpu):
    """The shapes that go in parts for their bytes, and gradients past the caches
    (560 x 128100: 143 MB), against float64 in pieces on the GPU."""
    V, N, T = 128100, 560, 1.3
    for dtype, n in ((BF, N), (FP, 300)):
        _say("megabytes", dtype)
        x = _on_gpu(n, V, seed=1, gpu=gpu, dtype=dtype).requires_grad_()
        ids = torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(2)).to(gpu)
        ids[5::7] = -100
        t_ids = torch.randint(0, V, (n, 70), generator=torch.Generator().manual_seed(3)).to(gpu)
        t_ids[3::5, 40:] = -1
        t_ids[2::9] = -1
        teacher = _rand(n, 70, seed=4, std=3.0).to(gpu)
        g = _rand(n, seed=5, std=1.0).to(gpu)
        o = da.fused_token_logprobs(x, ids, temperature=T)
        (d,) = torch.autograd.grad(o.logprobs, x, g)
        loss = da.fused_distillation_loss(x, t_ids, teacher, T)
        (e,) = torch.autograd.grad(loss, x, g)
        h = torch.finfo(dtype).eps / 2
        for lo in range(0, n, 70):
            r = slice(lo, lo + 70)
            logp = torch.log_softmax(x.detach()[r].double() / T, -1)
            p, l, out = logp.exp(), logp.abs(), ids[r] == -100
            at = ids[r].clamp(min=0).unsqueeze(-1)
            lp = logp.gather(-1, at).squeeze(-1).masked_fill(out, 0.0)
            assert ((o.logprobs[r].double() - lp).abs() <= U * (200 + 4 * lp.abs())).all()
            H, M2 = ov.moments(logp)
            assert ((o.entropy[r].double() - H.masked_fill(out, 0.0)).abs() <= U * (200 + 200 * H + 6 * M2)).all()
            gr = g[r].double().masked_fill(out, 0.0).unsqueeze(-1)
            want = (-gr * p).scatter_add_(-1, at, gr) / T
            tol = U * gr.abs() / T * (p * (3 * l + 220)).scatter_add_(-1, at, torch.full_like(gr, 4.0)) + h * want.abs()
            assert ((d[r].double() - want).abs() <= tol).all()
            none = (t_ids[r] < 0).all(-1, keepdim=True)
            q, lq = ov.teacher_probs(t_ids[r], teacher[r], T)
            at = t_ids[r].clamp(min=0)
            want = ov.distillation(logp, at, q, lq, T)
            lqa, la = lq.nan_to_num(0, 0, 0).abs(), l.gather(-1, at)
            tol = T * T * U * (q * ((3 * lqa + 40) * (lqa + la) + 220 + 4 * la + 3 * lqa)).sum(-1)
            assert ((loss[r].double() - want).abs() <= tol).all()
            gr = torch.where(none, 0.0, g[r].double().unsqueeze(-1) * T)
            want = (gr * p).scatter_add_(-1, at, -gr * q)
            tol = U * gr.abs() * (p * (3 * l + 260)).scatter_add_(-1, at, q * (3 * lqa + 44)) + h * want.abs()
            assert ((e[r].double() - want).abs() <= tol).all()


def _logprobs_agree(o, x, ids, T):
    """Every result against float64, in pieces of up to 9M values on the GPU."""
    N, V = x.shape
    k = 0 if o.top_ids is None else o.top_ids.shape[-1]
    step = max(1, (9 << 20) // V)
    for lo in range(0, N, step):
        r = slice(lo, lo + step)
        logp = torch.log_softmax(x[r].double() / T, -1)
        out = ids[r] == -100
        lp = logp.gather(-1, ids[r].clamp(min=0).unsqueeze(-1)).squeeze(-1).masked_fill(out, 0.0)
        assert ((o.logprobs[r].double() - lp).abs() <= U * (200 + 4 * lp.abs())).all()
        H, M2 = ov.moments(logp)
        assert ((o.entropy[r].double() - H.masked_fill(out, 0.0)).abs() <= U * (200 + 200 * H + 6 * M2)).all()
        z = x[r].double() / T
        lse, m = torch.logsumexp(z, -1).masked_fill(out, 0.0), z.amax(-1).abs()
        assert ((o.logsumexp[r].double() - lse).abs() <= U * (200 + 3 * m + lse.abs())).all()
        if k:
            top = torch.sort(x[r].float(), dim=-1, descending=True, stable=True).indices[:, :k]
            assert torch.equal(o.top_ids[r], top.masked_fill(out.unsqueeze(-1), -1))
            tl = logp.gather(-1, top).masked_fill(out.unsqueeze(-1), 0.0)
            assert ((o.top_logprobs[r].double() - tl).abs() <= U * (200 + 4 * tl.abs())).all()


def _distillation_agrees(loss, x, t_ids, teacher, T):
    N, V = x.shape
    step = max(1, (9 << 20) // V)
    for lo in range(0, N, step):
        r = slice(lo, lo + step)
        logp = torch.log_softmax(x[r].double() / T, -1)
        q, lq = ov.teacher_probs(t_ids[r], teacher[r], T)
        at = t_ids[r].clamp(min=0)
        lqa, la = lq.nan_to_num(0, 0, 0).abs(), logp.gather(-1, at).abs()
        tol = T * T * U * (q * ((3 * lqa + 40) * (lqa + la) + 220 + 4 * la + 3 * lqa)).sum(-1)
        assert ((loss[r].double() - ov.distillation(logp, at, q, lq, T)).abs() <= tol).all()


def _entries(N, V, K, gpu):
    t_ids = torch.randint(0, V, (N, K), generator=torch.Generator().manual_seed(3))
    t_ids[3::5, K // 2 :] = -1
    t_ids[2::9] = -1
    return t_ids.to(gpu), _rand(N, K, seed=4, std=3.0).to(gpu)


@pytest.mark.parametrize(
    "N,V,dtype,k",
    [
        (1100, 128100, BF, 5), (560, 128100, FP, 5),  # whole rows by 512 threads
        (2100, 65001, BF, 64), (2100, 32501, FP, 64),  # by 256
        (1100, 128100, BF, 0), (560, 128100, FP, 0),  # in parts
        (8400, 16001, BF, 0), (8400, 8001, FP, 0),  # as many bytes in rows of one part
    ],
)
def test_logits_past_the_caches(N, V, dtype, k, gpu):
    """Forwards that autograd does not record, from 256 MiB on: their loads go past
    the caches.  A seventh of the rows is left out."""
    _say("past the caches", N, V, dtype, k)
    x = _on_gpu(N, V, seed=N + V, gpu=gpu, dtype=dtype)
    assert x.numel() * x.element_size() >= 256 << 20
    ids = torch.randint(0, V, (N,), generator=torch.Generator().manual_seed(2)).to(gpu)
    ids[5::7] = -100
    _logprobs_agree(da.fused_token_logprobs(x, ids, top_k=k, temperature=1.3), x, ids, 1.3)


@pytest.mark.parametrize(
    "N,V,dtype,grad",
    [
        (1100, 128100, BF, False), (560, 128100, FP, False), (8400, 16001, BF, False), (8400, 8001, FP, False),
        (2100, 128100, BF, True), (1100, 128100, FP, True),
    ],
)
def test_distillations_past_the_caches(N, V, dtype, grad, gpu):
    """From 256 MiB on where no backward reads the logits again, from 512 MiB on
    where one does."""
    _say("distillation past the caches", N, V, dtype, grad)
    x = _on_gpu(N, V, seed=N + V, gpu=gpu, dtype=dtype)
    assert x.numel() * x.element_size() >= (512 if grad else 256) << 20
    t_ids, teacher = _entries(N, V, 40, gpu)
    loss = da.fused_distillation_loss(x.requires_grad_(grad), t_ids, teacher, 1.3).detach()
    _distillation_agrees(loss, x.detach(), t_ids, teacher, 1.3)


@pytest.mark.parametrize(
    "N,V,dtype,k",
    [
        (100, 128100, FP, 0), (70, 128100, FP, 20), (100, 128100, FP, 5), (60, 262144, FP, 0), (36, 262145, BF, 64), (20, 1 << 19, FP, 5),
        (130, 1 << 19, FP, 5), (120, 128100, FP, 5),  # whole
        (24, (1 << 21) + 1, FP, 0), (1, 5_000_001, BF, 0), (1, 20_000_000, FP, 0), (1, 1 << 25, BF, 0),
    ],
)
def test_few_long_rows(N, V, dtype, k, gpu):
    """Rows in up to 2442 parts, and the longest that a block reads by itself.  The sum's
    share is 400 u: of a whole row 16 + 64 + 10 additions and as many scalings of 3 u by a
    larger maximum, of one in parts 16 + 2 + 10 and 10 in the join; 3 ln V <= 52."""
    _say("long rows", N, V, dtype, k)
    x = _on_gpu(N, V, seed=N, gpu=gpu, dtype=dtype)
    ids = torch.randint(0, V, (N,), generator=torch.Generator().manual_seed(2)).to(gpu)
    ids[2::7] = -100
    t_ids, teacher = _entries(N, V, 40, gpu)
    o = da.fused_token_logprobs(x, ids, top_k=k, temperature=1.3)
    loss = da.fused_distillation_loss(x, t_ids, teacher, 1.3)
    for r in range(N):
        z = x[r].double() / 1.3
        lse = torch.logsumexp(z, -1)
        if ids[r] == -100:
            assert o.logprobs[r] == 0 and o.entropy[r] == 0 and o.logsumexp[r] == 0
        else:
            lp = z[ids[r]] - lse
            assert abs(o.logprobs[r].double() - lp) <= U * (400 + 4 * lp.abs())
            assert abs(o.logsumexp[r].double() - lse) <= U * (400 + 3 * z.amax().abs() + lse.abs())
            H, M2 = ov.moments(z - lse)
            assert abs(o.entropy[r].double() - H) <= U * (400 + 400 * H + 6 * M2)
            if k:
                top = torch.sort(x[r].float(), descending=True, stable=True).indices[:k]
                assert torch.equal(o.top_ids[r], top)
                assert ((o.top_logprobs[r].double() - (z[top] - lse)).abs() <= U * (400 + 4 * (z[top] - lse).abs())).all()
        q, lq = ov.teacher_probs(t_ids[r], teacher[r], 1.3)
        at = t_ids[r].clamp(min=0)
        lqa, la = lq.nan_to_num(0, 0, 0).abs(), (z[at] - lse).abs()
        want = 1.3**2 * torch.where(q == 0, 0.0, q * (lq - (z[at] - lse))).sum()
        assert abs(loss[r].double() - want) <= 1.3**2 * U * (q * ((3 * lqa + 40) * (lqa + la) + 420 + 4 * la + 3 * lqa)).sum()


def test_the_longest_row(gpu):
    """2^31 - 128 columns, forward and backward, in pieces against float64.  A lane of the
    join adds up 512 parts' sums: 540 additions and as many scalings of 3 u, 3 ln V <= 65:
    2300 u."""
    V, T = (1 << 31) - 128, 1.3
    _say("the longest row")
    x = torch.empty(1, V, dtype=BF, device=gpu).normal_(generator=torch.Generator(device=gpu).manual_seed(1)).requires_grad_()
    for token in (0, V - 1):
        ids = torch.tensor([token], device=gpu)
        o = da.fused_token_logprobs(x, ids, temperature=T)
        pieces = x.detach().view(-1).split(1 << 27)
        lse = torch.logsumexp(torch.stack([torch.logsumexp(c.double() / T, -1) for c in pieces]), -1)
        lp = x.detach()[0, token].double() / T - lse
        assert abs(o.logprobs.double() - lp) <= U * (2300 + 4 * lp.abs())
        assert abs(o.logsumexp.double() - lse) <= U * (2300 + 24 + lse)
    (d,) = torch.autograd.grad(o.logprobs.sum(), x)
    at = 0
    for c, e in zip(pieces, d.view(-1).split(1 << 27)):
        logp = c.double() / T - lse
        want = -logp.exp() / T
        tol = U * -want * (3 * logp.abs() + 2300) + 2.0**-8 * want.abs()
        at += c.numel()
        if at == V:
            want[-1] += 1 / T
            tol[-1] += 4 * U + 2.0**-8
        assert ((e.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("N,V", [(3, 128100), (200, 128100), (3, 20011), (600, 20011)])
def test_the_largest_of_moved_rows(N, V, gpu):
    """Thousands of values that are equal in their upper 16 bits and differ below them:
    more than compete in the fast search.  In parts, and by 512 and 256 threads."""
    for dtype in (FP, BF):
        x = (_on_gpu(N, V, seed=V, gpu=gpu, dtype=FP) + 1000.0).to(dtype)
        x[1] = 1000.0 - (x[1] - 1000.0).abs()  # the largest side by side at one value
        want = torch.sort(x.float(), dim=-1, descending=True, stable=True).indices
        for k in (1, 20, 64, 128):
            _say("moved", N, V, dtype, k)
            o = da.fused_token_logprobs(x, top_k=k)
            assert torch.equal(o.top_ids, want[:, :k])
            tl = torch.log_softmax(x.double(), -1).gather(-1, want[:, :k])
            assert ((o.top_logprobs.double() - tl).abs() <= U * (200 + 4 * tl.abs())).all()


def test_more_rows_than_a_launch_takes(gpu):
    """2^22 blocks a launch: rows of two columns, where log p is -log1p(exp(-d)) of
    their difference, to the tolerances above."""
    N = (1 << 22) + 37
    x = _on_gpu(N, 2, seed=1, gpu=gpu, dtype=FP).requires_grad_()
    ids = torch.zeros(N, dtype=torch.int32, device=gpu)
    ids[-5:] = torch.tensor([1, -100, 0, 1, 1])
    o = da.fused_token_logprobs(x, ids, top_k=1)
    (d,) = torch.autograd.grad(o.logprobs.sum(), x)
    z = x.detach().double()
    logp = torch.log_softmax(z, -1)
    out = ids == -100
    at = ids.clamp(min=0).long().unsqueeze(-1)
    lp = logp.gather(-1, at).squeeze(-1).masked_fill(out, 0.0)
    assert ((o.logprobs.double() - lp).abs() <= U * (200 + 4 * lp.abs())).all()
    assert torch.equal(o.top_ids.squeeze(-1), (z[:, 1] > z[:, 0]).long().masked_fill(out, -1))
    p = logp.exp()
    want = torch.zeros_like(p).scatter_(-1, at, 1.0) - p
    want[out] = 0.0
    assert ((d.double() - want).abs() <= U * (p * (3 * logp.abs() + 220) + 4) + U * want.abs()).all()
    loss = da.fused_distillation_loss(x, at, torch.zeros(N, 1, device=gpu))
    want = -logp.gather(-1, at).squeeze(-1)
    assert ((loss.double() - want).abs() <= U * (40 * want + 220 + 4 * want)).all()
    (d,) = torch.autograd.grad(loss[-9:].sum(), x)
    assert not d[:-9].any() and d[-9:].abs().sum() > 0


def test_a_wide_row(gpu):
    """2^20 + 3 columns: past what the largest are given for, and not else."""
    V = (1 << 20) + 3
    x = _on_gpu(2, V, seed=1, gpu=gpu, dtype=BF)
    with pytest.raises(ValueError, match="at most 524288"):
        da.fused_token_logprobs(x, top_k=1)
    x.requires_grad_()
    ids = torch.tensor([V - 1, 0], device=gpu)
    o = da.fused_token_logprobs(x, ids)
    logp = torch.log_softmax(x.detach().double(), -1)
    lp = logp.gather(-1, ids.unsqueeze(-1)).squeeze(-1)
    # twice the batches of 128100 columns, at most: twice the sum's share
    assert ((o.logprobs.double() - lp).abs() <= U * (400 + 4 * lp.abs())).all()
    (d,) = torch.autograd.grad(o.logprobs.sum(), x)
    p = logp.exp()
    want = torch.zeros_like(p).scatter_(-1, ids.unsqueeze(-1), 1.0) - p
    tol = U * (p * (3 * logp.abs() + 420)).scatter_add_(-1, ids.unsqueeze(-1), torch.full((2, 1), 4.0, device=gpu, dtype=torch.float64))
    assert ((d.double() - want).abs() <= tol + 2.0**-8 * want.abs()).all()
    # and the widest with them: 2^19
    y = _on_gpu(2, 1 << 19, seed=2, gpu=gpu, dtype=FP)
    top = da.fused_token_logprobs(y, top_k=128)
    assert torch.equal(top.top_ids, torch.sort(y, dim=-1, descending=True, stable=True).indices[:, :128])
