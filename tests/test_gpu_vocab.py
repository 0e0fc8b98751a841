"""The operators on a vocabulary's logits on the GPU against their float64
definitions (oracle/vocab.py) on the same inputs: every result and gradient, over
widths, alignments, types, masks and the cases that go wrong first (no rows, one
column, rows of nothing but -inf or of the type's lowest value, infinities and
NaN, ties in their thousands, ids outside the vocabulary, entries that occur twice,
offsets past 32 bits).

Tolerances, with u = 2^-24 the half step of float32 and h that of the gradient's
type, element by element.  With e = exp(z - m) and ln e = (x - m) / T:

  e        x - m, its scaling and the scale itself are a rounding each, v_exp_f32
           is off by at most a step:  (3 |ln e| + 2) u of e
  s        a term goes through at most 16 additions in a batch, one a batch
           (16 of them at 128128 columns and 256 threads), 10 over lanes and
           waves, and through as many scalings by a larger maximum, each (3 |d| + 3)
           u with the d adding up to |ln e|: with sum p |ln e| <= ln V <= 12
           less than 200 u of s, and so of ln s with logf's step
  logprob  (x - m) / T - ln s, both of one sign:  (200 + 4 |lp|) u
  entropy  ln s - (sum e ln e) / s, a term's error (6 |ln e| + 160) u:
           (200 + 200 H + 6 M2) u,  M2 = sum p ln^2 p
  lse      (200 + 3 |m| / T + |lse|) u
  p        e / s:  (3 |lp| + 210) u
  dx       p (a + b ln p) + c:  with G = |g| + sum |g_top| + |g_lse| + |g_H| (H +
           |lp| + 24), the row's terms and their cancelling parts:
           p / T (G (3 |lp| + 220) u + |g_H| tol(H)) + 4 u |c| / T + h |dx|
  q        expf of a difference, a sum of 128:  (3 |lq| + 40) u of q
  loss     T^2 u sum q ((3 |lq| + 40) (|lq| + |lp|) + 220 + 4 |lp| + 3 |lq|)
  dx       |g| T u (Q p (3 |lp| + 260) + sum q (3 |lq| + 44)) + h |dx|

What is below the smallest normal bf16 or float32, 2^-126, may be flushed.
"""

from __future__ import annotations

import sys
from types import SimpleNamespace

import pytest
import torch

import deberta_amd as da
from oracle import vocab as ov

pytestmark = pytest.mark.gpu

U = 2.0**-24
TINY = 2.0**-126
BF, FP = torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")


def _say(*a):
    print(*a, file=sys.stderr, flush=True)


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _rand(*shape, seed, dtype=FP, std=2.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def _ints(lo, hi, *shape, seed):
    return torch.randint(lo, hi, shape, generator=torch.Generator().manual_seed(seed))


def _within(name, got, want, tol):
    got, want = got.detach().double().cpu(), want.detach().double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.equal(got.isnan(), want.isnan()), name
    assert torch.equal(got.isinf(), want.isinf()) and torch.equal(got[got.isinf()], want[want.isinf()]), name
    over = ((got - want).abs() - tol).nan_to_num(0.0, 0.0, 0.0)
    assert (over <= 0).all(), (name, over.max().item(), (got - want).nan_to_num(0.0).abs().max().item())


def _check_logprobs(logits, ids, top_k, T=1.0, grads="all", ignore=-100, seed=1):
    """``logits`` on the GPU (a view, perhaps), ``ids`` on the CPU or None."""
    x = logits.detach().requires_grad_()
    rows, V = x.shape[:-1], x.shape[-1]
    o = da.fused_token_logprobs(x, None if ids is None else ids.to(x.device), top_k=top_k, temperature=T, ignore_index=ignore)
    c = logits.detach().cpu()
    c64 = c.double().requires_grad_()
    out = torch.zeros(rows, dtype=torch.bool) if ids is None else ids == ignore
    keep = lambda t: torch.where(out.view(out.shape + (1,) * (t.dim() - out.dim())), 0.0, t)  # noqa: E731
    z = torch.where(out.unsqueeze(-1), 0.0, c64)
    logp = ov.log_probs(z, T)
    H, M2 = ov.moments(logp)
    lse = ov.logsumexp(z, T)
    lp = logp.gather(-1, torch.where(out, 0, ids.long()).clamp(0, V - 1).unsqueeze(-1)).squeeze(-1) if ids is not None else None
    if ids is not None:
        lp = torch.where((ids >= 0) & (ids < V) | out, lp, NAN)
    tol_H = U * (200 + 200 * H.detach().nan_to_num() + 6 * M2.detach().nan_to_num())
    m = z.detach().amax(-1).nan_to_num(0.0, 0.0, 0.0).abs()
    results = [o.entropy, o.logsumexp]
    wants = [keep(H), keep(lse)]
    assert o.entropy.dtype == FP and o.logsumexp.dtype == FP
    _within("entropy", o.entropy, wants[0], tol_H)
    _within("lse", o.logsumexp, wants[1], U * (200 + 3 * m / T + lse.detach().nan_to_num(0, 0, 0).abs()))
    if ids is not None:
        results.append(o.logprobs)
        wants.append(keep(lp))
        _within("logprobs", o.logprobs, wants[-1], U * (200 + 4 * lp.detach().nan_to_num(0, 0, 0).abs()))
    else:
        assert o.logprobs is None
    if top_k:
        top = ov.largest(z.detach(), top_k)
        assert o.top_ids.dtype == torch.int64
        assert torch.equal(o.top_ids.cpu(), torch.where(out.unsqueeze(-1), -1, top))
        tl = logp.gather(-1, top)
        results.append(o.top_logprobs)
        wants.append(keep(tl))
        _within("top", o.top_logprobs, wants[-1], U * (200 + 4 * tl.detach().nan_to_num(0, 0, 0).abs()))
    else:
        assert o.top_ids is None and o.top_logprobs is None
    if not grads:
        return o
    if grads == "nll":
        results, wants = [o.logprobs], [keep(lp)]
    gs = [_rand(*t.shape, seed=seed + i, std=1.0) for i, t in enumerate(results)]
    (dx,) = torch.autograd.grad(results, x, [g.to(x.device) for g in gs])
    assert dx.dtype == x.dtype and dx.shape == x.shape
    (want,) = torch.autograd.grad(wants, c64, [g.double() for g in gs])
    bad = torch.zeros_like(out) if ids is None else ((ids < 0) | (ids >= V)) & ~out
    want = torch.where(bad.unsqueeze(-1), NAN, want)
    # a column without probability has no gradient; autograd's formulas multiply 0 by inf there
    dead = (c.double() == -INF) & ~z.detach().isnan().any(-1, keepdim=True) & (z.detach().amax(-1, keepdim=True) < INF)
    dead &= ~(z.detach() == -INF).all(-1, keepdim=True) & ~bad.unsqueeze(-1)
    by = dict(zip(["entropy", "lse", *(["lp"] if ids is not None else []), *(["top"] if top_k else [])] if grads == "all" else ["lp"], gs))
    zero = torch.zeros(rows, dtype=torch.float64)
    g_lp, g_h, g_l = (by.get(k, zero).double().abs() for k in ("lp", "entropy", "lse"))
    g_top = by["top"].double().abs().sum(-1) if "top" in by else zero
    l, p = logp.detach().nan_to_num(0, 0, 0).abs(), logp.detach().exp().nan_to_num()
    G = (g_lp + g_top + g_l + g_h * (H.detach().nan_to_num() + 24)).unsqueeze(-1) + g_h.unsqueeze(-1) * l
    term = torch.zeros_like(p)
    if "top" in by:
        term.scatter_add_(-1, top, by["top"].double().abs())
    if "lp" in by:
        term.scatter_add_(-1, ids.long().clamp(0, V - 1).unsqueeze(-1), g_lp.unsqueeze(-1))
    tol = p / T * (G * (3 * l + 220) * U + (g_h * tol_H).unsqueeze(-1)) + 4 * U * term / T
    if dead.any():
        sparse = torch.zeros_like(p)  # a given token of probability 0 keeps its own term
        if "lp" in by:
            sparse.scatter_add_(-1, ids.long().clamp(0, V - 1).unsqueeze(-1), torch.where(out | bad, 0.0, by["lp"].double()).unsqueeze(-1))
        if "top" in by:
            sparse.scatter_add_(-1, top, torch.where(out.unsqueeze(-1), 0.0, by["top"].double()))
        want = torch.where(dead, sparse / T, want)
    _within("dlogits", dx, want, tol + _half(x.dtype) * want.abs().nan_to_num() + TINY)
    return o


WIDTHS = [1, 2, 3, 7, 8, 9, 15, 16, 17, 63, 64, 65, 127, 129, 500, 1001, 2047, 8191, 8200, 16385, 50021, 128100]


@pytest.mark.parametrize("V", WIDTHS)
def test_widths(V, gpu):
    """Rows of every alignment: an odd width moves each row's start."""
    _say("widths", V)
    N = 9 if V < 20000 else 4
    for dtype, T in ((BF, 1.0), (FP, 0.7)):
        x = _rand(N, V, seed=V, dtype=dtype).to(gpu)
        ids = _ints(0, V, N, seed=V + 1)
        for k in sorted({0, 1, min(V, 5)}):
            _check_logprobs(x, ids, k, T)
        _check_logprobs(x, ids, 0, T, grads="nll")


@pytest.mark.parametrize("k", [2, 31, 64, 65, 127, 128])
@pytest.mark.parametrize("V", [128, 1000, 4099, 33000])
def test_largest(k, V, gpu):
    _say("largest", V, k)
    for dtype in (BF, FP):
        _check_logprobs(_rand(5, V, seed=k, dtype=dtype).to(gpu), None, k)


def test_all_of_a_row(gpu):
    for V in (1, 5, 64, 100, 128):
        _say("all", V)
        _check_logprobs(_rand(3, V, seed=V, dtype=BF).to(gpu), _ints(0, V, 3, seed=1), V)


@pytest.mark.parametrize("dtype", [BF, FP], ids=str)
@pytest.mark.parametrize("V", [300, 20011, 50021, 128100])
def test_ties_and_orders(V, dtype, gpu):
    """Values in the orders that a selection is worst at: all equal, two values,
    rising, falling, the largest side by side, zeros of both signs, one far out."""
    _say("ties", V, dtype)
    x = torch.empty(9, V)
    ramp = torch.linspace(-6, 6, V)
    x[0] = 2.5
    x[1] = (torch.arange(V) % 3 == 1).float()
    x[2], x[3] = ramp, ramp.flip(0)
    x[4] = -4.0
    x[4, 100:240] = 3.0 + torch.arange(140) % 7 * 0.125
    x[5] = torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0)
    x[6] = _rand(V, seed=3)
    x[6, V // 2] = 80.0
    x[7] = -3.0 - torch.arange(V) % 5 * 0.25
    x[8] = (_rand(V, seed=4) * 2).round()
    for k in (1, 17, 128):
        _check_logprobs(x.to(dtype).to(gpu), None, k, grads="" if V > 1000 else "all")


@pytest.mark.parametrize("dtype", [BF, FP], ids=str)
def test_masked_columns_and_rows(dtype, gpu):
    """-inf, the type's lowest value, NaN and infinities, in places of every kind."""
    V = 777
    lowest = torch.finfo(dtype).min
    x = _rand(12, V, seed=5, dtype=dtype)
    x[0, 5:] = -INF
    x[1, :700] = -INF
    x[2] = -INF
    x[3] = lowest
    x[4, ::2] = lowest
    x[5, 776] = NAN
    x[6, 0] = INF
    x[7, :400] = -INF
    x[7, 400] = INF
    x[8] = -INF
    x[8, 300] = 1.0
    x[9] = x[9] * 1000  # one token takes all
    x[10] = x[10] + 9984.0
    x[11] = -INF
    x[11, 7] = lowest
    ids = _ints(0, V, 12, seed=6)
    ids[0], ids[1], ids[8] = 3, 5, 299
    for T in (1.0, 0.5, 3.0):
        _say("masked", dtype, T)
        if T == 1.0:
            _check_logprobs(x.to(gpu), ids, 9, T)
        else:  # without what overflows in its scaling
            _check_logprobs(x[[0, 1, 2, 5, 6, 7, 8, 9]].to(gpu), ids[[0, 1, 2, 5, 6, 7, 8, 9]], 9, T)
    # a mask that leaves nothing: every token alike, whatever the temperature
    o = da.fused_token_logprobs(x[3:4].to(gpu), ids[3:4].to(gpu), temperature=0.25)
    want = torch.tensor(float(V)).log()
    assert abs(o.entropy.item() - want) <= 200 * U * 8 and abs(o.logprobs.item() + want) <= 230 * U


@pytest.mark.parametrize("dtype", [BF, FP], ids=str)
def test_signalling_nan_among_the_largest(dtype, gpu):
    """A NaN counts as -inf among the largest whichever its bits are, and hides no
    value beside it: quiet and signalling ones at the row's single values, in its
    vectors and in its segments, in whole rows and in rows in parts."""
    bits = {BF: (torch.int16, 0x7F81, -0x7F), FP: (torch.int32, 0x7F800001, -0x7FFFFF)}[dtype]
    for V, k in ((9, 9), (13, 1), (70, 5), (777, 20), (3001, 128), (90001, 7)):
        _say("signalling", dtype, V, k)
        g = torch.Generator().manual_seed(V)
        x = torch.randperm(4 * V, generator=g).view(4, V)
        x = (x % 256 - 128).to(dtype) if dtype == BF else (x - 2 * V).to(dtype)
        order = torch.rand(4, V, generator=g)
        raw = x.view(bits[0]).clone()
        few = order < 0.02
        few[0] = order[0] < 0.5
        few[1, :3] = few[1, -3:] = True  # beside the row's borders
        few[2] = False
        few[2, V // 2] = few[0, 1] = few[3, V - 2] = True
        raw[few] = bits[1]
        raw[3, order[3] < 0.1] = bits[2]  # with the sign
        x = raw.view(dtype)
        assert x.isnan().sum() == (raw == bits[1]).sum() + (raw == bits[2]).sum()
        clean = torch.where(x.isnan(), -INF, x.float())
        want = torch.sort(clean, dim=-1, descending=True, stable=True).indices[..., :k]
        for first in (0, 1, 3):  # where a row begins between two borders
            wide = torch.zeros(4, V + 5, dtype=bits[0])
            wide[:, first : first + V] = raw
            o = da.fused_token_logprobs(wide.to(gpu).view(dtype)[:, first : first + V], top_k=k)
            assert torch.equal(o.top_ids.cpu(), want), (V, k, first)
            assert o.top_logprobs.isnan().all() and o.logsumexp.isnan().all() and o.entropy.isnan().all()


def test_large_values_keep_their_differences(gpu):
    """Rows moved by a constant: their own rounding, not that of the constant's
    product with 1 / T (which is 2^-8 here), is what is left."""
    ids = _ints(0, 3001, 4, seed=8)
    x = _rand(4, 3001, seed=7, dtype=BF).float()
    for dtype in (FP, BF):
        _check_logprobs((x + 32768.0).to(dtype).to(gpu), ids, 4, 0.3)
    moved = (x + 32768.0) - 32768.0  # what the sum keeps of x
    b = da.fused_token_logprobs((x + 32768.0).to(gpu), ids.to(gpu), top_k=4, temperature=0.3)
    c = da.fused_token_logprobs(moved.to(gpu), ids.to(gpu), top_k=4, temperature=0.3)
    assert torch.equal(b.top_ids, c.top_ids)
    for p, q in ((b.logprobs, c.logprobs), (b.top_logprobs, c.top_logprobs)):
        assert ((p - q).abs() <= 2 * U * (200 + 4 * q.abs())).all()


def test_strides(gpu):
    """Rows of a wider tensor from odd offsets, rows that are one, columns with a
    stride, three dimensions, gradients that are broadcast or not contiguous."""
    ids = _ints(0, 1001, 6, seed=9)
    for dtype in (BF, FP):
        wide = _rand(6, 1111, seed=10, dtype=dtype).to(gpu)
        for first in (0, 1, 3, 4, 7):
            _say("strides", dtype, first)
            _check_logprobs(wide[:, first : first + 1001], ids, 5)
        _check_logprobs(wide[:1, 2:1003].expand(6, 1001), ids, 3)
        _check_logprobs(_rand(1001, 6, seed=11, dtype=dtype).to(gpu).t(), ids, 3)
        _check_logprobs(wide[:, ::2], _ints(0, 556, 6, seed=9), 3)
        _check_logprobs(_rand(2, 3, 400, seed=12, dtype=dtype).to(gpu).transpose(0, 1), _ints(0, 400, 3, 2, seed=9), 3)
        # rows that overlap in memory
        _check_logprobs(torch.as_strided(wide, (6, 1001), (10, 1)), ids, 2, grads="")
    x = _rand(2, 3, 100, seed=13).to(gpu).requires_grad_()
    ids = _ints(0, 100, 2, 3, seed=1).to(gpu)
    o = da.fused_token_logprobs(x, ids, top_k=2)
    (a,) = torch.autograd.grad(o.logprobs.sum() + 2 * o.entropy.sum(), x, retain_graph=True)
    g = torch.ones(3, 2, device=gpu).t()
    (b,) = torch.autograd.grad((o.logprobs, o.entropy), x, (g, 2 * g), retain_graph=True)
    assert torch.equal(a, b)
    wide = torch.zeros(2, 3, 4, device=gpu)
    wide[..., ::2] = _rand(2, 3, 2, seed=14).to(gpu)
    (a,) = torch.autograd.grad(o.top_logprobs, x, wide[..., ::2], retain_graph=True)
    (b,) = torch.autograd.grad(o.top_logprobs, x, wide[..., ::2].contiguous())
    assert torch.equal(a, b)


def test_rows_left_out_and_ids_outside(gpu):
    """Left-out rows are not read (they hold NaN), ids are int32 or int64."""
    for dtype in (BF, FP):
        x = _rand(8, 1003, seed=15, dtype=dtype)
        ids = _ints(0, 1003, 8, seed=16)
        ids[[1, 4]] = -100
        x[[1, 4]] = NAN
        for it in (torch.int64, torch.int32):
            _say("left out", dtype, it)
            _check_logprobs(x.to(gpu), ids.to(it), 6)
        ids[2], ids[3], ids[5] = 1003, -1, -(1 << 31)
        _check_logprobs(x.to(gpu), ids, 6)
        _check_logprobs(x.to(gpu), ids, 0, grads="nll")
        ids[6] = (1 << 40) + 3
        _check_logprobs(x.to(gpu), ids, 0, grads="nll")
        ids[0] = 7
        _check_logprobs(x[[0, 6]].to(gpu), ids[[0, 6]], 0, ignore=7, grads="nll")
    # an id outside whose result is not used adds nothing
    x = _rand(2, 50, seed=17).to(gpu).requires_grad_()
    o = da.fused_token_logprobs(x, torch.tensor([50, 1], device=gpu))
    (d,) = torch.autograd.grad(torch.where(o.logprobs.isnan(), 0.0, o.logprobs).sum(), x)
    assert (d[0] == 0).all() and d[1].isfinite().all() and d[1].abs().sum() > 0


@pytest.mark.parametrize("shape", [(0, 9), (3, 0, 9)], ids=str)
def test_no_rows(shape, gpu):
    x = torch.zeros(shape, device=gpu, requires_grad=True)
    rows = shape[:-1]
    o = da.fused_token_logprobs(x, torch.zeros(rows, dtype=torch.int64, device=gpu), top_k=3)
    loss = da.fused_distillation_loss(x, torch.zeros(*rows, 2, dtype=torch.int64, device=gpu), torch.zeros(*rows, 2, device=gpu))
    assert o.logprobs.shape == loss.shape == rows and o.top_ids.shape == (*rows, 3)
    (d,) = torch.autograd.grad(o.logprobs.sum() + loss.sum(), x)
    assert d.shape == shape


def test_many_rows(gpu):
    """More rows than run at once, of few columns."""
    for V, N in ((3, 70001), (131, 9000)):
        _say("many", V, N)
        x = _rand(N, V, seed=18, dtype=BF).to(gpu)
        _check_logprobs(x, _ints(-1, V, N, seed=19).masked_fill_(_ints(0, 5, N, seed=20) == 0, -100).clamp(min=-100), 2, grads="nll")


@pytest.mark.parametrize("dtype", [BF, FP], ids=str)
@pytest.mark.parametrize("N", [511, 512, 700])
def test_many_narrow_rows(N, dtype, gpu):
    """The blocks that such rows go to (fewer threads from 512 rows on), with ties in
    their hundreds, rows left out and the largest in every number."""
    for V, k, grads in ((130, 128, "all"), (1001, 5, "all"), (1001, 64, "nll"), (3001, 20, "nll")):
        _say("narrow", N, V, k, dtype)
        x = _rand(N, V, seed=V + k, dtype=dtype)
        x[::7] = x[::7].round()
        x[3::50] = 1.5
        ids = _ints(0, V, N, seed=V).masked_fill_(_ints(0, 6, N, seed=k) == 0, -100)
        _check_logprobs(x.to(gpu), ids, k, 1.5, grads=grads)
    _check_distill(_rand(N, 777, seed=3, dtype=dtype).to(gpu), _ints(-1, 777, N, 33, seed=4), _rand(N, 33, seed=5, std=3.0), 2.0)


def test_offsets_past_32_bits(gpu):
    """Rows that begin past 2^31 elements, and past 2^32 bytes; the rows between
    are left out.  Against the same rows by themselves, whose sums may go in
    another order: twice the tolerances above, of the bf16 gradient 2 h."""
    V, N = 128100, 17000
    ids = torch.full((N,), -100)
    picked = [0, 8001, 16764, 16765, 16998]  # 16764 x 128100 < 2^31 < 16765 x 128100
    ids[picked] = _ints(0, V, len(picked), seed=21)
    some = _rand(len(picked), V, seed=22, dtype=BF)
    x = torch.empty(N, V, dtype=BF, device=gpu)
    x[torch.tensor(picked, device=gpu)] = some.to(gpu)
    x.requires_grad_()
    _say("past 32 bits")
    o = da.fused_token_logprobs(x, ids.to(gpu), top_k=3)
    g = _rand(N, seed=23).to(gpu)
    (d,) = torch.autograd.grad(o.logprobs, x, g)
    y = some.to(gpu).requires_grad_()
    p = da.fused_token_logprobs(y, ids[picked].to(gpu), top_k=3)
    (e,) = torch.autograd.grad(p.logprobs, y, g[picked])
    assert torch.equal(o.top_ids[picked], p.top_ids)
    assert ((o.logprobs[picked] - p.logprobs).abs() <= 2 * U * (200 + 4 * p.logprobs.abs())).all()
    assert ((o.entropy[picked] - p.entropy).abs() <= 2 * U * (200 + 206 * 12 * 12)).all()  # H <= ln V, M2 <= its square
    assert ((d[picked].float() - e.float()).abs() <= 2.1 * 2.0**-8 * e.float().abs()).all()
    out = torch.ones(N, dtype=torch.bool, device=gpu)
    out[picked] = False
    assert (o.logprobs[out] == 0).all() and (o.top_ids[out] == -1).all()
    for i in range(0, N, 4000):  # no row between was written otherwise
        assert not d[i : i + 4000][out[i : i + 4000]].any()


# ---------------------------------------------------------------------------
# distillation


def _check_distill(logits, teacher_ids, teacher, T=1.0, lse=None, seed=1):
    x = logits.detach().requires_grad_()
    V = x.shape[-1]
    gpu = x.device
    loss = da.fused_distillation_loss(x, teacher_ids.to(gpu), teacher.to(gpu), T, None if lse is None else lse.to(gpu))
    ids = teacher_ids.long()
    none = (ids < 0).all(-1)
    bad = (ids >= V).any(-1)
    c64 = logits.detach().cpu().double().requires_grad_()
    z = torch.where(none.unsqueeze(-1), 0.0, c64)
    logp = ov.log_probs(z, T)
    q, log_q = ov.teacher_probs(ids, teacher, T, lse)
    inside = ids.clamp(0, V - 1)
    want = torch.where(bad, NAN, ov.distillation(logp, inside, q, log_q, T))
    lq, lp = log_q.nan_to_num(0, 0, 0).abs(), logp.detach().gather(-1, inside).nan_to_num(0, 0, 0).abs()
    if lse is not None:
        lq = lq + (teacher.double() / T).nan_to_num(0, 0, 0).abs()
    qs = q.nan_to_num()
    assert loss.dtype == FP
    _within("loss", loss, want, T * T * U * (qs * ((3 * lq + 40) * (lq + lp) + 220 + 4 * lp + 3 * lq)).sum(-1))
    g = _rand(*loss.shape, seed=seed, std=1.0)
    (dx,) = torch.autograd.grad(loss, x, g.to(gpu))
    assert dx.dtype == x.dtype
    p = logp.detach().exp()
    Q = q.sum(-1, keepdim=True)
    T_g = (g.double() * T).unsqueeze(-1)
    want = (T_g * p * Q).scatter_add_(-1, inside, -T_g * q)
    want = torch.where(none.unsqueeze(-1), 0.0, torch.where(bad.unsqueeze(-1), NAN, want))
    l = logp.detach().nan_to_num(0, 0, 0).abs()
    tol = p.nan_to_num() * Q.nan_to_num() * (3 * l + 260)
    tol.scatter_add_(-1, inside, qs * (3 * lq + 44))
    tol = T_g.abs() * U * tol + _half(x.dtype) * want.abs().nan_to_num()
    _within("dlogits", dx, want, tol + TINY)
    return loss


@pytest.mark.parametrize("K", [1, 2, 17, 63, 64, 65, 127, 128])
def test_distill_entries(K, gpu):
    for dtype, tt, T, V in ((BF, FP, 2.0, 1001), (FP, BF, 1.0, 300), (BF, BF, 0.5, 5003)):
        _say("distill", K, dtype, V)
        x = _rand(6, V, seed=K, dtype=dtype).to(gpu)
        ids = _ints(0, V, 6, K, seed=K + 1)  # with entries that occur twice
        teacher = _rand(6, K, seed=K + 2, dtype=tt, std=3.0)
        _check_distill(x, ids, teacher, T)
        ids[torch.rand(ids.shape, generator=torch.Generator().manual_seed(K)) < 0.3] = -1
        ids[2] = -7
        _check_distill(x, ids.to(torch.int32), teacher, T)
        lse = torch.logsumexp(teacher.float() / T, -1) + 0.2
        _check_distill(x, ids, teacher, T, lse)


@pytest.mark.parametrize("V", WIDTHS)
def test_distill_widths(V, gpu):
    _say("distill", V)
    N, K = (7, 5) if V < 20000 else (4, 33)
    for dtype in (BF, FP):
        x = _rand(N, V, seed=V, dtype=dtype).to(gpu)
        _check_distill(x, _ints(0, V, N, K, seed=V), _rand(N, K, seed=V + 1, std=3.0), 1.5)


def test_distill_one_token_many_times(gpu):
    """Every entry the same token: their terms add up."""
    x = _rand(3, 200, seed=1, dtype=BF).to(gpu)
    _check_distill(x, torch.full((3, 128), 77), _rand(3, 128, seed=2))


def test_distill_extreme_temperatures(gpu):
    """T^2 past float32 on either side.  One entry, so q = 1: the loss is
    T^2 (-log p), at a small T T (max - x), at a large one T^2 log V; a product
    with rounded log2(e) / T and ln 2, two with T, and a sum of V terms."""
    x = _rand(4, 101, seed=1)
    ids = x.argmin(-1, keepdim=True)
    zero = torch.zeros(4, 1)
    for T in (2.0**-100, 2.0**-70):
        loss = da.fused_distillation_loss(x.to(gpu), ids.to(gpu), zero.to(gpu), T).cpu().double()
        want = T * (x.double().amax(-1) - x.double().amin(-1))
        assert ((loss - want).abs() <= 8 * U * want).all(), T
    T = 2.0**60
    loss = da.fused_distillation_loss(x.to(gpu), ids.to(gpu), zero.to(gpu), T).cpu().double()
    want = T * T * torch.tensor(101.0, dtype=torch.float64).log()
    assert ((loss - want).abs() <= 230 * U * want).all()
    for T in (2.0**-100, 2.0**100):  # a vocabulary of one: no loss
        y = x[:, :1].to(gpu).requires_grad_()
        loss = da.fused_distillation_loss(y, torch.zeros(4, 1, dtype=torch.int64, device=gpu), zero.to(gpu), T)
        (d,) = torch.autograd.grad(loss.sum(), y)
        assert (loss == 0).all() and (d == 0).all()


@pytest.mark.parametrize("dtype", [BF, FP], ids=str)
def test_distill_masks(dtype, gpu):
    V, lowest = 333, torch.finfo(dtype).min
    x = _rand(10, V, seed=3, dtype=dtype)
    ids = _ints(0, V, 10, 6, seed=4)
    teacher = _rand(10, 6, seed=5)
    x[0, ids[0, 1]], teacher[0, 1] = -INF, -INF  # 0 of both
    x[1, ids[1, 2]] = -INF  # the loss is infinite
    teacher[2] = -INF  # no entry of a finite logit
    x[3] = -INF
    x[4] = lowest
    x[5, 17] = NAN
    x[6, 18] = INF
    teacher[7, 3] = NAN
    teacher[8] = torch.finfo(FP).min
    ids[9, 4] = V
    _say("distill masks", dtype)
    _check_distill(x.to(gpu), ids, teacher)
    # an id outside in a row whose loss is not used
    y = x[8:].to(gpu).requires_grad_()
    loss = da.fused_distillation_loss(y, ids[8:].to(gpu), teacher[8:].to(gpu))
    (d,) = torch.autograd.grad(torch.where(loss.isnan(), 0.0, loss).sum(), y)
    assert (d[1] == 0).all() and d[0].abs().sum() > 0


@pytest.mark.parametrize("dtype", [BF, FP], ids=str)
def test_distill_teachers_that_leave_float32(dtype, gpu):
    """A teacher whose logits / T leave float32: its largest is taken off first, so
    that a row of the type's lowest value is uniform."""
    x, ids, lowest = _rand(4, 333, seed=3, dtype=dtype).to(gpu), _ints(0, 333, 4, 3, seed=4), torch.finfo(FP).min
    teacher = _rand(4, 3, seed=5)
    teacher[0], teacher[2, 1] = lowest, lowest
    teacher[1] = 3e38 + 1e37 * torch.arange(3)
    _say("distill far teachers", dtype)
    for T in (0.5, 0.25):
        _check_distill(x, ids, teacher, T)
    _check_distill(x, ids, torch.full((4, 3), torch.finfo(BF).min, dtype=BF), 0.5)
    T, far = 2.0**-100, torch.tensor([[1e9, 1e9 - 64.0]]).repeat(4, 1).to(gpu)  # q = (1, 0): T (max - x), as in the test above of such temperatures
    c = x.cpu().double()
    loss = da.fused_distillation_loss(x, torch.stack((x.argmin(-1), x.argmax(-1)), -1), far, T).cpu().double()
    want = T * (c.amax(-1) - c.amin(-1))
    assert ((loss - want).abs() <= 8 * U * want).all()


def test_distill_from_a_teachers_pass(gpu):
    """What a pass at T stores, times T, are logits with a logsumexp of 0: the
    teacher's own probabilities at T."""
    T, K = 2.0, 40
    for dtype in (BF, FP):
        c = _rand(6, 1001, seed=31, dtype=dtype)
        t = da.fused_token_logprobs(c.to(gpu), top_k=K, temperature=T)
        lse = torch.zeros(6)
        _check_distill(_rand(6, 1001, seed=32, dtype=dtype).to(gpu), t.top_ids.cpu(), T * t.top_logprobs.cpu(), T, lse)
        loss = da.fused_distillation_loss(c.to(gpu), t.top_ids, T * t.top_logprobs, T, lse.to(gpu)).cpu().double()
        # of a student that is the teacher nothing: q = p to the pass' (200 + 4 |lp|) u, a product's and the loss' own
        lp = torch.log_softmax(c.double() / T, -1).gather(-1, t.top_ids.cpu())
        q, l = lp.exp(), lp.abs()
        assert (loss.abs() <= T * T * U * (q * ((6 * l + 40) * 2 * l + 2 * (220 + 8 * l))).sum(-1)).all()


def test_distill_strides(gpu):
    wide = _rand(6, 1111, seed=6, dtype=BF).to(gpu)
    ids, teacher = _ints(0, 1001, 6, 9, seed=7), _rand(6, 9, seed=8)
    for first in (0, 1, 5):
        _check_distill(wide[:, first : first + 1001], ids, teacher, 2.0)
    big = torch.zeros(6, 18, dtype=torch.int64)
    big[:, ::2] = ids
    a = _check_distill(wide[:, :1001], big[:, ::2], teacher, 2.0)
    b = da.fused_distillation_loss(wide[:, :1001], big.to(gpu)[:, ::2], teacher.to(gpu).t().contiguous().t(), 2.0)
    assert torch.equal(a, b)
    _check_distill(_rand(2, 3, 400, seed=9).to(gpu), _ints(0, 400, 2, 3, 4, seed=1), _rand(2, 3, 4, seed=2), 0.8)


# ---------------------------------------------------------------------------
# how they are called


def test_equal_inputs_give_equal_bits(gpu):
    x = _rand(300, 5003, seed=10, dtype=BF).to(gpu).requires_grad_()
    ids, t_ids, teacher = _ints(0, 5003, 300, seed=1).to(gpu), _ints(0, 40, 300, 64, seed=2).to(gpu), _rand(300, 64, seed=3).to(gpu)

    def once():
        o = da.fused_token_logprobs(x, ids, top_k=40)
        loss = da.fused_distillation_loss(x, t_ids, teacher, 2.0)
        d = torch.autograd.grad(o.logprobs.sum() + o.entropy.sum() + o.top_logprobs.sum() + loss.sum(), x)
        return [*o, loss, *d]

    first = once()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))


def test_a_forward_without_gradients_is_the_same(gpu):
    x = _rand(5, 2003, seed=11).to(gpu)
    ids = _ints(0, 2003, 5, seed=1).to(gpu)
    a = da.fused_token_logprobs(x, ids, top_k=4)
    b = da.fused_token_logprobs(x.clone().requires_grad_(), ids, top_k=4)
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and not a.entropy.requires_grad
    assert b.logprobs.requires_grad and b.entropy.requires_grad and b.top_logprobs.requires_grad and not b.top_ids.requires_grad
    c = da.fused_token_logprobs(x, ids.to(torch.int32))
    assert torch.equal(a.logprobs, c.logprobs) and c.top_ids is None


def test_gradients_of_single_results(gpu):
    """Each result's gradient by itself, and their sum."""
    x = _rand(4, 1501, seed=12).to(gpu).requires_grad_()
    ids = _ints(0, 1501, 4, seed=1).to(gpu)
    o = da.fused_token_logprobs(x, ids, top_k=3, temperature=1.4)
    parts = [torch.autograd.grad(t.sum(), x, retain_graph=True)[0] for t in (o.logprobs, o.entropy, o.logsumexp, o.top_logprobs)]
    (whole,) = torch.autograd.grad(o.logprobs.sum() + o.entropy.sum() + o.logsumexp.sum() + o.top_logprobs.sum(), x)
    total = sum(p.double() for p in parts)
    # each of five evaluations of p (a + b ln p) + c to 260 u of terms below 40
    assert (whole.double() - total).abs().max() <= 5 * 260 * U * 40 * max(p.abs().max().item() for p in parts)


def test_streams(gpu):
    x = _rand(64, 20011, seed=13, dtype=BF).to(gpu)
    ids = _ints(0, 20011, 64, seed=1).to(gpu)
    want = da.fused_token_logprobs(x, ids, top_k=8)
    torch.cuda.synchronize()
    outs = []
    for _ in range(3):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(da.fused_token_logprobs(x, ids, top_k=8))
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, want))


def test_capture_is_refused(gpu):
    x = _rand(2, 100, seed=1).to(gpu)
    ids = torch.zeros(2, dtype=torch.int64, device=gpu)
    da.fused_token_logprobs(x, ids)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    errors = []
    with torch.cuda.stream(s):
        graph.capture_begin()
        for call in (lambda: da.fused_token_logprobs(x, ids), lambda: da.fused_distillation_loss(x, ids[:, None], x[:, :1])):
            try:
                call()
            except RuntimeError as e:
                errors.append(str(e))
        y = x + 1  # noqa: F841 (a capture of nothing is an error)
        graph.capture_end()
    assert len(errors) == 2 and all("captur" in e for e in errors)


def test_no_second_derivative(gpu):
    x = _rand(2, 100, seed=1).to(gpu).requires_grad_()
    ids = torch.tensor([1, 2], device=gpu)
    for y in (da.fused_token_logprobs(x, ids).logprobs, da.fused_distillation_loss(x, ids[:, None], x[:, :1].detach())):
        (d,) = torch.autograd.grad(y.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="twice"):
            d.sum().backward()


def test_refusals(gpu):
    x, ids = _rand(3, 8, seed=1).to(gpu), torch.tensor([1, 2, 3], device=gpu)
    t_ids, teacher = ids[:, None], torch.zeros(3, 1, device=gpu)
    f, d = da.fused_token_logprobs, da.fused_distillation_loss
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        f(x.half(), ids)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        d(x, t_ids, teacher.half())
    with pytest.raises(TypeError, match="int64 or int32"):
        f(x, ids.float())
    for k in (-1, 9):
        with pytest.raises(ValueError, match="top_k"):
            f(x, ids, top_k=k)
    with pytest.raises(ValueError, match="at most 524288"):
        f(torch.zeros(1, (1 << 19) + 1, device=gpu), top_k=1)
    with pytest.raises(ValueError, match="shape"):
        f(x, ids[:2])
    with pytest.raises(ValueError, match="on cpu"):
        f(x, ids.cpu())
    with pytest.raises(ValueError, match="at least one column"):
        f(x[:, :0], ids)
    with pytest.raises(ValueError, match="K in"):
        d(x, torch.zeros(3, 129, dtype=torch.int64, device=gpu), torch.zeros(3, 129, device=gpu))
    with pytest.raises(ValueError, match="K in"):
        d(x, ids, teacher)
    with pytest.raises(ValueError, match="teacher_logits"):
        d(x, t_ids, teacher[:2])
    with pytest.raises(ValueError, match="teacher_lse"):
        d(x, t_ids, teacher, 1.0, torch.zeros(2, device=gpu))
    with pytest.raises(TypeError, match="float32"):
        d(x, t_ids, teacher, 1.0, torch.zeros(3, device=gpu, dtype=BF))
    with pytest.raises(ValueError, match="no gradient for the teacher"):
        d(x, t_ids, teacher.clone().requires_grad_())


def test_compiled_calls(gpu):
    """Under torch.compile the registered ops run, with their autograd."""
    x = _rand(6, 700, seed=14, dtype=BF).to(gpu).requires_grad_()
    ids, t_ids, teacher = _ints(0, 700, 6, seed=1).to(gpu), _ints(0, 700, 6, 5, seed=2).to(gpu), _rand(6, 5, seed=3).to(gpu)

    def step(x):
        o = da.fused_token_logprobs(x, ids, top_k=3)
        return o.logprobs.sum() + o.entropy.mean() + o.top_logprobs.sum(), da.fused_distillation_loss(x, t_ids, teacher, 2.0).sum(), o.top_ids

    a, b, tops = torch.compile(step)(x)
    (d,) = torch.autograd.grad(a + b, x)
    a2, b2, tops2 = step(x)
    (d2,) = torch.autograd.grad(a2 + b2, x)
    assert torch.equal(tops, tops2)
    # sums of 18 and of 6 float32 numbers in another order
    assert abs(a.item() - a2.item()) <= 40 * U * 18 * 20 and abs(b.item() - b2.item()) <= 40 * U * 6 * 100
    # two bf16 gradients are added, each off by half a step, and rounded again
    scale = d2.float().abs() + 1e-3
    assert ((d.float() - d2.float()).abs() <= 3 * 2.0**-8 * scale).all()


def test_ops_pass_opcheck(gpu):
    x = _rand(2, 30, seed=1).to(gpu).requires_grad_()
    ids = torch.tensor([1, 2], device=gpu)
    torch.library.opcheck(torch.ops.deberta_amd.token_logprobs, (x, ids, 3, 1.5, -100), test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(torch.ops.deberta_amd.token_logprobs, (x, None, 0, 1.0, -100), test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(torch.ops.deberta_amd.distill_loss, (x, ids[:, None], x.detach()[:, :1], None, 2.0),
                          test_utils=("test_schema", "test_faketensor"))


def test_training_step_of_teacher_and_student(gpu):
    """As they are used together: the teacher's pass stores its best tokens, the
    student learns from them and from the labels through one head; its gradients
    are those of the same step in torch operations."""
    torch.manual_seed(0)
    C, V, N = 64, 1500, 40
    config = SimpleNamespace(hidden_size=C, vocab_size=V, layer_norm_eps=1e-7)
    head, weight = da.FusedMLMHead(config).to(gpu), torch.nn.Parameter(_rand(V, C, seed=1, std=0.1).to(gpu))
    hidden = _rand(N, C, seed=2, std=1.0).to(gpu).requires_grad_()
    teacher = da.fused_token_logprobs(_rand(N, V, seed=3, dtype=BF).to(gpu), top_k=32, temperature=2.0)
    assert not teacher.top_logprobs.requires_grad
    labels = _ints(0, V, N, seed=4).masked_fill_(_ints(0, 3, N, seed=5) == 0, -100).to(gpu)
    loss, rows = head.forward_loss(hidden, weight, labels)
    loss = loss + head.forward_distillation(hidden, weight, teacher.top_ids, teacher.top_logprobs, 1.5)
    leaves = [hidden, weight, *head.parameters()]
    got = torch.autograd.grad(loss, leaves)

    F = torch.nn.functional
    copies = [t.detach().cpu().double().requires_grad_() for t in leaves]
    h, w = copies[:2]
    named = dict(zip([n for n, _ in head.named_parameters()], copies[2:]))
    z = F.layer_norm(F.gelu(F.linear(h, named["dense.weight"], named["dense.bias"])), (C,), named["LayerNorm.weight"], named["LayerNorm.bias"], 1e-7)
    z = F.linear(z, w, named["bias"])
    logp = ov.log_probs(z, 1.5)
    q, log_q = ov.teacher_probs(teacher.top_ids.cpu(), teacher.top_logprobs.cpu(), 1.5)
    want = F.cross_entropy(z, labels.cpu()) + ov.distillation(logp, teacher.top_ids.cpu(), q, log_q, 1.5).mean()
    # float32 products of 64 and 1500 terms: 1e-4 of a gradient's norm holds their roundings many times over
    assert abs(loss.item() - want.item()) <= 1e-4 * abs(want.item())
    for a, b in zip(got, torch.autograd.grad(want, copies)):
        assert (a.cpu().double() - b).norm() <= 1e-4 * b.norm()
    best = head.predict(hidden, weight, top_k=4)
    assert torch.equal(best.top_ids[:, 0], head(hidden, weight).argmax(-1))


@pytest.mark.parametrize("autocast", [False, True], ids=["bf16", "autocast"])
def test_training_step_in_bf16(autocast, gpu):
    """The same step with a head in bf16, and with one in float32 under bf16 autocast:
    bf16 logits go into the operators, gradients have their leaves' types.  Against
    float64 from the same values: the dense product, its bias, GELU, LayerNorm, the
    vocabulary's product and its bias round to bf16 forward, at most as many products and
    sums backward, and a logit's error of six half steps of the largest logit (here below
    5) moves p by 6 * 5 half steps.  All one way, with a factor of two for the GELU's
    slope: logits off by 12 half steps of the largest, a gradient by (12 + 12 + 30) 2^-8 of
    its norm."""
    torch.manual_seed(0)
    C, V, N, T = 64, 1500, 160, 1.5
    config = SimpleNamespace(hidden_size=C, vocab_size=V, layer_norm_eps=1e-7)
    kept = FP if autocast else BF
    head, weight = da.FusedMLMHead(config).to(gpu, kept), torch.nn.Parameter(_rand(V, C, seed=1, std=0.1, dtype=kept).to(gpu))
    with torch.no_grad():
        head.bias.copy_(_rand(V, seed=6, std=0.1).to(gpu))
        head.dense.bias.copy_(_rand(C, seed=7, std=0.1).to(gpu))
    hidden = _rand(N, C, seed=2, std=1.0, dtype=kept).to(gpu).requires_grad_()
    labels = _ints(0, V, N, seed=4).masked_fill_(_ints(0, 3, N, seed=5) == 0, -100).to(gpu)
    teacher = da.fused_token_logprobs(_rand(N, V, seed=3, dtype=BF).to(gpu), top_k=32)
    with torch.autocast("cuda", dtype=BF, enabled=autocast):
        logits = head(hidden, weight)
        mlm, rows = head.forward_loss(hidden, weight, labels)
        distil = head.forward_distillation(hidden, weight, teacher.top_ids, teacher.top_logprobs, T)
        best = head.predict(hidden, weight, top_k=4)
    assert logits.dtype == BF and mlm.dtype == distil.dtype == rows.entropy.dtype == FP
    # the operators read these logits
    _check_logprobs(logits.detach(), labels.cpu(), 4)
    assert torch.equal(best.top_ids, da.fused_token_logprobs(logits.detach(), top_k=4).top_ids)
    leaves = [hidden, weight, *head.parameters()]
    got = torch.autograd.grad(mlm + distil, leaves)

    F = torch.nn.functional
    copies = [t.detach().cpu().double().requires_grad_() for t in leaves]
    named = dict(zip([n for n, _ in head.named_parameters()], copies[2:]))
    z = F.layer_norm(F.gelu(F.linear(copies[0], named["dense.weight"], named["dense.bias"])), (C,), named["LayerNorm.weight"], named["LayerNorm.bias"], 1e-7)
    z = F.linear(z, copies[1], named["bias"])
    h, most = 2.0**-8, z.abs().max().item()
    assert most < 5
    assert (logits.detach().cpu().double() - z.detach()).abs().max() <= 12 * h * most
    logp = ov.log_probs(z, T)
    q, log_q = ov.teacher_probs(teacher.top_ids.cpu(), teacher.top_logprobs.cpu(), T)
    want = [F.cross_entropy(z, labels.cpu()), ov.distillation(logp, teacher.top_ids.cpu(), q, log_q, T).mean()]
    # a log probability moves by twice what the logits are off by (over T, times T^2)
    assert abs(mlm.item() - want[0].item()) <= 24 * h * most and abs(distil.item() - want[1].item()) <= 24 * h * most * T
    for leaf, a, b in zip(leaves, got, torch.autograd.grad(sum(want), copies)):
        assert a.dtype == leaf.dtype
        assert (a.cpu().double() - b).norm() <= 54 * h * b.norm(), leaf.shape
