"""Calls of the hidden-state operators on the GPU that need care on the way to
the kernels: tensors without memory of their own, wrapped and traced calls,
views with a pending sign, more rows than one launch holds, teams that take
several rows.  Tolerances as in test_gpu_hidden.py."""

from __future__ import annotations

import sys

import pytest
import torch

import deberta_amd as da
from deberta_amd import hidden
from oracle import hidden as oh
from tests._hidden import Wrapper
from tests.test_gpu_hidden import _rms_case

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float32
U = 2.0**-24
EPS = 1e-6
SEED = 0x3_1234_5678_9ABC


def _rand(*shape, seed, dtype=FP):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def test_wrapped_arguments_count(gpu):
    """A wrapper tensor as bias, residual, weight or ids gives what the plain
    tensor in it gives."""
    x, b, r, w = (_rand(*s, seed=k).to(gpu) for k, s in enumerate(((5, 24), (24,), (5, 24), (24,))))
    ids = torch.tensor([3, 0, 4], device=gpu)
    for call in (
        lambda b, r, w: da.fused_dropout(x, 0.5, bias=b, res=r, seed=SEED),
        lambda b, r, w: da.fused_add_rms_norm(x, w, bias=b, res=r)[0],
        lambda b, r, w: da.fused_add_rms_norm_fp8(x, w, bias=b, res=r)[0].view(torch.uint8),
    ):
        want = call(b, r, w)
        for k in range(3):
            args = [Wrapper(t) if i == k else t for i, t in enumerate((b, r, w))]
            assert torch.equal(call(*args), want)
    assert torch.equal(da.fused_embedding(Wrapper(ids), x), x[ids])


def test_tensors_without_memory_are_refused(gpu):
    """A plain tensor whose storage was freed has a null address, which must
    not read as an argument that was not given."""
    x, w = _rand(5, 24, seed=1).to(gpu), torch.ones(24, device=gpu)
    ext, seed = hidden._ext(), torch.tensor([SEED])

    def freed(*shape):
        t = torch.ones(shape, device=gpu)
        t.untyped_storage().resize_(0)
        return t

    row, vec = freed(5, 24), freed(24)
    shifted = torch.ones(30, device=gpu)
    part = shifted[6:]
    shifted.untyped_storage().resize_(0)  # its address alone is not null
    for call in (
        lambda: da.fused_dropout(x, 0.5, bias=vec, seed=SEED),
        lambda: da.fused_dropout(x, 0.5, bias=part, seed=SEED),
        lambda: da.fused_dropout(x, 0.5, res=row, seed=SEED),
        lambda: da.fused_dropout(row, 0.5, seed=SEED),
        lambda: da.fused_rms_norm(row, w),
        lambda: da.fused_rms_norm(x, vec),
        lambda: da.fused_add_rms_norm(x, w, bias=vec),
        lambda: da.fused_add_rms_norm(x, w, res=row),
        lambda: da.fused_add_rms_norm_fp8(x, w, res=row),
        lambda: da.fused_embedding(torch.zeros(2, dtype=torch.int64, device=gpu), row),
        lambda: ext.dropout_bwd(row, FP, FP, 100, seed),
        lambda: ext.rms_bwd(x, row, x, None, None, w, torch.ones(5, device=gpu), 0, None),
        lambda: ext.dropout_fwd(x, Wrapper(w), None, 100, seed),
        lambda: ext.dropout_fwd(x, None, None, 100, Wrapper(seed)),
    ):
        with pytest.raises(ValueError, match="no memory"):
            call()


class _Path(torch.nn.Module):
    def __init__(self, grad):
        super().__init__()
        for k, (name, shape) in enumerate((("table", (40, 64)), ("w", (64,)), ("b", (64,)))):
            setattr(self, name, torch.nn.Parameter(_rand(*shape, seed=k), requires_grad=grad))

    def forward(self, ids, res):
        e = da.fused_embedding(ids, self.table, padding_idx=0, scale=2.0)
        e = da.fused_dropout(e, 0.25, seed=SEED)
        return da.fused_add_rms_norm(e, self.w, bias=self.b, res=res, dropout_p=0.5, seed=SEED)


class _Eight(_Path):
    def forward(self, r):
        return da.fused_add_rms_norm_fp8(r, self.w, res=r)


def _traced(m, *inputs):
    """m's trace; memory freed afterwards holds NaN, which a result that is
    only allocated would return."""
    t = torch.jit.trace(m, inputs, check_trace=False)
    junk = [torch.full((3, 5, 64), float("nan"), device=inputs[0].device) for _ in range(8)]
    del junk
    return t


@pytest.mark.parametrize("grad", [False, True])
def test_traced_calls_compute(grad, gpu):
    """A traced module runs the kernels again on new inputs: equal to the
    eager calls, with gradients."""
    m = _Path(grad).to(gpu)
    ids, res = torch.randint(0, 40, (3, 5), generator=torch.Generator().manual_seed(1)).to(gpu), _rand(3, 5, 64, seed=5).to(gpu)
    traced = _traced(m, ids, res)
    ids, res = ids.flip(0), res * 2
    got, want = traced(ids, res), m(ids, res)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    if grad:
        dy = _rand(3, 5, 64, seed=6).to(gpu)
        g, h = (torch.autograd.grad(o, list(m.parameters()), (dy, dy)) for o in (got, want))
        assert all(torch.equal(a, b) for a, b in zip(g, h))


def test_traced_eight_bit_rows_compute(gpu):
    m, res = _Eight(False).to(gpu), _rand(3, 5, 64, seed=5).to(gpu)
    traced = _traced(m, res)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(traced(res * 3), m(res * 3)))


def test_a_traced_rtd_head_computes(gpu):
    from oracle import eager

    cfg = eager.make_config(hidden_size=64, num_attention_heads=4, intermediate_size=128, layer_norm_eps=1e-7, use_rmsnorm_heads=True)
    head = da.FusedRTDHead(cfg).to(gpu).eval()
    with torch.no_grad():
        h = _rand(2, 9, 64, seed=1).to(gpu)
        traced = _traced(head, h)
        assert torch.equal(traced(h * 2), head(h * 2))


def test_a_pending_sign_counts(gpu):
    """The imaginary part of a conjugated tensor is a view whose values are to
    be negated: equal to its copy in every argument and as a gradient."""
    z = torch.complex(_rand(6, 1, seed=1), _rand(6, 1, seed=2)).to(gpu)
    view = z.conj().imag  # one column: rows of stride 2 are read in place
    assert view.is_neg()
    zero = torch.zeros(1, device=gpu)
    assert torch.equal(da.fused_dropout(view, 0.0, bias=zero), view.clone())
    x, w, r = (_rand(*s, seed=k).to(gpu) for k, s in enumerate(((5, 24), (24,), (5, 24))))
    ids, neg = torch.tensor([1, 3], device=gpu), torch._neg_view
    seed = torch.tensor([SEED])
    rstd = torch.ones(5, device=gpu)
    for call in (
        lambda f: da.fused_dropout(f(x), 0.5, bias=f(w), res=f(r), seed=SEED),
        lambda f: da.fused_dropout(f(x.view(1, 5, 24)), 0.5, res=f(r[:1]).expand(1, 5, 24), seed=SEED),
        lambda f: da.fused_add_rms_norm(f(x), f(w), bias=f(w), res=f(r))[0],
        lambda f: da.fused_add_rms_norm_fp8(f(x), f(w), res=f(r))[0].view(torch.uint8),
        lambda f: da.fused_embedding(ids, f(x)),
        lambda f: hidden._hidden_dropout_bwd_impl(f(x), FP, FP, 100, seed)[1],
        lambda f: hidden._add_rms_norm_bwd_impl(f(x), f(r), f(r), None, None, f(w), rstd, 0, None)[0],
        lambda f: hidden._embed_bwd_impl(f(x[:2]), ids, 6, FP, -1, 1.0),
    ):
        assert torch.equal(call(neg), call(lambda t: -t))


def test_more_rows_than_one_launch_holds(gpu):
    """2^28 rows of eight columns are one more than 2^32 - 1 threads; the keep
    bits show that a row keeps its number.  A norm of eight values: 8 squares,
    8 additions, a division, a root and two products, under 24 half steps."""
    C, N = 8, (1 << 28) + 37
    rows = [0, 17, (1 << 28) - 17, (1 << 28) - 16, (1 << 28) - 1, 1 << 28, N - 2, N - 1]
    some, one = _rand(len(rows), C, seed=1, dtype=BF), torch.ones(C, dtype=torch.float64)
    x, w = torch.zeros(N, C, dtype=BF, device=gpu), torch.ones(C, device=gpu)
    x[rows] = some.to(gpu)
    z64 = some.double() * oh.keep_mask(rows, C, 32768, SEED) * 2
    y, z = da.fused_add_rms_norm(x, w, EPS, dropout_p=0.5, seed=SEED)
    assert torch.equal(z[rows].cpu().double(), z64)
    y64 = oh.rms_norm(z64, one, EPS)
    assert ((y[rows].cpu().double() - y64).abs() <= (24 * U + 2.0**-8) * y64.abs()).all()
    y[rows] = 0
    assert not y.view(torch.int16).any()
    del y, z
    with torch.no_grad():
        q, s, _ = da.fused_add_rms_norm_fp8(x, w, EPS)
    got = q[rows].cpu().float() * s[rows].cpu()
    y64 = oh.rms_norm(some.double(), one, EPS)
    assert ((got.double() - y64).abs() <= (2.0**-4 + 32 * U) * y64.abs() + 2.0**-10 * s[rows].cpu().double()).all()
    s[rows] = 1
    assert (s == 1).all()


# rows so that every shape of team takes two or three, the last ones fewer: 16 and
# 32 lanes, one wave of one and of two chunks, four, eight and sixteen waves, with
# column sums in registers and (past 8192 columns) in LDS, whole and cut rows
@pytest.mark.parametrize("N,C", [(20011, 33), (20011, 64), (9001, 200), (9001, 201), (5001, 301), (5001, 304), (5001, 1024),
                                 (5001, 777), (2501, 1025), (1301, 2048), (600, 2500), (600, 4096), (600, 5003), (600, 8192),
                                 (600, 8193), (600, 16384)])
@pytest.mark.parametrize("xt,rt,bt", [(BF, BF, FP), (BF, FP, BF), (FP, FP, FP)])
def test_rms_teams_of_several_rows(N, C, xt, rt, bt, gpu):
    print("rms", N, C, xt, rt, file=sys.stderr, flush=True)
    _rms_case(gpu, (N, C), xt, rt, FP, bt=bt, p=0.1)


def test_transforms_of_any_argument_raise(gpu):
    """torch.func's wrappers in another argument than the first: an error, not
    a result without them."""
    import torch.autograd.forward_ad as fwAD

    x, w, r = (_rand(*s, seed=k).to(gpu) for k, s in enumerate(((5, 24), (24,), (5, 24))))
    for call, t in (
        (lambda b: da.fused_dropout(x, 0.5, bias=b, seed=SEED), w),
        (lambda b: da.fused_dropout(x, 0.5, res=b, seed=SEED), r),
        (lambda b: da.fused_rms_norm(x, b), w),
        (lambda b: da.fused_add_rms_norm(x, w, bias=b)[0], w),
        (lambda b: da.fused_add_rms_norm(x, w, res=b)[0], r),
    ):
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(t.expand(3, *t.shape))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda v: call(v).sum())(t)
        with fwAD.dual_level(), pytest.raises(RuntimeError):
            call(fwAD.make_dual(t, torch.ones_like(t)))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda i: da.fused_embedding(i, x))(torch.zeros(3, 2, dtype=torch.int64, device=gpu))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda v: da.fused_add_rms_norm_fp8(x, v)[1])(w.expand(3, 24))


@pytest.mark.parametrize("N,C,group", [(2000, 1024, None), (700, 2048, 128), (900, 1023, None)])
def test_eight_bit_bytes_are_the_definitions(N, C, group, gpu):
    """Every byte is the float64 definition's rounded once, or its neighbour
    where the exact value lies on the border between the two as far as float32
    can tell: by twice y's error over the scale (that of the value, and of the
    scale at the group's largest) and four half steps of the value."""
    G = group or C
    x, res = _rand(N, C, seed=1, dtype=BF).to(gpu), _rand(N, C, seed=2, dtype=BF).to(gpu)
    w = (1 + 0.2 * _rand(C, seed=3)).to(gpu)
    with torch.no_grad():
        q, _, _ = da.fused_add_rms_norm_fp8(x, w, EPS, res=res, group_size=group)
        again = da.fused_add_rms_norm_fp8(x, w, EPS, res=res, group_size=group)[0]
    assert torch.equal(q.view(torch.uint8), again.view(torch.uint8))
    x64, r64, w64 = x.cpu().double(), res.cpu().double(), w.cpu().double()
    z64 = x64 + r64
    exact, s64 = oh.quantise(oh.rms_norm(z64, w64, EPS), G)
    got, want = q.float().cpu().double(), exact.float().to(torch.float8_e4m3fn).float().double()
    r = 1 / torch.sqrt(z64.square().mean(-1, keepdim=True) + EPS)
    e = w64.abs() * 96 * U * ((z64 * r).abs() + (x64.abs() + r64.abs()) * r)  # of y, as in test_gpu_hidden.py
    top = e.unflatten(-1, (C // G, G)).amax(-1).repeat_interleave(G, -1)
    s_el = s64.repeat_interleave(G, -1)
    tol = e / s_el + top / s_el * exact.abs() / 448 + 4 * U * exact.abs()
    other = got != want
    assert ((exact - (got + want) / 2).abs() <= tol)[other].all()
    assert ((got - want).abs() <= 2.0**-3 * torch.maximum(got.abs(), want.abs()).clamp(min=2.0**-6))[other].all()
