"""The operators on hidden states on the GPU against their float64 definitions
(oracle/hidden.py) on the same inputs: outputs and every gradient, over
widths, row counts, strides, types, masks and the cases that go wrong first
(no rows, one column, dropped infinities, ids outside the table, tokens that
cross the sums' borders, offsets past 32 bits).

Tolerances, with u = 2^-24 the half step of float32 and h that of the output's
type (bf16 2^-8, fp32 2^-24), element by element:

  dropout  y = (x + b) s + r takes three roundings and s one:  4 u M + h |y|,
           M = |x + b| s + |r|;  dx: 2 u |dx| + h |dx|;  dbias, a sum of at
           most D = 400 roundings in a row (rows of a thread, of a block, of
           the blocks):  D u sum|dx| + h |dbias|
  norm     sums of a row are taken over at most 64 values in a lane, 12
           additions over lanes and waves, of squares of z (each 5 u of M):
           with A = M r (M's share of the normed row) the normed value is
           off by e = 96 u (|n| + A), y by |w| e + h |y|;
           dz = r (g - n m) + v, m = mean(g n):  128 u (r (|g| + (|n| + A)
           mean(|g| (|n| + A))) + |v|) + h |dz|;  dw, D rows:  (128 + D) u
           sum(|dy| (|n| + A)) + h |dw|
  8 bits   half a step of e4m3 (2^-4 of the value, 2^-10 of the scale where it
           is subnormal) with y's own error; the scale by y's error / 448
  embed    out: 2 u + h;  dW: at most 72 + count / 32 additions in a row:
           that many u sum|dy scale| + h |dW|
"""

from __future__ import annotations

import sys
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

import deberta_amd as da
from deberta_amd import hidden
from oracle import hidden as oh

pytestmark = pytest.mark.gpu

U = 2.0**-24
BF, FP = torch.bfloat16, torch.float32
EPS = 1e-6
SEED = 0x3_1234_5678_9ABC
D = 400


def _say(*a):
    print(*a, file=sys.stderr, flush=True)


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _rand(*shape, seed, dtype, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def _within(name, got, want, tol):
    got, want = got.detach().double().cpu(), want.detach().double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.equal(got.isnan(), want.isnan()), name
    over = ((got - want).abs() - tol).nan_to_num(0.0)
    assert over.max().item() <= 0 if over.numel() else True, (name, over.max().item(), (got - want).abs().max().item())


def _leaf(t, gpu):
    return None if t is None else t.to(gpu).requires_grad_()


def _d(t):
    return None if t is None else t.double()


# ---------------------------------------------------------------------------
# dropout


def _dropout_case(gpu, shape, xt, rt, bt, p, seed=1, x=None, res=None, dy=None):
    """x, res and dy may be given as GPU views; else contiguous random ones."""
    C = shape[-1]
    t = round(p * 65536)
    s = 65536.0 / (65536 - t) if t < 65536 else 0.0
    x = _rand(*shape, seed=seed, dtype=xt).to(gpu) if x is None else x
    if res is None and rt is not None:
        res = _rand(*shape, seed=seed + 1, dtype=rt).to(gpu)
    bias = _rand(C, seed=seed + 2, dtype=bt).to(gpu) if bt is not None else None
    zt = xt if res is None else torch.promote_types(xt, res.dtype)
    dy = _rand(*shape, seed=seed + 3, dtype=zt).to(gpu) if dy is None else dy
    leaves = [v.detach().requires_grad_() if v is not None else None for v in (x, bias, res)]
    y = da.fused_dropout(leaves[0], p, bias=leaves[1], res=leaves[2], seed=SEED)
    assert y.dtype == zt
    grads = iter(torch.autograd.grad(y, [v for v in leaves if v is not None], dy))
    x64, b64, r64 = (None if v is None else v.cpu().double().requires_grad_() for v in (x, bias, res))
    ref = oh.dropout_add(x64, b64, r64, t, SEED)
    want = iter(torch.autograd.grad(ref, [v for v in (x64, b64, r64) if v is not None], dy.cpu().double()))
    M = (x64 if bias is None else x64 + b64).detach().abs() * s + (0 if res is None else r64.detach().abs())
    _within("y", y, ref, 4 * U * M + _half(zt) * ref.detach().abs())
    wx = next(want)
    _within("dx", next(grads), wx, (2 * U + _half(xt)) * wx.abs())
    if bias is not None:
        wb = next(want)
        total = wx.abs().reshape(-1, C).sum(0)
        _within("dbias", next(grads), wb, D * U * total + _half(bt) * wb.abs())
    if res is not None:
        wr = next(want)
        _within("dres", next(grads), wr, _half(res.dtype) * wr.abs())


@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (3, 8), (5, 9), (2, 5, 17), (257, 64), (33, 768), (4, 63, 513), (7, 2049),
                                   (3, 5000), (1300, 24)], ids=str)
def test_dropout(shape, gpu):
    _say("dropout", shape)
    _dropout_case(gpu, shape, BF, BF, FP, 0.1)
    _dropout_case(gpu, shape, FP, None, None, 0.5)


@pytest.mark.parametrize("xt,rt,bt", [(BF, None, None), (BF, FP, BF), (FP, BF, FP), (FP, FP, BF), (BF, BF, BF), (FP, None, FP)])
@pytest.mark.parametrize("p", [0.0, 0.25, 1.0])
def test_dropout_types(xt, rt, bt, p, gpu):
    if p == 0.0 and rt is None and bt is None:
        x = torch.ones(3, 8, device=gpu)
        assert da.fused_dropout(x, p) is x
        return
    _dropout_case(gpu, (6, 11, 100), xt, rt, bt, p)


def test_dropout_strides(gpu):
    """Columns of a wider tensor from an odd offset, a transposed batch, and a
    residual broadcast along the sequence."""
    big = _rand(40, 131, seed=9, dtype=BF).to(gpu)
    _dropout_case(gpu, (40, 77), BF, BF, FP, 0.3, x=big[:, 3:80], dy=_rand(40, 131, seed=8, dtype=BF).to(gpu)[:, 1:78])
    t = _rand(6, 4, 50, seed=7, dtype=FP).to(gpu).transpose(0, 1)
    _dropout_case(gpu, (4, 6, 50), FP, None, None, 0.3, x=t, res=t)
    head = _rand(4, 1, 65, seed=6, dtype=BF).to(gpu)
    _dropout_case(gpu, (4, 9, 65), BF, None, FP, 0.3, res=head.expand(4, 9, 65))
    # columns with a stride of their own are copied
    _dropout_case(gpu, (5, 33), FP, None, None, 0.3, x=_rand(33, 5, seed=5, dtype=FP).to(gpu).t())
    # one row repeated
    _dropout_case(gpu, (9, 33), FP, FP, None, 0.3, x=_rand(1, 33, seed=4, dtype=FP).to(gpu).expand(9, 33))


def test_dropout_masks_infinities_and_nan(gpu):
    """A dropped NaN or infinity leaves 0, forward and backward; a kept one
    passes."""
    keep = oh.keep_mask(16, 96, 32768, SEED).to(gpu)
    x = torch.ones(16, 96, device=gpu)
    for bad in (float("nan"), float("inf"), -float("inf"), torch.finfo(FP).min):
        v = torch.where(keep, x, torch.tensor(bad, device=gpu)).requires_grad_()
        y = da.fused_dropout(v, 0.5, seed=SEED)
        assert torch.equal(y, keep * 2.0)
        (dx,) = torch.autograd.grad(y, v, torch.where(keep, x, torch.tensor(bad, device=gpu)))
        assert torch.equal(dx, keep * 2.0)
    v = x.clone()
    r, c = keep.nonzero()[0].tolist()
    v[r, c] = float("nan")
    y = da.fused_dropout(v, 0.5, seed=SEED)
    assert y.isnan().sum().item() == 1 and y[r, c].isnan()


def test_dropout_seeds_and_the_cpu_path(gpu):
    x = torch.ones(64, 768, device=gpu)
    torch.manual_seed(3)
    a, b = da.fused_dropout(x, 0.1), da.fused_dropout(x, 0.1)
    assert not torch.equal(a, b)
    torch.manual_seed(3)
    assert torch.equal(a, da.fused_dropout(x, 0.1))
    assert torch.equal(da.fused_dropout(x, 0.1, seed=SEED).cpu(), da.fused_dropout(x.cpu(), 0.1, seed=SEED))
    assert torch.equal(da.fused_dropout(x, 0.1, seed=SEED) != 0, da.hidden_keep_mask(64, 768, 0.1, SEED, gpu))


def test_no_rows(gpu):
    x, w = torch.randn(0, 8, device=gpu, requires_grad=True), torch.ones(8, device=gpu, requires_grad=True)
    b = torch.ones(8, device=gpu, requires_grad=True)
    y = da.fused_dropout(x, 0.5, bias=b)
    gx, gb = torch.autograd.grad(y.sum(), (x, b))
    assert y.shape == (0, 8) and gx.shape == (0, 8) and (gb == 0).all()
    y, z = da.fused_add_rms_norm(x, w, res=torch.randn(0, 8, device=gpu))
    gx, gw = torch.autograd.grad(y.sum() + z.sum(), (x, w))
    assert gx.shape == (0, 8) and (gw == 0).all()
    with torch.no_grad():
        q, s, _ = da.fused_add_rms_norm_fp8(x, w)
    assert q.shape == (0, 8) and s.shape == (0, 1)
    table = torch.randn(5, 8, device=gpu, requires_grad=True)
    y = da.fused_embedding(torch.zeros(0, 3, dtype=torch.int64, device=gpu), table)
    (g,) = torch.autograd.grad(y.sum(), table)
    assert y.shape == (0, 3, 8) and (g == 0).all()


# ---------------------------------------------------------------------------
# RMS norm


def _rms_case(gpu, shape, xt=BF, rt=BF, wt=FP, bt=None, p=0.0, yt=None, use=("y", "z"), x=None, res=None, std=1.0, eps=EPS):
    C = shape[-1]
    t = round(p * 65536)
    x = _rand(*shape, seed=1, dtype=xt, std=std).to(gpu) if x is None else x
    if res is None and rt is not None:
        res = _rand(*shape, seed=2, dtype=rt, std=std).to(gpu)
    w = (1 + 0.3 * _rand(C, seed=3, dtype=FP)).to(wt).to(gpu)
    bias = _rand(C, seed=4, dtype=bt).to(gpu) if bt is not None else None
    zt = xt if res is None else torch.promote_types(xt, res.dtype)
    yt = zt if yt is None else yt
    dy, dz = _rand(*shape, seed=5, dtype=yt), _rand(*shape, seed=6, dtype=zt)
    leaves = [None if v is None else v.detach().requires_grad_() for v in (x, w, bias, res)]
    y, z = da.fused_add_rms_norm(leaves[0], leaves[1], eps, bias=leaves[2], res=leaves[3], dropout_p=p, seed=SEED if t else None,
                                 out_dtype=yt)
    assert y.dtype == yt and z.dtype == zt
    outs = [o for o, n in ((y, "y"), (z, "z")) if n in use]
    live = [v for v in leaves if v is not None]
    got = torch.autograd.grad(outs, live, [g.to(gpu) for g, n in ((dy, "y"), (dz, "z")) if n in use], allow_unused=True)

    ref = [None if v is None else v.detach().cpu().double().requires_grad_() for v in (x, w, bias, res)]
    z64 = oh.dropout_add(ref[0], ref[2], ref[3], t, SEED)
    y64 = oh.rms_norm(z64, ref[1], eps)
    outs = [o for o, n in ((y64, "y"), (z64, "z")) if n in use]
    want = torch.autograd.grad(outs, [v for v in ref if v is not None], [g.double() for g, n in ((dy, "y"), (dz, "z")) if n in use],
                               allow_unused=True)
    with torch.no_grad():
        s = 65536.0 / (65536 - t) if t < 65536 else 0.0
        M = (ref[0] if bias is None else ref[0] + ref[2]).abs() * s + (0 if res is None else ref[3].abs())
        r = 1 / torch.sqrt(z64.square().mean(-1, keepdim=True) + eps)
        n, A, w64 = (z64 * r).abs(), M * r, ref[1].abs()
        _within("z", z, z64, 4 * U * M + _half(zt) * z64.abs())
        _within("y", y, y64, w64 * 96 * U * (n + A) + _half(yt) * y64.abs())
        g = dy.double().abs() * w64 if "y" in use else torch.zeros_like(n)
        up = dz.double().abs() if "z" in use else torch.zeros_like(n)
        dz_tol = 128 * U * (r * (g + (n + A) * (g * (n + A)).mean(-1, keepdim=True)) + up)
        names = [k for k, v in zip(("dx", "dw", "dbias", "dres"), leaves) if v is not None]
        for name, a, b, leaf in zip(names, got, want, live):
            if b is None:
                b = torch.zeros(leaf.shape, dtype=torch.float64)
            if a is None:
                a = torch.zeros_like(leaf)
            assert a.dtype == leaf.dtype
            if name == "dx":
                tol = dz_tol * max(s, 1.0) + 2 * U * b.abs()
                if res is None and bias is None and not t and len(use) == 2:
                    # z is x itself: autograd adds its gradient v to the norm's part b - v, which the kernel
                    # has rounded to x's type, and rounds the sum: h |b - v| beside h |b|
                    tol = tol + _half(xt) * (b - dz.double()).abs()
            elif name == "dres":
                tol = dz_tol
            elif name == "dw":
                tol = (128 + D) * U * (dy.double().abs() * (n + A)).reshape(-1, C).sum(0)
            else:
                total = (want[0].abs() if want[0] is not None else torch.zeros_like(n)).reshape(-1, C).sum(0)
                tol = D * U * total + (dz_tol * max(s, 1.0)).reshape(-1, C).sum(0)
            _within(name, a, b, tol + _half(leaf.dtype) * b.abs())


WIDTHS = [1, 7, 8, 64, 511, 512, 513, 768, 1024, 1025, 2048, 2500, 4096, 5003, 8192, 8193, 16384]


@pytest.mark.parametrize("C", WIDTHS)
def test_rms_widths(C, gpu):
    _say("rms", C)
    _rms_case(gpu, (5, C), BF, BF, FP, bt=FP, p=0.1)
    _rms_case(gpu, (3, C), FP, None, FP)


@pytest.mark.parametrize("rows", [(1,), (3,), (4, 33), (1025,), (4100,)], ids=str)
def test_rms_rows(rows, gpu):
    _say("rms rows", rows)
    _rms_case(gpu, (*rows, 768), BF, FP, FP, bt=BF, p=0.2)
    _rms_case(gpu, (*rows, 40), FP, FP, BF)
    _rms_case(gpu, (*rows, 1032), BF, BF, BF, bt=FP)


@pytest.mark.parametrize("xt", [BF, FP])
@pytest.mark.parametrize("rt", [None, BF, FP])
@pytest.mark.parametrize("yt", [BF, FP])
@pytest.mark.parametrize("p,bt", [(0.0, None), (0.0, FP), (0.3, None), (0.3, BF)])
def test_rms_types(xt, rt, yt, p, bt, gpu):
    _rms_case(gpu, (2, 9, 200), xt, rt, BF, bt=bt, p=p, yt=yt)


@pytest.mark.parametrize("use", [("y",), ("z",)])
@pytest.mark.parametrize("p", [0.0, 0.5])
def test_rms_one_output_used(use, p, gpu):
    _rms_case(gpu, (6, 300), BF, BF, FP, bt=FP, p=p, use=use)


def test_rms_strides(gpu):
    big = _rand(40, 1331, seed=9, dtype=BF).to(gpu)
    _rms_case(gpu, (40, 777), BF, BF, FP, p=0.1, x=big[:, 5:782])
    head = _rand(4, 1, 130, seed=6, dtype=FP).to(gpu)
    _rms_case(gpu, (4, 9, 130), FP, None, FP, res=head.expand(4, 9, 130))
    t = _rand(6, 4, 500, seed=7, dtype=FP).to(gpu).transpose(0, 1)
    _rms_case(gpu, (4, 6, 500), FP, None, FP, x=t, res=t)
    _rms_case(gpu, (2, 3, 4, 56), BF, BF, BF, bt=BF)
    _rms_case(gpu, (56,), BF, BF, BF)


def test_rms_rows_of_zeros_and_cancelling_sums(gpu):
    """Rows of zeros have the norm 0 (their gradient goes by 1 / sqrt(eps));
    rows whose residual cancels x leave the small difference."""
    x = _rand(6, 96, seed=1, dtype=FP).to(gpu)
    x[2] = 0
    _rms_case(gpu, (6, 96), FP, None, FP, x=x, eps=1e-2)
    y, z = da.fused_add_rms_norm(x, torch.ones(96, device=gpu), res=-x)
    assert (y == 0).all() and (z == 0).all()
    y = da.fused_rms_norm(x * 1e-18, torch.ones(96, device=gpu), eps=0.0)
    assert y[2].isnan().all()  # 0 / 0 without an eps
    _rms_case(gpu, (6, 96), FP, None, FP, std=1e3)
    _rms_case(gpu, (6, 96), BF, BF, FP, std=1e-3, eps=1e-6)


def test_rms_nan_and_infinity_stay_in_their_rows(gpu):
    x = _rand(8, 600, seed=1, dtype=FP).to(gpu)
    x[3, 17], x[5, 599] = float("nan"), float("inf")
    clean = [0, 1, 2, 4, 6, 7]
    w = torch.ones(600, device=gpu)
    y = da.fused_rms_norm(x, w)
    assert y[3].isnan().all() and y[5, 599].isnan() and y[clean].isfinite().all()
    assert torch.equal(y[clean], da.fused_rms_norm(x[clean], w))


def test_rms_differences(gpu):
    """The gradient along a direction against differences of the kernel's own
    forward: L(x + h d) - L(x - h d) over 2 h, h = 2^-6.  The third derivative
    of a unit-scaled norm along a unit-scaled direction is below 20, so the
    formula's error is under 20 h^2 / 6 a value; the roundings of y (below 8)
    add 96 u 8 / h.  Both over 3 * 50 values of |dy| < 4."""
    h = 2.0**-6
    x, res, d = (_rand(3, 50, seed=k, dtype=FP).to(gpu) for k in (1, 2, 3))
    dy, dz = (_rand(3, 50, seed=k, dtype=FP).to(gpu) for k in (4, 5))
    w = torch.ones(50, device=gpu)

    def f(v):
        y, z = da.fused_add_rms_norm(v, w, EPS, res=res, dropout_p=0.3, seed=SEED)
        return (y.double() * dy).sum() + (z.double() * dz).sum()

    v = x.clone().requires_grad_()
    y, z = da.fused_add_rms_norm(v, w, EPS, res=res, dropout_p=0.3, seed=SEED)
    (g,) = torch.autograd.grad((y, z), v, (dy, dz))
    got, want = (g.double() * d).sum().item(), (f(x + h * d) - f(x - h * d)).item() / (2 * h)
    assert abs(got - want) <= 150 * 4 * (20 * h * h / 6 + 96 * U * 8 / h), (got, want)


# ---------------------------------------------------------------------------
# 8 bits


@pytest.mark.parametrize("shape,group", [((1, 1), None), ((3, 7), None), ((5, 96), 32), ((4, 9, 768), None), ((4, 9, 768), 128),
                                         ((2, 1024), 512), ((3, 1025), None), ((3, 2048), 64), ((2, 4096), 256), ((5, 5003), None),
                                         ((2, 8192), 128), ((3, 16384), 512), ((2, 16383), None), ((300, 64), 64)], ids=str)
@pytest.mark.parametrize("xt,rt", [(BF, BF), (FP, None), (BF, FP), (FP, BF)])
def test_fp8(shape, group, xt, rt, gpu):
    C = shape[-1]
    x = _rand(*shape, seed=1, dtype=xt).to(gpu)
    res = _rand(*shape, seed=2, dtype=rt).to(gpu) if rt is not None else None
    w = (1 + 0.3 * _rand(C, seed=3, dtype=FP)).to(gpu)
    bias = _rand(C, seed=4, dtype=BF).to(gpu) if rt is not None else None
    with torch.no_grad():
        q, scale, z = da.fused_add_rms_norm_fp8(x, w, EPS, bias=bias, res=res, group_size=group)
        y32, z2 = da.fused_add_rms_norm(x, w, EPS, bias=bias, res=res, out_dtype=FP)
    assert torch.equal(z, z2)
    G = group or C
    assert scale.shape == (*shape[:-1], C // G) and q.shape == shape
    # the quantisation of the kernel's own float32 y: the scale and every byte
    top = y32.unflatten(-1, (C // G, G)).abs().amax(-1)
    most = torch.full_like(top, 448.0)  # a tensor: torch divides by a number through its reciprocal
    assert torch.equal(scale, top / most)
    by = (y32.unflatten(-1, (C // G, G)) * (most / top).unsqueeze(-1)).clamp(-448, 448).flatten(-2).to(torch.float8_e4m3fn)
    assert torch.equal(q.view(torch.uint8), by.view(torch.uint8))
    # and the definition in float64
    z64 = oh.dropout_add(x.cpu().double(), _d(bias.cpu()) if bias is not None else None, _d(res.cpu()) if res is not None else None, 0, 0)
    y64 = oh.rms_norm(z64, w.cpu().double(), EPS)
    s64 = oh.quantise(y64, G)[1]
    M = (x.cpu().double() if bias is None else x.cpu().double() + bias.cpu().double()).abs()
    M = M if res is None else M + res.cpu().double().abs()
    r = 1 / torch.sqrt(z64.square().mean(-1, keepdim=True) + EPS)
    e = w.cpu().double().abs() * 96 * U * ((z64 * r).abs() + M * r)
    _within("scale", scale, s64, e.unflatten(-1, (C // G, G)).amax(-1) / 448 + 2 * U * s64)
    s_el = scale.cpu().double().repeat_interleave(G, -1)
    _within("values", q.float().cpu().double() * s_el, y64, 2.0**-4 * y64.abs() * (1 + 1e-5) + 2.0**-10 * s_el + 2 * e)


def test_fp8_zeros_tiny_nan_and_infinity(gpu):
    x = _rand(8, 128, seed=1, dtype=FP).to(gpu)
    w = torch.ones(128, device=gpu)
    x[1] = 0
    x[2, 70] = float("nan")
    x[3, 70] = -float("inf")
    with torch.no_grad():
        q, s, z = da.fused_add_rms_norm_fp8(x, w, group_size=64)
        assert z is x
        q1, s1, _ = da.fused_add_rms_norm_fp8(x, w)
        tiny, st, _ = da.fused_add_rms_norm_fp8(x[:1], w * 1e-37)
    v = q.float()
    assert (v[1] == 0).all() and (s[1] == 1).all() and (s1[1] == 1).all()
    assert v[2].isnan().all() and s[2].isnan().all()
    # an infinity: 1 / rms is 0, so the row is 0 but for inf * 0
    assert (v[3, :64] == 0).all() and v[3, 64:].isnan().all() and s[3, 0] == 1 and s[3, 1].isnan()
    assert q1.float()[3].isnan().all() and s1[3].isnan()
    assert (tiny.float() == 0).all() and (st == 1).all()
    rest = [0, 4, 5, 6, 7]
    with torch.no_grad():
        assert torch.equal(q.view(torch.uint8)[rest], da.fused_add_rms_norm_fp8(x[rest], w, group_size=64)[0].view(torch.uint8))


# ---------------------------------------------------------------------------
# embedding


def _embed_case(gpu, ids, V, C, wt=FP, yt=None, padding=None, scale=1.0, strided=False):
    w = _rand(V, C + 5, seed=1, dtype=wt).to(gpu)[:, 3:3 + C] if strided else _rand(V, C, seed=1, dtype=wt).to(gpu)
    yt = wt if yt is None else yt
    leaf = w.detach().requires_grad_()
    y = da.fused_embedding(ids.to(gpu), leaf, padding_idx=padding, scale=scale, out_dtype=yt)
    dy = _rand(*ids.shape, C, seed=2, dtype=yt)
    dyg = dy.to(gpu)
    if strided:
        dyg = torch.nn.functional.pad(dyg, (1, 2))[..., 1:1 + C]
    assert y.shape == (*ids.shape, C) and y.dtype == yt
    (dw,) = torch.autograd.grad(y, leaf, dyg)
    assert dw.dtype == wt
    flat = ids.reshape(-1).long()
    ok = (flat >= 0) & (flat < V)
    want = oh.embedding(flat.clamp(0, V - 1), w.cpu().double(), scale)
    want[~ok] = float("nan")
    want = want.view(y.shape)
    _within("out", y, want, (2 * U + _half(yt)) * want.abs().nan_to_num(0.0))
    pad = -1 if padding is None else padding % V
    dw64 = oh.embedding_grad(ids, dy.double(), V, pad, scale)
    total = oh.embedding_grad(ids, dy.double().abs(), V, pad, abs(scale))
    counts = torch.bincount(flat[ok], minlength=V).double()[:, None]
    _within("dw", dw, dw64, (72 + counts / 32) * U * total + _half(wt) * dw64.abs())
    return dw


def _zipf(n, V, seed):
    u = torch.rand(n, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)
    return (V ** u).long().clamp(0, V - 1)


@pytest.mark.parametrize("N", [1, 2, 63, 64, 65, 700, 4096, 4097, 9001])
@pytest.mark.parametrize("V", [1, 2, 511, 512, 50000])
def test_embedding_sizes(N, V, gpu):
    _say("embed", N, V)
    _embed_case(gpu, _zipf(N, V, N + V), V, 24, scale=1.5)


@pytest.mark.parametrize("C", [1, 3, 8, 9, 100, 511, 512, 513, 1024, 1300, 2056])
def test_embedding_widths(C, gpu):
    _say("embed", C)
    _embed_case(gpu, _zipf(2500, 3001, C).view(50, 50), 3001, C, BF, padding=0, scale=0.5)
    _embed_case(gpu, _zipf(300, 77, C), 77, C, FP, BF, padding=-1, strided=True)


@pytest.mark.parametrize("wt,yt", [(BF, BF), (BF, FP), (FP, BF), (FP, FP)])
@pytest.mark.parametrize("ids_t", [torch.int64, torch.int32])
def test_embedding_types(wt, yt, ids_t, gpu):
    _embed_case(gpu, _zipf(5000, 9000, 3).to(ids_t), 9000, 136, wt, yt, padding=1, scale=11.7)


@pytest.mark.parametrize("N", [5, 64, 1000, 6000, 40000])
def test_embedding_one_token(N, gpu):
    """Every position the same token (its sum crosses every border), the same
    between two others, and every position padding."""
    _embed_case(gpu, torch.full((N,), 7), 50, 72)
    ids = torch.full((N,), 30000)
    ids[0], ids[-1] = 2, 39999
    _embed_case(gpu, ids, 40000, 40)
    dw = _embed_case(gpu, torch.full((N,), 7), 50, 72, padding=7)
    assert (dw == 0).all()


@pytest.mark.parametrize("N", [200, 6000])
def test_embedding_ids_outside_the_table(N, gpu):
    ids = _zipf(N, 1000, 5)
    ids[3], ids[N // 2], ids[N - 1], ids[7] = -1, 1000, 1 << 40, -(1 << 40)
    _embed_case(gpu, ids, 1000, 48)
    ids = ids.clamp(-5, 1 << 30).to(torch.int32)
    _embed_case(gpu, ids, 1000, 48, padding=0)


def test_embedding_large_vocabulary_and_many_positions(gpu):
    """Three digits, and more positions than one run a sort workgroup."""
    _embed_case(gpu, torch.randint(0, 600000, (20000,), generator=torch.Generator().manual_seed(1)), 600000, 8)
    _embed_case(gpu, torch.randint(0, 262143, (3000,), generator=torch.Generator().manual_seed(2)), 262143, 8)
    _embed_case(gpu, torch.randint(0, 262144, (3000,), generator=torch.Generator().manual_seed(2)), 262144, 8)
    N = (1 << 20) + 4097
    ids = _zipf(N, 5000, 3)
    w = torch.zeros(5000, 2, device=gpu, requires_grad=True)
    y = da.fused_embedding(ids.to(gpu), w)
    (dw,) = torch.autograd.grad(y, w, torch.ones_like(y))
    assert torch.equal(dw[:, 0].cpu().long(), torch.bincount(ids, minlength=5000))  # counts: exact in float32


def test_embedding_equal_inputs_give_equal_bits(gpu):
    ids = _zipf(30000, 2000, 4).to(gpu)
    dy = _rand(30000, 200, seed=1, dtype=BF).to(gpu)
    a = hidden._embed_bwd_impl(dy, ids, 2000, FP, 0, 1.0)
    for _ in range(3):
        assert torch.equal(a, hidden._embed_bwd_impl(dy, ids, 2000, FP, 0, 1.0))


def test_embedding_module(gpu):
    emb = da.FusedEmbedding(300, 40, padding_idx=2, scale=2.0).to(gpu)
    ref = torch.nn.Embedding(300, 40, padding_idx=2).to(gpu)
    ref.load_state_dict(emb.state_dict(), strict=True)
    ids = torch.randint(0, 300, (4, 50), generator=torch.Generator().manual_seed(1)).to(gpu)
    dy = _rand(4, 50, 40, seed=2, dtype=FP).to(gpu)
    emb(ids).backward(dy)
    (ref(ids) * 2.0).backward(dy)
    assert torch.equal(emb(ids), ref(ids) * 2.0)
    assert (emb.weight.grad - ref.weight.grad).abs().max().item() <= 1e-5  # both sum a few float32 values below 8


# ---------------------------------------------------------------------------
# together, and the ways to call them


class _Net(torch.nn.Module):
    """A pre-norm block's path: embedding, dropout, residual + norm, twice."""

    def __init__(self):
        super().__init__()
        self.emb = da.FusedEmbedding(200, 96, padding_idx=0, scale=96**0.5)
        self.drop = da.FusedDropout(0.1)
        self.up, self.down = torch.nn.Linear(96, 160), torch.nn.Linear(160, 96)
        self.n1, self.n2 = da.FusedRMSNorm(96), da.FusedRMSNorm(96, dropout_p=0.2)

    def forward(self, ids):
        x = self.drop(self.emb(ids))
        h = self.n1(x)
        h = torch.nn.functional.linear(torch.nn.functional.gelu(self.up(h)), self.down.weight)
        y, z = self.n2(h, x, bias=self.down.bias)
        return y, z


def _net_reference(net, ids, seeds):
    p = {k: v.detach().cpu().double().requires_grad_() for k, v in net.named_parameters()}
    x = oh.dropout_add(oh.embedding(ids, p["emb.weight"], 96**0.5), None, None, round(0.1 * 65536), seeds[0])
    h = oh.rms_norm(x, p["n1.weight"], 1e-6)
    h = torch.nn.functional.gelu(h @ p["up.weight"].T + p["up.bias"]) @ p["down.weight"].T
    z = oh.dropout_add(h, p["down.bias"], x, round(0.2 * 65536), seeds[1])
    return p, oh.rms_norm(z, p["n2.weight"], 1e-6), z


def _net_run(net, ids, dy, dz):
    torch.manual_seed(17)
    y, z = net(ids)
    grads = torch.autograd.grad((y, z), list(net.parameters()), (dy, dz))
    return y, z, grads


def test_a_run_of_them_together(gpu):
    """Outputs and gradients of a block on all of them against float64:
    float32, two matrix products of at most 160 terms between, 1e-4 of each
    tensor's scale (400 half steps of 2^-24 a stage would be 2.4e-5)."""
    torch.manual_seed(5)
    net = _Net().to(gpu).train()
    ids = torch.randint(0, 200, (3, 40), generator=torch.Generator().manual_seed(1))
    ids[:, 30:] = 0
    dy, dz = (_rand(3, 40, 96, seed=k, dtype=FP).to(gpu) for k in (1, 2))
    y, z, grads = _net_run(net, ids.to(gpu), dy, dz)
    torch.manual_seed(17)
    seeds = [int(hidden.draw_dropout_seed().item()) for _ in range(2)]
    p, y64, z64 = _net_reference(net, ids, seeds)
    want = list(torch.autograd.grad((y64, z64), list(p.values()), (dy.cpu().double(), dz.cpu().double())))
    want[0][0] = 0.0  # the padding token
    for name, a, b in (("y", y, y64), ("z", z, z64), *zip(p, grads, want)):
        err = (a.detach().cpu().double() - b.detach()).abs().max().item()
        assert err <= 1e-4 * b.abs().max().item(), (name, err)


def test_eight_bit_rows_feed_a_scaled_product(gpu):
    """Serving in 8 bits as it is used: the norm's rows and scales straight
    into torch's row-scaled float8 product.  Against float64 on the values
    that q and the weight's bytes stand for, the product loses its float32
    sums (K u of the sum of magnitudes) and the bf16 of its result."""
    M, K, N = 64, 512, 256
    x, res = _rand(M, K, seed=1, dtype=BF).to(gpu), _rand(M, K, seed=2, dtype=BF).to(gpu)
    with torch.no_grad():
        q, scale, z = da.fused_add_rms_norm_fp8(x, torch.ones(K, device=gpu), res=res)
        w = _rand(N, K, seed=3, dtype=FP, std=0.05)
        ws = w.abs().amax(1, keepdim=True) / 448.0
        wq = (w / ws).to(torch.float8_e4m3fn)
        y = torch._scaled_mm(q, wq.to(gpu).t(), scale_a=scale, scale_b=ws.t().contiguous().to(gpu), out_dtype=BF)
    a = q.float().cpu().double() * scale.cpu().double()
    b = (wq.float().double() * ws.double()).t()
    _within("product", y, a @ b, (K * U + 4 * U) * (a.abs() @ b.abs()) + _half(BF) * (a @ b).abs())
    assert torch.equal(z, x + res)


def test_one_tensor_in_two_places(gpu):
    """x and the residual one leaf, a table looked up twice, a graph walked
    twice: gradients add up."""
    x = _rand(6, 200, seed=1, dtype=FP).to(gpu).requires_grad_()
    w = torch.ones(200, device=gpu)
    dy = _rand(6, 200, seed=2, dtype=FP).to(gpu)
    for p in (0.0, 0.5):
        y, z = da.fused_add_rms_norm(x, w, EPS, res=x, dropout_p=p, seed=SEED)
        (g,) = torch.autograd.grad((y, z), x, (dy, dy), retain_graph=True)
        (again,) = torch.autograd.grad((y, z), x, (dy, dy))
        assert torch.equal(g, again)
        u, v = x.detach().requires_grad_(), x.detach().requires_grad_()
        y, z = da.fused_add_rms_norm(u, w, EPS, res=v, dropout_p=p, seed=SEED)
        gu, gv = torch.autograd.grad((y, z), (u, v), (dy, dy))
        assert torch.equal(g, gu + gv)
        y = da.fused_dropout(x, p, res=x, seed=SEED)
        (g,) = torch.autograd.grad(y, x, dy)
        keep = oh.keep_mask(6, 200, round(p * 65536), SEED).to(gpu) / (1 - p)
        assert torch.equal(g, dy * keep + dy)
    table = _rand(30, 40, seed=3, dtype=FP).to(gpu).requires_grad_()
    a = torch.arange(10, device=gpu)
    y = da.fused_embedding(a, table) + da.fused_embedding(a.flip(0), table)
    (g,) = torch.autograd.grad(y.sum(), table)
    assert (g[:10] == 2).all() and (g[10:] == 0).all()
    # ids with strides of their own
    grid = torch.arange(24, device=gpu).view(4, 6)
    assert torch.equal(da.fused_embedding(grid.t(), table), table[grid.t()])
    assert torch.equal(da.fused_embedding(grid[:, ::2], table), table[grid[:, ::2]])


def test_only_some_inputs_need_gradients(gpu):
    x, r, b = (_rand(*s, seed=k, dtype=FP).to(gpu) for k, s in enumerate(((4, 60), (4, 60), (60,))))
    w = torch.ones(60, device=gpu)
    dy = _rand(4, 60, seed=5, dtype=FP).to(gpu)

    def grads(*which):
        t = [v.detach().requires_grad_(k in which) for k, v in zip("xrbw", (x, r, b, w))]
        y, z = da.fused_add_rms_norm(t[0], t[3], EPS, bias=t[2], res=t[1], dropout_p=0.25, seed=SEED)
        d = da.fused_dropout(t[0], 0.25, bias=t[2], res=t[1], seed=SEED)
        need = [v for v in t if v.requires_grad]
        out = [(y * dy).sum() + (z * dy).sum()] + ([(d * dy).sum()] if d.requires_grad else [])
        return dict(zip(which, torch.autograd.grad(sum(out), need)))

    full = grads("x", "r", "b", "w")
    for one in "xrbw":
        assert torch.equal(grads(one)[one], full[one])


def test_checkpointing_draws_the_same_bits(gpu):
    from torch.utils.checkpoint import checkpoint

    net = _Net().to(gpu).train()
    ids = torch.randint(0, 200, (3, 40), generator=torch.Generator().manual_seed(1)).to(gpu)
    dy, dz = (_rand(3, 40, 96, seed=k, dtype=FP).to(gpu) for k in (1, 2))
    want = _net_run(net, ids, dy, dz)
    torch.manual_seed(17)
    y, z = checkpoint(net, ids, use_reentrant=False)
    grads = torch.autograd.grad((y, z), list(net.parameters()), (dy, dz))
    assert torch.equal(y, want[0]) and all(torch.equal(a, b) for a, b in zip(grads, want[2]))


def test_compiled(gpu):
    """Under torch.compile the registered ops run: the same bits for equal
    seeds, with the autograd they register."""
    torch._dynamo.reset()
    w = torch.rand(64, generator=torch.Generator().manual_seed(1)).to(gpu).requires_grad_()
    x = _rand(4, 10, 64, seed=2, dtype=BF).to(gpu).requires_grad_()
    table = _rand(50, 64, seed=3, dtype=BF).to(gpu).requires_grad_()
    ids = torch.randint(0, 50, (4, 10), generator=torch.Generator().manual_seed(4)).to(gpu)
    seed = torch.tensor([SEED], dtype=torch.int64)

    def f(x, w, table, seed):
        e = da.fused_embedding(ids, table, padding_idx=0)
        e = da.fused_dropout(e, 0.1, seed=seed)
        y, z = da.fused_add_rms_norm(x, w, res=e, dropout_p=0.2, seed=seed)
        return y, z

    want = f(x, w, table, seed)
    gw = torch.autograd.grad([o.float().sum() + (o.float() ** 2).sum() for o in want], (x, w, table))
    g = torch.compile(f, backend="aot_eager", fullgraph=True)
    got = g(x, w, table, seed)
    gg = torch.autograd.grad([o.float().sum() + (o.float() ** 2).sum() for o in got], (x, w, table))
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert all(torch.equal(a, b) for a, b in zip(gw, gg))


def test_side_streams(gpu):
    """Two streams at once, each with its own work before the call."""
    x = _rand(512, 768, seed=1, dtype=BF).to(gpu)
    w = torch.ones(768, device=gpu, requires_grad=True)
    ids = _zipf(6000, 3000, 2).to(gpu)
    dy = _rand(6000, 64, seed=3, dtype=BF).to(gpu)
    want = da.fused_add_rms_norm(x * 2, w, res=x, dropout_p=0.1, seed=SEED)
    wantd = hidden._embed_bwd_impl(dy * 2, ids, 3000, FP, -1, 1.0)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        for s in (a, b):
            s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(a):
            got = da.fused_add_rms_norm(x * 2, w, res=x, dropout_p=0.1, seed=SEED)
        with torch.cuda.stream(b):
            gotd = hidden._embed_bwd_impl(dy * 2, ids, 3000, FP, -1, 1.0)
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(want, got)) and torch.equal(wantd, gotd)


def test_two_threads(gpu):
    """Two threads, each on its own stream, forward and backward at once (the
    calls release the interpreter's lock)."""
    x, res = _rand(300, 520, seed=1, dtype=BF).to(gpu), _rand(300, 520, seed=2, dtype=FP).to(gpu)
    ids = _zipf(5000, 700, 3).to(gpu)
    dys = [_rand(300, 520, seed=4, dtype=FP).to(gpu), _rand(5000, 520, seed=5, dtype=FP).to(gpu)]

    def norm():
        v, w = x.detach().requires_grad_(), torch.ones(520, device=gpu, requires_grad=True)
        y, z = da.fused_add_rms_norm(v, w, EPS, res=res, dropout_p=0.25, seed=SEED)
        return [y, z, *torch.autograd.grad((y, z), (v, w), (dys[0], dys[0]))]

    def table():
        t = torch.ones(700, 520, device=gpu, requires_grad=True)
        y = da.fused_dropout(da.fused_embedding(ids, t), 0.5, seed=SEED)
        return [y, *torch.autograd.grad(y, t, dys[1])]

    want = [norm(), table()]
    torch.cuda.synchronize()

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            outs = [(norm, table)[k]() for _ in range(8)]
            torch.cuda.current_stream().synchronize()
            return all(torch.equal(a, b) for out in outs for a, b in zip(out, want[k]))

    with ThreadPoolExecutor(2) as pool:
        assert list(pool.map(work, (0, 1))) == [True, True]


def test_under_capture_and_twice_differentiated_they_raise(gpu):
    x = torch.randn(4, 64, device=gpu)
    w = torch.ones(64, device=gpu)
    ids = torch.zeros(4, dtype=torch.int64, device=gpu)
    calls = [
        lambda: da.fused_dropout(x, 0.5, seed=1),
        lambda: da.fused_rms_norm(x, w),
        lambda: da.fused_add_rms_norm_fp8(x, w),
        lambda: da.fused_embedding(ids, x),
        lambda: hidden._embed_bwd_impl(x, ids, 4, FP, -1, 1.0),
        lambda: hidden._hidden_dropout_bwd_impl(x, FP, FP, 100, torch.tensor([1])),
    ]
    for call in calls:
        call()
    torch.cuda.synchronize()
    refused = []
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in calls:
            try:
                call()
            except RuntimeError as e:
                refused.append("capturing" in str(e))
        x + 1  # a graph needs work
    assert refused == [True] * len(calls)
    v = x.clone().requires_grad_()
    for y in (da.fused_dropout(v, 0.5, seed=1), da.fused_rms_norm(v, w)):
        (g,) = torch.autograd.grad(y, v, v * 1.0, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), v)


def test_other_transforms_raise(gpu):
    """Forward-mode tangents and torch.func have no rule here: an error, not a
    result without them."""
    import torch.autograd.forward_ad as fwAD

    x, w = torch.randn(4, 64, device=gpu), torch.ones(64, device=gpu)
    for call in (lambda v: da.fused_dropout(v, 0.5, seed=1), lambda v: da.fused_rms_norm(v, w),
                 lambda v: da.fused_embedding(torch.zeros(2, dtype=torch.int64, device=gpu), v)):
        with fwAD.dual_level():
            with pytest.raises(RuntimeError):
                call(fwAD.make_dual(x, torch.ones_like(x)))
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(x.expand(3, 4, 64))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda v: call(v).sum())(x)


def test_refusals_on_the_gpu(gpu):
    x, w = torch.randn(4, 64, device=gpu), torch.ones(64, device=gpu)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        da.fused_dropout(x.half(), 0.5)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        da.fused_rms_norm(x, w, out_dtype=torch.float16)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        da.fused_embedding(torch.zeros(2, dtype=torch.int64, device=gpu), x.double())
    with pytest.raises(ValueError, match="columns"):
        da.fused_rms_norm(torch.randn(2, 16385, device=gpu), torch.ones(16385, device=gpu))
    with pytest.raises(ValueError, match="on cpu"):
        da.fused_rms_norm(x, w.cpu())
    with pytest.raises(ValueError, match="on cpu"):
        da.fused_embedding(torch.zeros(2, dtype=torch.int64), x)
    with pytest.raises(ValueError, match="group_size"):
        da.fused_add_rms_norm_fp8(x, w, group_size=128)


def test_autocast_and_modules(gpu):
    from oracle import eager

    x = torch.randn(2, 9, 64, device=gpu)
    w = torch.ones(64, device=gpu)
    with torch.autocast("cuda", dtype=BF):
        y, z = da.fused_add_rms_norm(x.bfloat16(), w, res=x.bfloat16())
        assert y.dtype == FP and z.dtype == BF
    cfg = eager.make_config(hidden_size=64, num_attention_heads=4, intermediate_size=128, layer_norm_eps=1e-7,
                            hidden_dropout_prob=0.25, fused_hidden_dropout=True, use_rmsnorm_heads=True)
    # the fused dropout: the module on the GPU against the module on the CPU, one seed (fp32, 1e-4 of scale)
    for cls in (da.FusedSelfOutput, da.FusedRTDHead):
        cpu = cls(cfg).train()
        dev = cls(cfg).to(gpu).train()
        dev.load_state_dict(cpu.state_dict(), strict=True)
        outs = []
        for m, d in ((cpu, "cpu"), (dev, gpu)):
            torch.manual_seed(3)
            v = x.cpu().to(d).requires_grad_()
            out = m(v, v * 0.5) if cls is da.FusedSelfOutput else m(v)
            g = torch.autograd.grad(out, [v, *m.parameters()], torch.ones_like(out))
            outs.append([out, *g])
        for a, b in zip(*outs):
            err = (a.detach() - b.detach().cpu()).abs().max().item()
            assert err <= 1e-4 * max(1.0, a.abs().max().item()), err


# ---------------------------------------------------------------------------
# offsets past 32 bits


def test_far_rows(gpu):
    """Tensors of more than 2^32 bytes and 2^31 elements: the last rows against
    float64."""
    C, N = 2056, (1 << 20) + 5
    rows = [0, N // 2, N - 2, N - 1]
    x = torch.zeros(N, C, dtype=BF, device=gpu)
    some = _rand(len(rows), C, seed=1, dtype=BF)
    x[rows] = some.to(gpu)
    keep = oh.keep_mask(rows, C, 32768, SEED)
    y = da.fused_dropout(x, 0.5, seed=SEED)
    assert torch.equal(y[rows].cpu().double(), some.double() * keep * 2)
    del y
    w = torch.ones(C, device=gpu)
    y, z = da.fused_add_rms_norm(x, w, EPS, dropout_p=0.5, seed=SEED)
    z64 = some.double() * keep * 2
    y64 = oh.rms_norm(z64, torch.ones(C, dtype=torch.float64), EPS)
    assert torch.equal(z[rows].cpu().double(), z64)
    _within("y", y[rows], y64, (192 * U + _half(BF)) * y64.abs())
    del y, z
    with torch.no_grad():
        q, s, _ = da.fused_add_rms_norm_fp8(x, w, EPS)
    y64 = oh.rms_norm(some.double(), torch.ones(C, dtype=torch.float64), EPS)
    _within("q", q[rows].float() * s[rows], y64, 2.0**-4 * y64.abs() * (1 + 1e-5) + 2.0**-10 * s[rows].cpu().double() + 192 * U * y64.abs())
    del q, s
    ids = torch.tensor([N - 1, 3, N // 2, N - 1, N - 2], device=gpu)
    e = da.fused_embedding(ids, x)
    assert torch.equal(e, x[ids])
    dy = _rand(5, C, seed=2, dtype=BF).to(gpu)
    del x
    dw = hidden._embed_bwd_impl(dy, ids, N, BF, -1, 1.0)
    assert torch.equal(dw[N - 1], (dy[0].float() + dy[3].float()).bfloat16())
    assert torch.equal(dw[N - 2], dy[4]) and torch.equal(dw[N // 2], dy[2]) and torch.equal(dw[3], dy[1])
    dw[[N - 1, N - 2, N // 2, 3]] = 0
    assert not dw.view(torch.int16).any()


def test_far_rows_backward(gpu):
    """The gradients' last rows of more than 2^31 elements, all other rows zero."""
    C, N = 2056, (1 << 20) + 5
    rows = [0, N // 2, N - 2, N - 1]
    some = _rand(len(rows), C, seed=1, dtype=BF)
    dy = torch.zeros(N, C, dtype=BF, device=gpu)
    dy[rows] = some.to(gpu)
    seed = torch.tensor([SEED])
    keep = oh.keep_mask(rows, C, 32768, SEED)
    dx, db = hidden._hidden_dropout_bwd_impl(dy, BF, FP, 32768, seed)
    want = some.double() * keep * 2
    assert torch.equal(dx[rows].cpu().double(), want)
    # four values a column and zeros: three roundings
    _within("dbias", db, want.sum(0), 4 * U * want.abs().sum(0))
    del dx
    w, x = torch.ones(C, device=gpu), dy
    rstd = torch.ones(N, device=gpu)
    z64 = some.double()
    dx, _, dw, _ = hidden._add_rms_norm_bwd_impl(dy, None, x, None, None, w, rstd, 0, None)
    # g = z = dy, r = 1: dx = z (1 - mean(z^2)), a mean by at most 8 (lane) + 6 (lanes) + 8 (waves)
    # additions and a division, then a product and a difference
    m = z64.square().mean(-1, keepdim=True)
    wx = z64 * (1 - m)
    _within("dx", dx[rows], wx, _half(BF) * wx.abs() + 32 * U * z64.abs() * (1 + m))
    ww = z64.square().sum(0)
    _within("dw", dw, ww, 8 * U * ww)
