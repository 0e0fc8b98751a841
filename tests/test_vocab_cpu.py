"""The operators on a vocabulary's logits without a GPU: the torch path of CPU
tensors against the float64 definitions, its gradients against differences,
refusals of the functions and of the C entry points (before any device work),
which calls go into the extension, and the ops' fake implementations.

The CPU path computes in float32 over rows of at most 50 values within 40 of
each other: a log probability is a sum of terms below 50, an exp of one of them
and a sum of 50, less than 50 * (3 + 50) half steps of 2^-24 = 1.6e-4; those
that are summed with weights that add up to one stay within it.
"""

from __future__ import annotations

import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import deberta_amd as da
from deberta_amd import _lib, vocab
from oracle import vocab as ov
from tests._hidden import Wrapper

ROOT = Path(__file__).resolve().parents[1]
TOL = 1.6e-4
INF, NAN = float("inf"), float("nan")


def _rand(*shape, seed=0, dtype=torch.float32, std=3.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * std).to(dtype)


def _near(got, want):
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.isinf(), want.isinf())
    fine = want.isfinite()
    assert (got[fine].double() - want[fine].double()).abs().max().item() <= TOL if fine.any() else True


@pytest.mark.parametrize("T", [1.0, 0.6, 2.5])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
def test_cpu_logprobs(T, dtype):
    x = _rand(2, 6, 50, dtype=dtype)
    x[0, 1, 30:] = -INF
    x[0, 2, 5] = NAN
    x[0, 3, 6] = INF
    x[0, 4] = -INF
    x[1, 0] = 1.5  # ties: the first ones
    x[1, 1] = torch.finfo(torch.bfloat16 if dtype is torch.bfloat16 else torch.float32).min  # a mask that leaves nothing
    ids = torch.randint(0, 50, (2, 6), generator=torch.Generator().manual_seed(1))
    ids[1, 5] = -100
    ids[0, 1] = 40  # masked: -inf
    o = da.fused_token_logprobs(x, ids, top_k=7, temperature=T)
    logp = ov.log_probs(x, T)
    entropy, _ = ov.moments(logp)
    out = ids == -100
    wide = torch.promote_types(dtype, torch.float32)
    assert all(t.dtype == wide for t in (o.logprobs, o.entropy, o.logsumexp, o.top_logprobs)) and o.top_ids.dtype == torch.int64
    _near(o.logprobs, logp.gather(-1, ids.clamp(min=0).unsqueeze(-1)).squeeze(-1).masked_fill(out, 0))
    _near(o.entropy, entropy.masked_fill(out, 0))
    want = ov.logsumexp(x, T).masked_fill(out, 0)
    want[1, 1] = o.logsumexp[1, 1]  # of the type's lowest value, far out
    _near(o.logsumexp, want)
    assert (o.entropy[1, 1] - torch.log(torch.tensor(50.0))).abs() < 1e-5
    top = ov.largest(x, 7)
    assert torch.equal(o.top_ids, top.masked_fill(out.unsqueeze(-1), -1))
    assert o.top_ids[1, 0].tolist() == list(range(7))
    _near(o.top_logprobs, logp.gather(-1, top).masked_fill(out.unsqueeze(-1), 0))


def test_cpu_gradients_against_differences():
    x = _rand(3, 9, dtype=torch.float64)
    x[1, 4] = -20.0
    ids = torch.tensor([3, -100, 8], dtype=torch.int32)
    x = x.requires_grad_()

    def results(x):
        o = da.fused_token_logprobs(x, ids, top_k=3, temperature=1.7)
        return o.logprobs, o.entropy, o.logsumexp, o.top_logprobs

    assert torch.autograd.gradcheck(results, (x,))
    t_ids = torch.tensor([[1, 5, 5], [-1, -1, -1], [0, -1, 8]])
    teacher = _rand(3, 3, seed=3, dtype=torch.float64)
    assert torch.autograd.gradcheck(lambda x: da.fused_distillation_loss(x, t_ids, teacher, 1.7), (x,))
    lse = torch.logsumexp(teacher, -1) + 0.5
    assert torch.autograd.gradcheck(lambda x: da.fused_distillation_loss(x, t_ids, teacher, 1.0, lse), (x,))
    (d,) = torch.autograd.grad(da.fused_distillation_loss(x, t_ids, teacher, 1.7).sum(), x)
    assert (d[1] == 0).all()


def test_oracle_gradients_are_the_formulas():
    """The closed forms that the kernels compute."""
    x = _rand(4, 11, dtype=torch.float64)
    x[0, 3] = -INF
    x = x.requires_grad_()
    T, ids = 1.3, torch.tensor([2, 10, 0, 5])
    g, gh, gl = (_rand(4, seed=s, dtype=torch.float64) for s in (1, 2, 3))
    logp = ov.log_probs(x, T)
    entropy, _ = ov.moments(logp)
    lp = logp.gather(-1, ids[:, None]).squeeze(-1)
    (d,) = torch.autograd.grad((lp, entropy, ov.logsumexp(x, T)), x, (g, gh, gl))
    p = logp.detach().exp()
    ln = torch.where(p > 0, logp.detach(), 0.0)
    want = p * ((gl - g - gh * entropy.detach())[:, None] - gh[:, None] * ln)
    want[torch.arange(4), ids] += g
    assert (d - want / T).abs().max() < 1e-14
    t_ids = torch.tensor([[1, 4], [2, 2], [-1, 0], [10, 3]])
    q, log_q = ov.teacher_probs(t_ids, _rand(4, 2, seed=4), T)
    (d,) = torch.autograd.grad(ov.distillation(ov.log_probs(x, T), t_ids, q, log_q, T), x, g)
    want = p * q.sum(-1, keepdim=True)
    want.scatter_add_(-1, t_ids.clamp(min=0), -q)
    assert (d - want * T * g[:, None]).abs().max() < 1e-14


def test_cpu_rows_left_out_are_not_read():
    x = _rand(3, 8)
    x[1] = NAN
    x = x.requires_grad_()
    o = da.fused_token_logprobs(x, torch.tensor([1, 7, 2]), top_k=2, ignore_index=7)
    assert o.logprobs[1] == 0 and o.entropy[1] == 0 and o.logsumexp[1] == 0 and o.top_ids[1].tolist() == [-1, -1]
    (d,) = torch.autograd.grad(o.logprobs.sum() + o.entropy.sum() + o.top_logprobs.sum(), x)
    assert (d[1] == 0).all() and d.isfinite().all()
    loss = da.fused_distillation_loss(x, torch.tensor([[1], [-1], [2]]), torch.zeros(3, 1))
    (d,) = torch.autograd.grad(loss.sum(), x)
    assert loss[1] == 0 and (d[1] == 0).all() and d.isfinite().all()


@pytest.mark.parametrize("T", [1.0, 2.5])
def test_cpu_distillation(T):
    x = _rand(5, 50, dtype=torch.bfloat16)
    x[0, 7] = -INF
    ids = torch.randint(0, 50, (5, 4), generator=torch.Generator().manual_seed(2))
    ids[0, 1], ids[1, 2], ids[2] = 7, -1, -5
    teacher = _rand(5, 4, seed=3)
    teacher[0, 1] = -INF  # probability 0 where the student's is 0 too
    teacher[3] = -INF  # none left
    for lse in (None, torch.logsumexp(teacher / T, -1).nan_to_num(neginf=0.0) + 0.25):
        got = da.fused_distillation_loss(x, ids, teacher, T, lse)
        q, log_q = ov.teacher_probs(ids, teacher, T, lse)
        _near(got, ov.distillation(ov.log_probs(x, T), ids, q, log_q, T))
        assert got[2] == 0 and got[3] == 0 and got.isfinite().all()
    ids[0, 0] = 7
    assert da.fused_distillation_loss(x, ids, teacher, T)[0] == INF


def test_cpu_distillation_at_extreme_temperatures():
    """T^2 past float32 on either side: T (max - x), and no loss over one token."""
    x, zero = _rand(4, 101), torch.zeros(4, 1)
    want = 2.0**-100 * (x.double().amax(-1) - x.double().amin(-1))
    got = da.fused_distillation_loss(x, x.argmin(-1, keepdim=True), zero, 2.0**-100).double()
    assert ((got - want).abs() <= 8 * 2.0**-24 * want).all()
    for T in (2.0**-100, 2.0**100):
        assert (da.fused_distillation_loss(x[:, :1], zero[:, :1].long(), zero, T) == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
def test_cpu_distillation_takes_the_teachers_largest_off_before_its_scaling(dtype):
    """A teacher whose logits / T leave float32: rows of the type's lowest value are
    uniform, as they are on the device, and differences decide, not the values."""
    x, ids = _rand(4, 50, dtype=dtype), torch.randint(0, 50, (4, 3), generator=torch.Generator().manual_seed(2))
    teacher = _rand(4, 3, seed=3)
    teacher[0] = torch.finfo(torch.float32).min
    teacher[1] = 3e38 + 1e37 * torch.arange(3)
    teacher[2, 1] = torch.finfo(torch.float32).min  # probability 0
    for T in (0.5, 0.25):
        q, log_q = ov.teacher_probs(ids, teacher, T)
        assert (q[0] - 1 / 3).abs().max() < 1e-15 and q[1].tolist() == [0, 0, 1] and q[2, 1] == 0
        _near(da.fused_distillation_loss(x, ids, teacher, T), ov.distillation(ov.log_probs(x, T), ids, q, log_q, T))
    # q = (1, 0), so T^2 (-log p) = T (max - x): a product with 1 / T, two with T and a difference
    T, far = 2.0**-100, torch.tensor([[1e9, 1e9 - 64.0]]).expand(4, 2)
    ids = torch.stack((x.argmin(-1), x.argmax(-1)), -1)
    want = T * (x.double().amax(-1) - x.double().amin(-1))
    got = da.fused_distillation_loss(x, ids, far, T).double()
    assert ((got - want).abs() <= 8 * 2.0**-24 * want).all()


@pytest.mark.parametrize("shape", [(0, 9), (2, 0, 9)], ids=str)
def test_cpu_no_rows(shape):
    x = torch.zeros(shape)
    o = da.fused_token_logprobs(x, torch.zeros(shape[:-1], dtype=torch.int64), top_k=3)
    assert o.logprobs.shape == shape[:-1] and o.top_ids.shape == (*shape[:-1], 3)
    assert da.fused_distillation_loss(x, torch.zeros(*shape[:-1], 2, dtype=torch.int64), torch.zeros(*shape[:-1], 2)).shape == shape[:-1]


def test_refusals():
    x, ids = _rand(3, 8), torch.tensor([1, 2, 3])
    t_ids, teacher = torch.tensor([[1], [2], [3]]), torch.zeros(3, 1)
    f, d = da.fused_token_logprobs, da.fused_distillation_loss
    for T in (0.0, -1.0, INF, NAN, 2.0**-101):
        for call in (lambda: f(x, ids, temperature=T), lambda: d(x, t_ids, teacher, T)):
            with pytest.raises(ValueError, match="temperature"):
                call()
    for k in (-1, 9, 129):
        with pytest.raises(ValueError, match="top_k"):
            f(x, ids, top_k=k)
    with pytest.raises(ValueError, match="at most 524288"):
        f(torch.zeros(1, (1 << 19) + 1), top_k=1)
    with pytest.raises(ValueError, match="shape"):
        f(x, ids[:2])
    with pytest.raises(TypeError, match="int64 or int32"):
        f(x, ids.float())
    for bad in (8, -1):
        with pytest.raises(IndexError, match="outside"):
            f(x, torch.tensor([1, bad, 2]))
    with pytest.raises(ValueError, match="at least one column"):
        f(torch.zeros(3, 0), ids)
    with pytest.raises(TypeError, match="floating"):
        f(ids[None], torch.tensor([0]))
    with pytest.raises(ValueError, match="K in"):
        d(x, torch.zeros(3, 0, dtype=torch.int64), torch.zeros(3, 0))
    with pytest.raises(ValueError, match="K in"):
        d(x, torch.zeros(3, 129, dtype=torch.int64), torch.zeros(3, 129))
    with pytest.raises(ValueError, match="K in"):
        d(x, ids, teacher)
    with pytest.raises(ValueError, match="teacher_logits"):
        d(x, t_ids, torch.zeros(3, 2))
    with pytest.raises(ValueError, match="teacher_lse"):
        d(x, t_ids, teacher, 1.0, torch.zeros(2))
    with pytest.raises(IndexError, match="outside"):
        d(x, torch.tensor([[8], [1], [1]]), teacher)
    with pytest.raises(ValueError, match="no gradient for the teacher"):
        d(x, t_ids, teacher.requires_grad_())
    with torch.no_grad():
        d(x, t_ids, teacher)


@pytest.mark.parametrize("t", [1.0, 2.0, 0.7])
def test_what_a_teachers_pass_stores_gives_its_probabilities(t):
    """The documented ways from a pass at t to the loss at T: of a student that is the
    teacher, with q over the entries the loss of those alone, with the teacher's own
    probabilities nothing.  In float64, to far more than the roundings of 50 terms."""
    x, T, K = _rand(5, 50, dtype=torch.float64), 2.0, 12
    p = da.fused_token_logprobs(x, top_k=K, temperature=t)
    logp = torch.log_softmax(x / T, -1).gather(-1, p.top_ids)
    log_q = torch.log_softmax(x.gather(-1, p.top_ids) / T, -1)
    got = da.fused_distillation_loss(x, p.top_ids, t * p.top_logprobs, T)
    assert (got - T * T * (log_q.exp() * (log_q - logp)).sum(-1)).abs().max() < 1e-12
    if t == 1.0:
        assert torch.equal(got, da.fused_distillation_loss(x, p.top_ids, p.top_logprobs, T))
    if t == T:
        zeros = torch.zeros_like(p.entropy)
        assert da.fused_distillation_loss(x, p.top_ids, T * p.top_logprobs, T, zeros).abs().max() < 1e-12
        assert da.fused_distillation_loss(x, p.top_ids, x.gather(-1, p.top_ids), T, p.logsumexp).abs().max() < 1e-12


def test_a_teachers_types_are_the_devices():
    """float32 or bfloat16 logits and a float32 logsumexp, as on the GPU; float64
    beside a student in float64, which is computed so."""
    x, ids, teacher, lse = _rand(3, 8), torch.tensor([[1], [2], [3]]), torch.zeros(3, 1), torch.zeros(3)
    d = da.fused_distillation_loss
    for student in (x, x.bfloat16(), x.double()):
        for t in (torch.float16, torch.int64, torch.int32, torch.bool, torch.complex64):
            with pytest.raises(TypeError, match="teacher_logits: dtype must be float32 or bfloat16"):
                d(student, ids, teacher.to(t))
        for t in (torch.float16, torch.bfloat16, torch.int64):
            with pytest.raises(TypeError, match="teacher_lse must be float32"):
                d(student, ids, teacher, 1.0, lse.to(t))
        for t in (torch.float32, torch.bfloat16):
            assert d(student, ids, teacher.to(t), 1.0, lse).isfinite().all()
    for student in (x, x.bfloat16()):
        with pytest.raises(TypeError, match="teacher_logits: dtype must be float32 or bfloat16"):
            d(student, ids, teacher.double())
        with pytest.raises(TypeError, match="teacher_lse must be float32"):
            d(student, ids, teacher, 1.0, lse.double())
    assert d(x.double(), ids, teacher.double(), 1.0, lse.double()).dtype == torch.float64


# ---------------------------------------------------------------------------
# calls on device tensors, seen without one (see test_hidden_calls_cpu.py)


@pytest.fixture
def as_on_gpu(monkeypatch):
    """CPU tensors that say they are on the GPU."""
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))


def test_plain_tensors_go_into_the_extension(as_on_gpu):
    x = torch.randn(3, 8)
    for call in (lambda: da.fused_token_logprobs(x, torch.tensor([1, 2, 3]), top_k=2),
                 lambda: da.fused_distillation_loss(x, torch.tensor([[1], [2], [3]]), torch.zeros(3, 1))):
        with pytest.raises(ValueError, match="must be on the GPU"):
            call()


@pytest.mark.parametrize("which", ["logits", "ids", "teacher_ids", "teacher_logits", "teacher_lse"])
def test_a_wrapper_in_any_argument_sees_the_op(which, as_on_gpu):
    t = {"logits": torch.randn(3, 8), "ids": torch.tensor([1, 2, 3]), "teacher_ids": torch.tensor([[1], [2], [3]]),
         "teacher_logits": torch.zeros(3, 1), "teacher_lse": torch.zeros(3)}
    t[which] = Wrapper(t[which])
    calls = []
    if which in ("logits", "ids"):
        calls.append(lambda: da.fused_token_logprobs(t["logits"], t["ids"]))
    if which != "ids":
        calls.append(lambda: da.fused_distillation_loss(t["logits"], t["teacher_ids"], t["teacher_logits"], 1.0, t["teacher_lse"]))
    for call in calls:
        Wrapper.seen.clear()
        with pytest.raises(NotImplementedError):
            call()
        assert any("deberta_amd" in str(f) for f in Wrapper.seen)


def test_fake_shapes_and_cpu_refusal_of_the_ops():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty(2, 3, 50, dtype=torch.bfloat16, device="cuda")
        ids = torch.empty(2, 3, dtype=torch.int64, device="cuda")
        o = torch.ops.deberta_amd.token_logprobs(x, ids, 4, 1.0, -100)
        assert [tuple(t.shape) for t in o] == [(2, 3), (2, 3), (2, 3), (2, 3, 4), (2, 3, 4), (6, 4)]
        assert o[4].dtype == torch.int64 and o[0].dtype == torch.float32
        o = torch.ops.deberta_amd.token_logprobs(x, None, 0, 1.0, -100)
        assert [tuple(t.shape) for t in o] == [(0,), (2, 3), (2, 3), (2, 3, 0), (2, 3, 0), (6, 4)]
        assert torch.ops.deberta_amd.token_logprobs_bwd(None, o[1], None, None, x, None, None, o[5], 1.0, -100).dtype == x.dtype
        loss, stats = torch.ops.deberta_amd.distill_loss(x, ids[..., None], x[..., :1], None, 2.0)
        assert loss.shape == (2, 3) and stats.shape == (6, 4) and loss.dtype == torch.float32
        assert torch.ops.deberta_amd.distill_loss_bwd(loss, x, ids[..., None], x[..., :1], None, stats, 2.0).shape == x.shape
    with pytest.raises(NotImplementedError):
        torch.ops.deberta_amd.token_logprobs(torch.zeros(1, 8), None, 0, 1.0, -100)


# ---------------------------------------------------------------------------
# the C ABI


HEADER = ROOT / "include" / "dsa_vocab.h"
STRUCTS = (("dsa_logprobs_args", _lib.DsaLogprobsArgs), ("dsa_distill_args", _lib.DsaDistillArgs))


def test_header_matches_the_exports_and_structs(tmp_path):
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    assert sorted(set(re.findall(r"\b(dsa_[a-z_]+)\s*\([^;{]*\)\s*;", text))) == sorted(_lib.VOCAB_EXPORTS)
    lib = _lib.load()
    for name in _lib.VOCAB_EXPORTS:
        assert hasattr(lib, name), name
    limits = dict(re.findall(r"DSA_VOCAB_(\w+) = ([^,\n/]+)", text))
    assert int(limits["MAX_ENTRIES"]) == vocab.MAX_ENTRIES and eval(limits["MAX_TOP_V"]) == vocab.MAX_TOP_VOCAB
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    lines = [f'printf("{c} %zu\\n", sizeof({c}));' for c, _ in STRUCTS]
    lines += [f'printf("{c}.{f} %zu\\n", offsetof({c}, {f}));' for c, s in STRUCTS for f, _ in s._fields_]
    src = tmp_path / "probe.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "dsa_vocab.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0;\n}\n")
    subprocess.run([gcc, "-std=c99", "-I", str(HEADER.parent), str(src), "-o", str(tmp_path / "probe")], check=True)
    out = dict(line.rsplit(" ", 1) for line in subprocess.run([str(tmp_path / "probe")], capture_output=True, text=True).stdout.splitlines())
    for c, s in STRUCTS:
        assert int(out[c]) == ctypes.sizeof(s), c
        for f, _ in s._fields_:
            assert int(out[f"{c}.{f}"]) == getattr(s, f).offset, (c, f)


def _what_changes(v):
    """A case's name: the fields that it changes, without addresses, which differ
    from process to process."""
    return ",".join(v) if isinstance(v, dict) else str(v)


_KEEP = ctypes.create_string_buffer(4096)
_AT = (ctypes.addressof(_KEEP) + 255) // 256 * 256
_LOGPROBS = dict(logits=_AT, logits_stride=8, ids=_AT, ids_bytes=8, logprobs=_AT, entropy=_AT, lse=_AT, stats=_AT, N=2, V=8, dtype=0,
                 inv_temperature=1.0, dlogprobs=_AT, dlogits=_AT, dlogits_stride=8)
_DISTILL = dict(logits=_AT, logits_stride=8, teacher_ids=_AT, ids_bytes=8, teacher=_AT, loss=_AT, stats=_AT, dloss=_AT, dlogits=_AT,
                dlogits_stride=8, N=2, V=8, K=2, dtype=0, teacher_dtype=0, temperature=1.0)


@pytest.mark.parametrize("change,match", [
    (dict(dtype=2), "dtype"), (dict(N=-1), "N must"), (dict(N=(1 << 36) + 1), "N must"), (dict(V=0), "V must"), (dict(V=1 << 31), "V must"),
    (dict(inv_temperature=0.0), "inv_temperature"), (dict(inv_temperature=NAN), "inv_temperature"), (dict(inv_temperature=INF), "inv_temperature"),
    (dict(top_k=9), "top_k"), (dict(top_k=-1), "top_k"), (dict(top_k=1, V=(1 << 19) + 1, logits_stride=1 << 20, dlogits_stride=1 << 20), "at most"),
    (dict(ids_bytes=2), "ids_bytes"), (dict(logits=None), "logits are required"), (dict(logits=_AT + 2), "aligned"),
    (dict(logits_stride=-8), "stride"), (dict(ids=_AT + 4), "aligned"), (dict(stats=_AT + 4), "16-byte"),
], ids=_what_changes)
def test_logprobs_entry_points_refuse(change, match):
    lib = _lib.load()
    for name in ("dsa_logprobs_fwd", "dsa_logprobs_bwd"):
        assert getattr(lib, name)(ctypes.byref(_lib.DsaLogprobsArgs(**{**_LOGPROBS, **change})), None) != 0
        assert re.search(match, _lib.last_error()), _lib.last_error()


@pytest.mark.parametrize("name,change,match", [
    ("dsa_logprobs_fwd", dict(ids=None), "need ids"), ("dsa_logprobs_fwd", dict(top_k=2), "top_logprobs and top_ids"),
    ("dsa_logprobs_bwd", dict(stats=None), "stats are required"), ("dsa_logprobs_bwd", dict(dlogprobs=None), "a gradient"),
    ("dsa_logprobs_bwd", dict(ids=None), "need ids"), ("dsa_logprobs_bwd", dict(dtop=_AT), "top_k and top_ids"),
    ("dsa_logprobs_bwd", dict(dlogprobs_stride=2), "strides"), ("dsa_logprobs_bwd", dict(dlogits=None), "dlogits are required"),
    ("dsa_logprobs_bwd", dict(dlogits_stride=7), "overlap"), ("dsa_logprobs_bwd", dict(dlogits=_AT + 1), "aligned"),
], ids=_what_changes)
def test_logprobs_entry_points_refuse_what_one_needs(name, change, match):
    assert getattr(_lib.load(), name)(ctypes.byref(_lib.DsaLogprobsArgs(**{**_LOGPROBS, **change})), None) != 0
    assert re.search(match, _lib.last_error()), _lib.last_error()


@pytest.mark.parametrize("names,change,match", [
    ("both", dict(dtype=3), "dtype"), ("both", dict(teacher_dtype=3), "teacher_dtype"), ("both", dict(K=0), "K must"),
    ("both", dict(K=129), "K must"), ("both", dict(temperature=0.0), "temperature"), ("both", dict(temperature=NAN), "temperature"),
    ("both", dict(ids_bytes=1), "ids_bytes"), ("both", dict(teacher_ids=None), "teacher_ids"), ("both", dict(teacher=_AT + 1), "teacher's"),
    ("both", dict(logits=None), "logits are required"), ("both", dict(stats=_AT + 8), "16-byte"), ("dsa_distill_fwd", dict(loss=None), "loss"),
    ("dsa_distill_bwd", dict(stats=None), "stats and dloss"), ("dsa_distill_bwd", dict(dloss=None), "stats and dloss"),
    ("dsa_distill_bwd", dict(dloss_stride=3), "stride"), ("dsa_distill_bwd", dict(dlogits_stride=4), "overlap"),
], ids=_what_changes)
def test_distill_entry_points_refuse(names, change, match):
    for name in ("dsa_distill_fwd", "dsa_distill_bwd") if names == "both" else (names,):
        assert getattr(_lib.load(), name)(ctypes.byref(_lib.DsaDistillArgs(**{**_DISTILL, **change})), None) != 0
        assert re.search(match, _lib.last_error()), _lib.last_error()


def test_rows_in_parts_need_their_workspace():
    """Which the library sizes: for few long rows, for many bytes, and nothing
    for what one block a row reads."""
    lib, bytes_of = _lib.load(), _lib.load().dsa_vocab_workspace_bytes
    assert bytes_of(1, 128100, _lib.DSA_BF16, 0) > 0 and bytes_of(1, 128100, _lib.DSA_BF16, 5) > bytes_of(1, 128100, _lib.DSA_BF16, 0)
    assert bytes_of(1229, 128100, _lib.DSA_BF16, 0) > 0 and bytes_of(1229, 128100, _lib.DSA_BF16, 64) == 0
    assert bytes_of(512, 32768, _lib.DSA_BF16, 0) == 0 == bytes_of(0, 128100, _lib.DSA_F32, 0)
    # the most rows of the most columns: no product of theirs passes 64 bits
    assert 1 << 59 < bytes_of(1 << 36, (1 << 31) - 128, _lib.DSA_F32, 0) < 1 << 61
    a = {**_LOGPROBS, "V": 128100, "logits_stride": 128100, "N": 1}
    d = {**_DISTILL, "V": 128100, "logits_stride": 128100, "N": 1}
    need = bytes_of(1, 128100, _lib.DSA_F32, 0)
    for ws in (dict(), dict(workspace=_AT, workspace_bytes=need - 1), dict(workspace=_AT + 4, workspace_bytes=need)):
        assert lib.dsa_logprobs_fwd(ctypes.byref(_lib.DsaLogprobsArgs(**a, **ws)), None) != 0
        assert f"workspace needs {need} bytes" in _lib.last_error()
        assert lib.dsa_distill_fwd(ctypes.byref(_lib.DsaDistillArgs(**d, **ws)), None) != 0
        assert "workspace needs" in _lib.last_error()


def test_long_rows_go_in_parts():
    """However many bytes the rows are together, where they are few: a block reads a
    long row by itself for as long as it has columns, and its lanes add up as many
    terms one after the other."""
    bytes_of = _lib.load().dsa_vocab_workspace_bytes
    f32, bf16 = _lib.DSA_F32, _lib.DSA_BF16
    for N, V, dt, k in ((1, 10_000_000, f32, 0), (1, 20_000_000, f32, 0), (1, 1 << 25, bf16, 0), (36, 262144, f32, 0), (36, 262144, f32, 5),
                        (72, 262144, bf16, 5), (90, 262144, f32, 64), (20, 524288, f32, 5), (100, 524288, f32, 128), (100, 1 << 20, f32, 0), (100, 128100, f32, 5)):
        assert bytes_of(N, V, dt, k) > 0, (N, V, dt, k)
    # of more columns than this every row is, where no largest are asked for: a lane's chain
    # is 41 batches at most
    for N in (1, 10, 50, 100, 1000, 100_000):
        for V in (340_000, 1 << 20, 1 << 27):
            assert bytes_of(N, V, f32, 0) > 0 and bytes_of(N, V, bf16, 0) > 0, (N, V)
    # short rows are not, nor so many that whole ones fill the card
    for N, V, dt, k in ((1, 50021, f32, 0), (32, 64000, bf16, 0), (250, 262144, bf16, 0), (100, 128100, f32, 0), (200, 128100, bf16, 0), (8, 41000, f32, 5),
                        (200, 128100, bf16, 20), (256, 262144, f32, 64)):
        assert bytes_of(N, V, dt, k) == 0, (N, V, dt, k)


def test_null_arguments_are_errors():
    lib = _lib.load()
    for name in _lib.VOCAB_EXPORTS[1:]:
        assert getattr(lib, name)(None, None) != 0 and name in _lib.last_error()


# ---------------------------------------------------------------------------
# the head


def test_cpu_head_learns_and_predicts():
    """Its three uses on CPU tensors, against torch operations."""
    from types import SimpleNamespace

    torch.manual_seed(0)
    head = da.FusedMLMHead(SimpleNamespace(hidden_size=16, vocab_size=50, layer_norm_eps=1e-7))
    weight = torch.nn.Parameter(torch.randn(50, 16) * 0.1)
    assert sorted(head.state_dict()) == ["LayerNorm.bias", "LayerNorm.weight", "bias", "dense.bias", "dense.weight"]
    hidden, labels = torch.randn(2, 5, 16), torch.randint(0, 50, (2, 5))
    labels[0, :3] = -100
    loss, rows = head.forward_loss(hidden, weight, labels)
    want = torch.nn.functional.cross_entropy(head(hidden, weight).view(-1, 50), labels.view(-1))
    assert (loss - want).abs() < 1e-5 and rows.entropy.shape == (2, 5)
    loss.backward()
    assert weight.grad is not None and head.bias.grad.abs().sum() > 0
    best = head.predict(hidden, weight, top_k=3)
    assert torch.equal(best.top_ids[..., 0], head(hidden, weight).argmax(-1)) and not best.top_logprobs.requires_grad
    distil = head.forward_distillation(hidden, weight, best.top_ids, best.top_logprobs, 2.0)
    assert distil.requires_grad and distil.item() > 0
    none, _ = head.forward_loss(hidden, weight, torch.full((2, 5), -100))
    assert none == 0
