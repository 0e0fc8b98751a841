"""The operators on hidden states without a GPU: the keep bits against the
oracle's, the torch path of CPU tensors against float64, the oracle's own
gradients against differences, refusals of the functions and of the C entry
points (before any device work), and the ops' fake implementations.

The CPU path computes in float32: a sum of three terms and a norm over C <= 40
values lose at most about C + 8 half steps of 2^-24 on the scale of the
largest term of the row; values here are below 8, so 48 * 2^-24 * 8 < 3e-5
holds for outputs and 1e-4 for gradients, which multiply two of them.
"""

from __future__ import annotations

import ctypes
import re
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

import pytest
import torch

import deberta_amd as da
from deberta_amd import _lib, hidden
from oracle import hidden as oh

ROOT = Path(__file__).resolve().parents[1]
SEED = 0x1234_5678_9ABC


def _rand(*shape, seed=0, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64).to(dtype)


@pytest.mark.parametrize("rows,C,p", [(1, 1, 0.5), (3, 7, 0.1), (5, 8, 0.9), (17, 65, 0.25), (2, 768, 0.1)])
def test_keep_bits_match_the_oracle(rows, C, p):
    got = da.hidden_keep_mask(rows, C, p, SEED)
    assert torch.equal(got, oh.keep_mask(rows, C, round(p * 65536), SEED))


def test_keep_bits_of_far_rows_use_both_words_of_the_row():
    a = oh.keep_mask([5], 64, 32768, SEED)
    assert not torch.equal(a, oh.keep_mask([5 + (1 << 32)], 64, 32768, SEED))


def test_dropped_share_and_the_ends_of_p():
    keep = da.hidden_keep_mask(512, 512, 0.1, 7)
    # 2^18 draws of probability 0.1: five standard deviations are 0.003
    assert abs(1.0 - keep.float().mean().item() - 0.1) < 0.003
    assert da.hidden_keep_mask(4, 9, 0.0, 7).all() and not da.hidden_keep_mask(4, 9, 1.0, 7).any()


# p = 1 without a residual leaves zeros, whose norm's gradient goes by 1 / sqrt(eps)
@pytest.mark.parametrize("p,with_bias,with_res", [(p, b, r) for p in (0.0, 0.3, 1.0)
                                                  for b, r in ((False, False), (True, True), (False, True)) if p < 1 or r])
def test_cpu_path_matches_float64(p, with_bias, with_res):
    x, w = _rand(2, 5, 40, seed=1), 1 + 0.1 * _rand(40, seed=2)
    bias = _rand(40, seed=3) if with_bias else None
    res = _rand(2, 5, 40, seed=4) if with_res else None
    t = round(p * 65536)
    dy, dz = _rand(2, 5, 40, seed=5), _rand(2, 5, 40, seed=6)

    def run(fn, dtype):
        leaves = [v.to(dtype).requires_grad_() for v in (x, w, bias, res) if v is not None]
        it = iter(leaves)
        args = [next(it), next(it), next(it) if with_bias else None, next(it) if with_res else None]
        outs = fn(*args)
        live = [(o, g) for o, g in zip(outs, (dy.to(dtype), dz.to(dtype), dz.to(dtype))) if o.requires_grad]
        grads = torch.autograd.grad([o for o, _ in live], leaves, [g for _, g in live], allow_unused=True)
        return [o.detach() for o in outs], [torch.zeros(()) if g is None else g for g in grads]

    def ours(x, w, b, r):
        y, z = da.fused_add_rms_norm(x, w, 1e-6, bias=b, res=r, dropout_p=p, seed=SEED)
        return y, z, da.fused_dropout(x, p, bias=b, res=r, seed=SEED)

    def ref(x, w, b, r):
        z = oh.dropout_add(x, b, r, t, SEED)
        return oh.rms_norm(z, w, 1e-6), z, z

    for tol, a, b in zip((3e-5, 1e-4), run(ours, torch.float32), run(ref, torch.float64)):
        for u, v in zip(a, b):
            assert (u.double() - v).abs().max().item() <= tol


def test_cpu_path_of_float64_tensors_computes_in_float64():
    x, w, bias, res = _rand(3, 40, seed=1, dtype=torch.float64), _rand(40, seed=2), _rand(40, seed=3), _rand(3, 40, seed=4)
    t = round(0.3 * 65536)
    z = oh.dropout_add(x, bias.double(), res.double(), t, SEED)
    y = oh.rms_norm(z, w.double(), 1e-6)
    got_y, got_z = da.fused_add_rms_norm(x, w, 1e-6, bias=bias, res=res, dropout_p=0.3, seed=SEED)
    # 48 half steps of 2^-53 on values below 32: 2e-13
    for got, want in ((got_y, y), (got_z, z), (da.fused_dropout(x, 0.3, bias=bias, res=res, seed=SEED), z)):
        assert got.dtype == torch.float64 and (got - want).abs().max().item() < 2e-13
    ids, table = torch.tensor([2, 0]), _rand(3, 40, seed=5, dtype=torch.float64)
    assert torch.equal(da.fused_embedding(ids, table, scale=0.3), table[ids] * 0.3)
    leaves = [v.double().requires_grad_() for v in (x, w, bias, res)]
    assert torch.autograd.gradcheck(
        lambda x, w, b, r: da.fused_add_rms_norm(x, w, 1e-6, bias=b, res=r, dropout_p=0.3, seed=SEED), leaves)


def test_cpu_embedding_and_its_gradient():
    w = _rand(11, 6, seed=1).requires_grad_()
    ids = torch.tensor([[3, 0, 3], [10, 2, 0]])
    y = da.fused_embedding(ids, w, padding_idx=0, scale=2.5)
    dy = _rand(2, 3, 6, seed=2)
    (dw,) = torch.autograd.grad(y, w, dy)
    assert torch.allclose(y.double(), oh.embedding(ids, w.detach().double(), 2.5), rtol=1e-6)
    assert torch.allclose(dw.double(), oh.embedding_grad(ids, dy.double(), 11, 0, 2.5), rtol=1e-6, atol=1e-6)
    assert da.fused_embedding(ids, w, out_dtype=torch.bfloat16).dtype == torch.bfloat16


@pytest.mark.parametrize("group", [None, 32])
def test_cpu_fp8(group):
    x, w = _rand(3, 64, seed=1), 1 + 0.1 * _rand(64, seed=2)
    x[1] = 0.0
    x[2, 40] = float("nan")
    q, scale, z = da.fused_add_rms_norm_fp8(x, w, group_size=group)
    assert q.dtype == torch.float8_e4m3fn and z is x and scale.shape == (3, 2 if group else 1)
    want = oh.rms_norm(x.double(), w.double(), 1e-6)
    got = q.float().double() * scale.double().repeat_interleave(64 // scale.shape[1], 1)
    # half a step of e4m3 is 2^-4 of the value, or 2^-10 scales where it is subnormal
    assert ((got - want)[0].abs() <= 2.0**-4 * want[0].abs() * (1 + 1e-5) + 2.0**-10 * scale[0].max()).all()
    assert (scale[1] == 1).all() and (q[1].float() == 0).all()
    assert got[2].isnan().all()


def test_the_oracles_gradients_against_differences():
    x, w, b, r = (v.requires_grad_() for v in (_rand(3, 9, seed=1, dtype=torch.float64), _rand(9, seed=2, dtype=torch.float64),
                                               _rand(9, seed=3, dtype=torch.float64), _rand(3, 9, seed=4, dtype=torch.float64)))

    def f(x, w, b, r):
        z = oh.dropout_add(x, b, r, 20000, SEED)
        return oh.rms_norm(z, w, 1e-6), z

    assert torch.autograd.gradcheck(f, (x, w, b, r))
    ids = torch.tensor([1, 4, 1, 0, 4, 4])
    table = _rand(5, 3, seed=5, dtype=torch.float64).requires_grad_()
    assert torch.autograd.gradcheck(lambda t: oh.embedding(ids, t, 1.5), (table,))
    dy = _rand(6, 3, seed=6, dtype=torch.float64)
    (dw,) = torch.autograd.grad(oh.embedding(ids, table, 1.5), table, dy)
    assert torch.allclose(dw, oh.embedding_grad(ids, dy, 5, -1, 1.5))


def test_seeds():
    x = torch.ones(4, 100)
    torch.manual_seed(3)
    a, b = da.fused_dropout(x, 0.5), da.fused_dropout(x, 0.5)
    assert not torch.equal(a, b)
    torch.manual_seed(3)
    assert torch.equal(da.fused_dropout(x, 0.5), a)
    s = torch.tensor([9], dtype=torch.int64)
    assert torch.equal(da.fused_dropout(x, 0.5, seed=s), da.fused_dropout(x, 0.5, seed=9))
    assert da.fused_dropout(x, 0.5, training=False) is x and da.fused_dropout(x, 0.0) is x
    for bad in (-1, 1 << 63, 1.5, torch.tensor([1.0]), torch.tensor([1, 2])):
        with pytest.raises(ValueError, match="seed"):
            da.fused_dropout(x, 0.5, seed=bad)


def test_refusals():
    x, w = torch.randn(3, 8), torch.ones(8)
    for p in (-0.1, 1.1, float("nan"), 2.0**-18, 1 - 2.0**-18):
        with pytest.raises(ValueError, match="probability"):
            da.fused_dropout(x, p)
    with pytest.raises(ValueError, match="x's shape"):
        da.fused_dropout(x, 0.5, res=torch.randn(8))
    with pytest.raises(ValueError, match="bias"):
        da.fused_dropout(x, 0.5, bias=torch.randn(7))
    with pytest.raises(ValueError, match="last dimension"):
        da.fused_dropout(torch.tensor(1.0), 0.5)
    with pytest.raises(ValueError, match="weight"):
        da.fused_rms_norm(x, torch.ones(9))
    for g in (0, 16, 48, 1024, 64):
        with pytest.raises(ValueError, match="group_size"):
            da.fused_add_rms_norm_fp8(torch.randn(2, 96), torch.ones(96), group_size=g)
    with pytest.raises(RuntimeError, match="no gradient"):
        da.fused_add_rms_norm_fp8(x, w.clone().requires_grad_())
    with pytest.raises(TypeError, match="ids"):
        da.fused_embedding(torch.tensor([1.0]), torch.randn(4, 4))
    with pytest.raises(ValueError, match="padding_idx"):
        da.fused_embedding(torch.tensor([1]), torch.randn(4, 4), padding_idx=4)
    with pytest.raises(ValueError, match="weight"):
        da.fused_embedding(torch.tensor([1]), torch.randn(4))


# --- the C entry points ------------------------------------------------------------------
def _lib_or_fail():
    if not _lib.LIB_PATH.exists():
        pytest.fail(f"{_lib.LIB_PATH} is not built (run python -m deberta_amd._build)")
    return _lib.load()


def test_structs_match_the_c_header(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    structs = (("dsa_dropout_args", _lib.DsaDropoutArgs), ("dsa_rms_args", _lib.DsaRmsArgs), ("dsa_embed_args", _lib.DsaEmbedArgs))
    lines = [f'printf("{c} %zu\\n", sizeof({c}));' for c, _ in structs]
    lines += [f'printf("{c}.{f} %zu\\n", offsetof({c}, {f}));' for c, s in structs for f, _ in s._fields_]
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "dsa_block.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0;\n}\n")
    subprocess.run([gcc, "-std=c99", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    out = dict(ln.rsplit(" ", 1) for ln in subprocess.run([str(exe)], capture_output=True, text=True).stdout.splitlines())
    for c, s in structs:
        assert int(out[c]) == ctypes.sizeof(s), c
        for f, _ in s._fields_:
            assert int(out[f"{c}.{f}"]) == getattr(s, f).offset, (c, f)
    header = (ROOT / "include" / "dsa_block.h").read_text()
    for name, value in re.findall(r"(DSA_BLOCK_[A-Z]+) = (\d+)", header):
        assert getattr(_lib, name) == int(value)


def _buffers():
    keep = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(keep) + 255) // 256 * 256
    return keep, at


def _refused(entry, a, match):
    """The call fails with this message (in a thread of its own: the error text
    is the thread's)."""
    lib = _lib_or_fail()

    def call():
        return getattr(lib, entry)(None if a is None else ctypes.byref(a), None), _lib.last_error()

    with ThreadPoolExecutor(1) as pool:
        rc, text = pool.submit(call).result()
    assert rc != 0 and re.search(match, text), (rc, text)


def test_dropout_entry_refuses():
    keep, at = _buffers()
    good = dict(x=at, x_stride=8, y=at, y_stride=8, N=2, C=8, threshold=100)
    for entry in ("dsa_dropout_fwd", "dsa_dropout_bwd", "dsa_add_rms_fwd", "dsa_add_rms_quant", "dsa_add_rms_bwd",
                  "dsa_embed_fwd", "dsa_embed_bwd"):
        _refused(entry, None, "null arguments")
    for change, match in (
        (dict(N=0), "N in"), (dict(N=1 << 31), "N in"), (dict(C=0), "C >= 1"), (dict(threshold=65537), "threshold"),
        (dict(x=None), "bad x"), (dict(x=at + 2), "bad x"), (dict(x_stride=-1), "bad x"), (dict(x_dtype=2), "bad x"),
        (dict(res=at + 1, rows_per_group=2), "bad res"), (dict(res=at), "bad res"), (dict(bias=at, bias_dtype=7), "bad bias"),
        (dict(y_dtype=_lib.DSA_BF16), "bad y"),
    ):
        _refused("dsa_dropout_fwd", _lib.DsaDropoutArgs(**{**good, **change}), match)
    back = dict(dy=at, dy_stride=8, dx=at, dx_stride=8, N=2, C=8, threshold=100)
    for change, match in ((dict(dx=None), "dx or dbias"), (dict(dbias=at, N=100000), "workspace"), (dict(dy=None), "bad dy")):
        _refused("dsa_dropout_bwd", _lib.DsaDropoutArgs(**{**back, **change}), match)


def test_rms_entry_refuses():
    keep, at = _buffers()
    good = dict(x=at, x_stride=64, weight=at, y=at, y_stride=64, z=at, z_stride=64, rstd=at, scales=at, N=2, C=64)
    for entry, change, match in (
        ("dsa_add_rms_fwd", dict(C=16385), r"C in \[1, 16384\]"),
        ("dsa_add_rms_fwd", dict(weight=None), "bad weight"),
        ("dsa_add_rms_bwd", dict(dy=at, dy_stride=64, rstd=None), "rstd"),
        ("dsa_add_rms_fwd", dict(y_stride=63), "bad y"),
        ("dsa_add_rms_fwd", dict(z_stride=63), "bad z"),
        ("dsa_add_rms_fwd", dict(threshold=70000), "threshold"),
        ("dsa_add_rms_quant", dict(scales=None), "scales"),
        ("dsa_add_rms_quant", dict(group_size=48), "group_size"),
        ("dsa_add_rms_quant", dict(group_size=128), "group_size"),
        ("dsa_add_rms_quant", dict(group_size=16), "group_size"),
        ("dsa_add_rms_bwd", dict(dy=None), "bad dy"),
        ("dsa_add_rms_bwd", dict(dy=at, dy_stride=64, dweight=at), "workspace"),
        ("dsa_add_rms_bwd", dict(dy=at, dy_stride=64, dres=at), "bad dres"),
        ("dsa_add_rms_bwd", dict(dy=at, dy_stride=64, dbias=at), "bad dbias"),
    ):
        _refused(entry, _lib.DsaRmsArgs(**{**good, **change}), match)


def test_embed_entry_refuses():
    keep, at = _buffers()
    good = dict(ids=at, ids_bytes=8, weight=at, weight_stride=8, y=at, y_stride=8, N=2, V=5, C=8, padding=-1, scale=1.0)
    for change, match in (
        (dict(V=0), "V in"), (dict(V=(1 << 31) - 1), "V in"), (dict(ids_bytes=2), "int64 or int32"), (dict(ids=at + 4), "bad ids"),
        (dict(weight=None), "bad weight"), (dict(y=None), "bad y"),
    ):
        _refused("dsa_embed_fwd", _lib.DsaEmbedArgs(**{**good, **change}), match)
    for change, match in (
        (dict(dy=None), "bad dy"), (dict(dy=at, dy_stride=8), "dweight"), (dict(dy=at, dy_stride=8, dweight=at + 8), "dweight"),
        (dict(dy=at, dy_stride=8, dweight=at), "workspace"),
    ):
        _refused("dsa_embed_bwd", _lib.DsaEmbedArgs(**{**good, **change}), match)


def test_workspaces_cover_the_partial_sums():
    lib = _lib_or_fail()
    for N in (1, 63, 64, 5000, 16384, 300000):
        for C in (1, 8, 513, 768, 4096):
            # up to 16 rows a thread of at most 512 one block takes all and needs none
            assert lib.dsa_block_workspace_bytes(_lib.DSA_BLOCK_DROPOUT, N, C) >= (8 * C if N > 16 * 512 else 0)
            assert lib.dsa_block_workspace_bytes(_lib.DSA_BLOCK_RMS, N, C) >= 8 * C
            # keys and positions, and two partial sums a chunk of at most 64 positions
            assert lib.dsa_embed_workspace_bytes(N, C, 1000) >= 8 * N + 2 * C * 4 * -(-N // 64)
    assert lib.dsa_embed_workspace_bytes(0, 8, 5) == 0


# --- the host side for PyTorch tensors ---------------------------------------------------
def test_extension_is_built_and_refuses_cpu_tensors():
    ext = hidden._ext()
    x, w = torch.randn(3, 8), torch.ones(8)
    for call in (lambda: ext.dropout(x, None, None, 100, torch.tensor([1])), lambda: ext.rms(x, None, None, w, 1e-6, x.dtype, 0, None),
                 lambda: ext.quant(x, None, None, w, 1e-6, 0), lambda: ext.embed(torch.tensor([1]), x, -1, 1.0, x.dtype),
                 lambda: ext.embed_bwd(x, torch.tensor([0, 1, 2]), 4, x.dtype, -1, 1.0)):
        with pytest.raises(ValueError, match="must be on the GPU"):
            call()


# --- the ops -----------------------------------------------------------------------------
def test_fake_shapes_and_cpu_refusal():
    from torch._subclasses.fake_tensor import FakeTensorMode

    ops = torch.ops.deberta_amd
    with FakeTensorMode():
        x, res, w = torch.randn(2, 8, 64, dtype=torch.bfloat16), torch.randn(2, 8, 64), torch.randn(64)
        seed = torch.zeros(1, dtype=torch.int64)
        assert ops.hidden_dropout(x, w, res, 100, seed).dtype == torch.float32
        y, z, rstd = ops.add_rms_norm(x, w, res, w, 1e-6, torch.bfloat16, 100, seed)
        assert y.dtype == torch.bfloat16 and z.dtype == torch.float32 and z.shape == x.shape and rstd.shape == (16,)
        assert ops.add_rms_norm(x, None, None, w, 1e-6, torch.bfloat16, 0, None)[1].shape == (0,)
        dx, dres, dw, db = ops.add_rms_norm_bwd(y, z, x, w, res, w, rstd, 100, seed)
        assert dx.dtype == x.dtype and dres.dtype == res.dtype and dw.shape == db.shape == (64,)
        q, s, z = ops.add_rms_norm_quant(x, None, res, w, 1e-6, 32)
        assert q.dtype == torch.float8_e4m3fn and s.shape == (2, 8, 2) and z.dtype == torch.float32
        ids = torch.zeros(2, 8, dtype=torch.int64)
        e = ops.embed(ids, torch.randn(10, 64), -1, 1.0, torch.bfloat16)
        assert e.shape == (2, 8, 64) and e.dtype == torch.bfloat16
        assert ops.embed_bwd(e, ids, 10, torch.float32, -1, 1.0).shape == (10, 64)
    with pytest.raises(NotImplementedError):
        ops.hidden_dropout(torch.randn(2, 64), None, None, 100, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(NotImplementedError):
        ops.embed(torch.zeros(2, dtype=torch.int64), torch.randn(4, 4), -1, 1.0, torch.float32)


def test_modules():
    norm = da.FusedRMSNorm(16, eps=1e-5)
    x, res = torch.randn(3, 16), torch.randn(3, 16)
    assert torch.equal(norm(x), da.fused_rms_norm(x, norm.weight, 1e-5))
    y, z = norm(x, res)
    assert torch.equal(z, x + res)
    drop = da.FusedDropout(0.5).eval()
    assert drop(x) is x
    y, z = da.FusedRMSNorm(16, dropout_p=0.1).eval()(x)
    assert z is x
    emb = da.FusedEmbedding(9, 4, padding_idx=-1, scale=3.0)
    ref = torch.nn.Embedding(9, 4, padding_idx=-1)
    ref.load_state_dict(emb.state_dict(), strict=True)
    ids = torch.tensor([[0, 8, 2]])
    assert torch.allclose(emb(ids), ref(ids) * 3.0)
    assert hidden.norm_out_dtype(x.bfloat16(), res) == torch.float32


def test_rtd_head_with_rms_norm_on_cpu():
    from oracle import eager

    cfg = eager.make_config(hidden_size=32, num_attention_heads=4, intermediate_size=64, layer_norm_eps=1e-7, use_rmsnorm_heads=True)
    head = da.FusedRTDHead(cfg).eval()
    assert set(head.state_dict()) == {"dense.weight", "dense.bias", "norm.weight", "classifier.weight", "classifier.bias"}
    with torch.no_grad():
        head.norm.weight.mul_(1.5)
    h = _rand(2, 6, 32, seed=3)
    z = h.double() + h[:, :1].double()
    y = oh.rms_norm(z, head.norm.weight.double(), head.norm.eps)
    y = torch.nn.functional.gelu(y @ head.dense.weight.double().T + head.dense.bias.double())
    want = (y @ head.classifier.weight.double().T + head.classifier.bias.double()).squeeze(-1)
    assert (head(h).double() - want).abs().max().item() <= 1e-5


def test_fused_hidden_dropout_on_cpu():
    """dense without its bias, then bias, dropout and residual at once: the
    same as by hand with the same seed."""
    from oracle import eager

    cfg = eager.make_config(hidden_size=32, num_attention_heads=4, intermediate_size=64, layer_norm_eps=1e-7,
                            hidden_dropout_prob=0.25, fused_hidden_dropout=True)
    m = da.FusedSelfOutput(cfg).train()
    x, res = _rand(2, 6, 32, seed=3), _rand(2, 6, 32, seed=4)
    torch.manual_seed(11)
    got = m(x, res)
    torch.manual_seed(11)
    seed = int(hidden.draw_dropout_seed().item())
    z = oh.dropout_add(x.double() @ m.dense.weight.double().T, m.dense.bias.double(), res.double(), 16384, seed)
    want = torch.nn.functional.layer_norm(z, (32,), m.LayerNorm.weight.double(), m.LayerNorm.bias.double(), 1e-7)
    assert (got.double() - want).abs().max().item() <= 3e-5
    assert torch.equal(m.eval()(x, res), da.FusedSelfOutput.forward(m, x, res))
