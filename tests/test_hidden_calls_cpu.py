"""How calls of the hidden-state operators are routed and checked, without a
GPU: what goes past ``torch.ops`` into the extension and what must not, which
extension is loaded, where seeds are drawn, what the build needs, and what the
torch path of CPU tensors sums in.

A call on device tensors is seen here by letting CPU tensors say that they are
on the GPU: the extension then refuses those calls that reach its own part, and
those that it leaves to the registered op find no CPU kernel there.
"""

from __future__ import annotations

import ctypes
import re
import shutil
import subprocess
import types
from pathlib import Path

import pytest
import torch

import deberta_amd as da
from deberta_amd import _build, _lib, hidden
from oracle import hidden as oh
from tests._hidden import Wrapper


@pytest.fixture
def as_on_gpu(monkeypatch):
    """CPU tensors that say they are on the GPU."""
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))


def _calls(x, bias, res, w, ids):
    return {
        "dropout": lambda: da.fused_dropout(x, 0.5, bias=bias, res=res, seed=1),
        "rms": lambda: da.fused_add_rms_norm(x, w, bias=bias, res=res),
        "quant": lambda: da.fused_add_rms_norm_fp8(x, w, bias=bias, res=res),
        "embed": lambda: da.fused_embedding(ids, x),
    }


def test_plain_tensors_go_into_the_extension(as_on_gpu):
    x, w = torch.randn(3, 8), torch.nn.Parameter(torch.ones(8), requires_grad=False)
    for call in _calls(x, w, x, w, torch.tensor([1])).values():
        with pytest.raises(ValueError, match="must be on the GPU"):  # its check, on what it was given
            call()


@pytest.mark.parametrize("which", ["bias", "res", "weight", "ids"])
def test_a_wrapper_in_any_argument_sees_the_op(which, as_on_gpu):
    """The extension reads addresses, and a wrapper has none: a bias or a
    residual of that kind would be left out of the result."""
    x, b, r, w, ids = torch.randn(3, 8), torch.ones(8), torch.randn(3, 8), torch.ones(8), torch.tensor([1])
    if which == "bias":
        b = Wrapper(b)
    elif which == "res":
        r = Wrapper(r)
    elif which == "weight":
        w = Wrapper(w)
    else:
        ids = Wrapper(ids)
    reached = {"bias": ("dropout", "rms", "quant"), "res": ("dropout", "rms", "quant"), "weight": ("rms", "quant"),
               "ids": ("embed",)}[which]
    calls = _calls(x, b, r, w, ids)
    for name in reached:
        Wrapper.seen.clear()
        with pytest.raises(NotImplementedError):  # the op, on tensors that are on the CPU after all
            calls[name]()
        assert any("deberta_amd" in str(f) for f in Wrapper.seen), name


def test_a_traced_call_is_the_op(as_on_gpu, monkeypatch):
    """torch.jit.trace records what the extension allocates, not what it
    launches: a trace of its calls would return memory that nothing wrote."""
    seen = []

    def op(name):  # an exception inside the tracer would leave it half done
        return lambda *args: seen.append(name) or (args[1] if name == "embed" else (args[0], args[0], args[0]))

    names = ["hidden_dropout", "add_rms_norm", "add_rms_norm_quant", "embed"]
    for name in names:
        monkeypatch.setattr(torch.ops.deberta_amd, name, op(name))
    x, w, ids = torch.randn(3, 8), torch.ones(8), torch.tensor([1])

    def f(v):
        for call in _calls(x, w, x, w, ids).values():
            call()
        return v + 1

    torch.jit.trace(f, (x,), check_trace=False)
    assert seen == names


@pytest.mark.parametrize("wt", [torch.bfloat16, torch.float16, torch.float32])
def test_cpu_embedding_gradient_sums_in_float32(wt):
    """A token at 4000 positions: 4000 additions in float32 and one rounding,
    on the sum of magnitudes (torch's own gradient of a bf16 table stops
    growing at 256 times a position's)."""
    u, h = 2.0**-24, torch.finfo(wt).eps / 2
    table = torch.randn(5, 6, generator=torch.Generator().manual_seed(1)).to(wt).requires_grad_()
    ids = torch.full((4000,), 3)
    ids[::1000] = 1
    for out, dy in ((wt, torch.ones(4000, 6, dtype=wt)),
                    (torch.float32, torch.randn(4000, 6, generator=torch.Generator().manual_seed(2)))):
        y = da.fused_embedding(ids, table, padding_idx=1, scale=0.5, out_dtype=out)
        assert y.dtype == out and torch.equal(y, (table.detach().float()[ids] * 0.5).to(out))
        (g,) = torch.autograd.grad(y, table, dy)
        want = oh.embedding_grad(ids, dy.double(), 5, 1, 0.5)
        most = oh.embedding_grad(ids, dy.double().abs(), 5, 1, 0.5)
        assert g.dtype == wt and ((g.double() - want).abs() <= 4001 * u * most + h * want.abs()).all()


@pytest.fixture
def fresh_ext():
    hidden._ext.cache_clear()
    yield
    hidden._ext.cache_clear()


@pytest.mark.parametrize("change", [None, {"abi_version": -1}, {"torch_version": "1.0.0"}], ids=str)
def test_an_extension_of_another_build_is_refused(change, fresh_ext, monkeypatch):
    """It would pass structs of another layout to the library."""
    own = hidden._ext()
    old = types.ModuleType("_hidden_ext")  # change None: one from before the versions were kept
    if change is not None:
        vars(old).update({"abi_version": own.abi_version, "torch_version": own.torch_version, **change})
    monkeypatch.setattr(da, "_hidden_ext", old)
    hidden._ext.cache_clear()
    with pytest.raises(RuntimeError, match="rebuild"):
        hidden._ext()


def test_the_headers_version_is_the_loaders():
    header = (Path(__file__).resolve().parents[1] / "include" / "dsa.h").read_text()
    (version,) = re.findall(r"#define DSA_VERSION (\d+)", header)
    assert int(version) == _lib.EXPECTED_VERSION == _lib.load().dsa_version() == hidden._ext().abi_version


def test_the_build_without_gcc_takes_rocms_compiler(monkeypatch, tmp_path):
    """hipcc needs no g++, and neither does the extension."""
    which = shutil.which
    monkeypatch.setattr(shutil, "which", lambda name: None if name in ("g++", "c++") else which(name))
    compile_cmd, _ = _build._ext_commands(tmp_path / "ext.o", tmp_path / "ext.so")
    assert Path(compile_cmd[0]).name == "clang++"
    subprocess.run([*(a for a in compile_cmd if a != "-O2"), "-fsyntax-only"], check=True)


def test_the_build_without_torchs_headers_builds_the_kernels(monkeypatch, tmp_path):
    built = []
    monkeypatch.setattr(_build, "_compile", lambda sources, out, verbose: built.append(out) or out)
    monkeypatch.setattr(_build, "_ext_include", lambda: [tmp_path] * 4)
    monkeypatch.setattr(_build, "EXT_PATH", tmp_path / "_hidden_ext.so")
    _build.EXT_PATH.write_text("an earlier build's")
    with pytest.warns(UserWarning, match="custom_function.h"):
        assert _build.build() == _build.LIB_PATH
    assert built == [_build.PROBE_PATH, _build.LIB_PATH] and not _build.EXT_PATH.exists()


def test_seeds_are_on_the_cpu_whatever_the_default_device():
    """As under torch.set_default_device("cuda"): a seed of the default device
    was refused, and would have been drawn from its generator."""
    x = torch.ones(4, 100)
    torch.manual_seed(3)
    want = da.fused_dropout(x, 0.5), da.fused_dropout(x, 0.5, seed=9), da.hidden_keep_mask(4, 100, 0.5, 9)
    torch.manual_seed(3)
    with torch.device("meta"):
        got = da.fused_dropout(x, 0.5), da.fused_dropout(x, 0.5, seed=9), da.hidden_keep_mask(4, 100, 0.5, 9)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_embedding_from_a_given_table():
    """nn.Embedding's constructor for a given table, which passes arguments
    that FusedEmbedding's own does not take."""
    table = torch.randn(9, 4)
    ids = torch.tensor([[0, 8, 2]])
    emb = da.FusedEmbedding.from_pretrained(table, padding_idx=-1, scale=3.0)
    assert emb.weight.data_ptr() == table.data_ptr() and not emb.weight.requires_grad and emb.padding_idx == 8
    assert type(emb) is da.FusedEmbedding and (emb.num_embeddings, emb.embedding_dim) == (9, 4)
    assert torch.equal(emb(ids), table[ids] * 3.0) and torch.equal(table[8], emb.weight[8])
    emb = da.FusedEmbedding.from_pretrained(table, freeze=False)
    emb(ids).sum().backward()
    assert emb.weight.grad[0].eq(1).all() and emb.weight.grad[1].eq(0).all()
    with pytest.raises(ValueError, match="shape"):
        da.FusedEmbedding.from_pretrained(table[0])


def test_the_embeddings_backward_refuses_columns_past_32_bit_offsets():
    """Its byte offsets inside a row are 32-bit: 2^30 float32 columns."""
    lib = _lib.load()
    keep = ctypes.create_string_buffer(512)
    at = (ctypes.addressof(keep) + 255) // 256 * 256
    args = dict(ids=at, ids_bytes=8, dy=at, dy_stride=8, dweight=at, N=2, V=5, padding=-1, scale=1.0)
    for C, match in (((1 << 30) + 1, "2\\^30 columns"), (1 << 30, "workspace")):
        assert lib.dsa_embed_bwd(ctypes.byref(_lib.DsaEmbedArgs(C=C, **args)), None) != 0
        assert re.search(match, _lib.last_error())


def test_the_library_holds_no_norm_kernel_that_no_width_reaches():
    """Lanes, chunks and waves a row of the norm's kernels in the library: the
    forward's two chunks a lane and the backward's one between 2049 and 8192
    columns, and what both take elsewhere."""
    nm = shutil.which("nm")
    if nm is None:
        pytest.skip("nm not available")
    names = subprocess.run([nm, "-C", str(_lib.LIB_PATH)], capture_output=True, text=True, check=True).stdout
    both = {(16, 1, 1), (32, 1, 1), (64, 1, 1), (64, 2, 1), (64, 1, 4), (64, 2, 16)}
    for kernel, between in (("rms_fwd_kernel", {(64, 2, 4), (64, 2, 8)}), ("rms_bwd_kernel", {(64, 1, 8), (64, 1, 16)})):
        found = re.findall(kernel + r"<(\d+), (\d+), (\d+)", names)
        assert {tuple(map(int, t)) for t in found} == both | between


@pytest.mark.parametrize("group", [None, 64])
def test_cpu_bytes_round_the_product_that_the_kernel_rounds(group):
    """y * (448 / m), not y / (m / 448): a few bytes in a million differ, and
    CPU tensors would not give the GPU's."""
    x, w = torch.randn(4096, 512, generator=torch.Generator().manual_seed(1)), 1 + 0.2 * torch.randn(512, generator=torch.Generator().manual_seed(2))
    q, scale, _ = da.fused_add_rms_norm_fp8(x, w, group_size=group)
    y = da.fused_rms_norm(x, w).unflatten(-1, (512 // (group or 512), group or 512))
    m = y.abs().amax(-1, keepdim=True)
    most = torch.full_like(m, 448.0)
    assert torch.equal(scale, (m / most).squeeze(-1))
    want = (y * (most / m)).clamp(-448, 448).flatten(-2).to(torch.float8_e4m3fn)
    assert torch.equal(q.view(torch.uint8), want.view(torch.uint8))


def test_cpu_bytes_of_a_group_that_is_not_finite():
    x = torch.ones(3, 64)
    x[0, 3], x[1, 40] = float("inf"), float("nan")
    q, scale, _ = da.fused_add_rms_norm_fp8(x, torch.ones(64), group_size=32)
    # an infinity leaves a norm of 0 in its row but for inf * 0
    assert scale[0, 0].isnan() and q[0, :32].float().isnan().all() and scale[0, 1] == 1 and (q[0, 32:].float() == 0).all()
    assert scale[1].isnan().all() and q[1].float().isnan().all() and q[2].float().isfinite().all()
