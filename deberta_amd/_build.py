"""Builds ``libdsa.so`` (the HIP kernels and their C ABI) in-tree with hipcc for
gfx950, and ``_hidden_ext.so`` (the host side of the operators on hidden
states and on a vocabulary's logits: PyTorch tensors and autograd over that C
ABI) with g++, or the ROCm toolchain's own clang++ where there is no g++."""

from __future__ import annotations

import os
import shutil
import subprocess
import sysconfig
import tempfile
import warnings
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
CSRC_DIR = PKG_DIR / "csrc"
LIB_PATH = PKG_DIR / "libdsa.so"
# (source, macros): one translation unit each, compiled in parallel and linked
SOURCES = (
    ("dsa_inst.hip", ("-DDSA_T=bf16", "-DDSA_D=64")),
    ("dsa_inst.hip", ("-DDSA_T=float", "-DDSA_D=64")),
    ("dsa_inst.hip", ("-DDSA_T=bf16", "-DDSA_D=32")),
    ("dsa_inst.hip", ("-DDSA_T=float", "-DDSA_D=32")),
    ("dsa_capi.hip", ()),
    ("dsa_hidden.hip", ()),
    ("dsa_rms_inst.hip", ("-DDSA_TX=bf16", "-DDSA_TR=bf16")),
    ("dsa_rms_inst.hip", ("-DDSA_TX=bf16", "-DDSA_TR=float")),
    ("dsa_rms_inst.hip", ("-DDSA_TX=float", "-DDSA_TR=bf16")),
    ("dsa_rms_inst.hip", ("-DDSA_TX=float", "-DDSA_TR=float")),
    ("dsa_vocab.hip", ()),
)
# bench.py's MFMA throughput probe (include/dsa_probe.h), a library of its own
PROBE_PATH = PKG_DIR / "libdsa_probe.so"
PROBE_SOURCES = (("dsa_probe.hip", ()),)
# the operators on hidden states and logits for PyTorch tensors: host code (it includes vocab_ext.h), linked to libdsa.so
EXT_PATH = PKG_DIR / "_hidden_ext.so"
EXT_SOURCE = CSRC_DIR / "hidden_ext.cpp"
ARCH = "gfx950"

# Packed fp32 VALU ops are kept out of the generated code: hipcc otherwise
# forms v_pk_{add,mul,fma}_f32 from plain float arithmetic.
HIPCC_FLAGS = (
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-Xclang",
    "-target-feature",
    "-Xclang",
    "-packed-fp32-ops",
)


def hipcc_path() -> str:
    """Locate hipcc (PATH first, then the ROCm install)."""
    found = shutil.which("hipcc")
    if found:
        return found
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    cand = Path(rocm) / "bin" / "hipcc"
    if cand.exists():
        return str(cand)
    raise RuntimeError("hipcc not found: libdsa.so cannot be built without the ROCm toolchain")


def _compile(sources, out: Path, verbose: bool) -> Path:
    """Compile every (source, macros) pair to an object, at most one hipcc per
    CPU at a time, and link them into ``out``."""
    with tempfile.TemporaryDirectory(dir=out.parent, prefix="_build") as tmp_dir:
        objs = [str(Path(tmp_dir) / f"{n}.o") for n in range(len(sources))]
        cmds = [
            [hipcc_path(), *HIPCC_FLAGS, "-c", *macros, str(CSRC_DIR / src), "-o", obj]
            for (src, macros), obj in zip(sources, objs)
        ]
        with ThreadPoolExecutor(max_workers=min(len(cmds), len(os.sched_getaffinity(0)))) as pool:
            list(pool.map(_run, cmds))
        tmp = out.with_suffix(".so.tmp")
        link = [hipcc_path(), f"--offload-arch={ARCH}", "-fPIC", "-shared", *objs, "-o", str(tmp)]
        _run(link)
        if verbose:
            for cmd in (*cmds, link):
                print(" ".join(cmd))
    os.replace(tmp, out)
    return out


def _host_compiler() -> str:
    """A C++ compiler for host code: hipcc brings one."""
    rocm = Path(os.environ.get("ROCM_PATH", "/opt/rocm"))
    for found in (shutil.which("g++"), shutil.which("c++"), rocm / "llvm" / "bin" / "clang++", shutil.which("clang++")):
        if found and Path(found).exists():
            return str(found)
    raise RuntimeError("no C++ compiler found: _hidden_ext.so cannot be built")


def _ext_include() -> list[Path]:
    """The extension's header folders: torch's, Python's and ROCm's."""
    import torch

    root = Path(torch.__file__).resolve().parent / "include"
    return [root, root / "torch" / "csrc" / "api" / "include", Path(sysconfig.get_paths()["include"]),
            Path(os.environ.get("ROCM_PATH", "/opt/rocm")) / "include"]


def _missing_headers() -> list[str]:
    """What the extension includes and this machine does not have (an
    installation of torch or Python without its C++ headers)."""
    torch_include, _, python_include, _ = _ext_include()
    need = (torch_include / "torch" / "csrc" / "autograd" / "custom_function.h", python_include / "Python.h")
    return [str(p) for p in need if not p.exists()]


def _ext_commands(obj: Path, out: Path) -> tuple[list[str], list[str]]:
    """(compile, link) of the extension.  It finds libdsa.so beside itself and
    torch's libraries where the process has loaded them."""
    import torch

    cxx, root, include = _host_compiler(), Path(torch.__file__).resolve().parent, _ext_include()
    flags = ["-O2", "-std=c++17", "-fPIC", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
             f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    compile_cmd = [cxx, *flags, *(f"-isystem{p}" for p in include), "-c", str(EXT_SOURCE), "-o", str(obj)]
    libs = ("torch", "torch_cpu", "torch_hip", "c10", "c10_hip", "torch_python")
    link_cmd = [cxx, "-shared", str(obj), f"-L{root / 'lib'}", *(f"-l{n}" for n in libs), f"-L{PKG_DIR}", "-l:libdsa.so",
                "-Wl,-rpath,$ORIGIN", "-o", str(out)]
    return compile_cmd, link_cmd


def _run(cmd) -> None:
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"{Path(cmd[0]).name} failed ({proc.returncode}):\n{' '.join(cmd)}\n{proc.stdout}\n{proc.stderr}")


def build(verbose: bool = False) -> Path:
    """Compile every source: ``deberta_amd/libdsa.so`` (the kernels and their
    C ABI), ``deberta_amd/libdsa_probe.so`` (the MFMA probe) and
    ``deberta_amd/_hidden_ext.so`` (the hidden-state and vocabulary operators'
    host side).

    Always recompiles.  Each library is written to a temporary name first and
    renamed into place, so a process that already loaded the old file keeps a
    consistent image.

    Where torch's or Python's C++ headers are not installed the kernels are
    built alone, with a warning: the operators on hidden states and logits then
    raise on device tensors, everything else runs.
    """
    missing = _missing_headers()
    if missing:
        warnings.warn(f"{EXT_PATH.name} is not built, {', '.join(missing)} not found: the operators on hidden states and logits will not run")
        EXT_PATH.unlink(missing_ok=True)  # not to be taken for this build's
        _compile(PROBE_SOURCES, PROBE_PATH, verbose)
        return _compile(SOURCES, LIB_PATH, verbose)
    with tempfile.TemporaryDirectory(dir=PKG_DIR, prefix="_build") as tmp_dir, ThreadPoolExecutor(1) as pool:
        tmp = EXT_PATH.with_suffix(".so.tmp")
        compile_cmd, link_cmd = _ext_commands(Path(tmp_dir) / "ext.o", tmp)
        ext = pool.submit(_run, compile_cmd)
        _compile(PROBE_SOURCES, PROBE_PATH, verbose)
        lib = _compile(SOURCES, LIB_PATH, verbose)
        ext.result()
        _run(link_cmd)
        os.replace(tmp, EXT_PATH)
        if verbose:
            print(" ".join(compile_cmd))
            print(" ".join(link_cmd))
    return lib


if __name__ == "__main__":
    print(build(verbose=True))
