"""Calls of the hidden-state operators on the GPU that need care on the way to
the kernels: tensors without memory of their own, wrapped and traced calls,
views with a pending sign, more rows than one launch holds, teams that take
several rows.  Tolerances as in test_gpu_hidden.py."""

from __future__ import annotations

import pytest
import torch

import deberta_amd as da
from deberta_amd import hidden
from tests._hidden import Wrapper

pytestmark = pytest.mark.gpu

FP = torch.float32
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
        lambda: ext.dropout(x, Wrapper(w), None, 100, seed),
        lambda: ext.dropout(x, None, None, 100, Wrapper(seed)),
    ):
        with pytest.raises(ValueError, match="no memory"):
            call()
