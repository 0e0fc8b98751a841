"""Operators on a layer's hidden states, on the HIP kernels of libdsa.so
(include/dsa_block.h):

  fused_embedding          token lookup with scaling; its gradient sums the
                           positions of each token in their order (no float
                           atomics: equal inputs give equal bits)
  fused_dropout            dropout(x + bias) + res; the keep bits come from a
                           counter-based generator, no mask is stored
  fused_add_rms_norm       z = dropout(x + bias) + res and y = RMSNorm(z)
  fused_rms_norm           RMSNorm(x)
  fused_add_rms_norm_fp8   the same with y in float8_e4m3fn and scales, for
                           serving

and the modules FusedEmbedding, FusedDropout and FusedRMSNorm on them.

The kernels take float32 and bfloat16 tensors of any width, row stride and
element alignment; arithmetic, sums and statistics are float32, and every
result is rounded once.  In plain eager mode the functions go through
csrc/hidden_ext.cpp (checks, memory, launches and autograd nodes in C++: the
host time of a call is what bounds these operators on small batches).  CPU
tensors run the same operators in torch operations (float64 ones in float64),
dropout with the same keep bits.  The ops under the functions
(``deberta_amd::hidden_dropout``, ``add_rms_norm``, ``add_rms_norm_quant``,
``embed`` and the backwards) take device tensors only; like the package's
other ops they have fake implementations and autograd, are not twice
differentiable, and refuse a stream that is capturing a HIP graph.

Dropout's keep bits are a function of a 64-bit seed and the position: the
value at row r (all leading dimensions flattened) and column c is kept where
16 bits of Philox4x32-10 (J. K. Salmon, M. A. Moraes, R. O. Dror, D. E. Shaw,
"Parallel random numbers: as easy as 1, 2, 3", SC 2011) with counter ``(c // 8,
r & 0xffffffff, r >> 32, 0x68696464)`` and the seed's low and high words as the
key, of word ``(c % 8) // 2`` the low half for even c and the high half for odd
c, are at least ``round(65536 p)``.  Kept values are scaled by 65536 / (65536 -
round(65536 p)).  A dropped value is 0 whatever it was (a NaN or an infinity
included).
"""

from __future__ import annotations

import functools
from typing import Any, Optional, Union

import torch
import torch.nn as nn
from torch import Tensor

from deberta_amd import _eager, _lib
from deberta_amd._build import EXT_PATH
from deberta_amd.ops import draw_dropout_seed, dropout_threshold

_TAGS = (torch.Tag.cudagraph_unsafe,)  # as the package's other ops
_MASK32 = 0xFFFFFFFF
_DOMAIN = 0x68696464  # the last word of hidden dropout's counters
FP8_MAX = 448.0  # the largest value of float8_e4m3fn
MAX_RMS_WIDTH = 16384


@functools.lru_cache(maxsize=None)
def _ext() -> Any:
    """The host side of the operators on the GPU (csrc/hidden_ext.cpp).  Its
    functions named like an operator return None for a call that the registered
    op has to see: one that is traced, or with a wrapper among its tensors."""
    _lib.load()  # and checks its version
    if not EXT_PATH.exists():
        raise RuntimeError(
            f"{EXT_PATH} is missing: the operators on hidden states are not built. Run `python -m deberta_amd._build` first."
        )
    from deberta_amd import _hidden_ext

    # an extension left from an earlier build would pass its own structs to the library, or hold torch's older ones
    built = (getattr(_hidden_ext, "abi_version", None), getattr(_hidden_ext, "torch_version", None))
    need = (_lib.EXPECTED_VERSION, torch.__version__.split("+")[0])
    if built != need:
        raise RuntimeError(f"{EXT_PATH} was built for (ABI, torch) versions {built}, expected {need}; rebuild it")
    return _hidden_ext


def _cpu_args(what: str, x: Tensor, bias: Optional[Tensor], res: Optional[Tensor], weight: Optional[Tensor] = None) -> None:
    """The checks of the torch path."""
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"{what}: x needs a last dimension of at least one column, got shape {tuple(x.shape)}")
    for name, t in (("bias", bias), ("weight", weight)):
        if t is not None and tuple(t.shape) != (x.shape[-1],):
            raise ValueError(f"{what} {name} must have shape ({x.shape[-1]},), got {tuple(t.shape)}")
    if res is not None and res.shape != x.shape:
        raise ValueError(f"{what}: res must have x's shape {tuple(x.shape)}, got {tuple(res.shape)}")
    for name, t in (("bias", bias), ("res", res), ("weight", weight)):
        if t is not None and t.device != x.device:
            raise ValueError(f"{what}: {name} is on {t.device}, x is on {x.device}")


def _stream_dtype(x: Tensor, res: Optional[Tensor]) -> torch.dtype:
    return x.dtype if res is None else torch.promote_types(x.dtype, res.dtype)


def _wide_dtype(t: torch.dtype) -> torch.dtype:
    """The type that the torch path computes results of type t in."""
    return torch.promote_types(t, torch.float32)


# ---------------------------------------------------------------------------
# dropout's arguments


def _threshold(p: float) -> int:
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability must be in [0, 1], got {p}")
    t = dropout_threshold(p)
    if t in (0, 65536) and p not in (0.0, 1.0):
        raise ValueError(f"dropout probability {p} has no form in units of 1/65536 (0 < p < 2^-17 or 1 - 2^-17 < p < 1)")
    return t


def _seed_tensor(seed: Union[None, int, Tensor]) -> Tensor:
    if seed is None:
        return draw_dropout_seed()
    if isinstance(seed, int) and not isinstance(seed, bool):
        if not 0 <= seed < 1 << 63:
            raise ValueError(f"dropout seed must be in [0, 2^63), got {seed}")
        return torch.tensor([seed], dtype=torch.int64, device="cpu")
    if not isinstance(seed, Tensor) or seed.numel() != 1 or seed.dtype != torch.int64 or seed.device.type != "cpu":
        raise ValueError("dropout seed must be an int or an int64 CPU tensor of one element")
    return seed


def hidden_keep_mask(rows: int, C: int, p: float, seed: Union[int, Tensor], device: Union[str, torch.device] = "cpu") -> Tensor:
    """Hidden dropout's keep bits as a ``(rows, C)`` bool tensor, in torch
    operations (the kernels never store them)."""
    t, s = _threshold(p), int(_seed_tensor(seed).item())
    groups = (C + 7) // 8
    r = torch.arange(rows, device=device)[:, None]
    c0 = torch.arange(groups, device=device)[None, :].expand(rows, groups)
    c1, c2 = (r & _MASK32).expand(rows, groups), (r >> 32).expand(rows, groups)
    c3 = torch.full_like(c0, _DOMAIN)
    k0, k1 = s & _MASK32, (s >> 32) & _MASK32
    for _ in range(10):  # 64-bit products wrap; their two words are exact
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (p1 >> 32 & _MASK32) ^ c1 ^ k0, p1 & _MASK32, (p0 >> 32 & _MASK32) ^ c3 ^ k1, p0 & _MASK32
        k0, k1 = (k0 + 0x9E3779B9) & _MASK32, (k1 + 0xBB67AE85) & _MASK32
    words = torch.stack([c0, c1, c2, c3], dim=-1)
    return torch.stack([words & 0xFFFF, words >> 16], dim=-1).reshape(rows, 8 * groups)[:, :C] >= t


def _cpu_sum(x: Tensor, bias: Optional[Tensor], res: Optional[Tensor], t: int, seed: Optional[Tensor]) -> Tensor:
    """dropout(x + bias) + res in torch operations, not rounded."""
    wide = _wide_dtype(_stream_dtype(x, res))
    z = x.to(wide)
    if bias is not None:
        z = z + bias.to(wide)
    if t:
        C = x.shape[-1]
        keep = hidden_keep_mask(x.numel() // C, C, t / 65536.0, seed, x.device).view(x.shape)
        z = torch.where(keep, z * (65536.0 / (65536 - t) if t < 65536 else 0.0), 0.0)
    return z if res is None else z + res.to(wide)


# ---------------------------------------------------------------------------
# dropout


def _hidden_dropout_impl(
    x: Tensor, bias: Optional[Tensor], res: Optional[Tensor], dropout_t: int, dropout_seed: Optional[Tensor]
) -> Tensor:
    """``dropout(x + bias) + res`` in x's type promoted with res's."""
    return _ext().dropout_fwd(x, bias, res, dropout_t, dropout_seed)


def _hidden_dropout_bwd_impl(
    dy: Tensor, dx_dtype: torch.dtype, bias_dtype: Optional[torch.dtype], dropout_t: int, dropout_seed: Optional[Tensor]
) -> tuple[Tensor, Tensor]:
    """(dx in ``dx_dtype``, dbias in ``bias_dtype``, empty where that is None)."""
    return _ext().dropout_bwd(dy, dx_dtype, bias_dtype, dropout_t, dropout_seed)


hidden_dropout = torch.library.custom_op(
    "deberta_amd::hidden_dropout", _hidden_dropout_impl, mutates_args=(), device_types="cuda", tags=_TAGS
)
hidden_dropout_bwd = torch.library.custom_op(
    "deberta_amd::hidden_dropout_bwd", _hidden_dropout_bwd_impl, mutates_args=(), device_types="cuda", tags=_TAGS
)


@hidden_dropout.register_fake
def _hidden_dropout_fake(x, bias, res, dropout_t, dropout_seed):
    return x.new_empty(x.shape, dtype=_stream_dtype(x, res))


@hidden_dropout_bwd.register_fake
def _hidden_dropout_bwd_fake(dy, dx_dtype, bias_dtype, dropout_t, dropout_seed):
    dbias = dy.new_empty((0 if bias_dtype is None else dy.shape[-1],), dtype=bias_dtype or dx_dtype)
    return dy.new_empty(dy.shape, dtype=dx_dtype), dbias


def _hidden_dropout_setup(ctx, inputs, output):
    x, bias, res, dropout_t, seed = inputs
    ctx.save_for_backward(seed)
    ctx.dropout_t, ctx.x_dtype = dropout_t, x.dtype
    ctx.bias_dtype = None if bias is None else bias.dtype
    ctx.res_dtype = None if res is None else res.dtype


def _hidden_dropout_backward(ctx, dy):
    (seed,) = ctx.saved_tensors
    dx = dbias = dres = None
    for_x, for_bias, for_res = ctx.needs_input_grad[:3]
    if for_x or for_bias:
        dx, dbias = hidden_dropout_bwd(dy, ctx.x_dtype, ctx.bias_dtype if for_bias else None, ctx.dropout_t, seed)
    if for_res:
        dres = dy if dy.dtype is ctx.res_dtype else dy.to(ctx.res_dtype)
    return dx, (dbias if for_bias else None), dres, None, None


torch.library.register_autograd("deberta_amd::hidden_dropout", _hidden_dropout_backward, setup_context=_hidden_dropout_setup)


def fused_dropout(
    x: Tensor,
    p: float,
    bias: Optional[Tensor] = None,
    res: Optional[Tensor] = None,
    training: bool = True,
    seed: Union[None, int, Tensor] = None,
) -> Tensor:
    """``dropout(x + bias) + res`` in one kernel, in x's type promoted with
    res's.  ``bias`` has shape ``(C,)``; ``res`` has x's shape (a view
    broadcast along the second of three dimensions is read in place).

    ``p`` is rounded to a multiple of 1/65536.  ``seed``: an int in [0, 2^63)
    or an int64 CPU tensor of one element; by default one is drawn from
    torch's CPU generator (``torch.manual_seed`` reproduces it, and activation
    checkpointing draws the same one again).  Calls with one seed and one
    shape drop the same positions."""
    t = _threshold(p) if training else 0
    if not t and bias is None and res is None:
        return x
    s = _seed_tensor(seed) if t else None
    if not x.is_cuda:
        _cpu_args("fused_dropout", x, bias, res)
        return _cpu_sum(x, bias, res, t, s).to(_stream_dtype(x, res))
    if _eager.eager(x):
        y = _ext().dropout(x, bias, res, t, s)
        if y is not None:
            return y
    return torch.ops.deberta_amd.hidden_dropout(x, bias, res, t, s)


# ---------------------------------------------------------------------------
# residual + RMS norm


def _plain(bias: Optional[Tensor], res: Optional[Tensor], dropout_t: int) -> bool:
    """z is x itself."""
    return bias is None and res is None and not dropout_t


def _add_rms_norm_impl(
    x: Tensor,
    bias: Optional[Tensor],
    res: Optional[Tensor],
    weight: Tensor,
    eps: float,
    out_dtype: torch.dtype,
    dropout_t: int,
    dropout_seed: Optional[Tensor],
) -> tuple[Tensor, Tensor, Tensor]:
    """(y in ``out_dtype``, z = dropout(x + bias) + res, 1 / rms per row); z is
    empty where it is x itself."""
    return _ext().rms_fwd(x, bias, res, weight, eps, out_dtype, dropout_t, dropout_seed)


def _add_rms_norm_bwd_impl(
    dy: Tensor,
    dz: Optional[Tensor],
    x: Tensor,
    bias: Optional[Tensor],
    res: Optional[Tensor],
    weight: Tensor,
    rstd: Tensor,
    dropout_t: int,
    dropout_seed: Optional[Tensor],
) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """(dx, dres, dweight, dbias) for the gradients of y and (optional) of z.
    dres is empty without a residual and where it equals dx (no dropout, one
    type); dbias is empty without a bias."""
    return _ext().rms_bwd(dy, dz, x, bias, res, weight, rstd, dropout_t, dropout_seed)


def _add_rms_norm_quant_impl(
    x: Tensor, bias: Optional[Tensor], res: Optional[Tensor], weight: Tensor, eps: float, group_size: int
) -> tuple[Tensor, Tensor, Tensor]:
    """(y as float8_e4m3fn, its scales, z); z is empty where it is x itself.
    ``group_size`` 0: one scale a row."""
    return _ext().quant_fwd(x, bias, res, weight, eps, group_size)


add_rms_norm = torch.library.custom_op(
    "deberta_amd::add_rms_norm", _add_rms_norm_impl, mutates_args=(), device_types="cuda", tags=_TAGS
)
add_rms_norm_bwd = torch.library.custom_op(
    "deberta_amd::add_rms_norm_bwd", _add_rms_norm_bwd_impl, mutates_args=(), device_types="cuda", tags=_TAGS
)
add_rms_norm_quant = torch.library.custom_op(
    "deberta_amd::add_rms_norm_quant", _add_rms_norm_quant_impl, mutates_args=(), device_types="cuda", tags=_TAGS
)


@add_rms_norm.register_fake
def _add_rms_norm_fake(x, bias, res, weight, eps, out_dtype, dropout_t, dropout_seed):
    z = x.new_empty((0,) if _plain(bias, res, dropout_t) else x.shape, dtype=_stream_dtype(x, res))
    return x.new_empty(x.shape, dtype=out_dtype), z, x.new_empty((x.numel() // x.shape[-1],), dtype=torch.float32)


@add_rms_norm_bwd.register_fake
def _add_rms_norm_bwd_fake(dy, dz, x, bias, res, weight, rstd, dropout_t, dropout_seed):
    apart = res is not None and (dropout_t or res.dtype != x.dtype)
    return (
        x.new_empty(x.shape),
        x.new_empty(x.shape if apart else (0,), dtype=res.dtype if apart else x.dtype),
        weight.new_empty(weight.shape),
        bias.new_empty(bias.shape) if bias is not None else weight.new_empty((0,)),
    )


@add_rms_norm_quant.register_fake
def _add_rms_norm_quant_fake(x, bias, res, weight, eps, group_size):
    groups = x.shape[-1] // group_size if group_size else 1
    z = x.new_empty((0,) if _plain(bias, res, 0) else x.shape, dtype=_stream_dtype(x, res))
    return (
        x.new_empty(x.shape, dtype=torch.float8_e4m3fn),
        x.new_empty((*x.shape[:-1], groups), dtype=torch.float32),
        z,
    )


def _add_rms_norm_setup(ctx, inputs, output):
    x, bias, res, weight, eps, out_dtype, dropout_t, seed = inputs
    y, z, rstd = output
    ctx.mark_non_differentiable(*((rstd, z) if _plain(bias, res, dropout_t) else (rstd,)))
    ctx.save_for_backward(x, bias, res, weight, rstd, seed)
    ctx.dropout_t, ctx.out_dtype = dropout_t, out_dtype
    ctx.set_materialize_grads(False)


def _add_rms_norm_backward(ctx, dy, dz, drstd):
    x, bias, res, weight, rstd, seed = ctx.saved_tensors
    if dy is None and dz is None:
        return (None,) * 8
    if dy is None:  # only z was used
        dy = torch.zeros(x.shape, dtype=ctx.out_dtype, device=x.device)
    dx, dres, dweight, dbias = add_rms_norm_bwd(dy, dz, x, bias, res, weight, rstd, ctx.dropout_t, seed)
    if res is None:
        dres = None
    elif not (ctx.dropout_t or res.dtype != x.dtype):
        dres = dx
    return dx, (dbias if bias is not None else None), dres, dweight, None, None, None, None


torch.library.register_autograd("deberta_amd::add_rms_norm", _add_rms_norm_backward, setup_context=_add_rms_norm_setup)


def norm_out_dtype(x: Tensor, res: Optional[Tensor]) -> torch.dtype:
    """A norm's result type: float32 under CUDA autocast (torch runs its
    norms in float32 there), else the promoted type of its inputs."""
    if torch.is_autocast_enabled("cuda"):
        return torch.float32
    return _stream_dtype(x, res)


def fused_add_rms_norm(
    x: Tensor,
    weight: Tensor,
    eps: float = 1e-6,
    bias: Optional[Tensor] = None,
    res: Optional[Tensor] = None,
    dropout_p: float = 0.0,
    training: bool = True,
    seed: Union[None, int, Tensor] = None,
    out_dtype: Optional[torch.dtype] = None,
) -> tuple[Tensor, Tensor]:
    """``(y, z)`` in one kernel: the residual stream ``z = dropout(x + bias) +
    res`` in x's type promoted with res's (x itself where there is nothing to
    add or drop), and its norm ``y = z / sqrt(mean(z^2) + eps) * weight`` in
    ``out_dtype`` (by default float32 under autocast, else z's type).

    y is computed from z before z is rounded.  The squares are summed in
    float32: a row whose squares pass its range (values over about 1e17) has
    the norm 0.  ``dropout_p``, ``training`` and ``seed`` as in
    :func:`fused_dropout`.  Rows of at most 16384 columns."""
    t = _threshold(dropout_p) if training else 0
    s = _seed_tensor(seed) if t else None
    out_dtype = norm_out_dtype(x, res) if out_dtype is None else out_dtype
    if not x.is_cuda:
        _cpu_args("fused_add_rms_norm", x, bias, res, weight)
        z = _cpu_sum(x, bias, res, t, s)
        y = z * torch.rsqrt(z.square().mean(-1, keepdim=True) + eps) * weight.to(z.dtype)
        return y.to(out_dtype), (x if _plain(bias, res, t) else z.to(_stream_dtype(x, res)))
    if _eager.eager(x):
        out = _ext().rms(x, bias, res, weight, float(eps), out_dtype, t, s)
        if out is not None:
            return out
    y, z, _ = torch.ops.deberta_amd.add_rms_norm(x, bias, res, weight, float(eps), out_dtype, t, s)
    return y, (x if _plain(bias, res, t) else z)


def fused_rms_norm(x: Tensor, weight: Tensor, eps: float = 1e-6, out_dtype: Optional[torch.dtype] = None) -> Tensor:
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension (see
    :func:`fused_add_rms_norm`)."""
    return fused_add_rms_norm(x, weight, eps, out_dtype=out_dtype)[0]


def fused_add_rms_norm_fp8(
    x: Tensor,
    weight: Tensor,
    eps: float = 1e-6,
    bias: Optional[Tensor] = None,
    res: Optional[Tensor] = None,
    group_size: Optional[int] = None,
) -> tuple[Tensor, Tensor, Tensor]:
    """``(q, scales, z)``: :func:`fused_add_rms_norm` without dropout, with y in
    8 bits for the next matrix product: ``y = q * scales``, q float8_e4m3fn of
    x's shape and scales float32 ``(..., 1)``, one a row, or ``(..., C /
    group_size)``, one for each ``group_size`` columns (32, 64, 128, 256 or 512).

    With m the group's largest ``|y|`` the scale is m / 448 and q is ``y * (448 /
    m)`` rounded to nearest even, both in float32 (a y between two bytes may go
    to the other one than ``y / scale`` would): m itself becomes 448.  A group of zeros (or
    below the normal float32 range) has the scale 1 and q 0; one with a NaN or an
    infinity has the scale NaN and q NaN.  For serving: there is no gradient,
    and a call under autograd whose inputs need one raises."""
    g = 0 if group_size is None else int(group_size)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, res)):
        raise RuntimeError("fused_add_rms_norm_fp8 has no gradient: call it under torch.no_grad()")
    if group_size is not None and g == 0:
        raise ValueError("group_size must be 32, 64, 128, 256 or 512, or None for one scale a row")
    if not x.is_cuda:
        _cpu_args("fused_add_rms_norm_fp8", x, bias, res, weight)
        C = x.shape[-1]
        if g and (g not in (32, 64, 128, 256, 512) or C % g):
            raise ValueError(f"group_size must be 32, 64, 128, 256 or 512 and divide the width {C}, got {g}")
        z = _cpu_sum(x, bias, res, 0, None)
        y = z * torch.rsqrt(z.square().mean(-1, keepdim=True) + eps) * weight.to(z.dtype)
        y = y.unflatten(-1, (C // (g or C), g or C))
        top = y.abs().amax(-1, keepdim=True)
        tiny, finite = top < FP8_MAX * 2.0**-126, top.isfinite()
        scale = torch.where(finite, torch.where(tiny, 1.0, top / FP8_MAX), torch.nan)
        # a tensor above: torch divides a number through the reciprocal
        factor = torch.where(finite, torch.where(tiny, 1.0, torch.full_like(top, FP8_MAX) / top), torch.nan)
        q = (y * factor).clamp(-FP8_MAX, FP8_MAX).flatten(-2).to(torch.float8_e4m3fn)
        return q, scale.squeeze(-1).float(), (x if _plain(bias, res, 0) else z.to(_stream_dtype(x, res)))
    if _eager.eager(x):
        out = _ext().quant(x, bias, res, weight, float(eps), g)
        if out is not None:
            return out
    q, scale, z = torch.ops.deberta_amd.add_rms_norm_quant(x, bias, res, weight, float(eps), g)
    return q, scale, (x if _plain(bias, res, 0) else z)


# ---------------------------------------------------------------------------
# embedding


def _embed_impl(ids: Tensor, weight: Tensor, padding_idx: int, scale: float, out_dtype: torch.dtype) -> Tensor:
    """``scale * weight[ids]`` in ``out_dtype``; a row of NaN where an id is
    outside the table.  ``padding_idx`` (-1: none) matters to the gradient
    only."""
    return _ext().embed_fwd(ids, weight, padding_idx, scale, out_dtype)


def _embed_bwd_impl(
    dy: Tensor, ids: Tensor, num_embeddings: int, weight_dtype: torch.dtype, padding_idx: int, scale: float
) -> Tensor:
    """The gradient of the whole table, in ``weight_dtype``."""
    return _ext().embed_bwd(dy, ids, num_embeddings, weight_dtype, padding_idx, scale)


embed = torch.library.custom_op("deberta_amd::embed", _embed_impl, mutates_args=(), device_types="cuda", tags=_TAGS)
embed_bwd = torch.library.custom_op("deberta_amd::embed_bwd", _embed_bwd_impl, mutates_args=(), device_types="cuda", tags=_TAGS)


@embed.register_fake
def _embed_fake(ids, weight, padding_idx, scale, out_dtype):
    return weight.new_empty((*ids.shape, weight.shape[1]), dtype=out_dtype)


@embed_bwd.register_fake
def _embed_bwd_fake(dy, ids, num_embeddings, weight_dtype, padding_idx, scale):
    return dy.new_empty((num_embeddings, dy.shape[-1]), dtype=weight_dtype)


def _embed_setup(ctx, inputs, output):
    ids, weight, padding_idx, scale, _ = inputs
    ctx.save_for_backward(ids)
    ctx.table = (weight.shape[0], weight.dtype, padding_idx, scale)


def _embed_backward(ctx, dy):
    (ids,) = ctx.saved_tensors
    return None, embed_bwd(dy, ids, *ctx.table), None, None, None


torch.library.register_autograd("deberta_amd::embed", _embed_backward, setup_context=_embed_setup)


def fused_embedding(
    ids: Tensor,
    weight: Tensor,
    padding_idx: Optional[int] = None,
    scale: float = 1.0,
    out_dtype: Optional[torch.dtype] = None,
) -> Tensor:
    """``scale * weight[ids]`` in ``out_dtype`` (by default weight's type), for
    int64 or int32 ``ids`` of any shape.

    The gradient is dense, in weight's type: for each token the sum over its
    positions in their order, in float32; zero for the padding token
    (``padding_idx``, negative from the end) and tokens that do not occur.  An
    id outside the table gives a row of NaN and adds to no gradient (on CPU
    tensors torch raises)."""
    if weight.dim() != 2:
        raise ValueError(f"fused_embedding: weight must be (V, C), got shape {tuple(weight.shape)}")
    V = weight.shape[0]
    if padding_idx is None:
        pad = -1
    else:
        if not -V <= padding_idx < V:
            raise ValueError(f"fused_embedding: padding_idx {padding_idx} is outside the table of {V} rows")
        pad = padding_idx % V
    out_dtype = weight.dtype if out_dtype is None else out_dtype
    if not weight.is_cuda:
        if ids.dtype not in (torch.int64, torch.int32):
            raise TypeError(f"fused_embedding: ids must be int64 or int32, got {ids.dtype}")
        wide = _wide_dtype(weight.dtype)
        if torch.is_grad_enabled() and weight.requires_grad:
            weight = weight.to(wide)  # before the lookup: its gradient sums a token's positions in this type
        y = torch.nn.functional.embedding(ids, weight, padding_idx=None if pad < 0 else pad)
        return (y.to(wide) * scale).to(out_dtype)
    if _eager.eager(weight):
        y = _ext().embed(ids, weight, pad, float(scale), out_dtype)
        if y is not None:
            return y
    return torch.ops.deberta_amd.embed(ids, weight, pad, float(scale), out_dtype)


# ---------------------------------------------------------------------------
# modules


class FusedEmbedding(nn.Embedding):
    """``nn.Embedding`` (its parameter, its state dict) on
    :func:`fused_embedding`, with a scale (``sqrt(embedding_dim)`` in some
    models) and an output type of its own, e.g. bfloat16 from float32
    weights."""

    def __init__(
        self,
        num_embeddings: int,
        embedding_dim: int,
        padding_idx: Optional[int] = None,
        scale: float = 1.0,
        out_dtype: Optional[torch.dtype] = None,
        device=None,
        dtype=None,
    ) -> None:
        super().__init__(num_embeddings, embedding_dim, padding_idx, device=device, dtype=dtype)
        self.scale = float(scale)
        self.out_dtype = out_dtype

    @classmethod
    def from_pretrained(
        cls,
        embeddings: Tensor,
        freeze: bool = True,
        padding_idx: Optional[int] = None,
        scale: float = 1.0,
        out_dtype: Optional[torch.dtype] = None,
    ) -> "FusedEmbedding":
        """A module on the given ``(V, C)`` table (not a copy), as
        ``nn.Embedding.from_pretrained``."""
        if embeddings.dim() != 2:
            raise ValueError(f"FusedEmbedding: embeddings must be (V, C), got shape {tuple(embeddings.shape)}")
        emb = cls(*embeddings.shape, padding_idx, scale, out_dtype, device="meta")
        emb.weight = nn.Parameter(embeddings, requires_grad=not freeze)
        return emb

    def forward(self, ids: Tensor) -> Tensor:
        return fused_embedding(ids, self.weight, self.padding_idx, self.scale, self.out_dtype)


class FusedDropout(nn.Module):
    """:func:`fused_dropout` with the module's ``p``, in training mode."""

    def __init__(self, p: float = 0.5) -> None:
        super().__init__()
        _threshold(p)
        self.p = float(p)

    def forward(self, x: Tensor, bias: Optional[Tensor] = None, res: Optional[Tensor] = None) -> Tensor:
        return fused_dropout(x, self.p, bias=bias, res=res, training=self.training)

    def extra_repr(self) -> str:
        return f"p={self.p}"


class FusedRMSNorm(nn.Module):
    """:func:`fused_add_rms_norm` with the module's ``weight``: ``(y, z)`` with
    the residual stream z; only y where the module has no ``dropout_p`` and
    neither ``res`` nor ``bias`` is given (z is then x)."""

    def __init__(self, hidden_size: int, eps: float = 1e-6, dropout_p: float = 0.0, device=None, dtype=None) -> None:
        super().__init__()
        _threshold(dropout_p)
        self.weight = nn.Parameter(torch.ones(hidden_size, device=device, dtype=dtype))
        self.eps = float(eps)
        self.dropout_p = float(dropout_p)

    def forward(self, x: Tensor, res: Optional[Tensor] = None, bias: Optional[Tensor] = None):
        if res is None and bias is None and not self.dropout_p:
            return fused_rms_norm(x, self.weight, self.eps)
        return fused_add_rms_norm(
            x, self.weight, self.eps, bias=bias, res=res, dropout_p=self.dropout_p, training=self.training
        )

    def extra_repr(self) -> str:
        return f"{self.weight.shape[0]}, eps={self.eps}, dropout_p={self.dropout_p}"
