"""The operators on hidden states restated in float64 on the CPU: hidden
dropout, the residual RMS norm (and its 8-bit output) and the embedding.

TEST INFRASTRUCTURE ONLY (see oracle/__init__.py).

Everything is written in torch operations that autograd differentiates, so
that a parity test takes the gradients from here; the keep bits come from
``oracle.dropout.philox4x32_10`` (numpy, pinned by published vectors).
"""

from __future__ import annotations

from typing import Optional

import numpy as np
import torch

from oracle.dropout import philox4x32_10

DOMAIN = 0x68696464
FP8_MAX = 448.0


def keep_mask(rows, C: int, threshold: int, seed: int) -> torch.Tensor:
    """Hidden dropout's kept positions, bool ``(len(rows), C)``: value (r, c)
    by the 16-bit half ``c % 2`` of word ``(c % 8) // 2`` of Philox4x32-10 at
    counter (c // 8, r low, r high, DOMAIN) under the seed's words.  ``rows``:
    row numbers, or their count."""
    r = np.arange(rows, dtype=np.uint64) if isinstance(rows, int) else np.asarray(rows, dtype=np.uint64)
    groups = (C + 7) // 8
    ctr = np.empty((len(r), groups, 4), dtype=np.uint64)
    ctr[..., 0] = np.arange(groups, dtype=np.uint64)[None, :]
    ctr[..., 1] = (r & np.uint64(0xFFFFFFFF))[:, None]
    ctr[..., 2] = (r >> np.uint64(32))[:, None]
    ctr[..., 3] = DOMAIN
    x = philox4x32_10(ctr, (seed & 0xFFFFFFFF, seed >> 32))
    halves = np.stack([x & np.uint32(0xFFFF), x >> np.uint32(16)], axis=-1)
    return torch.from_numpy(halves.reshape(len(r), 8 * groups)[:, :C].astype(np.int64) >= threshold)


def dropout_add(
    x: torch.Tensor,
    bias: Optional[torch.Tensor],
    res: Optional[torch.Tensor],
    threshold: int,
    seed: int,
) -> torch.Tensor:
    """``dropout(x + bias) + res``: kept values scaled by 65536 / (65536 -
    threshold), dropped ones 0 whatever they were."""
    z = x if bias is None else x + bias
    if threshold:
        keep = keep_mask(x.numel() // x.shape[-1], x.shape[-1], threshold, seed).view(x.shape)
        z = torch.where(keep, z, torch.zeros((), dtype=z.dtype))
        if threshold < 65536:
            z = z * (65536.0 / (65536 - threshold))
    return z if res is None else z + res


def rms_norm(z: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    return z / torch.sqrt(z.square().mean(-1, keepdim=True) + eps) * weight


def quantise(y: torch.Tensor, group: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(y / scale before its rounding to 8 bits, scale): one scale for each
    ``group`` columns, the largest magnitude / 448."""
    y = y.unflatten(-1, (y.shape[-1] // group, group))
    top = y.abs().amax(-1, keepdim=True)
    scale = torch.where(top < FP8_MAX * 2.0**-126, torch.ones_like(top), top / FP8_MAX)
    return (y / scale).flatten(-2), scale.squeeze(-1)


def embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float) -> torch.Tensor:
    return weight[ids.long()] * scale


def embedding_grad(ids: torch.Tensor, dy: torch.Tensor, V: int, padding: int, scale: float) -> torch.Tensor:
    """dW, the padding token's row and ids outside the table left out."""
    C = dy.shape[-1]
    flat, rows = ids.reshape(-1).long(), dy.reshape(-1, C)
    ok = (flat >= 0) & (flat < V) & (flat != padding)
    return torch.zeros(V, C, dtype=dy.dtype).index_add_(0, flat[ok], rows[ok]) * scale
