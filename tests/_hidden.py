"""Helpers of the hidden-state operators' call tests."""

from __future__ import annotations

import torch


class Wrapper(torch.Tensor):
    """A tensor whose values lie in another one (as a sharded parameter's do)."""

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device)

    def __init__(self, inner):
        self.inner = inner

    seen: list = []

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        cls.seen.append(func)
        args = [a.inner if isinstance(a, Wrapper) else a for a in args]
        return func(*args, **(kwargs or {}))
