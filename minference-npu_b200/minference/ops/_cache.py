"""Shared checks of the cache operators: views, lengths, overlap."""

from __future__ import annotations

import torch
import torch.nn.functional as F

from .. import _native

MAX_HEAD_DIM = 128


def check_same(name: str, x: torch.Tensor, like: torch.Tensor, shape: tuple) -> None:
    """`x` has the given shape and `like`'s dtype and device."""
    if not isinstance(x, torch.Tensor) or tuple(x.shape) != tuple(shape):
        got = tuple(x.shape) if isinstance(x, torch.Tensor) else type(x).__name__
        raise ValueError(f"{name} must be {tuple(shape)}, got {got}")
    if x.dtype != like.dtype:
        raise TypeError(f"{name} is {x.dtype}, expected {like.dtype}")
    if x.device != like.device:
        raise ValueError(f"{name} is on {x.device}, expected {like.device}")


def check_query(q: torch.Tensor, Hkv: int) -> None:
    _native.require_cuda(q)
    _native.dtype_code(q)
    if Hkv < 1 or q.shape[1] % Hkv:
        raise ValueError(f"{q.shape[1]} query heads over {Hkv} key/value heads")
    if not 1 <= q.shape[-1] <= MAX_HEAD_DIM:
        raise NotImplementedError(
            f"head_dim={q.shape[-1]}: the sm_100a kernels take 1 to {MAX_HEAD_DIM}")


def lengths_arg(name: str, x, n: int, cap: int, device: torch.device):
    """int32 device tensor [n] of valid rows, or None (every row)."""
    if x is None:
        return None
    if not isinstance(x, torch.Tensor) or x.dtype.is_floating_point or x.dtype.is_complex \
            or x.dtype == torch.bool:
        raise TypeError(f"{name} must be an integer tensor")
    if tuple(x.shape) != (n,):
        raise ValueError(f"{name} must be ({n},), got {tuple(x.shape)}")
    if x.dtype != torch.int32:
        x = x.clamp(0, cap).to(torch.int32)
    return x.to(device).contiguous()


def _aligned(x: torch.Tensor) -> bool:
    """Rows that 16-byte loads and tensor maps can read (dimensions of one entry
    have no stride)."""
    if x.stride(-1) != 1 or x.data_ptr() % 16:
        return False
    return all(x.shape[i] <= 1 or (x.stride(i) > 0 and x.stride(i) % 8 == 0) for i in range(3))


def rows_view(x: torch.Tensor, D: int) -> torch.Tensor:
    """`x` with its head dim padded to D by zeros and 16-byte rows; `x` itself
    where it has them already."""
    if x.shape[-1] != D:
        return F.pad(x, (0, D - x.shape[-1]))
    return x if _aligned(x) else x.clone(memory_format=torch.contiguous_format)


def span(x: torch.Tensor) -> tuple[int, int]:
    """Addresses [first, end) that a strided view covers."""
    if x.numel() == 0:
        return 0, 0
    last = sum((n - 1) * s for n, s in zip(x.shape, x.stride()))
    return x.data_ptr(), x.data_ptr() + (last + 1) * x.element_size()


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def check_output(name: str, x: torch.Tensor) -> None:
    """Every element of an output view has its own address."""
    need = 1
    for n, s in sorted(zip(x.shape, x.stride()), key=lambda t: t[1]):
        if n > 1:
            if s < need:
                raise ValueError(f"{name} has overlapping rows (strides {x.stride()})")
            need = s * (n - 1) + need
