"""Shared checks of the cache operators: views, lengths, overlap."""

from __future__ import annotations

import torch
import torch.nn.functional as F

from .. import _native

MAX_HEAD_DIM = 128


_DTYPES = {torch.float16: _native.MI_F16, torch.bfloat16: _native.MI_BF16}


def check_same(name: str, x: torch.Tensor, like: torch.Tensor, shape: tuple) -> None:
    """`x` has the given shape and `like`'s dtype and device."""
    if isinstance(x, torch.Tensor) and x.shape == shape and x.dtype is like.dtype \
            and x.get_device() == like.get_device():
        return
    if not isinstance(x, torch.Tensor) or x.shape != shape:
        got = tuple(x.shape) if isinstance(x, torch.Tensor) else type(x).__name__
        raise ValueError(f"{name} must be {tuple(shape)}, got {got}")
    if x.dtype is not like.dtype:
        raise TypeError(f"{name} is {x.dtype}, expected {like.dtype}")
    raise ValueError(f"{name} is on {x.device}, expected {like.device}")


def check_query(q: torch.Tensor, Hkv: int) -> int:
    """dtype code of q."""
    _native.require_cuda(q)
    code = _DTYPES.get(q.dtype)
    if code is None:
        code = _native.dtype_code(q)  # raises
    if Hkv < 1 or q.shape[1] % Hkv:
        raise ValueError(f"{q.shape[1]} query heads over {Hkv} key/value heads")
    if not 1 <= q.shape[3] <= MAX_HEAD_DIM:
        raise NotImplementedError(
            f"head_dim={q.shape[3]}: the sm_100a kernels take 1 to {MAX_HEAD_DIM}")
    return code


def lengths_arg(name: str, x, n: int, cap: int, device: torch.device):
    """int32 device tensor [n] of valid rows."""
    if not isinstance(x, torch.Tensor) or x.dtype.is_floating_point or x.dtype.is_complex \
            or x.dtype == torch.bool:
        raise TypeError(f"{name} must be an integer tensor")
    if x.shape != (n,):
        raise ValueError(f"{name} must be ({n},), got {tuple(x.shape)}")
    if x.dtype is not torch.int32:
        # in 64 bits: a narrow type need not hold the capacity
        x = x.to(torch.int64).clamp(0, cap).to(torch.int32)
    if x.get_device() != device.index:
        x = x.to(device)
    return x if x.is_contiguous() else x.contiguous()


def rows_arg(x: torch.Tensor, pad: int, hold: list) -> tuple[int, int, int, int]:
    """(address, strides) of `x`'s rows for the C structs: the head dim with `pad`
    zeros behind it, rows that 16-byte loads and tensor maps can read.  A view
    without them is copied; `hold` then keeps the copy until the launch."""
    p = x.data_ptr()
    b, h, s, d = x.stride()
    if not pad and d == 1 and not (p | (b | h | s) << 1) & 15 and b > 0 and h > 0 and s > 0:
        return p, b, h, s
    if pad:
        x = F.pad(x, (0, pad))
    elif d != 1 or p & 15 or any(
            n > 1 and (t <= 0 or t % 8) for n, t in zip(x.shape[:3], (b, h, s))):
        x = x.clone(memory_format=torch.contiguous_format)
    hold.append(x)
    return x.data_ptr(), x.stride(0), x.stride(1), x.stride(2)


def span(x: torch.Tensor) -> tuple[int, int]:
    """Addresses [first, end) that a strided view covers."""
    n = x.numel()
    if n == 0:
        return 0, 0
    if x.is_contiguous():
        p = x.data_ptr()
        return p, p + n * x.element_size()
    last = sum((n - 1) * s for n, s in zip(x.shape, x.stride()))
    return x.data_ptr(), x.data_ptr() + (last + 1) * x.element_size()


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Two views may share an element (views that interleave do not)."""
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1 and not _interleaved(a, b)


def _interleaved(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Some stride tells the views apart: modulo it, each covers one stretch of
    addresses (what its dimensions of other strides reach), clear of the other's."""
    dims = [[(n, s * x.element_size()) for n, s in zip(x.shape, x.stride()) if n > 1]
            for x in (a, b)]
    for step in {s for d in dims for _, s in d if s > 0}:
        na, nb = (sum((n - 1) * s for n, s in d if s % step) + x.element_size()
                  for d, x in zip(dims, (a, b)))
        gap = (b.data_ptr() - a.data_ptr()) % step
        if na <= gap and gap + nb <= step:
            return True
    return False


def check_output(name: str, x: torch.Tensor) -> None:
    """Every element of an output view has its own address."""
    if x.is_contiguous():
        return
    need = 1
    for n, s in sorted(zip(x.shape, x.stride()), key=lambda t: t[1]):
        if n > 1:
            if s < need:
                raise ValueError(f"{name} has overlapping rows (strides {x.stride()})")
            need = s * (n - 1) + need
