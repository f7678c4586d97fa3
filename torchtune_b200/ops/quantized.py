"""A key/value cache in 4 or 8 bits: its rows, and the kernels that write, read and attend over them (``csrc/quantized_cache.cu``, ``csrc/quantized_attention.cu``)."""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple, Optional, Tuple

import torch

from ._lib import check, lib, stream_ptr
from .mask import AttentionMask

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}  # of rows that are written
HEAD_DIMS = (64, 96, 128, 256)  # that the attention kernel has


class QuantizedRows(NamedTuple):
    """The keys (or the values) of a cache: one row of codes and scales per batch row, head and slot.

    ``codes`` uint8 ``[batch, heads, slots, d * bits / 8]``, ``scales`` bf16 ``[batch, heads, slots, d / 32]``; ``d`` is a multiple of 32, ``bits`` 4 or 8.  Seen as ``[4, d / 32, 8]``, a row's channels
    with the same middle index are a group; channel ``c`` stands for ``scale[group] * (code[c] - 2^(bits - 1))``.  Of 4 bits two codes share a byte, the even channel in the low half."""

    codes: torch.Tensor
    scales: torch.Tensor

    @property
    def head_dim(self) -> int:
        return self.scales.shape[-1] * 32

    @property
    def bits(self) -> int:
        return self.codes.shape[-1] * 8 // self.head_dim

    @property
    def slots(self) -> int:
        return self.codes.shape[2]

    @classmethod
    def zeros(cls, batch: int, slots: int, heads: int, head_dim: int, bits: int, device=None) -> "QuantizedRows":
        """Rows that read as zeros.  Every head's rows start on 16 bytes, whatever the number of slots."""
        if bits not in (4, 8):
            raise ValueError(f"a quantised cache has 4 or 8 bits, not {bits}")
        if head_dim <= 0 or head_dim % 32:
            raise ValueError(f"a quantised cache needs a head dimension that is a multiple of 32, not {head_dim}")
        held = -(-slots // 8) * 8
        codes = torch.zeros(batch, heads, held, head_dim * bits // 8, dtype=torch.uint8, device=device)
        scales = torch.zeros(batch, heads, held, head_dim // 32, dtype=torch.bfloat16, device=device)
        return cls(codes[:, :, :slots], scales[:, :, :slots])

    def first(self, slots: int) -> "QuantizedRows":
        """The first ``slots`` slots (a view)."""
        return QuantizedRows(self.codes[:, :, :slots], self.scales[:, :, :slots])

    def batch(self, rows: int) -> "QuantizedRows":
        """The first ``rows`` batch rows (a view)."""
        return QuantizedRows(self.codes[:rows], self.scales[:rows])


def validate(rows: QuantizedRows, name: str) -> None:
    codes, scales = rows
    if codes.dim() != 4 or scales.dim() != 4 or codes.shape[:3] != scales.shape[:3]:
        raise ValueError(f"{name}: codes {tuple(codes.shape)} and scales {tuple(scales.shape)} are not [batch, heads, slots, ...] of the same rows")
    if codes.dtype != torch.uint8 or scales.dtype != torch.bfloat16:
        raise ValueError(f"{name}: codes are uint8 and scales bfloat16, not {codes.dtype} and {scales.dtype}")
    if scales.shape[3] == 0 or codes.shape[3] not in (scales.shape[3] * 16, scales.shape[3] * 32):
        raise ValueError(f"{name}: rows of {codes.shape[3]} bytes with {scales.shape[3]} scales are neither 4 nor 8 bits (32 channels share a scale)")
    if codes.device != scales.device:
        raise ValueError(f"{name}: codes and scales are on different devices")


def validate_pair(k_rows: QuantizedRows, v_rows: QuantizedRows) -> None:
    validate(k_rows, "k_rows")
    validate(v_rows, "v_rows")
    if k_rows.codes.shape != v_rows.codes.shape or k_rows.scales.shape != v_rows.scales.shape or k_rows.codes.device != v_rows.codes.device:
        raise ValueError(f"keys {tuple(k_rows.codes.shape)} and values {tuple(v_rows.codes.shape)} of a cache have the same shape, bits and device")


def _here(t: torch.Tensor) -> "_OnDevice":
    return _OnDevice(t.device.index)


class _OnDevice:
    """Makes the device of the operands the current one, if it is not (kernels launch on the current device's stream)."""

    def __init__(self, index: int) -> None:
        self.index, self.was = index, -1

    def __enter__(self) -> None:
        if self.index != torch.cuda.current_device():
            self.was = torch.cuda.current_device()
            torch.cuda.set_device(self.index)

    def __exit__(self, *exc) -> None:
        if self.was >= 0:
            torch.cuda.set_device(self.was)


def _inner(rows: QuantizedRows) -> bool:
    """Whether each row's codes and scales lie one behind the other."""
    return rows.codes.stride(3) == 1 and (rows.scales.stride(3) == 1 or rows.scales.shape[3] == 1)


def append(k: torch.Tensor, v: torch.Tensor, k_rows: QuantizedRows, v_rows: QuantizedRows, slots: torch.Tensor) -> None:
    b, s, h, d = k.shape
    if k.stride(3) != 1:
        k = k.contiguous()
    if v.stride(3) != 1:
        v = v.contiguous()
    if not (_inner(k_rows) and _inner(v_rows)):
        raise ValueError("the codes and scales of a row have to lie one behind the other")
    strides = (ctypes.c_longlong * 18)(*k.stride()[:3], *v.stride()[:3], *k_rows.codes.stride()[:3], *k_rows.scales.stride()[:3], *v_rows.codes.stride()[:3], *v_rows.scales.stride()[:3])
    with _here(k):
        check(lib().ttb_quantized_append(k.data_ptr(), v.data_ptr(), k_rows.codes.data_ptr(), k_rows.scales.data_ptr(), v_rows.codes.data_ptr(), v_rows.scales.data_ptr(), strides,
                                         slots.data_ptr(), _TYPES[k.dtype], b, s, h, d, k_rows.bits, k_rows.slots, stream_ptr()), "quantised append")


def read(k_rows: QuantizedRows, v_rows: QuantizedRows, start: int, stop: int, dtype: torch.dtype) -> Tuple[torch.Tensor, torch.Tensor]:
    b, h = k_rows.codes.shape[:2]
    n, d = stop - start, k_rows.head_dim
    k = torch.empty(b, n, h, d, dtype=dtype, device=k_rows.codes.device)
    v = torch.empty_like(k)
    if k.numel() == 0:
        return k, v
    if not (_inner(k_rows) and _inner(v_rows)):
        raise ValueError("the codes and scales of a row have to lie one behind the other")
    strides = (ctypes.c_longlong * 12)(*k_rows.codes.stride()[:3], *k_rows.scales.stride()[:3], *v_rows.codes.stride()[:3], *v_rows.scales.stride()[:3])
    with _here(k):
        check(lib().ttb_quantized_read(k_rows.codes.data_ptr(), k_rows.scales.data_ptr(), v_rows.codes.data_ptr(), v_rows.scales.data_ptr(), strides, k.data_ptr(), v.data_ptr(), b, start, n, h, d,
                                       k_rows.bits, int(dtype == torch.float32), stream_ptr()), "quantised read")
    return k, v


def attends(s: int, hq: int, k_rows: QuantizedRows, v_rows: QuantizedRows) -> bool:
    """Whether the kernel for few queries takes these rows; the visibility words of a cluster of 16 CTAs bound the number of slots."""
    d, group = k_rows.head_dim, hq // k_rows.codes.shape[1]
    if d not in HEAD_DIMS or s * group > (8 if d == 256 else 16) or -(-k_rows.slots // 512) * (s + 1) * 4 > 16384:
        return False
    for rows in (k_rows, v_rows):
        codes, scales = rows
        if not _inner(rows) or codes.stride(2) != codes.shape[3] or scales.stride(2) != scales.shape[3]:
            return False
        if (codes.data_ptr() | scales.data_ptr() | codes.stride(0) | codes.stride(1) | 2 * scales.stride(0) | 2 * scales.stride(1)) & 15:
            return False
    return True


def attention(q: torch.Tensor, k_rows: QuantizedRows, v_rows: QuantizedRows, mask: AttentionMask, scale: Optional[float]) -> torch.Tensor:
    b, s, hq, d = q.shape
    hkv, n = k_rows.codes.shape[1], k_rows.slots
    q = q.contiguous()
    if q.data_ptr() % 16:
        q = q.clone()
    o = torch.empty_like(q)
    seen, start, offset, window, sinks = None, None, -1, 0, 0
    if mask.bool_mask is not None:
        seen = mask.bool_mask if mask.bool_mask.dim() == 3 else mask.bool_mask[:, 0]
        if seen.dtype != torch.bool or not seen.device == q.device:
            seen = seen.to(device=q.device, dtype=torch.bool)
        seen = seen.expand(b, s, n)
        if seen.stride(2) != 1 and n > 1:
            seen = seen.contiguous()
    elif mask.key_start is not None:
        start = mask.key_start.to(device=q.device, dtype=torch.int32).contiguous()
        offset = mask.query_start
    elif mask.causal:
        offset, window, sinks = n - s, mask.window, mask.sinks if mask.window else 0
    strides = (ctypes.c_longlong * 8)(*k_rows.codes.stride()[:2], *k_rows.scales.stride()[:2], *v_rows.codes.stride()[:2], *v_rows.scales.stride()[:2])
    with _here(q):
        check(lib().ttb_quantized_attention(q.data_ptr(), k_rows.codes.data_ptr(), k_rows.scales.data_ptr(), v_rows.codes.data_ptr(), v_rows.scales.data_ptr(), strides, o.data_ptr(),
                                            None if seen is None else seen.data_ptr(), 0 if seen is None else seen.stride(0), 0 if seen is None else seen.stride(1),
                                            None if start is None else start.data_ptr(), offset, window, sinks, b, s, n, hq, hkv, d, k_rows.bits,
                                            1.0 / math.sqrt(d) if scale is None else float(scale), stream_ptr()), "attention over a quantised cache")
    return o
