"""A key/value cache in 4 or 8 bits: its rows, and the kernels that write, read and attend over them (``csrc/quantized_cache.cu``, ``csrc/quantized_attention.cu``)."""
from __future__ import annotations

import math
import struct
from typing import NamedTuple, Optional, Tuple

import torch

from ._lib import check, lib, stream_ptr
from .mask import AttentionMask

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}  # of rows that are written
_pack_append, _pack_read, _pack_attention = (struct.Struct(f"={n}q").pack for n in (32, 25, 30))  # arguments of a call, as its struct in the kernel's source has them
HEAD_DIMS = (64, 96, 128, 256)  # that the attention kernel has


class QuantizedRows(NamedTuple):
    """The keys (or the values) of a cache: one row of codes and scales per batch row, head and slot.

    ``codes`` uint8 ``[batch, heads, slots, d * bits / 8]``, ``scales`` bf16 ``[batch, heads, slots, d / 32]``; ``d`` is a multiple of 32, ``bits`` 4 or 8.  Seen as ``[4, d / 32, 8]``, a row's channels
    with the same middle index are a group; channel ``c`` stands for ``scale[group] * (code[c] - 2^(bits - 1))``.  Of 4 bits two codes share a byte, the even channel in the low half.
    ``count``: how many of the slots are meant (:meth:`first`), ``-1`` for all."""

    codes: torch.Tensor
    scales: torch.Tensor
    count: int = -1

    @property
    def head_dim(self) -> int:
        return self.scales.shape[3] * 32

    @property
    def bits(self) -> int:
        return self.codes.shape[3] * 8 // self.head_dim

    @property
    def slots(self) -> int:
        return self.codes.shape[2] if self.count < 0 else self.count

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
        return cls(codes, scales, slots)

    def first(self, slots: int) -> "QuantizedRows":
        """The first ``slots`` slots."""
        if not 0 <= slots <= self.slots:
            raise ValueError(f"{slots} of {self.slots} slots")
        return QuantizedRows(self.codes, self.scales, slots)

    def batch(self, rows: int) -> "QuantizedRows":
        """The first ``rows`` batch rows (a view)."""
        return QuantizedRows(self.codes[:rows], self.scales[:rows], self.count)


def sizes(k_rows: QuantizedRows, v_rows: QuantizedRows) -> Tuple[int, int, int, int, int]:
    """``(batch, heads, slots, head_dim, bits)`` of the keys and values of a cache; an error if they are not a pair of rows."""
    kc, ks, n = k_rows
    vc, vs, vn = v_rows
    a, g, device = kc.shape, ks.shape, kc.device
    if len(a) == 4 and len(g) == 4 and a == vc.shape and g == vs.shape and n == vn and kc.dtype is vc.dtype is torch.uint8 and ks.dtype is vs.dtype is torch.bfloat16:
        b, h, held, row = a
        groups = g[3]
        if (g[0] == b and g[1] == h and g[2] == held and n <= held and groups > 0 and (row == groups * 16 or row == groups * 32)
                and device == vc.device and device == ks.device and device == vs.device):
            return b, h, held if n < 0 else n, groups * 32, row // (groups * 4)
    for name, (codes, scales, count) in (("k_rows", k_rows), ("v_rows", v_rows)):
        if codes.dim() != 4 or scales.dim() != 4 or codes.shape[:3] != scales.shape[:3] or count > codes.shape[2]:
            raise ValueError(f"{name}: codes {tuple(codes.shape)} and scales {tuple(scales.shape)} are not [batch, heads, slots, ...] of the same rows")
        if codes.dtype != torch.uint8 or scales.dtype != torch.bfloat16:
            raise ValueError(f"{name}: codes are uint8 and scales bfloat16, not {codes.dtype} and {scales.dtype}")
        if scales.shape[3] == 0 or codes.shape[3] not in (scales.shape[3] * 16, scales.shape[3] * 32):
            raise ValueError(f"{name}: rows of {codes.shape[3]} bytes with {scales.shape[3]} scales are neither 4 nor 8 bits (32 channels share a scale)")
    raise ValueError(f"keys {tuple(kc.shape)} on {kc.device} and values {tuple(vc.shape)} on {vc.device} of a cache have the same shape, bits, slots and device")


def plain(*rows: QuantizedRows) -> bool:
    """Whether these are ordinary tensors, whose address a kernel can be given."""
    for codes, scales, _ in rows:
        if type(codes) is not torch.Tensor or type(scales) is not torch.Tensor:
            return False
    return True


def _on(t: torch.Tensor, call, *args) -> int:
    """Calls a kernel with the device of its operands as the current one (kernels launch on the current device's stream)."""
    if t.get_device() == torch._C._cuda_getDevice():
        return call(*args, stream_ptr())
    with torch.cuda.device(t.device):
        return call(*args, stream_ptr())


def _steps(rows: QuantizedRows) -> Tuple[int, ...]:
    """Strides of batch, head and slot, of codes and of scales."""
    codes, scales = rows.codes.stride(), rows.scales.stride()
    if codes[3] != 1 or (scales[3] != 1 and rows.scales.shape[3] > 1):
        raise ValueError("the codes and scales of a row have to lie one behind the other")
    return codes[:3] + scales[:3]


def append(k: torch.Tensor, v: torch.Tensor, k_rows: QuantizedRows, v_rows: QuantizedRows, slots: torch.Tensor, bits: int) -> None:
    b, s, h, d = k.shape
    if k.stride(3) != 1:
        k = k.contiguous()
    if v.stride(3) != 1:
        v = v.contiguous()
    call = _pack_append(k.data_ptr(), v.data_ptr(), k_rows.codes.data_ptr(), k_rows.scales.data_ptr(), v_rows.codes.data_ptr(), v_rows.scales.data_ptr(), *k.stride()[:3], *v.stride()[:3],
                        *_steps(k_rows), *_steps(v_rows), slots.data_ptr(), _TYPES[k.dtype], b, s, h, d, bits, k_rows.slots)
    check(_on(k, lib().ttb_quantized_append, call), "quantised append")


def read(k_rows: QuantizedRows, v_rows: QuantizedRows, start: int, stop: int, dtype: torch.dtype, size: Tuple[int, int, int, int, int]) -> Tuple[torch.Tensor, torch.Tensor]:
    b, h, _, d, bits = size
    n = stop - start
    codes = k_rows.codes
    k = codes.new_empty((b, n, h, d), dtype=dtype)
    v = torch.empty_like(k)
    if b and n and h:
        call = _pack_read(codes.data_ptr(), k_rows.scales.data_ptr(), v_rows.codes.data_ptr(), v_rows.scales.data_ptr(), *_steps(k_rows), *_steps(v_rows), k.data_ptr(), v.data_ptr(), b, start,
                          n, h, d, bits, dtype == torch.float32)
        check(_on(codes, lib().ttb_quantized_read, call), "quantised read")
    return k, v


def layout(s: int, hq: int, k_rows: QuantizedRows, v_rows: QuantizedRows, size: Tuple[int, int, int, int, int]) -> Optional[Tuple[int, ...]]:
    """Addresses, and batch and head strides, of codes and scales for the kernel of few queries, or ``None`` where it does not take these rows; the visibility words of a cluster of 8 CTAs bound the number of slots."""
    _, h, n, d, bits = size
    if d not in HEAD_DIMS or s * (hq // h) > (8 if d == 256 else 16) or (-(-n // 256) * (s + 2) + 1) * 4 > 16384:
        return None
    row, groups = d * bits // 8, d // 32
    kc, ks, _ = k_rows
    vc, vs, _ = v_rows
    c0, c1, c2, c3 = kc.stride()
    g0, g1, g2, g3 = ks.stride()
    d0, d1, d2, d3 = vc.stride()
    h0, h1, h2, h3 = vs.stride()
    if not (c2 == d2 == row and g2 == h2 == groups and c3 == g3 == d3 == h3 == 1) or (c0 | c1 | d0 | d1 | 2 * (g0 | g1 | h0 | h1)) & 15:
        return None
    at = kc.data_ptr(), ks.data_ptr(), vc.data_ptr(), vs.data_ptr()
    if (at[0] | at[1] | at[2] | at[3]) & 15:
        return None
    return (*at, c0, c1, g0, g1, d0, d1, h0, h1)


def attention(q: torch.Tensor, mask: AttentionMask, scale: Optional[float], size: Tuple[int, int, int, int, int], steps: Tuple[int, ...]) -> torch.Tensor:
    b, s, hq, d = q.shape
    _, hkv, n, _, bits = size
    q = q.contiguous()
    if q.data_ptr() & 15:
        q = q.clone()
    o = torch.empty_like(q)
    seen, seen_b, seen_r, start, offset, window, sinks = 0, 0, 0, None, -1, 0, 0
    m = mask.bool_mask
    if m is not None:
        m = m if m.dim() == 3 else m[:, 0]
        if m.dtype is not torch.bool or m.device != q.device:
            m = m.to(device=q.device, dtype=torch.bool)
        if m.shape[0] != b or m.shape[1] != s:
            m = m.expand(b, s, n)
        seen_b, seen_r, unit = m.stride()
        if unit != 1 and n > 1:
            m = m.contiguous()
            seen_b, seen_r, _ = m.stride()
        seen = m.data_ptr()
    elif mask.key_start is not None:
        start = mask.key_start.to(device=q.device, dtype=torch.int32).contiguous()
        offset = mask.query_start
    elif mask.causal:
        offset, window = n - s, min(max(mask.window, 0), n)
        sinks = min(max(mask.sinks, 0), n) if window else 0
    work, floats = None, 0
    if (n if window == 0 else min(n, window + sinks)) >= 6144 and b * hkv * 8 < 592:
        # Few and long rows are split further than a cluster reaches.  The kernel's model never does that to shorter rows.  To more than 73 pairs of a batch row and a key head it would in places (93 pairs of
        # 130 000 slots: 11 splits instead of 4, 14 % by the model, not measured); they are not offered a workspace, which holds 128 results of a row.
        floats = 128 * b * s * hq * (d + 4)
        work = torch.empty(floats, dtype=torch.float32, device=q.device)
    call = _pack_attention(q.data_ptr(), *steps, o.data_ptr(), seen, seen_b, seen_r, 0 if start is None else start.data_ptr(), offset, window, sinks, b, s, n, hq, hkv, d, bits,
                           0 if work is None else work.data_ptr(), floats)
    check(_on(q, lib().ttb_quantized_attention, call, 1.0 / math.sqrt(d) if scale is None else float(scale)), "attention over a quantised cache")
    return o
