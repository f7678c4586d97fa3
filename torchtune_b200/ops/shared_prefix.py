"""Attention of rows that share a long prefix (``csrc/shared_prefix.cu``)."""
from __future__ import annotations

import math
import struct
from typing import Optional

import torch

from ._lib import check, err_word, launch, lib

HEAD_DIMS = (64, 128)  # that the kernel has
_pack = struct.Struct("=31q").pack  # the kernel source's Call
_WITHOUT = (0,) * 23  # addresses and steps, where only sizes count


def check_arguments(q, k_prefix, v_prefix, k, v, prefix_start, prefix_stop, lengths) -> None:
    a, b, c = q.shape, k_prefix.shape, k.shape
    if len(a) != 4 or len(b) != 4 or len(c) != 4 or b != v_prefix.shape or c != v.shape:
        raise ValueError(f"queries {tuple(a)}, prefix {tuple(b)} and {tuple(v_prefix.shape)}, own {tuple(c)} and {tuple(v.shape)} are not [rows, tokens, heads, channels] with keys like values")
    if a[0] != c[0] or b[2:] != c[2:] or a[3] != c[3] or c[2] == 0 or a[2] % c[2] or a[2] == 0 or (b[0] == 0) != (a[0] == 0) or (b[0] and a[0] % b[0]):
        raise ValueError(f"{a[0]} rows of {a[2]} query heads of {a[3]} channels, {b[0]} prompts and {c[0]} rows with {b[2]} and {c[2]} key heads of {b[3]} and {c[3]}: rows are a multiple of the "
                         "prompts, query heads of the key heads")
    if not (q.dtype == k_prefix.dtype == v_prefix.dtype == k.dtype == v.dtype) or not q.dtype.is_floating_point:
        raise ValueError(f"queries, keys and values have one floating-point type, not {q.dtype}, {k_prefix.dtype}, {v_prefix.dtype}, {k.dtype} and {v.dtype}")
    if not (q.device == k_prefix.device == v_prefix.device == k.device == v.device):
        raise ValueError("queries, keys and values are on one device")
    for name, t, n in (("prefix_start", prefix_start, b[0]), ("prefix_stop", prefix_stop, b[0]), ("lengths", lengths, a[0])):
        if t is not None and (t.dtype != torch.int32 or t.shape != (n,) or t.device != q.device):
            raise ValueError(f"{name} is int32 of [{n}] on {q.device}, not {t.dtype} of {tuple(t.shape)} on {t.device}")


def suits(q: torch.Tensor, k: torch.Tensor, prompts: int) -> bool:
    """Whether the kernels have these sizes: query rows are numbered in 32 bits, and their tokens are found by a multiplication that is exact below 2^32 over the query heads of a key head."""
    rows, s, hq, d = q.shape
    group = hq // k.shape[2]
    return d in HEAD_DIMS and k.shape[2] <= 256 and rows * s * hq < 2**31 and rows // prompts * s * group * group < 2**32


def _steady(t: torch.Tensor) -> torch.Tensor:
    """``t``, if copies of tiles of one head can read it where it is, or a copy."""
    if t.is_contiguous():
        return t if t.data_ptr() & 15 == 0 else t.clone()
    steps = t.stride()
    if steps[3] == 1 and t.data_ptr() & 15 == 0 and all(n == 1 or (step > 0 and step % 8 == 0) for n, step in zip(t.shape[:3], steps)):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _steps(t: torch.Tensor):
    """Steps of batch, slot and head; those of dimensions of size 1 are not used, but have to be in range."""
    b, n, h, d = t.shape
    if t.is_contiguous():
        return n * h * d, h * d, d
    return [step if n > 1 else d for n, step in zip((b, n, h), t.stride())]


def attention(q, k_prefix, v_prefix, k, v, prefix_start, prefix_stop, lengths, scale: Optional[float]) -> torch.Tensor:
    rows, s, hq, d = q.shape
    q = q.contiguous()
    if q.data_ptr() & 15:
        q = q.clone()
    o = torch.empty_like(q)
    k_prefix, v_prefix, k, v = _steady(k_prefix), _steady(v_prefix), _steady(k), _steady(v)
    prefix_start, prefix_stop, lengths = (t if t is None or t.is_contiguous() else t.contiguous() for t in (prefix_start, prefix_stop, lengths))
    library = lib()
    sizes = (k_prefix.shape[0], rows, s, hq, k.shape[2], d, k_prefix.shape[1], k.shape[1])
    floats = launch(q, library.ttb_shared_prefix_floats, _pack(*_WITHOUT, *sizes))
    if floats < 0:
        check(floats, "attention over a shared prefix")
    work = q.new_empty((floats,), dtype=torch.float32)
    call = _pack(q.data_ptr(), o.data_ptr(), k_prefix.data_ptr(), v_prefix.data_ptr(), k.data_ptr(), v.data_ptr(), _at(prefix_start), _at(prefix_stop), _at(lengths), work.data_ptr(), floats,
                 *_steps(k_prefix), *_steps(v_prefix), *_steps(k), *_steps(v), *sizes)
    check(launch(q, library.ttb_shared_prefix_attention, call, 1.0 / math.sqrt(d) if scale is None else float(scale), err_word(q.device).data_ptr()), "attention over a shared prefix")
    return o


def _at(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()
