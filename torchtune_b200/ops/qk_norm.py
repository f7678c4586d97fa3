"""Norms of queries and keys per head with the rotation of their positions (``csrc/qk_norm_rope.cu``): one pass forward, one backward, and one that also fills a key/value cache."""
from __future__ import annotations

import struct
from typing import Optional, Tuple

import torch

from ._lib import check, launch, lib

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_pack = struct.Struct("=53q").pack  # the kernel source's Call
_NONE = (0, 0, 0)


def positions(input_pos: Optional[torch.Tensor], b: int, s: int, table_len: int) -> Optional[torch.Tensor]:
    """``input_pos`` of ``[b, s]``, ``[1, s]``, ``[s]``, or ``[b]`` for one token per row, as ``[b, s]`` (a view); ``None`` stays, if the table has as many positions as there are tokens."""
    if input_pos is None:
        if s > table_len:
            raise ValueError(f"{s} tokens, but angles for {table_len} positions")
        return None
    shape = input_pos.shape
    if input_pos.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"positions are int32 or int64, not {input_pos.dtype}")
    if shape == (b, s):
        return input_pos
    if s == 1 and shape == (b,):
        return input_pos.view(b, 1)
    if shape == (s,) or shape == (1, s):
        return input_pos.view(1, s).expand(b, s)
    raise ValueError(f"positions {tuple(shape)} do not fit {b} rows of {s} tokens")


def check_arguments(q: torch.Tensor, k: torch.Tensor, gains: Tuple[Optional[torch.Tensor], Optional[torch.Tensor]], cache: torch.Tensor) -> None:
    a, c, t, device = q.shape, k.shape, cache.shape, q.device
    if len(a) != 4 or len(c) != 4 or a[:2] != c[:2] or a[3] != c[3] or a[3] % 2 or a[2] == 0 or c[2] == 0 or a[3] == 0:
        raise ValueError(f"queries {tuple(a)} and keys {tuple(c)} are not [rows, tokens, heads, channels] of the same rows, tokens and (even) channels")
    if q.dtype is not k.dtype or not q.dtype.is_floating_point:
        raise ValueError(f"queries and keys have one floating-point type, not {q.dtype} and {k.dtype}")
    if k.device != device or cache.device != device:
        raise ValueError(f"queries on {q.device}, keys on {k.device} and angles on {cache.device} are not on one device")
    if len(t) != 3 or t[0] == 0 or t[1] * 2 != a[3] or t[2] != 2 or not cache.dtype.is_floating_point:
        raise ValueError(f"angles {tuple(t)} are not [positions, {a[3] // 2}, 2] (cosine and sine)")
    for gain in gains:
        if gain is not None and (gain.shape != (a[3],) or gain.device != device or not gain.dtype.is_floating_point):
            raise ValueError(f"a gain {tuple(gain.shape)} of {gain.dtype} on {gain.device} is not [{a[3]}] on {q.device}")


def suits(q: torch.Tensor, k: torch.Tensor, cache: torch.Tensor) -> bool:
    """Whether the kernels have this type and size."""
    b, s, h, d = q.shape
    return q.dtype in _TYPES and d % 16 == 0 and d <= 512 and cache.dtype is torch.float32 and b * s * (h + 2 * k.shape[2]) < 2**31


def _steady(t: torch.Tensor) -> torch.Tensor:
    """``t``, if its rows of one head can be read in 16-byte pieces, or a copy."""
    b, s, h, d = t.stride()
    if d != 1 or (b | s | h) & 7 or t.data_ptr() & 15:
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _aligned(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    if t is None or (t.is_contiguous() and t.data_ptr() & 15 == 0):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _at(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _launch_pos(pos: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    if pos is None:
        return None
    if pos.dtype is not torch.int32:
        pos = pos.clamp(-1, 2**31 - 1).to(torch.int32)  # what does not fit stays out of range
    return pos.contiguous()


def _gains(q: torch.Tensor, gain_q: Optional[torch.Tensor], gain_k: Optional[torch.Tensor]):
    """Both in the type of the queries, or both in 32 bits."""
    if (gain_q is None or gain_q.dtype is q.dtype) and (gain_k is None or gain_k.dtype is q.dtype):
        return gain_q, gain_k
    return tuple(g if g is None else g.float() for g in (gain_q, gain_k))


def _is_wide(gain_q: Optional[torch.Tensor], gain_k: Optional[torch.Tensor]) -> bool:
    gain = gain_q if gain_q is not None else gain_k
    return gain is not None and gain.dtype is torch.float32


def _forward(q, k, v, gain_q, gain_k, cache, pos, eps, interleaved, norm_first, out_k, out_v, slots):
    b, s, hq, d = q.shape
    hk, held = k.shape[2], cache.shape[0]
    q, k, cache, gain_q, gain_k = _steady(q), _steady(k), _aligned(cache), _aligned(gain_q), _aligned(gain_k)
    out_q = q.new_empty((b, s, hq, d))
    if v is None:
        out_k = k.new_empty((b, s, hk, d))
        xv, yv, steps_v, to_k, to_v, heads_v, slot_count = 0, 0, _NONE, (s * hk * d, hk * d, d), _NONE, 0, 0
    else:
        v = _steady(v)
        xv, yv, steps_v, to_k, to_v, heads_v, slot_count = v.data_ptr(), out_v.data_ptr(), v.stride()[:3], out_k.stride()[:3], out_v.stride()[:3], hk, out_k.shape[1]
    call = _pack(q.data_ptr(), k.data_ptr(), xv, out_q.data_ptr(), out_k.data_ptr(), yv, 0, 0, _at(gain_q), _at(gain_k), *q.stride()[:3], *k.stride()[:3], *steps_v,
                 s * hq * d, hq * d, d, *to_k, *to_v, 0, 0, 0, 0, 0, 0, cache.data_ptr(), _at(pos), _at(slots), 0, 0, 0, 0, b, s, hq, hk, heads_v, d,
                 held, slot_count, _TYPES[q.dtype], _is_wide(gain_q, gain_k), interleaved, not norm_first)
    check(launch(q, lib().ttb_qk_norm_rope, call, eps), "norm and rotation of queries and keys")
    return out_q, out_k


class _QKNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, gain_q, gain_k, cache, pos, eps, interleaved, norm_first):
        out = _forward(q, k, None, gain_q, gain_k, cache, pos, eps, interleaved, norm_first, None, None, None)
        ctx.save_for_backward(q, k, gain_q, gain_k, cache, pos)
        ctx.how = eps, interleaved, norm_first
        return out

    @staticmethod
    def backward(ctx, dy_q, dy_k):
        if torch.is_grad_enabled():
            raise RuntimeError("the gradients of qk_norm_rope are not differentiable themselves")
        q, k, gain_q, gain_k, cache, pos = ctx.saved_tensors
        eps, interleaved, norm_first = ctx.how
        need_q, need_k, need_gq, need_gk = ctx.needs_input_grad[:4]
        b, s, hq, d = q.shape
        hk, held = k.shape[2], cache.shape[0]
        q, k, dy_q, dy_k, cache, gain_q, gain_k = _steady(q), _steady(k), _steady(dy_q), _steady(dy_k), _aligned(cache), _aligned(gain_q), _aligned(gain_k)
        dq, dk = q.new_empty((b, s, hq, d)), k.new_empty((b, s, hk, d))
        d_gq = torch.empty_like(gain_q) if need_gq and gain_q is not None else None
        d_gk = torch.empty_like(gain_k) if need_gk and gain_k is not None else None
        work, rows = None, 0
        if d_gq is not None or d_gk is not None:
            rows = lib().ttb_qk_norm_rope_rows()
            work = q.new_empty((rows, d), dtype=torch.float32)
        call = _pack(q.data_ptr(), k.data_ptr(), 0, dq.data_ptr(), dk.data_ptr(), 0, dy_q.data_ptr(), dy_k.data_ptr(), _at(gain_q), _at(gain_k), *q.stride()[:3], *k.stride()[:3], 0, 0, 0,
                     s * hq * d, hq * d, d, s * hk * d, hk * d, d, 0, 0, 0, *dy_q.stride()[:3], *dy_k.stride()[:3], cache.data_ptr(), _at(pos), 0, _at(work), rows,
                     _at(d_gq), _at(d_gk), b, s, hq, hk, 0, d, held, 0, _TYPES[q.dtype], _is_wide(gain_q, gain_k), interleaved, not norm_first)
        check(launch(q, lib().ttb_qk_norm_rope_bwd, call, eps), "gradients of the norm and rotation of queries and keys")
        return dq if need_q else None, dk if need_k else None, d_gq, d_gk, None, None, None, None, None


def norm_rope(q, k, gain_q, gain_k, cache, pos, eps: float, interleaved: bool, norm_first: bool, differentiated: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    gain_q, gain_k = _gains(q, gain_q, gain_k)
    pos = _launch_pos(pos)
    if differentiated:
        return _QKNormRope.apply(q, k, gain_q, gain_k, cache, pos, eps, interleaved, norm_first)
    return _forward(q, k, None, gain_q, gain_k, cache, pos, eps, interleaved, norm_first, None, None, None)


def append_suits(*caches: torch.Tensor) -> bool:
    """Whether the kernel can write to these caches."""
    for t in caches:
        b, s, h, d = t.stride()
        if d != 1 or (b | s | h) & 7 or t.data_ptr() & 15:
            return False
    return True


def norm_rope_append(q, k, v, gain_q, gain_k, cache, pos, k_cache, v_cache, slots, eps: float, interleaved: bool, norm_first: bool) -> torch.Tensor:
    gain_q, gain_k = _gains(q, gain_q, gain_k)
    return _forward(q, k, v, gain_q, gain_k, cache, _launch_pos(pos), eps, interleaved, norm_first, k_cache, v_cache, slots)[0]
