"""Log-probabilities of given tokens with the entropy and the likeliest alternatives (``csrc/token_stats.cu``)."""
from __future__ import annotations

import math
import struct
from typing import NamedTuple, Optional, Tuple

import torch

from ._lib import check, launch, lib

MAX_TOP = 64
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_LOG2E = math.log2(math.e)
_pack = struct.Struct("=19q").pack  # the kernel source's Call


class TokenStatistics(NamedTuple):
    """Of logits ``[..., V]``: ``logprobs`` and ``entropy`` fp32 ``[...]``, and with ``top`` alternatives ``top_logprobs`` fp32 and ``top_tokens`` int64 ``[..., top]``, the likeliest first."""

    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: Optional[torch.Tensor]
    top_tokens: Optional[torch.Tensor]


def check_arguments(logits: torch.Tensor, tokens: torch.Tensor, temperature: float, top: int) -> None:
    if logits.dim() == 0 or logits.shape[:-1] != tokens.shape or logits.shape[-1] == 0:
        raise ValueError(f"logits {tuple(logits.shape)} are not one row for each of the tokens {tuple(tokens.shape)}")
    if not logits.dtype.is_floating_point:
        raise ValueError(f"logits are floating-point numbers, not {logits.dtype}")
    if tokens.dtype != torch.int64 or tokens.device != logits.device:
        raise ValueError(f"tokens are int64 on {logits.device}, not {tokens.dtype} on {tokens.device}")
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError(f"a temperature is a positive number, not {temperature}")
    if not 0 <= top <= min(MAX_TOP, logits.shape[-1]):
        raise ValueError(f"0 to {min(MAX_TOP, logits.shape[-1])} alternatives, not {top}")


def _rows(logits: torch.Tensor) -> Tuple[torch.Tensor, int, int, int]:
    """Logits whose rows lie one after the other or are a slice of a batch, and where: steps of the outer and the inner dimension, and the latter's size."""
    v = logits.shape[-1]
    if logits.stride(-1) != 1 and v > 1:
        logits = logits.contiguous()
    if logits.dim() == 3 and not logits.is_contiguous():
        return logits, logits.stride(0), logits.stride(1), logits.shape[1]
    flat = logits.reshape(-1, v)
    return flat, 0, flat.stride(0), flat.shape[0]


def _at(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def forward(logits, tokens, temperature: float, top: int, ignore: int, keep: bool):
    x, *steps = _rows(logits)
    v, rows, shape = logits.shape[-1], tokens.numel(), tokens.shape
    tokens = tokens.contiguous()
    logprobs = logits.new_empty(shape, dtype=torch.float32)
    entropy = torch.empty_like(logprobs)
    top_logprobs = logits.new_empty((*shape, top), dtype=torch.float32) if top else None
    top_tokens = tokens.new_empty((*shape, top)) if top else None
    stats = logprobs.new_empty((rows, 2)) if keep else None
    call = _pack(x.data_ptr(), *steps, rows, v, _TYPES[x.dtype], top, ignore, tokens.data_ptr(), logprobs.data_ptr(), entropy.data_ptr(), _at(stats), _at(top_logprobs), _at(top_tokens), 0, 0, 0, 0)
    check(launch(x, lib().ttb_token_stats, call, _LOG2E / temperature, 1.0 / temperature), "statistics of tokens")
    return TokenStatistics(logprobs, entropy, top_logprobs, top_tokens), tokens, stats


class _TokenStatistics(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, temperature, top, ignore):
        out, tokens, stats = forward(logits, tokens, temperature, top, ignore, True)
        ctx.save_for_backward(logits, tokens, stats, out.entropy, out.top_tokens)
        ctx.how = temperature, top, ignore
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(out.top_tokens)
        return tuple(out)

    @staticmethod
    def backward(ctx, g, h, k, _):
        if torch.is_grad_enabled():
            raise RuntimeError("the gradients of token_statistics are not differentiable themselves")
        logits, tokens, stats, entropy, top_tokens = ctx.saved_tensors
        temperature, top, ignore = ctx.how
        if g is None and h is None and k is None:
            return None, None, None, None, None
        g, h, k = (t if t is None or t.is_contiguous() else t.contiguous() for t in (g, h, k))
        x, *steps = _rows(logits)
        dx = logits.new_empty(logits.shape)
        call = _pack(x.data_ptr(), *steps, tokens.numel(), logits.shape[-1], _TYPES[x.dtype], top, ignore, tokens.data_ptr(), 0, entropy.data_ptr(), stats.data_ptr(), 0, _at(top_tokens),
                     _at(g), _at(h), _at(k), dx.data_ptr())
        check(launch(x, lib().ttb_token_stats_bwd, call, _LOG2E / temperature, 1.0 / temperature), "gradient of statistics of tokens")
        return dx, None, None, None, None


def suits(logits: torch.Tensor, top: int) -> bool:
    """Whether the kernels take these: with alternatives, a CTA has room for the maxima of 1024 segments of 256 elements, and a row has eight CTAs."""
    v = logits.shape[-1]
    return logits.dtype in _TYPES and v <= (2_000_000 if top else 2**31 - 512) and logits.numel() // v < 2**27


def token_statistics(logits, tokens, temperature: float, top: int, ignore: int, differentiated: bool) -> TokenStatistics:
    if differentiated:
        return TokenStatistics(*_TokenStatistics.apply(logits, tokens, temperature, top, ignore))
    return forward(logits, tokens, temperature, top, ignore, False)[0]
