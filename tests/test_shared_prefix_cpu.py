"""Attention of rows that share a prefix: the plain statement against attention over each row's own keys, and what it refuses."""
import math

import pytest
import torch

from torchtune_b200 import ops
from torchtune_b200.ops import _lib


def _inputs(prompts, rows, s, n, m, hq, hkv, d, dtype=torch.float64, seed=0):
    g = torch.Generator().manual_seed(seed)
    make = lambda *shape: torch.randn(*shape, generator=g, dtype=torch.float64).to(dtype)  # noqa: E731
    return make(rows, s, hq, d), make(prompts, n, hkv, d), make(prompts, n, hkv, d), make(rows, m, hkv, d), make(rows, m, hkv, d)


def _int(*values):
    return torch.tensor(values, dtype=torch.int32)


def _by_hand(q, kp, vp, k, v, row, i, h, start, stop, length, scale):
    group, prompt = q.shape[2] // k.shape[2], row * kp.shape[0] // q.shape[0]
    head, at = h // group, length - q.shape[1] + i
    pairs = [(kp[prompt, j, head], vp[prompt, j, head]) for j in range(start, stop)] + [(k[row, j, head], v[row, j, head]) for j in range(0, at + 1)]
    if not pairs:
        return torch.zeros(q.shape[3], dtype=q.dtype)
    w = [math.exp(scale * float(q[row, i, h] @ a)) for a, _ in pairs]
    return sum(x * b for x, (_, b) in zip(w, pairs)) / sum(w)


@pytest.mark.parametrize("prompts,rows,s,n,m,hq,hkv,d", [(1, 1, 1, 1, 1, 1, 1, 2), (2, 6, 2, 5, 4, 4, 2, 4), (1, 3, 3, 4, 7, 3, 1, 4), (3, 3, 1, 6, 2, 2, 2, 8)])
def test_statement_against_the_definition(prompts, rows, s, n, m, hq, hkv, d):
    t = _inputs(prompts, rows, s, n, m, hq, hkv, d)
    start, stop = torch.arange(prompts).int() % n, torch.full((prompts,), n - (n > 1)).int()
    lengths = (torch.arange(rows).int() + s).clamp(max=m)
    out = ops.shared_prefix_attention(*t, prefix_start=start, prefix_stop=stop, lengths=lengths, scale=0.3)
    for row in range(rows):
        p = row * prompts // rows
        for i in range(s):
            for h in range(hq):
                want = _by_hand(*t, row, i, h, int(start[p]), max(int(stop[p]), int(start[p])), int(lengths[row]), 0.3)
                torch.testing.assert_close(out[row, i, h], want, rtol=1e-10, atol=1e-12)


def test_same_as_attention_over_joined_keys():
    q, kp, vp, k, v = _inputs(2, 6, 3, 9, 5, 4, 2, 16, torch.float32)
    out = ops.shared_prefix_attention(q, kp, vp, k, v)
    keys, values = (torch.cat([a.repeat_interleave(3, 0), b], 1) for a, b in ((kp, k), (vp, v)))
    want = ops.attention(q, keys, values, ops.AttentionMask(causal=True))
    torch.testing.assert_close(out, want, rtol=1e-5, atol=1e-5)


def test_nothing_to_see():
    q, kp, vp, k, v = _inputs(2, 4, 2, 5, 3, 2, 1, 4)
    out = ops.shared_prefix_attention(q, kp, vp, k, v, prefix_start=_int(5, 0), lengths=_int(0, 1, 2, 0))
    assert not out[0].any()  # no prefix, no token of its own
    assert not out[1, 0].any() and torch.equal(out[1, 1, 0], v[1, 0, 0])  # the second query sees the one token
    assert out[2:].abs().sum(-1).min() > 0
    empty = ops.shared_prefix_attention(q, kp[:, :0], vp[:, :0], k[:, :0], v[:, :0])
    assert empty.shape == q.shape and not empty.any()


def test_numbers_out_of_range_are_cut_off():
    t = _inputs(1, 2, 1, 4, 3, 2, 2, 4)
    assert torch.equal(ops.shared_prefix_attention(*t, prefix_start=_int(-3), prefix_stop=_int(9), lengths=_int(7, 3)), ops.shared_prefix_attention(*t))
    none = ops.shared_prefix_attention(*t, prefix_start=_int(9), lengths=_int(-2, 1))
    assert not none[0].any() and none[1].any()


def test_hidden_slots_have_no_influence():
    q, kp, vp, k, v = _inputs(2, 4, 2, 6, 5, 2, 1, 4)
    how = dict(prefix_start=_int(1, 0), prefix_stop=_int(6, 4), lengths=_int(2, 3, 4, 5))
    want = ops.shared_prefix_attention(q, kp, vp, k, v, **how)
    for t in (kp, vp):
        t[0, :1], t[1, 4:] = float("nan"), float("inf")
    for t in (k, v):
        t[0, 2:], t[1, 3:], t[2, 4:] = float("inf"), float("nan"), -float("inf")
    assert torch.equal(ops.shared_prefix_attention(q, kp, vp, k, v, **how), want)


def test_gradients_against_differences():
    t = [x.requires_grad_() for x in _inputs(1, 2, 2, 3, 3, 2, 1, 2)]
    assert torch.autograd.gradcheck(lambda *a: ops.shared_prefix_attention(*a, prefix_start=_int(1), lengths=_int(2, 3)), t)


def test_refusals():
    q, kp, vp, k, v = _inputs(2, 4, 1, 5, 3, 4, 2, 4)
    call = lambda **how: ops.shared_prefix_attention(**{**dict(q=q, k_prefix=kp, v_prefix=vp, k=k, v=v), **how})  # noqa: E731
    call()
    for how in (dict(q=q[:3]), dict(q=q[0]), dict(q=q[:, :, :3]), dict(q=q[..., :2]), dict(k=k[:, :2]), dict(v_prefix=vp[:1]), dict(k_prefix=kp[:, :, :1], v_prefix=vp[:, :, :1]), dict(q=q.float()),
                dict(v=v.float()), dict(k_prefix=kp[:0], v_prefix=vp[:0]), dict(k_prefix=kp.expand(2, 5, 2, 4)[:, :, :, :2], v_prefix=vp[..., :2]), dict(prefix_start=_int(0)),
                dict(prefix_stop=torch.tensor([1, 2])), dict(lengths=_int(1, 1)), dict(lengths=torch.ones(4)), dict(k_prefix=torch.cat([kp, kp[:1]]), v_prefix=torch.cat([vp, vp[:1]]))):
        with pytest.raises(ValueError):
            call(**how)
    assert ops.shared_prefix_attention(q[:0], kp[:0], vp[:0], k[:0], v[:0]).shape == (0, 1, 4, 4)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_statement_does_not_repeat_the_prefix(dtype):
    """Nothing of the size of every row's own copy of its prompt's keys is made, forward or backward."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Largest(TorchDispatchMode):
        size = 0

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            out = func(*args, **(kwargs or {}))
            for t in out if isinstance(out, (tuple, list)) else (out,):
                if isinstance(t, torch.Tensor):
                    self.size = max(self.size, t.numel() if t._base is None else 0)
            return out

    prompts, rows, n, d = 2, 48, 160, 64
    t = [x.requires_grad_() for x in _inputs(prompts, rows, 1, n, 3, 4, 2, d, dtype)]
    with Largest() as seen:
        ops.shared_prefix_attention(*t, prefix_start=_int(3, 0)).square().sum().backward()
    assert seen.size <= 2 * rows * 4 * (n + 3) < rows * n * 2 * d / 4


@pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="the kernel library is not built")
def test_kernels_refuse_more_tiles_than_they_count():
    """Tiles of 64 keys of all heads are numbered in 32 bits."""
    from torchtune_b200.ops import shared_prefix

    def floats(prompts, rows, hkv, prefix, own):
        return _lib.lib().ttb_shared_prefix_floats(shared_prefix._pack(*shared_prefix._WITHOUT, prompts, rows, 1, hkv, hkv, 64, prefix, own), None)

    assert floats(1, 4, 8, 100, 100) > 0 and floats(1, 1, 256, 2**23 * 64 - 64, 64) > 0
    for sizes in ((1, 1, 256, 2**23 * 64, 64), (2**20, 2**20, 256, 32000, 64), (1, 2**21, 128, 64, 6400), (1, 1, 256, 64, 2**29)):
        assert floats(*sizes) == -3


@pytest.mark.parametrize("prompts,rows,s", [(2, 4, 0), (0, 0, 1), (0, 0, 0)])
def test_nothing_is_differentiated_too(prompts, rows, s):
    """No rows or no tokens: the output is part of the graph as others are."""
    t = [x.requires_grad_() for x in _inputs(prompts, rows, s, 5, 3, 4, 2, 8, torch.float32)]
    out = ops.shared_prefix_attention(*t, prefix_start=torch.zeros(prompts, dtype=torch.int32), lengths=torch.zeros(rows, dtype=torch.int32))
    assert out.shape == t[0].shape
    grads = torch.autograd.grad(out.sum(), t)
    assert not any(g.any() for g in grads)
