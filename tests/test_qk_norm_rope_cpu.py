"""Norms of queries and keys per head with the rotation in the same pass: the plain statement against the definition and against differences, what it refuses, and the write to a cache."""
import pytest
import torch

from torchtune_b200 import ops
from torchtune_b200.ops import reference


def _table(n, d):
    angle = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    return torch.stack([angle.cos(), angle.sin()], -1).float()


def _inputs(b, s, hq, hk, d, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    make = lambda *shape: torch.randn(*shape, generator=g, dtype=torch.float64).to(dtype)  # noqa: E731
    return make(b, s, hq, d), make(b, s, hk, d), 1 + 0.2 * make(d), 1 + 0.2 * make(d)


def _by_hand(x, gain, angles, eps, interleaved, norm_first):
    """One head row in scalars."""
    d = len(x)
    pairs = [(2 * i, 2 * i + 1) if interleaved else (i, i + d // 2) for i in range(d // 2)]

    def turn(v):
        y = list(v)
        for i, (a, b) in enumerate(pairs):
            c, s = (float(t) for t in angles[i])
            y[a], y[b] = v[a] * c - v[b] * s, v[b] * c + v[a] * s
        return y

    def norm(v):
        r = (sum(t * t for t in v) / d + eps) ** -0.5
        return [t * r for t in v]

    x = [float(t) for t in x]
    w = [1.0] * d if gain is None else [float(t) for t in gain]
    scaled = lambda v: [a * b for a, b in zip(v, w)]  # noqa: E731
    return turn(scaled(norm(x))) if norm_first else scaled(norm(turn(x)))


@pytest.mark.parametrize("gains", [True, False])
@pytest.mark.parametrize("norm_first", [True, False])
@pytest.mark.parametrize("interleaved", [True, False])
def test_statement_against_scalars(interleaved, norm_first, gains):
    q, k, gq, gk = _inputs(2, 3, 2, 1, 6, torch.float64)
    table = 1.25 * _table(9, 6)  # angles' cosines and sines may be scaled
    pos = torch.tensor([[4, 0, 8], [1, 1, 2]])
    if not gains:
        gq = gk = None
    out = ops.qk_norm_rope(q, k, gq, gk, table, pos, eps=1e-3, interleaved=interleaved, norm_first=norm_first)
    for got, x, gain in zip(out, (q, k), (gq, gk)):
        assert got.dtype == torch.float64
        for at in ((0, 0, 0), (1, 2, x.shape[2] - 1), (0, 1, 0)):
            want = torch.tensor(_by_hand(x[at], gain, table[pos[at[:2]]], 1e-3, interleaved, norm_first), dtype=torch.float64)
            torch.testing.assert_close(got[at], want, rtol=1e-12, atol=1e-12)


def test_gradients_against_differences():
    q, k, gq, gk = _inputs(1, 2, 2, 1, 4, torch.float64, seed=1)
    table = _table(5, 4)
    for interleaved in (True, False):
        for norm_first in (True, False):
            leaves = [t.clone().requires_grad_() for t in (q, k, gq, gk)]
            assert torch.autograd.gradcheck(lambda *t: ops.qk_norm_rope(*t, table, torch.tensor([3, 1]), eps=1e-2, interleaved=interleaved, norm_first=norm_first), leaves)


def test_positions_of_every_form():
    q, k, gq, gk = _inputs(3, 1, 2, 1, 16)
    table = _table(10, 16)
    full = ops.qk_norm_rope(q, k, gq, gk, table, torch.tensor([[2], [5], [9]]))
    row = ops.qk_norm_rope(q, k, gq, gk, table, torch.tensor([2, 5, 9], dtype=torch.int32))
    assert torch.equal(full[0], row[0]) and torch.equal(full[1], row[1])
    q, k, gq, gk = _inputs(2, 4, 2, 1, 16)
    default = ops.qk_norm_rope(q, k, gq, gk, table)
    for pos in (torch.arange(4), torch.arange(4)[None], torch.arange(4).expand(2, 4)):
        assert torch.equal(default[0], ops.qk_norm_rope(q, k, gq, gk, table, pos)[0])


def test_same_as_the_two_operators_of_their_own():
    q, k, gq, gk = _inputs(2, 5, 4, 2, 32)
    table = _table(8, 32)
    for interleaved in (True, False):
        want = ops.rope(ops.rms_norm(q, gq, 1e-6), table, None, interleaved)
        got = ops.qk_norm_rope(q, k, gq, gk, table, interleaved=interleaved)[0]
        # fp32 throughout on both sides: a few roundings of values up to about 5 apart
        torch.testing.assert_close(got, want, rtol=1e-6, atol=4e-6)


def test_refusals():
    q, k, gq, gk = _inputs(2, 3, 4, 2, 16)
    table = _table(8, 16)
    call = lambda **how: ops.qk_norm_rope(**{**dict(q=q, k=k, q_gain=gq, k_gain=gk, cache=table), **how})  # noqa: E731
    call()
    wrong = [dict(k=k[:1]), dict(k=k[:, :2]), dict(k=k[..., :8]), dict(k=k.double()), dict(q=q[0]), dict(q_gain=gq[:8]), dict(k_gain=gk[None]), dict(cache=table[:, :4]),
             dict(cache=table[:2]), dict(cache=table[0]), dict(input_pos=torch.arange(4)), dict(input_pos=torch.arange(3).float()), dict(input_pos=torch.tensor([0, 1, 8])),
             dict(input_pos=torch.tensor([0, -1, 2])), dict(input_pos=torch.zeros(3, 3, dtype=torch.int64)), dict(q=q.int(), k=k.int()), dict(q=q[:, :, :0]), dict(q_gain=gq.int())]
    for how in wrong:
        with pytest.raises(ValueError):
            call(**how)


def _append(**how):
    q, k, gq, gk = _inputs(2, 3, 4, 2, 16)
    caches = [torch.full((2, 9, 2, 16), 7.0) for _ in range(2)]
    args = {**dict(q=q, k=k, v=-k, q_gain=gq, k_gain=gk, cache=_table(20, 16), input_pos=torch.tensor([[4, 5, 6], [11, 12, 13]]), k_cache=caches[0], v_cache=caches[1],
                   slots=torch.tensor([7, 2, 4])), **how}
    return args, ops.qk_norm_rope_append(**args)


def test_append_writes_the_slots_and_nothing_else():
    a, out = _append()
    want = ops.qk_norm_rope(a["q"], a["k"], a["q_gain"], a["k_gain"], a["cache"], a["input_pos"])
    assert torch.equal(out, want[0])
    assert torch.equal(a["k_cache"][:, a["slots"]], want[1]) and torch.equal(a["v_cache"][:, a["slots"]], a["v"])
    others = [0, 1, 3, 5, 6, 8]
    assert (a["k_cache"][:, others] == 7).all() and (a["v_cache"][:, others] == 7).all()


def test_append_refusals():
    caches = lambda *shape, dtype=torch.float32: dict(k_cache=torch.zeros(*shape, dtype=dtype), v_cache=torch.zeros(*shape, dtype=dtype))  # noqa: E731
    g = torch.zeros(2, 3, 2, 16)
    for how in (dict(v=g[:, :2]), dict(v=g.double()), caches(1, 9, 2, 16), caches(3, 9, 2, 16), caches(2, 9, 1, 16), caches(2, 9, 2, 16, dtype=torch.bfloat16), dict(v_cache=torch.zeros(2, 8, 2, 16)),
                dict(slots=torch.tensor([0, 1])), dict(slots=torch.tensor([0, 1, 2], dtype=torch.int32)), dict(slots=torch.arange(6)[::2]), dict(v=g.clone().requires_grad_())):
        with pytest.raises(ValueError):
            _append(**how)
    with pytest.raises(IndexError):
        _append(slots=torch.tensor([0, 1, 9]))


def test_nothing_to_do():
    table = _table(4, 16)
    gain = torch.ones(16)
    for b, s in ((0, 2), (2, 0)):
        q, k = ops.qk_norm_rope(torch.zeros(b, s, 2, 16), torch.zeros(b, s, 1, 16), gain, gain, table)
        assert q.shape == (b, s, 2, 16) and k.shape == (b, s, 1, 16)


def test_zeros_and_non_finite_rows_stay_apart():
    q, k, gq, gk = _inputs(1, 4, 2, 1, 16)
    q[0, 0, 0] = 0.0
    q[0, 1, 0, 3] = float("inf")
    q[0, 2, 0, 3] = float("nan")
    out = reference.norm_rope(q, gq, _table(4, 16), None, 1e-6, True, True)
    assert not out[0, 0, 0].any() and out[0, 1, 0].isnan().any() and out[0, 2, 0].isnan().all()
    assert out[0, :, 1].isfinite().all() and out[0, 3].isfinite().all()


def test_plain_writes_leave_out_slots_that_a_cache_does_not_have():
    """What stands in for the kernel on a device must not reach outside of the cache."""
    cache, values = torch.randn(2, 5, 3, 4), torch.randn(2, 4, 3, 4)
    want = cache.clone()
    want[:, 3], want[:, 0] = values[:, 0], values[:, 3]
    reference.write_known_slots(cache, torch.tensor([3, 5, -1, 0]), values)
    assert torch.equal(cache, want)
    reference.write_known_slots(cache, torch.tensor([2**40, -(2**40), 7, 9]), values)
    assert torch.equal(cache, want)
    empty = cache[:, :0].clone()
    reference.write_known_slots(empty, torch.tensor([0, 1, 2, 3]), values)
    with pytest.raises((IndexError, RuntimeError)):
        reference.write_slots(cache, torch.tensor([3, 5, 1, 0]), values)


@pytest.mark.parametrize("shape", [(2, 0), (0, 3), (0, 0)])
def test_nothing_is_differentiated_too(shape):
    """No rows or no tokens: outputs are part of the graph as others are, and gains have gradients of zeros."""
    q, k = (torch.randn(*shape, h, 16, requires_grad=True) for h in (4, 2))
    gains = [torch.ones(16, requires_grad=True) for _ in range(2)]
    for pos in (None, torch.zeros(shape, dtype=torch.int32)):
        a, b = ops.qk_norm_rope(q, k, *gains, _table(8, 16), pos)
        assert a.shape == q.shape and b.shape == k.shape
        grads = torch.autograd.grad(a.sum() + b.sum(), (q, k, *gains))
        assert [g.shape for g in grads] == [q.shape, k.shape, (16,), (16,)] and not any(g.any() for g in grads)
