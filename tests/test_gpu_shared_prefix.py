"""Attention of rows that share a prefix, on the kernels, against the statement in 64 bits."""
import pytest
import torch

from torchtune_b200 import ops
from torchtune_b200.ops import _lib, reference

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _inputs(prompts, rows, s, n, m, hq, hkv, d, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    make = lambda *shape: torch.randn(*shape, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
    return make(rows, s, hq, d), make(prompts, n, hkv, d), make(prompts, n, hkv, d), make(rows, m, hkv, d), make(rows, m, hkv, d)


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _check(out, q, kp, vp, k, v, start=None, stop=None, lengths=None, scale=None):
    wide = [t.double() for t in (q, kp, vp, k, v)]
    want = reference.shared_prefix_attention(*wide, start, stop, lengths, scale)
    # probabilities are rounded to bf16 for the second product, scores are sums of d products in 32 bits (128 of them are below 2^-13 off at these sizes), the result is rounded once
    size = reference.shared_prefix_attention(*wide[:2], wide[2].abs(), wide[3], wide[4].abs(), start, stop, lengths, scale)
    far = (out.double() - want).abs() - (2.0**-8 * want.abs() + (2.0**-8 + 2.0**-12) * size)
    assert out.dtype == torch.bfloat16 and out.shape == q.shape
    assert (far <= 0).all(), float(far.max())
    _lib.check_device_errors()
    return out


@pytest.mark.parametrize("prompts,rows,s,n,m,hq,hkv,d", [
    (1, 1, 1, 1, 1, 1, 1, 64), (1, 4, 1, 61, 17, 4, 1, 64), (1, 1, 1, 64, 64, 8, 8, 128), (2, 6, 2, 65, 63, 8, 2, 128), (1, 16, 1, 700, 130, 32, 8, 128), (3, 48, 1, 333, 129, 10, 2, 64),
    (1, 64, 1, 200, 40, 16, 4, 128), (2, 70, 3, 150, 90, 15, 3, 128), (1, 3, 40, 90, 200, 8, 2, 64), (1, 2, 9, 300, 77, 16, 1, 128), (4, 4, 1, 128, 192, 3, 3, 128), (1, 8, 1, 20011, 33, 8, 2, 128),
    (1, 256, 1, 77, 5, 4, 4, 64)])
def test_against_64_bits(prompts, rows, s, n, m, hq, hkv, d):
    t = _inputs(prompts, rows, s, n, m, hq, hkv, d)
    _check(ops.shared_prefix_attention(*t), *t)
    g = torch.Generator().manual_seed(rows)
    start, stop = (torch.randint(0, n + 1, (prompts,), generator=g) for _ in range(2))
    start, stop = torch.minimum(start, stop).int().to(DEV), torch.maximum(start, stop).int().to(DEV)
    lengths = torch.randint(0, m + 1, (rows,), generator=g).int().to(DEV)
    _check(ops.shared_prefix_attention(*t, prefix_start=start, prefix_stop=stop, lengths=lengths, scale=0.2), *t, start, stop, lengths, 0.2)


def test_without_a_prefix_or_without_tokens_of_their_own():
    q, kp, vp, k, v = _inputs(2, 8, 2, 100, 70, 8, 2, 64)
    _check(ops.shared_prefix_attention(q, kp[:, :0], vp[:, :0], k, v), q, kp[:, :0], vp[:, :0], k, v)
    _check(ops.shared_prefix_attention(q, kp, vp, k[:, :0], v[:, :0]), q, kp, vp, k[:, :0], v[:, :0])
    assert not ops.shared_prefix_attention(q, kp[:, :0], vp[:, :0], k[:, :0], v[:, :0]).any()
    assert ops.shared_prefix_attention(q[:0], kp[:0], vp[:0], k[:0], v[:0]).shape == (0, 2, 8, 64)
    start, lengths = _int([100, 3]), _int([0, 1, 2, 3, 0, 1, 70, 69])
    out = _check(ops.shared_prefix_attention(q, kp, vp, k, v, prefix_start=start, lengths=lengths), q, kp, vp, k, v, start, None, lengths)
    assert not out[0].any() and not out[1, 0].any() and out[1, 1].any() and out[4].any()


def test_hidden_slots_have_no_influence():
    q, kp, vp, k, v = _inputs(2, 8, 1, 300, 200, 8, 2, 128)
    how = dict(prefix_start=_int([70, 0]), prefix_stop=_int([300, 201]), lengths=_int([1, 63, 64, 65, 127, 128, 129, 0]))
    want = ops.shared_prefix_attention(q, kp, vp, k, v, **how)
    for bad in (float("nan"), float("inf")):
        for t in (kp, vp):
            t[0, :70], t[1, 201:] = bad, -bad
        for t in (k, v):
            for row, n in enumerate(how["lengths"].tolist()):
                t[row, n:] = bad
        assert torch.equal(ops.shared_prefix_attention(q, kp, vp, k, v, **how), want)
    _lib.check_device_errors()


def test_numbers_out_of_range_are_cut_off():
    t = _inputs(1, 2, 1, 90, 30, 4, 2, 64)
    assert torch.equal(ops.shared_prefix_attention(*t, prefix_start=_int([-5]), prefix_stop=_int([2**31 - 1]), lengths=_int([31, 2**31 - 1])), ops.shared_prefix_attention(*t))
    low = -(2**31)
    none = ops.shared_prefix_attention(*t, prefix_start=_int([2**31 - 1]), prefix_stop=_int([low]), lengths=_int([low, 1]))
    assert not none[0].any() and none[1].any()


@pytest.mark.parametrize("scale", [0.0, -0.1, 3.0])
def test_scales(scale):
    t = _inputs(1, 6, 1, 150, 70, 8, 2, 64)
    t[0].mul_(0.25)  # scores stay where 32 bits hold them to 2^-12
    _check(ops.shared_prefix_attention(*t, scale=scale), *t, scale=scale)


def test_scores_that_grow_along_the_keys():
    """The running maximum moves in every tile."""
    q, kp, vp, k, v = _inputs(1, 5, 1, 640, 260, 4, 1, 64)
    q.fill_(0.5)
    kp.copy_((torch.arange(640, device=DEV)[None, :, None, None] / 40).to(torch.bfloat16).expand_as(kp))
    k.copy_((18 + torch.arange(260, device=DEV)[None, :, None, None] / 40).to(torch.bfloat16).expand_as(k))
    _check(ops.shared_prefix_attention(q, kp, vp, k, v), q, kp, vp, k, v)
    _check(ops.shared_prefix_attention(q, kp.flip(1), vp, k, v), q, kp.flip(1), vp, k, v)


def test_non_finite_keys_that_are_seen():
    q, kp, vp, k, v = _inputs(1, 3, 1, 100, 50, 2, 2, 64)
    want = ops.shared_prefix_attention(q, kp, vp, k, v)
    k[1, 20, 0] = float("nan")
    out = ops.shared_prefix_attention(q, kp, vp, k, v)
    assert out[1, :, 0].isnan().all() and torch.equal(out[[0, 2]], want[[0, 2]]) and torch.equal(out[1, :, 1], want[1, :, 1])


def test_layouts():
    """Caches that are parts of larger ones, heads first, or at odd addresses."""
    q, kp, vp, k, v = _inputs(2, 6, 1, 130, 50, 8, 2, 64)
    want = ops.shared_prefix_attention(q, kp, vp, k, v)
    held = torch.randn(9, 80, 2, 64, device=DEV).to(torch.bfloat16)
    held[:6, :50] = k
    assert torch.equal(ops.shared_prefix_attention(q, kp, vp, held[:6, :50], v), want)
    turned = kp.transpose(1, 2).contiguous().transpose(1, 2)
    both = torch.cat([vp, vp], -1)[..., 64:]
    assert torch.equal(ops.shared_prefix_attention(q, turned, both, k, v), want)
    odd = torch.empty(v.numel() + 1, device=DEV, dtype=torch.bfloat16)[1:].view_as(v).copy_(v)
    assert torch.equal(ops.shared_prefix_attention(q, kp, vp, k, odd), want)
    wide = torch.cat([q, q], 2)[:, :, 8:]
    assert torch.equal(ops.shared_prefix_attention(wide, kp, vp, k, v), want)
    twice = kp[:1].expand(2, -1, -1, -1), vp[:1].expand(2, -1, -1, -1)
    _check(ops.shared_prefix_attention(q, *twice, k, v), q, *twice, k, v)


def test_what_has_no_kernel():
    q, kp, vp, k, v = _inputs(1, 2, 1, 10, 5, 2, 1, 64)
    with pytest.raises(ops.KernelFallbackError):
        ops.shared_prefix_attention(*(t[..., :32] for t in (q, kp, vp, k, v)))
    with pytest.raises(ops.KernelFallbackError):
        ops.shared_prefix_attention(q.requires_grad_(), kp, vp, k, v)
    wide = [t.detach().float() for t in (q, kp, vp, k, v)]
    torch.testing.assert_close(ops.shared_prefix_attention(*wide), reference.shared_prefix_attention(*(t.double() for t in wide), None, None, None, None).float(), rtol=1e-5, atol=1e-5)


def test_sizes_beyond_the_kernels_indices():
    with pytest.raises(ops.KernelFallbackError):
        ops.shared_prefix_attention(*_inputs(1, 1, 1, 3, 2, 257, 257, 64))
    with pytest.raises(ops.KernelFallbackError):
        ops.shared_prefix_attention(*_inputs(1, 5, 1, 3, 2, 30011, 1, 64))


def test_streams_recordings_and_lengths_that_move_on():
    t = _inputs(2, 8, 1, 400, 200, 8, 2, 128)
    lengths = _int([1] * 8)
    call = lambda: ops.shared_prefix_attention(*t, lengths=lengths)  # noqa: E731
    assert torch.equal(call(), call())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, call())
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, call()))
    for n in (1, 64, 65, 200, 0):
        lengths.fill_(n)
        for graph, out in graphs:
            out.zero_()
        for graph, out in graphs:
            graph.replay()
        for graph, out in graphs:
            assert torch.equal(out, call())
        _check(graphs[0][1], *t, lengths=lengths)


def test_same_as_attention_over_joined_keys():
    q, kp, vp, k, v = _inputs(2, 8, 1, 300, 60, 8, 2, 128)
    keys, values = (torch.cat([a.repeat_interleave(4, 0), b], 1) for a, b in ((kp, k), (vp, v)))
    want = ops.attention(q, keys, values, ops.AttentionMask(causal=True))
    size = ops.attention(q, keys, values.abs(), ops.AttentionMask(causal=True)).float()
    # both are within the bound of _check
    assert ((ops.shared_prefix_attention(q, kp, vp, k, v).float() - want.float()).abs() <= 2.0**-7 * want.float().abs() + 2 * (2.0**-8 + 2.0**-12) * 1.01 * size).all()


@pytest.mark.parametrize("d,hq,hkv,n,m", [(64, 8, 2, 3, 2), (128, 8, 8, 40, 25), (64, 64, 1, 100, 0), (128, 16, 4, 0, 70)])
def test_probabilities_are_not_rounded_to_16_bits(d, hq, hkv, n, m):
    """Values that cancel: outputs are far smaller than what they are sums of, whose roundings would show."""
    q, kp, vp, k, v = _inputs(2, 40, 1, n, m, hq, hkv, d)
    q.mul_(0.25), vp.sign_(), v.sign_()
    out = ops.shared_prefix_attention(q, kp, vp, k, v).double()
    want = reference.shared_prefix_attention(*(t.double() for t in (q, kp, vp, k, v)), None, None, None, None)
    # the output's rounding; 2^-16 of a probability as two bf16 numbers; scores, sums of d <= 128 products whose sizes add up to less than 4 with the scale: 128 * 4 * 2^-24 = 2^-15; exponentials, sums and
    # joins: some 50 roundings of 2^-24.  Sizes of values are 1.
    far = (out - want).abs() - (2.0**-8 * want.abs() + 2.0**-16 + 2.0**-15 + 2.0**-18)
    assert (far <= 0).all(), float(far.max())
    _lib.check_device_errors()


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_non_finite_values_that_are_seen(bad):
    """They reach the channel of the queries that see them and nothing else."""
    q, kp, vp, k, v = _inputs(2, 6, 1, 100, 70, 4, 2, 64)
    lengths = _int([70, 21, 20, 70, 70, 0])
    want = ops.shared_prefix_attention(q, kp, vp, k, v, lengths=lengths)
    v[:3, 20, 1, 5] = bad  # rows 0 and 1 see it, row 2 ends in front of it
    vp[1, 3, 0, 7] = bad  # rows 3 to 5
    out = ops.shared_prefix_attention(q, kp, vp, k, v, lengths=lengths)
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[:2, :, 2:, 5] = True
    hit[3:, :, :2, 7] = True
    assert not out[hit].isfinite().any() and torch.equal(out[~hit], want[~hit])
