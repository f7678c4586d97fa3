"""Norms of queries and keys per head with the rotation, on the kernels: against the statement in 64 bits, at the sizes, layouts and types that they distinguish."""
import pytest
import torch

from torchtune_b200 import ops
from torchtune_b200.ops import _lib, reference

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _table(n, d):
    angle = torch.arange(n, dtype=torch.float64, device=DEV)[:, None] * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=DEV) / d)
    return torch.stack([angle.cos(), angle.sin()], -1).float()


def _inputs(b, s, hq, hk, d, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    make = lambda *shape: torch.randn(*shape, generator=g, device=DEV)  # noqa: E731
    return make(b, s, hq, d).to(dtype), (3 * make(b, s, hk, d)).to(dtype), (1 + 0.3 * make(d)).to(dtype), (1 + 0.3 * make(d)).to(dtype)


def _step(dtype):
    return torch.finfo(dtype).eps / 2


def _close(got, want, size, roundings):
    """One rounding of the result, and ``roundings`` of 32 bits of values of ``size``."""
    bound = _step(got.dtype) * want.abs() + roundings * 2.0**-24 * size
    worst = ((got.double() - want).abs() - bound).max()
    assert worst <= 0, f"off by {float(worst)} more than the bound"


def _check_forward(x, gain, out, table, pos, eps, interleaved, norm_first):
    want = reference.norm_rope(x.double(), None if gain is None else gain.double(), table, pos, eps, interleaved, norm_first)
    # the sum of squares (up to 32 terms of a lane, 5 of a tree), its root, three products and a rotation of values up to the largest of the head
    _close(out, want, want.abs().amax(-1, keepdim=True), 64)


@pytest.mark.parametrize("norm_first", [True, False])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("b,s,hq,hk,d,dtype", [
    (1, 1, 1, 1, 16, torch.bfloat16), (2, 3, 4, 2, 64, torch.bfloat16), (3, 7, 5, 1, 48, torch.bfloat16), (1, 33, 32, 8, 128, torch.bfloat16), (2, 5, 3, 3, 96, torch.float16),
    (2, 9, 6, 2, 256, torch.float32), (1, 4, 2, 1, 512, torch.bfloat16), (2, 11, 7, 2, 80, torch.float32), (2, 901, 17, 6, 128, torch.bfloat16)])
def test_forward_and_gradients(b, s, hq, hk, d, dtype, interleaved, norm_first):
    q, k, gq, gk = _inputs(b, s, hq, hk, d, dtype)
    table, eps = 1.1 * _table(s + 5, d), 1e-5
    pos = torch.randint(0, s + 5, (b, s), device=DEV)
    leaves = [t.clone().requires_grad_() for t in (q, k, gq, gk)]
    out = ops.qk_norm_rope(*leaves, table, pos, eps=eps, interleaved=interleaved, norm_first=norm_first)
    dy = [torch.randn_like(t) for t in out]
    grads = torch.autograd.grad(out, leaves, dy)
    for i, (x, gain) in enumerate(((q, gq), (k, gk))):
        assert out[i].dtype == dtype and out[i].is_contiguous()
        _check_forward(x, gain, out[i], table, pos, eps, interleaved, norm_first)
        x64, w64 = x.double().requires_grad_(), gain.double().requires_grad_()
        want = torch.autograd.grad(reference.norm_rope(x64, w64, table, pos, eps, interleaved, norm_first), (x64, w64), dy[i].double())
        x64 = x64.detach()
        r = 1.1 * (x64.square().mean(-1, keepdim=True) + eps).rsqrt() if norm_first else (1.21 * x64.square().mean(-1, keepdim=True) + eps).rsqrt() * 1.1
        top = 1.6 * dy[i].double().abs().amax(-1, keepdim=True) * gain.double().abs().max()  # of dn: a rotation of a pair is up to sqrt(2), the table 1.1 long
        n = x64.abs().amax(-1, keepdim=True) * r * 1.5
        assert grads[i].dtype == dtype
        # two sums, a product, a difference of values up to top (1 + n), and a rotation
        _close(grads[i], want[0], r * top * (1 + n), 128)
        # sums of up to 8 terms of a lane, 5 steps of a tree, 8 warps, 10 rows of the workspace and 6 steps of a tree, of values up to top n
        _close(grads[2 + i], want[1], (top * n / gain.double().abs().max()).sum(), 128)


def test_types_of_gains():
    q, k, gq, gk = _inputs(2, 3, 4, 2, 64)
    table = _table(8, 64)
    for a, c in ((gq.float(), gk.float()), (gq.float(), gk), (None, gk), (gq, None), (None, None), (gq.half(), gk)):
        leaves = [None if g is None else g.clone().requires_grad_() for g in (a, c)]
        x = q.clone().requires_grad_()
        out = ops.qk_norm_rope(x, k, *leaves, table)
        _check_forward(q, a, out[0], table, None, 1e-6, True, True)
        _check_forward(k, c, out[1], table, None, 1e-6, True, True)
        (out[0].float().sum() + out[1].float().square().sum()).backward()
        for g in leaves:
            assert g is None or (g.grad.dtype == g.dtype and g.grad.abs().sum() > 0)


def test_layouts():
    """Queries, keys and gradients that are parts of one projection, transposed heads, and rows that start at odd addresses."""
    b, s, d = 2, 6, 64
    table = _table(s, d)
    wide = torch.randn(b, s, 8 * d, device=DEV).to(torch.bfloat16).requires_grad_()
    q, k = wide[..., : 6 * d].view(b, s, 6, d), wide[..., 6 * d :].view(b, s, 2, d)
    gain = torch.ones(d, device=DEV, dtype=torch.bfloat16)
    apart = ops.qk_norm_rope(q.detach().contiguous(), k.detach().contiguous(), gain, gain, table)
    out = ops.qk_norm_rope(q, k, gain, gain, table)
    assert torch.equal(out[0], apart[0]) and torch.equal(out[1], apart[1])
    dy = torch.randn(b, s, 8, d, device=DEV).to(torch.bfloat16)
    out[0].backward(dy[:, :, :6], retain_graph=True)  # no gradient of the keys
    assert not wide.grad[..., 6 * d :].any() and wide.grad[..., : 6 * d].any()
    turned = q.detach().transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(ops.qk_norm_rope(turned, k.detach(), gain, gain, table)[0], apart[0])
    odd = torch.empty(q.numel() + 1, device=DEV, dtype=torch.bfloat16)[1:].view_as(q).copy_(q.detach())
    odd_gain = torch.ones(d + 1, device=DEV, dtype=torch.bfloat16)[1:]
    assert torch.equal(ops.qk_norm_rope(odd, k.detach(), odd_gain, gain, table)[0], apart[0])
    rounded = table.to(torch.bfloat16)
    assert torch.equal(ops.qk_norm_rope(q.detach(), k.detach(), gain, gain, rounded)[0], ops.qk_norm_rope(q.detach(), k.detach(), gain, gain, rounded.float())[0])
    spread = torch.ones((), device=DEV, dtype=torch.bfloat16).expand(b, s, 6, d)
    x = q.detach().clone().requires_grad_()
    (g1,) = torch.autograd.grad(ops.qk_norm_rope(x, k.detach(), gain, gain, table)[0], x, spread)
    (g2,) = torch.autograd.grad(ops.qk_norm_rope(x, k.detach(), gain, gain, table)[0], x, spread.contiguous())
    assert torch.equal(g1, g2)


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("b,s,hq,hk,d,dtype", [(1, 1, 32, 8, 128, torch.bfloat16), (16, 1, 16, 8, 64, torch.bfloat16), (3, 5, 4, 1, 80, torch.float32), (2, 601, 32, 8, 128, torch.float16)])
def test_append(b, s, hq, hk, d, dtype, interleaved):
    q, k, gq, gk = _inputs(b, s, hq, hk, d, dtype)
    v = torch.randn_like(k)
    held = torch.full((2, b, s + 7, hk, d + 16), 5.0, device=DEV, dtype=dtype)
    k_cache, v_cache = held[0, ..., :d], held[1, ..., :d]  # rows that lie apart
    slots = torch.arange(3, 3 + s, device=DEV)
    pos = torch.randint(0, 50, (b,) if s == 1 else (b, s), device=DEV, dtype=torch.int32)
    table = _table(50, d)
    out = ops.qk_norm_rope_append(q, k, v, gq, gk, table, pos, k_cache, v_cache, slots, interleaved=interleaved)
    want = ops.qk_norm_rope(q, k, gq, gk, table, pos, interleaved=interleaved)
    assert torch.equal(out, want[0]) and torch.equal(k_cache[:, slots], want[1]) and torch.equal(v_cache[:, slots], v)
    held[0, :, 3 : 3 + s, :, :d], held[1, :, 3 : 3 + s, :, :d] = 5.0, 5.0
    assert (held == 5).all()


def test_indices_out_of_range_are_counted_and_write_nothing():
    q, k, gq, gk = _inputs(2, 3, 4, 2, 64)
    table = _table(8, 64)
    _lib.index_violations()
    far = ops.qk_norm_rope(q, k, gq, gk, table, torch.tensor([[0, 8, 2**40], [1, -1, 7]], device=DEV))
    assert _lib.index_violations() == 3
    near = ops.qk_norm_rope(q, k, gq, gk, table, torch.tensor([[0, 0, 0], [1, 0, 7]], device=DEV))
    assert torch.equal(far[0], near[0]) and torch.equal(far[1], near[1])
    caches = [torch.zeros(2, 4, 2, 64, device=DEV, dtype=torch.bfloat16) for _ in range(2)]
    ops.qk_norm_rope_append(q, k, k, gq, gk, table, None, *caches, torch.tensor([-1, 2, 4], device=DEV))
    assert _lib.index_violations() == 4  # two slots of two rows
    for c in caches:
        assert c[:, 2].any() and not c[:, [0, 1, 3]].any()


def test_empty_and_head_dimensions_without_a_kernel():
    table, gain = _table(4, 24), torch.ones(24, device=DEV)
    q, k = ops.qk_norm_rope(torch.zeros(0, 3, 2, 24, device=DEV), torch.zeros(0, 3, 1, 24, device=DEV), gain, gain, table)
    assert q.shape == (0, 3, 2, 24) and k.shape == (0, 3, 1, 24)
    x = torch.randn(2, 3, 2, 24, device=DEV)
    _check_forward(x, gain, ops.qk_norm_rope(x, x, gain, gain, table)[0], table, None, 1e-6, True, True)
    with pytest.raises(ops.KernelFallbackError):
        ops.qk_norm_rope(x.bfloat16(), x.bfloat16(), gain, gain, table)


def test_streams_and_recordings():
    q, k, gq, gk = _inputs(2, 64, 16, 8, 128)
    table = _table(64, 128)
    want = ops.qk_norm_rope(q, k, gq, gk, table)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.qk_norm_rope(q, k, gq, gk, table)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])

    leaves = [t.clone().requires_grad_() for t in (q, k, gq, gk)]
    dy = [torch.randn_like(t) for t in want]

    def step():
        return torch.autograd.grad(ops.qk_norm_rope(*leaves, table), leaves, dy)

    eager = step()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two recordings do not share a workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, step()))
    for graph, out in graphs:
        for t in out:
            t.zero_()
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_plain_writes_leave_out_slots_that_a_cache_does_not_have():
    """Head sizes and types without a kernel: as the kernel does."""
    for d, dtype in ((24, torch.float32), (16, torch.float64)):
        q, k, v = (torch.randn(2, 4, h, d, device=DEV, dtype=dtype) for h in (4, 2, 2))
        table = torch.randn(20, d // 2, 2, device=DEV)
        caches = [torch.randn(2, 9, 2, d, device=DEV, dtype=dtype) for _ in range(2)]
        want = [c.clone() for c in caches]
        out_q, out_k = ops.qk_norm_rope(q, k, None, None, table)
        for c, new in zip(want, (out_k, v)):
            c[:, 8], c[:, 2] = new[:, 0], new[:, 3]
        got = ops.qk_norm_rope_append(q, k, v, None, None, table, None, *caches, torch.tensor([8, 9, -1, 2], device=DEV))
        assert torch.equal(got, out_q) and all(torch.equal(a, b) for a, b in zip(caches, want))
