"""Log-probabilities, entropies, alternatives and their gradients on the kernels, against the statement in 64 bits."""
import pytest
import torch

from torchtune_b200 import ops
from torchtune_b200.ops import _lib, reference

pytestmark = pytest.mark.gpu

DEV = "cuda"
INF = float("inf")
STEP = 2.0**-24


def _logits(*shape, seed=0, dtype=torch.bfloat16, spread=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (spread * torch.randn(*shape, generator=g, device=DEV)).to(dtype)


def _check(logits, tokens, temperature=1.0, top=0, grads=True, seed=1):
    """All outputs and the gradient with random weights against 64 bits."""
    v = logits.shape[-1]
    x = logits.detach().clone().requires_grad_(grads)
    with torch.set_grad_enabled(grads):
        s = ops.token_statistics(x, tokens, temperature=temperature, top=top)
    x64 = logits.double().requires_grad_(grads)
    want = reference.token_statistics(x64, tokens, temperature, top, -100)
    # a thread adds up v / 2048 vectors of 8, the CTA's threads 8 steps more; exponentials are 4 steps off and twice their argument's, which is below 60
    sums = 140 + v / 2048
    bound = STEP * (sums + 4 * want[0].abs())
    assert ((s.logprobs.double() - want[0]).abs() <= bound).all(), float((s.logprobs.double() - want[0]).abs().max())
    assert ((s.entropy.double() - want[1]).abs() <= STEP * 2 * sums * (1 + want[1])).all(), float((s.entropy.double() - want[1]).abs().max())
    if top:
        assert torch.equal(s.top_tokens, want[3])
        assert ((s.top_logprobs.double() - want[2]).abs() <= STEP * (sums + 4 * want[2].abs())).all()
    if not grads:
        return s
    g = torch.Generator(device=DEV).manual_seed(seed)
    weights = [torch.randn(t.shape, generator=g, device=DEV) for t in s[: 3 if top else 2]]
    (got,) = torch.autograd.grad(s[: len(weights)], x, weights)
    (exact,) = torch.autograd.grad(want[: len(weights)], x64, [w.double() for w in weights])
    assert got.dtype == logits.dtype and got.shape == logits.shape
    logp = torch.log_softmax(x64.detach() / temperature, -1)
    each = sum(w.double().abs().reshape(*tokens.shape, -1).sum(-1) for w in (weights[0], *weights[2:]))[..., None] + weights[1].double().abs()[..., None] * (want[1].detach()[..., None] + logp.abs())
    info = torch.finfo(got.dtype)
    bound = info.eps / 2 * exact.abs().clamp(min=info.tiny) + STEP * ((sums + 4 * logp.abs()) * logp.exp() * each + 8 * (each if top else weights[0].abs()[..., None])) / temperature + 1e-36
    bound = torch.where(torch.isfinite(bound), bound, torch.zeros_like(bound))
    far = (got.double() - exact).abs() - bound
    assert (far <= 0).all(), float(far.max())
    return s


@pytest.mark.parametrize("top", [0, 1, 20, 64])
@pytest.mark.parametrize("rows,v,dtype,temperature", [
    (1, 64, torch.float32, 1.0), (5, 257, torch.bfloat16, 0.7), (3, 2048, torch.float16, 1.3), (2, 4099, torch.bfloat16, 1.0), (40, 32003, torch.bfloat16, 0.9), (7, 50257, torch.float32, 0.5),
    (16, 128256, torch.float32, 1.0), (3, 151936, torch.bfloat16, 1.0), (700, 5001, torch.float16, 1.0)])
def test_against_64_bits(rows, v, dtype, temperature, top):
    logits = _logits(rows, v, dtype=dtype)
    tokens = torch.randint(0, v, (rows,), device=DEV)
    tokens[0] = logits[0].argmax()
    if rows > 2:
        tokens[1], tokens[2] = v - 1, -100
    _check(logits, tokens, temperature, top)


@pytest.mark.parametrize("v", [1, 2, 7, 8, 9, 31, 255])
def test_small_vocabularies(v):
    for dtype in (torch.bfloat16, torch.float32):
        _check(_logits(9, v, dtype=dtype), torch.arange(9, device=DEV) % v, top=min(v, 64))


@pytest.mark.parametrize("order", ["up", "down", "equal", "blocks"])
def test_alternatives_whatever_the_order(order):
    """Rows whose largest logits lie together, which a choice by parts could miss, and rows of ties."""
    v = 33000
    x = torch.arange(v, device=DEV, dtype=torch.float32) / 1000
    x = {"up": x, "down": x.flip(0), "equal": torch.zeros_like(x), "blocks": (torch.arange(v, device=DEV) // 300 % 7).float()}[order]
    for rows in (1, 600):
        s = _check(x.expand(rows, v).contiguous(), torch.zeros(rows, dtype=torch.int64, device=DEV), top=64, grads=rows == 1)
        assert s.top_tokens[0].tolist() == torch.sort(x, descending=True, stable=True).indices[:64].tolist()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,v,top", [(3, 700, 7), (700, 1, 1), (700, 33, 32), (700, 255, 0), (700, 1026, 12), (700, 2049, 64), (700, 8200, 33), (611, 8001, 20), (2000, 32003, 5), (4736 + 13, 900, 3)])
def test_many_short_rows(rows, v, top, dtype):
    """Rows of one warp each: a lane adds up v / 256 <= 126 vectors, and there are 13 steps more, which stays below the 140 steps of _check."""
    logits, tokens = _logits(rows, v, dtype=dtype), torch.randint(0, v, (rows,), device=DEV)
    tokens[::7] = -100
    _check(logits, tokens, 0.8, top)


@pytest.mark.parametrize("order", ["up", "down", "equal", "blocks"])
def test_alternatives_of_many_short_rows_whatever_the_order(order):
    for v in (200, 3000, 9000):
        x = torch.arange(v, device=DEV, dtype=torch.float32) / 1000
        x = {"up": x, "down": x.flip(0), "equal": torch.zeros_like(x), "blocks": (torch.arange(v, device=DEV) // 300 % 7).float()}[order]
        for top in (3, 32, 64):
            s = _check(x.expand(400, v).contiguous(), torch.zeros(400, dtype=torch.int64, device=DEV), top=top, grads=False)
            assert torch.equal(s.top_tokens, torch.sort(x, descending=True, stable=True).indices[:top].expand(400, top))


def test_short_rows_that_are_not_finite():
    x = _logits(640, 3000, dtype=torch.float32)
    x[0, 3:], x[1], x[2, 17], x[3, 2001], x[4, ::2] = -INF, -INF, float("nan"), INF, -INF
    x[5] = torch.finfo(torch.float32).min
    tokens = torch.ones(640, dtype=torch.int64, device=DEV)
    for top in (5, 40):
        s = ops.token_statistics(x, tokens, top=top)
        want = reference.token_statistics(x.double(), tokens, 1.0, top, -100)
        assert torch.equal(s.top_tokens, want[3])
        for a, b in zip(s[:3], want[:3]):
            torch.testing.assert_close(a.double(), b, rtol=2e-5, atol=2e-5, equal_nan=True)


def test_masked_and_non_finite_logits():
    v, low = 5000, torch.finfo(torch.float32).min
    x = _logits(8, v, dtype=torch.float32)
    x[0, 3:] = -INF  # three tokens are left
    x[1] = -INF
    x[2] = low
    x[3, 1:4999] = low
    x[4, 17] = float("nan")
    x[5, 4001] = INF
    x[6, ::2] = -INF
    x[7, :4096] = -INF  # whole segments
    tokens = torch.tensor([2, 0, 9, 0, 1, 1, 1, 4999], device=DEV)
    for case in (x, x[:, 1:]):  # rows that begin at odd addresses too
        s = ops.token_statistics(case, tokens, top=5)
        want = reference.token_statistics(case.double(), tokens, 1.0, 5, -100) if case.shape[1] == v else None
        if want is None:
            continue
        assert torch.equal(s.top_tokens, want[3])
        for a, b in zip(s[:3], want[:3]):
            torch.testing.assert_close(a.double(), b, rtol=2e-5, atol=2e-5, equal_nan=True)
        assert s.logprobs[[1, 4, 5]].isnan().all() and s.entropy[[1, 4, 5]].isnan().all() and s.logprobs[[0, 2, 3, 6, 7]].isfinite().all()
    leaf = x[[0, 2, 3, 6, 7]].requires_grad_()
    s = ops.token_statistics(leaf, tokens[[0, 2, 3, 6, 7]], top=2)
    (g,) = torch.autograd.grad(s.logprobs.sum() + s.entropy.sum() + s.top_logprobs[:, 0].sum(), leaf)
    assert g.isfinite().all() and not g[0, 3:].any() and not g[4, :4096].any()


@pytest.mark.parametrize("v", [1000, 70001])
def test_batches_that_share_their_logits(v):
    """Expanded along the batch, along the rows or both: every row its own token, and the results of a copy (whose rows of an odd width begin elsewhere, so that sums run in another order)."""
    for shape in ((1, 5, v), (60, 1, v), (1, 1, v)):
        leaf = _logits(*shape).requires_grad_()
        shared = leaf.expand(60, 5, v)
        tokens = torch.randint(0, v, (60, 5), device=DEV)
        s, want = ops.token_statistics(shared, tokens, top=3), _check(shared.detach().contiguous(), tokens, top=3, grads=False)
        assert torch.equal(s.top_tokens, want.top_tokens)
        for a, b in zip(s[:3], want[:3]):
            assert ((a - b).abs() <= 4 * STEP * (180 + 4 * b.abs()) * (1 + b.abs())).all()
        (g,) = torch.autograd.grad(s.logprobs.sum(), leaf)
        assert g.shape == leaf.shape and g.isfinite().all()
        if v % 8 == 0:
            (same,) = torch.autograd.grad(ops.token_statistics(shared.contiguous(), tokens, top=3).logprobs.sum(), leaf)
            assert torch.equal(g, same)


def test_gradients_of_rows_that_are_not_finite():
    """NaN reaches the gradient of a row with any weight; a row without weight (padding, say) has zeros."""
    x = _logits(6, 3000)
    x[0, 17], x[1] = float("nan"), -INF
    x[2, 5] = INF
    x[3, 99] = float("nan")
    leaf = x.requires_grad_()
    s = ops.token_statistics(leaf, torch.tensor([1, 2, 3, -100, 4, -100], device=DEV), top=3)
    for weight in (torch.ones(6, device=DEV), torch.zeros(6, device=DEV)):
        (g,) = torch.autograd.grad(s.logprobs, leaf, weight, retain_graph=True)
        assert not g[3].any() and not g[5].any() and g[4].isfinite().all()
        assert bool(weight.any()) == bool(g[:3].isnan().all()) == bool(g[4].any()) and (bool(weight.any()) or not g.any())
    (g,) = torch.autograd.grad(s.top_logprobs, leaf, torch.tensor([1.0, -1.0, 0.0], device=DEV).expand(6, 3))  # weights that add up to 0
    assert g[:4].isnan().all() and g[4:].isfinite().all() and g[4:].any(1).all()


def test_layouts():
    """Slices of a batch are read where they are; other layouts are copied; gradients have the logits' shape."""
    whole = _logits(3, 40, 1003)
    tokens = torch.randint(0, 1003, (3, 17), device=DEV)
    part = whole[:, 5:22]
    apart = ops.token_statistics(part.contiguous(), tokens, top=3)
    before = torch.cuda.memory_stats()["allocated_bytes.all.allocated"]
    s = ops.token_statistics(part, tokens, top=3)
    assert torch.cuda.memory_stats()["allocated_bytes.all.allocated"] - before < part.numel() * 2  # no copy
    # rows of an odd width begin at another address in a copy, and their sums run in another order: both are within the bound of _check
    def near(a, b):
        return bool(((a - b).abs() <= 2 * STEP * (141 + 4 * b.abs())).all())

    assert near(s.logprobs, apart.logprobs) and near(s.top_logprobs, apart.top_logprobs) and torch.equal(s.top_tokens, apart.top_tokens)
    assert ((s.entropy - apart.entropy).abs() <= 4 * STEP * 141 * (1 + apart.entropy)).all()
    turned = part.transpose(-1, -2).contiguous().transpose(-1, -2)
    assert torch.equal(ops.token_statistics(turned, tokens, top=3).logprobs, apart.logprobs)
    _check(part, tokens, top=3)
    leaf = whole.clone().requires_grad_()
    ops.token_statistics(leaf[:, 5:22], tokens).logprobs.sum().backward()
    assert not leaf.grad[:, :5].any() and not leaf.grad[:, 22:].any()
    again = part.contiguous().requires_grad_()
    ops.token_statistics(again, tokens).logprobs.sum().backward()
    # two roundings to bf16 of values 2 * 141 roundings of 32 bits apart
    assert ((leaf.grad[:, 5:22] - again.grad).abs() <= 2.0**-7 * again.grad.abs() + 2 * STEP * 141).all()
    one = ops.token_statistics(part[0, 0], tokens[0, 0], top=3)
    assert one.logprobs.shape == () and torch.equal(one.top_tokens, apart.top_tokens[0, 0])
    strided = ops.token_statistics(part, torch.stack([tokens, tokens], -1)[..., 0], top=3)
    assert torch.equal(strided.logprobs, s.logprobs)


def test_gradients_of_parts_of_the_result():
    logits, tokens = _logits(6, 3001), torch.randint(0, 3001, (6,), device=DEV)
    x64 = logits.double().requires_grad_()
    want = reference.token_statistics(x64, tokens, 1.0, 4, -100)
    for i in range(3):
        leaf = logits.clone().requires_grad_()
        s = ops.token_statistics(leaf, tokens, top=4)
        (g,) = torch.autograd.grad(s[i].sum(), leaf)
        (exact,) = torch.autograd.grad(want[i].sum(), x64, retain_graph=True)
        torch.testing.assert_close(g.double(), exact, rtol=2.0**-8, atol=1e-5)
    assert not s.top_tokens.requires_grad


def test_tokens_out_of_range_are_counted():
    logits = _logits(4, 99)
    _lib.index_violations()
    leaf = logits.clone().requires_grad_()
    s = ops.token_statistics(leaf, torch.tensor([99, -1, -100, 5], device=DEV))
    assert _lib.index_violations() == 2 and not s.logprobs[:3].any() and s.logprobs[3] < 0
    (g,) = torch.autograd.grad(s.logprobs.sum(), leaf)
    assert not g[:3].any() and g[3].any()


def test_results_do_not_change_and_recordings_hold_their_own():
    logits, tokens = _logits(9, 32003), torch.randint(0, 32003, (9,), device=DEV)
    leaf = logits.clone().requires_grad_()

    def step():
        s = ops.token_statistics(leaf, tokens, top=7)
        (g,) = torch.autograd.grad(s.logprobs.sum() - s.entropy.sum(), leaf)
        return (*(t.detach() for t in s), g)

    eager = step()
    assert all(torch.equal(a, b) for a, b in zip(eager, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert all(torch.equal(a, b) for a, b in zip(eager, step()))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for t in out:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, out))


def test_rows_beyond_32_bits():
    """Rows that begin behind 2^31 elements."""
    v, rows = 128256, 17000
    logits = torch.zeros(rows, v, dtype=torch.bfloat16, device=DEV)
    logits[-1] = _logits(v)
    tokens = torch.full((rows,), 7, device=DEV)
    s = ops.token_statistics(logits, tokens, top=2)
    want = reference.token_statistics(logits[-1:].double(), tokens[-1:], 1.0, 2, -100)
    assert torch.equal(s.top_tokens[-1:], want[3])
    torch.testing.assert_close(s.logprobs[-1:].double(), want[0], rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(s.entropy[-1:].double(), want[1], rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,v,top", [(640, 1000, 5), (640, 3000, 40), (640, 12000, 64), (3, 50000, 7)])
def test_rows_of_nan_keep_the_first_index(rows, v, top, dtype):
    """All of them equal and above all numbers: the choice of one alternative after the other, too, begins at index 0."""
    x = _logits(rows, v, dtype=dtype)
    x[::2] = float("nan")
    x[1::4, 0] = float("nan")
    s = ops.token_statistics(x, torch.zeros(rows, dtype=torch.int64, device=DEV), top=top)
    assert torch.equal(s.top_tokens, torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top])
    assert s.top_logprobs[::2].isnan().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,v", [(700, 600), (700, 9001), (300, 70000), (3, 128256)])
def test_sure_tokens(rows, v, dtype):
    """One token far above another one, and nothing else: probabilities do not go above 1 nor entropies below 0."""
    g = torch.Generator(device=DEV).manual_seed(2)
    x = torch.full((rows, v), -80.0, device=DEV)
    first, sure = torch.randint(0, 8, (rows,), generator=g, device=DEV), 256 + torch.randint(0, 8, (rows,), generator=g, device=DEV)  # the same lane's elements
    x.scatter_(1, first[:, None], 0.0)
    x.scatter_(1, sure[:, None], 12 + 5 * torch.rand(rows, 1, generator=g, device=DEV))
    x = x.to(dtype)
    s = ops.token_statistics(x, sure, top=2)
    want = reference.token_statistics(x.double(), sure, 1.0, 2, -100)
    assert (s.logprobs <= 0).all() and (s.top_logprobs <= 0).all() and (s.entropy >= 0).all()
    # sums of 1 + 2^-17 and less: a rounding for each of some 12 joins of lanes and warps; t is below 2^-12 and its roundings nothing; the logarithm is one step off, the product with ln 2 half of one
    assert (s.logprobs.double() - want[0]).abs().max() <= 16 * STEP
    assert (s.top_logprobs[:, 0].double() - want[2][:, 0]).abs().max() <= 16 * STEP
    assert (s.entropy.double() - want[1]).abs().max() <= 16 * STEP


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("copies", [1, 100])
@pytest.mark.parametrize("skip", [1, 3, 7])
def test_masked_and_non_finite_logits_at_odd_addresses(skip, copies, dtype):
    """Rows that do not begin on 16 bytes and end anywhere, few and many: their first and last elements are read one by one."""
    v, low = 5001, torch.finfo(dtype).min
    x = _logits(8 * copies, v + skip, dtype=dtype).view(copies, 8, v + skip)
    x[:, 0, skip + 3 :] = -INF  # three tokens are left
    x[:, 1] = -INF
    x[:, 2] = low
    x[:, 3, skip + 1 : -1] = low
    x[:, 4, skip] = float("nan")
    x[:, 5, -1] = INF
    x[:, 6, ::2] = -INF
    x[:, 7, : 4096 + skip] = -INF  # whole segments
    x[:, :, :skip] = float("nan")  # in front of the rows
    case = x.view(8 * copies, v + skip)[:, skip:]
    tokens = torch.tensor([2, 0, 9, 0, 1, 1, 1 - skip % 2 + 1, v - 1], device=DEV).repeat(copies)
    leaf = case.detach().requires_grad_()
    s = ops.token_statistics(leaf, tokens, top=5)
    want = reference.token_statistics(case.double(), tokens, 1.0, 5, -100)
    assert torch.equal(s.top_tokens, want[3])
    for a, b in zip(s[:3], want[:3]):
        torch.testing.assert_close(a.detach().double(), b, rtol=2e-5, atol=2e-5, equal_nan=True)
    (g,) = torch.autograd.grad(s.logprobs.sum() + s.entropy.sum(), leaf)
    g = g.view(copies, 8, v)
    assert g[:, [1, 4, 5]].isnan().all() and g[:, [0, 2, 3, 7]].isfinite().all() and not g[:, 0, 3:].any() and not g[:, 7, :4096].any() and g[:, 7, 4096:].any(-1).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_one_logit_is_certain(dtype):
    """And so is one beside infinitely low ones: nothing is left to round."""
    one = _logits(900, 1, dtype=dtype)
    few = torch.cat([one, torch.full((900, 30), -INF, device=DEV, dtype=dtype)], 1)
    for x in (one, few):
        leaf = x.requires_grad_()
        s = ops.token_statistics(leaf, torch.zeros(900, dtype=torch.int64, device=DEV), temperature=0.7, top=1)
        (g,) = torch.autograd.grad(s.logprobs.sum() + 3 * s.entropy.sum(), leaf)
        assert not s.logprobs.any() and not s.entropy.any() and not s.top_logprobs.any() and not g.any()
