"""Attention with a sliding window beside which the first tokens (of each document) stay visible: kernels against the definition in float64."""
import warnings

import pytest
import torch

pytestmark = pytest.mark.gpu

from torchtune_b200 import ops
from torchtune_b200.ops.mask import AttentionMask


@pytest.fixture(autouse=True)
def _check_device_errors():
    yield
    from torchtune_b200.ops._lib import check_device_errors

    torch.cuda.synchronize()
    check_device_errors()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(*shape, seed):
    return torch.randn(*shape, generator=_gen(seed), device="cuda").to(torch.bfloat16)


def _docs(b, s, mean, seed=0):
    border = torch.rand(b, s, generator=_gen(seed), device="cuda") < 1.0 / mean
    border[:, 0] = False
    return border.cumsum(1).to(torch.int32)


def _visible(sq, sk, window, sinks, docs=None):
    i, j = torch.arange(sq, device="cuda")[:, None] + sk - sq, torch.arange(sk, device="cuda")[None, :]
    seen, first = j <= i, torch.zeros(1, 1, sk, dtype=torch.long, device="cuda")
    if docs is not None:
        seen = seen & (docs[:, :, None] == docs[:, None, :])
        first = torch.stack([torch.searchsorted(d.contiguous(), d.contiguous()) for d in docs])[:, None, :]
    return (seen & ((i - j < window) | (j - first < sinks))).expand(1 if docs is None else docs.shape[0], sq, sk)


def _formula(q, k, v, d_o, seen, scale):
    """Output and gradients in float64, a key head at a time."""
    b, s, hq, d = q.shape
    hkv = k.shape[2]
    out, dq, dk, dv = (torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in (q, q, k, v))
    square = torch.zeros_like(out)
    for h in range(hkv):
        group = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
        qd, dod = (t[:, :, group].double().permute(0, 2, 1, 3) for t in (q, d_o))
        kd, vd = (t[:, :, h].double()[:, None] for t in (k, v))
        p = torch.softmax((qd @ kd.transpose(-1, -2) * scale).masked_fill(~seen[:, None], float("-inf")), -1)
        o = p @ vd
        ds = p * (dod @ vd.transpose(-1, -2) - (dod * o).sum(-1, keepdim=True)) * scale
        out[:, :, group], dq[:, :, group] = o.permute(0, 2, 1, 3), (ds @ kd).permute(0, 2, 1, 3)
        square[:, :, group] = (p.square() @ vd.square()).permute(0, 2, 1, 3)
        dk[:, :, h], dv[:, :, h] = (ds.transpose(-1, -2) @ qd).sum(1), (p.transpose(-1, -2) @ dod).sum(1)
    return out, square, dq, dk, dv


def _near(got, want, square):
    # as for the other attention kernels: the result is rounded to 8 bits, and so is every weight before it meets its value (14 standard deviations)
    bound = 2.0**-8 * want.abs() + 2.0**-6 * square.sqrt()
    assert ((got.double() - want).abs() <= bound).all(), float(((got.double() - want).abs() - bound).max())


def _check_gradients(got, want, d_o, out, scale):
    """Weights, dS and the output inside delta are rounded to 8 bits (2^-9 each of terms without a common sign), the result too: 2^-7 of the norm of a row, twice that allowed, and a
    sixty-fourth of the typical row for rows whose terms cancel.  Where a query sees one key, dP - delta is 0 in exact arithmetic and the difference of two fp32 sums of d products here: off by at
    most 2^-22 |dO| |v| (a sum of up to 128 terms in any order, twice), so a row by 2^-22 |dO| |v| |k| scale, and three norms of d standard normals, each below 1.5 sqrt(d), times
    a scale of up to 3 / sqrt(d) are below 2^4 d.

    Where a query sees few keys, dS is small beside delta = sum dO o, whose o is rounded to 8 bits: errors of at most 2^-9 |o| with a standard deviation of 2^-9 |o| / sqrt(3), of random signs,
    so 2^-9 |dO o| / sqrt(3) in delta and at most that times scale and the largest |k|, 1.5 sqrt(d), in a row of dQ (weights add up to 1); eight standard deviations are 2^-9 x 4.7."""
    delta = 4.7 * 2.0**-9 * (d_o.double() * out).norm(dim=-1) * abs(scale) * 1.5 * out.shape[-1] ** 0.5
    for name, a, w in zip(("dq", "dk", "dv"), got, want):
        rows = w.norm(dim=-1)
        off = (a.double() - w).norm(dim=-1)
        bound = (delta if name == "dq" else 0.0) + 2.0**-6 * rows + 2.0**-6 * rows.square().mean().sqrt() + 2.0**-18 * w.shape[-1]
        assert (off <= bound).all(), (name, float((off - bound).max()), float(rows.max()))


CASES = [  # s, window, sinks, documents of about this length (0: none)
    (1, 1, 0, 0), (2, 1, 1, 0), (63, 5, 1, 0), (128, 128, 4, 0), (129, 16, 4, 0), (257, 100, 130, 0), (300, 1, 2, 0), (400, 64, 0, 0), (513, 129, 7, 0), (1000, 100, 4, 0), (1000, 3, 300, 0),
    (777, 900, 5, 0), (2000, 250, 3, 0), (130, 20, 3, 40), (1000, 60, 2, 300), (1000, 100, 140, 500), (640, 30, 1, 5), (1537, 200, 4, 3000), (384, 1, 1, 128),
]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("s, window, sinks, mean", CASES)
def test_forward_and_backward(s, window, sinks, mean, d):
    b, hq, hkv = 2, 4, 2
    q, k, v, d_o = (_randn(b, s, h, d, seed=i) for i, h in ((1, hq), (2, hkv), (3, hkv), (4, hq)))
    docs = _docs(b, s, mean) if mean else None
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = ops.attention(*leaves, AttentionMask(window=window, sinks=sinks, doc_ids=docs))
    grads = torch.autograd.grad(out, leaves, d_o)
    want, square, *wants = _formula(*(t.detach() for t in leaves), d_o, _visible(s, s, window, sinks, docs), d**-0.5)
    _near(out, want, square)
    _check_gradients(grads, wants, d_o, want, d**-0.5)
    with torch.no_grad():
        _near(ops.attention(*leaves, AttentionMask(window=window, sinks=sinks, doc_ids=docs)), want, square)  # a few queries take another kernel


@pytest.mark.parametrize("s, window, sinks, mean", CASES)
def test_every_pair_that_is_visible_counts_and_no_other(s, window, sinks, mean):
    """Queries of zeros: all visible keys weigh the same, so one pair too many or too few shows."""
    if window > 300:
        window = 300
    b, d = 2, 64
    docs = _docs(b, s, mean, seed=7) if mean else None
    q, k = torch.zeros(b, s, 1, d, device="cuda", dtype=torch.bfloat16), _randn(b, s, 1, d, seed=2)
    v, d_o = (_randn(b, s, 1, d, seed=i).sign() for i in (3, 4))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = ops.attention(*leaves, AttentionMask(window=window, sinks=sinks, doc_ids=docs))
    (dv,) = torch.autograd.grad(out, v, d_o)
    seen = _visible(s, s, window, sinks, docs).double().expand(b, s, s)
    count = seen.sum(-1, keepdim=True)
    want = (seen @ v[:, :, 0].double()) / count  # weights are 1 on the way: the sum is exact
    assert ((out[:, :, 0].double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-20).all()
    weight = seen / count
    want = weight.transpose(1, 2) @ d_o[:, :, 0].double()
    # weights 1 / count are rounded by at most 2^-9 of each, without a common sign: eight standard deviations, below the smallest weight up to 600 queries
    bound = 2.0**-8 * want.abs() + 2.0**-6 * weight.square().sum(1)[:, :, None].sqrt()
    assert ((dv[:, :, 0].double() - want).abs() <= bound).all()


@pytest.mark.parametrize("hq, hkv", [(1, 1), (6, 2), (8, 1), (5, 5)])
def test_head_layouts_and_scales(hq, hkv):
    s, d = 300, 64
    for scale in (0.3, -0.2, 0.0):
        q, k, v, d_o = (_randn(1, s, h, d, seed=i + hq) for i, h in ((1, hq), (2, hkv), (3, hkv), (4, hq)))
        leaves = [t.requires_grad_() for t in (q, k, v)]
        out = ops.attention(*leaves, AttentionMask(window=70, sinks=5), scale=scale)
        grads = torch.autograd.grad(out, leaves, d_o)
        want, square, *wants = _formula(*(t.detach() for t in leaves), d_o, _visible(s, s, 70, 5), scale)
        _near(out, want, square)
        _check_gradients(grads, wants, d_o, want, scale)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("s, sk", [(1, 1), (1, 2), (1, 700), (1, 4099), (3, 333), (4, 64), (100, 700), (130, 131), (256, 1000), (17, 2000)])
@pytest.mark.parametrize("window, sinks", [(1, 0), (16, 4), (200, 1), (64, 500), (5000, 3)])
def test_queries_at_the_end_of_the_keys(s, sk, window, sinks, d):
    q, k, v, d_o = (_randn(2, n, h, d, seed=i + s) for i, n, h in ((1, s, 8), (2, sk, 2), (3, sk, 2), (4, s, 8)))
    mask = AttentionMask(window=window, sinks=sinks)
    want, square, *wants = _formula(q, k, v, d_o, _visible(s, sk, window, sinks), d**-0.5)
    with torch.no_grad():
        _near(ops.attention(q, k, v, mask), want, square)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = ops.attention(*leaves, mask)
    _near(out, want, square)
    if s > 1 or sk < 5:
        _check_gradients(torch.autograd.grad(out, leaves, d_o), wants, d_o, want, d**-0.5)
    else:  # one query: keys that it does not see have gradients of exactly 0
        grads = torch.autograd.grad(out, leaves, d_o)
        hidden = ~_visible(s, sk, window, sinks)[0, 0]
        assert not grads[1][:, hidden].any() and not grads[2][:, hidden].any()
        _check_gradients(grads[:1], wants[:1], d_o, want, d**-0.5)


def test_a_batch_row_does_not_reach_into_the_next():
    """Infinities and NaN in one row, in front of and behind the others' ends, leave those as they are."""
    for docs in (None, _docs(3, 200, 60)):
        q, k, v, d_o = (_randn(3, 200, h, 64, seed=i) for i, h in ((1, 4), (2, 2), (3, 2), (4, 4)))
        mask = AttentionMask(window=50, sinks=3, doc_ids=docs)

        def run():
            leaves = [t.clone().requires_grad_() for t in (q, k, v)]
            out = ops.attention(*leaves, mask)
            return [out.detach(), *torch.autograd.grad(out, leaves, d_o)]

        clean = run()
        for t in (q, k, v, d_o):
            t[1] = float("nan")
        q[1, ::2], k[1, 1::2] = float("inf"), float("-inf")
        spoilt = run()
        for a, c in zip(clean, spoilt):
            # dQ is summed by atomics, whose order differs from run to run: fp32 sums of five blocks, then 8 bits
            assert ((a[::2].float() - c[::2].float()).abs() <= 2.0**-7 * a[::2].float().abs() + 1e-5).all()
            assert torch.equal(a[::2], c[::2]) or a.shape == q.shape


def test_strided_and_odd_inputs():
    base = _randn(2, 300, 8, 72, seed=1)
    q, k, v = base[:, :, :4, 3:67], base[:, :, 4:6, 8:], base[:, :, 6:, 1:65]
    mask = AttentionMask(window=40, sinks=3)
    want, square, *_ = _formula(q, k, v, q, _visible(300, 300, 40, 3), 64**-0.5)
    _near(ops.attention(q, k, v, mask), want, square)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ops.attention(*leaves, mask)
    d_o = _randn(2, 4, 300, 65, seed=5)[..., 1:].transpose(1, 2)
    full = _formula(q, k, v, d_o, _visible(300, 300, 40, 3), 64**-0.5)
    _check_gradients(torch.autograd.grad(out, leaves, d_o), full[2:], d_o, full[0], 64**-0.5)
    # the same keys for all batch rows: their gradient is the sum
    one = k[:1].detach().requires_grad_()
    out = ops.attention(q, one.expand(2, -1, -1, -1), v, mask)
    (grad,) = torch.autograd.grad(out, one, d_o)
    want = _formula(q, k[:1].expand(2, -1, -1, -1), v, d_o, _visible(300, 300, 40, 3), 64**-0.5)[3].sum(0, keepdim=True)
    assert (grad.double() - want).norm() <= 2.0**-6 * want.norm()


def test_long_documents_meet_their_first_tokens():
    """Documents of very different lengths in one row, borders on and beside the borders of tiles."""
    lengths = [1, 127, 128, 1, 255, 300, 2, 700, 22]
    ids = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths)).to(device="cuda", dtype=torch.int32)[None]
    s = ids.shape[1]
    q, k, v, d_o = (_randn(1, s, h, 128, seed=i) for i, h in ((1, 2), (2, 1), (3, 1), (4, 2)))
    for window, sinks in ((7, 2), (130, 1), (1, 128), (300, 0), (40, 600)):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = ops.attention(*leaves, AttentionMask(window=window, sinks=sinks, doc_ids=ids))
        grads = torch.autograd.grad(out, leaves, d_o)
        want, square, *wants = _formula(q, k, v, d_o, _visible(s, s, window, sinks, ids), 128**-0.5)
        _near(out, want, square)
        _check_gradients(grads, wants, d_o, want, 128**-0.5)


def test_gradient_against_differences():
    s, d = 200, 64
    q, k, v, d_o, u = (_randn(1, s, h, d, seed=i) for i, h in ((1, 2), (2, 1), (3, 1), (4, 2), (5, 1)))
    seen = _visible(s, s, 30, 4)
    for which in (1, 2):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        grad = torch.autograd.grad(ops.attention(*leaves, AttentionMask(window=30, sinks=4)), leaves, d_o)[which]
        step, ends = 1e-4, []
        for sign in (1, -1):
            moved = [t.double() for t in (q, k, v)]
            moved[which] = moved[which] + sign * step * u.double()
            ends.append((_formula(*moved, d_o, seen, d**-0.5)[0] * d_o.double()).sum())
        slope = float((ends[0] - ends[1]) / (2 * step))
        # the product with a random direction: the gradient's relative error of 2^-7 of |grad| |u| / sqrt(size), over a sum of its size; eight standard deviations
        spread = float(grad.double().norm()) * 2.0**-7 * 8
        assert abs(float((grad.double() * u.double()).sum()) - slope) <= spread


def test_the_same_forward_twice_on_another_stream_and_recorded():
    q, k, v, d_o = (_randn(1, 700, h, 64, seed=i) for i, h in ((1, 4), (2, 2), (3, 2), (4, 4)))
    mask = AttentionMask(window=100, sinks=4)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = ops.attention(*leaves, mask)
    grads = torch.autograd.grad(out, leaves, d_o)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ops.attention(*leaves, mask)
        grads_again = torch.autograd.grad(again, leaves, d_o)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, again) and torch.equal(grads[1], grads_again[1]) and torch.equal(grads[2], grads_again[2])
    static = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    graph = torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(ops.attention(*static, mask), static, d_o)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        recorded = ops.attention(*static, mask)
        recorded_grads = torch.autograd.grad(recorded, static, d_o)
    for seed in (11, 12):
        fresh = [_randn(*t.shape, seed=seed + i) for i, t in enumerate(static)]
        with torch.no_grad():
            for t, f in zip(static, fresh):
                t.copy_(f)
        graph.replay()
        leaves = [f.requires_grad_() for f in fresh]
        out = ops.attention(*leaves, mask)
        grads = torch.autograd.grad(out, leaves, d_o)
        assert torch.equal(recorded, out) and torch.equal(recorded_grads[1], grads[1]) and torch.equal(recorded_grads[2], grads[2])


def test_what_the_kernels_do_not_take_is_not_computed_otherwise():
    q, k = _randn(1, 40, 2, 64, seed=1), _randn(1, 20, 2, 64, seed=2)
    from torchtune_b200.ops import KernelFallbackError

    for mask, keys in ((AttentionMask(window=5, sinks=2, chunk=8), q), (AttentionMask(window=5, sinks=2), k)):
        with pytest.raises(KernelFallbackError):
            ops.attention(q, keys, keys, mask)
    with pytest.raises(KernelFallbackError):
        ops.attention(q, q, q, AttentionMask(window=5, sinks=2), softcap=10.0)


def test_a_model_is_tuned_and_generates_with_windows():
    """A training step of a windowed decoder, packed, and generation over its quantised cache: gradients exist, and cached steps agree with the whole pass."""
    from torchtune_b200 import generation
    from torchtune_b200.models.mistral import mistral

    torch.manual_seed(2)
    with torch.device("cuda"):
        model = mistral(vocab_size=304, num_layers=2, num_heads=4, num_kv_heads=2, embed_dim=256, intermediate_dim=256, max_seq_len=512, sliding_window_size=40, attention_sinks=3).to(torch.bfloat16)
    tokens = torch.randint(1, 304, (2, 300), generator=_gen(3), device="cuda")
    model(tokens, mask=AttentionMask(doc_ids=_docs(2, 300, 90))).float().logsumexp(-1).mean().backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in model.parameters())
    assert any(bool(p.grad.any()) for p in model.layers[0].attn.parameters())
    model.eval()
    with torch.no_grad():
        whole = model(tokens)
        with torch.device("cuda"):
            model.setup_caches(2, torch.bfloat16, decoder_max_seq_len=320)
        causal = torch.ones(320, 320, dtype=torch.bool, device="cuda").tril().expand(2, 320, 320)
        steps = [model(tokens[:, a:z], input_pos=torch.arange(a, z, device="cuda").expand(2, -1), mask=causal[:, a:z]) for a, z in ((0, 290), (290, 291), (291, 300))]
    steps = torch.cat(steps, 1)
    assert (steps.float() - whole.float()).norm() <= 2.0**-5 * whole.float().norm()  # bf16 activations of two layers, rounded at other places
    for layer in model.layers:
        layer.attn.kv_cache, layer.attn.cache_enabled = None, False
    with torch.device("cuda"):
        model.setup_caches(2, torch.bfloat16, decoder_max_seq_len=320, kv_cache_bits=4)
    out, _ = generation.generate(model, tokens[:, :200], max_generated_tokens=10, pad_id=0, top_k=1)
    assert out.shape == (2, 210)


def test_no_queries_and_what_does_not_fit():
    mask = AttentionMask(window=4, sinks=1)
    k = _randn(2, 5, 2, 64, seed=1).requires_grad_()
    q = k[:, :0].detach().requires_grad_()
    out = ops.attention(q, k, k, mask)
    assert out.shape == (2, 0, 2, 64)
    assert not torch.autograd.grad(out.sum(), k)[0].any()
    x = _randn(2, 9, 2, 64, seed=2)
    for q, k, v, m in ((x, x[:1], x[:1], mask), (x, x, x[:, :8], mask), (x, x.float(), x, mask), (x, x[..., :32], x[..., :32], mask), (x, x, x, AttentionMask(window=4, sinks=1, doc_ids=_docs(2, 8, 3)))):
        with pytest.raises(ValueError):
            ops.attention(q, k, v, m)
    one = _docs(1, 9, 3)
    assert torch.equal(ops.attention(x, x, x, AttentionMask(window=4, sinks=1, doc_ids=one)), ops.attention(x, x, x, AttentionMask(window=4, sinks=1, doc_ids=one.expand(2, 9))))
    y = x.clone().requires_grad_()
    (grad,) = torch.autograd.grad(ops.attention(y, y, y, mask).float().square().sum(), y, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.float().sum().backward()


def test_saved_tensors_are_asked_for_once():
    """What activation checkpointing allows and offloading pays for."""
    from torchtune_b200.models.mistral import mistral
    from torchtune_b200.modules import TransformerSelfAttentionLayer
    from torchtune_b200.training.memory import set_activation_checkpointing

    unpacked = []

    def unpack(packed):
        unpacked.append(packed[0])
        return packed[1]

    numbers = iter(range(1000))
    q, k, v, d_o = (_randn(1, 90, h, 64, seed=i) for i, h in ((1, 4), (2, 2), (3, 2), (4, 4)))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (next(numbers), t), unpack):
        out = ops.attention(*leaves, AttentionMask(window=20, sinks=2, doc_ids=_docs(1, 90, 30)))
    torch.autograd.grad(out, leaves, d_o)
    assert unpacked and len(set(unpacked)) == len(unpacked)

    grads = []
    tokens = torch.randint(1, 304, (2, 300), generator=_gen(3), device="cuda")
    for recomputed in (False, True):
        torch.manual_seed(2)
        with torch.device("cuda"):
            model = mistral(vocab_size=304, num_layers=2, num_heads=4, num_kv_heads=2, embed_dim=256, intermediate_dim=256, max_seq_len=512, sliding_window_size=40, attention_sinks=3).to(torch.bfloat16)
        if recomputed:
            set_activation_checkpointing(model, {TransformerSelfAttentionLayer})
        for mask in (None, AttentionMask(doc_ids=_docs(2, 300, 90))):
            model(tokens, mask=mask).float().logsumexp(-1).mean().backward()
        grads.append([p.grad for p in model.parameters()])
    # the recomputed forward is the same bit for bit; dQ is summed by atomics, and where another order tips its rounding an element moves by 2^-8 of itself
    for a, b in zip(*grads):
        assert (a.float() - b.float()).norm() <= 2.0**-6 * a.float().norm()


def test_attention_over_key_ranges_does_not_drop_first_tokens(monkeypatch):
    """Latent and span attention take one range of keys per query: a window with first tokens beside it is refused, or computed by the statement."""
    from torchtune_b200.modules import Linear, SpanAttention
    from torchtune_b200.ops import KernelFallbackError

    torch.manual_seed(1)
    with torch.device("cuda"):
        attn = SpanAttention(embed_dim=128, num_heads=4, num_kv_heads=2, key_dim=32, value_dim=32, scale=0.2, **{f"{n}_proj": Linear(128, w, bias=False) for n, w in (("q", 128), ("k", 64), ("v", 64), ("output", 128))})
    attn = attn.to(torch.bfloat16)
    x = _randn(2, 60, 128, seed=1)
    for docs in (None, _docs(2, 60, 20)):
        mask = AttentionMask(window=5, sinks=2, doc_ids=docs)
        with torch.no_grad():
            with pytest.raises(KernelFallbackError):
                attn(x, mask=mask)
            with monkeypatch.context() as m:
                m.setenv("TTB_STRICT", "0")
                m.setattr(ops, "fallback_counts", {})
                with pytest.warns(RuntimeWarning):
                    got = attn(x, mask=mask)
            with ops.use_reference_ops():
                want = attn(x, mask=_visible(60, 60, 5, 2, docs).expand(2, 60, 60))
        # bf16 projections by two GEMMs and an attention that are rounded alike but for the order of fp32 sums
        assert (got.float() - want.float()).norm() <= 2.0**-6 * want.float().norm()


def test_windows_over_other_numbers_of_keys_can_do_what_the_statement_can(monkeypatch):
    """Second derivatives, transforms of functions, mixed types and broadcasts of a window without first tokens: all of them the statement's."""
    monkeypatch.setattr(ops, "fallback_counts", {})
    base = _randn(2, 20, 2, 72, seed=2)
    q, k, v, d_o = _randn(2, 6, 4, 64, seed=1), base[..., 3:67], base[..., 8:], _randn(2, 6, 4, 64, seed=4)  # strided keys, values at an odd address
    mask = AttentionMask(window=5)

    def twice():
        leaves = [t.clone(memory_format=torch.preserve_format).requires_grad_() for t in (q, k, v)]
        parts = [leaves[0], leaves[1].expand(2, -1, -1, -1), leaves[2].transpose(1, 2).contiguous().transpose(1, 2)]
        first = torch.autograd.grad(ops.attention(*parts, mask), leaves, d_o, create_graph=True)
        return [*first, *torch.autograd.grad(sum(t.float().square().sum() for t in first), leaves)]

    def some():  # not all of them have gradients
        x = k.clone().requires_grad_()
        (first,) = torch.autograd.grad(ops.attention(q, x, v, mask), x, d_o, create_graph=True)
        return torch.autograd.grad(first.float().square().sum(), x)

    def tied():  # the same tensor as keys and values, and queries made of it
        x = k.clone().requires_grad_()
        (first,) = torch.autograd.grad(ops.attention(torch.cat([x, -x], 2)[:, :6] * 0.5, x, x, mask), x, d_o, create_graph=True)
        return [first, *torch.autograd.grad(first.float().square().sum(), x)]

    calls = [
        twice,
        some,
        tied,
        lambda: [torch.func.vmap(lambda t: ops.attention(t, k, v, mask))(torch.stack([q, -q]))],
        lambda: [torch.func.grad(lambda t: ops.attention(q, t, v, mask).float().square().sum())(k)],
        lambda: list(torch.func.jvp(lambda t: ops.attention(q, k, t, mask), (v,), (v,))),
        lambda: [ops.attention(q, k.float(), v, mask)],
        lambda: [ops.attention(q, k[:1], v[:1], mask), ops.attention(q, k, v[:, :, :1], mask)],
        lambda: [ops.attention(q[:1, :1].expand(65536, 1, 4, 64), k[:1, :2].expand(65536, 2, 2, 64), v[:1, :2].expand(65536, 2, 2, 64), mask)],
    ]
    for call in calls:
        with pytest.raises(ops.KernelFallbackError):
            call()
        with monkeypatch.context() as m:
            m.setenv("TTB_STRICT", "0")
            with warnings.catch_warnings():
                warnings.simplefilter("ignore")
                got = call()
        with ops.use_reference_ops():
            want = call()
        for a, w in zip(got, want, strict=True):
            assert a.dtype == w.dtype and torch.equal(a, w)
    # one backward pass, whose gradients nobody differentiates, is the kernels'
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    torch.autograd.grad(ops.attention(*leaves, mask), leaves, d_o)


def test_more_rows_and_key_heads_than_a_grid_dimension_has():
    """Gradients of first positions that meet in a workspace, of 65 536 pairs of a batch row and a key head."""
    b, s, h = 1024, 129, 64
    q, k, v, d_o = (_randn(b, s, h, 64, seed=i) for i in range(4))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    mask = AttentionMask(window=1, sinks=1)
    out = ops.attention(*leaves, mask)
    grads = torch.autograd.grad(out, leaves, d_o)
    at = [0, 511, 1023]
    for got in (out, *grads):
        assert got.isfinite().all()
    parts = [t.detach()[at] for t in leaves]
    want, square, *wants = _formula(*parts, d_o[at], _visible(s, s, 1, 1), 64**-0.5)
    _near(out[at], want, square)
    _check_gradients([g[at] for g in grads], wants, d_o[at], want, 64**-0.5)


@pytest.mark.parametrize("bits", [None, 4, 8])
def test_cached_steps_of_a_windowed_decoder_see_the_window(bits):
    """Prompt and single tokens of left-padded rows: what the windowed model does by itself, the same weights without a window do under a mask of the window."""
    from torchtune_b200.models.mistral import mistral

    arch = dict(vocab_size=304, num_layers=2, num_heads=4, num_kv_heads=2, embed_dim=256, intermediate_dim=256, max_seq_len=256)
    models = []
    for kwargs in (dict(sliding_window_size=30, attention_sinks=3), {}):
        torch.manual_seed(2)
        with torch.device("cuda"):
            model = mistral(**arch, **kwargs).to(torch.bfloat16).eval()
            model.setup_caches(2, torch.bfloat16, decoder_max_seq_len=140, kv_cache_bits=bits)
        models.append(model)
    tokens = torch.randint(1, 304, (2, 130), generator=_gen(3), device="cuda")
    start = torch.tensor([0, 21], device="cuda")[:, None, None]
    i, j = torch.arange(130, device="cuda")[:, None], torch.arange(140, device="cuda")
    causal = (j <= i) & ((j >= start) | (i == j))
    window = causal & ((i - j < 30) | (j - start < 3))
    with torch.no_grad():
        for a, z in ((0, 120), (120, 121), (121, 129), (129, 130)):
            pos = torch.arange(a, z, device="cuda").expand(2, -1)
            own, given = (m(tokens[:, a:z], input_pos=pos, mask=mask[:, a:z]) for m, mask in zip(models, (causal, window)))
            assert torch.equal(own, given)
        # and the window counts
        pos = torch.full((2, 1), 130, device="cuda")
        last = (torch.arange(140, device="cuda") <= 130)[None, None].expand(2, 1, 140) & (j >= start)
        own, all_keys = (m(tokens[:, :1], input_pos=pos, mask=last) for m in models)
        assert not torch.equal(own, all_keys)
