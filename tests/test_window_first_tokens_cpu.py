"""Masks of a sliding window beside which the first tokens stay visible: their dense form, the plain statement's gradients, models that use them."""
import pytest
import torch

from torchtune_b200 import ops
from torchtune_b200.ops import reference
from torchtune_b200.ops.mask import AttentionMask


def _visible(sq, sk, window, sinks, docs=None):
    """By the words of the definition, pair by pair."""
    b = 1 if docs is None else docs.shape[0]
    m = torch.zeros(b, sq, sk, dtype=torch.bool)
    for r in range(b):
        for i in range(sq):
            at = i + sk - sq
            for j in range(at + 1):
                first = 0
                if docs is not None:
                    if docs[r, at] != docs[r, j]:
                        continue
                    first = int((docs[r] == docs[r, at]).nonzero()[0])
                m[r, i, j] = at - j < window or j - first < sinks
    return m


DOCS = torch.tensor([[0] * 5 + [1] * 1 + [2] * 9, [4] * 15], dtype=torch.int32)


@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (3, 2), (4, 20), (20, 3)])
def test_dense_masks(window, sinks):
    mask = AttentionMask(window=window, sinks=sinks)
    assert torch.equal(mask.dense(1, 15, 15, "cpu"), _visible(15, 15, window, sinks))
    packed = AttentionMask(window=window, sinks=sinks, doc_ids=DOCS)
    assert torch.equal(packed.dense(2, 15, 15, "cpu"), _visible(15, 15, window, sinks, DOCS))
    assert torch.equal(packed.to("cpu").dense(2, 15, 15, "cpu"), packed.dense(2, 15, 15, "cpu"))
    assert torch.equal(AttentionMask(window=window).dense(1, 9, 9, "cpu"), _visible(9, 9, window, 0))


@pytest.mark.parametrize("sq", [1, 4, 11])
@pytest.mark.parametrize("docs", [False, True])
def test_plain_attention_and_its_gradients(sq, docs):
    if docs and sq < 11:
        return  # documents go with whole sequences
    g = torch.Generator().manual_seed(sq)
    ids = torch.tensor([[0] * 4 + [1] * 7], dtype=torch.int32) if docs else None
    q, k, v, d_o, u = (torch.randn(1, n, h, 8, generator=g, dtype=torch.float64) for n, h in ((sq, 4), (11, 2), (11, 2), (sq, 4), (sq, 4)))
    mask = AttentionMask(window=3, sinks=2, doc_ids=ids)
    seen = _visible(sq, 11, 3, 2, ids)

    def formula(q, k, v):
        score = torch.einsum("bqgnd,bkgd->bgnqk", q.view(1, sq, 2, 2, 8), k) * 8**-0.5
        return torch.einsum("bgnqk,bkgd->bqgnd", torch.softmax(score.masked_fill(~seen[:, None, None], float("-inf")), -1), v).reshape(1, sq, 4, 8)

    leaves = [t.float().requires_grad_() for t in (q, k, v)]
    out = ops.attention(*leaves, mask)
    wide = [t.requires_grad_() for t in (q, k, v)]
    want = formula(*wide)
    assert (out.double() - want).abs().max() <= 1e-5  # fp32 sums of at most 11 terms of size 10
    grads, wants = torch.autograd.grad(out, leaves, d_o.float()), torch.autograd.grad(want, wide, d_o)
    for a, w in zip(grads, wants):
        assert (a.double() - w).abs().max() <= 1e-4
    step = 1e-5
    with torch.no_grad():
        slope = ((formula(q + step * u, k, v) - formula(q - step * u, k, v)) * d_o).sum() / (2 * step)
    assert abs(float((grads[0].double() * u).sum() - slope)) <= 1e-4


def test_a_decoder_with_windows_and_first_tokens():
    """Whole sequences by the structured mask and cached steps by boolean ones see the same tokens."""
    from torchtune_b200.models.mistral import mistral

    arch = dict(vocab_size=60, num_layers=2, num_heads=4, num_kv_heads=2, embed_dim=64, intermediate_dim=64, max_seq_len=64)
    torch.manual_seed(5)
    model = mistral(**arch, sliding_window_size=6, attention_sinks=2).eval()
    torch.manual_seed(5)
    full = mistral(**arch).eval()
    tokens = torch.randint(0, 60, (2, 20), generator=torch.Generator().manual_seed(1))
    with torch.no_grad():
        want = model(tokens)
        assert not torch.allclose(want, full(tokens))
        dense = _visible(20, 20, 6, 2).expand(2, 20, 20)
        assert (full(tokens, mask=dense) - want).abs().max() <= 1e-4
        docs = torch.tensor([[0] * 8 + [1] * 12, [0] * 20], dtype=torch.int32)
        packed = model(tokens, mask=AttentionMask(doc_ids=docs))
        assert (full(tokens, mask=_visible(20, 20, 6, 2, docs)) - packed).abs().max() <= 1e-4
        model.setup_caches(2, torch.float32, decoder_max_seq_len=24)
        causal = torch.ones(24, 24, dtype=torch.bool).tril().expand(2, 24, 24)
        got = [model(tokens[:, a:z], input_pos=torch.arange(a, z).expand(2, -1), mask=causal[:, a:z]) for a, z in ((0, 11), (11, 12), (12, 20))]
        assert (torch.cat(got, 1) - want).abs().max() <= 1e-4
    with pytest.raises(ValueError):
        mistral(**arch, attention_sinks=2)


def test_windows_over_a_quantised_cache_and_left_padded_rows():
    from torchtune_b200 import generation
    from torchtune_b200.models.mistral import mistral

    torch.manual_seed(6)
    model = mistral(vocab_size=60, num_layers=2, num_heads=4, num_kv_heads=2, embed_dim=128, intermediate_dim=64, max_seq_len=64, sliding_window_size=5, attention_sinks=2).eval()
    prompt = torch.randint(1, 60, (1, 9), generator=torch.Generator().manual_seed(2))
    padded = torch.cat([torch.zeros(1, 4, dtype=torch.long), prompt], 1)
    both = torch.cat([padded, torch.randint(1, 60, (1, 13), generator=torch.Generator().manual_seed(3))])
    results = []
    for p, n in ((prompt, 1), (both, 2)):
        model.setup_caches(n, torch.float32, decoder_max_seq_len=24, kv_cache_bits=8)
        results.append(generation.generate(model, p, max_generated_tokens=8, pad_id=0, top_k=1)[1][0])
        for layer in model.layers:
            layer.attn.kv_cache, layer.attn.cache_enabled = None, False
    # padding changes neither positions nor what is seen: the same sums in another order
    assert (results[0] - results[1]).abs().max() <= 1e-3 * results[0].abs().max()


def test_which_calls_are_windows_of_the_kernels():
    from torchtune_b200.ops._cuda_attention import takes_window, unsupported_reason

    q, k = torch.zeros(1, 8, 4, 64), torch.zeros(1, 9, 2, 64)
    ids = torch.zeros(1, 8, dtype=torch.int32)
    takes = lambda q, k, softcap=0.0, **mask: takes_window(q, k, AttentionMask(**mask), softcap)  # noqa: E731
    assert takes(q, q[:, :, :2], window=4, sinks=1) and takes(q, q[:, :, :2], window=4, sinks=1, doc_ids=ids) and takes(q, k, window=4) and takes(q, k, window=4, sinks=2, softcap=None)
    for kind in (dict(window=4), dict(sinks=2), dict(window=4, sinks=2, causal=False), dict(window=4, sinks=2, chunk=4), dict(window=4, sinks=2, bool_mask=torch.ones(1, 8, 8, dtype=torch.bool))):
        assert not takes(q, q[:, :, :2], **kind)
    assert not takes(q, q[:, :, :2], window=4, sinks=2, softcap=30.0) and not takes(q, k, window=4, sinks=2, doc_ids=ids) and not takes(k, q[:, :, :1], window=4, sinks=2)
    assert not takes(q, torch.zeros(1, 8, 3, 64), window=4, sinks=2)
    assert "first tokens" in unsupported_reason(q, q[:, :, :2], AttentionMask(window=4, sinks=2, chunk=4))
    assert unsupported_reason(q, q[:, :, :2], AttentionMask(window=4)) is None  # the general kernels


def test_fields_of_a_mask_keep_their_places():
    dense = torch.ones(1, 2, 2, dtype=torch.bool)
    mask = AttentionMask(False, None, 0, 0, dense, None, 1)
    assert mask.bool_mask is dense and mask.query_start == 1 and mask.sinks == 0


def test_one_range_of_keys_does_not_stand_for_a_window_and_first_tokens():
    from torchtune_b200.modules._spans import make_bounds

    assert make_bounds(AttentionMask(window=4, sinks=2), 2, 15, 0, "cpu") is None
    assert make_bounds(AttentionMask(window=4, sinks=2, doc_ids=DOCS), 2, 15, 0, "cpu") is None
    assert torch.equal(make_bounds(AttentionMask(window=4), 1, 6, 0, "cpu").lo, torch.tensor([[0, 0, 0, 0, 1, 2]], dtype=torch.int32))
    assert make_bounds(AttentionMask(sinks=2), 1, 6, 0, "cpu").lo is None  # first tokens of no window: causal


def test_windows_that_stay_with_the_statement():
    """Transforms, and without first tokens what the statement broadcasts or converts; with them these calls are refused elsewhere."""
    from torchtune_b200.ops._cuda_attention import window_reason

    q, k = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 9, 2, 64, dtype=torch.bfloat16)
    plain, first = AttentionMask(window=4), AttentionMask(window=4, sinks=1)
    assert window_reason(q, k, k, plain) is None and window_reason(q, k, k, first) is None
    for keys, values in ((k.float(), k.float()), (k, k.float()), (k[:1], k[:1]), (k, k[:, :, :1]), (k[..., :32], k[..., :32])):
        assert window_reason(q, keys, values, plain) is not None and window_reason(q, keys, values, first) is None
    reasons = []
    torch.func.vmap(lambda t: reasons.append(window_reason(t, k, k, first)) or t)(q[None])
    torch.func.jvp(lambda t: reasons.append(window_reason(q, t, k, plain)) or t, (k,), (k,))
    with torch.autograd.forward_ad.dual_level():
        reasons.append(window_reason(q, k, k, plain))
    assert len(reasons) == 3 and all(reasons)
    many = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16)
    assert window_reason(many.expand(65536, 1, 1, 64), many.expand(65536, 2, 1, 64), many.expand(65536, 2, 1, 64), plain) is not None


class _Widest(torch.utils._python_dispatch.TorchDispatchMode):
    """Notes the most bytes that a result of an operation has."""

    most = 0

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        for t in out if isinstance(out, (tuple, list)) else (out,):
            if isinstance(t, torch.Tensor):
                self.most = max(self.most, t.numel() * t.element_size())
        return out


@pytest.mark.parametrize("sinks", [0, 3])
def test_dense_masks_are_narrowed_without_wider_copies(sinks):
    from torchtune_b200.models._factory import _window_first_mask_mod

    mod = _window_first_mask_mod(5, sinks)
    causal = torch.ones(40, 64, dtype=torch.bool).tril(11).expand(2, 40, 64)
    with _Widest() as widest:
        got = mod(causal, 2, 40)
    assert widest.most <= causal.numel()
    i, j = torch.arange(40)[:, None] + 11, torch.arange(64)
    want = (j <= i) & ((i - j < 5) | (j < sinks))
    assert torch.equal(got, want.expand(2, 40, 64))
    # left-padded rows, a row that sees itself only, rows without a key, and a mask with a dimension of heads
    start = torch.tensor([7, 0])[:, None, None]
    padded = causal & (j >= start)
    padded[0, 0], padded[1, 5] = False, False
    padded[1, 6] = j == 17
    want = padded & ((i - j < 5) | (j - start < sinks))
    assert torch.equal(mod(padded, 2, 40), want) and torch.equal(mod(padded[:, None], 2, 40), want[:, None])
    assert torch.equal(mod(AttentionMask(causal=False, bool_mask=padded), 2, 40), want)
    assert mod(padded[:, :0], 2, 0).shape == (2, 0, 64)
