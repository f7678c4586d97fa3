"""A key/value cache in 4 or 8 bits: its format, what writing, reading and attending refuse, and a cached decoder, all on plain statements."""
import pytest
import torch

from torchtune_b200 import ops
from torchtune_b200.ops import QuantizedRows, reference
from torchtune_b200.ops.mask import AttentionMask


def _rows(b, slots, h, d, bits):
    return QuantizedRows.zeros(b, slots, h, d, bits), QuantizedRows.zeros(b, slots, h, d, bits)


def _value(codes, scales, bits, d, c):
    """Channel ``c`` of one row, from the words of the format."""
    code = int(codes[c]) if bits == 8 else (int(codes[c // 2]) >> (4 * (c % 2))) & 15
    return (code - 2 ** (bits - 1)) * float(scales[(c % (d // 4)) // 8])


@pytest.mark.parametrize("d", [32, 96, 128])
@pytest.mark.parametrize("bits", [4, 8])
def test_a_row_stands_for_its_nearest_codes(bits, d):
    x = torch.randn(2, 3, 2, d, generator=torch.Generator().manual_seed(d)).to(torch.bfloat16)
    k_rows, v_rows = _rows(2, 7, 2, d, bits)
    ops.quantized_append(x, -x, k_rows, v_rows, torch.arange(2, 5))
    k, v = ops.quantized_read(k_rows, v_rows, 2, 5, torch.float32)
    half = 2 ** (bits - 1)
    for b, i, h in ((0, 0, 0), (1, 2, 1)):
        row = x[b, i, h].double()
        for c in range(d):
            assert float(k[b, i, h, c]) == _value(k_rows.codes[b, h, 2 + i], k_rows.scales[b, h, 2 + i], bits, d, c)
        for j in range(d // 32):
            at = [c for c in range(d) if (c % (d // 4)) // 8 == j]
            top = max(at, key=lambda c: (abs(float(row[c])), -c))
            step = float(row[top]) / -half  # exact for bf16
            assert float(k_rows.scales[b, h, 2 + i, j]) == step
            for c in at:
                error = abs(float(k[b, i, h, c]) - float(row[c]))
                # the nearest code, but for +h, which does not exist
                assert error <= abs(step) / 2 or (float(row[c]) / step > half - 1 and float(k[b, i, h, c]) == (half - 1) * step)
    # the opposite values have opposite scales and the same codes
    assert torch.equal(k_rows.codes, v_rows.codes) and torch.equal(k_rows.scales, -v_rows.scales) and torch.equal(k, -v)
    untouched = [0, 1, 5, 6]
    assert not k_rows.codes[:, :, untouched].any() and not k_rows.scales[:, :, untouched].any()


@pytest.mark.parametrize("bits", [4, 8])
def test_groups_of_zeros_ties_and_non_finite_values(bits):
    x = torch.randn(1, 5, 1, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    group = [c for c in range(64) if (c % 16) // 8 == 1]
    x[0, 0, 0, group] = 0.0
    x[0, 1, 0, group] = torch.linspace(-1, 1, 32).to(torch.bfloat16)  # -1 and 1 are equally large: the first counts
    x[0, 2, 0, group[3]] = float("inf")
    x[0, 3, 0, group[3]] = float("nan")
    x[0, 4, 0, group] = 1e-40  # its scale underflows or is coarse: nothing turns into NaN
    k_rows, v_rows = _rows(1, 5, 1, 64, bits)
    ops.quantized_append(x, x, k_rows, v_rows, torch.arange(5))
    k, _ = ops.quantized_read(k_rows, v_rows, dtype=torch.float32)
    others = [c for c in range(64) if c not in group]
    assert not k[0, 0, 0, group].any()
    assert float(k[0, 1, 0, group[0]]) == -1.0 and float(k_rows.scales[0, 0, 1, 1]) == 1.0 / 2 ** (bits - 1)
    assert float(k[0, 1, 0, group[-1]]) == 1.0 - 1.0 / 2 ** (bits - 1)
    assert k[0, 2, 0, group].isnan().all() and k[0, 3, 0, group].isnan().all()
    assert k[0, :, 0, others].isfinite().all() and k[0, 4].isfinite().all()


def test_rows_are_views_with_their_own_sizes():
    rows = QuantizedRows.zeros(3, 13, 2, 64, 4)
    assert rows.codes.shape == (3, 2, 16, 32) and rows.scales.shape == (3, 2, 16, 2) and rows.bits == 4 and rows.head_dim == 64 and rows.slots == 13
    part = rows.batch(2).first(5)
    assert part.codes.shape[0] == 2 and part.slots == 5 and part.codes.data_ptr() == rows.codes.data_ptr()
    for slots in (-1, 6):
        with pytest.raises(ValueError):
            part.first(slots)
    assert QuantizedRows.zeros(1, 3, 1, 32, 8).bits == 8
    with pytest.raises(ValueError):
        ops.quantized_read(rows, rows.first(3))
    with pytest.raises(ValueError):
        ops.quantized_read(*(QuantizedRows(rows.codes, rows.scales, 17) for _ in "kv"))
    for bits, d in ((2, 64), (4, 48), (8, 0)):
        with pytest.raises(ValueError):
            QuantizedRows.zeros(1, 4, 1, d, bits)


def test_writing_refuses_what_does_not_fit():
    k_rows, v_rows = _rows(2, 8, 2, 64, 4)
    x = torch.zeros(2, 3, 2, 64)
    at = torch.arange(3)
    for slots in (torch.arange(6, 9), torch.tensor([-1, 0, 1]), torch.tensor([1, 1, 1]), torch.tensor([0, 2, 4]), torch.arange(2), torch.arange(3, dtype=torch.int32)):
        with pytest.raises(ValueError):
            ops.quantized_append(x, x, k_rows, v_rows, slots)
    assert not k_rows.codes.any()
    for k, v in ((x[:1], x[:1]), (x[..., :32], x[..., :32]), (x[:, :, :1], x[:, :, :1]), (x, x[:, :2]), (x, x.half()), (x.int(), x.int()), (x.double(), x.double())):
        with pytest.raises(ValueError):
            ops.quantized_append(k, v, k_rows, v_rows, at)
    with pytest.raises(ValueError):
        ops.quantized_append(x, x, k_rows, QuantizedRows.zeros(2, 8, 2, 64, 8), at)
    with pytest.raises(ValueError):
        ops.quantized_append(x, x, k_rows, QuantizedRows(v_rows.codes, v_rows.scales.float()), at)
    ops.quantized_append(x[:, :0], x[:, :0], k_rows, v_rows, at[:0])
    for start, stop in ((-1, 2), (3, 2), (0, 9)):
        with pytest.raises(ValueError):
            ops.quantized_read(k_rows, v_rows, start, stop)
    with pytest.raises(ValueError):
        ops.quantized_read(k_rows, v_rows, dtype=torch.int32)
    assert ops.quantized_read(k_rows, v_rows, 4, 4)[0].shape == (2, 0, 2, 64)


def _filled(b, n, h, d, bits, seed=0):
    g = torch.Generator().manual_seed(seed)
    k_rows, v_rows = _rows(b, n, h, d, bits)
    ops.quantized_append(torch.randn(b, n, h, d, generator=g), torch.randn(b, n, h, d, generator=g), k_rows, v_rows, torch.arange(n))
    return k_rows, v_rows


def test_attention_refuses_what_does_not_fit():
    k_rows, v_rows = _filled(2, 8, 2, 64, 4)
    q = torch.randn(2, 3, 4, 64)
    for x in (q[:1], q[..., :32], q[:, :, :3], q[0]):
        with pytest.raises(ValueError):
            ops.quantized_attention(x, k_rows, v_rows)
    masks = [AttentionMask(causal=False, window=4), AttentionMask(doc_ids=torch.zeros(2, 8, dtype=torch.int32)), AttentionMask(chunk=4), AttentionMask(bool_mask=torch.ones(2, 3, 7, dtype=torch.bool)),
             AttentionMask(bool_mask=torch.ones(2, 4, 3, 8, dtype=torch.bool)), AttentionMask(key_start=torch.zeros(2, dtype=torch.int32), query_start=6),
             AttentionMask(key_start=torch.zeros(3, dtype=torch.int32)), AttentionMask(key_start=torch.zeros(2, dtype=torch.int32), window=3)]
    for mask in masks:
        with pytest.raises(ValueError):
            ops.quantized_attention(q, k_rows, v_rows, mask)
    with pytest.raises(ValueError):
        ops.quantized_attention(torch.randn(2, 9, 4, 64), k_rows, v_rows, AttentionMask())
    assert not ops.quantized_attention(q, k_rows.first(0), v_rows.first(0)).any()
    assert ops.quantized_attention(q[:, :0], k_rows, v_rows).shape == (2, 0, 4, 64)


@pytest.mark.parametrize("mask", [AttentionMask(causal=False), AttentionMask(), AttentionMask(window=3, sinks=2), AttentionMask(window=1), "bool", "start"])
def test_attention_is_that_of_the_values_the_cache_stands_for(mask):
    k_rows, v_rows = _filled(2, 11, 2, 64, 8)
    q = torch.randn(2, 2, 6, 64, generator=torch.Generator().manual_seed(3))
    i, j = torch.arange(2)[:, None] + 9, torch.arange(11)[None, :]
    if mask == "bool":
        dense = torch.rand(2, 2, 11, generator=torch.Generator().manual_seed(4)) < 0.5
        dense[1, 0] = False  # a query that sees nothing
        mask = AttentionMask(causal=False, bool_mask=dense)
    elif mask == "start":
        mask = AttentionMask(key_start=torch.tensor([0, 4], dtype=torch.int32), query_start=5)
        dense = (j <= i - 4) & (j >= torch.tensor([0, 4])[:, None, None])
    else:
        dense = torch.ones(2, 2, 11, dtype=torch.bool)
        if mask.causal:
            dense = dense & (j <= i)
        if mask.window:
            dense = dense & ((i - j < mask.window) | (j < mask.sinks))
    got = ops.quantized_attention(q, k_rows, v_rows, mask, scale=0.3)
    k, v = (t.double() for t in ops.quantized_read(k_rows, v_rows, dtype=torch.float32))
    score = torch.einsum("bqgnd,bkgd->bgnqk", q.double().view(2, 2, 2, 3, 64), k) * 0.3
    p = torch.softmax(score.masked_fill(~dense[:, None, None], float("-inf")), -1).nan_to_num()
    want = torch.einsum("bgnqk,bkgd->bqgnd", p, v).reshape(2, 2, 6, 64)
    # fp32 sums of at most 64 products of size 10 and 11 terms: 2^-24 x 100
    assert (got.double() - want).abs().max() <= 1e-5


def test_gradients_reach_the_queries():
    k_rows, v_rows = _filled(1, 5, 1, 32, 8)
    q = torch.randn(1, 2, 2, 32, generator=torch.Generator().manual_seed(5), dtype=torch.float64).float().requires_grad_()
    out = ops.quantized_attention(q, k_rows, v_rows, AttentionMask())
    (grad,) = torch.autograd.grad(out.sum(), q)
    k, v = ops.quantized_read(k_rows, v_rows, dtype=torch.float32)
    (want,) = torch.autograd.grad(reference.attention(q, k, v, causal=True).sum(), q)
    assert torch.equal(grad, want)


# ------------------------------------------------------------------------------------------------------------------------- decoders


def _decoder(**kwargs):
    from torchtune_b200.models.llama2 import llama2

    torch.manual_seed(7)
    return llama2(**{**dict(vocab_size=50, num_layers=2, num_heads=4, num_kv_heads=2, embed_dim=128, max_seq_len=64, intermediate_dim=64), **kwargs}).eval()


class _RoundTrip(torch.nn.Module):
    """Stands for quantised values in an ordinary cache: rounds what it is given as the format does."""

    def __init__(self, cache, bits):
        super().__init__()
        self.cache, self.bits = cache, bits

    def __getattr__(self, name):
        return super().__getattr__(name) if name in ("cache", "bits") else getattr(self.cache, name)

    def update(self, k, v):
        return self.cache.update(*(reference.dequantize_rows(*reference.quantize_rows(t, self.bits), torch.float32) for t in (k, v)))


@pytest.mark.parametrize("bits", [4, 8])
def test_a_decoder_sees_what_its_quantised_caches_stand_for(bits):
    from torchtune_b200.modules import QuantizedKVCache

    model, plain = _decoder(), _decoder()
    model.setup_caches(2, torch.float32, decoder_max_seq_len=20, kv_cache_bits=bits)
    plain.setup_caches(2, torch.float32, decoder_max_seq_len=20)
    for layer in plain.layers:
        layer.attn.kv_cache = _RoundTrip(layer.attn.kv_cache, bits)
    cache = model.layers[0].attn.kv_cache
    assert type(cache) is QuantizedKVCache and cache.bits == bits and cache.k_codes.dtype == torch.uint8 and not any("codes" in k for k in model.state_dict())
    tokens = torch.randint(0, 50, (2, 9), generator=torch.Generator().manual_seed(1))
    mask = torch.tril(torch.ones(9, 20, dtype=torch.bool)).expand(2, 9, 20)
    with torch.no_grad():
        for a, z in ((0, 6), (6, 7), (7, 9)):
            pos = torch.arange(a, z).expand(2, -1)
            got, want = (m(tokens[:, a:z], input_pos=pos, mask=mask[:, a:z]) for m in (model, plain))
            # both fp32; sums of up to 128 products in another order, two layers: a thousand roundings of 2^-24
            assert (got - want).abs().max() <= 1e-4 * want.abs().max()
        assert cache.size == 9
        before = got
        model.reset_caches()
        assert cache.size == 0 and not cache.k_codes.any()
        for a, z in ((0, 6), (6, 9)):
            got = model(tokens[:, a:z], input_pos=torch.arange(a, z).expand(2, -1), mask=mask[:, a:z])
        assert (got[:, -2:] - before).abs().max() <= 1e-4 * before.abs().max()
        one = model.layers[0].attn.kv_cache
        with pytest.raises(AssertionError):
            one.append(torch.zeros(2, 12, 2, 32), torch.zeros(2, 12, 2, 32))
        with pytest.raises(ValueError):
            one.append(torch.zeros(3, 1, 2, 32), torch.zeros(3, 1, 2, 32))
        k, v = one.update(torch.ones(1, 1, 2, 32), torch.ones(1, 1, 2, 32))
        assert k.shape == (1, 20, 2, 32) and k.dtype == torch.float32 and torch.equal(k[:, 9], torch.ones(1, 2, 32))


def test_caches_in_few_bits_are_refused_where_they_do_not_apply():
    with pytest.raises(ValueError):
        _decoder().setup_caches(1, torch.float32, decoder_max_seq_len=8, kv_cache_bits=3)
    with pytest.raises(ValueError):
        _decoder(num_heads=8).setup_caches(1, torch.float32, decoder_max_seq_len=8, kv_cache_bits=4)  # 16 channels per head
    from torchtune_b200.models.llama3_2_vision import llama3_2_vision_decoder

    fused = llama3_2_vision_decoder(vocab_size=50, num_layers=2, fusion_interval=2, num_special_tokens=2, num_heads=2, num_kv_heads=2, embed_dim=64, max_seq_len=16, encoder_max_seq_len=4,
                                    intermediate_dim=32)
    with pytest.raises(ValueError):
        fused.setup_caches(1, torch.float32, encoder_max_seq_len=4, decoder_max_seq_len=8, kv_cache_bits=4)


def test_generation_on_quantised_caches():
    from torchtune_b200 import generation
    from torchtune_b200.modules import delete_kv_caches, local_kv_cache

    model = _decoder()
    prompt = torch.tensor([[0, 0, 5, 6, 7], [3, 4, 5, 6, 7]])
    with local_kv_cache(model, batch_size=2, device=torch.device("cpu"), dtype=torch.float32, decoder_max_seq_len=16, kv_cache_bits=8):
        tokens, logits = generation.generate(model, prompt, max_generated_tokens=6, pad_id=0, top_k=1)
    assert tokens.shape == (2, 11) and logits.isfinite().all()
    model.setup_caches(2, torch.float32, decoder_max_seq_len=16)
    plain, _ = generation.generate(model, prompt, max_generated_tokens=1, pad_id=0, top_k=1)
    assert torch.equal(tokens[:, 5], plain[:, 5])  # logits of random weights lie further apart than 8 bits move them
    delete_kv_caches(model)


def test_generate_recipe_with_a_quantised_cache(tmp_path, tune_path, monkeypatch, caplog):
    from helpers import run_tune, write_tiny_hf_checkpoint
    from tokenizer_assets import write_sentencepiece_model
    from torchtune_b200.models.llama2 import llama2

    arch = dict(vocab_size=200, num_layers=1, num_heads=2, num_kv_heads=1, embed_dim=64, max_seq_len=128, intermediate_dim=64, norm_eps=1e-5)
    write_tiny_hf_checkpoint(tmp_path / "ckpt", arch=arch, builder=llama2)
    (tmp_path / "tok").mkdir()
    sp = write_sentencepiece_model(tmp_path / "tok", vocab_size=200)
    model = " ".join(f"model.{k}={v}" for k, v in arch.items())
    run_tune(tune_path, f"run generate --config generation model._component_=torchtune_b200.models.llama2.llama2 {model} checkpointer.checkpoint_dir={tmp_path / 'ckpt'} "
             f"checkpointer.checkpoint_files=[model-00001-of-00001.safetensors] device=cpu dtype=fp32 output_dir={tmp_path / 'out'} tokenizer.path={sp} max_new_tokens=6 prompt.user=hello "
             "kv_cache_bits=4", monkeypatch)
    assert "tokens/sec" in caplog.text


def test_a_cache_keeps_its_types_when_a_model_changes_its_own():
    model = _decoder()
    model.setup_caches(1, torch.float32, decoder_max_seq_len=8, kv_cache_bits=4)
    cache = model.layers[0].attn.kv_cache
    cache.append(torch.randn(1, 3, 2, 32), torch.randn(1, 3, 2, 32))
    scales = cache.k_scales.clone()
    model.to(torch.bfloat16).float()
    assert cache.k_scales.dtype == torch.bfloat16 and torch.equal(cache.k_scales, scales) and cache.k_codes.dtype == torch.uint8 and cache.cache_pos.dtype == torch.int64


@pytest.mark.parametrize("bits", [4, 8])
def test_scales_do_not_pass_through_a_models_new_type(bits):
    """Scales below the smallest number of fp16 and above its largest."""
    model = _decoder()
    model.setup_caches(1, torch.float32, decoder_max_seq_len=8, kv_cache_bits=bits)
    cache = model.layers[1].attn.kv_cache
    x = torch.randn(1, 6, 2, 32, generator=torch.Generator().manual_seed(1)) * torch.tensor([1e-30, 1e-6, 1e-3, 1.0, 1e8, 1e30])[:, None, None]
    cache.append(x, -x)
    want = [t.clone() for t in (cache.k_scales, cache.v_scales, cache.k_codes, cache.v_codes)]
    for convert in (torch.nn.Module.half, torch.nn.Module.double, lambda m: m.to("cpu", torch.float16), lambda m: m.to(torch.bfloat16), torch.nn.Module.float):
        convert(model)
        assert all(torch.equal(a, b) for a, b in zip(want, (cache.k_scales, cache.v_scales, cache.k_codes, cache.v_codes)))
        assert cache.k_scales.dtype == cache.v_scales.dtype == torch.bfloat16 and dict(cache.named_buffers())["k_scales"] is cache.k_scales
    meta = _decoder()
    meta.setup_caches(1, torch.float32, decoder_max_seq_len=8, kv_cache_bits=bits)
    meta.to("meta").half()
    assert meta.layers[0].attn.kv_cache.k_scales.dtype == torch.bfloat16 and meta.layers[0].attn.kv_cache.k_scales.device.type == "meta"
    meta.to_empty(device="cpu")
    assert meta.layers[0].attn.kv_cache.k_scales.dtype == torch.bfloat16 and meta.layers[0].attn.kv_cache.k_scales.device.type == "cpu"


def test_a_cache_whose_buffers_were_exchanged_takes_as_many_rows_as_they_have():
    from torchtune_b200.modules import KVCache, QuantizedKVCache

    plain = KVCache(2, 8, 1, 32, torch.float32)
    plain.k_cache, plain.v_cache = torch.zeros(3, 8, 1, 32), torch.zeros(3, 8, 1, 32)
    x = torch.randn(3, 2, 1, 32, generator=torch.Generator().manual_seed(1))
    assert torch.equal(plain.update(x, -x)[0][:, :2], x)
    few = QuantizedKVCache(2, 8, 1, 32, 8)
    for name, t in QuantizedKVCache(3, 8, 1, 32, 8).named_buffers():
        setattr(few, name, t)
    assert few.update(x, -x)[0].shape == (3, 8, 1, 32)
    for cache in (plain, few):
        with pytest.raises(ValueError, match="batch size of 3"):
            cache.update(x.repeat(2, 1, 1, 1), x.repeat(2, 1, 1, 1))
