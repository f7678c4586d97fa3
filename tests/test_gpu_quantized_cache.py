"""Kernels of a key/value cache in 4 or 8 bits: writing and reading against the plain statement bit for bit, attention against the definition in float64."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from torchtune_b200 import ops
from torchtune_b200.ops import QuantizedRows, reference
from torchtune_b200.ops.mask import AttentionMask


@pytest.fixture(autouse=True)
def _check_device_errors():
    yield
    from torchtune_b200.ops._lib import check_device_errors

    torch.cuda.synchronize()
    check_device_errors()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _zeros(b, slots, h, d, bits):
    return [QuantizedRows.zeros(b, slots, h, d, bits, device="cuda") for _ in range(2)]


def _filled(b, n, h, d, bits, seed=0):
    k_rows, v_rows = _zeros(b, n, h, d, bits)
    g = _gen(seed)
    k, v = (torch.randn(b, n, h, d, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    ops.quantized_append(k * torch.exp(0.3 * torch.randn(h, d, generator=g, device="cuda")).to(torch.bfloat16), v, k_rows, v_rows, torch.arange(n, device="cuda"))
    return k_rows, v_rows


# ------------------------------------------------------------------------------------------------------------------------ writing and reading


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("bits", [4, 8])
def test_written_and_read_as_the_plain_statement_does(bits, d, dtype):
    for b, s, h, at, seed in ((1, 1, 1, 0, 1), (2, 7, 3, 5, 2), (3, 70, 2, 1, 3)):
        x = [(torch.randn(b, s, h, d, generator=_gen(seed + i), device="cuda") * 3).to(dtype) for i in range(2)]
        rows = _zeros(b, at + s + 2, h, d, bits)
        ops.quantized_append(*x, *rows, torch.arange(at, at + s, device="cuda"))
        for part, r in zip(x, rows):
            codes, scales = reference.quantize_rows(part.cpu().transpose(1, 2), bits)
            assert torch.equal(r.codes[:, :, at : at + s].cpu(), codes) and torch.equal(r.scales[:, :, at : at + s].cpu(), scales)
            rest = [i for i in range(at + s + 2) if not at <= i < at + s]
            assert not r.codes[:, :, rest].any() and not r.scales[:, :, rest].any()
        for out in (torch.bfloat16, torch.float32, torch.float16):
            got = ops.quantized_read(*rows, at, at + s, out)
            for y, r in zip(got, rows):
                want = reference.dequantize_rows(r.codes.cpu(), r.scales.cpu(), torch.float32)[:, :, at : at + s].transpose(1, 2).to(out)
                assert y.is_contiguous() and torch.equal(y.cpu(), want)


@pytest.mark.parametrize("bits", [4, 8])
def test_ties_zeros_and_non_finite_values(bits):
    x = torch.randint(-16, 17, (1, 64, 2, 64), generator=_gen(4), device="cuda").to(torch.bfloat16) / 4  # many ties, equal magnitudes of both signs
    x[0, 3, 0] = 0.0
    x[0, 4, 0, 5], x[0, 5, 1, 9], x[0, 6, 0, 7], x[0, 6, 0, 1] = float("inf"), float("nan"), float("-inf"), float("nan")
    x[0, 7] = 1e-40
    x[0, 8, 0, 0] = 3.3e38
    rows = _zeros(1, 64, 2, 64, bits)
    ops.quantized_append(x, -x, *rows, torch.arange(64, device="cuda"))
    got = ops.quantized_read(*rows, dtype=torch.float32)
    for y, part in zip(got, (x, -x)):
        codes, scales = reference.quantize_rows(part.cpu(), bits)
        want = reference.dequantize_rows(codes, scales, torch.float32)
        assert torch.equal(y.cpu().nan_to_num(nan=12345.0), want.nan_to_num(nan=12345.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bits", [4, 8])
def test_strided_keys_and_rows(bits, dtype):
    both = torch.randn(4, 9, 6, 131, generator=_gen(5), device="cuda").to(dtype)
    k, v = both[::2, 1:8, :3, 1:129], both[1::2, 1:8, 3:, 3:131]  # two bytes off a vector's address; every other batch row
    wide = _zeros(5, 20, 6, 128, bits)
    rows = [QuantizedRows(r.codes[1:5:2, ::2], r.scales[1:5:2, ::2]) for r in wide]
    ops.quantized_append(k, v, *rows, torch.arange(20, device="cuda")[4:11])
    for part, r, all_rows in zip((k, v), rows, wide):
        codes, scales = reference.quantize_rows(part.cpu().transpose(1, 2), bits)
        assert torch.equal(r.codes[:, :, 4:11].cpu(), codes) and torch.equal(r.scales[:, :, 4:11].cpu(), scales)
        assert not all_rows.codes[::2].any() and not all_rows.codes[:, 1::2].any() and not all_rows.codes[:, :, :4].any() and not all_rows.codes[:, :, 11:].any()
    got = ops.quantized_read(*rows, 4, 11)
    for y, r in zip(got, rows):
        assert torch.equal(y.cpu(), reference.dequantize_rows(r.codes.cpu(), r.scales.cpu(), torch.bfloat16)[:, :, 4:11].transpose(1, 2))


def test_slots_outside_the_cache_or_out_of_order_are_not_written():
    from torchtune_b200.ops._lib import index_violations

    index_violations()
    x = torch.randn(2, 3, 2, 64, generator=_gen(6), device="cuda").to(torch.bfloat16)
    for slots, written in (([6, 7, 8], [6, 7]), ([-2, -1, 0], [0]), ([2, 2, 2], [2]), ([5, 4, 3], [5]), ([1, 2, 1], [1, 2])):
        rows = _zeros(2, 8, 2, 64, 4)
        ops.quantized_append(x, x, *rows, torch.tensor(slots, device="cuda"))
        held = rows[0].scales.ne(0).any(-1).any(0).any(0).nonzero().flatten().tolist()
        assert held == written
        assert index_violations() == 2 * (3 - len(written))  # once per token and batch row


# ---------------------------------------------------------------------------------------------------------------------------------- attention


def _check(q, k_rows, v_rows, mask, dense, scale=None, spread=False):
    with torch.no_grad():
        got = ops.quantized_attention(q, k_rows, v_rows, mask, scale=scale)
    b, s, hq, d = q.shape
    k, v = (t.double() for t in ops.quantized_read(k_rows, v_rows, dtype=torch.float32))
    k, v = (torch.where(dense.any(1)[:, :, None, None], t, 0.0) for t in (k, v))  # what nobody sees may be anything
    score = torch.einsum("bqgnd,bkgd->bgnqk", q.double().view(b, s, k.shape[2], -1, d), k) * (d**-0.5 if scale is None else scale)
    p = torch.softmax(score.masked_fill(~dense[:, None, None], float("-inf")), -1).nan_to_num()
    want, square = (torch.einsum("bgnqk,bkgd->bqgnd", w, t).reshape(b, s, hq, d) for w, t in ((p, v), (p.square(), v.square())))
    # The result is rounded to 8 bits (at most 2^-9 of it; twice that here); so is every weight times its scale: errors of at most 2^-9 of the terms, without a common sign, so eight times 2^-9 of the
    # terms' root of squares bounds their sum (14 standard deviations).  Scores: fp32 sums whose terms are at most 136 |q| |scale|: at these sizes 1e-4, a twentieth of a weight's rounding.
    bound = 2.0**-8 * want.abs() + 2.0**-6 * square.sqrt()
    if spread:
        # Values of very different sizes: where the largest have the code 0, the small ones are what is left.  The kernel's fp32 sums hold codes (below 2^bits) and take 2^(bits - 1) off, so they pass
        # through numbers of sum p |scale| 2^bits; at most 2^5 steps of a warp and joins, each off by at most 2^-23 of that.
        size = torch.where(dense.any(1)[:, None, :, None], v_rows.scales[:, :, : v_rows.slots].double(), 0.0).abs().amax(-1)
        bound = bound + 2.0 ** (v_rows.bits - 18) * torch.einsum("bgnqk,bgk->bqgn", p, size).reshape(b, s, hq, 1)
    assert ((got.double() - want).abs() <= bound).all(), float(((got.double() - want).abs() - bound).max())
    return got


def _queries(b, s, hq, d, seed=9):
    return torch.randn(b, s, hq, d, generator=_gen(seed), device="cuda").to(torch.bfloat16)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 65, 127, 129, 500, 1025, 4097])
def test_every_length(n, d, bits):
    k_rows, v_rows = _filled(2, n, 2, d, bits, seed=n)
    _check(_queries(2, 1, 8, d), k_rows, v_rows, AttentionMask(), torch.ones(2, 1, n, dtype=torch.bool, device="cuda"))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("s, group", [(1, 1), (1, 3), (1, 8), (2, 4), (8, 1), (3, 2), (1, 16), (4, 4), (16, 1), (3, 5)])
def test_head_layouts_and_several_queries(s, group, d, bits):
    if d == 256 and s * group > 8:
        pytest.skip("read back instead; the other attention has no kernel for 256 channels")
    n = 77
    k_rows, v_rows = _filled(3, n, 2, d, bits, seed=s * 16 + group)
    j, i = torch.arange(n, device="cuda"), torch.arange(s, device="cuda")[:, None] + n - s
    _check(_queries(3, s, 2 * group, d), k_rows, v_rows, AttentionMask(), (j <= i).expand(3, s, n))
    _check(_queries(3, s, 2 * group, d), k_rows, v_rows, None, torch.ones(3, s, n, dtype=torch.bool, device="cuda"), scale=-0.07)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (5, 3), (32, 32), (33, 31), (100, 64), (250, 33), (600, 2), (40, 700)])
@pytest.mark.parametrize("n, s", [(1, 1), (64, 1), (290, 1), (517, 4)])
def test_windows_and_first_tokens(n, s, window, sinks, bits):
    k_rows, v_rows = _filled(2, n, 2, 64, bits, seed=n)
    j, i = torch.arange(n, device="cuda"), torch.arange(s, device="cuda")[:, None] + n - s
    dense = (j <= i) & ((i - j < window) | (j < sinks))
    _check(_queries(2, s, 8, 64), k_rows, v_rows, AttentionMask(window=window, sinks=sinks), dense.expand(2, s, n))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("s", [1, 3])
def test_boolean_masks_with_anything_behind_them(s, bits):
    """Scattered masks, queries without a key, one mask for all rows or queries, and infinities and NaN where nobody looks."""
    n = 333
    k_rows, v_rows = _filled(4, n, 2, 128, bits, seed=3)
    dense = torch.rand(4, s, n, generator=_gen(8), device="cuda") < torch.tensor([0.5, 0.02, 0.9, 0.3], device="cuda")[:, None, None]
    dense[3, 0] = False
    dense[1, :, 64:200] = False
    unseen = (~dense.any(1)).nonzero()
    for x, (b, j) in enumerate(unseen.tolist()):
        for rows in (k_rows, v_rows):
            rows.scales[b, :, j] = (float("nan"), float("inf"), -3e38)[x % 3]
    q = _queries(4, s, 8, 128)
    got = _check(q, k_rows, v_rows, AttentionMask(causal=False, bool_mask=dense), dense)
    assert not got[3, 0].any()
    assert torch.equal(got, ops.quantized_attention(q, k_rows, v_rows, AttentionMask(causal=False, bool_mask=dense[:, None])))
    strided = torch.zeros(4, 2 * s, n + 5, dtype=torch.bool, device="cuda")
    strided[:, ::2, 5:] = dense
    assert torch.equal(got, ops.quantized_attention(q, k_rows, v_rows, AttentionMask(causal=False, bool_mask=strided[:, ::2, 5:])))
    assert torch.equal(got, ops.quantized_attention(q, k_rows, v_rows, AttentionMask(causal=False, bool_mask=dense.transpose(1, 2).contiguous().transpose(1, 2))))
    k_rows, v_rows = _filled(4, n, 2, 128, bits, seed=3)
    _check(q, k_rows, v_rows, AttentionMask(causal=False, bool_mask=dense[2:3, :1]), dense[2:3, :1].expand(4, s, n))


def test_a_slot_that_one_query_sees_and_another_does_not():
    """A NaN in a slot reaches the queries that see it and no others."""
    k_rows, v_rows = _filled(1, 40, 1, 64, 4)
    v_rows.scales[0, 0, 39] = float("nan")
    q = _queries(1, 2, 2, 64)
    got = ops.quantized_attention(q, k_rows, v_rows, AttentionMask())
    assert got[0, 1].isnan().all()
    k_rows2, v_rows2 = _filled(1, 40, 1, 64, 4)
    assert torch.equal(got[0, 0], ops.quantized_attention(q, k_rows2, v_rows2, AttentionMask())[0, 0])


def test_left_padded_rows():
    n, s = 150, 2
    start = torch.tensor([0, 31, 32, 120, 149], dtype=torch.int32, device="cuda")
    k_rows, v_rows = _filled(5, n, 2, 64, 4)
    j, i = torch.arange(n, device="cuda"), torch.arange(s, device="cuda")[:, None] + 120
    dense = (j <= i) & (j >= start[:, None, None])
    got = _check(_queries(5, s, 4, 64), k_rows, v_rows, AttentionMask(key_start=start, query_start=120), dense)
    assert not got[4].any()


def test_slots_behind_the_last_are_not_read():
    """The first slots of a larger cache, whose others hold NaN; the last one of the last head ends the memory."""
    for n in (1, 30, 61, 64):
        k_rows, v_rows = _filled(2, 64, 2, 64, 4)
        for r in (k_rows, v_rows):
            r.scales[:, :, n:] = float("nan")
        _check(_queries(2, 1, 8, 64), k_rows.first(n), v_rows.first(n), AttentionMask(), torch.ones(2, 1, n, dtype=torch.bool, device="cuda"))


def test_views_and_odd_strides():
    k_rows, v_rows = _filled(6, 100, 4, 128, 4)
    part = [QuantizedRows(r.codes[1::2, 1:3], r.scales[1::2, 1:3], 100) for r in (k_rows, v_rows)]
    seen = torch.ones(3, 1, 100, dtype=torch.bool, device="cuda")
    got = _check(_queries(3, 1, 8, 128), *part, AttentionMask(), seen)
    q = torch.randn(3, 1, 8, 257, generator=_gen(9), device="cuda").to(torch.bfloat16)
    _check(q[..., 1:129], *part, AttentionMask(), seen)
    # rows that do not start on 16 bytes are read back first
    loose = [QuantizedRows(r.codes[:, :, :99].contiguous(), r.scales[:, :, :99].contiguous()) for r in part]
    near = ops.quantized_attention(_queries(3, 1, 8, 128), *loose, AttentionMask())
    assert torch.allclose(near.float(), ops.quantized_attention(_queries(3, 1, 8, 128), part[0].first(99), part[1].first(99), AttentionMask()).float(), atol=2.0**-6)
    assert got.shape == (3, 1, 8, 128)


@pytest.mark.parametrize("bits", [4, 8])
def test_many_queries_read_the_cache_back(bits):
    n = s = 200
    k_rows, v_rows = _filled(2, n, 2, 64, bits)
    q = _queries(2, s, 8, 64)
    k, v = ops.quantized_read(k_rows, v_rows)
    assert torch.equal(ops.quantized_attention(q, k_rows, v_rows, AttentionMask()), ops.attention(q, k, v, AttentionMask()))


def test_addresses_past_32_bits():
    b, n = 18, 131072
    rows = _zeros(b, n, 8, 256, 8)
    assert rows[0].codes.numel() > 2**32
    x = torch.randn(1, 4, 8, 256, generator=_gen(1), device="cuda").to(torch.bfloat16)
    last = [QuantizedRows(r.codes[-1:], r.scales[-1:]) for r in rows]
    ops.quantized_append(x.expand(b, 4, 8, 256), x.expand(b, 4, 8, 256), *rows, torch.arange(n - 4, n, device="cuda"))
    assert torch.equal(ops.quantized_read(*rows, n - 4, n)[0][-1], ops.quantized_read(*last, n - 4, n)[0][0])
    small = _zeros(1, 4, 8, 256, 8)
    ops.quantized_append(x, x, *small, torch.arange(4, device="cuda"))
    q = _queries(1, 1, 8, 256)
    mask = torch.zeros(1, 1, n, dtype=torch.bool, device="cuda")
    mask[..., -4:] = True
    got = ops.quantized_attention(q.expand(b, 1, 8, 256), *rows, AttentionMask(causal=False, bool_mask=mask))
    assert torch.equal(got, ops.quantized_attention(q, *small).expand_as(got))


def test_the_same_twice_and_on_another_stream():
    k_rows, v_rows = _filled(1, 9000, 8, 128, 4)
    q = _queries(1, 1, 32, 128)
    a = ops.quantized_attention(q, k_rows, v_rows)
    assert torch.equal(a, ops.quantized_attention(q, k_rows, v_rows))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = torch.randn(1, 1, 8, 128, generator=_gen(2), device="cuda").to(torch.bfloat16)
        ops.quantized_append(x, x, k_rows, v_rows, torch.tensor([77], device="cuda"))
        c = ops.quantized_attention(q, k_rows, v_rows)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(c, ops.quantized_attention(q, k_rows, v_rows)) and not torch.equal(a, c)


def test_recorded_and_replayed():
    """Two recordings that share nothing but the cache, replayed in turn with new tokens and slots."""
    b, n = 2, 96
    k_rows, v_rows = _zeros(b, n, 2, 64, 4)
    plain_k, plain_v = _zeros(b, n, 2, 64, 4)
    x = torch.randn(b, 1, 2, 64, device="cuda").to(torch.bfloat16)
    q, slot = _queries(b, 1, 8, 64), torch.zeros(1, dtype=torch.int64, device="cuda")
    mask = torch.zeros(b, 1, n, dtype=torch.bool, device="cuda")

    def step(k_rows, v_rows):
        ops.quantized_append(x, -x, k_rows, v_rows, slot)
        return ops.quantized_attention(q, k_rows, v_rows, AttentionMask(causal=False, bool_mask=mask))

    step(*_zeros(b, n, 2, 64, 4))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(k_rows, v_rows)
        graphs.append((graph, out))
    for i in range(n):
        x.copy_(torch.randn(b, 1, 2, 64, generator=_gen(100 + i), device="cuda"))
        q.copy_(torch.randn(b, 1, 8, 64, generator=_gen(500 + i), device="cuda"))
        slot.fill_(i)
        mask[..., i] = True
        graph, out = graphs[i % 2]
        graph.replay()
        assert torch.equal(out, step(plain_k, plain_v)), i


# --------------------------------------------------------------------------------------------------------------------------------- decoders


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim", [256, 512])
def test_generation_recorded_and_step_by_step(bits, dim, monkeypatch):
    """Recorded decode steps on quantised caches give what the modules give, for left-padded prompts and on caches that are used again."""
    from torchtune_b200 import generation
    from torchtune_b200.generation._step_graph import StepGraph
    from torchtune_b200.models.llama2 import llama2

    torch.manual_seed(3)
    with torch.device("cuda"):
        model = llama2(vocab_size=304, num_layers=2, num_heads=4, num_kv_heads=2, embed_dim=dim, max_seq_len=128, intermediate_dim=512).to(torch.bfloat16).eval()
        model.setup_caches(3, torch.bfloat16, decoder_max_seq_len=61, kv_cache_bits=bits)
    prompt = torch.randint(1, 304, (3, 23), generator=_gen(1), device="cuda")
    prompt[1, :7] = 0
    recorded = []
    real = StepGraph._record
    monkeypatch.setattr(StepGraph, "_record", lambda self, *a: (recorded.append(1), real(self, *a))[1])

    def run():
        model.reset_caches()
        return generation.generate(model, prompt, max_generated_tokens=30, pad_id=0, temperature=0.8, top_k=20, rng=_gen(5))

    tokens, logits = run()
    assert recorded
    again, logits_again = run()
    with monkeypatch.context() as m:
        m.setattr(StepGraph, "suits", staticmethod(lambda *a: False))
        plain, plain_logits = run()
    assert torch.equal(tokens, again) and torch.equal(logits, logits_again)
    assert torch.equal(tokens, plain) and torch.equal(logits, plain_logits)


def test_a_decode_step_attends_to_what_the_cache_stands_for():
    from torchtune_b200.models.llama2 import llama2

    torch.manual_seed(4)
    with torch.device("cuda"):
        model = llama2(vocab_size=304, num_layers=1, num_heads=8, num_kv_heads=2, embed_dim=512, max_seq_len=256, intermediate_dim=512).to(torch.bfloat16).eval()
        model.setup_caches(2, torch.bfloat16, decoder_max_seq_len=200, kv_cache_bits=4)
    attn = model.layers[0].attn
    x = torch.randn(2, 150, 512, generator=_gen(2), device="cuda").to(torch.bfloat16)
    causal = torch.ones(150, 200, dtype=torch.bool, device="cuda").tril().expand(2, 150, 200)
    with torch.no_grad():
        attn(x[:, :149], x[:, :149], mask=causal[:, :149], input_pos=torch.arange(149, device="cuda").expand(2, -1))
        got = attn(x[:, 149:], x[:, 149:], mask=causal[:, 149:], input_pos=torch.full((2, 1), 149, device="cuda"))
        k, v = ops.quantized_read(*attn.kv_cache.rows(2))
        q = attn.pos_embeddings(attn.q_proj(x[:, 149:]).view(2, 1, 8, 64), input_pos=torch.full((2, 1), 149, device="cuda"))
        want = attn.output_proj(ops.attention(q, k, v, AttentionMask(causal=False, bool_mask=causal[:, 149:])).reshape(2, 1, 512))
    assert attn.kv_cache.size == 150 and not attn.kv_cache.k_scales[:, :, 150:].any()
    # values rounded to bf16 on the way (2^-9 of each) and 150 of them averaged; the projection adds its own rounding to both sides
    assert (got.float() - want.float()).norm() <= 2.0**-6 * want.float().norm()


def test_every_quotient_of_two_bf16_numbers():
    """All pairs of significands, at several exponents apart: the codes are those of exact division, ties included."""
    sig = torch.arange(128, 256, device="cuda", dtype=torch.float64)
    for bits in (4, 8):
        half = 2 ** (bits - 1)
        for shift in range(0, bits + 2):
            # a group per divisor: the largest value, then 31 dividends at a time
            largest = sig * 2.0**-3
            for sign in (1.0, -1.0):
                rows = []
                for start in range(0, 128, 31):
                    part = sig[start : start + 31] * 2.0 ** (-3 - shift)
                    part = torch.nn.functional.pad(part, (0, 31 - part.shape[0]))
                    group = torch.cat([largest[:, None] * sign, part[None, :].expand(128, -1)], 1)
                    group[group.abs() > group[:, :1].abs()] = 0.0  # the first one has to be the largest
                    rows.append(group)
                x = torch.cat(rows)[None, :, None, :].to(torch.bfloat16)
                cache = _zeros(1, x.shape[1], 1, 32, bits)
                ops.quantized_append(x, x, *cache, torch.arange(x.shape[1], device="cuda"))
                got = ops.quantized_read(*cache, dtype=torch.float32)[0][0, :, 0].double()
                wide = x[0, :, 0].double()
                step = wide[:, :1] / -half
                want = (wide / step).round().clamp(-half, half - 1) * step
                assert torch.equal(got, want)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("power", [-70, -30, 20, 40, 60, 100])
def test_large_and_small_values(power, bits):
    """Values, and keys against queries, far from 1: the powers of two that the kernel works with stay within fp32."""
    k_rows, v_rows = _filled(2, 300, 2, 64, bits, seed=2)
    q = _queries(2, 1, 8, 64)
    seen = torch.ones(2, 1, 300, dtype=torch.bool, device="cuda")
    v_rows.scales.mul_(2.0**power)
    got = _check(q, k_rows, v_rows, AttentionMask(), seen)
    assert got.any()
    k_rows.scales.mul_(2.0**-power)
    assert torch.equal(got, _check((q.float() * 2.0**power).to(torch.bfloat16), k_rows, v_rows, AttentionMask(), seen))


@pytest.mark.parametrize("bits", [4, 8])
def test_values_of_very_different_sizes(bits):
    """Scales that grow along the slots: every warp moves to a smaller power of two on the way; a row whose largest scales lie in slots that it does not see."""
    k_rows, v_rows = _filled(3, 700, 1, 128, bits, seed=2)
    v_rows.scales[:, :, :700] *= (2.0 ** torch.linspace(-6, 40, 700, device="cuda"))[:, None].to(torch.bfloat16)
    dense = torch.ones(3, 1, 700, dtype=torch.bool, device="cuda")
    dense[1, :, 300:] = False
    v_rows.scales[1, :, 300:] = 3e38
    dense[2, :, 600:] = torch.rand(100, generator=_gen(4), device="cuda") < 0.5
    _check(_queries(3, 1, 4, 128), k_rows, v_rows, AttentionMask(causal=False, bool_mask=dense), dense, spread=True)
    _check(_queries(3, 1, 4, 128), k_rows, v_rows, AttentionMask(causal=False, bool_mask=dense), dense, scale=2.0, spread=True)


def test_a_query_that_is_not_finite_spoils_its_own_rows_only():
    k_rows, v_rows = _filled(2, 100, 2, 64, 4)
    q = _queries(2, 2, 8, 64)
    clean = ops.quantized_attention(q, k_rows, v_rows, AttentionMask())
    spoilt = q.clone()
    spoilt[0, 1, 3, 5], spoilt[1, 0, 7, 0] = float("nan"), float("inf")
    got = ops.quantized_attention(spoilt, k_rows, v_rows, AttentionMask())
    assert got[0, 1, 3].isnan().all() and got[1, 0, 7].isnan().all()
    same = torch.ones(2, 2, 8, dtype=torch.bool, device="cuda")
    same[0, 1, 3] = same[1, 0, 7] = False
    assert torch.equal(got[same], clean[same])


def test_few_long_rows_recorded():
    """The split that meets in a workspace, in two recordings at once."""
    k_rows, v_rows = _filled(1, 20000, 2, 64, 4)
    q = [_queries(1, 1, 8, 64, seed=i) for i in (1, 2)]
    want = [ops.quantized_attention(x, k_rows, v_rows) for x in q]
    static, graphs = [x.clone() for x in q], []
    for x in static:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.quantized_attention(x, k_rows, v_rows)
        graphs.append((graph, out))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(4):
        for i, (x, (graph, _), stream) in enumerate(zip(static, graphs, streams)):
            x.copy_(q[(i + turn) % 2])
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                graph.replay()
        for stream in streams:
            torch.cuda.current_stream().wait_stream(stream)
        for i, (_, out) in enumerate(graphs):
            assert torch.equal(out, want[(i + turn) % 2])
    dense = torch.rand(1, 1, 20000, generator=_gen(3), device="cuda") < 0.4
    _check(q[0], k_rows, v_rows, AttentionMask(causal=False, bool_mask=dense), dense)
    assert not ops.quantized_attention(q[0], k_rows, v_rows, AttentionMask(causal=False, bool_mask=torch.zeros_like(dense))).any()


@pytest.mark.parametrize("d, bits", [(64, 8), (128, 4), (256, 8)])
@pytest.mark.parametrize("n, window", [(6143, 0), (6144, 0), (6271, 0), (6305, 0), (12345, 0), (30011, 0), (30011, 6139), (30011, 6140), (30011, 20000)])
def test_lengths_where_few_rows_are_split_further(n, window, d, bits):
    k_rows, v_rows = _filled(1, n, 1, d, bits, seed=n)
    at = torch.arange(n, device="cuda")
    dense = ((at > n - 1 - window) | (at < 4))[None, None] if window else torch.ones(1, 1, n, dtype=torch.bool, device="cuda")
    _check(_queries(1, 1, 4, d), k_rows, v_rows, AttentionMask(causal=True, window=window, sinks=4 if window else 0), dense)


@pytest.mark.parametrize("kind", ["all", "causal", "window", "bool"])
@pytest.mark.parametrize("d, bits", [(64, 4), (96, 4), (96, 8), (128, 8), (256, 4)])
@pytest.mark.parametrize("b, s, group", [(2, 1, 4), (1, 3, 4), (2, 4, 4), (1, 1, 5), (3, 16, 1), (1, 1, 16)])
def test_several_rows_that_meet_in_a_workspace(b, s, group, d, bits, kind):
    """One and two tiles of query rows, several queries, batch rows and key heads, whose slots are split further than a cluster reaches."""
    if d == 256 and s * group > 8:
        pytest.skip("read back instead; the other attention has no kernel for 256 channels")
    n, h = 20011, 2
    k_rows, v_rows = _filled(b, n, h, d, bits, seed=s * group)
    j, i = torch.arange(n, device="cuda"), torch.arange(s, device="cuda")[:, None] + n - s
    dense, mask = {
        "all": (torch.ones(b, s, n, dtype=torch.bool, device="cuda"), AttentionMask(causal=False)),
        "causal": ((j <= i).expand(b, s, n), AttentionMask()),
        "window": (((j <= i) & ((i - j < 15000) | (j < 77))).expand(b, s, n), AttentionMask(window=15000, sinks=77)),
        "bool": (torch.rand(b, s, n, generator=_gen(6), device="cuda") < 0.3, None),
    }[kind]
    if mask is None:
        dense[-1, -1] = False  # the last query sees nothing
        mask = AttentionMask(causal=False, bool_mask=dense)
    got = _check(_queries(b, s, h * group, d), k_rows, v_rows, mask, dense)
    assert kind != "bool" or not got[-1, -1].any()
