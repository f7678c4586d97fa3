"""Norm and rotation, attention over shared prompts and statistics of tokens together, as rollouts use them, and the decoders and the generation that call them."""
import pytest
import torch
import torch.nn.functional as F

from torchtune_b200 import generation, ops
from torchtune_b200.generation import _group
from torchtune_b200.models.llama2 import llama2
from torchtune_b200.models.qwen3 import qwen3
from torchtune_b200.ops import _lib, reference

pytestmark = pytest.mark.gpu

DEV = "cuda"
_T = dict(vocab_size=500, num_layers=2, num_heads=8, num_kv_heads=2, embed_dim=256, intermediate_dim=512, max_seq_len=512)


def _qwen(**how):
    torch.manual_seed(0)
    with torch.device(DEV):
        model = qwen3(**_T, head_dim=64, norm_eps=1e-6, q_proj_bias=False, k_proj_bias=False, v_proj_bias=False, q_norm=True, k_norm=True, **how)
    return model.to(torch.bfloat16).eval()


def _llama():
    torch.manual_seed(0)
    with torch.device(DEV):
        return llama2(**{**_T, "num_heads": 4}).to(torch.bfloat16).eval()


def _prompts():
    p = torch.randint(1, 500, (3, 70), generator=torch.Generator().manual_seed(3)).to(DEV)
    p[0, :31] = 0
    p[2, :1] = 0
    return p


def test_steps_of_all_three_recorded_and_replayed():
    """Four steps of 2 prompts with 3 answers each, from projections to statistics, against the chain in 64 bits."""
    prompts, rows, n, hq, hk, d, vocab = 2, 6, 150, 8, 2, 128, 3003
    g = torch.Generator(device=DEV).manual_seed(0)
    make = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
    angle = torch.arange(300, dtype=torch.float64, device=DEV)[:, None] * 1e4 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=DEV) / d)
    table = torch.stack([angle.cos(), angle.sin()], -1).float()
    kp, vp, gq, gk, w = make(prompts, n, hk, d), make(prompts, n, hk, d), 1 + 0.1 * make(d), 1 + 0.1 * make(d), make(vocab, hq * d)
    k_own, v_own = (torch.zeros(rows, 8, hk, d, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    starts = torch.tensor([0, 40], dtype=torch.int32, device=DEV)
    pos = (n - starts).repeat_interleave(3)[:, None].contiguous()
    lengths, slot = torch.ones(rows, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int64, device=DEV)
    q, k, v = make(rows, 1, hq, d), make(rows, 1, hk, d), make(rows, 1, hk, d)
    tokens = torch.randint(0, vocab, (rows,), device=DEV)

    def step():
        a = ops.qk_norm_rope_append(q, k, v, gq, gk, table, pos, k_own, v_own, slot, interleaved=False)
        o = ops.shared_prefix_attention(a, kp, vp, k_own, v_own, prefix_start=starts, lengths=lengths)
        s = ops.token_statistics(ops.linear(o.reshape(rows, hq * d), w) * 0.2, tokens, top=5)
        pos.add_(1), lengths.add_(1), slot.add_(1)
        return o, s

    with torch.no_grad():
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o, s = step()
        wide = lambda t: t.double()  # noqa: E731
        keys, values = [], []
        pos.copy_((n - starts).repeat_interleave(3)[:, None]), lengths.fill_(1), slot.zero_()
        for i in range(4):
            for t in (q, k, v):
                t.copy_(make(*t.shape))
            at = pos.clone()
            graph.replay()
            a = reference.norm_rope(wide(q), wide(gq), table, at, 1e-6, False, True).to(torch.bfloat16)
            keys.append(reference.norm_rope(wide(k), wide(gk), table, at, 1e-6, False, True).to(torch.bfloat16)), values.append(v.clone())
            want = reference.shared_prefix_attention(*(wide(t) for t in (a, kp, vp, torch.cat(keys, 1), torch.cat(values, 1))), starts, None, None, None)
            # one step of bf16 in queries and keys moves scores of up to 6 by 2^-8 of that and the probabilities as much again; outputs are below 1
            assert (wide(o) - want).abs().max() < 6 * 2.0**-8
            exact = reference.token_statistics(wide(F.linear(o.reshape(rows, -1), w) * 0.2), tokens, 1.0, 5, -100)
            close = wide(ops.linear(o.reshape(rows, hq * d), w) * 0.2)
            mine = reference.token_statistics(close, tokens, 1.0, 5, -100)
            assert torch.equal(s.top_tokens, mine[3])
            for x, y in zip(s[:3], mine[:3]):
                torch.testing.assert_close(wide(x), y, rtol=2e-5, atol=2e-5)
            assert (s.entropy - exact[1]).abs().max() < 0.05
        assert torch.equal(k_own[:, :4], torch.cat(keys, 1)) or (k_own[:, :4].float() - torch.cat(keys, 1).float()).abs().max() < 0.04  # a tie of the rounding may fall either way
        assert torch.equal(v_own[:, :4], torch.cat(values, 1)) and not k_own[:, 4:].any()
    _lib.check_device_errors()


@pytest.mark.parametrize("build", [_llama, _qwen, lambda: _qwen(fuse_qk_norm=True)])
def test_groups_generate_from_the_models_own_distributions(build, monkeypatch):
    model, prompts, n = build(), _prompts(), 9
    how = dict(samples=4, max_generated_tokens=n, temperature=0.9)
    tokens, logits = generation.generate_group(model, prompts, rng=torch.Generator(DEV).manual_seed(5), **how)
    assert tokens.shape == (12, 79) and logits.shape == (12, n, 500) and torch.equal(tokens[:, :70], prompts.repeat_interleave(4, 0))
    real = F.pad(prompts.repeat_interleave(4, 0) != 0, (0, n), value=True)
    with torch.no_grad():
        whole = model(tokens, mask=generation.get_causal_mask_from_padding_mask(real), input_pos=generation.get_position_ids_from_padding_mask(real))[:, 69:-1].float()
    # the same sums of bf16 products in another order and with other roundings between them: a few steps of bf16 of the logits' size
    assert (logits.float() - whole).norm() / whole.norm() < 4 * 2.0**-8
    # as it is and recorded are the same
    monkeypatch.setattr(_group.StepGraph, "suits", staticmethod(lambda *a: False))
    plain = generation.generate_group(model, prompts, rng=torch.Generator(DEV).manual_seed(5), **how)
    assert torch.equal(plain[0], tokens) and torch.equal(plain[1], logits)
    _lib.check_device_errors()


def test_two_groups_one_after_the_other_and_stops():
    model, prompts = _qwen(fuse_qk_norm=True), _prompts()
    how = dict(max_generated_tokens=12, temperature=1.0, stop_tokens=list(range(0, 500, 9)))
    first = generation.generate_group(model, prompts, samples=3, rng=torch.Generator(DEV).manual_seed(1), **how)
    other = generation.generate_group(model, prompts[1:, 20:], samples=5, rng=torch.Generator(DEV).manual_seed(2), **how)
    again = generation.generate_group(model, prompts, samples=3, rng=torch.Generator(DEV).manual_seed(1), **how)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1]) and other[0].shape[0] == 10
    assert not model.caches_are_setup()


def test_fused_norms_in_training_and_in_cached_steps():
    plain, fused = _qwen(), _qwen(fuse_qk_norm=True)
    tokens = torch.randint(0, 500, (2, 200), device=DEV)
    grads = []
    for model in (plain, fused):
        out = model(tokens)
        F.cross_entropy(out.float().flatten(0, 1), tokens.flatten()).backward()
        grads.append([out.detach().float()] + [p.grad.float() for p in model.parameters()])
    for a, b in zip(*grads):
        # gradients of two layers with bf16 activations, one rounding apart
        assert (a - b).norm() / a.norm() < 0.03
    outs = []
    for model in (plain, fused):
        with torch.device(DEV):
            model.setup_caches(2, torch.bfloat16, decoder_max_seq_len=256)
        mask = torch.tril(torch.ones(256, 256, dtype=torch.bool, device=DEV)).unsqueeze(0)
        with torch.no_grad():
            first = model(tokens[:, :190], mask=mask[:, :190], input_pos=torch.arange(190, device=DEV))
            rest = [model(tokens[:, i : i + 1], mask=mask[:, i : i + 1], input_pos=torch.full((2,), i, device=DEV)) for i in range(190, 200)]
        outs.append(torch.cat([first, *rest], 1).float())
    assert (outs[0] - outs[1]).norm() / outs[0].norm() < 0.03 and (outs[1] - grads[1][0]).norm() / grads[1][0].norm() < 0.03
    assert _lib.index_violations() == 0


def test_recorded_steps_run_count_and_end_with_their_caches(monkeypatch):
    """A generation of this length records a step and replays it; the host's count is the device's, and a step too many is refused."""
    model, prompts, replays = _qwen(fuse_qk_norm=True), _prompts(), []
    replay = torch.cuda.CUDAGraph.replay
    monkeypatch.setattr(torch.cuda.CUDAGraph, "replay", lambda self: replays.append(1) or replay(self))
    generation.generate_group(model, prompts, samples=2, max_generated_tokens=9)
    assert len(replays) == 7  # eight steps, of which the first runs as it is
    real, device = prompts != 0, prompts.device
    with torch.no_grad(), generation.shared_prompts(model, 70 - real.sum(1), 6, 70, 5) as groups:
        model(prompts, input_pos=generation.get_position_ids_from_padding_mask(real), mask=generation.get_causal_mask_from_padding_mask(real))
        groups.begin()
        tokens = torch.ones(6, 1, dtype=torch.long, device=device)
        step = _group._Steps(model, groups, torch.full((6, 1), 70, dtype=torch.int32, device=device), tokens.clone(), True)
        for i in range(5):
            step(tokens)
            assert groups.steps == i + 1 == int(groups.slot)
        assert step.graph is not None
        with pytest.raises(AssertionError, match="full"):
            step(tokens)
        assert groups.steps == 5 == int(groups.slot)
        del step
    _lib.check_device_errors()
