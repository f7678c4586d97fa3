"""Answers that share their prompts, decoders with norm and rotation as one operator, and GRPO with both and the policy's entropy, on plain statements."""
import json
import re

import pytest
import torch

from torchtune_b200 import generation, ops, rlhf
from torchtune_b200.models.gemma2 import gemma2
from torchtune_b200.models.llama2 import llama2
from torchtune_b200.models.qwen3 import lora_qwen3_0_6b_base, qwen3, qwen3_0_6b_base
from torchtune_b200.modules import KVCache, PromptGroups, SharedPrefixKVCache

_T = dict(vocab_size=90, num_layers=2, num_heads=4, num_kv_heads=2, embed_dim=32, intermediate_dim=48, max_seq_len=64)


def _qwen(**how):
    torch.manual_seed(0)
    model = qwen3(**_T, head_dim=16, norm_eps=1e-6, q_proj_bias=False, k_proj_bias=False, v_proj_bias=False, q_norm=True, k_norm=True, **how).eval()
    with torch.no_grad():
        for p in model.parameters():
            p.mul_(1.5) if p.dim() > 1 else p.add_(0.1 * torch.randn(p.shape))
    return model


def _llama():
    torch.manual_seed(0)
    return llama2(**_T).eval()


def _prompts(padded):
    p = torch.randint(1, 90, (3, 7), generator=torch.Generator().manual_seed(3))
    if padded:
        p[0, :4] = 0
        p[2, :1] = 0
    if padded == "inside":  # ids of padding that no token sees
        p[1, 2], p[2, 4:6] = 0, 0
    return p


@pytest.mark.parametrize("padded", [False, True, "inside"])
@pytest.mark.parametrize("stop", [None, list(range(40, 60))])
@pytest.mark.parametrize("build", [_llama, _qwen, lambda: _qwen(fuse_qk_norm=True)])
def test_groups_are_what_repeated_prompts_generate(build, stop, padded):
    model, prompts, n = build(), _prompts(padded), 6
    how = dict(max_generated_tokens=n, temperature=0.8, top_k=20, stop_tokens=stop)
    tokens, logits = generation.generate_group(model, prompts, samples=4, rng=torch.Generator().manual_seed(5), **how)
    assert not model.caches_are_setup()
    model.setup_caches(12, torch.float32, decoder_max_seq_len=7 + n)
    want, want_logits = generation.generate(model, prompts.repeat_interleave(4, 0), rng=torch.Generator().manual_seed(5), **how)
    assert torch.equal(tokens, want)
    torch.testing.assert_close(logits, want_logits, rtol=1e-4, atol=1e-4)
    assert generation.generate_group(build(), prompts, samples=1, max_generated_tokens=1, return_logits=False)[1] is None


def test_groups_refuse_what_they_cannot_share():
    model, prompts = _llama(), _prompts(False)
    call = lambda m=model, p=prompts, **how: generation.generate_group(m, p, **{**dict(samples=2, max_generated_tokens=2), **how})  # noqa: E731
    call()
    right = prompts.clone()
    right[1, 6] = 0
    for how in (dict(p=right), dict(p=prompts[0]), dict(samples=0), dict(max_generated_tokens=0), dict(p=prompts[:, :0]),
                dict(m=gemma2(**_T, head_dim=16, hidden_capping_value=20.0, final_capping_value=10.0, sliding_window_size=8, query_pre_attn_scalar=24))):
        with pytest.raises(ValueError):
            call(**how)
    model.setup_caches(2, torch.float32)
    with pytest.raises(ValueError):
        call()
    assert type(model.layers[0].attn.kv_cache) is KVCache  # what was there stays


def test_a_shared_cache_refuses_other_batches_and_masks():
    groups = PromptGroups(torch.tensor([0, 2]), 6)
    cache = SharedPrefixKVCache(groups, 5, 3, 2, 16, torch.float32)
    with pytest.raises(ValueError):
        cache.reserve(6, 5)
    with pytest.raises(ValueError):
        cache.reserve(2, 4)
    cache.append(torch.ones(2, 5, 2, 16), torch.ones(2, 5, 2, 16))
    groups.begin()
    with pytest.raises(ValueError):
        cache.reserve(2, 1)
    with pytest.raises(ValueError):
        cache.reserve(6, 2)
    cache.append(torch.ones(6, 1, 2, 16), torch.full((6, 1, 2, 16), 2.0))
    q = torch.zeros(6, 1, 4, 16)
    out = cache.attend(q, ops.AttentionMask(causal=True))
    torch.testing.assert_close(out[0], torch.full((1, 4, 16), 7 / 6))
    torch.testing.assert_close(out[5], torch.full((1, 4, 16), 5 / 4))  # two slots of padding
    for mask in (ops.AttentionMask(causal=False), ops.AttentionMask(causal=True, window=3), ops.AttentionMask(causal=False, bool_mask=torch.ones(6, 1, 8, dtype=torch.bool))):
        with pytest.raises(ValueError):
            cache.attend(q, mask)
    with pytest.raises(ValueError):
        cache.attend(q, ops.AttentionMask(causal=True), softcap=3.0)


def test_fused_norms_change_nothing_but_roundings():
    plain, fused = _qwen(), _qwen(fuse_qk_norm=True)
    tokens = torch.randint(0, 90, (2, 9), generator=torch.Generator().manual_seed(1))
    a, b = plain(tokens), fused(tokens)
    torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-4)
    for model, out in ((plain, a), (fused, b)):
        out.square().mean().backward()
    for (name, p), q in zip(plain.named_parameters(), fused.parameters()):
        torch.testing.assert_close(p.grad, q.grad, rtol=1e-3, atol=1e-5, msg=name)
    # cached, in one piece and token by token, and with caches in few bits
    for bits in (None, 8):
        outs = []
        for model in (plain, fused):
            model = model.eval()
            model.setup_caches(2, torch.float32, decoder_max_seq_len=32, **({} if bits is None or model.layers[0].attn.head_dim % 32 else dict(kv_cache_bits=bits)))
            mask = torch.tril(torch.ones(32, 32, dtype=torch.bool)).unsqueeze(0)
            with torch.no_grad():
                first = model(tokens[:, :6], mask=mask[:, :6], input_pos=torch.arange(6))
                rest = [model(tokens[:, i : i + 1], mask=mask[:, i : i + 1], input_pos=torch.full((2,), i)) for i in range(6, 9)]
            outs.append(torch.cat([first, *rest], 1))
            for layer in model.layers:
                layer.attn.kv_cache, layer.attn.cache_enabled = None, False
        torch.testing.assert_close(*outs, rtol=1e-4, atol=1e-4)
        torch.testing.assert_close(outs[0], a.detach(), rtol=1e-3, atol=1e-3)


def test_builders_take_the_switch():
    with torch.device("meta"):
        model = qwen3_0_6b_base(fuse_qk_norm=True)
        assert all(layer.attn.fuse_qk_norm for layer in model.layers)
        assert not any(layer.attn.fuse_qk_norm for layer in qwen3_0_6b_base().layers)
        assert lora_qwen3_0_6b_base(["q_proj"], fuse_qk_norm=True).layers[0].attn.fuse_qk_norm


def test_statistics_of_responses():
    logits = torch.randn(2, 5, 30, requires_grad=True)
    tokens = torch.randint(0, 30, (2, 5))
    s = rlhf.logits_to_statistics(logits, tokens, 0.9, top=4)
    torch.testing.assert_close(s.logprobs, rlhf.logits_to_logprobs(logits, tokens, 0.9))
    assert s.top_tokens.shape == (2, 5, 4) and s.entropy.requires_grad


def test_grpo_recipe_with_shared_prompts_and_entropy(tmp_path, tune_path, monkeypatch):
    from helpers import run_tune, write_tiny_hf_checkpoint
    from test_recipe_grpo import ARCH
    from tokenizer_assets import write_sentencepiece_model

    ckpt = tmp_path / "policy"
    write_tiny_hf_checkpoint(ckpt, arch=ARCH, builder=llama2)
    (tmp_path / "tok").mkdir()
    sp = write_sentencepiece_model(tmp_path / "tok", vocab_size=200)
    qa = tmp_path / "qa.json"
    qa.write_text(json.dumps([{"question": f"what is {i} plus {i}", "answer": str(2 * i)} for i in range(8)]))
    logs = {}
    for name, more in (("plain", "log_entropy=True"), ("shared", "log_entropy=True share_prompts=True"), ("bonus", "entropy_coeff=0.5")):
        out = tmp_path / name
        run_tune(tune_path, f"run dev/grpo_full_finetune_distributed --config tiny/llama2_grpo checkpointer.checkpoint_dir={ckpt} tokenizer.path={sp} dataset.data_files={qa} output_dir={out} "
                 f"metric_logger.filename=log.txt {more}", monkeypatch)
        text = (out / "logs" / "log.txt").read_text()
        logs[name] = {k: [float(x) for x in re.findall(rf"\b{k}:(\S+)", text)] for k in ("loss", "entropy", "rewards", "response_lengths")}
        assert all(len(v) == 2 and all(x == x for x in v) for v in logs[name].values())
        assert all(0 < x < 5.4 for x in logs[name]["entropy"])  # of 200 tokens: below log 200
    # the same draws from the same distributions
    for k in ("rewards", "response_lengths"):
        assert logs["plain"][k] == logs["shared"][k]
    assert logs["bonus"]["loss"][0] == pytest.approx(logs["plain"]["loss"][0] - 0.5 * logs["bonus"]["entropy"][0], abs=1e-3)


def test_entropy_bonus_does_not_depend_on_the_size_of_the_pieces():
    """Answers of 1 to 6 tokens: gradients and the logged entropy of one pass over all of them and of pieces."""
    from torchtune_b200.dev.grpo import GRPOSimpleLoss, GRPOTrajectory
    from torchtune_b200.engine.grpo import GRPOTrainer

    n, ctx, m = 5, 4, 6
    g = torch.Generator().manual_seed(4)
    tokens = torch.randint(1, 90, (n, ctx + m), generator=g)
    pad = torch.arange(m) >= torch.tensor([1, 6, 3, 2, 5])[:, None]
    ones = torch.ones(n, ctx + m, dtype=torch.bool)
    traj = GRPOTrajectory(query_responses=tokens, logprobs=torch.randn(n, m, generator=g) - 4, ref_logprobs=torch.randn(n, m, generator=g) - 4, advantages=torch.randn(n, generator=g),
                          masks=generation.get_causal_mask_from_padding_mask(ones), position_ids=generation.get_position_ids_from_padding_mask(ones), response_padding_masks=pad, seq_lens=None, answers=None)
    seen = []
    for size in (5, 1, 2):
        trainer = GRPOTrainer.__new__(GRPOTrainer)
        trainer._model = _llama()
        trainer._device, trainer.parallel, trainer._lr_scheduler, trainer._clip_grad_norm, trainer.global_step = torch.device("cpu"), None, None, None, 0
        trainer._forward_batch_size, trainer._temperature, trainer._log_entropy, trainer._entropy_coeff, trainer._loss_fn = size, 0.9, True, 0.7, GRPOSimpleLoss(kl_coeff=0.1)
        grads = []

        class Keep:
            def step(self, of=trainer._model):
                grads.extend(p.grad.clone() for p in of.parameters())

            def zero_grad(self, set_to_none):
                pass

        trainer._optimizer = Keep()
        stats = trainer.grpo_step(traj, ctx)
        seen.append((stats.metadata["entropy"], stats.loss, *grads))
    logits = _llama()(tokens)[:, ctx - 1 : -1] / 0.9
    h = -(torch.softmax(logits, -1) * torch.log_softmax(logits, -1)).sum(-1)
    want = torch.stack([row[~p].mean() for row, p in zip(h, pad)]).mean()
    torch.testing.assert_close(seen[0][0], want.detach(), rtol=1e-5, atol=1e-5)
    for other in seen[1:]:
        for a, b in zip(seen[0], other):
            torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-6)


@pytest.mark.parametrize("build", [_llama, lambda: _qwen(fuse_qk_norm=True)])
def test_a_shared_cache_that_is_full_says_so(build):
    """More steps than it was made for: as of any cache, before anything is written."""
    model, prompts = build(), _prompts(False)
    step = lambda pos: model(torch.ones(6, 1, dtype=torch.long), input_pos=torch.full((6, 1), pos), mask=ops.AttentionMask(causal=True))  # noqa: E731
    with torch.no_grad(), generation.shared_prompts(model, torch.zeros(3, dtype=torch.int64), 6, 7, 2) as groups:
        model(prompts, input_pos=torch.arange(7), mask=torch.tril(torch.ones(1, 7, 7, dtype=torch.bool)))
        for _ in range(2):  # the same caches may answer anew
            groups.begin()
            for i in range(2):
                step(7 + i)
                groups.advance()
            assert groups.steps == int(groups.slot) == 2
            held = [layer.attn.kv_cache.own_k.clone() for layer in model.layers]
            with pytest.raises(AssertionError, match="full"):
                step(9)
            assert all(torch.equal(a, layer.attn.kv_cache.own_k) for a, layer in zip(held, model.layers))
