"""Several answers to each prompt: a prompt is read and kept once, whatever the number of its answers."""
from __future__ import annotations

from contextlib import contextmanager
from typing import Iterator, List, Optional, Tuple

import torch

from ..modules import MultiHeadAttention, PromptGroups, SharedPrefixKVCache, TransformerDecoder, TransformerSelfAttentionLayer
from ..ops.mask import AttentionMask
from ._generation import _exponential_like, get_causal_mask_from_padding_mask, get_position_ids_from_padding_mask, last_logits, sample, update_stop_tokens_tracker
from ._step_graph import StepGraph, _alone


def _refusal(model) -> Optional[str]:
    """Why a model's rows cannot share their prompts."""
    if type(model) is not TransformerDecoder or model.loop is not None or model.pos_embeddings is not None or model.num_output_chunks or model.skip_output_layer or model.output_hidden_states:
        return "prompts are shared in plain decoders, which return logits"
    for layer in model.layers:
        attn = getattr(layer, "attn", None)
        if getattr(layer, "inner_cls", type(layer)) is not TransformerSelfAttentionLayer or layer.mask_mod is not None or not isinstance(attn, MultiHeadAttention) or type(attn).forward is not MultiHeadAttention.forward:
            return "prompts are shared in decoders whose layers are plain self-attention without masks of their own"
        if attn.softcap > 0.0 or getattr(attn, "context_parallel", None) is not None or (attn.training and attn.attn_dropout):
            return "prompts are shared in attention without soft caps, dropout or sharded sequences"
        if attn.kv_cache is not None:
            return "the model has caches already (delete_kv_caches)"
    return None


@contextmanager
def shared_prompts(model: TransformerDecoder, starts: torch.Tensor, rows: int, prompt_len: int, max_new_tokens: int) -> Iterator[PromptGroups]:
    """Gives all layers of a plain decoder a :class:`~torchtune_b200.modules.SharedPrefixKVCache` for ``rows`` answers to prompts whose first real slots are ``starts`` (``[prompts]``), until the block
    is left."""
    why = _refusal(model)
    if why is not None:
        raise ValueError(why)
    if starts.shape[0] == 0 or rows % starts.shape[0]:
        raise ValueError(f"{rows} rows are not the same number of answers to each of {starts.shape[0]} prompts")
    groups = PromptGroups(starts, rows)
    layers = [layer.attn for layer in model.layers]
    before = model.decoder_max_cache_seq_len
    model.decoder_max_cache_seq_len = prompt_len + max_new_tokens
    try:
        for attn in layers:
            attn.kv_cache = SharedPrefixKVCache(groups, prompt_len, max_new_tokens, attn.num_kv_heads, attn.head_dim, model.tok_embeddings.weight.dtype)
            attn.cache_enabled = True
        yield groups
    finally:
        model.decoder_max_cache_seq_len = before
        for attn in layers:
            attn.kv_cache, attn.cache_enabled = None, False


class _Steps:
    """The step of one token per row, recorded once it has run as it is (where that may be: see :class:`StepGraph`) and replayed from then on."""

    def __init__(self, model: TransformerDecoder, groups: PromptGroups, pos: torch.Tensor, tokens: torch.Tensor, recorded: bool) -> None:
        self.model, self.groups, self.pos, self.tokens, self.recorded = model, groups, pos, tokens, recorded
        self.graph: Optional[torch.cuda.CUDAGraph] = None
        self.ran = False

    def _body(self) -> torch.Tensor:
        logits = self.model(self.tokens, input_pos=self.pos, mask=AttentionMask(causal=True))[:, -1]
        self.pos.add_(1)
        self.groups.advance()
        return logits

    def __call__(self, tokens: torch.Tensor) -> torch.Tensor:
        self.tokens.copy_(tokens)
        if not self.recorded or not self.ran:
            self.ran = True
            return self._body()
        if self.graph is None:
            if not _alone():
                return self._body()
            device = tokens.device
            graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream(device=device)
            stream.wait_stream(torch.cuda.current_stream(device))
            with torch.cuda.stream(stream):
                graph.capture_begin(capture_error_mode="thread_local")
                try:
                    self.logits = self._body()
                finally:
                    graph.capture_end()
            torch.cuda.current_stream(device).wait_stream(stream)
            self.graph = graph  # and this step is counted
        else:
            self.model.layers[0].attn.kv_cache.reserve(self.groups.rows, 1)  # raises when the cache is full
            self.groups.steps += 1
        self.graph.replay()
        return self.logits.clone()


@torch.no_grad()
def generate_group(
    model: TransformerDecoder,
    prompt: torch.Tensor,
    *,
    samples: int,
    max_generated_tokens: int,
    pad_id: int = 0,
    temperature: float = 1.0,
    top_k: Optional[int] = None,
    stop_tokens: Optional[List[int]] = None,
    rng: Optional[torch.Generator] = None,
    return_logits: bool = True,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``samples`` answers to each of ``prompt`` (``[prompts, s]``, left-padded with ``pad_id`` when lengths differ): what :func:`generate` returns for every prompt repeated ``samples`` times,
    ``(tokens [prompts * samples, s + n], logits [prompts * samples, n, vocab])``, but prompts are read once and their keys and values kept and, in every step, read once.  The model is a plain
    decoder (rotary or no positions, no windows or soft caps) without caches; it gets its own for the call.  With the same ``rng`` draws are those of :func:`generate`."""
    if prompt.dim() != 2 or prompt.numel() == 0 or samples < 1 or max_generated_tokens < 1:
        raise ValueError(f"prompts {tuple(prompt.shape)} are not [prompts, tokens], or {samples} answers of {max_generated_tokens} tokens are none")
    device, (prompts, length), rows = prompt.device, prompt.shape, prompt.shape[0] * samples
    real = prompt != pad_id
    starts = length - real.sum(1)
    asked = prompt
    if not bool((real == (torch.arange(length, device=device) >= starts[:, None])).all()):
        # ids of padding inside a prompt, which no token sees: without them, so that a prompt's tokens are one run
        if not bool((real[:, -1] | ~real.any(1)).all()):
            raise ValueError("prompts are padded on the left: the last token of a prompt is a real one")
        order = torch.sort(real.to(torch.int8), dim=1, stable=True).indices
        prompt, real = prompt.gather(1, order), real.gather(1, order)
    if bool(real.all()):
        mask, pos = torch.tril(torch.ones(length, length, dtype=torch.bool, device=device)).unsqueeze(0), torch.arange(length, device=device).unsqueeze(0)
    else:
        mask, pos = get_causal_mask_from_padding_mask(real), get_position_ids_from_padding_mask(real)

    def draw() -> Optional[torch.Tensor]:
        return None if rng is None else _exponential_like((rows, model.tok_embeddings.num_embeddings), device, rng)

    with shared_prompts(model, starts, rows, length, max_generated_tokens) as groups:
        logits = last_logits(model, prompt, input_pos=pos, mask=mask).repeat_interleave(samples, 0)
        tokens = sample(logits.clone(), temperature=temperature, top_k=top_k, q=draw())
        out, kept = [tokens], [logits.unsqueeze(1)] if return_logits else None
        groups.begin()
        first = (length - starts).to(torch.int32).repeat_interleave(samples)[:, None].contiguous()
        step = _Steps(model, groups, first, torch.empty_like(tokens), max_generated_tokens > 4 and StepGraph.suits(model, prompt, (SharedPrefixKVCache,)))
        stop = torch.tensor(stop_tokens, device=device, dtype=tokens.dtype) if stop_tokens else None
        reached = torch.zeros(rows, dtype=torch.bool, device=device)
        keep = [torch.ones(rows, 1, dtype=torch.bool, device=device)]
        while True:
            if stop is not None:
                reached = update_stop_tokens_tracker(tokens, stop, reached)
                if bool(reached.all()):
                    break
            if len(out) == max_generated_tokens:
                break
            keep.append(~reached[:, None])
            logits = step(tokens)
            tokens = sample(logits.clone(), temperature=temperature, top_k=top_k, q=draw())
            out.append(tokens)
            if kept is not None:
                kept.append(logits.unsqueeze(1))
        del step  # and with it its recording, before the caches that it reads
    alive = torch.cat(keep, 1)
    answers = torch.where(alive, torch.cat(out, 1), torch.full_like(alive, pad_id, dtype=tokens.dtype))
    result = torch.cat([asked.repeat_interleave(samples, 0), answers.to(prompt.dtype)], 1)
    return result, None if kept is None else torch.cat(kept, 1) * alive[..., None]
