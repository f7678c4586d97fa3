"""Rollouts of a group of answers to one prompt, operator by operator: norms of queries and keys per head with the position rotation in the same pass (and the write to
the cache), attention of rows that share a long prefix, and log-probabilities of given tokens with the entropy and the likeliest alternatives.

``run`` is one pass through an operator, in elementary torch operations or, with ``own``, by the calls that a user makes.

* ``rotate``: per head ``z = x / sqrt(mean(x²) + eps) · gain``, then pairs of channels are turned by the table's angle for the token's position; or, with ``after``, turned first and normalised
  then.  With ``grads`` forward and backward, gains' gradients among them; with ``slots`` the keys and values of the new tokens go to their slots of a cache.
* ``prefix``: row ``r`` of a batch belongs to prompt ``r // (rows / prompts)``.  Its queries see the prompt's keys from the prompt's first real token on (prompts are padded on the left) and
  the keys of its own answer up to their own position; a row's queries are the last of its ``length`` tokens.
* ``stats``: of ``z = logits / temperature`` the log-probability of a given token, the entropy ``-Σ p log p``, and the ``top`` largest logits (of equal ones the lower index first) with
  their log-probabilities; with ``grads`` the gradient of the first two as well.

Sizes are those of decoders that the recipes serve: 16 to 64 query heads on 8 key heads of 64 or 128 channels, vocabularies of 32 000 to 151 936."""
from __future__ import annotations

import math
from typing import Any, Dict, List, Optional, Tuple

import torch

own = False

DEV = "cuda"
HKV = 8
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed() -> List[Dict[str, Any]]:
    return [
        # One decode step of 16 rollouts: the new token's queries and keys, and the write to the cache (the smallest call; launches count).
        dict(name="rotate_token", kind="rotate", batch=16, new=1, hq=32, d=128, interleaved=False, after=False, gains=True, grads=False, slots=1024, at=731),
        # Prompts of a batch enter their cache.
        dict(name="rotate_prompts", kind="rotate", batch=4, new=1999, hq=32, d=128, interleaved=False, after=False, gains=True, grads=False, slots=4096, at=0),
        # Fine-tuning, forward and backward: four rows of 2048 tokens.
        dict(name="rotate_train", kind="rotate", batch=4, new=2048, hq=32, d=128, interleaved=False, after=False, gains=True, grads=True, slots=0, at=0),
        # The other order and layout, without gains, on smaller heads and odd lengths, forward and backward.
        dict(name="rotate_train_after", kind="rotate", batch=3, new=517, hq=16, d=64, interleaved=True, after=True, gains=False, grads=True, slots=0, at=0),
        # A short question and four answers that have just begun: the smallest attention.
        dict(name="prefix_chat", kind="prefix", prompts=1, rows=4, queries=1, prefix=61, pad=0, slots=64, length=17, hq=32, d=64),
        # Rollouts of a batch of padded prompts, answers of different lengths.
        dict(name="prefix_rollouts", kind="prefix", prompts=4, rows=64, queries=1, prefix=613, pad=200, slots=512, length=391, hq=32, d=128),
        # One long document, sixteen answers: few rows, so the keys have to be split.
        dict(name="prefix_document", kind="prefix", prompts=1, rows=16, queries=1, prefix=32003, pad=0, slots=512, length=300, hq=32, d=128),
        # Many rollouts of long prompts with three drafted tokens each: the largest attention.
        dict(name="prefix_drafts", kind="prefix", prompts=8, rows=256, queries=3, prefix=4096, pad=500, slots=1024, length=1001, hq=32, d=128),
        # The sampled tokens of 16 rollouts with 20 alternatives each: few rows.
        dict(name="stats_token", kind="stats", rows=16, vocab=128256, dtype="fp32", top=20, temperature=1.0, grads=False),
        # All tokens of a batch of finished answers, with alternatives.
        dict(name="stats_answers", kind="stats", rows=4136, vocab=128256, dtype="bf16", top=5, temperature=0.7, grads=False),
        # The policy's own log-probabilities with an entropy bonus, forward and backward: the largest case.
        dict(name="stats_train", kind="stats", rows=4096, vocab=151936, dtype="bf16", top=0, temperature=1.0, grads=True),
        # A vocabulary of an odd size, in which rows begin at any address, forward and backward.
        dict(name="stats_train_odd", kind="stats", rows=333, vocab=32003, dtype="bf16", top=3, temperature=0.9, grads=True),
    ]


def _log(rng, low: int, high: int) -> int:
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng) -> Dict[str, Any]:
    kind = rng.choice(["rotate", "prefix", "stats"])
    if kind == "rotate":
        grads = rng.random() < 0.5
        batch = _log(rng, 1, 64)
        new = _log(rng, 1, max(1, 8192 // batch)) if grads else rng.choice([1, _log(rng, 2, max(2, 8192 // batch))])
        at = 0 if grads else rng.choice([0, _log(rng, 1, 1000)])
        return dict(kind=kind, batch=batch, new=new, hq=rng.choice([8, 16, 32, 40, 64]), d=rng.choice([64, 128]), interleaved=rng.random() < 0.4, after=rng.random() < 0.3,
                    gains=rng.random() < 0.8, grads=grads, slots=0 if grads else at + new + rng.randint(0, 100), at=at)
    if kind == "prefix":
        prompts, hq = _log(rng, 1, 16), rng.choice([8, 16, 32, 40, 64])
        rows = prompts * _log(rng, 1, max(1, 256 // prompts))
        queries = rng.choice([1, 1, 1, 2, 3, 4])
        prefix = _log(rng, 1, min(40000, 65536 // prompts, 96_000_000 // (rows * queries * hq)))
        slots = _log(rng, queries, max(queries, min(2048, 262144 // rows)))
        return dict(kind=kind, prompts=prompts, rows=rows, queries=queries, prefix=prefix, pad=rng.choice([0, rng.randint(0, prefix)]), slots=slots, length=rng.randint(queries, slots),
                    hq=hq, d=rng.choice([64, 128]))
    grads = rng.random() < 0.5
    vocab = rng.choice([32000, 50257, 128256, 151936, _log(rng, 500, 160000)])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    rows = _log(rng, 1, min(8192, (300_000_000 if dtype == "fp32" else 500_000_000) // vocab))
    return dict(kind=kind, rows=rows, vocab=vocab, dtype=dtype, top=rng.choice([0, rng.randint(1, 32)]), temperature=rng.choice([1.0, round(rng.uniform(0.3, 1.5), 2)]), grads=grads)


# ------------------------------------------------------------------------------------------------------------------------------------- cases


def _normal(g: torch.Generator, *shape: int, scale: float = 1.0) -> torch.Tensor:
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(torch.bfloat16)


def prepare(case: Dict[str, Any], seed: int) -> Dict[str, Any]:
    g = torch.Generator(device=DEV).manual_seed(seed)
    state: Dict[str, Any] = {"case": case}
    if case["kind"] == "rotate":
        b, s, d = case["batch"], case["new"], case["d"]
        # outputs of projections: heads differ in size
        spread = lambda h: torch.exp(0.5 * torch.randn(h, 1, generator=g, device=DEV))  # noqa: E731
        state["q"] = (torch.randn(b, s, case["hq"], d, generator=g, device=DEV) * spread(case["hq"])).to(torch.bfloat16)
        state["k"] = (torch.randn(b, s, HKV, d, generator=g, device=DEV) * spread(HKV)).to(torch.bfloat16)
        state["gains"] = tuple((1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(torch.bfloat16) for _ in range(2)) if case["gains"] else (None, None)
        length = case["at"] + s + 64
        angle = torch.arange(length, device=DEV, dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d)
        state["table"] = torch.stack([angle.cos(), angle.sin()], -1).float()
        state["pos"] = None
        if case["grads"]:
            state["dq"], state["dk"] = _normal(g, b, s, case["hq"], d), _normal(g, b, s, HKV, d)
        else:
            # rows are padded on the left: their positions lag behind the slots
            lag = torch.randint(0, case["at"] + 1, (b, 1), generator=g, device=DEV)
            state["pos"] = (torch.arange(case["at"], case["at"] + s, device=DEV)[None] - lag).to(torch.int32)
            state["v"] = _normal(g, b, s, HKV, d)
            state["slots"] = torch.arange(case["at"], case["at"] + s, device=DEV)
            state["k_cache"], state["v_cache"] = (torch.zeros(b, case["slots"], HKV, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        return state
    if case["kind"] == "prefix":
        p, r, d = case["prompts"], case["rows"], case["d"]
        state["q"] = _normal(g, r, case["queries"], case["hq"], d)
        state["k_prefix"], state["v_prefix"] = _normal(g, p, case["prefix"], HKV, d), _normal(g, p, case["prefix"], HKV, d)
        state["k"], state["v"] = _normal(g, r, case["slots"], HKV, d), _normal(g, r, case["slots"], HKV, d)
        starts, lengths = _spread(case)
        state["starts"] = starts.to(DEV)[torch.randperm(p, generator=g, device=DEV)].int()
        state["lengths"] = lengths.to(DEV)[torch.randperm(r, generator=g, device=DEV)].int()
        return state
    rows, v = case["rows"], case["vocab"]
    # a language model is sure of some tokens and not of others: rows differ in width
    logits = torch.randn(rows, v, generator=g, device=DEV)
    logits *= 1.0 + 3.0 * torch.rand(rows, 1, generator=g, device=DEV)
    state["logits"] = logits.to(TYPES[case["dtype"]])
    likely = logits.argmax(1)
    del logits
    state["tokens"] = torch.where(torch.rand(rows, generator=g, device=DEV) < 0.7, likely, torch.randint(0, v, (rows,), generator=g, device=DEV))
    if case["grads"]:
        state["d_logprobs"], state["d_entropy"] = (torch.randn(rows, generator=g, device=DEV) for _ in range(2))
        if case["top"]:
            state["d_top"] = torch.randn(rows, case["top"], generator=g, device=DEV)
    return state


def _spread(case: Dict[str, Any]) -> Tuple[torch.Tensor, torch.Tensor]:
    """First real slot of each prompt, from 0 to ``pad``, and length of each answer, from half of ``length`` to all of it; in an order that the seed changes."""
    starts = torch.linspace(0, case["pad"], case["prompts"]).long()
    lengths = torch.linspace(max(case["queries"], case["length"] // 2), case["length"], case["rows"]).long()
    return starts, lengths


def run(state: Dict[str, Any]) -> Dict[str, torch.Tensor]:
    return {"rotate": _run_rotate, "prefix": _run_prefix, "stats": _run_stats}[state["case"]["kind"]](state, state["case"])


# ------------------------------------------------------------------------------------------------------------------------------- plain forms


def _turn(x: torch.Tensor, cs: torch.Tensor, interleaved: bool, back: bool = False) -> torch.Tensor:
    """Pairs of channels turned by the angles whose cosines and sines are ``cs`` ``[..., 1, d / 2, 2]``, or back."""
    x = x.unflatten(-1, (-1, 2)) if interleaved else x.unflatten(-1, (2, -1)).transpose(-1, -2)
    cos, sin = cs[..., 0], -cs[..., 1] if back else cs[..., 1]
    y = torch.stack([x[..., 0] * cos - x[..., 1] * sin, x[..., 1] * cos + x[..., 0] * sin], -1)
    return (y if interleaved else y.transpose(-1, -2)).flatten(-2)


def _rotate(x: torch.Tensor, gain: Optional[torch.Tensor], cs: torch.Tensor, case: Dict[str, Any], dy: Optional[torch.Tensor] = None):
    """The operator on one of queries and keys, and with ``dy`` the gradients of input and gain, in 32 bits."""
    x, w, turn = x.float(), 1.0 if gain is None else gain.float(), case["interleaved"]
    u = _turn(x, cs, turn) if case["after"] else x
    r = (u.square().mean(-1, keepdim=True) + EPS).rsqrt()
    n = u * r
    y = n * w if case["after"] else _turn(n * w, cs, turn)
    if dy is None:
        return y, None, None
    dz = dy.float() if case["after"] else _turn(dy.float(), cs, turn, back=True)
    dw = None if gain is None else (dz * n).sum((0, 1, 2)).to(gain.dtype)
    dn = dz * w
    du = r * (dn - n * (dn * n).mean(-1, keepdim=True))
    return y, _turn(du, cs, turn, back=True) if case["after"] else du, dw


def _run_rotate(st, case):
    q, k, (gq, gk) = st["q"], st["k"], st["gains"]
    how = dict(eps=EPS, interleaved=case["interleaved"], norm_first=not case["after"])
    if own:
        from torchtune_b200 import ops

        if not case["grads"]:
            return {"q": ops.qk_norm_rope_append(q, k, st["v"], gq, gk, st["table"], st["pos"], st["k_cache"], st["v_cache"], st["slots"], **how), "k": st["k_cache"], "v": st["v_cache"]}
        leaves = [t.detach().requires_grad_() for t in (q, k, gq, gk) if t is not None]
        out = ops.qk_norm_rope(*leaves[:2], *(leaves[2:] or (None, None)), st["table"], **how)
        grads = torch.autograd.grad(out, leaves, (st["dq"], st["dk"]))
        return {"q": out[0].detach(), "k": out[1].detach(), **dict(zip(("dq", "dk", "dgq", "dgk"), grads))}
    bf = torch.bfloat16
    if not case["grads"]:
        cs = st["table"][st["pos"].long()][:, :, None]
        st["k_cache"][:, st["slots"]] = _rotate(k, gk, cs, case)[0].to(bf)
        st["v_cache"][:, st["slots"]] = st["v"]
        return {"q": _rotate(q, gq, cs, case)[0].to(bf), "k": st["k_cache"], "v": st["v_cache"]}
    cs = st["table"][None, : case["new"], None]
    yq, dq, dgq = _rotate(q, gq, cs, case, st["dq"])
    yk, dk, dgk = _rotate(k, gk, cs, case, st["dk"])
    out = {"q": yq.to(bf), "k": yk.to(bf), "dq": dq.to(bf), "dk": dk.to(bf)}
    return {**out, "dgq": dgq, "dgk": dgk} if case["gains"] else out


def _run_prefix(st, case):
    if own:
        from torchtune_b200 import ops

        with torch.no_grad():
            return {"out": ops.shared_prefix_attention(st["q"], st["k_prefix"], st["v_prefix"], st["k"], st["v"], prefix_start=st["starts"], lengths=st["lengths"])}
    p, (r, s, hq, d) = case["prompts"], st["q"].shape
    g = hq // HKV
    q = st["q"].float().view(r, s, HKV, g, d).permute(0, 2, 3, 1, 4) * d**-0.5  # [r, hkv, g, s, d]
    shared = q.view(p, r // p, HKV, g, s, d).transpose(1, 2).reshape(p, HKV, -1, d)  # [p, hkv, rows of the prompt, d]
    kp, vp, k, v = (st[x].float().transpose(1, 2) for x in ("k_prefix", "v_prefix", "k", "v"))
    a = shared @ kp.transpose(-1, -2)
    a.masked_fill_((torch.arange(case["prefix"], device=DEV) < st["starts"][:, None])[:, None, None], float("-inf"))
    b = (q.reshape(r, HKV, g * s, d) @ k.transpose(-1, -2)).view(r, HKV, g, s, -1)
    last = st["lengths"][:, None] - s + torch.arange(s, device=DEV)  # [r, s]
    b.masked_fill_((torch.arange(case["slots"], device=DEV) > last[..., None])[:, None, None], float("-inf"))
    a = a.view(p, HKV, r // p, g, s, -1).transpose(1, 2).reshape(r, HKV, g, s, -1)
    top = torch.maximum(a.amax(-1, keepdim=True), b.amax(-1, keepdim=True))
    top = torch.where(top.isfinite(), top, torch.zeros_like(top))
    a, b = a.sub_(top).exp_(), b.sub_(top).exp_()
    total = a.sum(-1, keepdim=True) + b.sum(-1, keepdim=True)
    o = (a.view(p, r // p, HKV, g, s, -1).transpose(1, 2).reshape(p, HKV, -1, case["prefix"]) @ vp).view(p, HKV, r // p, g, s, d).transpose(1, 2).reshape(r, HKV, g, s, d)
    o = o + (b.view(r, HKV, g * s, -1) @ v).view(r, HKV, g, s, d)
    o = o / torch.where(total > 0, total, torch.ones_like(total))
    return {"out": o.permute(0, 3, 1, 2, 4).reshape(r, s, hq, d).to(torch.bfloat16)}


def _largest(x: torch.Tensor, top: int) -> torch.Tensor:
    """Indices of the ``top`` largest of each row, of equal ones the lower index first."""
    bits = x.float().view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)  # as the numbers themselves
    key = (order << 20) + ((1 << 20) - 1 - torch.arange(x.shape[-1], device=x.device))
    return (1 << 20) - 1 - (key.topk(top, dim=-1).values & ((1 << 20) - 1))


def _run_stats(st, case):
    x, tokens, top = st["logits"], st["tokens"], case["top"]
    names = ("logprobs", "entropy", "top_logprobs", "top_tokens")
    if own:
        from torchtune_b200 import ops

        how = dict(temperature=case["temperature"], top=top)
        if not case["grads"]:
            with torch.no_grad():
                s = ops.token_statistics(x, tokens, **how)
            return {n: t for n, t in zip(names, s) if t is not None}
        leaf = x.detach().requires_grad_()
        s = ops.token_statistics(leaf, tokens, **how)
        (dx,) = torch.autograd.grad(s[: 3 if top else 2], leaf, [st["d_logprobs"], st["d_entropy"]] + ([st["d_top"]] if top else []))
        return {**{n: t.detach() for n, t in zip(names, s) if t is not None}, "dlogits": dx}
    z = x.float() / case["temperature"]
    z = z - z.amax(-1, keepdim=True)
    logp = z - z.exp().sum(-1, keepdim=True).log()
    del z
    p = logp.exp()
    entropy = -(p * logp).sum(-1)
    out = {"logprobs": logp.gather(-1, tokens[:, None])[:, 0], "entropy": entropy}
    if top:
        out["top_tokens"] = _largest(x, top)
        out["top_logprobs"] = logp.gather(-1, out["top_tokens"])
    if case["grads"]:
        # d log p_t / dz_v = [v = t] - p_v, dH / dz_v = -p_v (log p_v + H)
        g1, g2 = st["d_logprobs"][:, None], st["d_entropy"][:, None]
        whole = g1 + st["d_top"].sum(-1, keepdim=True) if top else g1
        dz = logp.add_(entropy[:, None]).mul_(g2).add_(whole).mul_(p).neg_()
        dz.scatter_add_(-1, tokens[:, None], g1)
        if top:
            dz.scatter_add_(-1, out["top_tokens"], st["d_top"])
        out["dlogits"] = dz.div_(case["temperature"]).to(x.dtype)
    return {n: out[n] for n in (*names, "dlogits") if n in out}


def work(case: Dict[str, Any]) -> Dict[str, float]:
    if case["kind"] == "rotate":
        tokens, d = case["batch"] * case["new"], case["d"]
        values = tokens * (case["hq"] + HKV) * d
        if case["grads"]:  # inputs and outputs' gradients read, outputs and inputs' gradients written
            return {"bytes": values * 8, "flops": 24.0 * values}
        return {"bytes": values * 4 + tokens * HKV * d * 4, "flops": 8.0 * values}
    if case["kind"] == "prefix":
        starts, lengths = _spread(case)
        s, d, hq = case["queries"], case["d"], case["hq"]
        prefix, own_keys = float((case["prefix"] - starts).sum()), float(lengths.sum())
        pairs = prefix * (case["rows"] // case["prompts"]) * s + own_keys * s - case["rows"] * s * (s - 1) / 2
        return {"bytes": (prefix + own_keys) * HKV * d * 4 + case["rows"] * s * hq * d * 4, "flops": 4.0 * pairs * hq * d}
    values, size = case["rows"] * case["vocab"], 4 if case["dtype"] == "fp32" else 2
    return {"bytes": values * size * (2 if case["grads"] else 1) + case["rows"] * (16 + 12 * case["top"]), "flops": (14.0 if case["grads"] else 6.0) * values}


# -------------------------------------------------------------------------------------------------------------------- the definition, in 64 bits


def _exact_rotate(st, case):
    d = case["d"]
    first = torch.arange(0, d, 2, device=DEV) if case["interleaved"] else torch.arange(d // 2, device=DEV)
    second = first + (1 if case["interleaved"] else d // 2)
    pos = torch.arange(case["new"], device=DEV).expand(case["batch"], -1) if st["pos"] is None else st["pos"].long()
    # the rotation of a token as a matrix
    cos, sin = st["table"].double()[pos, :, 0], st["table"].double()[pos, :, 1]
    m = torch.zeros(*pos.shape, d, d, dtype=torch.float64, device=DEV)
    m[:, :, first, first], m[:, :, first, second] = cos, -sin
    m[:, :, second, first], m[:, :, second, second] = sin, cos

    def one(x, gain, dy):
        x = x.double().detach().requires_grad_()
        w = torch.ones(d, dtype=torch.float64, device=DEV) if gain is None else gain.double()
        w.requires_grad_()
        norm = lambda t: t / (t.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt()  # noqa: E731
        turn = lambda t: torch.einsum("bsij,bshj->bshi", m, t)  # noqa: E731
        y = norm(turn(x)) * w if case["after"] else turn(norm(x) * w)
        return (y.detach(), *(torch.autograd.grad(y, (x, w), dy.double()) if dy is not None else (None, None)))

    yq, dq, dgq = one(st["q"], st["gains"][0], st.get("dq"))
    yk, dk, dgk = one(st["k"], st["gains"][1], st.get("dk"))
    if case["grads"]:
        out = {"q": yq, "k": yk, "dq": dq, "dk": dk}
        return {**out, "dgq": dgq, "dgk": dgk} if case["gains"] else out
    kc, vc = st["k_cache"].double(), st["v_cache"].double()
    stop = case["at"] + case["new"]
    kc[:, case["at"] : stop], vc[:, case["at"] : stop] = yk, st["v"].double()
    return {"q": yq, "k": kc, "v": vc}


def _exact_prefix(st, case):
    r, s, hq, d = st["q"].shape
    out = torch.zeros(r, s, hq, d, dtype=torch.float64, device=DEV)
    starts, lengths = st["starts"].tolist(), st["lengths"].tolist()
    for row in range(r):
        prompt = row * case["prompts"] // r
        keys, values = (torch.cat([st[x + "_prefix"][prompt, starts[prompt] :], st[x][row, : lengths[row]]]).double().repeat_interleave(hq // HKV, 1) for x in "kv")
        score = torch.einsum("shd,nhd->hsn", st["q"][row].double(), keys) / math.sqrt(d)
        n = keys.shape[0]
        ahead = torch.arange(n, device=DEV)[None, :] > torch.arange(n - s, n, device=DEV)[:, None]
        out[row] = torch.einsum("hsn,nhd->shd", torch.softmax(score.masked_fill(ahead, -math.inf), -1), values)
    return {"out": out}


def _exact_stats(st, case):
    parts: List[Dict[str, torch.Tensor]] = []
    for r0 in range(0, case["rows"], 256):
        part = slice(r0, r0 + 256)
        x = st["logits"][part].double().requires_grad_(case["grads"])
        dist = torch.log_softmax(x / case["temperature"], -1)
        lp = dist[torch.arange(x.shape[0], device=DEV), st["tokens"][part]]
        h = -torch.where(dist > -math.inf, dist.exp() * dist, 0.0).sum(-1)
        res = {"logprobs": lp.detach(), "entropy": h.detach()}
        loss = (lp * st["d_logprobs"][part] + h * st["d_entropy"][part]).sum() if case["grads"] else None
        if case["top"]:
            best = torch.sort(x.detach(), dim=-1, descending=True, stable=True).indices[:, : case["top"]]
            top = dist.gather(-1, best)
            res.update(top_logprobs=top.detach(), top_tokens=best)
            if case["grads"]:
                loss = loss + (top * st["d_top"][part]).sum()
        if case["grads"]:
            res["dlogits"] = torch.autograd.grad(loss, x)[0]
        parts.append(res)
    return {n: torch.cat([p[n] for p in parts]) for n in parts[0]}


def exact(case: Dict[str, Any], seed: int) -> Optional[Dict[str, torch.Tensor]]:
    st = prepare(case, seed)
    if case["kind"] == "rotate":
        return _exact_rotate(st, case)
    if case["kind"] == "prefix":
        return _exact_prefix(st, case)
    return _exact_stats(st, case)
