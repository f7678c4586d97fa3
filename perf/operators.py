"""Attention over long contexts with a bounded cache, operator by operator: a key/value cache that is quantised as it is written and read back, attention of
single tokens over that cache, and attention with a sliding window and a few first tokens that stay visible.

``run`` is one pass through an operator, in elementary torch operations or, with ``own``, by the calls that a user makes.  A quantised cache keeps, per row of one
token and head, ``d`` codes of 4 or 8 bits and ``d / 32`` bf16 scales.  Seen as ``[4, d / 32, 8]``, a row's channels with the same middle index share a scale, so
that a quarter of the row holds eight channels of every group.  The scale is the group's value of largest magnitude (the first of equals) divided by
``-2^(bits - 1)``, the code of that value therefore ``-2^(bits - 1)`` itself, and every other one the nearest that exists.  Codes are stored with ``2^(bits - 1)`` added, of 4 bits
two to a byte, the even channel in the low half.  Rows of a head lie one behind the other: ``[batch, heads, slots, ...]``.

Head counts are those of the Llama-3 decoders that the recipes serve: 32 query heads on 8 key heads of 128 channels (8B) or 64 (1B)."""
from __future__ import annotations

import math
from typing import Any, Dict, List, Optional, Tuple

import torch

own = False

DEV = "cuda"
HQ, HKV = 32, 8


def listed() -> List[Dict[str, Any]]:
    return [
        # Decoding: the new token of 16 rollouts enters the cache (the smallest write; launches count).
        dict(name="append_token", kind="append", bits=4, batch=16, new=1, at=731, slots=1024, d=128),
        # A long prompt enters the cache and is read back for its own attention: the largest write and read.
        dict(name="append_long_prompt", kind="append", bits=4, batch=2, new=8000, at=0, slots=8192, d=128),
        # Prompts of an instruction data set, in 8 bits, 64 channels per head, an odd length behind an odd start (a second turn).
        dict(name="append_turn_8bit", kind="append", bits=8, batch=8, new=333, at=117, slots=1024, d=64),
        # One short chat turn: a single token over 61 cached ones, the smallest attention.
        dict(name="attend_chat", kind="attend", bits=4, batch=1, queries=1, keys=61, slots=64, d=64, mask="last", window=0, sinks=0),
        # Rollouts of left-padded prompts in a cache that is not full: a boolean mask, as generation hands it over.
        dict(name="attend_rollouts", kind="attend", bits=4, batch=16, queries=1, keys=732, slots=1024, d=128, mask="bool", window=0, sinks=0),
        # One long document: few rows, so the keys have to be split.
        dict(name="attend_document", kind="attend", bits=4, batch=1, queries=1, keys=65003, slots=65536, d=128, mask="last", window=0, sinks=0),
        # Many rollouts of long answers: the largest cache.
        dict(name="attend_batch", kind="attend", bits=4, batch=64, queries=1, keys=4096, slots=4096, d=128, mask="last", window=0, sinks=0),
        # Three drafted tokens at once over a cache in 8 bits, 64 channels per head.
        dict(name="attend_draft_8bit", kind="attend", bits=8, batch=16, queries=3, keys=4111, slots=4352, d=64, mask="last", window=0, sinks=0),
        # Endless chat: a window of the newest tokens and four first ones out of a long 4-bit cache.
        dict(name="attend_window", kind="attend", bits=4, batch=8, queries=1, keys=16001, slots=16384, d=128, mask="last", window=2048, sinks=4),
        # The same on an unquantised cache.
        dict(name="window_token", kind="window", batch=8, queries=1, keys=8012, d=128, window=2048, sinks=4, doc=0),
        # Fine-tuning with that mask, forward and backward: one long document, heads of 128 channels; the largest case.
        dict(name="window_train_8b", kind="window", batch=1, queries=6000, keys=6000, d=128, window=1024, sinks=4, doc=0),
        # Packed documents of odd lengths, heads of 64 channels, forward and backward: each document keeps its own first tokens.
        dict(name="window_train_1b_packed", kind="window", batch=4, queries=1413, keys=1413, d=64, window=200, sinks=3, doc=611),
    ]


def _log(rng, low: int, high: int) -> int:
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng) -> Dict[str, Any]:
    kind = rng.choice(["append", "attend", "attend", "window"])
    d = rng.choice([64, 128])
    if kind == "append":
        bits = rng.choice([4, 8])
        new = rng.choice([1, _log(rng, 2, 8000)])
        batch = _log(rng, 1, max(1, min(64, 16000 // new)))
        at = rng.choice([0, _log(rng, 1, 4000)])
        return dict(kind=kind, bits=bits, batch=batch, new=new, at=at, slots=at + new + rng.randint(0, 200), d=d)
    if kind == "attend":
        keys = _log(rng, 1, 65000)
        batch = _log(rng, 1, max(1, min(64, 260000 // keys)))
        mask = rng.choice(["last", "last", "bool"])
        window = rng.choice([0, 0, _log(rng, 1, 4096)]) if mask == "last" else 0
        queries = rng.choice([1, 1, rng.randint(1, min(4, keys))])
        return dict(kind=kind, bits=rng.choice([4, 4, 8]), batch=batch, queries=queries, keys=keys, slots=keys + rng.randint(0, 100), d=d, mask=mask, window=window,
                    sinks=rng.randint(1, 16) if window else 0)
    window, sinks = _log(rng, 16, 4096), rng.randint(1, 64)
    if rng.random() < 0.3:
        keys = _log(rng, 1, 20000)
        return dict(kind=kind, batch=_log(rng, 1, max(1, min(32, 64000 // keys))), queries=1, keys=keys, d=d, window=window, sinks=sinks, doc=0)
    keys = _log(rng, 33, 5500)
    return dict(kind=kind, batch=_log(rng, 1, max(1, min(8, 20_000_000 // keys**2))), queries=keys, keys=keys, d=d, window=window, sinks=sinks,
                doc=rng.choice([0, _log(rng, 16, max(17, keys))]))


# ------------------------------------------------------------------------------------------------------------------------------- plain forms


def _groups(x: torch.Tensor) -> torch.Tensor:
    return x.view(*x.shape[:-1], 4, x.shape[-1] // 32, 8)


def _quantize(x: torch.Tensor, bits: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Codes (one per channel, with 2^(bits - 1) added) and bf16 scales of the rows of ``x``."""
    half = 2 ** (bits - 1)
    g = _groups(x.float()).transpose(-3, -2).flatten(-2)  # [..., group, 32], channels in order
    first = g.abs().max(-1, keepdim=True).indices  # the first of equals
    scale = (g.gather(-1, first).squeeze(-1) / -half).to(torch.bfloat16)
    s = scale.float()[..., None]
    code = torch.where((s != 0) & s.isfinite(), g / s, torch.zeros_like(g)).round().clamp(-half, half - 1) + half
    code = code.unflatten(-1, (4, 8)).transpose(-3, -2).reshape(x.shape).to(torch.uint8)
    return code, scale


def _pack(code: torch.Tensor, bits: int) -> torch.Tensor:
    return code if bits == 8 else code[..., 0::2] | code[..., 1::2] << 4


def _values(codes: torch.Tensor, scales: torch.Tensor, bits: int) -> torch.Tensor:
    c = codes if bits == 8 else torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    v = _groups(c.float() - 2 ** (bits - 1)) * scales.float()[..., None, :, None]
    return v.view(c.shape)


def _visible(case: Dict[str, Any], doc_ids: Optional[torch.Tensor], device) -> torch.Tensor:
    """``[batch or 1, queries, keys]``: the queries are the last of the keys, a key is at or before its query, and inside the window or among the first of its document."""
    i = torch.arange(case["queries"], device=device).view(1, -1, 1) + case["keys"] - case["queries"]
    j = torch.arange(case["keys"], device=device).view(1, 1, -1)
    seen = j <= i
    first = torch.zeros_like(j)
    if doc_ids is not None:
        same = doc_ids[:, :, None] == doc_ids[:, None, :]
        seen, first = seen & same, same.int().argmax(-1)[:, None, :]
    if case["window"]:
        seen = seen & ((i - j < case["window"]) | (j - first < case["sinks"]))
    return seen


def _attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, seen: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``q`` [b, queries, hq, d], ``k``, ``v`` [b, hkv, keys, d] in 32 bits → output like ``q`` and weights [b, hkv, group, queries, keys]."""
    b, s, hq, d = q.shape
    qh = q.view(b, s, k.shape[1], -1, d).permute(0, 2, 3, 1, 4)
    score = (qh @ k.transpose(-1, -2).unsqueeze(2)).mul_(d**-0.5).masked_fill_(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top.isfinite(), top, torch.zeros_like(top))).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total > 0, total, torch.ones_like(total)))
    return (p @ v.unsqueeze(2)).permute(0, 3, 1, 2, 4).reshape(b, s, hq, d), p


# ------------------------------------------------------------------------------------------------------------------------------------- cases


def _rows(g: torch.Generator, *shape: int, spread: float = 0.0) -> torch.Tensor:
    """Random rows; ``spread``: how much the channels differ in size, as those of keys do."""
    x = torch.randn(*shape, generator=g, device=DEV)
    if spread:
        x = x * torch.exp(spread * torch.randn(shape[-2], shape[-1], generator=g, device=DEV))
    return x.to(torch.bfloat16)


def _slots_for(slots: int) -> int:
    return -(-slots // 32) * 32


def _documents(g: torch.Generator, batch: int, length: int, mean: int) -> torch.Tensor:
    """Document ids of packed rows; documents have about ``mean`` tokens."""
    starts = torch.rand(batch, length, generator=g, device=DEV) < 1.0 / mean
    starts[:, 0] = False
    return starts.cumsum(1).to(torch.int32)


def prepare(case: Dict[str, Any], seed: int) -> Dict[str, Any]:
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind, d = case["kind"], case["d"]
    state: Dict[str, Any] = {"case": case}
    if kind == "window":
        b, s, n = case["batch"], case["queries"], case["keys"]
        state.update(q=_rows(g, b, s, HQ, d), k=_rows(g, b, n, HKV, d, spread=0.3), v=_rows(g, b, n, HKV, d))
        state["docs"] = _documents(g, b, n, case["doc"]) if case["doc"] else None
        if s == n:
            state["dout"] = _rows(g, b, s, HQ, d)
        return state
    b, slots = case["batch"], _slots_for(case["slots"])
    if kind == "append":
        # the projections leave keys and values side by side in one row
        kv = _rows(g, b, case["new"], 2 * HKV, d, spread=0.3)
        state.update(k=kv[:, :, :HKV], v=kv[:, :, HKV:], slots=torch.arange(case["at"], case["at"] + case["new"], device=DEV))
        for n in "kv":
            state[n + "_codes"] = torch.zeros(b, HKV, slots, d * case["bits"] // 8, dtype=torch.uint8, device=DEV)
            state[n + "_scales"] = torch.zeros(b, HKV, slots, d // 32, dtype=torch.bfloat16, device=DEV)
        return state
    state["q"] = _rows(g, b, case["queries"], HQ, d)
    for n in "kv":
        state[n + "_codes"] = torch.zeros(b, HKV, slots, d * case["bits"] // 8, dtype=torch.uint8, device=DEV)
        state[n + "_scales"] = torch.zeros(b, HKV, slots, d // 32, dtype=torch.bfloat16, device=DEV)
        code, scale = _quantize(_rows(g, b, case["keys"], HKV, d, spread=0.3 if n == "k" else 0.0).transpose(1, 2), case["bits"])
        state[n + "_codes"][:, :, : case["keys"]] = _pack(code, case["bits"])
        state[n + "_scales"][:, :, : case["keys"]] = scale
    state["mask"] = None
    if case["mask"] == "bool":  # left-padded rows, slots that are not filled yet
        start = (torch.rand(b, 1, 1, generator=g, device=DEV) * case["keys"] * 0.6).long()
        j = torch.arange(slots, device=DEV)
        i = torch.arange(case["queries"], device=DEV).view(1, -1, 1) + case["keys"] - case["queries"]
        state["mask"] = (j >= start) & (j <= i)
    return state


def run(state: Dict[str, Any]) -> Dict[str, torch.Tensor]:
    case = state["case"]
    return {"append": _run_append, "attend": _run_attend, "window": _run_window}[case["kind"]](state, case)


def _run_append(st, case):
    first, last = case["at"], case["at"] + case["new"]
    if own:
        from torchtune_b200 import ops

        k_rows, v_rows = ops.QuantizedRows(st["k_codes"], st["k_scales"]), ops.QuantizedRows(st["v_codes"], st["v_scales"])
        ops.quantized_append(st["k"], st["v"], k_rows, v_rows, st["slots"])
        k, v = ops.quantized_read(k_rows, v_rows, first, last)
        return {"k": k, "v": v}
    code, scale = _quantize(torch.stack([st["k"], st["v"]]).transpose(2, 3), case["bits"])
    code = _pack(code, case["bits"])
    st["k_codes"][:, :, st["slots"]], st["v_codes"][:, :, st["slots"]] = code[0], code[1]
    st["k_scales"][:, :, st["slots"]], st["v_scales"][:, :, st["slots"]] = scale[0], scale[1]
    k, v = (_values(st[n + "_codes"][:, :, first:last], st[n + "_scales"][:, :, first:last], case["bits"]).transpose(1, 2) for n in "kv")
    return {"k": k.to(torch.bfloat16).contiguous(), "v": v.to(torch.bfloat16).contiguous()}


def _run_attend(st, case):
    if own:
        from torchtune_b200 import ops

        k_rows, v_rows = ops.QuantizedRows(st["k_codes"], st["k_scales"]), ops.QuantizedRows(st["v_codes"], st["v_scales"])
        if st["mask"] is not None:
            mask = ops.AttentionMask(causal=False, bool_mask=st["mask"])
        else:
            mask = ops.AttentionMask(causal=True, window=case["window"], sinks=case["sinks"])
            k_rows, v_rows = k_rows.first(case["keys"]), v_rows.first(case["keys"])
        return {"out": ops.quantized_attention(st["q"], k_rows, v_rows, mask)}
    n = case["keys"] if st["mask"] is None else st["mask"].shape[-1]
    k, v = (_values(st[x + "_codes"][:, :, :n], st[x + "_scales"][:, :, :n], case["bits"]) for x in "kv")
    seen = _visible(case, None, DEV) if st["mask"] is None else st["mask"]
    return {"out": _attention(st["q"].float(), k, v, seen)[0].to(torch.bfloat16)}


def _run_window(st, case):
    q, k, v = st["q"], st["k"], st["v"]
    if own:
        from torchtune_b200 import ops

        mask = ops.AttentionMask(causal=True, window=case["window"], sinks=case["sinks"], doc_ids=st["docs"])
        if "dout" not in st:
            with torch.no_grad():
                return {"out": ops.attention(q, k, v, mask)}
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = ops.attention(*leaves, mask)
        grads = torch.autograd.grad(out, leaves, st["dout"])
        return {"out": out.detach(), "dq": grads[0], "dk": grads[1], "dv": grads[2]}
    seen = _visible(case, st["docs"], DEV)
    kf, vf = k.float().transpose(1, 2), v.float().transpose(1, 2)
    out, p = _attention(q.float(), kf, vf, seen)
    if "dout" not in st:
        return {"out": out.to(torch.bfloat16)}
    # dV = Pᵀ dO, dS = P (dO Vᵀ - rowsum(dO o O)), dQ = dS K / sqrt(d), dK = dSᵀ Q / sqrt(d); a key head's gradients sum over its query heads
    b, s, hq, d = q.shape
    do = st["dout"].float()
    split = lambda t: t.reshape(b, s, HKV, -1, d).permute(0, 2, 3, 1, 4)  # noqa: E731
    delta = (split(do) * split(out)).sum(-1, keepdim=True)
    dv = (p.transpose(-1, -2) @ split(do)).sum(2)
    ds = (split(do) @ vf.unsqueeze(2).transpose(-1, -2)).sub_(delta).mul_(p).mul_(d**-0.5)
    del p
    dq = (ds @ kf.unsqueeze(2)).permute(0, 3, 1, 2, 4).reshape(b, s, hq, d)
    dk = (ds.transpose(-1, -2) @ split(q.float())).sum(2)
    bf = torch.bfloat16
    return {"out": out.to(bf), "dq": dq.to(bf), "dk": dk.transpose(1, 2).to(bf), "dv": dv.transpose(1, 2).to(bf)}


def _pairs(case: Dict[str, Any]) -> int:
    """Visible pairs of a query and a key of one batch row (documents: by their mean length)."""
    total, length = 0, case["keys"]
    docs = [length] if not case.get("doc") else [min(case["doc"], length)] * max(1, length // case["doc"])
    for n in docs:
        w = case["window"] or n
        for i in range(max(0, n - case["queries"]), n):
            total += min(i + 1, w + (min(case["sinks"], max(0, i + 1 - w)) if case["window"] else 0))
    return total


def work(case: Dict[str, Any]) -> Dict[str, float]:
    b, d = case["batch"], case["d"]
    if case["kind"] == "append":  # new keys and values read, codes and scales written, what they stand for returned
        values = 2 * b * case["new"] * HKV * d
        return {"bytes": values * (2 + case["bits"] / 8 + 1 / 16 + 2), "flops": 4 * values}
    pairs = _pairs(case)
    flops = 4.0 * b * pairs * HQ * d
    reach = min(case["keys"], case["window"] + case["queries"] - 1 + case["sinks"]) if case["window"] else case["keys"]
    out = 2 * b * case["queries"] * HQ * d * 2
    if case["kind"] == "attend":
        return {"bytes": 2 * b * reach * HKV * d * (case["bits"] / 8 + 1 / 16) + out, "flops": flops}
    if case["queries"] < case["keys"] or case["keys"] == 1:
        return {"bytes": 2 * b * reach * HKV * d * 2 + out, "flops": flops}
    # forward, and five products of the same size backward; q, k, v, dO read, O and three gradients written
    return {"bytes": 2 * out + 2 * (2 * b * case["keys"] * HKV * d * 2), "flops": flops * 3.5}


# -------------------------------------------------------------------------------------------------------------------- the definition, in 64 bits


def _stored64(x: torch.Tensor, bits: int) -> torch.Tensor:
    """What a cache stands for after rows ``x`` have been written to it."""
    half = 2.0 ** (bits - 1)
    out, quarter = torch.zeros(x.shape, dtype=torch.float64, device=x.device), x.shape[-1] // 4
    for j in range(x.shape[-1] // 32):
        at = torch.cat([torch.arange(t * quarter + 8 * j, t * quarter + 8 * j + 8, device=x.device) for t in range(4)])
        part = x.double()[..., at]
        big = part.abs().amax(-1, keepdim=True)
        place = torch.where(part.abs() == big, torch.arange(32, device=x.device), 32).amin(-1, keepdim=True)
        step = torch.gather(part, -1, place).div(-half).to(torch.bfloat16).double()
        code = torch.where(step == 0, torch.zeros_like(part), part / torch.where(step == 0, torch.ones_like(step), step))
        out[..., at] = torch.clamp(torch.round(code), -half, half - 1) * step
    return out


def _rows64(codes: torch.Tensor, scales: torch.Tensor, bits: int, d: int) -> torch.Tensor:
    out, quarter = torch.empty(*codes.shape[:-1], d, dtype=torch.float64, device=codes.device), d // 4
    for c in range(d):
        raw = codes[..., c] if bits == 8 else (codes[..., c // 2] >> (4 * (c % 2))) % 16
        out[..., c] = (raw.double() - 2.0 ** (bits - 1)) * scales[..., (c % quarter) // 8].double()
    return out


def exact(case: Dict[str, Any], seed: int) -> Optional[Dict[str, torch.Tensor]]:
    st = prepare(case, seed)
    if case["kind"] == "append":
        return {"k": _stored64(st["k"], case["bits"]), "v": _stored64(st["v"], case["bits"])}
    q = st["q"].double()
    b, s, hq, d = q.shape
    group, n = hq // HKV, case["keys"]
    grads = case["kind"] == "window" and "dout" in st
    names = ("out", "dq", "dk", "dv") if grads else ("out",)
    res = {x: torch.zeros(st[{"out": "q", "dq": "q", "dk": "k", "dv": "v"}[x]].shape, dtype=torch.float64, device=DEV) for x in names}
    i, j = torch.arange(s, device=DEV)[:, None] + n - s, torch.arange(n, device=DEV)[None, :]
    for r in range(b):
        if case["kind"] == "attend" and st["mask"] is not None:
            seen = st["mask"][r]
            width = seen.shape[-1]
        else:
            seen, width = j <= i, n
            start = torch.zeros(n, dtype=torch.long, device=DEV)
            docs = st.get("docs")
            if docs is not None:
                seen = seen & (docs[r][:, None] == docs[r][None, :])
                start = torch.searchsorted(docs[r].contiguous(), docs[r].contiguous())
            if case["window"]:
                seen = seen & ((j > i - case["window"]) | (j < start[None, :] + case["sinks"]))
        for h in range(HKV):
            if case["kind"] == "attend":
                k, v = (_rows64(st[x + "_codes"][r, h, :width], st[x + "_scales"][r, h, :width], case["bits"], d) for x in "kv")
            else:
                k, v = st["k"][r, :, h].double(), st["v"][r, :, h].double()
            for x in range(h * group, (h + 1) * group):
                score = (q[r, :, x] @ k.T / math.sqrt(d)).masked_fill(~seen, -math.inf)
                p = torch.nan_to_num(torch.softmax(score, -1))
                o = p @ v
                res["out"][r, :, x] = o
                if grads:
                    do = st["dout"][r, :, x].double()
                    ds = p * (do @ v.T - (do * o).sum(-1, keepdim=True)) / math.sqrt(d)
                    res["dq"][r, :, x] = ds @ k
                    res["dk"][r, :, h] += ds.T @ q[r, :, x]
                    res["dv"][r, :, h] += p.T @ do
    return res
