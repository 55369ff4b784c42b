"""Decoding from a paged cache of bounded size, as timed cases: single tokens
attend over pages of the model's type, each key's attention weight is summed up
on the way, and the keys with the least of it are evicted from the pages.

A decode step attends from each sequence's latest token, or its last few, over
the sequence's pages (``decode``); with the sums kept for every key and KV head,
or for all heads together, it also adds each key's softmax weights to them
(``weigh``); every so often, or once behind a long prompt, a sequence's pages are
cut down to a budget (``evict``): the first keys, the most recent ones and the
heaviest of the others stay, moved together in their order, each head's own or
the same for all heads. Shapes are those of the Qwen3 layers that bench.py and
the tests use (1.7B: 16 query heads over 8 KV heads; 8B: 32 over 8; 14B: 40 over
8; 30B-A3B: 32 over 4; head size 128) and, in the drawn cases, a head size of 64.
"""

from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def listed() -> list[dict]:
    return [
        # decode steps: one sequence with a short context (latency), one with
        # a long one, a few tokens at a time as a draft's check has them, the
        # accuracy comparisons' type, and an ordinary batch of long contexts
        dict(name="decode_1_of_600", kind="decode", dtype="bf16", batch=1, rows=1, context=600, q_heads=32, heads=8,
             dim=128, block=16),
        dict(name="decode_1_of_32k", kind="decode", dtype="f16", batch=1, rows=1, context=32749, q_heads=32, heads=4,
             dim=128, block=16),
        dict(name="decode_9_of_3k_rows_4", kind="decode", dtype="bf16", batch=9, rows=4, context=2999, q_heads=40,
             heads=8, dim=128, block=16),
        dict(name="decode_f32_5_of_2k", kind="decode", dtype="f32", batch=5, rows=1, context=2047, q_heads=16, heads=8,
             dim=128, block=16),
        dict(name="decode_64_of_16k", kind="decode", dtype="bf16", batch=64, rows=1, context=16384, q_heads=32,
             heads=8, dim=128, block=16),
        # the same with the keys' weights summed up: one short sequence, a
        # batch, and the last tokens of two prompts, whose weights decide what
        # of the prompt stays
        dict(name="weigh_1_of_1000", kind="weigh", dtype="f16", batch=1, rows=1, context=1000, q_heads=16, heads=8,
             dim=128, block=16, shared=False),
        dict(name="weigh_24_of_8k", kind="weigh", dtype="bf16", batch=24, rows=1, context=8192, q_heads=32, heads=8,
             dim=128, block=16, shared=False),
        dict(name="weigh_2_of_8k_rows_32", kind="weigh", dtype="bf16", batch=2, rows=32, context=8000, q_heads=32,
             heads=4, dim=128, block=16, shared=True),
        # evictions: one key of a sequence that outgrew its budget, prompts cut
        # down for each head by itself, float32 pages of 64 tokens, and a batch
        # halved with one choice for all heads
        dict(name="evict_1025_to_1024", kind="evict", dtype="bf16", batch=1, context=1025, keep=1024, first=4,
             recent=64, heads=8, dim=128, block=16, shared=False),
        dict(name="evict_4_of_8k_to_2k", kind="evict", dtype="f16", batch=4, context=8192, keep=2048, first=4,
             recent=32, heads=8, dim=128, block=16, shared=False),
        dict(name="evict_f32_7_of_2k_to_700", kind="evict", dtype="f32", batch=7, context=2000, keep=700, first=0,
             recent=33, heads=4, dim=128, block=64, shared=False),
        dict(name="evict_32_of_8k_to_4k", kind="evict", dtype="bf16", batch=32, context=8192, keep=4096, first=16,
             recent=256, heads=8, dim=128, block=16, shared=True),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["decode", "decode", "weigh", "weigh", "evict", "evict"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    common = dict(kind=kind, dtype=dtype, dim=rng.choice([128, 128, 64]), block=rng.choice([16, 16, 16, 32, 64, 5]))
    q_heads, heads = rng.choice([(16, 8), (32, 8), (40, 8), (32, 4), (8, 2), (6, 1)])
    most = 2 if dtype == "f32" else 4  # the batch's 16K keys, at most
    if kind == "evict":
        batch = _log_int(rng, 1, 32)
        context = _log_int(rng, 40, min(16384, 65536 * most // batch))
        first, recent = rng.choice([0, 1, 4]), rng.choice([0, 8, 16, 32])
        keep = max(first + recent, int(context * rng.uniform(0.05, 1.0)))
        return dict(common, batch=batch, context=context, keep=keep, first=first, recent=recent, heads=heads,
                    shared=rng.choice([False, False, True]))
    batch = _log_int(rng, 1, 64)
    case = dict(common, batch=batch, rows=rng.choice([1, 1, 1, 2, 3, 4]), q_heads=q_heads, heads=heads,
                context=_log_int(rng, 20, min(32768, 65536 * most // batch)))
    if kind == "weigh":
        case["shared"] = rng.choice([False, False, True])
        if rng.random() < 0.25:  # a prompt's last tokens
            case.update(rows=rng.choice([16, 32, 33]), batch=rng.choice([1, 2, 3]), context=_log_int(rng, 100, 8192))
    return case


# ------------------------------------------------------------------ inputs


def _package():
    path = os.path.join(os.getcwd(), "pic-kvcache_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from cacheblend_vllm import attention, kv_layout

    return attention, kv_layout


def _randn(g: torch.Generator, *shape: int, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _lengths(case: dict) -> np.ndarray:
    """Ragged lengths, the first the longest; the same for every seed, so that
    its inputs cost the same."""
    longest = case["context"]
    lens = np.random.default_rng(17).integers(max(1, longest // 4), longest + 1, case["batch"])
    lens[0] = longest
    return lens


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype, heads, dim, block = case["kind"], DTYPES[case["dtype"]], case["heads"], case["dim"], case["block"]
    lens, width = _lengths(case), -(-case["context"] // block)
    # the sequences' pages, in random order
    used = -(-lens // block)
    order = np.random.default_rng(seed).permutation(int(used.sum()) + 8)
    tables = np.zeros((case["batch"], width), dtype=np.int32)
    at = 0
    for i, n in enumerate(used):
        tables[i, :n] = order[at:at + n]
        at += n
    state = dict(case=case, pages=_randn(g, 2, len(order), block, heads, dim, dtype=dtype),
                 tables=torch.from_numpy(tables).cuda(), lens=torch.from_numpy(lens.astype(np.int32)).cuda())
    if kind != "evict":
        # queries that prefer some keys, as a model's do: logits of a standard deviation of 2
        state["query"] = (2 * _randn(g, case["batch"], case["rows"], case["q_heads"], dim)).to(dtype)
    if kind != "decode":
        # sums over a few steps before: most keys light, a few heavy, some that no step looked at
        sums = torch.exp(1.5 * _randn(g, case["batch"], 1 if case["shared"] else heads, width * block))
        state["weights"] = torch.where(sums > 0.4, 4.0 / case["context"] * sums, 0.0)
    return state


# ------------------------------------------------- a pass, in its plain form


def _attend(state: dict):
    """The rows' outputs, and what their softmax weights add up to for each key and KV head."""
    case, query, tables, lens = state["case"], state["query"], state["tables"], state["lens"]
    rows, heads = case["rows"], case["heads"]
    pages = state["pages"][:, tables.long()].flatten(2, 3)  # [2, batch, keys, heads, dim]
    q = query.float().unflatten(2, (heads, -1)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [batch, heads, group * rows, dim]
    k = pages[0].float().permute(0, 2, 3, 1).contiguous()
    logits = torch.matmul(q, k).mul_(case["dim"] ** -0.5).unflatten(2, (-1, rows))
    # the rows are the context's last tokens
    last = lens[:, None] - rows + torch.arange(rows, device="cuda")
    seen = torch.arange(k.shape[3], device="cuda") <= last[..., None]
    logits.masked_fill_(~seen[:, None, None], -math.inf)
    top = logits.amax(dim=-1, keepdim=True).clamp_min(torch.finfo(logits.dtype).min)
    p = logits.sub_(top).exp_()
    p.div_(p.sum(dim=-1, keepdim=True).clamp_min(1e-30))  # a row that sees nothing stays zero
    p = p.flatten(2, 3)
    out = torch.matmul(p, pages[1].float().transpose(1, 2).contiguous())
    out = out.unflatten(2, (-1, rows)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return out.to(query.dtype), p


def _evict(state: dict):
    case, pages, tables, lens = state["case"], state["pages"], state["tables"].long(), state["lens"].long()
    block, weights = case["block"], state["weights"]
    batch, sets, places = weights.shape
    at = torch.arange(places, device="cuda")
    n, keep = lens[:, None, None], lens.clamp_max(case["keep"])[:, None, None]
    always = (at < case["first"]) | (at >= n - case["recent"]) | (n <= case["keep"])
    # what stays always before the others, by weight, and what lies behind the context last
    order = torch.where(at < n, torch.where(always, math.inf, weights), -math.inf)
    rank = order.sort(dim=-1, descending=True, stable=True).indices
    kept = torch.zeros_like(rank, dtype=torch.bool).scatter_(2, rank, (at < keep).expand_as(rank))
    source = torch.where(kept, at, places).sort(dim=-1).values  # the kept keys in their order, then `places`
    b, m, to = (source < places).nonzero(as_tuple=True)
    at_from = source[b, m, to]
    new_weights = torch.where(at < n, 0.0, weights)
    new_weights[b, m, to] = weights[b, m, at_from]
    per_set = pages.flatten(1, 2).unflatten(2, (sets, -1))  # [2, slots, sets, heads of a set, dim]
    slot = lambda i: tables[b, i // block] * block + i % block  # noqa: E731
    per_set[:, slot(to), m] = per_set[:, slot(at_from), m]
    return {"lens": keep.flatten().int(), "weights": new_weights, "pages": pages}


def run(state: dict):
    case, kind = state["case"], state["case"]["kind"]
    if not own:
        if kind == "evict":
            return _evict(state)
        out, p = _attend(state)
        if kind == "decode":
            return out
        added = p.sum(dim=2)
        state["weights"].add_(added.sum(dim=1, keepdim=True) if case["shared"] else added)
        return {"out": out, "weights": state["weights"]}
    attention, kv_layout = _package()
    if kind == "evict":
        weights = state["weights"].clone()  # a pass leaves the sums to the next one on the same state
        lens = kv_layout.evict_paged_kv(state["pages"], state["tables"], state["lens"], case["block"], weights,
                                        case["keep"], first=case["first"], recent=case["recent"])
        return {"lens": lens, "weights": weights, "pages": state["pages"]}
    out = attention.paged_attention(state["query"], state["pages"], state["tables"], state["lens"], case["block"],
                                    case["dim"] ** -0.5, key_weights=state.get("weights"))
    return out if kind == "decode" else {"out": out, "weights": state["weights"]}


# ----------------------------------------------------- work and exact values


def work(case: dict) -> dict:
    es, dim, heads, lens = BYTES[case["dtype"]], case["dim"], case["heads"], _lengths(case).astype(np.int64)
    total = int(lens.sum())
    # tables and lengths, and the sums of each key read and written once
    rest = 4 * int((-(-lens // case["block"])).sum()) + 4 * len(lens)
    if case["kind"] != "decode":
        rest += 8 * total * (1 if case["shared"] else heads)
    if case["kind"] != "evict":
        return {"bytes": total * 2 * heads * dim * es + 2 * case["batch"] * case["rows"] * case["q_heads"] * dim * es + rest,
                "flops": 4 * case["rows"] * case["q_heads"] * dim * total}
    # rows behind the first evicted key move: of N keys that may go E go, and
    # before the first of them lie (N - E) / (E + 1) in the mean
    gone = np.maximum(lens - case["keep"], 0)
    free = np.maximum(lens - case["first"] - case["recent"], 0)
    moved = np.where(gone > 0, case["keep"] - case["first"] - (free - gone) / (gone + 1), 0)
    return {"bytes": int(np.maximum(moved, 0).sum()) * 4 * heads * dim * es + rest, "flops": total}


def _exact_attend(case: dict, state: dict):
    rows, heads, dim, block = case["rows"], case["heads"], case["dim"], case["block"]
    group = case["q_heads"] // heads
    out = torch.zeros(state["query"].shape, dtype=torch.float64, device="cuda")
    weights = state["weights"].double() if case["kind"] == "weigh" else None
    for b, n in enumerate(state["lens"].tolist()):
        held = state["pages"][:, state["tables"][b, :-(-n // block)].long()].flatten(1, 2)[:, :n].double()
        for i in range(rows):
            seen = n - rows + 1 + i
            if seen <= 0:
                continue
            q = state["query"][b, i].double().reshape(heads, group, dim)
            p = torch.softmax(torch.bmm(q, held[0, :seen].permute(1, 2, 0).contiguous()) * dim ** -0.5, dim=-1)
            out[b, i] = torch.bmm(p, held[1, :seen].permute(1, 0, 2).contiguous()).reshape(-1, dim)
            if weights is not None:
                weights[b, :, :seen] += p.sum(dim=(0, 1)) if case["shared"] else p.sum(dim=1)
    return out if weights is None else {"out": out, "weights": weights}


def _exact_evict(case: dict, state: dict):
    block, first, recent = case["block"], case["first"], case["recent"]
    pages, weights, tables = state["pages"].double(), state["weights"].double(), state["tables"].long()
    sets = weights.shape[1]
    size = case["heads"] // sets
    lens = []
    for b, n in enumerate(state["lens"].tolist()):
        lens.append(min(n, case["keep"]))
        if n <= case["keep"]:
            continue
        slots = (tables[b][:, None] * block + torch.arange(block, device="cuda")).flatten()[:n]
        rows = pages.flatten(1, 2)[:, slots]
        for m in range(sets):
            middle = weights[b, m, first:n - recent].cpu().numpy()
            best = np.lexsort((np.arange(len(middle)), -middle))[:case["keep"] - first - recent]
            stay = np.concatenate([np.arange(first), first + np.sort(best), np.arange(n - recent, n)])
            stay = torch.from_numpy(stay).cuda()
            pages.flatten(1, 2)[:, slots[:len(stay)], m * size:(m + 1) * size] = rows[:, stay, m * size:(m + 1) * size]
            mine = weights[b, m, :n].clone()
            weights[b, m, :n] = 0
            weights[b, m, :len(stay)] = mine[stay]
    return {"lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "weights": weights, "pages": pages}


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    return _exact_evict(case, state) if case["kind"] == "evict" else _exact_attend(case, state)
