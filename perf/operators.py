"""A request's own keys and values, as timed cases: appended to the paged cache
with the rotation applied on the way, held there in the model's type or in 4
bits, read back, and attended to by whole prompts and by single tokens.

A prefill appends the prompt's rows to the pages (``append``; ``append4`` for
4-bit pages, followed by the read-back that a store or a blend makes of them)
and attends causally within each packed prompt (``prompt``); a later request
reads stored 4-bit rows (``gather4``); a decode step appends one token a
sequence and attends over the 4-bit pages (``decode4``). Shapes are those of
the Qwen3 layers that bench.py and the tests use (1.7B: 16 query heads over 8
KV heads; 8B: 32 over 8; 14B: 40 over 8; 30B-A3B: 32 over 4; head size 128)
and, in the drawn cases, a head size of 64.

A 4-bit row holds, per head, the 4-bit codes of its dims (dim 2i in the low
half of byte i), then for every 32 dims a bf16 step and a bf16 offset; a dim's
value is offset + step * code.
"""

from __future__ import annotations

import math
import os
import sys
from types import SimpleNamespace

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
BLOCK = 16   # tokens per vLLM block
GROUP = 32   # dims that share a step and an offset
POSITIONS = 40960  # rows of the rotary table


def listed() -> list[dict]:
    return [
        # one decoded token of an 8B layer into the pages: latency
        dict(name="append_1", kind="append", dtype="bf16", tokens=1, q_heads=32, heads=8, dim=128, neox=True),
        # the rows of an 8K prefill batch of the same layer
        dict(name="append_8k", kind="append", dtype="bf16", tokens=8192, q_heads=32, heads=8, dim=128, neox=True),
        # a batch of 61 decoded tokens, and an 8K prefill, into 4-bit pages;
        # then their read-back
        dict(name="append4_61", kind="append4", dtype="f16", tokens=61, q_heads=16, heads=8, dim=128, neox=False),
        dict(name="append4_8k", kind="append4", dtype="bf16", tokens=8192, q_heads=32, heads=8, dim=128, neox=True),
        # stored 4-bit rows of a short prompt and of a long one, read back
        dict(name="gather4_333", kind="gather4", dtype="f16", tokens=333, heads=8, dim=128),
        dict(name="gather4_65k", kind="gather4", dtype="bf16", tokens=65531, heads=4, dim=128),
        # decode steps: one sequence with a short context, one with a long
        # one, and an ordinary batch of ragged contexts
        dict(name="decode4_1_of_700", kind="decode4", dtype="bf16", batch=1, rows=1, context=700, q_heads=32,
             heads=8, dim=128),
        dict(name="decode4_1_of_32k", kind="decode4", dtype="f16", batch=1, rows=1, context=32749, q_heads=32,
             heads=4, dim=128),
        dict(name="decode4_64_of_16k", kind="decode4", dtype="bf16", batch=64, rows=1, context=16384, q_heads=32,
             heads=8, dim=128),
        # prefills: one short prompt, an ordinary batch of packed prompts
        # in float32 (the accuracy comparisons' type), and a long batch
        dict(name="prompt_509", kind="prompt", dtype="f16", prompts=1, longest=509, q_heads=32, heads=8, dim=128),
        dict(name="prompt_f32_4_of_1k", kind="prompt", dtype="f32", prompts=4, longest=1024, q_heads=16, heads=8,
             dim=128),
        dict(name="prompt_3_of_8k", kind="prompt", dtype="bf16", prompts=3, longest=8192, q_heads=32, heads=8,
             dim=128),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["append", "append4", "gather4", "decode4", "decode4", "decode4", "prompt", "prompt", "prompt"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    dim = rng.choice([128, 128, 64])
    q_heads, heads = rng.choice([(16, 8), (32, 8), (40, 8), (32, 4), (8, 2)])
    if kind in ("append", "append4"):
        return dict(kind=kind, dtype=dtype, tokens=_log_int(rng, 1, 8192), q_heads=q_heads, heads=heads, dim=dim,
                    neox=rng.choice([True, True, False]))
    if kind == "gather4":
        return dict(kind=kind, dtype=dtype, tokens=_log_int(rng, 1, 32768), heads=heads, dim=dim)
    if kind == "decode4":
        batch = _log_int(rng, 1, 64)
        return dict(kind=kind, dtype=dtype, batch=batch, rows=rng.choice([1, 1, 1, 2, 3, 4]),
                    context=_log_int(rng, 20, min(32768, 16384 * 64 // batch)), q_heads=q_heads, heads=heads, dim=dim)
    if dtype == "f32":
        prompts, q_heads, heads = rng.choice([1, 2, 4]), *rng.choice([(16, 8), (8, 2)])
        return dict(kind=kind, dtype=dtype, prompts=prompts, longest=_log_int(rng, 5, 1024), q_heads=q_heads,
                    heads=heads, dim=dim)
    prompts = _log_int(rng, 1, 24)
    q_heads, heads = rng.choice([(16, 8), (32, 8), (32, 4), (8, 2)])
    return dict(kind=kind, dtype=dtype, prompts=prompts, longest=_log_int(rng, 5, min(8192, 24576 // prompts)),
                q_heads=q_heads, heads=heads, dim=dim)


# ------------------------------------------------------------------ inputs


def _package():
    path = os.path.join(os.getcwd(), "pic-kvcache_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from cacheblend_vllm import attention, kv_layout

    return attention, kv_layout


def _rope(dim: int, neox: bool) -> SimpleNamespace:
    """What the append reads of a model's rotary embedding."""
    inv = 1.0 / (1e6 ** (torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim))
    angle = torch.arange(POSITIONS, dtype=torch.float64, device="cuda")[:, None] * inv
    return SimpleNamespace(head_size=dim, rotary_dim=dim, is_neox_style=neox,
                           cos_sin_cache=torch.cat([angle.cos(), angle.sin()], dim=-1).float())


def _randn(g: torch.Generator, *shape: int, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _slots(seed: int, blocks: int, tokens: int) -> torch.Tensor:
    order = np.random.default_rng(seed).permutation(blocks)
    slots = (order[:, None] * BLOCK + np.arange(BLOCK)[None, :]).reshape(-1)[:tokens]
    return torch.from_numpy(slots).cuda()


def _row_bytes(dim: int) -> int:
    return dim // GROUP * (GROUP // 2 + 4)


def _pages4(g: torch.Generator, blocks: int, heads: int, dim: int) -> torch.Tensor:
    """One layer of 4-bit pages [2, blocks, BLOCK, heads, row bytes]: uniform
    codes, steps around the ~0.27 of 32 N(0, 1) values, offsets half their
    range below zero."""
    groups = dim // GROUP
    lead = (2, blocks, BLOCK, heads)
    codes = torch.randint(0, 256, (*lead, dim // 2), generator=g, device="cuda", dtype=torch.uint8)
    step = (0.27 * torch.exp(0.2 * _randn(g, *lead, groups))).bfloat16()
    offset = (step.float() * (-7.5 + _randn(g, *lead, groups))).bfloat16()
    both = torch.stack([step, offset], dim=-1).flatten(-2).view(torch.uint8)
    return torch.cat([codes, both], dim=-1)


def _lengths(seed: int, count: int, longest: int) -> np.ndarray:
    """Ragged lengths, the first the longest."""
    lens = np.random.default_rng(seed).integers(max(1, longest // 4), longest + 1, count)
    lens[0] = longest
    return lens


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype, heads, dim = case["kind"], DTYPES[case["dtype"]], case["heads"], case["dim"]
    state = dict(kind=kind, dtype=dtype, scale=dim ** -0.5)
    if kind in ("append", "append4"):
        n, q_heads = case["tokens"], case["q_heads"]
        # as many pages again as the tokens fill, in random order
        blocks = 2 * ((n + BLOCK - 1) // BLOCK) + 8
        # the projection's output rows: queries, keys and values side by side
        qkv = _randn(g, n, q_heads + 2 * heads, dim, dtype=dtype)
        start = int(np.random.default_rng(seed).integers(0, POSITIONS - n))
        if kind == "append":
            pages = _randn(g, 2, blocks, BLOCK, heads, dim, dtype=dtype)
        else:
            pages = _pages4(g, blocks, heads, dim)
        return dict(state, pages=pages, query=qkv[:, :q_heads], key=qkv[:, q_heads:q_heads + heads],
                    value=qkv[:, q_heads + heads:], slots=_slots(seed, blocks, n), rope=_rope(dim, case["neox"]),
                    positions=torch.arange(start, start + n, device="cuda"))
    if kind == "gather4":
        n = case["tokens"]
        blocks = (n + BLOCK - 1) // BLOCK + 8
        return dict(state, pages=_pages4(g, blocks, heads, dim), slots=_slots(seed, blocks, n))
    if kind == "decode4":
        # one set of lengths per size, so that every seed's inputs cost the same
        lens = _lengths(17, case["batch"], case["context"])
        per = (case["context"] + BLOCK - 1) // BLOCK
        blocks = int(((lens + BLOCK - 1) // BLOCK).sum()) + 8
        order = np.random.default_rng(seed).permutation(blocks)
        tables = np.zeros((case["batch"], per), dtype=np.int32)
        at = 0
        for i, n in enumerate((lens + BLOCK - 1) // BLOCK):
            tables[i, :n] = order[at:at + n]
            at += n
        query = _randn(g, case["batch"], case["rows"], case["q_heads"], dim, dtype=dtype)
        return dict(state, pages=_pages4(g, blocks, heads, dim), query=query,
                    tables=torch.from_numpy(tables).cuda(), lens=torch.from_numpy(lens.astype(np.int32)).cuda())
    lens = _lengths(17, case["prompts"], case["longest"])
    total = int(lens.sum())
    ends = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    return dict(state, query=_randn(g, total, case["q_heads"], dim, dtype=dtype),
                key=_randn(g, total, heads, dim, dtype=dtype), value=_randn(g, total, heads, dim, dtype=dtype),
                ends=torch.from_numpy(ends).cuda(), longest=case["longest"])


# ------------------------------------------------- a pass, in its plain form


def _turn(x: torch.Tensor, rope, positions: torch.Tensor, real: torch.dtype = torch.float32) -> torch.Tensor:
    """Rotated rows [tokens, heads, dim]."""
    x = x.to(real)
    cos, sin = rope.cos_sin_cache[positions][:, None].to(real).chunk(2, dim=-1)
    half = x.shape[-1] // 2
    a, b = (x[..., :half], x[..., half:]) if rope.is_neox_style else (x[..., 0::2], x[..., 1::2])
    a, b = a * cos - b * sin, b * cos + a * sin
    return torch.cat([a, b], dim=-1) if rope.is_neox_style else torch.stack([a, b], dim=-1).flatten(-2)


def _codes(x: torch.Tensor) -> torch.Tensor:
    """64-bit rows [..., dim] (values lie on the codes' borders) as 4-bit rows
    [..., row bytes]: the offset is the lowest value, rounded down to bf16, the
    step a 15th of the rest, rounded to float32 and up to bf16; a code is the
    nearest whole number to the rest times the step's float32 inverse."""
    x = x.unflatten(-1, (-1, GROUP))
    low, high = x.amin(dim=-1, keepdim=True), x.amax(dim=-1, keepdim=True)
    near = low.float()
    near = torch.where(near.double() > low, near.nextafter(torch.full_like(near, -math.inf)), near)
    bits = near.view(torch.int32)
    offset = (torch.where(near < 0, bits + 0xffff, bits) & -0x10000).view(torch.float32)
    step = ((high - offset) / 15).float()
    step = ((step.view(torch.int32) + 0xffff) & -0x10000).view(torch.float32)
    inverse = (1 / step.double()).float()
    code = torch.where(step > 0, torch.round((x - offset) * inverse), 0.0).clamp(0, 15)
    code = code.to(torch.uint8).flatten(-2)
    both = torch.cat([step, offset], dim=-1).bfloat16().flatten(-2).view(torch.uint8)
    return torch.cat([code[..., 0::2] | code[..., 1::2] << 4, both], dim=-1)


def _values(rows: torch.Tensor, dim: int, real: torch.dtype = torch.float32) -> torch.Tensor:
    """The values [..., dim] that 4-bit rows [..., row bytes] stand for."""
    codes, both = rows[..., :dim // 2], rows[..., dim // 2:].contiguous().view(torch.bfloat16).to(real)
    code = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).to(real).unflatten(-1, (-1, GROUP))
    return (both[..., 1::2, None] + both[..., 0::2, None] * code).flatten(-2)


def _append(state: dict):
    query = _turn(state["query"], state["rope"], state["positions"]).to(state["dtype"])
    flat = state["pages"].flatten(1, 2)
    if state["kind"] == "append":
        flat[0][state["slots"]] = _turn(state["key"], state["rope"], state["positions"]).to(state["dtype"])
        flat[1][state["slots"]] = state["value"]
        return {"query": query, "pages": state["pages"]}
    flat[0][state["slots"]] = _codes(_turn(state["key"], state["rope"], state["positions"], torch.float64))
    flat[1][state["slots"]] = _codes(state["value"].double())
    return {"query": query, "rows": _gather4(state)}


def _gather4(state: dict) -> torch.Tensor:
    rows = state["pages"].flatten(1, 2)[:, state["slots"]]
    return _values(rows, rows.shape[-1] // (GROUP // 2 + 4) * GROUP).to(state["dtype"])


def _softmax(logits: torch.Tensor) -> torch.Tensor:
    """Along the last dimension, in place; a row of -inf only becomes zero."""
    top = logits.amax(dim=-1, keepdim=True).clamp_min(torch.finfo(logits.dtype).min)
    p = logits.sub_(top).exp_()
    return p.div_(p.sum(dim=-1, keepdim=True).clamp_min(1e-30))


def _decode4(state: dict) -> torch.Tensor:
    query, tables, lens = state["query"], state["tables"], state["lens"]
    batch, rows, q_heads, dim = query.shape
    pages = state["pages"][:, tables.long()].flatten(2, 3)  # [2, batch, keys, heads, bytes]
    heads, keys = pages.shape[3], pages.shape[2]
    q = query.float().unflatten(2, (heads, -1)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [batch, heads, group * rows, dim]
    k = _values(pages[0], dim).permute(0, 2, 3, 1).contiguous()
    logits = torch.matmul(q, k).mul_(state["scale"]).unflatten(2, (-1, rows))
    # the rows are the context's last tokens
    last = lens[:, None] - rows + torch.arange(rows, device="cuda")
    seen = torch.arange(keys, device="cuda") <= last[..., None]
    p = _softmax(logits.masked_fill_(~seen[:, None, None], -math.inf)).flatten(2, 3)
    out = torch.matmul(p, _values(pages[1], dim).transpose(1, 2).contiguous())
    return out.unflatten(2, (-1, rows)).permute(0, 3, 1, 2, 4).flatten(2, 3).to(state["dtype"])


def _prompt(state: dict) -> torch.Tensor:
    query, key, value, ends, longest = (state[k] for k in ("query", "key", "value", "ends", "longest"))
    heads, dim = key.shape[1:]
    lens = ends[1:] - ends[:-1]
    at = torch.arange(longest, device="cuda")
    # every prompt padded to the longest: [prompts, longest, ...]
    place = (ends[:-1, None] + at).clamp_max(query.shape[0] - 1).long()
    q = query[place].float().unflatten(2, (heads, -1)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    k = key[place].float().permute(0, 2, 3, 1).contiguous()
    logits = torch.matmul(q, k).mul_(state["scale"]).unflatten(2, (-1, longest))
    hidden = (at[None, :] > at[:, None]) | (at >= lens[:, None, None])  # [prompts, query, key]
    p = _softmax(logits.masked_fill_(hidden[:, None, None], -math.inf)).flatten(2, 3)
    out = torch.matmul(p, value[place].float().transpose(1, 2).contiguous())
    out = out.unflatten(2, (-1, longest)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return out[at < lens[:, None]].to(state["dtype"])


def run(state: dict):
    kind = state["kind"]
    if not own:
        return {"append": _append, "append4": _append, "gather4": _gather4, "decode4": _decode4,
                "prompt": _prompt}[kind](state)
    attention, kv_layout = _package()
    if kind == "prompt":
        return attention.prompt_attention(state["query"], state["key"], state["value"], state["ends"], state["scale"])
    if kind == "decode4":
        return attention.paged_attention_int4(state["query"], state["pages"], state["tables"], state["lens"], BLOCK,
                                              state["scale"])
    if kind == "gather4":
        return kv_layout.gather_paged_kv_int4(state["pages"], state["slots"], BLOCK, state["dtype"])
    query = kv_layout.append_paged_kv(state["key"], state["value"], state["pages"], state["slots"], BLOCK,
                                      positions=state["positions"], rotary_emb=state["rope"], query=state["query"])
    if kind == "append":
        return {"query": query, "pages": state["pages"]}
    return {"query": query, "rows": kv_layout.gather_paged_kv_int4(state["pages"], state["slots"], BLOCK,
                                                                   state["dtype"])}


# ----------------------------------------------------- work and exact values


def work(case: dict) -> dict:
    kind, es, heads, dim = case["kind"], BYTES[case["dtype"]], case["heads"], case["dim"]
    row, row4 = 2 * heads * dim * es, 2 * heads * _row_bytes(dim)  # a token's K and V
    if kind == "append":
        # inputs, slot, position and table row in; query and pages out
        n, q_row = case["tokens"], case["q_heads"] * dim * es
        return {"bytes": n * (2 * q_row + 2 * row + 16 + 4 * dim), "flops": 3 * n * (case["q_heads"] + heads) * dim}
    if kind == "append4":
        # the same with 4-bit rows, and the read-back
        n, q_row = case["tokens"], case["q_heads"] * dim * es
        return {"bytes": n * (2 * q_row + 2 * row + 2 * row4 + 24 + 4 * dim),
                "flops": n * (3 * case["q_heads"] + 17 * heads) * dim}
    if kind == "gather4":
        return {"bytes": case["tokens"] * (row + row4 + 8), "flops": 4 * case["tokens"] * heads * dim}
    q_heads = case["q_heads"]
    if kind == "decode4":
        total, rows = int(_lengths(17, case["batch"], case["context"]).sum()), case["rows"]
        return {"bytes": total * row4 + 2 * case["batch"] * rows * q_heads * dim * es + 4 * (total // BLOCK),
                "flops": 4 * rows * q_heads * dim * total}
    lens = _lengths(17, case["prompts"], case["longest"]).astype(np.int64)
    total, pairs = int(lens.sum()), int((lens * (lens + 1) // 2).sum())
    return {"bytes": total * (2 * q_heads * dim * es + row), "flops": 4 * q_heads * dim * pairs}


def _exact_rows(state: dict, case: dict):
    """Rotated queries and keys in 64 bits, as complex numbers times e^(i angle)."""
    rope, dim = state["rope"], case["dim"]
    table = rope.cos_sin_cache.double()[state["positions"]]
    turn = torch.complex(table[:, :dim // 2], table[:, dim // 2:])[:, None]

    def turned(x):
        x = x.double()
        pairs = torch.complex(x[..., :dim // 2], x[..., dim // 2:]) if rope.is_neox_style else \
            torch.view_as_complex(x.reshape(*x.shape[:-1], dim // 2, 2))
        pairs = pairs * turn
        if rope.is_neox_style:
            return torch.cat([pairs.real, pairs.imag], dim=-1)
        return torch.view_as_real(pairs).reshape(x.shape)

    return turned(state["query"]), turned(state["key"])


def _exact_held(x: torch.Tensor) -> torch.Tensor:
    """What 4-bit rows of the 64-bit rows x stand for."""

    def rounded(v, up):  # the next bfloat16 at or above (below)
        near = v.bfloat16()
        past = near.double() < v if up else near.double() > v
        return torch.where(past, near.nextafter(torch.full_like(near, math.inf if up else -math.inf)), near).double()

    parts = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    offset = rounded(parts.min(dim=-1, keepdim=True).values, False)
    step = rounded(((parts.max(dim=-1, keepdim=True).values - offset) / 15).float().double(), True)
    code = ((parts - offset) * step.reciprocal().float().double()).nan_to_num(0.0).round().clamp(0, 15)
    return (offset + step * code).reshape(x.shape)


def _exact_read(rows: torch.Tensor, dim: int) -> torch.Tensor:
    """4-bit rows [..., row bytes] as 64-bit values."""
    groups = dim // GROUP
    pairs = rows[..., :dim // 2].to(torch.int16)
    code = torch.empty(*rows.shape[:-1], dim, dtype=torch.float64, device=rows.device)
    code[..., 0::2], code[..., 1::2] = pairs % 16, pairs // 16
    words = rows[..., dim // 2:].to(torch.int32)
    bits = (words[..., 0::2] + 256 * words[..., 1::2]) << 16
    real = bits.view(torch.float32).double().reshape(*rows.shape[:-1], groups, 2)
    return code * real[..., 0].repeat_interleave(GROUP, dim=-1) + real[..., 1].repeat_interleave(GROUP, dim=-1)


def _exact_decode(state: dict, case: dict) -> torch.Tensor:
    rows, dim, group = case["rows"], case["dim"], case["q_heads"] // case["heads"]
    out = torch.zeros(state["query"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(state["lens"].tolist()):
        blocks = state["tables"][b, :(n + BLOCK - 1) // BLOCK].long()
        held = _exact_read(state["pages"][:, blocks].flatten(1, 2)[:, :n], dim)  # [2, n, heads, dim]
        for i in range(rows):
            seen = n - rows + 1 + i
            if seen <= 0:
                continue
            q = state["query"][b, i].double().reshape(case["heads"], group, dim)
            k = held[0, :seen].permute(1, 2, 0).contiguous()
            p = torch.softmax(torch.bmm(q, k) * state["scale"], dim=-1)
            out[b, i] = torch.bmm(p, held[1, :seen].permute(1, 0, 2).contiguous()).reshape(-1, dim)
    return out


def _exact_prompt(state: dict, case: dict) -> torch.Tensor:
    group = case["q_heads"] // case["heads"]
    out = torch.empty(state["query"].shape, dtype=torch.float64, device="cuda")
    ends = state["ends"].tolist()
    for lo, hi in zip(ends[:-1], ends[1:]):
        later = torch.ones(hi - lo, hi - lo, dtype=torch.bool, device="cuda").triu(1)
        for h in range(case["q_heads"]):
            k = state["key"][lo:hi, h // group].double().t().contiguous()
            logits = (state["query"][lo:hi, h].double() @ k) * state["scale"]
            p = torch.softmax(logits.masked_fill_(later, -math.inf), dim=1)
            out[lo:hi, h] = p @ state["value"][lo:hi, h // group].double().contiguous()
    return out


def exact(case: dict, seed: int):
    state, kind, dim = prepare(case, seed), case["kind"], case["dim"]
    if kind == "prompt":
        return _exact_prompt(state, case)
    if kind == "decode4":
        return _exact_decode(state, case)
    if kind == "gather4":
        return _exact_read(state["pages"].flatten(1, 2)[:, state["slots"]], dim)
    query, key = _exact_rows(state, case)
    if kind == "append4":
        return {"query": query, "rows": torch.stack([_exact_held(key), _exact_held(state["value"].double())])}
    pages = state["pages"].double()
    pages.flatten(1, 2)[:, state["slots"]] = torch.stack([key, state["value"].double()])
    return {"query": query, "pages": pages}
