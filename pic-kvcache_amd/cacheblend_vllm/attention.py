"""Attention on MI355X: of the selected queries, of packed prompts, and of single
tokens over 4-bit pages.

``blend_attention`` keeps the signature of ``Qwen3BlendExecutor._attention``
(cacheblend_vllm/ascend.py:798-846): queries ``[Nq, Hq, D]`` at absolute
positions ``q_positions`` attend causally (key ``k`` visible iff ``k <=
q_positions[i]``) to the layer buffer's keys/values ``[Nk, Hkv, D]`` with GQA
head sharing. It runs in ``cbk_blend_attention``: a flash-style MFMA kernel
that evaluates the mask in place (so the reference's cached
``[1, 1, Nq, Nk]`` mask, ``state.attention_mask``, is never built) and rounds
the logits as the reference's bf16/f16 einsum and ``* scale`` do.
"""

from __future__ import annotations

import torch

from . import _native
from .kv_layout import KVLayer, int4_geometry, paged_layer, rows_apart


def blend_attention(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    q_positions: torch.Tensor,
    scale: float,
    state=None,
) -> torch.Tensor:
    """Reference ascend.py:798-846 (``state`` is accepted for the signature;
    the mask needs no cache here). Returns ``[Nq, Hq, D]`` in the input dtype."""
    for name, t in (("query", query), ("key", key), ("value", value)):
        _native.require_device(t, name)
        if t.dim() != 3:
            raise ValueError(f"{name} must be [tokens, heads, head_size]")
        if t.stride(2) != 1 or t.stride(1) != t.shape[2]:
            raise ValueError(f"{name} rows must hold contiguous heads")
    nq, hq, d = query.shape
    nk, hkv, dk = key.shape
    if value.shape != key.shape or dk != d:
        raise ValueError("key/value shapes do not match the query head size")
    if key.dtype != query.dtype or value.dtype != query.dtype:
        raise ValueError("query, key and value must share a dtype")
    if query.dtype not in _native.DTYPE_CODES:
        raise ValueError(f"dtype {query.dtype} is not supported")
    if hq % hkv:
        raise ValueError(f"query heads ({hq}) must be divisible by KV heads ({hkv})")
    if q_positions.numel() != nq:
        raise ValueError(f"{q_positions.numel()} positions for {nq} queries")
    if q_positions.device.type == "cpu" and nq:
        lo, hi = int(q_positions.min()), int(q_positions.max())
        if lo < 0 or hi >= nk:
            raise IndexError(f"query positions in [{lo}, {hi}] outside the {nk} keys")
    pos = q_positions.to(device=query.device, dtype=torch.int64).contiguous()
    out = torch.empty((nq, hq, d), dtype=query.dtype, device=query.device)
    if nq == 0:
        return out
    lib = _native.load()
    # partial results of the keys' ranges, from torch's allocator on every
    # call: a captured graph then owns its own
    dtype_code = _native.DTYPE_CODES[query.dtype]
    # (under 256 keys every call takes one range: 0.7 us less of the host)
    nbytes = lib.cbk_blend_attention_workspace_bytes(nq, nk, hq, hkv, d, dtype_code) if nk >= 256 else 0
    ws = None
    if nbytes:
        try:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=query.device)
        except torch.cuda.OutOfMemoryError:
            nbytes = 0  # one range, which needs no scratch
    rc = lib.cbk_blend_attention_ws(
        query.data_ptr(), query.stride(0), pos.data_ptr(), nq,
        key.data_ptr(), key.stride(0), value.data_ptr(), value.stride(0), nk, hq, hkv, d,
        float(scale), dtype_code, out.data_ptr(), out.stride(0),
        _native.ptr(ws), nbytes, _native.stream_handle(query.device),
    )
    _native.check(rc, "blend_attention")
    return out


def _whole_int32(t: torch.Tensor, device: torch.device) -> torch.Tensor:
    """Whole numbers as int32 on ``device``; what int32 does not hold stays out of range."""
    if t.dtype != torch.int32:
        if t.dtype.is_floating_point or t.dtype.is_complex or t.dtype == torch.bool:
            raise ValueError(f"whole numbers expected, got {t.dtype}")
        if t.dtype in (torch.int64, torch.uint32, torch.uint64):
            t = t.to(torch.int64).clamp(-1, (1 << 31) - 1)
    return t if t.dtype == torch.int32 and t.device == device else t.to(device=device, dtype=torch.int32)


def _check_out(out: torch.Tensor, query: torch.Tensor) -> None:
    """An output of ``query``'s shape and type whose rows lie apart."""
    if out.shape != query.shape or out.dtype != query.dtype or out.device != query.device:
        raise ValueError(f"out must be {tuple(query.shape)} {query.dtype} on {query.device}")
    if out.stride(-1) != 1:
        raise ValueError("out rows must hold contiguous dims")
    if not rows_apart(out):
        raise ValueError("out rows must not overlap")


def _prompt_ends(ends: torch.Tensor, tokens: int, name: str, device: torch.device) -> torch.Tensor:
    if ends.dim() != 1 or ends.numel() == 0:
        raise ValueError(f"{name} must be [sequences + 1], got {tuple(ends.shape)}")
    if ends.device.type == "cpu":
        if int(ends[0]) < 0 or int(ends[-1]) > tokens or bool((ends[1:] < ends[:-1]).any()):
            raise IndexError(f"{name} must rise within the {tokens} tokens")
    return _whole_int32(ends, device).contiguous()


def _pieces(t: torch.Tensor, es: int, strided: bool = False) -> bool:
    """16-byte aligned rows of whole dims; ``strided``: tokens within 2^24 elements."""
    return (t.stride(2) == 1 and (t.data_ptr() | t.stride(0) * es | t.stride(1) * es) % 16 == 0
            and not (strided and t.stride(0) >= 1 << 24))


def prompt_attention(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    cu_seqlens: torch.Tensor,
    scale: float,
    cu_seqlens_k: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Causal attention of packed prompts: a prefill.

    ``query`` ``[tokens, q_heads, head_size]``, ``key`` and ``value`` ``[tokens,
    kv_heads, head_size]`` hold the sequences one after another, sequence ``s`` from
    ``cu_seqlens[s]`` to ``cu_seqlens[s + 1]`` (with ``cu_seqlens_k``, keys and values
    from ``cu_seqlens_k[s]`` to ``cu_seqlens_k[s + 1]``). A sequence's last query is its
    last key: with more keys than queries the first keys are context from before
    (a chunk of a longer prompt), with fewer the first queries see nothing and are
    zero. Head sizes 64 and 128; logits, softmax and sums in float32. For the product
    with the values the softmax's terms are rounded to the inputs' type (float16: terms
    below 2^-14 of the largest of the first 32 keys' to 2^-25 of that, none below);
    float32 terms and products hold 24 bits.

    Tokens before the first sequence and behind the last (padding) are zero in a
    new output and left as they are in ``out``. What a query does not see may hold
    anything, infinities and NaN among it. Rows that are not 16-byte aligned are
    copied first.

    ``cu_seqlens`` on the host is checked (``IndexError``); on the device it is not
    read back: ends past the tensors are taken as their end, and ends that fall,
    which no batch has, leave ``out``'s rows undefined (nothing else is touched).
    """
    for name, t in (("query", query), ("key", key), ("value", value)):
        _native.require_device(t, name)
        if t.dim() != 3:
            raise ValueError(f"{name} must be [tokens, heads, head_size]")
    total, hq, d = query.shape
    total_k, hkv, dk = key.shape
    if value.shape != key.shape or dk != d:
        raise ValueError("key/value shapes do not match the query head size")
    if key.dtype != query.dtype or value.dtype != query.dtype:
        raise ValueError("query, key and value must share a dtype")
    device = query.device
    if key.device != device or value.device != device:
        raise ValueError("query, key and value must share a device")
    if query.dtype not in _native.DTYPE_CODES:
        raise ValueError(f"dtype {query.dtype} is not supported")
    if d not in (64, 128):
        raise ValueError(f"head size {d}: 64 or 128 supported")
    if hkv == 0 or hq == 0 or hq % hkv:
        raise ValueError(f"query heads ({hq}) must be divisible by KV heads ({hkv})")
    if cu_seqlens_k is None and total_k != total:
        raise ValueError(f"{total_k} keys for {total} queries need cu_seqlens_k")
    ends_q = _prompt_ends(cu_seqlens, total, "cu_seqlens", device)
    ends_k = ends_q if cu_seqlens_k is None else _prompt_ends(cu_seqlens_k, total_k, "cu_seqlens_k", device)
    batch = ends_q.numel() - 1
    if ends_k.numel() != batch + 1:
        raise ValueError(f"{ends_k.numel()} ends of keys for {batch + 1} of queries")
    fresh = out is None
    if fresh:
        out = torch.empty((total, hq, d), dtype=query.dtype, device=device)
    else:
        _check_out(out, query)
    if total == 0 or batch == 0:
        return out.zero_() if fresh else out
    es = query.element_size()
    copied = {"memory_format": torch.contiguous_format}
    q = query if _pieces(query, es) else query.clone(**copied)
    k = key if _pieces(key, es, True) else key.clone(**copied)
    v = value if _pieces(value, es, True) else value.clone(**copied)
    o = out if _pieces(out, es) else out.clone(**copied)
    lib = _native.load()
    # partial results of the keys' ranges, from torch's allocator on every
    # call: a captured graph then owns its own
    code = _native.DTYPE_CODES[query.dtype]
    nbytes = _native.on_device(device, lib.cbk_prompt_attention_workspace_bytes, total, total_k, batch, hq, hkv, d, code)
    ws = None
    if nbytes:
        try:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        except torch.cuda.OutOfMemoryError:
            nbytes = 0  # one range, which needs no scratch
    rc = _native.on_device(
        device, lib.cbk_prompt_attention, q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
        v.data_ptr(), v.stride(0), v.stride(1), ends_q.data_ptr(), ends_k.data_ptr(), batch, total, total_k, hq, hkv, d,
        float(scale), code, o.data_ptr(), o.stride(0), o.stride(1), int(fresh), _native.ptr(ws), nbytes,
        _native.stream_handle(device),
    )
    _native.check(rc, "prompt_attention")
    if o is not out:
        out.copy_(o)
    return out


def paged_attention_int4(
    query: torch.Tensor,
    kv_layer: KVLayer,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    block_size: int,
    scale: float,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of each sequence's latest tokens over its context in 4-bit pages
    (``kv_layout.append_paged_kv`` to a ``uint8`` layer): a decode step.

    ``query`` is ``[batch, q_heads, head_size]``, one token a sequence, or ``[batch,
    rows, q_heads, head_size]``: the last ``rows`` tokens, each of which sees the
    keys up to its own. Key ``k`` of sequence ``b`` is in page ``block_tables[b, k //
    block_size]``; ``context_lens[b]`` counts the keys, those of ``query``'s tokens
    among them (append before attending). Head sizes 64 and 128; logits, softmax
    and sums in float32, whatever the queries' type: 16-bit queries enter the first
    product exactly, or to 2^-36 of their row's largest element, the softmax's terms
    the second to 2^-16 of themselves (float32: 2^-23).

    Lengths on the host are checked, and the tables where both are there
    (``IndexError``). On the device they are not read back: lengths are clamped
    to what a table holds, a page outside the cache holds no keys, and a row that
    sees no key is zero.
    """
    _native.require_device(query, "query")
    if query.dim() not in (3, 4):
        raise ValueError("query must be [batch, q_heads, head_size] or [batch, rows, q_heads, head_size]")
    if query.dtype not in _native.DTYPE_CODES:
        raise ValueError(f"dtype {query.dtype} is not supported")
    desc, row, plane = paged_layer(kv_layer, block_size)
    hkv, d = int4_geometry(plane.dtype, row)
    device = query.device
    if plane.device != device:
        raise ValueError(f"query is on {device}, the cache on {plane.device}")
    q = query if query.dim() == 4 else query.unsqueeze(1)
    batch, rows, hq = q.shape[:3]
    if q.shape[3] != d:
        raise ValueError(f"query head size {q.shape[3]} does not match the pages' {d}")
    if d not in (64, 128):
        raise ValueError(f"head size {d}: 64 or 128 supported")
    if hkv == 0 or hq % hkv or (hq == 0 and batch * rows):
        raise ValueError(f"query heads ({hq}) must be divisible by KV heads ({hkv})")
    if q.stride(3) != 1:
        raise ValueError("query rows must hold contiguous dims")
    if block_tables.dim() != 2 or block_tables.shape[0] != batch or context_lens.numel() != batch:
        raise ValueError(f"{tuple(block_tables.shape)} block tables and {context_lens.numel()} lengths for {batch} sequences")
    width = block_tables.shape[1]
    if context_lens.device.type == "cpu" and batch:
        lo, hi = int(context_lens.min()), int(context_lens.max())
        if lo < 0 or hi > width * block_size:
            raise IndexError(f"context lengths in [{lo}, {hi}] outside the {width} blocks of {block_size}")
        if block_tables.device.type == "cpu":
            used = torch.arange(width) * block_size < context_lens.reshape(-1, 1)
            pages = block_tables[used]
            if pages.numel() and (int(pages.min()) < 0 or int(pages.max()) >= desc.num_blocks):
                raise IndexError(f"block tables hold pages outside [0, {desc.num_blocks})")
    if out is None:
        out = torch.empty(query.shape, dtype=query.dtype, device=device)
    else:
        _check_out(out, query)
    if batch * rows * hq == 0:
        return out
    tables = _whole_int32(block_tables, device)
    if width and tables.stride(1) != 1:
        tables = tables.contiguous()
    lens = _whole_int32(context_lens, device)
    if not lens.is_contiguous():
        lens = lens.contiguous()
    o = out if out.dim() == 4 else out.unsqueeze(1)
    lib = _native.load()
    nbytes = _native.on_device(device, lib.cbk_paged_attention_int4_workspace_bytes, batch, rows, hq, hkv, d,
                               width * block_size, _native.DTYPE_CODES[query.dtype])
    # from torch's allocator on every call: a captured graph then owns its own
    ws = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=device)
    rc = _native.on_device(
        device, lib.cbk_paged_attention_int4, q.data_ptr(), q.stride(0), q.stride(1), q.stride(2), batch, rows, hq,
        desc, hkv, d, tables.data_ptr() if width else None, tables.stride(0), width, lens.data_ptr(), float(scale),
        _native.DTYPE_CODES[query.dtype], o.data_ptr(), o.stride(0), o.stride(1), o.stride(2), ws.data_ptr(), ws.numel(),
        _native.stream_handle(device),
    )
    _native.check(rc, "paged_attention_int4")
    return out
