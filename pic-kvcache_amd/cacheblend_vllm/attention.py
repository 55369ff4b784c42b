"""Attention on MI355X: of the selected queries, of packed prompts, and of single
tokens over pages of their own type or of 4 bits.

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

import functools

import torch

from . import _native
from .kv_layout import (KVLayer, check_key_weights, check_tables, device_tables, int4_geometry, paged_layer, rows_apart,
                        strides_apart, whole_int32)


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


def _check_out(out: torch.Tensor, query: torch.Tensor) -> None:
    """An output of ``query``'s shape and type whose rows lie apart."""
    if out.shape != query.shape or out.dtype != query.dtype or out.device != query.device:
        raise ValueError(f"out must be {tuple(query.shape)} {query.dtype} on {query.device}")
    if out.stride(-1) != 1:
        raise ValueError("out rows must hold contiguous dims")
    if not rows_apart(out):
        raise ValueError("out rows must not overlap")


def _meets_otherwise(out: torch.Tensor, query: torch.Tensor) -> bool:
    """Whether an output of ``query``'s shape shares memory with it other than element for element."""
    if query.numel() == 0:
        return False
    shape, strides, o_strides = query.shape, query.stride(), out.stride()
    apart, es = out.data_ptr() - query.data_ptr(), query.element_size()
    if apart == 0:
        return any(n > 1 and a != b for n, a, b in zip(shape, strides, o_strides))
    if apart >= es * (1 + sum((n - 1) * a for n, a in zip(shape, strides))) or \
            -apart >= es * (1 + sum((n - 1) * a for n, a in zip(shape, o_strides))):
        return False
    # between each other in one tensor
    return apart % es != 0 or strides != o_strides or not strides_apart((2, *shape), (abs(apart) // es, *strides))


def _prompt_ends(ends: torch.Tensor, tokens: int, name: str, device: torch.device) -> torch.Tensor:
    if ends.dim() != 1 or ends.numel() == 0:
        raise ValueError(f"{name} must be [sequences + 1], got {tuple(ends.shape)}")
    if ends.device.type == "cpu":
        if int(ends[0]) < 0 or int(ends[-1]) > tokens or bool((ends[1:] < ends[:-1]).any()):
            raise IndexError(f"{name} must rise within the {tokens} tokens")
    return whole_int32(ends, device).contiguous()


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


def _check_tokens(query: torch.Tensor) -> None:
    _native.require_device(query, "query")
    if query.dim() not in (3, 4):
        raise ValueError("query must be [batch, q_heads, head_size] or [batch, rows, q_heads, head_size]")
    if query.dtype not in _native.DTYPE_CODES:
        raise ValueError(f"dtype {query.dtype} is not supported")


def _decode_tensors(query, plane, desc, hkv, d, block_tables, context_lens, block_size, out):
    """The checks that attention over pages of any type makes of a step's tensors:
    (batch, rows, query heads, the query's strides, out, its strides, tables, lengths),
    strides of sequences, rows and heads, tables and lengths as the kernels take them."""
    device = query.device
    if plane.device != device:
        raise ValueError(f"query is on {device}, the cache on {plane.device}")
    shape, strides = query.shape, query.stride()
    one = len(shape) == 3  # one token a sequence
    batch, rows, hq = (shape[0], 1, shape[1]) if one else shape[:3]
    if shape[-1] != d:
        raise ValueError(f"query head size {shape[-1]} does not match the pages' {d}")
    if d not in (64, 128):
        raise ValueError(f"head size {d}: 64 or 128 supported")
    if hkv == 0 or hq % hkv or (hq == 0 and batch * rows):
        raise ValueError(f"query heads ({hq}) must be divisible by KV heads ({hkv})")
    if strides[-1] != 1:
        raise ValueError("query rows must hold contiguous dims")
    check_tables(block_tables, context_lens, batch, block_size, desc.num_blocks)
    if out is None:
        # (of a contiguous query in half the time)
        out = torch.empty_like(query) if query.is_contiguous() else torch.empty(shape, dtype=query.dtype, device=device)
    else:
        _check_out(out, query)
    o_strides = out.stride()
    if one:
        strides, o_strides = (strides[0], 0, strides[1]), (o_strides[0], 0, o_strides[1])
    if batch * rows * hq == 0:
        return batch, rows, hq, strides[:3], out, o_strides[:3], None, None
    return batch, rows, hq, strides[:3], out, o_strides[:3], *device_tables(block_tables, context_lens, device)


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
    _check_tokens(query)
    desc, row, plane = paged_layer(kv_layer, block_size)
    hkv, d = int4_geometry(plane.dtype, row)
    batch, rows, hq, q_strides, out, o_strides, tables, lens = _decode_tensors(
        query, plane, desc, hkv, d, block_tables, context_lens, block_size, out)
    device = query.device
    width = block_tables.shape[1]
    if batch * rows * hq == 0:
        return out
    lib = _native.load()
    nbytes = _native.on_device(device, lib.cbk_paged_attention_int4_workspace_bytes, batch, rows, hq, hkv, d,
                               width * block_size, _native.DTYPE_CODES[query.dtype])
    # from torch's allocator on every call: a captured graph then owns its own
    ws = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=device)
    rc = _native.on_device(
        device, lib.cbk_paged_attention_int4, query.data_ptr(), *q_strides, batch, rows, hq,
        desc, hkv, d, tables.data_ptr() if width else None, tables.stride(0), width, lens.data_ptr(), float(scale),
        _native.DTYPE_CODES[query.dtype], out.data_ptr(), *o_strides, ws.data_ptr(), ws.numel(),
        _native.stream_handle(device),
    )
    _native.check(rc, "paged_attention_int4")
    return out


@functools.lru_cache(maxsize=256)  # steps of one shape ask again and again (0.7 us a call)
def _paged_workspace_bytes(device: torch.device, *sizes: int) -> int:
    return max(_native.on_device(device, _native.load().cbk_paged_attention_workspace_bytes, *sizes), 256)


def paged_attention(
    query: torch.Tensor,
    kv_layer: KVLayer,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    block_size: int,
    scale: float,
    out: torch.Tensor | None = None,
    key_weights: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of each sequence's latest tokens over its context in pages of the
    queries' type: a decode step. (Over 4-bit pages: :func:`paged_attention_int4`.)

    ``query`` is ``[batch, q_heads, head_size]``, one token a sequence, or ``[batch,
    rows, q_heads, head_size]``: the last ``rows`` tokens, each of which sees the
    keys up to its own. Key ``k`` of sequence ``b`` is in page ``block_tables[b, k //
    block_size]``; ``context_lens[b]`` counts the keys, those of ``query``'s tokens
    among them (append before attending). Head sizes 64 and 128. ``out`` may be ``query``; where it
    shares memory with it otherwise the queries are copied first. Logits, softmax and sums in
    float32. For the product with the values the softmax's terms are held to
    2^-16 (bf16) or 2^-22 (float16, those below 2^-8 of the largest to 2^-30 of that).

    ``key_weights`` ``[batch, kv_heads, keys]``, float32, at least as many keys as the
    tables hold: to every key of the context is added, in place, what the softmax
    weights of the rows and of the KV head's query heads give it together;
    ``[batch, 1, keys]``: of all heads. Summed over the steps they say which keys
    matter (``kv_layout.evict_paged_kv``). The call then takes scratch for the logits,
    4 bytes for each row, query head and key of the tables; in 16 bits not where a set of weights has
    512 rows (128 a KV head) and many keys, which it multiplies a second time instead. Scratch and
    the split of the work go by the tables' width: best cut to the longest context
    (``block_tables[:, :n]``).

    Lengths on the host are checked, and the tables where both are there
    (``IndexError``). On the device they are not read back: lengths are clamped
    to what a table holds, a page outside the cache holds no keys, and a row that
    sees no key is zero. What a row does not see may hold anything, infinities and
    NaN among it.
    """
    _check_tokens(query)
    desc, row, plane = paged_layer(kv_layer, block_size)
    if out is not None and out.shape == query.shape and out.dtype == query.dtype:
        # the weights may need the queries after the outputs, and a place another place's after its own
        if (key_weights is not None and out.data_ptr() == query.data_ptr()) or _meets_otherwise(out, query):
            query = query.clone()
    if plane.dtype != query.dtype or len(row) != 2:
        raise ValueError(f"the pages hold {plane.dtype} rows {tuple(row)}, the queries are {query.dtype}")
    hkv, d = row
    batch, rows, hq, q_strides, out, o_strides, tables, lens = _decode_tensors(
        query, plane, desc, hkv, d, block_tables, context_lens, block_size, out)
    device = query.device
    width = block_tables.shape[1]
    sets, w = 0, (None, 0, 0)
    if key_weights is not None:
        sets, *strides = check_key_weights(key_weights, batch, hkv, width * block_size, device)
        w = (key_weights.data_ptr(), *strides)
    if batch * rows * hq == 0:
        return out
    lib = _native.load()
    code = _native.DTYPE_CODES[query.dtype]
    nbytes = _paged_workspace_bytes(device, batch, rows, hq, hkv, d, width * block_size, code, sets)
    # from torch's allocator on every call: a captured graph then owns its own
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    rc = _native.on_device(
        device, lib.cbk_paged_attention, query.data_ptr(), *q_strides, batch, rows, hq, desc,
        hkv, d, tables.data_ptr() if width else None, tables.stride(0), width, lens.data_ptr(), float(scale), code,
        out.data_ptr(), *o_strides, *w, sets, ws.data_ptr(), nbytes,
        _native.stream_handle(device),
    )
    _native.check(rc, "paged_attention")
    return out
