"""The operators over a request's own keys and values, in 64 bits with numpy:
rotation to a position, 4-bit rows, attention of single tokens and of packed
prompts. TEST INFRASTRUCTURE ONLY, as the rest of this package."""

from __future__ import annotations

import numpy as np

GROUP = 32


def rotate(x: np.ndarray, cos_sin: np.ndarray, positions: np.ndarray, neox: bool) -> np.ndarray:
    """``x`` [T, H, D] with its first ``cos_sin.shape[1]`` dims turned to the positions."""
    x = np.asarray(x, dtype=np.float64)
    n = cos_sin.shape[1]
    table = np.asarray(cos_sin, dtype=np.float64)[np.asarray(positions)][:, None]
    c, s = table[..., :n // 2], table[..., n // 2:]
    out = x.copy()
    a, b = (np.s_[..., :n // 2], np.s_[..., n // 2:n]) if neox else (np.s_[..., 0:n:2], np.s_[..., 1:n:2])
    out[a] = x[a] * c - x[b] * s
    out[b] = x[b] * c + x[a] * s
    return out


def rotate_terms(x: np.ndarray, cos_sin: np.ndarray, positions: np.ndarray, neox: bool) -> np.ndarray:
    """The sum of the absolute terms of :func:`rotate`'s values: their rounding's scale."""
    n = cos_sin.shape[1]
    half = np.concatenate([np.abs(cos_sin[:, :n // 2]), -np.abs(cos_sin[:, n // 2:])], axis=1)
    first = rotate(np.abs(x), half, positions, neox)   # |x c| + |y s|, |y c| - |x s|
    half[:, n // 2:] *= -1
    second = rotate(np.abs(x), half, positions, neox)  # |x c| - |y s|, |y c| + |x s|
    return np.maximum(first, second)


def _bf16_down(x: np.ndarray) -> np.ndarray:
    """The highest bf16 value not above ``x`` (64 bits)."""
    with np.errstate(over="ignore"):
        f = x.astype(np.float32)
    f = np.where(f.astype(np.float64) > x, np.nextafter(f, np.float32(-np.inf)), f).astype(np.float32)
    bits = f.view(np.uint32).astype(np.uint64)
    bits = np.where(f < 0, bits + 0xffff, bits) & 0xffff0000
    return bits.astype(np.uint32).view(np.float32)


def int4_encode(x: np.ndarray) -> np.ndarray:
    """4-bit rows [..., D / 32 * 20] uint8 of 64-bit rows [..., D]."""
    x = np.asarray(x, dtype=np.float64)
    d = x.shape[-1]
    parts = x.reshape(*x.shape[:-1], d // GROUP, GROUP)
    with np.errstate(all="ignore"):
        finite = np.isfinite(parts).all(axis=-1, keepdims=True)
        offset = _bf16_down(parts.min(axis=-1, keepdims=True))
        step = ((parts.max(axis=-1, keepdims=True) - offset) / 15).astype(np.float32)
        step = ((step.view(np.uint32) + np.uint32(0xffff)) & np.uint32(0xffff0000)).view(np.float32)
        step = np.where(step < np.float32(2.0 ** -126), np.float32(0), step)
        inverse = np.where(step > 0, np.float32(1) / step, np.float32(0)).astype(np.float64)
        good = finite & np.isfinite(offset)
        code = np.clip(np.rint((parts - offset) * inverse), 0, 15)
        code = np.where(good & (inverse > 0), code, 0).astype(np.uint8).reshape(*x.shape[:-1], d)
        nan = np.uint32(0x7fc00000).view(np.float32)
        both = np.concatenate([np.where(good, step, nan), np.where(good, offset, nan)], axis=-1).astype(np.float32)
    words = (both.view(np.uint32) >> 16).astype(np.uint16).reshape(*x.shape[:-1], d // GROUP * 2)
    return np.concatenate([code[..., 0::2] | code[..., 1::2] << 4, words.view(np.uint8)], axis=-1)


def int4_decode(rows: np.ndarray) -> np.ndarray:
    """The values [..., D] (64 bits) of 4-bit rows."""
    groups = rows.shape[-1] // (GROUP // 2 + 4)
    d = groups * GROUP
    code = np.empty((*rows.shape[:-1], d), dtype=np.float64)
    code[..., 0::2], code[..., 1::2] = rows[..., :d // 2] & 15, rows[..., :d // 2] >> 4
    words = np.ascontiguousarray(rows[..., d // 2:]).view(np.uint16).astype(np.uint32) << 16
    both = words.view(np.float32).astype(np.float64).reshape(*rows.shape[:-1], groups, 2)
    return both[..., 1].repeat(GROUP, axis=-1) + both[..., 0].repeat(GROUP, axis=-1) * code


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, last: np.ndarray, scale: float):
    """Rows ``q`` [N, Hq, D] over keys and values [M, H, D], row i up to key
    ``last[i]`` (below 0: none, a zero row); returns the outputs, and sum p |v|."""
    n, hq, d = q.shape
    m, h, _ = k.shape
    out, mass = np.zeros((n, hq, d)), np.zeros((n, hq, d))
    hidden = np.arange(m)[None, :] > np.asarray(last)[:, None]
    rows = ~hidden.all(axis=1)
    for j in range(hq):
        with np.errstate(invalid="ignore"):
            x = (q[:, j].astype(np.float64) @ k[:, j // (hq // h)].astype(np.float64).T) * scale
        x[hidden] = -np.inf
        x = x[rows]
        p = np.exp(x - x.max(axis=1, keepdims=True)) if x.size else x
        p /= p.sum(axis=1, keepdims=True)
        values = v[:, j // (hq // h)].astype(np.float64)
        out[rows, j], mass[rows, j] = p @ values, p @ np.abs(values)
    return out, mass


def prompt_attention(q, k, v, ends_q, ends_k, scale):
    """Packed sequences, causal: a sequence's last query sees all of its keys."""
    out, mass = np.zeros(q.shape), np.zeros(q.shape)
    for a, b, c, d in zip(ends_q[:-1], ends_q[1:], ends_k[:-1], ends_k[1:]):
        if b > a and d > c:
            last = np.arange(b - a) + (d - c) - (b - a)
            out[a:b], mass[a:b] = attend(q[a:b], k[c:d], v[c:d], last, scale)
    return out, mass


def paged_attention_int4(q, k_pages, v_pages, tables, lens, scale):
    """q [B, R, Hq, D], a sequence's rows its context's last tokens; 4-bit pages
    [blocks, block size, H, bytes]. Pages out of range hold no keys."""
    out, mass = np.zeros(q.shape), np.zeros(q.shape)
    blocks, size = k_pages.shape[:2]
    for b in range(q.shape[0]):
        at = np.arange(lens[b])
        page = np.asarray(tables[b])[at // size]
        held = (page >= 0) & (page < blocks)
        if not held.any():
            continue
        k, v = (int4_decode(p[page[held], at[held] % size]) for p in (k_pages, v_pages))
        # the keys left, by their places: row i sees those up to its own
        last = np.searchsorted(at[held], np.arange(q.shape[1]) + lens[b] - q.shape[1], side="right") - 1
        out[b], mass[b] = attend(q[b], k, v, last, scale)
    return out, mass


def paged_attention(q, k_pages, v_pages, tables, lens, scale):
    """q [B, R, Hq, D], a sequence's rows its context's last tokens; pages [blocks,
    block size, H, D]. Pages out of range hold no keys. Returns the outputs, sum p |v|,
    and [B, H, keys of the tables]: each key's weights, summed over rows and the KV head's
    query heads."""
    out, mass = np.zeros(q.shape), np.zeros(q.shape)
    blocks, size, heads = k_pages.shape[:3]
    rows, group = q.shape[1], q.shape[2] // heads
    added = np.zeros((q.shape[0], heads, np.asarray(tables).shape[1] * size))
    for b in range(q.shape[0]):
        at = np.arange(lens[b])
        page = np.asarray(tables[b])[at // size]
        held = (page >= 0) & (page < blocks)
        at = at[held]
        k, v = (p[page[held], at % size].astype(np.float64) for p in (k_pages, v_pages))
        for r in range(rows):
            seen = at <= lens[b] - rows + r
            if not seen.any():
                continue
            for h in range(q.shape[2]):
                with np.errstate(invalid="ignore", over="ignore"):
                    x = k[seen, h // group] @ q[b, r, h].astype(np.float64) * scale
                    p = np.exp(x - x.max())
                    p /= p.sum()
                    out[b, r, h] = p @ v[seen, h // group]
                    mass[b, r, h] = p @ np.abs(v[seen, h // group])
                added[b, h // group, at[seen]] += p
    return out, mass, added


def evict(weights: np.ndarray, length: int, keep: int, first: int, recent: int) -> np.ndarray:
    """The keys, in order, that stay of ``length`` keys with these weights: the
    ``first`` first, the ``recent`` last, and of the others the heaviest (NaN above
    all, -0 as 0, ties to the lower index) up to ``keep`` keys together."""
    keep = max(keep, first + recent)
    if length <= keep:
        return np.arange(length)
    middle = np.arange(first, length - recent)
    w = np.asarray(weights, dtype=np.float64)[middle] + 0.0
    order = np.lexsort((middle, np.where(np.isnan(w), -np.inf, -w), ~np.isnan(w)))
    return np.concatenate([np.arange(first), np.sort(middle[order[:keep - first - recent]]),
                           np.arange(length - recent, length)])
