"""GPU: attention of single tokens over pages of their own type, and the keys'
weights, against 64 bits.

Tolerance of a row. A logit sums D products (exact in 16 bits) in float32, then is
scaled, the reference maximum taken off and exp2 taken: fewer than D + 16 roundings
of at most 2^-24 of the sum of the absolute terms (their largest exceeds the logit
and the maximum). The weights then lose 2^-16 (bf16: two parts of 8 bits each;
float16: 2^-22, and at most 2^-30 of the largest weight where they are below 2^-8
of it; float32: none) on the way into the second product, whose sums take, of 32
keys at a time in two parts, at most 8 roundings a tile of a wave, and the merges'.
A relative change e of every weight moves an output by at most 2 e sum p |v|; last
comes the type's own half step. A key's sum of weights has the weights' own error,
without the parts', a rounding for each row and head, and two for the sum before."""

import numpy as np
import pytest
import torch

from cacheblend_vllm import _native
from cacheblend_vllm import kv_layout as KL
from cacheblend_vllm.attention import paged_attention
from oracle import operators as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
PARTS = {BF16: 2.0 ** -16, F16: 2.0 ** -22, F32: 0.0}


def _pages(g, blocks, size, heads, d, dtype, layout="merged_first"):
    pool = torch.randn(2, blocks, size, heads, d, generator=g).to(dtype)
    if layout == "merged_block":
        return pool.transpose(0, 1).contiguous().to(DEV)
    pool = pool.to(DEV)
    return pool if layout == "merged_first" else (pool[0], pool[1])


def _tables(g, lens, blocks, size, width):
    """Every sequence's pages: distinct while they last, the rest of a table out of range."""
    order, tables, at = torch.randperm(blocks, generator=g), torch.full((len(lens), width), -7, dtype=torch.int32), 0
    for i, n in enumerate(lens):
        used = (n + size - 1) // size
        tables[i, :used] = order[torch.arange(at, at + used) % blocks]
        at += used
    return tables


def _numpy(pages):
    return tuple(p.double().cpu().numpy() for p in KL.kv_planes(pages))


def _terms(q, k, tables, lens, scale):
    """[B, R, Hq]: the largest sum of a logit's absolute terms."""
    size, heads = k.shape[1:3]
    out = np.zeros(q.shape[:3])
    for b, n in enumerate(lens):
        at = np.arange(n)
        page = np.asarray(tables[b])[at // size]
        ok = (page >= 0) & (page < k.shape[0])
        if ok.any():
            keys = np.abs(k[page[ok], at[ok] % size]).repeat(q.shape[2] // heads, axis=1)
            out[b] = np.einsum("rhd,nhd->rhn", np.abs(q[b]), keys).max(axis=-1) * abs(scale)
    return out


def _compare(q, pages, tables, lens, scale, got, weights=None, before=None):
    """``got`` and the weights against 64 bits, within the docstring's bound."""
    dtype = got.dtype
    qn = q.double().cpu().numpy()
    k, v = _numpy(pages)
    want, mass, added = R.paged_attention(qn, k, v, tables, lens, scale)
    terms = _terms(qn, k, tables, lens, scale)
    e = (qn.shape[3] + 16) * 2.0 ** -24 * terms  # of each weight
    n = np.asarray(lens).reshape(-1, 1, 1)
    tol = (2 * (e + PARTS[dtype]) + (n / 4 + 64) * 2.0 ** -24)[..., None] * mass
    if dtype == F16:
        tol = tol + (n * 2.0 ** -30)[..., None] * np.abs(v).max()
    tol = tol + torch.finfo(dtype).eps / 2 * np.abs(want) + (2.0 ** -25 if dtype == F16 else 1e-30)
    err = np.abs(got.double().cpu().numpy().reshape(want.shape) - want)
    print(f"  worst {float((err / tol).max()):.3f} of the bound", flush=True)
    assert np.all(err <= tol)
    for b, m in enumerate(lens):  # rows without keys are zero, not merely small
        for r in range(want.shape[1]):
            if m - want.shape[1] + r < 0:
                assert not got.reshape(want.shape)[b, r].any()
    if weights is None:
        return
    old, new = before.double().cpu().numpy(), weights.double().cpu().numpy()
    if old.shape[1] == 1:
        added = added.sum(axis=1, keepdims=True)
    total = old.copy()
    total[..., :added.shape[2]] += added
    heads = qn.shape[1] * qn.shape[2] / old.shape[1]
    e = 2 * e.max(axis=(1, 2)).reshape(-1, 1, 1) + (heads + n / 16 + 64) * 2.0 ** -24
    tol = 2.0 ** -22 * np.abs(total) + 1e-37
    tol[..., :added.shape[2]] += e * added
    err = np.abs(new - total)
    print(f"  weights: worst {float((err / tol).max()):.3f} of the bound", flush=True)
    assert np.all(err <= tol)
    for b, m in enumerate(lens):  # sums behind the context stay as they are
        assert np.array_equal(new[b, :, m:], old[b, :, m:])


def _check(dtype, hq, hkv, d, lens, rows=None, size=16, layout="merged_first", seed=0, blocks=None, scale=None, more=0,
           sets=None):
    print(f"paged attention {dtype} {hq}/{hkv}x{d} rows {rows} lens {lens[:6]} size {size} {layout} sets {sets}", flush=True)
    g = torch.Generator().manual_seed(seed)
    width = max((n + size - 1) // size for n in lens) + more
    blocks = blocks or max(1, sum((n + size - 1) // size for n in lens))
    pages = _pages(g, blocks, size, hkv, d, dtype, layout)
    tables = _tables(g, lens, blocks, size, width)
    q = torch.randn(len(lens), rows or 1, hq, d, generator=g).to(dtype)
    scale = d ** -0.5 if scale is None else scale
    give = q if rows else q[:, 0]
    weights = before = None
    if sets:
        weights = torch.rand(len(lens), sets, width * size + 3, generator=g).to(DEV)
        before = weights.clone()
    got = paged_attention(give.to(DEV), pages, tables.to(DEV), torch.tensor(lens, device=DEV), size, scale,
                          key_weights=weights)
    torch.cuda.synchronize()
    assert got.shape == give.shape and got.dtype == dtype
    _compare(q, pages, tables.numpy(), lens, scale, got, weights, before)
    return pages, tables, q, got


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (8, 8, 64), (5, 1, 128), (12, 1, 64), (40, 2, 128), (22, 11, 64)])
def test_decode_against_64_bits(dtype, hq, hkv, d):
    _check(dtype, hq, hkv, d, [1, 0, 15, 16, 17, 31, 32, 33, 63, 64, 65, 300, 1000], seed=hq + d)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,hq,hkv,d", [(2, 8, 2, 128), (3, 4, 4, 64), (4, 32, 4, 128), (17, 6, 2, 64), (33, 6, 3, 128)])
def test_several_rows_see_up_to_their_own_token(rows, hq, hkv, d, dtype):
    _check(dtype, hq, hkv, d, [rows, 1, 64, 65, 64 + rows, 500, 0, 2], rows=rows, seed=rows)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,hq,hkv,d", [(1, 32, 8, 128), (1, 7, 7, 64), (4, 10, 2, 128), (32, 8, 2, 64), (2, 3, 1, 128)])
def test_key_weights(rows, hq, hkv, d, dtype):
    for sets in {1, hkv}:
        _check(dtype, hq, hkv, d, [33, 1, 0, 700, 257, rows], rows=rows, sets=sets, seed=rows + sets)


@pytest.mark.parametrize("size,layout", [(1, "merged_first"), (5, "merged_block"), (16, "separate"), (48, "merged_first"),
                                         (256, "merged_block")])
def test_block_sizes_and_layouts(size, layout):
    for d in (64, 128):
        _check(BF16, 8, 2, d, [333, 64, 7, 700], size=size, layout=layout, seed=size, more=3, sets=2)
        _check(F32, 8, 2, d, [333, 64, 7, 70], size=size, layout=layout, seed=size, more=3)


@pytest.mark.parametrize("lens", [[20000], [1] * 200, [4096, 1, 4096], [0, 0, 777, 0], [130] * 70 + [9000], [0, 0]])
def test_ranges_that_share_sequences_and_the_other_way_round(lens):
    _check(BF16, 8, 2, 64, lens, seed=len(lens), blocks=700, more=40, sets=1)
    _check(F16, 16, 4, 128, lens, seed=len(lens) + 1, blocks=500, more=1)
    _check(F32, 4, 4, 64, lens, seed=len(lens) + 2, blocks=500, more=1, sets=4)


def test_scales_and_wide_logits():
    # logits of hundreds: a few keys hold all the weight; none; and a negative scale
    for scale in (3.0, -0.2, 0.0, 1e-30):
        _check(F32, 8, 2, 128, [500, 70], scale=scale, seed=9, sets=2)
        _check(BF16, 8, 2, 64, [500, 70], scale=scale, seed=10, sets=1)
        _check(F16, 8, 2, 128, [500, 70], scale=scale, seed=11)


def test_pages_out_of_range_hold_no_keys():
    g = torch.Generator().manual_seed(11)
    pages = _pages(g, 6, 16, 2, 64, BF16)
    tables = torch.tensor([[0, -1, 3], [99, 6, -5], [2, 1 << 30, 4]], dtype=torch.int32)
    lens = [45, 40, 33]
    q = torch.randn(3, 2, 4, 64, generator=g).to(BF16)
    before = torch.rand(3, 2, 48, generator=g).to(DEV)
    weights = before.clone()
    got = paged_attention(q.to(DEV), pages, tables.to(DEV), torch.tensor(lens, device=DEV), 16, 0.125, key_weights=weights)
    _compare(q, pages, tables.numpy(), lens, 0.125, got, weights, before)
    assert not got[1].any() and torch.equal(weights[1], before[1]) and torch.equal(weights[0, :, 16:32], before[0, :, 16:32])
    # 64-bit tables: what 32 bits do not hold is out of range, not another page
    wide = tables.long()
    wide[0, 1], wide[2, 1] = 1 << 32, (1 << 32) + 2
    again = paged_attention(q.to(DEV), pages, wide.to(DEV), torch.tensor(lens, device=DEV), 16, 0.125)
    assert torch.equal(again, got)


def test_lengths_on_the_device_are_clamped():
    g = torch.Generator().manual_seed(12)
    pages = _pages(g, 4, 16, 2, 128, BF16)
    tables = torch.arange(4, dtype=torch.int32, device=DEV)[None].expand(3, 4)
    q = torch.randn(3, 8, 128, generator=g).to(BF16).to(DEV)
    w = torch.zeros(3, 2, 64, device=DEV)
    got = paged_attention(q, pages, tables, torch.tensor([64, 1000, -3], device=DEV), 16, 0.1, key_weights=w)
    want = paged_attention(q, pages, tables, torch.tensor([64, 64, 0], device=DEV), 16, 0.1)
    assert torch.equal(got, want) and not got[2].any() and not w[2].any()
    # every softmax adds up to 1
    assert torch.allclose(w[:2].sum(dim=2), torch.full((2, 2), 4.0, device=DEV), rtol=1e-5)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,hq", [(3, 4), (9, 6)])
def test_what_a_row_does_not_see_may_be_anything(rows, hq, dtype):
    g = torch.Generator().manual_seed(13)
    for d in (64, 128):
        clean = _pages(g, 8, 16, 2, d, dtype)
        tables = torch.tensor([[5, 2, 7]], dtype=torch.int32, device=DEV)
        q = torch.randn(1, rows, hq, d, generator=g).to(dtype).to(DEV)
        lens = torch.tensor([40], device=DEV)
        run = lambda pages, query=q: paged_attention(query, pages, tables, lens, 16, 0.1)  # noqa: E731
        want = run(clean)
        for value in (float("nan"), float("inf")):
            dirty = clean.clone()
            dirty[:, 7, 8:] = value       # behind the context
            dirty[:, [0, 1, 3, 4, 6]] = value
            assert torch.equal(run(dirty), want)
            # the newest tokens' values: only the rows that see them may notice
            dirty[1, 7, 7, 1, 3], dirty[1, 7, 6, 0, d - 1] = value, -value
            got = run(dirty)
            same = torch.ones(1, rows, hq, d, dtype=torch.bool, device=DEV)
            same[0, -1, hq // 2:, 3] = False
            same[0, -2:, :hq // 2, d - 1] = False
            assert torch.equal(got[same], want[same])
            bad = got[~same]
            assert bool(bad.isnan().all()) if value != value else bool(bad.isinf().all())
            dirty[0, 7, 7] = value        # and its key
            got = run(dirty)
            assert torch.equal(got[:, :-1][same[:, :-1]], want[:, :-1][same[:, :-1]])
            assert bool(got[:, -1].isnan().all())
        # a NaN or an infinity in one query stays in its row and head
        bad = q.clone()
        bad[0, 1, 2, 5], bad[0, 0, 3, 9] = float("nan"), float("inf")
        got = run(clean, bad)
        other = torch.ones(1, rows, hq, dtype=torch.bool, device=DEV)
        other[0, 1, 2] = other[0, 0, 3] = False
        assert torch.equal(got[other], want[other]) and bool(got[~other].isnan().all())


def test_values_and_logits_near_the_ends_of_a_type():
    g = torch.Generator().manual_seed(14)
    tables = torch.tensor([[1, 0, 2, 3]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([64], device=DEV)
    for dtype, top in ((BF16, 3e38), (F16, 60000.0), (F32, 3e38)):
        for d in (64, 128):
            pages = _pages(g, 4, 16, 2, d, dtype)
            q = torch.randn(1, 4, d, generator=g).to(dtype).to(DEV)
            pages[1] = top  # equal values: their mean, rounded
            got = paged_attention(q, pages, tables, lens, 16, 0.1)
            # float32 sums of float32 terms: 2 roundings a key, and the type's half step
            assert bool(((got.double() / float(pages[1, 0, 0, 0, 0]) - 1).abs() <= 2.0 ** -16 + torch.finfo(dtype).eps / 2).all())
            # one key's logit past all others': its value, exactly
            pages = _pages(g, 4, 16, 2, d, dtype)
            q[:] = 1.0
            pages[0] = -1.0
            pages[0, 2, 5] = 100.0 if dtype == F16 else 1e30
            got = paged_attention(q, pages, tables, lens, 16, 1e6)
            want = pages[1, 2, 5].repeat_interleave(2, dim=0)[None]
            assert torch.equal(got, want)
            # logits of -inf have no weight, +inf is no number
            pages[0, 2, 5], pages[0, 1, 0] = -1.0, -float("inf")
            assert bool(paged_attention(q, pages, tables, lens, 16, 1.0).isfinite().all())
            pages[0, 1, 0] = float("inf")
            assert bool(paged_attention(q, pages, tables, lens, 16, 1.0).isnan().all())


def test_strides_and_alignments():
    g = torch.Generator().manual_seed(15)
    for dtype in (BF16, F32):
        for d in (64, 128):
            # blocks longer than used, pages at an odd element, padded rows of queries and outputs
            room = torch.randn(2 * 6 * 20 * 2 * d + 1, generator=g).to(dtype).to(DEV)
            pages = room[1:].view(2, 6, 20, 2, d)
            tables = torch.tensor([[3, 9, 1, 9, 5, 9], [0, 9, 2, 9, 4, 9]], dtype=torch.int32, device=DEV)[:, ::2]
            lens = [40, 48]
            wide = torch.randn(2, 3, 9, d + 1, generator=g).to(dtype).to(DEV)
            q = wide[:, 1:, 1:, :d]
            out = torch.full((2, 2, 10, d + 3), 7.0, dtype=dtype, device=DEV)
            pool = torch.rand(4, 2, 70, generator=g).to(DEV)
            weights, before = pool[1::2, :, 1:], pool[1::2, :, 1:].clone()
            kept = pool.clone()
            got = paged_attention(q, pages, tables, torch.tensor(lens), 16, 0.1, out=out[:, :, 1:9, 2:d + 2], key_weights=weights)
            _compare(q, pages[:, :, :16], tables.cpu().numpy(), lens, 0.1, got, weights, before)
            out[:, :, 1:9, 2:d + 2] = 7.0
            assert bool((out == 7.0).all())
            pool[1::2, :, 1:] = kept[1::2, :, 1:]
            assert torch.equal(pool, kept)


def test_offsets_past_32_bits():
    # two planes of 3 GB: the last pages lie past 2^32 bytes from the base
    blocks = 400_000
    pages = torch.empty(2, blocks, 16, 4, 64, dtype=BF16, device=DEV)
    g = torch.Generator().manual_seed(16)
    tables = torch.tensor([[blocks - 1, 3, blocks // 2]], dtype=torch.int32)
    pages[:, tables[0].long()] = torch.randn(2, 3, 16, 4, 64, generator=g).to(BF16).to(DEV)
    q = torch.randn(1, 1, 8, 64, generator=g).to(BF16)
    got = paged_attention(q.to(DEV), pages, tables.to(DEV), torch.tensor([41], device=DEV), 16, 0.125)
    small = pages[:, tables[0].long()]
    _compare(q, small, np.array([[0, 1, 2]]), [41], 0.125, got)


def test_streams_graphs_and_repeats():
    g = torch.Generator().manual_seed(17)
    pages = _pages(g, 300, 16, 8, 128, BF16)
    lens = torch.tensor([2000, 77, 1500], device=DEV)
    tables = _tables(g, lens.tolist(), 300, 16, 130).to(DEV)
    q = torch.randn(3, 32, 128, generator=g).to(BF16).to(DEV)
    w0 = torch.rand(3, 8, 130 * 16, generator=g).to(DEV)

    def once():
        w = w0.clone()
        return paged_attention(q, pages, tables, lens, 16, 0.09, key_weights=w), w

    want = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = once()
        again = once()
    torch.cuda.current_stream().wait_stream(side)
    for pair in (got, again):
        assert torch.equal(pair[0], want[0]) and torch.equal(pair[1], want[1])
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    w = w0.clone()
    with torch.cuda.graph(graph):
        out = paged_attention(q, pages, tables, lens, 16, 0.09, key_weights=w)
    w_other = w0.clone()
    with torch.cuda.graph(other):
        out_other = paged_attention(q, pages, tables, lens, 16, 0.09, key_weights=w_other)
    for n in (2000, 1033, 1):  # lengths may change between replays
        lens[0] = n
        want = once()
        for gr, o, ww in ((graph, out, w), (other, out_other, w_other)):
            ww.copy_(w0)
            gr.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, want[0]) and torch.equal(ww, want[1])


def test_refusals():
    pages = torch.zeros(2, 4, 16, 2, 64, dtype=BF16, device=DEV)
    tables, lens = torch.zeros(1, 4, dtype=torch.int32), torch.tensor([20])
    q = torch.zeros(1, 4, 64, dtype=BF16, device=DEV)

    def refused(error, match, query=q, kv=pages, t=tables, n=lens, size=16, **kw):
        with pytest.raises(error, match=match):
            paged_attention(query, kv, t, n, size, 0.1, **kw)

    refused(RuntimeError, "device", query=q.cpu())
    refused(ValueError, "query must be", query=q[0])
    refused(ValueError, "the pages hold", query=q.half())
    refused(ValueError, "not supported", query=q.double())
    refused(ValueError, "divisible", query=torch.zeros(1, 3, 64, dtype=BF16, device=DEV))
    refused(ValueError, "head size", query=torch.zeros(1, 4, 128, dtype=BF16, device=DEV))
    refused(ValueError, "64 or 128", query=torch.zeros(1, 4, 32, dtype=BF16, device=DEV),
            kv=torch.zeros(2, 4, 16, 2, 32, dtype=BF16, device=DEV))
    refused(ValueError, "block tables", t=tables.expand(2, 4))
    refused(ValueError, "lengths", n=torch.tensor([20, 20]))
    refused(ValueError, "whole numbers", t=tables.float())
    refused(IndexError, "context lengths", n=torch.tensor([65]))
    refused(IndexError, "context lengths", n=torch.tensor([-1]))
    refused(IndexError, "block tables", t=torch.full((1, 4), 4, dtype=torch.int32))
    refused(ValueError, "block_size", size=17)
    refused(ValueError, "out must be", out=torch.zeros(1, 4, 64, device=DEV))
    refused(ValueError, "overlap", out=torch.zeros(1, 1, 64, dtype=BF16, device=DEV).expand(1, 4, 64))
    for w in (torch.zeros(1, 2, 63, device=DEV), torch.zeros(1, 3, 64, device=DEV), torch.zeros(2, 2, 64, device=DEV),
              torch.zeros(2, 64, device=DEV)):
        refused(ValueError, "key weights are", key_weights=w)
    refused(ValueError, "float32", key_weights=torch.zeros(1, 2, 64, device=DEV, dtype=BF16))
    refused(ValueError, "float32", key_weights=torch.zeros(1, 2, 64))
    refused(ValueError, "contiguous keys", key_weights=torch.zeros(1, 2, 128, device=DEV)[..., ::2])
    refused(ValueError, "overlap", key_weights=torch.zeros(1, 1, 64, device=DEV).expand(1, 2, 64))
    with pytest.raises(ValueError, match="scale"):
        paged_attention(q, pages, tables, lens, 16, float("nan"))
    # nothing to do
    assert paged_attention(q[:0], pages, tables[:0], lens[:0], 16, 0.1).shape == (0, 4, 64)
    assert not paged_attention(q, pages, tables[:, :0], torch.tensor([0]), 16, 0.1).any()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_tables_of_more_than_the_caches_hold(dtype):
    # room for 600 MB of keys and values, which are then read past the caches; few are there
    es = 4 if dtype is F32 else 2
    more = 600_000_000 // (4 * 16 * 2 * 4 * 128 * es)
    _check(dtype, 8, 4, 128, [700, 33, 0, 290], seed=18, more=more)
    _check(dtype, 8, 4, 128, [700, 33, 0, 290], rows=2, sets=4, seed=19, more=more)
    _check(dtype, 8, 8, 64, [700, 33, 0, 290], size=48, sets=1, seed=20, more=more)


def test_outputs_in_the_queries_place():
    g = torch.Generator().manual_seed(21)
    for lens, rows in (([300, 40], 1), ([9000, 40, 2], 3), ([5000], 33)):  # whole and in ranges
        n = sum((x + 15) // 16 for x in lens)
        pages, tables = _pages(g, n, 16, 2, 64, BF16), _tables(g, lens, n, 16, (max(lens) + 15) // 16).to(DEV)
        q = torch.randn(len(lens), rows, 8, 64, generator=g).to(BF16).to(DEV)
        want = paged_attention(q, pages, tables, torch.tensor(lens), 16, 0.2)
        got = paged_attention(q, pages, tables, torch.tensor(lens), 16, 0.2, out=q)
        assert got is q and torch.equal(q, want)
    # with key weights, from logits and from a second product of the keys
    for rows, width in ((1, 20), (64, 800)):
        pages, tables = _pages(g, 20, 16, 2, 64, BF16), torch.randint(0, 20, (1, width), generator=g).int().to(DEV)
        q = torch.randn(1, rows, 8, 64, generator=g).to(BF16).to(DEV)
        pairs = []
        for out in (None, q):
            weights = torch.zeros(1, 1, width * 16, device=DEV)
            pairs.append((paged_attention(q, pages, tables, torch.tensor([300]), 16, 0.2, out=out, key_weights=weights), weights))
        assert pairs[1][0] is q and torch.equal(pairs[0][0], q) and torch.equal(pairs[0][1], pairs[1][1])
        # the entry point refuses the latter
        desc, _, _ = KL.paged_layer(pages, 16)
        lens, ws = torch.tensor([300], dtype=torch.int32, device=DEV), torch.empty(1 << 26, dtype=torch.uint8, device=DEV)
        rc = _native.load().cbk_paged_attention(
            q.data_ptr(), 0, 512, 64, 1, rows, 8, desc, 2, 64, tables.data_ptr(), width, width, lens.data_ptr(), 0.2, 1,
            q.data_ptr(), 0, 512, 64, weights.data_ptr(), 0, 0, 1, ws.data_ptr(), ws.numel(), _native.stream_handle(DEV))
        assert rc == (_native.CBK_OK if rows == 1 else _native.CBK_ERR_INVALID)


def test_logits_of_minus_infinity_weigh_nothing():
    # products of -3e38 and 3e38: rows of nothing else are zero, others go by the keys left
    g = torch.Generator().manual_seed(22)
    lens = [100, 1000]
    pages = _pages(g, 70, 16, 1, 64, F32)
    tables = _tables(g, lens, 70, 16, 63).to(DEV)
    pages[0] = 0.0
    pages[0, ..., 0] = -3e38
    q = torch.zeros(2, 2, 64, device=DEV)
    q[:, 0, 0] = 3e38
    weights = torch.zeros(2, 1, 63 * 16, device=DEV)
    got = paged_attention(q, pages, tables, torch.tensor(lens), 16, 1.0, key_weights=weights)
    assert not got[:, 0].any() and bool(got[:, 1].any(dim=1).all())
    for b, n in enumerate(lens):  # the second head's weights: equal
        assert torch.allclose(weights[b, 0, :n], torch.full((n,), 1.0 / n, device=DEV), rtol=2e-6) and not weights[b, 0, n:].any()
    # one key with another logit
    pages[0, tables[1, 30], 5, 0, 0] = 0.0
    got = paged_attention(q, pages, tables, torch.tensor(lens), 16, 1.0)
    assert not got[0, 0].any() and torch.equal(got[1, 0], pages[1, tables[1, 30], 5, 0])


def test_calls_that_need_no_scratch_take_none():
    g = torch.Generator().manual_seed(23)
    pages, lens = _pages(g, 8, 16, 2, 128, BF16), torch.tensor([60, 33], dtype=torch.int32, device=DEV)
    tables = torch.arange(8, dtype=torch.int32, device=DEV).view(2, 4)
    q = torch.randn(2, 4, 128, generator=g).to(BF16).to(DEV)
    lib, out = _native.load(), torch.empty_like(q)
    desc, _, _ = KL.paged_layer(pages, 16)
    assert lib.cbk_paged_attention_workspace_bytes(2, 1, 4, 2, 128, 64, 1, 0) == 0
    args = (q.data_ptr(), 512, 512, 128, 2, 1, 4, desc, 2, 128, tables.data_ptr(), 4, 4, lens.data_ptr(), 0.1, 1, out.data_ptr(),
            512, 512, 128)
    assert lib.cbk_paged_attention(*args, None, 0, 0, 0, None, 0, _native.stream_handle(DEV)) == _native.CBK_OK
    assert torch.equal(out, paged_attention(q, pages, tables, lens, 16, 0.1))
    # with key weights there is some to give
    need = lib.cbk_paged_attention_workspace_bytes(2, 1, 4, 2, 128, 64, 1, 1)
    w = torch.zeros(2, 1, 64, device=DEV)
    assert need > 0
    for ws, n in ((None, need), (w.data_ptr(), need - 1)):
        rc = lib.cbk_paged_attention(*args, w.data_ptr(), 64, 64, 1, ws, n, _native.stream_handle(DEV))
        assert rc == _native.CBK_ERR_WORKSPACE


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,hq,hkv,d,sets", [(64, 8, 1, 128, 1), (33, 16, 4, 64, 1), (129, 4, 4, 128, 1), (40, 64, 4, 64, 4)])
def test_key_weights_of_many_rows(rows, hq, hkv, d, sets, dtype):
    # with room for many keys without logits in scratch (from 128 rows a KV head and 512 a set on)
    assert _native.load().cbk_paged_attention_workspace_bytes(6, rows, hq, hkv, d, 160 * 16, 1, sets) < 6 * 2560 * rows * hq * 4
    for more in (0, 150):
        _check(dtype, hq, hkv, d, [33, 1, 0, 700, 257, rows], rows=rows, sets=sets, seed=rows + sets, more=more)
    _check(dtype, hq, hkv, d, [333, 64], size=5, rows=rows, sets=sets, seed=rows, more=1300)


def test_key_weights_of_many_rows_where_pages_are_missing():
    g = torch.Generator().manual_seed(24)
    pages = _pages(g, 6, 16, 2, 64, BF16)
    pages[:, 5] = float("nan")  # of keys past the lengths
    tables = torch.full((3, 300), 5, dtype=torch.int32)
    tables[:, :4] = torch.tensor([[0, -1, 3, 5], [99, 6, -5, 1], [2, 1 << 30, 4, 5]])
    lens, rows = [45, 40, 33], 64
    q = torch.randn(3, rows, 16, 64, generator=g).to(BF16)
    before = torch.rand(3, 1, 4800, generator=g).to(DEV)
    weights = before.clone()
    got = paged_attention(q.to(DEV), pages, tables.to(DEV), torch.tensor(lens, device=DEV), 16, 0.125, key_weights=weights)
    _compare(q, pages, tables.numpy(), lens, 0.125, got, weights, before)
    assert torch.equal(weights[1], before[1]) and torch.equal(weights[0, :, 16:32], before[0, :, 16:32])


def test_many_rows_in_graphs():
    g = torch.Generator().manual_seed(25)
    pages, tables = _pages(g, 60, 16, 2, 128, BF16), torch.randint(0, 60, (2, 450), generator=g).int().to(DEV)
    lens = torch.tensor([900, 70], device=DEV, dtype=torch.int32)
    q = torch.randn(2, 40, 16, 128, generator=g).to(BF16).to(DEV)
    w0 = torch.rand(2, 1, 7200, generator=g).to(DEV)

    def once():
        w = w0.clone()
        return paged_attention(q, pages, tables, lens, 16, 0.09, key_weights=w), w

    once()
    graph, w = torch.cuda.CUDAGraph(), w0.clone()
    with torch.cuda.graph(graph):
        out = paged_attention(q, pages, tables, lens, 16, 0.09, key_weights=w)
    for n in (900, 33, 0, 5000):
        lens[0] = n
        want = once()
        w.copy_(w0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(w, want[1])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,hq,d", [(1, 4, 128), (1, 8, 64), (3, 4, 128), (9, 6, 64), (40, 4, 128)])
def test_infinities_that_all_rows_see(rows, hq, d, dtype):
    """An infinite value that has any weight is the row's, of opposite ones there is no sum; other dims notice nothing."""
    inf, nan = float("inf"), float("nan")
    for lens, size, sets in (([70], 16, None), ([70, 64], 5, 2), ([600], 16, 1), ([9000, 100], 16, None), ([9000, 100], 16, 2),
                             ([300] * 40, 48, 2), ([2600] * 3, 16, 1)):
        g = torch.Generator().manual_seed(rows + d + len(lens))
        blocks = sum((n + size - 1) // size for n in lens)
        clean = _pages(g, blocks, size, 2, d, dtype)
        tables = _tables(g, lens, blocks, size, (max(lens) + size - 1) // size)
        q = torch.randn(len(lens), rows, hq, d, generator=g).to(dtype).to(DEV)

        def run(pages):
            w = torch.zeros(len(lens), sets, tables.shape[1] * size, device=DEV) if sets else None
            return paged_attention(q, pages, tables.to(DEV), torch.tensor(lens), size, 0.1, key_weights=w), w

        want, weights = run(clean)
        dirty = clean.clone()

        def put(key, head, dim, value):
            dirty[1, tables[0, key // size], key % size, head, dim] = value

        early = [2, 0, 19, 1, 29, 17, 25]  # keys of the first sequence that every row sees
        put(early[0], 0, 3, inf)
        put(early[1], 0, 6, -inf)
        put(early[2], 0, d - 1, -inf)
        put(early[3], 1, 8, inf)
        put(early[4], 1, 8, -inf)
        put(early[5], 1, 9, nan)
        put(early[6], 1, 3, inf)
        put(lens[0] - rows, 1, d - 2, inf)  # the first row's own
        got, again = run(dirty)
        half = hq // 2
        expect = want.clone()
        expect[0, :, :half, 3], expect[0, :, half:, 3], expect[0, :, half:, d - 2] = inf, inf, inf
        expect[0, :, :half, 6], expect[0, :, :half, d - 1] = -inf, -inf
        expect[0, :, half:, 8], expect[0, :, half:, 9] = nan, nan
        assert torch.equal(got.isnan(), expect.isnan()), (lens, size, sets)
        assert torch.equal(got.nan_to_num(nan=7.0, posinf=inf, neginf=-inf), expect.nan_to_num(nan=7.0, posinf=inf, neginf=-inf))
        assert not sets or torch.equal(again, weights)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,hq,hkv,d,width", [(3, 8, 2, 64, 40), (5, 8, 2, 128, 600), (20, 8, 2, 64, 300), (40, 4, 2, 128, 3),
                                                 (33, 16, 4, 64, 1300), (150, 8, 1, 128, 1300)])
def test_rows_without_a_number_weigh_only_what_they_see(rows, hq, hkv, d, width, dtype):
    """A NaN or an infinity in a query makes its row's weights NaN, those of the keys that the row sees; later keys
    and pages out of range keep the other rows' sums to the last bit. By logits in scratch, and by a second product."""
    g = torch.Generator().manual_seed(rows + width)
    lens = [45, 40, 33, 0]
    pages = _pages(g, 12, 16, hkv, d, dtype)
    pages[0, :, ::2, :, 5] = pages[0, :, ::2, :, 5].abs() + 1  # an infinity in a query meets both signs
    pages[0, :, 1::2, :, 5] = -pages[0, :, 1::2, :, 5].abs() - 1
    tables = torch.zeros(4, width, dtype=torch.int32)
    tables[:, :3] = torch.tensor([[0, 6, 3], [4, -1, 5], [7, 1 << 30, 2], [1, 1, 1]])
    clean = torch.randn(4, rows, hq, d, generator=g).to(dtype)
    held = [np.array([0 <= int(tables[b, k // 16]) < 12 for k in range(n)], dtype=bool) for b, n in enumerate(lens)]
    for sets in {1, hkv}:
        before = torch.rand(4, sets, width * 16, generator=g)

        def run(q):
            w = before.to(DEV)
            return paged_attention(q.to(DEV), pages, tables.to(DEV), torch.tensor(lens, device=DEV), 16, 0.1, key_weights=w), w.cpu()

        want, weights = run(clean)
        for value in (float("nan"), float("inf"), -float("inf")):
            for b, r, h in ((0, 0, 0), (0, rows - 2, hq - 1), (1, rows - 1, 1), (2, 1, hq - 1)):
                q = clean.clone()
                q[b, r, h, 5] = value
                got, w = run(q)
                seen = held[b] & (np.arange(lens[b]) <= lens[b] - rows + r)
                none = torch.zeros_like(weights, dtype=torch.bool)
                none[b, h // (hq // sets), :lens[b]] = torch.from_numpy(seen)
                assert torch.equal(w.isnan(), none), (sets, value, b, r, h)
                assert torch.equal(w[~none], weights[~none])
                other = torch.ones(4, rows, hq, dtype=torch.bool)
                other[b, r, h] = False
                assert torch.equal(got.cpu()[other], want.cpu()[other])
                assert bool(got[b, r, h].isnan().all()) if seen.any() else not got[b, r, h].any()


def test_outputs_over_the_queries_otherwise():
    """Outputs that share memory with other places' queries: of other strides, or moved by a sequence or a head."""
    g = torch.Generator().manual_seed(26)
    batch, hq, d = 1500, 8, 64
    pages = _pages(g, 50, 16, 2, d, BF16)
    tables, lens = torch.randint(0, 50, (batch, 3), generator=g).int().to(DEV), torch.full((batch,), 40, device=DEV)
    whole = torch.randn(batch + 1, hq, d, generator=g).to(BF16)

    def views(room):
        flat = room.flatten()
        yield room[:batch], flat[:batch * hq * d].view(hq, batch, d).transpose(0, 1)
        yield room[:batch], room[1:]
        yield room[1:], room[:batch]
        yield room[:batch], flat[d:d + batch * hq * d].view(batch, hq, d)
        yield room[:batch, None], flat[:batch * hq * d].view(hq, batch, 1, d).permute(1, 2, 0, 3)

    for i in range(5):
        for weigh in (False, True):
            q, out = list(views(whole.to(DEV)))[i]
            want = paged_attention(q, pages, tables, lens, 16, 0.2)
            w = torch.zeros(batch, 1, 48, device=DEV) if weigh else None
            got = paged_attention(q, pages, tables, lens, 16, 0.2, out=out, key_weights=w)
            assert got is out and torch.equal(out, want), (i, weigh)
    # beside each other in one tensor they share nothing
    room = torch.randn(batch, 2, hq, d, generator=g).to(BF16).to(DEV)
    q = room[:, 0].clone()
    want = paged_attention(q, pages, tables, lens, 16, 0.2)
    paged_attention(room[:, 0], pages, tables, lens, 16, 0.2, out=room[:, 1])
    assert torch.equal(room[:, 1], want) and torch.equal(room[:, 0], q)
