"""GPU: attention of single tokens over 4-bit pages, against 64 bits.

Tolerance of a row. A logit sums, per 32 dims, products of a query element
with a whole number below 16, exact, and then step times that sum and offset
times the query's sum: fewer than 64 float32 roundings on the way, of at most
2^-24 of the sum of the absolute terms each; taking it to log2 units and the
reference maximum off rounds it three times more. 16-bit queries are cut into
parts that hold an element to 2^-10 where the row's largest is 128 to 256, so to
2^-17 of that one. The weights then lose 2^-16 (two bf16 parts, the second
rounded; float32: three, 2^-23), their sums at most one rounding a key of a lane
and the merges'. A relative change e of every weight moves an output by at most
2 e sum p |v|; last comes the type's own half step. With codes, |v| is replaced
by what a value's products hold: step * 144 (the codes are 128 to 143 there,
and 128 is taken off; float32: step * 16) + |offset|, rounded as often."""

import numpy as np
import pytest
import torch

from cacheblend_vllm import kv_layout as KL
from cacheblend_vllm.attention import paged_attention_int4
from oracle import operators as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _pages(g, blocks, size, heads, d, layout="merged_first", spread=1.0):
    """4-bit pages of normal values, per token of a spread of its own."""
    x = torch.randn(2, blocks, size, heads, d, generator=g, dtype=torch.float64)
    x *= torch.exp(spread * torch.randn(2, blocks, size, 1, 1, generator=g, dtype=torch.float64) / 2)
    pool = torch.from_numpy(R.int4_encode(x.numpy()))
    if layout == "merged_block":
        return pool.transpose(0, 1).contiguous().to(DEV)
    pool = pool.to(DEV)
    return pool if layout == "merged_first" else (pool[0], pool[1])


def _tables(g, lens, blocks, size, width):
    """Every sequence's pages: distinct, the rest of a table out of range."""
    order, tables, at = torch.randperm(blocks, generator=g), torch.full((len(lens), width), -7, dtype=torch.int32), 0
    for i, n in enumerate(lens):
        used = (n + size - 1) // size
        tables[i, :used] = order[torch.arange(at, at + used) % blocks]
        at += used
    return tables


def _bound(q, pages, tables, lens, scale, dtype, want, mass):
    """The docstring's bound, per sequence, row and head (coarse over dims)."""
    k_pages, v_pages = (p.cpu().numpy() for p in KL.kv_planes(pages))
    size, heads, d = k_pages.shape[1], k_pages.shape[2], q.shape[3]
    exact = dtype == F32

    # steps and offsets [.., groups]
    def held(p):
        words = np.ascontiguousarray(p[..., d // 2:]).view(np.uint16).astype(np.uint32) << 16
        both = words.view(np.float32).reshape(*p.shape[:-1], d // 32, 2)
        return np.abs(both[..., 0]), np.abs(both[..., 1])

    tol = np.zeros(want.shape)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        at = np.arange(n)
        page = np.asarray(tables[b])[at // size]
        ok = (page >= 0) & (page < k_pages.shape[0])
        if not ok.any():
            continue
        (ks, ko), (vs, vo) = (held(p[page[ok], at[ok] % size]) for p in (k_pages, v_pages))  # [n, heads, groups]
        hk, hv = 16 * ks + ko, (16 if exact else 144) * vs + vo
        qs = np.abs(q[b]).reshape(q.shape[1], q.shape[2], d // 32, 32).sum(axis=-1)  # [rows, hq, groups]
        group = q.shape[2] // heads
        terms = np.einsum("rhg,nhg->rhn", qs, hk.repeat(group, axis=1)).max(axis=-1) * abs(scale)
        e = 67 * 2.0 ** -24 * terms + (2.0 ** -22 if exact else 2.0 ** -15) + (n / 16 + 64) * 2.0 ** -24
        if not exact:  # the queries' parts
            cut = 2.0 ** -17 * np.abs(q[b]).max(axis=-1) * 32 * 15 * ks.sum(axis=-1).max(axis=0).repeat(group)
            e = e + abs(scale) * cut
        values = hv.max(axis=0).repeat(group, axis=0).repeat(32, axis=1)  # [hq, d]
        tol[b] = 2 * e[..., None] * mass[b] + (n / 16 + 64) * 2.0 ** -24 * values
    return tol + torch.finfo(dtype).eps / 2 * np.abs(want) + (2.0 ** -25 if dtype == F16 else 1e-30)


def _check(dtype, hq, hkv, d, lens, rows=None, size=16, layout="merged_first", seed=0, blocks=None, scale=None, more=0,
           spread=1.0):
    print(f"int4 attention {dtype} {hq}/{hkv}x{d} rows {rows} lens {lens[:6]} size {size} {layout}", flush=True)
    g = torch.Generator().manual_seed(seed)
    width = max((n + size - 1) // size for n in lens) + more
    blocks = blocks or max(1, sum((n + size - 1) // size for n in lens))
    pages = _pages(g, blocks, size, hkv, d, layout, spread)
    tables = _tables(g, lens, blocks, size, width)
    q = torch.randn(len(lens), rows or 1, hq, d, generator=g).to(dtype)
    scale = d ** -0.5 if scale is None else scale
    give = q if rows else q[:, 0]
    got = paged_attention_int4(give.to(DEV), pages, tables.to(DEV), torch.tensor(lens, device=DEV), size, scale)
    torch.cuda.synchronize()
    assert got.shape == give.shape and got.dtype == dtype
    k, v = (p.cpu().numpy() for p in KL.kv_planes(pages))
    qn = q.double().numpy()
    want, mass = R.paged_attention_int4(qn, k, v, tables.numpy(), lens, scale)
    tol = _bound(qn, pages, tables.numpy(), lens, scale, dtype, want, mass)
    err = np.abs(got.double().cpu().numpy().reshape(want.shape) - want)
    print(f"  worst {float((err / tol).max()):.3f} of the bound, relative {np.linalg.norm(err) / max(1e-30, np.linalg.norm(want)):.2e}",
          flush=True)
    assert np.all(err <= tol)
    # rows without keys are zero, not merely small
    for b, n in enumerate(lens):
        for r in range(want.shape[1]):
            if n - want.shape[1] + r < 0:
                assert not got.reshape(want.shape)[b, r].any()
    return pages, tables, q, got


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (8, 8, 64), (5, 1, 128), (12, 1, 64), (40, 2, 128)])
def test_decode_against_64_bits(dtype, hq, hkv, d):
    _check(dtype, hq, hkv, d, [1, 0, 63, 64, 65, 300, 1000, 17], seed=hq + d)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,hq,hkv,d", [(2, 8, 2, 128), (3, 4, 4, 64), (4, 32, 4, 128), (17, 6, 2, 64)])
def test_several_rows_see_up_to_their_own_token(rows, hq, hkv, d, dtype):
    _check(dtype, hq, hkv, d, [rows, 1, 64, 65, 64 + rows, 500, 0, 2], rows=rows, seed=rows)


@pytest.mark.parametrize("size,layout", [(1, "merged_first"), (5, "merged_block"), (16, "separate"), (48, "merged_first"),
                                         (256, "merged_block")])
def test_block_sizes_and_layouts(size, layout):
    for d in (64, 128):
        _check(BF16, 8, 2, d, [333, 64, 7, 700], size=size, layout=layout, seed=size, more=3)


@pytest.mark.parametrize("lens", [[20000], [1] * 200, [4096, 1, 4096], [0, 0, 777, 0], [130] * 70 + [9000]])
def test_ranges_that_share_sequences_and_the_other_way_round(lens):
    _check(BF16, 8, 2, 64, lens, seed=len(lens), blocks=700, more=40)
    _check(F16, 16, 4, 128, lens, seed=len(lens) + 1, blocks=500)


def test_scales_and_wide_logits():
    # logits of hundreds: a few keys hold all the weight; none; and a negative scale
    for scale in (3.0, -0.2, 0.0, 1e-30):
        _check(F32, 8, 2, 128, [500, 70], scale=scale, seed=9, spread=2.0)
        _check(BF16, 8, 2, 64, [500, 70], scale=scale, seed=10, spread=2.0)


def test_pages_out_of_range_hold_no_keys():
    g = torch.Generator().manual_seed(11)
    pages = _pages(g, 6, 16, 2, 64)
    tables = torch.tensor([[0, -1, 3], [99, 6, -5], [2, 1 << 30, 4]], dtype=torch.int32)
    lens = [45, 40, 33]
    q = torch.randn(3, 2, 4, 64, generator=g).to(BF16)
    got = paged_attention_int4(q.to(DEV), pages, tables.to(DEV), torch.tensor(lens, device=DEV), 16, 0.125)
    k, v = (p.cpu().numpy() for p in KL.kv_planes(pages))
    want, mass = R.paged_attention_int4(q.double().numpy(), k, v, tables.numpy(), lens, 0.125)
    tol = _bound(q.double().numpy(), pages, tables.numpy(), lens, 0.125, BF16, want, mass)
    assert np.all(np.abs(got.double().cpu().numpy() - want) <= tol)
    assert not got[1].any()
    # 64-bit tables: what 32 bits do not hold is out of range, not another page
    wide = tables.long()
    wide[0, 1], wide[2, 1] = 1 << 32, (1 << 32) + 2
    again = paged_attention_int4(q.to(DEV), pages, wide.to(DEV), torch.tensor(lens, device=DEV), 16, 0.125)
    assert torch.equal(again, got)


def test_lengths_on_the_device_are_clamped():
    g = torch.Generator().manual_seed(12)
    pages = _pages(g, 4, 16, 2, 128)
    tables = torch.arange(4, dtype=torch.int32, device=DEV)[None].expand(3, 4)
    q = torch.randn(3, 8, 128, generator=g).to(BF16).to(DEV)
    got = paged_attention_int4(q, pages, tables, torch.tensor([64, 1000, -3], device=DEV), 16, 0.1)
    want = paged_attention_int4(q, pages, tables, torch.tensor([64, 64, 0], device=DEV), 16, 0.1)
    assert torch.equal(got, want) and not got[2].any()


def test_what_a_row_does_not_see_may_be_anything():
    # the newest token's rows hold NaN: only its own row may notice; so may
    # what lies behind the context and in no table
    g = torch.Generator().manual_seed(13)
    for d in (64, 128):
        clean = _pages(g, 8, 16, 2, d)
        tables = torch.tensor([[5, 2, 7]], dtype=torch.int32, device=DEV)
        q = torch.randn(1, 3, 4, d, generator=g).to(F16).to(DEV)
        lens = torch.tensor([40], device=DEV)
        want = paged_attention_int4(q, clean, tables, lens, 16, 0.1)
        dirty = clean.clone()
        nan = torch.from_numpy(R.int4_encode(np.full((2, d), np.nan))).to(DEV)
        dirty[:, 7, 7] = nan          # token 39: the last row's own
        dirty[:, 7, 8:] = 255         # behind the context
        dirty[:, [0, 1, 3, 4, 6]] = 255
        got = paged_attention_int4(q, dirty, tables, lens, 16, 0.1)
        assert torch.equal(got[:, :2], want[:, :2]), d
        assert bool(got[:, 2].isnan().all())
        # a NaN or an infinity in one query stays in its row and head
        bad = q.clone()
        bad[0, 1, 2, 5], bad[0, 0, 3, 9] = float("nan"), float("inf")
        got = paged_attention_int4(bad, clean, tables, lens, 16, 0.1)
        other = torch.ones(1, 3, 4, dtype=torch.bool, device=DEV)
        other[0, 1, 2] = other[0, 0, 3] = False
        assert torch.equal(got[other], want[other])
        assert bool(got[0, 1, 2].isnan().all()) and bool(got[0, 0, 3].isnan().all())


def test_strides_of_queries_and_outputs():
    g = torch.Generator().manual_seed(14)
    pages, lens = _pages(g, 20, 16, 2, 128), torch.tensor([90, 17], device=DEV)
    tables = _tables(g, [90, 17], 20, 16, 9).to(DEV)
    qkv = torch.randn(2, 2, 8 + 4, 128, generator=g).to(BF16).to(DEV)
    q = qkv[:, :, 2:10]
    want = paged_attention_int4(q.contiguous(), pages, tables, lens, 16, 0.1)
    assert torch.equal(paged_attention_int4(q, pages, tables, lens, 16, 0.1), want)
    out = torch.zeros(2, 2, 8, 200, dtype=BF16, device=DEV)
    got = paged_attention_int4(q, pages, tables[:, :6], lens, 16, 0.1, out=out[..., 3:131])
    assert torch.equal(got, want) and not out[..., :3].any() and not out[..., 131:].any()
    flipped = q.transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.randn(2, 2, 8, 129, generator=g).to(BF16).to(DEV)
    odd[..., 1:] = q
    for other in (flipped, odd[..., 1:]):
        assert torch.equal(paged_attention_int4(other, pages, tables, lens, 16, 0.1), want)
    shared = paged_attention_int4(q[:1].expand(2, 2, 8, 128), pages, tables[:1].expand(2, 9), lens[:1].expand(2), 16, 0.1)
    assert torch.equal(shared[0], want[0]) and torch.equal(shared[1], want[0])
    # pages at 4-byte alignment take other transfers, the same sums
    raw = torch.zeros(pages.numel() + 4, dtype=torch.uint8, device=DEV)
    moved = raw[4:].view(pages.shape)
    moved.copy_(pages)
    assert torch.equal(paged_attention_int4(q, moved, tables, lens, 16, 0.1), want)


def test_pages_past_32_bits():
    # 5 GB of pages: rows on both sides of 2^32 bytes
    blocks = 5 * (1 << 30) // (2 * 16 * 8 * 80)
    pages = torch.zeros(blocks, 2, 16, 8, 80, dtype=torch.uint8, device=DEV)
    g = torch.Generator().manual_seed(15)
    few = _pages(g, 6, 16, 8, 128)
    at = torch.tensor([0, blocks - 1, blocks // 2, 7, blocks - 3, blocks * 9 // 10], device=DEV)
    pages[at] = few.transpose(0, 1)
    q = torch.randn(1, 32, 128, generator=g).to(BF16).to(DEV)
    lens = torch.tensor([91], device=DEV)
    got = paged_attention_int4(q, pages, at[None], lens, 16, 0.1)
    want = paged_attention_int4(q, few, torch.arange(6, device=DEV)[None], lens, 16, 0.1)
    assert torch.equal(got, want)


def test_two_graphs_and_a_side_stream():
    g = torch.Generator().manual_seed(16)
    pages = _pages(g, 300, 16, 2, 128)
    lens = torch.tensor([3000, 40, 900], device=DEV)
    tables = _tables(g, [3000, 40, 900], 300, 16, 200).to(DEV)
    qs = [torch.randn(3, 8, 128, generator=g).to(BF16).to(DEV) for _ in range(2)]
    want = [paged_attention_int4(q, pages, tables, lens, 16, 0.1) for q in qs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = paged_attention_int4(qs[0], pages, tables, lens, 16, 0.1)
    side.synchronize()
    assert torch.equal(got, want[0])
    graphs, outs = [], []
    for q in qs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(paged_attention_int4(q, pages, tables, lens, 16, 0.1))
    for rep in range(3):
        for o in outs:
            o.fill_(float("nan"))
        paged_attention_int4(qs[1], pages, tables, lens, 16, 0.3)
        # both at once, on streams of their own
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want)), rep


def test_a_prefill_then_decode_steps_through_4_bit_pages():
    """append, then attend over what the pages hold, token by token."""
    from types import SimpleNamespace

    g = torch.Generator().manual_seed(17)
    heads, q_heads, d, size = 2, 8, 128, 16
    angle = torch.rand(64, d // 2, generator=g) * 6
    rope = SimpleNamespace(head_size=d, rotary_dim=d, is_neox_style=True,
                           cos_sin_cache=torch.cat([angle.cos(), angle.sin()], dim=1).to(DEV))
    pages = torch.zeros(2, 6, size, heads, KL.int4_row_bytes(d), dtype=torch.uint8, device=DEV)
    tables = torch.tensor([[4, 1, 3]], dtype=torch.int32)
    slot = (tables[0].long()[:, None] * size + torch.arange(size)).reshape(-1)
    x = torch.randn(40, q_heads + 2 * heads, d, generator=g).to(BF16).to(DEV)
    q, k, v = x.split([q_heads, heads, heads], dim=1)
    KL.append_paged_kv(k[:37], v[:37], pages, slot[:37], size, torch.arange(37), rope)
    for t in range(37, 40):
        turned = KL.append_paged_kv(k[t:t + 1], v[t:t + 1], pages, slot[t:t + 1], size, torch.tensor([t]), rope,
                                    query=q[t:t + 1])
        got = paged_attention_int4(turned, pages, tables.to(DEV), torch.tensor([t + 1]), size, d ** -0.5)
        held = KL.gather_paged_kv_int4(pages, slot[:t + 1], size, F32).double().cpu().numpy()
        qn = turned.double().cpu().numpy()
        want, mass = R.attend(qn, held[0], held[1], np.array([t]), d ** -0.5)
        tol = _bound(qn[:, None], pages, tables.numpy(), [t + 1], d ** -0.5, BF16, want[:, None], mass[:, None])[:, 0]
        assert np.all(np.abs(got.double().cpu().numpy() - want) <= tol)


def test_int4_attention_refuses():
    pages = torch.zeros(2, 4, 16, 2, 80, dtype=torch.uint8, device=DEV)
    q = torch.zeros(1, 4, 128, dtype=BF16, device=DEV)
    tables, lens = torch.zeros(1, 3, dtype=torch.int32, device=DEV), torch.tensor([5])

    def refuse(error, word, q=q, layer=pages, t=tables, n=lens, **more):
        with pytest.raises(error, match=word):
            paged_attention_int4(q, layer, t, n, 16, 1.0, **more)

    refuse(RuntimeError, "ROCm device tensor", q=q.cpu())
    refuse(ValueError, "query must be", q=q[0])
    refuse(ValueError, "not supported", q=q.double())
    refuse(ValueError, "4-bit pages", layer=pages.view(torch.int8))
    refuse(ValueError, "does not match", q=q[..., :64])
    refuse(ValueError, "must be contiguous", q=q[..., :32], layer=pages[..., :20])
    refuse(ValueError, "64 or 128", q=q[..., :32], layer=pages[..., :20].contiguous())
    refuse(ValueError, "divisible", q=q[:, :3])
    refuse(ValueError, "contiguous dims", q=torch.zeros(1, 128, 4, dtype=BF16, device=DEV).transpose(1, 2))
    refuse(ValueError, "block tables", t=tables[0])
    refuse(ValueError, "lengths", n=torch.tensor([1, 2]))
    refuse(IndexError, "context lengths", n=torch.tensor([49]))
    refuse(IndexError, "context lengths", n=torch.tensor([-1]))
    refuse(IndexError, "pages outside", t=torch.tensor([[4, 0, 0]]))
    refuse(ValueError, "whole numbers", t=tables.float())
    refuse(ValueError, "out must be", out=q[:, :2])
    refuse(ValueError, "must not overlap", out=q[:, :1].expand(1, 4, 128))
    refuse(ValueError, "must not overlap", q=q[:, None].expand(1, 2, 4, 128),
           out=q.new_zeros(1, 1, 4, 128).expand(1, 2, 4, 128))
    with pytest.raises(ValueError, match="finite"):
        paged_attention_int4(q, pages, tables, lens, 16, float("inf"))
    assert paged_attention_int4(q[:0], pages, tables[:0], lens[:0], 16, 1.0).shape == (0, 4, 128)
    # pages past the context's are not looked at
    paged_attention_int4(q, pages, torch.tensor([[3, 99, -1]]), torch.tensor([16]), 16, 1.0)
    assert not paged_attention_int4(q, pages, tables[:, :0], torch.tensor([0]), 16, 1.0).any()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("hkv", [3, 5, 6, 7, 10, 12, 16])
def test_counts_of_kv_heads(hkv, dtype):
    # workgroups of 3 to 8 waves, several of them a range (more than 8 heads), several
    # waves a head; a long sequence that ranges share beside short ones
    _check(dtype, 2 * hkv, hkv, 128, [1, 1900, 0, 63, 33], seed=hkv)
    _check(dtype, 3 * hkv, hkv, 64, [300, 2, 700], rows=2, seed=hkv + 1)
