"""GPU: appending rows to the paged cache with the rotation on the way, in the
cache's type and in 4 bits, and reading 4-bit rows back, against 64 bits.

Tolerances. A rotated value is x c - y s in float32: three roundings of at most
2^-24 of |x c| + |y s| each, then one of half a step of the type (2^-9 relative
for bf16's 8 bits ... eps / 2; float16 below 2^-14: half of 2^-24). Values and
4-bit rows are exact: the products are exact in 64 bits, kernel and restatement
round once, in the same place."""

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from cacheblend_vllm import kv_layout as KL
from oracle import operators as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _rope(rows, head_size, rotary_dim, neox, dtype=F32, seed=0):
    angle = torch.rand(rows, rotary_dim // 2, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * 6 - 3
    return SimpleNamespace(head_size=head_size, rotary_dim=rotary_dim, is_neox_style=neox,
                           cos_sin_cache=torch.cat([angle.cos(), angle.sin()], dim=1).to(dtype).to(DEV))


def _rows(g, *shape, dtype):
    return torch.randn(*shape, generator=g).to(dtype).to(DEV)


def _np(t):
    return t.double().cpu().numpy()


def _close(got, want, terms, dtype, what):
    tol = torch.finfo(dtype).eps / 2 * np.abs(want) + 2.0 ** -22 * terms + (2.0 ** -25 if dtype == F16 else 2.0 ** -130)
    err = np.abs(_np(got) - want)
    worst = float((err / tol).max()) if err.size else 0.0
    print(f"{what}: worst {worst:.3f} of the bound", flush=True)
    assert np.all(err <= tol)


def _layout(name, blocks, size, row, dtype, fill):
    if name == "merged_block":
        return torch.full((blocks, 2, size, *row), fill, dtype=dtype, device=DEV)
    pool = torch.full((2, blocks, size, *row), fill, dtype=dtype, device=DEV)
    return pool if name == "merged_first" else (pool[0], pool[1])


def _check(tokens, q_heads, heads, d, dtype, rotary_dim, neox, layout="merged_first", int4=False, size=16, seed=0,
           table=F32, wide=0, rows=400):
    """One call against the restatement, everything around the rows untouched."""
    print(f"append {tokens} {q_heads}/{heads}x{d} {dtype} rot {rotary_dim} neox {neox} {layout} int4 {int4} wide {wide}",
          flush=True)
    g = torch.Generator().manual_seed(seed)
    blocks = (tokens + size - 1) // size + 3
    row = (heads, KL.int4_row_bytes(d)) if int4 else (heads, d)
    pages = _layout(layout, blocks, size, row, torch.uint8 if int4 else dtype, 3)
    # queries, keys and values side by side (wide: more between the tokens)
    qkv = _rows(g, tokens, (q_heads + 2 * heads) * d + wide, dtype=dtype)
    q, k, v = qkv[:, :(q_heads + 2 * heads) * d].unflatten(1, (-1, d)).split([q_heads, heads, heads], dim=1)
    slots = torch.randperm(blocks * size, generator=g)[:tokens]
    pos = torch.randint(0, rows, (tokens,), generator=g)
    rope = _rope(rows, d, rotary_dim, neox, table, seed) if rotary_dim else None
    key_out = torch.empty(tokens, heads, d, dtype=dtype, device=DEV)
    out = KL.append_paged_kv(k, v, pages, slots, size, positions=pos if rope else None, rotary_emb=rope,
                             query=q if q_heads else None, key_out=key_out)
    torch.cuda.synchronize()
    table_np, pos_np = (_np(rope.cos_sin_cache), pos.numpy()) if rope else (np.zeros((rows, 0)), pos.numpy())
    want_k = R.rotate(_np(k), table_np, pos_np, neox)
    terms = R.rotate_terms(_np(k), table_np, pos_np, neox) * bool(rotary_dim)
    _close(key_out, want_k, terms, dtype, "key_out")
    if q_heads:
        _close(out, R.rotate(_np(q), table_np, pos_np, neox),
               R.rotate_terms(_np(q), table_np, pos_np, neox) * bool(rotary_dim), dtype, "query")
    else:
        assert out is None
    planes = [p.flatten(0, 1) for p in KL.kv_planes(pages)]
    here = slots.to(DEV)
    rest = torch.ones(blocks * size, dtype=torch.bool, device=DEV)
    rest[here] = False
    for p in planes:
        assert bool((p[rest] == 3).all())
    if int4:
        assert np.array_equal(planes[0][here].cpu().numpy(), R.int4_encode(want_k))
        assert np.array_equal(planes[1][here].cpu().numpy(), R.int4_encode(_np(v)))
    else:
        assert torch.equal(planes[0][here], key_out)
        assert torch.equal(planes[1][here], v)
    return pages, here


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("tokens,q_heads,heads,d", [(1, 32, 8, 128), (77, 6, 2, 64), (333, 5, 1, 128), (40, 0, 3, 16)])
def test_append_in_the_caches_type(tokens, q_heads, heads, d, neox, dtype):
    _check(tokens, q_heads, heads, d, dtype, d, neox, seed=tokens + d)


@pytest.mark.parametrize("layout", ["merged_first", "merged_block", "separate"])
@pytest.mark.parametrize("int4", [False, True])
def test_append_layouts_and_block_sizes(layout, int4):
    _check(50, 8, 2, 64, BF16, 64, True, layout, int4, size=5)
    _check(50, 8, 2, 64, F16, 0, True, layout, int4, size=1)


# sizes that leave the 16-byte pieces: partial rotation, odd halves, odd dims, rows at odd strides
@pytest.mark.parametrize("d,rotary,neox,wide,dtype,int4", [
    (128, 64, True, 0, BF16, False), (80, 80, True, 0, F16, False), (80, 20, False, 0, F32, False),
    (10, 6, True, 0, BF16, False), (3, 2, False, 0, F16, False), (512, 512, True, 0, BF16, False),
    (128, 128, True, 3, BF16, False), (64, 64, False, 1, F32, False), (1, 0, True, 0, BF16, False),
    (32, 32, True, 0, BF16, True), (96, 96, True, 0, F16, True), (96, 96, False, 0, F32, True),
    (160, 40, True, 0, BF16, True), (128, 128, True, 5, F16, True), (256, 256, False, 0, BF16, True),
    (512, 512, True, 0, F32, True),
])
def test_append_general_rows(d, rotary, neox, wide, dtype, int4):
    _check(37, 3, 2, d, dtype, rotary, neox, int4=int4, wide=wide, seed=d)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("tokens,d", [(1, 128), (333, 64), (61, 128)])
def test_append_in_4_bits_and_read_back(tokens, d, neox, dtype):
    pages, slots = _check(tokens, 4, 2, d, dtype, d, neox, int4=True, seed=tokens)
    rows = np.stack([p.flatten(0, 1)[slots].cpu().numpy() for p in KL.kv_planes(pages)])
    for want_type in (BF16, F16, F32):
        got = KL.gather_paged_kv_int4(pages, slots, 16, want_type)
        want = torch.from_numpy(R.int4_decode(rows).astype(np.float32)).to(want_type)
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("table", [BF16, F16, torch.float64])
def test_append_table_types(table):
    _check(20, 4, 2, 64, BF16, 64, True, table=table)
    _check(20, 4, 2, 20, F32, 12, True, table=table)


def test_values_of_4_bit_rows_out_of_the_ordinary():
    # constant rows, whole numbers, huge and tiny ranges, infinities and NaN
    v = torch.zeros(8, 1, 64)
    v[0], v[1, 0, 3], v[2, 0, 40], v[3, 0, 5] = 7.3, float("nan"), float("inf"), float("-inf")
    v[4, 0] = (torch.arange(64) % 16) - 4.0
    v[5, 0] = torch.linspace(-3e38, 3e38, 64)
    v[6, 0] = torch.linspace(-1e-38, 2e-38, 64)
    v[7, 0] = -3.4e38
    v = v.to(DEV)
    pages = torch.zeros(2, 2, 4, 1, 40, dtype=torch.uint8, device=DEV)
    KL.append_paged_kv(v, v, pages, torch.arange(8), 4)
    rows = pages.flatten(1, 2).cpu().numpy()
    want = R.int4_encode(_np(v))
    # a NaN's sign and payload are not part of the format
    values = [R.int4_decode(x) for x in (rows[0], rows[1], want)]
    assert np.array_equal(values[0], values[2], equal_nan=True) and np.array_equal(values[1], values[2], equal_nan=True)
    got = KL.gather_paged_kv_int4(pages, torch.arange(8), 4, F32).cpu().numpy()
    assert np.array_equal(got[0], values[2].astype(np.float32), equal_nan=True)


def test_outputs_in_place_and_rows_that_share_an_input():
    g = torch.Generator().manual_seed(5)
    for d, rot in ((128, 128), (80, 48)):
        for neox in (True, False):
            qkv = _rows(g, 65, 10, d, dtype=BF16)
            keep = qkv.clone()
            q, k, v = qkv.split([6, 2, 2], dim=1)
            pages = torch.zeros(2, 6, 16, 2, d, dtype=BF16, device=DEV)
            rope, pos = _rope(100, d, rot, neox), torch.arange(65, device=DEV)
            out = KL.append_paged_kv(k, v, pages, torch.arange(65), 16, pos, rope, query=q, query_out=q, key_out=k)
            assert out is q
            fresh = torch.zeros_like(pages)
            kq = torch.empty_like(k)
            want = KL.append_paged_kv(keep[:, 6:8], keep[:, 8:], fresh, torch.arange(65), 16, pos, rope,
                                      query=keep[:, :6], key_out=kq)
            assert torch.equal(q, want) and torch.equal(k, kq) and torch.equal(v, keep[:, 8:])
            assert torch.equal(pages, fresh)
    # one value row for every token and head
    one = _rows(g, 1, 1, 64, dtype=F16).expand(20, 3, 64)
    pages = torch.zeros(2, 2, 16, 3, 64, dtype=F16, device=DEV)
    KL.append_paged_kv(one, one, pages, torch.arange(20), 16)
    assert bool((pages.flatten(1, 2)[:, :20] == one).all())


@pytest.mark.parametrize("int4", [False, True])
def test_padding_and_places_out_of_range_on_the_device(int4):
    g = torch.Generator().manual_seed(6)
    d, heads = 64, 2
    row = KL.int4_row_bytes(d) if int4 else d
    pages = torch.full((2, 4, 8, heads, row), 9, dtype=torch.uint8 if int4 else BF16, device=DEV)
    k, v, q = (_rows(g, 7, heads, d, dtype=BF16) for _ in range(3))
    slots = torch.tensor([3, -1, 32, 5, 1 << 40, 7, 31], device=DEV)
    pos = torch.tensor([0, 1, 2, -1, 3, 50, 49], device=DEV)
    kept = torch.empty_like(k)
    out = KL.append_paged_kv(k, v, pages, slots, 8, pos, _rope(50, d, d, True), query=q, key_out=kept)
    flat = pages.flatten(1, 2)
    written = [i for i in range(32) if not bool((flat[:, i] == 9).all())]
    assert written == [3, 31]  # not 5 and 7: their positions are outside the table
    for x in (out, kept):
        assert not x[3].any() and not x[5].any() and x[1].any() and x[2].any()
    if int4:
        got = KL.gather_paged_kv_int4(pages, slots, 8, F32)
        assert not got[:, [1, 2, 4]].any() and got[:, 0].any()


def test_gather_into_views_and_other_strides():
    g = torch.Generator().manual_seed(7)
    pages = torch.randint(0, 256, (5, 2, 4, 3, 40), generator=g, dtype=torch.uint8)
    both = torch.randn(5, 2, 4, 3, 4, generator=g).to(BF16).view(torch.uint8)
    pages[..., 32:] = both
    pages = pages.to(DEV)
    slots = torch.tensor([0, 19, 7, 7, 3])
    want = KL.gather_paged_kv_int4(pages, slots, 4, F16)
    rows = pages.transpose(0, 1).flatten(1, 2)[:, slots.to(DEV)].cpu().numpy()
    assert torch.equal(want.cpu(), torch.from_numpy(R.int4_decode(rows).astype(np.float32)).to(F16))
    for out in (torch.zeros(2, 5, 3, 64, dtype=F16, device=DEV),
                torch.zeros(5, 2, 3, 64, dtype=F16, device=DEV).transpose(0, 1),
                torch.zeros(2, 5, 3, 65, dtype=F16, device=DEV)[..., 1:],
                torch.zeros(2, 9, 3, 64, dtype=F16, device=DEV)[:, 2:7]):
        assert KL.gather_paged_kv_int4(pages, slots, 4, out=out) is out
        assert torch.equal(out, want)
    assert KL.gather_paged_kv_int4(pages, slots[:0], 4).shape == (2, 0, 3, 64)


def test_4_bit_rows_move_as_any_paged_rows():
    # stored and brought back by the byte movers, then read as values
    pages, slots = _check(45, 4, 2, 128, BF16, 128, True, int4=True)
    chunk = KL.gather_paged_kv(pages, slots, 16)
    other = torch.zeros(2, 9, 16, 2, 80, dtype=torch.uint8, device=DEV)
    moved = torch.randperm(9 * 16)[:45]
    KL.scatter_paged_kv(chunk, other, moved, 16)
    assert torch.equal(KL.gather_paged_kv_int4(other, moved, 16), KL.gather_paged_kv_int4(pages, slots, 16))


def test_append_on_a_side_stream_and_in_a_graph():
    g = torch.Generator().manual_seed(8)
    k, v, q = _rows(g, 9, 2, 128, dtype=BF16), _rows(g, 9, 2, 128, dtype=BF16), _rows(g, 9, 4, 128, dtype=BF16)
    pos, slots = torch.arange(9, device=DEV), torch.arange(3, 12, device=DEV)
    rope = _rope(64, 128, 128, True)
    for int4 in (False, True):
        pages = torch.zeros(2, 2, 16, 2, 80 if int4 else 128, dtype=torch.uint8 if int4 else BF16, device=DEV)
        want = KL.append_paged_kv(k, v, pages, slots, 16, pos, rope, query=q)
        held = pages.clone()
        side = torch.cuda.Stream()
        pages.zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = KL.append_paged_kv(k, v, pages, slots, 16, pos, rope, query=q)
        side.synchronize()
        assert torch.equal(got, want) and torch.equal(pages, held)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = KL.append_paged_kv(k, v, pages, slots, 16, pos, rope, query=q)
        for rep in range(3):
            pages.zero_()
            out.zero_()
            q.mul_(2)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want * 2 ** (rep + 1)) and torch.equal(pages, held), rep
        q.div_(8)


def test_append_and_gather_refuse():
    k = torch.zeros(3, 2, 64, dtype=BF16, device=DEV)
    pages = torch.zeros(2, 4, 16, 2, 64, dtype=BF16, device=DEV)
    p4 = torch.zeros(2, 4, 16, 2, 40, dtype=torch.uint8, device=DEV)
    slots, pos, rope = torch.arange(3), torch.arange(3), _rope(10, 64, 64, True)

    def refuse(error, word, key=k, value=k, layer=pages, s=slots, **more):
        with pytest.raises(error, match=word):
            KL.append_paged_kv(key, value, layer, s, 16, **more)

    refuse(IndexError, "slot_mapping", s=torch.tensor([0, 1, 64]))
    refuse(IndexError, "slot_mapping", s=torch.tensor([0, 1, -1]))
    refuse(ValueError, "slots for", s=torch.arange(2))
    refuse(IndexError, "positions", positions=torch.tensor([0, 1, 10]), rotary_emb=rope)
    refuse(ValueError, "positions for", positions=torch.arange(2), rotary_emb=rope)
    refuse(ValueError, "come together", positions=pos)
    refuse(ValueError, "come together", rotary_emb=rope)
    refuse(ValueError, "rotary_dim", positions=pos, rotary_emb=_rope(10, 128, 128, True))
    refuse(ValueError, "cos_sin_cache is", positions=pos,
           rotary_emb=SimpleNamespace(head_size=64, rotary_dim=32, is_neox_style=True, cos_sin_cache=rope.cos_sin_cache))
    refuse(ValueError, "two-dimensional", positions=pos,
           rotary_emb=SimpleNamespace(head_size=64, is_neox_style=True, cos_sin_cache=None))
    refuse(ValueError, "key must be", key=k.flatten(1))
    refuse(ValueError, "not supported", key=k.double(), value=k.double())
    refuse(ValueError, "dtype and device", value=k.half())
    refuse(ValueError, "value has shape", value=k[:, :1])
    refuse(ValueError, "the pages hold", key=k.half(), value=k.half())
    refuse(ValueError, "the pages hold", key=k[:, :1], value=k[:, :1])
    refuse(ValueError, "do not hold rows", layer=p4[:, :, :, :1])
    refuse(ValueError, "4-bit pages", layer=p4[..., :36].contiguous())
    refuse(ValueError, "contiguous dims", value=torch.zeros(3, 64, 2, dtype=BF16, device=DEV).transpose(1, 2))
    refuse(ValueError, "query has shape", query=k[:2])
    refuse(ValueError, "needs a query", query_out=k.clone())
    refuse(ValueError, "must not overlap", key_out=k[:1].expand(3, 2, 64))
    refuse(ValueError, "must not overlap", query=k, query_out=k[:, :1].expand(3, 2, 64))
    with pytest.raises(ValueError, match="4-bit pages"):
        KL.gather_paged_kv_int4(pages, slots, 16)
    with pytest.raises(ValueError, match="not supported"):
        KL.gather_paged_kv_int4(p4, slots, 16, torch.float64)
    with pytest.raises(ValueError, match="expected"):
        KL.gather_paged_kv_int4(p4, slots, 16, out=torch.zeros(2, 3, 2, 128, device=DEV))
    with pytest.raises(IndexError, match="slot_mapping"):
        KL.gather_paged_kv_int4(p4, torch.tensor([64]), 16)
    assert KL.append_paged_kv(k[:0], k[:0], pages, slots[:0], 16) is None
    empty = KL.append_paged_kv(k[:0], k[:0], p4, slots[:0], 16, query=k[:0])
    assert empty.shape == (0, 2, 64)


@pytest.mark.parametrize("int4", [False, True])
@pytest.mark.parametrize("d,rotary", [(128, 128), (40, 24)])  # 16-byte pieces, and row by row
def test_outputs_whose_heads_lie_outside_the_tokens(d, rotary, int4):
    g = torch.Generator().manual_seed(31)
    d = 96 if int4 and d % 32 else d
    row = (2, KL.int4_row_bytes(d)) if int4 else (2, d)
    pages = [torch.zeros(2, 3, 16, *row, dtype=torch.uint8 if int4 else BF16, device=DEV) for _ in range(3)]
    q, k, v = (_rows(g, 33, h, d, dtype=BF16) for h in (4, 2, 2))
    slots, pos, rope = torch.randperm(48, generator=g)[:33], torch.arange(33), _rope(40, d, rotary, True)
    key = torch.empty_like(k)
    want = KL.append_paged_kv(k, v, pages[0], slots, 16, pos, rope, query=q, key_out=key)
    q_out, k_out = (torch.empty(h, 33, d, dtype=BF16, device=DEV).transpose(0, 1) for h in (4, 2))
    got = KL.append_paged_kv(k, v, pages[1], slots, 16, pos, rope, query=q, query_out=q_out, key_out=k_out)
    assert got is q_out and torch.equal(got, want) and torch.equal(k_out, key) and torch.equal(pages[1], pages[0])
    # in place, the inputs head by head
    q2, k2 = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k))
    KL.append_paged_kv(k2, v, pages[2], slots, 16, pos, rope, query=q2, query_out=q2, key_out=k2)
    assert torch.equal(q2, want) and torch.equal(k2, key) and torch.equal(pages[2], pages[0])
