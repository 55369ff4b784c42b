"""What attention over paged KV and eviction promise, by cases whose answers are known without them,
and the entry points' refusals, which come before anything is launched."""

import math

import numpy as np
import pytest
import torch

from cacheblend_vllm import _native
from cacheblend_vllm.attention import paged_attention
from cacheblend_vllm.kv_layout import evict_paged_kv
from oracle import operators as R


@pytest.mark.parametrize("weights,length,keep,first,recent,want", [
    ([5, 1, 4, 2, 3], 5, 3, 0, 0, [0, 2, 4]),            # the heaviest, in their order
    ([1, 5, 4, 3, 2], 5, 3, 1, 1, [0, 1, 4]),            # the ends stay, whatever they weigh
    ([9, 9, 9, 9, 9], 5, 2, 0, 0, [0, 1]),               # ties: the lower index
    ([0.0, -0.0, 0.0, -1.0], 4, 2, 0, 0, [0, 1]),        # -0 is 0
    ([math.inf, 1, math.nan, 2], 4, 2, 0, 0, [0, 2]),    # NaN above infinity
    ([-math.inf, 1, -2, 2], 4, 3, 0, 0, [1, 2, 3]),
    ([1, 2, 3], 3, 3, 0, 0, [0, 1, 2]),                  # nothing to do
    ([1, 2, 3, 4], 2, 1, 0, 0, [1]),                     # keys behind the length do not count
    ([1, 2, 3, 4], 4, 1, 2, 1, [0, 1, 3]),               # the ends come before the keep
    ([], 0, 0, 0, 0, []),
])
def test_which_keys_stay(weights, length, keep, first, recent, want):
    assert R.evict(np.array(weights), length, keep, first, recent).tolist() == want


def test_attention_from_pages_of_one_key_each():
    """Equal keys: rows average the values they see, and every key gets each row's equal share."""
    rows, heads, group, n, d = 2, 2, 3, 5, 4
    v = np.arange(n * heads * d, dtype=np.float64).reshape(n, heads, d)
    tables = np.array([[3, 0, 99, 4, 1, 2]])  # the third key's page does not exist
    pages = np.zeros((2, n, 1, heads, d))
    for key, page in enumerate(tables[0, :n]):
        if page < n:
            pages[1, page, 0] = v[key]
    q = np.random.default_rng(0).standard_normal((1, rows, heads * group, d))
    out, mass, added = R.paged_attention(q, pages[0], pages[1], tables, [n], 0.5)
    for r, seen in enumerate(([0, 1, 3], [0, 1, 3, 4])):
        for h in range(heads * group):
            np.testing.assert_allclose(out[0, r, h], v[seen, h // group].mean(0), rtol=1e-14)
    want = group * np.array([1 / 3 + 1 / 4, 1 / 3 + 1 / 4, 0, 1 / 3 + 1 / 4, 1 / 4, 0])
    np.testing.assert_allclose(added[0], np.stack([want] * heads), rtol=1e-14)
    np.testing.assert_allclose(mass, np.abs(out), rtol=1e-14)


def test_attention_from_pages_agrees_with_the_4_bit_pages_restatement():
    """The same keys and values, once as 4-bit pages and once as what these decode to."""
    rng = np.random.default_rng(1)
    k, v = (rng.standard_normal((6, 4, 2, 32)).astype(np.float32) for _ in range(2))
    coded = [R.int4_encode(x) for x in (k, v)]
    plain = [R.int4_decode(x) for x in coded]
    q = rng.standard_normal((2, 3, 4, 32))
    tables, lens = np.array([[5, 0, 2], [-1, 3, 1]]), [11, 2]
    a, _ = R.paged_attention_int4(q, *coded, tables, lens, 0.2)
    b, _, added = R.paged_attention(q, *plain, tables, lens, 0.2)
    np.testing.assert_allclose(a, b, rtol=1e-13, atol=1e-15)
    # a sequence that sees no key at all; the other's weights sum to its rows and heads
    assert not b[1].any() and not added[1].any()
    assert math.isclose(added[0].sum(), 3 * 4, rel_tol=1e-13)


def test_cpu_tensors_are_refused():
    q, pages = torch.zeros(2, 1, 4, 64), torch.zeros(2, 3, 4, 2, 64)
    tables, lens = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="ROCm device tensor"):
        paged_attention(q, pages, tables, lens, 4, 1.0)
    with pytest.raises(RuntimeError, match="ROCm device tensor"):
        evict_paged_kv(pages, tables, lens, 4, torch.zeros(2, 2, 12), 4)


def _desc():
    return _native.KVDesc(0x10000, 0x20000, 8, 16, 16 * 512, 512, 512)


def _attention(lib, **over):
    a = dict(q=0x1000, qb=512, qr=512, qh=128, batch=2, rows=1, hq=4, kv=_desc(), hkv=2, dim=128, tables=0x2000, ts=4, width=4,
             lens=0x3000, scale=0.1, dtype=1, out=0x4000, ob=512, orow=512, oh=128, weights=0x5000, wb=128, wset=64, sets=2,
             ws=0x100000, nbytes=1 << 40, stream=None)
    a.update(over)
    return lib.cbk_paged_attention(*a.values())


@pytest.mark.parametrize("over,word", [
    (dict(kv=None), b"NULL"), (dict(dtype=3), b"dtype"), (dict(dim=96), b"64 or 128"), (dict(hkv=3), b"bytes"),
    (dict(dtype=0), b"bytes"), (dict(scale=float("inf")), b"finite"), (dict(width=-1), b"width"), (dict(ts=-1), b"width"),
    (dict(hq=5), b"divisible"), (dict(rows=0), b"rows"), (dict(rows=1 << 16), b"rows"), (dict(batch=-1), b"batch"),
    (dict(batch=1 << 16), b"batch"), (dict(width=1 << 28, ts=1 << 28), b"context"), (dict(sets=3), b"3 sets"),
    (dict(sets=0), b"0 sets"),
])
def test_attention_entry_refuses(over, word):
    lib = _native.load()
    assert _attention(lib, **over) == _native.CBK_ERR_INVALID
    assert word in lib.cbk_last_error(), lib.cbk_last_error()


def _evict(lib, **over):
    a = dict(kv=_desc(), tables=0x2000, ts=4, width=4, lens=0x3000, batch=2, weights=0x5000, wb=128, wset=64, sets=2, keep=20,
             keeps=None, first=4, recent=8, new=0x6000, ws=0x100000, nbytes=0, stream=None)
    a.update(over)
    return lib.cbk_paged_evict(*a.values())


@pytest.mark.parametrize("over,word", [
    (dict(kv=None), b"NULL"), (dict(keep=-1), b"keep"), (dict(keeps=0x7000), b"keep"), (dict(keep=11), b"keep 11"),
    (dict(first=-1), b"first and recent"), (dict(recent=-1), b"first and recent"), (dict(first=1 << 31), b"first and recent"),
    (dict(sets=3), b"3 sets"), (dict(sets=0), b"0 sets"), (dict(width=-1), b"width"), (dict(ts=-1), b"width"),
    (dict(width=1 << 28), b"context"), (dict(batch=-1), b"batch"), (dict(batch=1 << 30), b"batch"),
    (dict(batch=1 << 20, width=1 << 20, keep=1 << 24), b"too many tiles"), (dict(batch=1 << 21), b"batch"), (dict(lens=None), b"NULL"), (dict(new=None), b"NULL"),
    (dict(weights=None), b"NULL"), (dict(tables=None), b"NULL"),
])
def test_evict_entry_refuses(over, word):
    lib = _native.load()
    assert _evict(lib, **over) == _native.CBK_ERR_INVALID
    assert word in lib.cbk_last_error(), lib.cbk_last_error()
    assert _evict(lib, batch=0) == _native.CBK_OK


def test_evict_workspace():
    lib = _native.load()
    need = lib.cbk_paged_evict_workspace_bytes(_desc(), 4, 2, 2, 20)
    assert need > 0
    assert _evict(lib, nbytes=need - 1) == _native.CBK_ERR_WORKSPACE
    assert _evict(lib, ws=None, nbytes=need) == _native.CBK_ERR_WORKSPACE
    assert _evict(lib, ws=0x100080, nbytes=need) == _native.CBK_ERR_INVALID and b"256" in lib.cbk_last_error()
    # lengths of their own may be as long as the tables; what is refused has no size
    assert lib.cbk_paged_evict_workspace_bytes(_desc(), 4, 2, 2, -1) >= need
    assert lib.cbk_paged_evict_workspace_bytes(_desc(), 4, 2, 3, 20) == 0


@pytest.mark.parametrize("over", [dict(new=0x3000), dict(new=0x3004), dict(new=0x2ffc),
                                  dict(new=0x7000, keep=-1, keeps=0x7000), dict(new=0x7004, keep=-1, keeps=0x7000)])
def test_new_lengths_over_what_is_still_read(over):
    """Sets of heads read a sequence's length and keep by themselves, while the first of them writes the new length."""
    lib = _native.load()
    assert _evict(lib, **over) == _native.CBK_ERR_INVALID
    assert b"new lengths" in lib.cbk_last_error(), lib.cbk_last_error()
    # beside them they are as good as anywhere (the scratch is missing next)
    for new in (0x3008, 0x2ff8, 0x7008):
        assert _evict(lib, new=new, keep=-1, keeps=0x7000) == _native.CBK_ERR_WORKSPACE


@pytest.mark.parametrize("over", [dict(ob=1024), dict(oh=192), dict(rows=2, orow=1024)])
def test_outputs_in_the_queries_place_with_other_strides(over):
    lib = _native.load()
    base = dict(weights=None, out=0x1000)
    assert _attention(lib, **base, **over) == _native.CBK_ERR_INVALID
    assert b"strides" in lib.cbk_last_error(), lib.cbk_last_error()


def test_which_outputs_meet_the_queries():
    from cacheblend_vllm.attention import _meets_otherwise

    def meets(query, out):
        """By the addresses of all elements."""
        mine, its = (torch.arange(4096).as_strided(t.shape, t.stride(), t.storage_offset()) for t in (query, out))
        return bool(torch.isin(mine, its).any()) and not torch.equal(mine, its)

    room = torch.zeros(4096)
    a = room[:1024].view(4, 4, 64)
    sure = [(a, a), (a, room[1024:2048].view(4, 4, 64)), (a, room[:1024].view(4, 4, 64).transpose(0, 1)), (a, room[256:1280].view(4, 4, 64)),
            (a, room[64:1088].view(4, 4, 64)), (a, room[1:1025].view(4, 4, 64)), (room[256:1280].view(4, 4, 64), a)]
    both = room.view(8, 2, 4, 64)
    sure += [(both[:, 0], both[:, 1]), (both[:, 1], both[:, 0]), (both[:4, 0], both[4:, 0]), (both[:7, 1], both[1:, 0])]
    beside = room.view(8, 4, 128)
    sure += [(beside[..., :64], beside[..., 64:]), (beside[:, :2], beside[:, 2:]), (beside[:, :3], beside[:, 1:])]
    for query, out in sure:
        assert _meets_otherwise(out, query) == meets(query, out), (query.shape, query.stride(), out.stride(), out.storage_offset())
    # one head or one sequence: its stride does not count
    one = room[:64].view(1, 1, 64)
    assert not _meets_otherwise(one.as_strided((1, 1, 64), (7, 9, 1)), one)
    assert not _meets_otherwise(room[:0].view(0, 4, 64), room[:0].view(0, 4, 64))
    # memory that is not the same at all
    assert not _meets_otherwise(torch.zeros(4, 4, 64), a)


@pytest.mark.parametrize("apart", [0, 511, -256])
def test_keys_and_values_in_the_same_rows_do_not_move(apart):
    """The two planes move by themselves, so that one would write rows that the other has yet to read."""
    lib = _native.load()
    kv = _native.KVDesc(0x10000, 0x10000 + apart, 8, 16, 16 * 1024, 1024, 512)
    assert _evict(lib, kv=kv) == _native.CBK_ERR_INVALID
    assert b"same rows" in lib.cbk_last_error(), lib.cbk_last_error()
    assert lib.cbk_paged_evict_workspace_bytes(kv, 4, 2, 2, 20) == 0
    # beside each other they do (the scratch is missing next)
    for apart in (512, -512):
        kv = _native.KVDesc(0x10000, 0x10000 + apart, 8, 16, 16 * 1024, 1024, 512)
        assert _evict(lib, kv=kv) == _native.CBK_ERR_WORKSPACE
