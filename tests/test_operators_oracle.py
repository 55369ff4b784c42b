"""CPU: the 64-bit restatement of the operators over a request's own keys and
values against closed forms and torch, and the C entries' refusals (no kernel
is launched)."""

import numpy as np
import pytest
import torch

from cacheblend_vllm import _native
from cacheblend_vllm.kv_layout import append_paged_kv, gather_paged_kv_int4, int4_geometry, int4_row_bytes
from oracle import operators as R


def _table(rows, n, seed=0):
    angle = np.random.default_rng(seed).uniform(-3, 3, (rows, n // 2))
    return np.concatenate([np.cos(angle), np.sin(angle)], axis=1)


@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("d,n", [(64, 64), (40, 24), (6, 2)])
def test_rotation_is_a_turn_of_each_pair(d, n, neox):
    x = np.random.default_rng(1).standard_normal((5, 3, d))
    table, pos = _table(9, n), np.array([0, 8, 3, 3, 7])
    got = R.rotate(x, table, pos, neox)
    a, b = (x[..., :n // 2], x[..., n // 2:n]) if neox else (x[..., 0:n:2], x[..., 1:n:2])
    turned = (a + 1j * b) * (table[pos, :n // 2] + 1j * table[pos, n // 2:])[:, None]
    c, e = (got[..., :n // 2], got[..., n // 2:n]) if neox else (got[..., 0:n:2], got[..., 1:n:2])
    np.testing.assert_allclose(c + 1j * e, turned, rtol=0, atol=1e-14)
    assert np.array_equal(got[..., n:], x[..., n:])
    assert np.all(R.rotate_terms(x, table, pos, neox) >= np.abs(got) - 1e-12)


@pytest.mark.parametrize("scale", [1.0, 1e-30, 1e30, 1e-39])
def test_4_bit_rows_hold_values_within_half_a_step(scale):
    x = np.random.default_rng(2).standard_normal((50, 128)) * scale
    x[3] = 7.25 * scale
    x[4, 40:50] *= 1000
    rows = R.int4_encode(x)
    assert rows.shape == (50, int4_row_bytes(128))
    got = R.int4_decode(rows)
    parts = x.reshape(50, 4, 32)
    span = parts.max(axis=-1) - parts.min(axis=-1)
    # the offset's rounding widens the span by up to 2^-7 of the lowest value; the
    # step is rounded up by up to 2^-7 (2^-126: where steps end)
    step = (span + np.abs(parts.min(axis=-1)) * 2.0 ** -7) / 15 * (1 + 2.0 ** -7) + 2.0 ** -126
    whole = scale >= 1e-30
    bound = (step / 2 * (1 + 2.0 ** -20)).repeat(32, axis=-1) if whole else (16 * step).repeat(32, axis=-1)
    assert np.all(np.abs(got - x) <= bound)


def test_4_bit_rows_of_special_values():
    x = np.zeros((5, 64))
    x[1, 3], x[2, 40], x[3, 5] = np.nan, np.inf, -np.inf
    x[4, :32] = np.arange(32) % 16 - 4.0  # whole numbers: step 1, held as they are
    got = R.int4_decode(R.int4_encode(x))
    assert np.array_equal(got[0], np.zeros(64))
    assert np.isnan(got[1, :32]).all() and np.array_equal(got[1, 32:], np.zeros(32))
    assert np.isnan(got[2, 32:]).all() and np.isnan(got[3, :32]).all()
    assert np.array_equal(got[4], x[4])
    huge = np.full((1, 32), -3.4e38)  # below bf16's range
    assert np.isnan(R.int4_decode(R.int4_encode(huge))).all()
    assert np.array_equal(R.int4_decode(np.zeros((2, 20), dtype=np.uint8)), np.zeros((2, 32)))


def test_attention_restatement_against_torch():
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(n, h, 16, generator=g, dtype=torch.float64) for n, h in ((12, 4), (20, 2), (20, 2)))
    ends_q, ends_k = [0, 5, 5, 12], [0, 9, 12, 20]
    got, mass = R.prompt_attention(q.numpy(), k.numpy(), v.numpy(), ends_q, ends_k, 0.3)
    for a, b, c, d in ((0, 5, 0, 9), (5, 12, 12, 20)):
        x = torch.einsum("qhd,khd->hqk", q[a:b], k[c:d].repeat_interleave(2, dim=1)) * 0.3
        late = torch.arange(d - c)[None] > torch.arange(b - a)[:, None] + (d - c) - (b - a)
        p = x.masked_fill(late, float("-inf")).softmax(dim=-1)
        want = torch.einsum("hqk,khd->qhd", p, v[c:d].repeat_interleave(2, dim=1))
        np.testing.assert_allclose(got[a:b], want.numpy(), rtol=1e-12, atol=1e-14)
    assert np.all(mass >= np.abs(got) - 1e-12)
    # more queries than keys: the first rows see none
    got, _ = R.prompt_attention(q.numpy(), k.numpy(), v.numpy(), [0, 12], [0, 2], 0.3)
    assert not got[:10].any() and got[10:].any()


def test_paged_4_bit_attention_restatement():
    g = np.random.default_rng(4)
    pages = R.int4_encode(g.standard_normal((2, 7, 4, 2, 32)))
    q = g.standard_normal((3, 2, 4, 32))
    tables = np.array([[5, 0, 2], [1, -1, 9], [3, 3, 3]])
    got, _ = R.paged_attention_int4(q, pages[0], pages[1], tables, [9, 6, 1], 0.2)
    k, v = (R.int4_decode(p[[5, 0, 2]].reshape(12, 2, 20)[:9]) for p in pages)
    np.testing.assert_allclose(got[0], R.attend(q[0], k, v, [7, 8], 0.2)[0], rtol=1e-13)
    k, v = (R.int4_decode(p[1]) for p in pages)  # the pages past the first hold no keys
    np.testing.assert_allclose(got[1], R.attend(q[1], k, v, [3, 3], 0.2)[0], rtol=1e-13)
    assert not got[2, 0].any()  # a context of one token: the first of two rows sees nothing


# ----------------------------------------------------------------- refusals


def test_4_bit_geometry():
    assert [int4_row_bytes(d) for d in (32, 64, 128)] == [20, 40, 80]
    for d in (0, -32, 33, 48):
        with pytest.raises(ValueError, match="multiple of 32"):
            int4_row_bytes(d)
    assert int4_geometry(torch.uint8, (2, 80)) == (2, 128)
    for bad in ((torch.float32, (2, 80)), (torch.uint8, (160,)), (torch.uint8, (2, 72)), (torch.uint8, (2, 0))):
        with pytest.raises(ValueError, match="4-bit pages"):
            int4_geometry(*bad)


def test_cpu_tensors_are_refused():
    rows, pages = torch.zeros(2, 1, 32), torch.zeros(2, 3, 4, 1, 32)
    with pytest.raises(RuntimeError, match="ROCm device tensor"):
        append_paged_kv(rows, rows, pages, torch.tensor([0, 1]), 4)
    with pytest.raises(RuntimeError, match="ROCm device tensor"):
        gather_paged_kv_int4(torch.zeros(2, 3, 4, 1, 20, dtype=torch.uint8), torch.tensor([0]), 4)


def _append(lib, desc, **over):
    a = dict(slots=0x1000, tokens=4, key=0x2000, kt=256, kh=128, value=0x3000, vt=256, vh=128, query=0x4000, qt=512,
             qh=128, q_heads=4, heads=2, dim=128, dtype=1, int4=0, pos=0x5000, table=0x6000, row=128, rows=100, tdt=0,
             rot=128, neox=1, qo=0x7000, qot=512, qoh=128, ko=None, kot=0, koh=0, stream=None)
    a.update(over)
    return lib.cbk_paged_append(desc, *a.values())


@pytest.mark.parametrize("over,word", [
    (dict(tokens=-1), b"num_tokens"), (dict(dtype=7), b"dtype 7"), (dict(heads=0), b"heads"),
    (dict(dim=0), b"head_dim"), (dict(dim=513), b"head_dim"), (dict(dim=64), b"rows are"),
    (dict(slots=None), b"NULL"), (dict(value=None), b"NULL"), (dict(query=None), b"query"), (dict(qo=None), b"query"),
    (dict(table=None), b"table"), (dict(rows=0), b"table"), (dict(rot=0), b"rotary_dim"), (dict(rot=129), b"rotary_dim"),
    (dict(rot=130), b"rotary_dim"), (dict(row=64), b"table row"), (dict(tdt=5), b"table dtype"),
    (dict(int4=1), b"4-bit row"), (dict(int4=1, dim=100), b"multiple of 32"), (dict(tokens=1 << 31), b"num_tokens"),
    (dict(tokens=1 << 30), b"exceed one launch"),
])
def test_append_entry_refuses(over, word):
    lib = _native.load()
    desc = _native.KVDesc(0x10000, 0x20000, 8, 16, 16 * 512, 512, 512)
    assert _append(lib, desc, **over) == _native.CBK_ERR_INVALID
    assert word in lib.cbk_last_error(), lib.cbk_last_error()
    assert _append(lib, desc, tokens=0) == _native.CBK_OK


def test_4_bit_entries_refuse_misaligned_pages():
    lib = _native.load()
    good = (0x10000, 0x20000, 8, 16, 16 * 160, 160, 160)
    for i, v in ((0, 0x10002), (1, 0x20001), (4, 16 * 160 + 2), (5, 161)):
        fields = list(good)
        fields[i] = v
        fields[4] = max(fields[4], 16 * fields[5])
        desc = _native.KVDesc(*fields)
        assert _append(lib, desc, int4=1) == _native.CBK_ERR_INVALID
        assert b"4-byte aligned" in lib.cbk_last_error()
        assert lib.cbk_paged_gather_int4(desc, 0x1000, 4, 2, 128, 1, 0x2000, 0x3000, 512, None) == _native.CBK_ERR_INVALID
        assert b"4-byte aligned" in lib.cbk_last_error()


@pytest.mark.parametrize("args,word", [
    ((0x1000, -1, 2, 128, 1, 0x2000, 0x3000, 512), b"num_tokens"), ((0x1000, 4, 2, 128, 9, 0x2000, 0x3000, 512), b"dtype"),
    ((0x1000, 4, 2, 96, 1, 0x2000, 0x3000, 512), b"4-bit row"), ((0x1000, 4, 2, 100, 1, 0x2000, 0x3000, 512), b"multiple"),
    ((None, 4, 2, 128, 1, 0x2000, 0x3000, 512), b"NULL"), ((0x1000, 4, 2, 128, 1, 0x2000, 0x3000, 504), b"stride"),
    ((0x1000, 4, 2, 128, 1, 0x2008, 0x3000, 512), b"16-byte"),
    ((0x1000, 1 << 30, 2, 128, 1, 0x2000, 0x3000, 512), b"too many rows"),
])
def test_int4_gather_entry_refuses(args, word):
    lib = _native.load()
    desc = _native.KVDesc(0x10000, 0x20000, 8, 16, 16 * 160, 160, 160)
    assert lib.cbk_paged_gather_int4(desc, *args, None) == _native.CBK_ERR_INVALID
    assert word in lib.cbk_last_error(), lib.cbk_last_error()


def _decode(lib, desc, **over):
    a = dict(q=0x1000, qb=512, qr=512, qh=128, batch=2, rows=1, hq=4, kv=desc, hkv=2, dim=128, tables=0x2000, ts=4, width=4,
             lens=0x3000, scale=0.1, dtype=1, out=0x4000, ob=512, orow=512, oh=128, ws=0x10000, nbytes=1 << 40, stream=None)
    a.update(over)
    return lib.cbk_paged_attention_int4(*a.values())


@pytest.mark.parametrize("over,word", [
    (dict(dtype=4), b"dtype"), (dict(dim=96), b"64 or 128"), (dict(hkv=3), b"4-bit row"), (dict(scale=float("nan")), b"finite"),
    (dict(width=-1), b"width"), (dict(hq=5), b"divisible"), (dict(rows=0), b"rows"), (dict(batch=-1), b"batch"),
    (dict(batch=1 << 16), b"batch"), (dict(width=1 << 28, ts=1 << 28), b"context"),
])
def test_int4_attention_entry_refuses(over, word):
    lib = _native.load()
    desc = _native.KVDesc(0x10000, 0x20000, 8, 16, 16 * 160, 160, 160)
    assert _decode(lib, desc, **over) == _native.CBK_ERR_INVALID
    assert word in lib.cbk_last_error(), lib.cbk_last_error()


def _prompt(lib, **over):
    a = dict(q=0x1000, qt=512, qh=128, k=0x2000, kt=256, kh=128, v=0x3000, vt=256, vh=128, ends_q=0x100, ends_k=0x200,
             batch=2, total_q=10, total_k=10, hq=4, hkv=2, dim=128, scale=0.1, dtype=1, out=0x4000, ot=512, oh=128, zero=1,
             ws=None, nbytes=0, stream=None)
    a.update(over)
    return lib.cbk_prompt_attention(*a.values())


@pytest.mark.parametrize("over,word", [
    (dict(dtype=3), b"dtype"), (dict(dim=80), b"64 or 128"), (dict(hq=3), b"divisible"), (dict(total_q=-1), b"tokens"),
    (dict(total_k=1 << 30), b"tokens"), (dict(batch=-1), b"batch"), (dict(batch=0), b"without a sequence"),
    (dict(q=None), b"NULL"), (dict(k=None), b"NULL"), (dict(ends_q=None), b"NULL"), (dict(out=None), b"NULL"),
    (dict(scale=float("inf")), b"finite"), (dict(q=0x1008), b"16-byte"), (dict(vt=260), b"16-byte"), (dict(oh=132), b"16-byte"),
    (dict(kt=1 << 24), b"2^24"), (dict(total_q=1 << 29, hq=8, hkv=2), b"too large"),
])
def test_prompt_entry_refuses(over, word):
    lib = _native.load()
    assert _prompt(lib, **over) == _native.CBK_ERR_INVALID
    assert word in lib.cbk_last_error(), lib.cbk_last_error()
    assert _prompt(lib, total_q=0) == _native.CBK_OK


def test_rows_that_lie_apart():
    from cacheblend_vllm.kv_layout import rows_apart

    x = torch.zeros(6, 4, 10)
    for t in (x, x.transpose(0, 1), x[:, ::2], x[..., 2:8], x[:1].expand(1, 4, 10), x.permute(1, 0, 2)[::2], x[:0],
              x.as_strided((3, 4, 5), (5, 30, 1)), x.as_strided((1, 2, 3), (0, 3, 1))):
        assert rows_apart(t), (t.shape, t.stride())
    for t in (x[:1].expand(6, 4, 10), x[:, :1].expand(6, 4, 10), x.as_strided((3, 4, 5), (5, 12, 1)),
              x.as_strided((3, 4, 5), (4, 40, 1))):
        assert not rows_apart(t), (t.shape, t.stride())
