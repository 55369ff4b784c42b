"""GPU: eviction from paged KV. Rows and weights move as they are, so everything is
compared bit for bit; and a decode loop of append, attention with the keys' weights
and eviction, against the same in 64 bits."""

import numpy as np
import pytest
import torch

from cacheblend_vllm import _native
from cacheblend_vllm import kv_layout as KL
from cacheblend_vllm.attention import paged_attention
from oracle import operators as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF16, F16, F32, U8 = torch.bfloat16, torch.float16, torch.float32, torch.uint8


def _bytes(g, shape, dtype):
    """Any bits: rows are moved, not read."""
    es = torch.empty((), dtype=dtype).element_size()
    raw = torch.randint(0, 256, (*shape[:-1], shape[-1] * es), generator=g, dtype=torch.uint8)
    return raw.view(dtype)


def _pool(g, blocks, size, row, dtype, layout="merged_first"):
    pool = _bytes(g, (2, blocks, size, *row), dtype)
    if layout == "merged_block":
        return pool.transpose(0, 1).contiguous().to(DEV)
    pool = pool.to(DEV)
    return pool if layout == "merged_first" else (pool[0], pool[1])


def _planes(layer):
    return torch.stack([p.contiguous() for p in KL.kv_planes(layer)]).view(torch.uint8).cpu().clone()


def _weights(g, batch, sets, keys, kind="mass"):
    w = torch.exp(1.5 * torch.randn(batch, sets, keys, generator=g))
    if kind == "mass":  # some that no row looked at
        w = torch.where(w > 0.4, w, 0.0)
    elif kind == "ties":
        w = torch.randint(0, 4, (batch, sets, keys), generator=g).float()
    elif kind == "equal":
        w = torch.full((batch, sets, keys), 0.25)
    elif kind == "odd":  # signs, zeros of both, infinities, NaN of both signs, subnormal numbers
        w = torch.randn(batch, sets, keys, generator=g)
        pick = torch.randint(0, 12, (batch, sets, keys), generator=g)
        for i, v in enumerate((0.0, -0.0, float("inf"), -float("inf"), float("nan"), 1e-45, -1e-45)):
            w[pick == i] = v
        bits = w.view(torch.int32)
        bits[pick == 7] = -0x3f0000  # 0xffc10000, a NaN
    return w


def _want(planes, tables, lens, size, weights, keeps, first, recent, heads):
    """Pages (as bytes), weights and lengths after the eviction."""
    planes, weights = planes.clone(), weights.clone()
    sets = weights.shape[1]
    blocks = planes.shape[1]
    rows = planes.flatten(3).unflatten(3, (sets, -1))  # a view: [2, blocks, tokens, sets, bytes]
    new_lens = []
    for b, n in enumerate(lens):
        stay_n = max(keeps[b], first + recent)
        new_lens.append(min(n, stay_n))
        if n <= stay_n:
            continue
        at = np.arange(n)
        page, off = np.asarray(tables[b])[at // size].astype(np.int64), at % size
        ok = (page >= 0) & (page < blocks)
        for m in range(sets):
            stay = R.evict(weights[b, m].numpy(), n, keeps[b], first, recent)
            assert len(stay) == stay_n
            to = np.arange(stay_n)
            good = ok[stay] & ok[to]
            s, t = stay[good], to[good]
            rows[:, page[t], off[t], m] = rows[:, page[s], off[s], m].clone()
            old = weights[b, m, :n].clone()
            weights[b, m, :n] = 0
            weights[b, m, :stay_n] = old[torch.from_numpy(stay)]
    return planes, weights, new_lens


def _check(row, dtype, lens, keep, first=0, recent=0, size=16, layout="merged_first", shared=False, kind="mass", seed=0,
           more=0, blocks=None, device_lens=True):
    keeps = [keep] * len(lens) if isinstance(keep, int) else list(keep)
    print(f"evict {dtype} {row} lens {lens[:6]} keep {keeps[:4]} {first} {recent} size {size} {layout} {shared} {kind}", flush=True)
    g = torch.Generator().manual_seed(seed)
    width = max((n + size - 1) // size for n in lens) + more
    used = sum((n + size - 1) // size for n in lens)
    blocks = blocks or used + 3
    layer = _pool(g, blocks, size, row, dtype, layout)
    order, at = torch.randperm(blocks, generator=g), 0
    tables = torch.full((len(lens), width), -5, dtype=torch.int32)
    for i, n in enumerate(lens):
        k = (n + size - 1) // size
        tables[i, :k] = order[at:at + k]
        at += k
    sets = 1 if shared else row[0]
    weights = _weights(g, len(lens), sets, width * size + 5, kind)
    planes = _planes(layer)
    want = _want(planes, tables, lens, size, weights, keeps, first, recent, row[0])
    on = weights.to(DEV)
    give = torch.tensor(lens, device=DEV if device_lens else "cpu")
    got = KL.evict_paged_kv(layer, tables.to(DEV) if device_lens else tables, give, size, on,
                            keep if isinstance(keep, int) else torch.tensor(keeps, device=DEV if device_lens else "cpu"),
                            first=first, recent=recent)
    torch.cuda.synchronize()
    assert got.dtype == torch.int32 and got.tolist() == want[2]
    same = on.cpu().view(torch.int32) == want[1].view(torch.int32)
    assert bool(same.all()), f"weights differ at {(~same).nonzero()[:4].tolist()}"
    same = _planes(layer) == want[0]
    assert bool(same.all()), f"pages differ at {(~same).nonzero()[:4].tolist()}"


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("row,dtype", [((8, 128), BF16), ((2, 64), F16), ((4, 128), F32), ((1, 128), BF16), ((8, 80), U8),
                                       ((3, 40), U8), ((5, 7), U8), ((3, 3), BF16)])
def test_rows_of_any_type(row, dtype, shared):
    _check(row, dtype, [700, 0, 1, 100, 333, 99, 101], 100, first=4, recent=16, shared=shared, seed=row[0])


@pytest.mark.parametrize("kind", ["mass", "ties", "equal", "odd"])
def test_ties_signs_and_numbers_that_are_none(kind):
    for keep, first, recent in ((50, 0, 0), (50, 1, 7), (8, 1, 7), (299, 0, 0), (1, 0, 0), (0, 0, 0), (300, 10, 10)):
        _check((2, 64), BF16, [300, 1025, 51], keep, first, recent, kind=kind, seed=keep)


@pytest.mark.parametrize("size,layout", [(1, "merged_first"), (5, "merged_block"), (16, "separate"), (48, "merged_first"),
                                         (256, "merged_block")])
def test_block_sizes_and_layouts(size, layout):
    for shared in (False, True):
        _check((4, 64), BF16, [333, 64, 7, 700], 60, 2, 9, size=size, layout=layout, shared=shared, seed=size, more=3)


@pytest.mark.parametrize("n", [2, 3, 1023, 1024, 1025, 2048, 2049])
def test_lengths_about_a_pass_of_the_choice(n):
    for keep in {1, n // 2, n - 1}:
        _check((2, 64), F16, [n], keep, seed=n, kind="ties")


def test_one_key_of_many_and_many_of_few():
    # rows that move by one place, tile after tile; by nearly all; lengths of their own to keep
    for shared in (False, True):
        _check((4, 128), BF16, [5000], 4999, 4, 64, shared=shared, seed=1)
        _check((4, 128), BF16, [5000, 4500], 4400, shared=shared, seed=2)
        _check((4, 128), BF16, [5000], 37, 4, 9, shared=shared, seed=3)
        _check((8, 128), BF16, [5000, 300, 0, 4097], [4096, 0, 5, 4097], 2, 3, shared=shared, seed=4)
        _check((8, 128), BF16, [3000, 300, 2900], [5, 299, 1000], 2, 3, shared=shared, seed=5, device_lens=False)
    _check((1, 4096), F32, [2000], 1500, seed=6)   # a row of more than a tile's pieces a thread
    _check((1, 10000), F32, [300], 200, 3, 5, seed=7)
    _check((9, 1001), U8, [600], 500, seed=8, shared=True)  # 9009 bytes, one by one


def test_a_long_sequence_and_many_short_ones():
    _check((2, 128), BF16, [40000], 20000, 4, 128, seed=9)
    _check((2, 64), BF16, [33] * 300, 32, 1, 8, seed=10, kind="ties")
    _check((1, 64), BF16, list(range(1, 200)), 64, 4, 4, seed=11, shared=True)


def test_pages_out_of_range_do_not_move():
    g = torch.Generator().manual_seed(12)
    layer = _pool(g, 6, 16, (2, 64), BF16)
    tables = torch.tensor([[0, -1, 3, 1], [99, 6, -5, 2], [4, 1 << 30, 5, -1]], dtype=torch.int32)
    lens, keeps = [60, 50, 64], [20, 9, 40]
    weights = _weights(g, 3, 2, 64)
    want = _want(_planes(layer), tables, lens, 16, weights, keeps, 0, 0, 2)
    on = weights.to(DEV)
    got = KL.evict_paged_kv(layer, tables.to(DEV), torch.tensor(lens, device=DEV), 16, on, torch.tensor(keeps, device=DEV))
    assert got.tolist() == want[2] and torch.equal(on.cpu(), want[1]) and torch.equal(_planes(layer), want[0])


def test_lengths_and_keeps_on_the_device_are_clamped():
    g = torch.Generator().manual_seed(13)
    layer = _pool(g, 8, 16, (2, 64), BF16)
    tables = torch.arange(8, dtype=torch.int32).reshape(2, 4)
    weights = _weights(g, 2, 2, 64)
    want = _want(_planes(layer), tables, [64, 0], 16, weights, [7, 7], 3, 4, 2)
    on = weights.to(DEV)
    got = KL.evict_paged_kv(layer, tables.to(DEV), torch.tensor([1000, -9], device=DEV), 16, on,
                            torch.tensor([-3, 2], device=DEV), first=3, recent=4)
    assert got.tolist() == [7, 0] and torch.equal(on.cpu(), want[1]) and torch.equal(_planes(layer), want[0])


def test_shared_pages_end():
    # pages of two tables: what they hold afterwards is undefined, the rest is not
    g = torch.Generator().manual_seed(14)
    layer = _pool(g, 40, 16, (4, 64), BF16)
    tables = torch.stack([torch.arange(30), torch.arange(30)]).int()
    tables[1, 20:] = 3
    before = _planes(layer)
    weights = _weights(g, 2, 4, 480).to(DEV)
    got = KL.evict_paged_kv(layer, tables.to(DEV), torch.tensor([480, 470], device=DEV), 16, weights, 200)
    torch.cuda.synchronize()
    assert got.tolist() == [200, 200]
    assert torch.equal(_planes(layer)[:, 30:], before[:, 30:])


def test_strides():
    # blocks longer than used, an odd first element, sums with rows apart
    g = torch.Generator().manual_seed(15)
    for dtype in (BF16, F32):
        room = _bytes(g, (2 * 9 * 20 * 2 * 64 + 1,), dtype).to(DEV)
        layer = room[1:].view(2, 9, 20, 2, 64)
        tables = torch.tensor([[3, 9, 1, 9, 5, 9], [0, 9, 2, 9, 4, 9]], dtype=torch.int32, device=DEV)[:, ::2]
        lens, size = [40, 48], 16
        pool = torch.rand(4, 2, 70, generator=g).to(DEV)
        weights = pool[1::2, :, 1:]
        cut = _planes(layer)
        want = _want(cut[:, :, :16].contiguous(), tables.cpu(), lens, size, weights.cpu(), [11, 11], 1, 2, 2)
        kept = pool.clone()
        got = KL.evict_paged_kv(layer, tables, torch.tensor(lens), size, weights, 11, first=1, recent=2)
        assert got.tolist() == [11, 11] and torch.equal(weights.cpu(), want[1])
        after = _planes(layer)
        assert torch.equal(after[:, :, :16], want[0]) and torch.equal(after[:, :, 16:], cut[:, :, 16:])
        pool[1::2, :, 1:] = kept[1::2, :, 1:]
        assert torch.equal(pool, kept)


def test_offsets_past_32_bits():
    blocks = 400_000  # two planes of 3 GB
    layer = torch.empty(2, blocks, 16, 4, 64, dtype=BF16, device=DEV)
    g = torch.Generator().manual_seed(16)
    tables = torch.tensor([[blocks - 1, 3, blocks // 2, blocks - 7]], dtype=torch.int32)
    own = tables[0].long()
    layer[:, own] = torch.randn(2, 4, 16, 4, 64, generator=g).to(BF16).to(DEV)
    small = layer[:, own].contiguous()
    weights = _weights(g, 1, 4, 64)
    want = _want(_planes(small), torch.arange(4)[None], [61], 16, weights, [30], 2, 5, 4)
    on = weights.to(DEV)
    KL.evict_paged_kv(layer, tables.to(DEV), torch.tensor([61], device=DEV), 16, on, 30, first=2, recent=5)
    assert torch.equal(on.cpu(), want[1]) and torch.equal(_planes(layer[:, own].contiguous()), want[0])


def test_streams_and_graphs():
    g = torch.Generator().manual_seed(17)
    first = _pool(g, 200, 16, (8, 64), BF16)
    lens0 = [1500, 60, 1400]
    tables = torch.full((3, 100), -1, dtype=torch.int32)
    order, at = torch.randperm(200, generator=g), 0
    for i, n in enumerate(lens0):
        k = (n + 15) // 16
        tables[i, :k] = order[at:at + k]
        at += k
    on_tables = tables.to(DEV)
    w0 = _weights(g, 3, 8, 1600)
    lens = torch.tensor(lens0, device=DEV)
    layer, weights = first.clone(), w0.to(DEV)

    def check(n):
        want = _want(_planes(first), tables, n, 16, w0, [700] * 3, 4, 32, 8)
        assert torch.equal(weights.cpu(), want[1]) and torch.equal(_planes(layer), want[0])
        return want[2]

    def reset():
        layer.copy_(first)
        weights.copy_(w0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = KL.evict_paged_kv(layer, on_tables, lens, 16, weights, 700, first=4, recent=32)
    torch.cuda.current_stream().wait_stream(side)
    assert got.tolist() == check(lens0)
    reset()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = KL.evict_paged_kv(layer, on_tables, lens, 16, weights, 700, first=4, recent=32)
    layer2, weights2 = first.clone(), w0.to(DEV)
    with torch.cuda.graph(other):
        out2 = KL.evict_paged_kv(layer2, on_tables, lens, 16, weights2, 700, first=4, recent=32)
    for n in ([1500, 60, 1400], [701, 700, 1], [1333, 0, 1399]):  # lengths may change between replays
        lens.copy_(torch.tensor(n))
        reset()
        layer2.copy_(first)
        weights2.copy_(w0.to(DEV))
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        assert out.tolist() == check(n) == out2.tolist()
        assert torch.equal(layer2, layer) or bool((layer2.view(torch.int16) == layer.view(torch.int16)).all())
        assert torch.equal(weights, weights2)


def test_refusals():
    layer = torch.zeros(2, 4, 16, 2, 64, dtype=BF16, device=DEV)
    tables, lens = torch.zeros(1, 4, dtype=torch.int32), torch.tensor([16])
    w = torch.zeros(1, 2, 64, device=DEV)

    def refused(error, match, kv=layer, t=tables, n=lens, size=16, weights=w, keep=8, **kw):
        with pytest.raises(error, match=match):
            KL.evict_paged_kv(kv, t, n, size, weights, keep, **kw)

    refused(RuntimeError, "device", kv=layer.cpu())
    refused(ValueError, "block_size", size=17)
    refused(ValueError, "lengths", n=torch.tensor([16, 16]))
    refused(ValueError, "block tables", t=tables[0])
    refused(IndexError, "context lengths", n=torch.tensor([65]))
    refused(IndexError, "block tables", t=torch.full((1, 4), -1, dtype=torch.int32))
    refused(ValueError, "key weights are", weights=torch.zeros(1, 2, 63, device=DEV))
    refused(ValueError, "key weights are", weights=torch.zeros(1, 3, 64, device=DEV))
    refused(ValueError, "float32", weights=w.half())
    refused(ValueError, "overlap", weights=torch.zeros(1, 1, 64, device=DEV).expand(1, 2, 64))
    refused(ValueError, "together", keep=7, first=4, recent=4)
    refused(ValueError, "together", keep=-1)
    refused(ValueError, "together", keep=torch.tensor([7]), first=4, recent=4)
    refused(ValueError, "negative", first=-1)
    refused(ValueError, "numbers to keep", keep=torch.tensor([7, 7]))
    refused(ValueError, "whole numbers", keep=torch.tensor([7.0]))
    assert KL.evict_paged_kv(layer, tables[:0], lens[:0], 16, w[:0], 8).shape == (0,)
    assert KL.evict_paged_kv(layer, tables[:, :0], torch.tensor([0]), 16, w, 8).tolist() == [0]
    # a scratch that is too small is an error, not a fault
    desc, _, _ = KL.paged_layer(layer, 16)
    lib = _native.load()
    ws = torch.empty(256, dtype=torch.uint8, device=DEV)
    new = torch.empty(1, dtype=torch.int32, device=DEV)
    on = tables.to(DEV), lens.int().to(DEV)
    rc = lib.cbk_paged_evict(desc, on[0].data_ptr(), 4, 4, on[1].data_ptr(), 1, w.data_ptr(), 128, 64, 2, 8, None, 0, 0,
                             new.data_ptr(), ws.data_ptr(), 256, _native.stream_handle(DEV))
    assert rc == _native.CBK_ERR_WORKSPACE


@pytest.mark.parametrize("dtype,shared", [(BF16, False), (F32, True)])
def test_a_decode_loop_with_a_bounded_cache(dtype, shared):
    """Prefill's last rows weigh the prompt, then every step appends a token, attends and,
    past the budget, evicts; outputs and weights against 64 bits with the same choices."""
    g = torch.Generator().manual_seed(18)
    batch, hq, heads, d, size, keep, first, recent, rows = 3, 8, 4, 64, 16, 40, 2, 6, 5
    lens = [90, 40, 33]
    width = 8
    layer = torch.zeros(2, batch * width, size, heads, d, dtype=dtype, device=DEV)
    tables = torch.randperm(batch * width, generator=g).reshape(batch, width).int()
    on_tables = tables.to(DEV)
    sets = 1 if shared else heads
    weights = torch.zeros(batch, sets, width * size, device=DEV)
    book = [[[[] for _ in range(heads)] for _ in range(2)] for _ in range(batch)]  # rows of [b][plane][head], 64 bits
    sums = [[np.zeros(0) for _ in range(sets)] for _ in range(batch)]
    half = torch.finfo(dtype).eps / 2

    def append(counts, at):
        n = sum(counts)
        k, v = (torch.randn(n, heads, d, generator=g).to(dtype) for _ in range(2))
        b = np.repeat(np.arange(batch), counts)
        pos = np.concatenate([np.arange(a, a + c) for a, c in zip(at, counts)])
        slots = tables.numpy()[b, pos // size].astype(np.int64) * size + pos % size
        KL.append_paged_kv(k.to(DEV), v.to(DEV), layer, torch.from_numpy(slots).to(DEV), size)
        for i, s in enumerate(b):
            for p, x in enumerate((k, v)):
                for h in range(heads):
                    book[s][p][h].append(x[i, h].double().numpy())
        for s in range(batch):
            sums[s] = [np.concatenate([w, np.zeros(counts[s])]) for w in sums[s]]

    def attend(q, n):
        got = paged_attention(q.to(DEV), layer, on_tables, n, size, 0.2, key_weights=weights)
        for s in range(batch):
            for h in range(hq):
                k, v = (np.stack(book[s][p][h // (hq // heads)]) for p in range(2))
                for r in range(q.shape[1]):
                    seen = len(k) - q.shape[1] + r + 1
                    x = k[:seen] @ q[s, r, h].double().numpy() * 0.2
                    p = np.exp(x - x.max())
                    p /= p.sum()
                    sums[s][h // (hq // sets)][:seen] += p
                    # weights off by at most 2^-14 of themselves (the bound above, for logits' terms under 100)
                    tol = half * np.abs(p @ v[:seen]) + 2.0 ** -13 * (p @ np.abs(v[:seen])) + 1e-30
                    assert np.all(np.abs(got[s, r, h].double().cpu().numpy() - p @ v[:seen]) <= tol)
        for s in range(batch):
            for m in range(sets):
                mine = weights[s, m].double().cpu().numpy()
                assert np.allclose(mine[:len(sums[s][m])], sums[s][m], rtol=2.0 ** -13, atol=0)
                assert not mine[len(sums[s][m]):].any()

    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    append(lens, [0] * batch)
    attend(torch.randn(batch, rows, hq, d, generator=g).to(dtype), n)
    at = lens
    for step in range(14):
        # the choice is made on the device's own sums: ties within rounding are its
        host = weights.cpu().numpy()
        n = KL.evict_paged_kv(layer, on_tables, n, size, weights, keep, first=first, recent=recent)
        for s in range(batch):
            for m in range(sets):
                stay = R.evict(host[s, m], len(sums[s][m]), keep, first, recent)
                sums[s][m] = sums[s][m][stay]
                for h in range(m * (heads // sets), (m + 1) * (heads // sets)):
                    for p in range(2):
                        book[s][p][h] = [book[s][p][h][i] for i in stay]
        at = n.tolist()
        assert at == [len(sums[s][0]) for s in range(batch)]
        append([1] * batch, at)
        n = n + 1
        attend(torch.randn(batch, 1, hq, d, generator=g).to(dtype), n)
    assert n.tolist() == [41, 41, 41]


def test_more_tiles_than_a_launch_has_workgroups():
    # 60000 sequences with room for 40 rows of 32 KB, a tile each, in two planes; two move any
    _check((256, 128), U8, [48] + [0] * 59998 + [47], 40, 3, 2, shared=True, seed=7)


def test_long_tables_of_short_sequences():
    _check((4, 64), BF16, [333, 0, 64, 700, 5] * 20, 60, 4, 8, seed=8, more=900)
    _check((4, 64), BF16, [333, 0, 64, 700, 5] * 20, [300, 7, 60, 20, 0] * 20, 0, 0, seed=9, more=900, shared=True)


@pytest.mark.parametrize("first,recent,keep", [(9000, 100, 10000), (100, 9000, 10000), (8192, 8192, 16400), (16500, 0, 16501),
                                               (0, 16500, 16501), (8191, 1, 8192)])
def test_ends_longer_than_a_pass_of_the_choice(first, recent, keep):
    _check((1, 32), BF16, [20000, 17000, keep, keep + 1], keep, first, recent, kind="mass", seed=first)
    _check((2, 16), BF16, [20000], keep, first, recent, kind="ties", seed=recent, shared=True)


def test_keys_and_values_in_one_tensor_are_refused():
    pages = torch.zeros(4, 16, 2, 64, dtype=BF16, device=DEV)
    tables, lens, w = torch.arange(4, dtype=torch.int32)[None], torch.tensor([60]), torch.zeros(1, 2, 64, device=DEV)
    for layer in ((pages, pages), pages.expand(2, 4, 16, 2, 64)):
        with pytest.raises(ValueError, match="same rows"):
            KL.evict_paged_kv(layer, tables, lens, 16, w, 8)
