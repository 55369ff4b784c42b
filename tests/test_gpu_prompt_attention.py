"""GPU: causal attention of packed prompts, against 64 bits.

Tolerance, 16 bits. A logit is a float32 sum of head_size exact products: at
most head_size + 8 roundings of 2^-24 of the sum of their absolute values (the
last few for the units and the reference maximum). A weight is rounded to the
type, eps / 2 of itself, or half of 2^-24 where float16 is below its normal
range (the row's sum is at least 1 then); the sum is of the rounded weights. A
relative change e of every weight moves an output by at most 2 e sum p |v|.
The output's sums round once a key at most, and the output by half its own
step. float32: the same without the weights' rounding."""

import numpy as np
import pytest
import torch

from cacheblend_vllm.attention import prompt_attention
from oracle import operators as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _ends(lens, first=0):
    return [first + n for n in np.concatenate([[0], np.cumsum(lens)]).tolist()]


def _bound(q, k, v, ends_q, ends_k, scale, dtype, want, mass):
    tol = np.zeros(want.shape)
    group, d = q.shape[1] // k.shape[1], q.shape[2]
    half = torch.finfo(dtype).eps / 2
    for a, b, c, e in zip(ends_q[:-1], ends_q[1:], ends_k[:-1], ends_k[1:]):
        if b == a or e == c:
            continue
        n = e - c
        # the largest sum of absolute products of any of the sequence's keys
        terms = np.einsum("qhd,hd->qh", np.abs(q[a:b]), np.abs(k[c:e]).max(axis=0).repeat(group, axis=0))
        weight = (d + 8) * 2.0 ** -24 * abs(scale) * terms + (0 if dtype == F32 else half) + (n + 64) * 2.0 ** -24
        tol[a:b] = 2 * weight[..., None] * mass[a:b]
        if dtype == F16:
            tol[a:b] += n * 2.0 ** -25 * np.abs(v[c:e]).max()
    return tol + half * np.abs(want) + (2.0 ** -25 if dtype == F16 else 1e-30)


def _make(g, total_q, total_k, hq, hkv, d, dtype):
    return (torch.randn(n, h, d, generator=g).to(dtype) for n, h in ((total_q, hq), (total_k, hkv), (total_k, hkv)))


def _compare(got, q, k, v, ends_q, ends_k, scale, dtype):
    qn, kn, vn = (t.double().numpy() for t in (q, k, v))
    want, mass = R.prompt_attention(qn, kn, vn, ends_q, ends_k, scale)
    tol = _bound(qn, kn, vn, ends_q, ends_k, scale, dtype, want, mass)
    err = np.abs(got.double().cpu().numpy() - want)
    inside = slice(ends_q[0], ends_q[-1])
    if err[inside].size:
        print(f"  worst {float((err / tol)[inside].max()):.3f} of the bound, "
              f"relative {np.linalg.norm(err) / max(1e-30, np.linalg.norm(want)):.2e}", flush=True)
    assert np.all(err <= tol)
    return mass


def _check(dtype, hq, hkv, d, lens, keys=None, seed=0, scale=None, before=0, behind=0):
    print(f"prompt {dtype} {hq}/{hkv}x{d} lens {lens[:6]} keys {(keys or [])[:6]} around {before} {behind}", flush=True)
    g = torch.Generator().manual_seed(seed)
    ends_q = _ends(lens, before)
    ends_k = ends_q if keys is None else _ends(keys, before)
    q, k, v = _make(g, ends_q[-1] + behind, ends_k[-1] + behind, hq, hkv, d, dtype)
    scale = d ** -0.5 if scale is None else scale
    give_k = None if keys is None else torch.tensor(ends_k, device=DEV)
    got = prompt_attention(q.to(DEV), k.to(DEV), v.to(DEV), torch.tensor(ends_q, device=DEV), scale, give_k)
    torch.cuda.synchronize()
    assert got.shape == q.shape and got.dtype == dtype
    mass = _compare(got, q, k, v, ends_q, ends_k, scale, dtype)
    # rows of no sequence, and rows that see nothing, are zero
    assert not got.cpu()[torch.from_numpy(~mass.any(axis=-1))].any()
    return q, k, v, got


TYPES = [BF16, F16, F32]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (8, 8, 64), (5, 1, 128), (12, 4, 64), (40, 8, 128)])
def test_packed_prompts_against_64_bits(dtype, hq, hkv, d):
    _check(dtype, hq, hkv, d, [1, 33, 0, 64, 130, 31, 32, 257], seed=hq + d)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", [[1], [2], [1000], [700, 1, 1, 900], [1] * 150, [16] * 70 + [300]])
def test_lengths(lens, dtype):
    _check(dtype, 8, 2, 128, lens, seed=len(lens))
    _check(dtype, 6, 2, 64, lens, seed=len(lens) + 1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,keys", [
    ([64], [2000]), ([1, 1, 1], [300, 1, 77]), ([40, 33], [100, 500]),  # chunks of longer prompts
    ([50, 10, 100], [3, 0, 99]),                                        # fewer keys than queries
    ([0, 5, 0], [40, 5, 7]), ([200, 7], [200, 1500]), ([1] * 80, list(range(1, 81))),
])
def test_more_and_fewer_keys_than_queries(lens, keys, dtype):
    _check(dtype, 8, 2, 128, lens, keys, seed=len(lens) + lens[0])
    _check(dtype, 4, 1, 64, lens, keys, seed=len(lens) + lens[0] + 1)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_around_the_sequences(dtype):
    q, k, v, _ = _check(dtype, 8, 2, 64, [40, 90], seed=3, before=7, behind=300)
    out = torch.full(q.shape, 5.0, dtype=dtype, device=DEV)
    ends = torch.tensor([7, 47, 137], device=DEV)
    got = prompt_attention(q.to(DEV), k.to(DEV), v.to(DEV), ends, 0.125, out=out)
    assert got is out and bool((out[:7] == 5).all()) and bool((out[137:] == 5).all())
    _compare(torch.cat([out[:7] * 0, out[7:137], out[137:] * 0]), q, k, v, ends.tolist(), ends.tolist(), 0.125, dtype)
    # the same through key ranges (a chunk with much context)
    _check(dtype, 8, 2, 64, [20], [1500], seed=4, before=7, behind=50)


@pytest.mark.parametrize("dtype", TYPES)
def test_hundreds_of_sequences(dtype):
    g = torch.Generator().manual_seed(20)
    lens = torch.randint(0, 9, (600,), generator=g).tolist()
    lens[37], lens[599] = 150, 70
    _check(dtype, 4, 2, 64, lens, seed=20, before=3, behind=40)
    _check(dtype, 4, 2, 128, lens, [n + 5 for n in lens], seed=21)


def test_thousands_of_sequences_and_ends_that_do_not_rise():
    g = torch.Generator().manual_seed(26)
    lens = torch.randint(0, 3, (5000,), generator=g).tolist()
    q, k, v, got = _check(BF16, 2, 1, 64, lens, seed=26, before=1, behind=2)
    # out of order: taken as they stand, within the tensors
    ends = torch.tensor(_ends(lens, 1))
    ends[2000:3000] = ends[2000:3000].flip(0)
    ends[4000] = -5
    ends[4500] = 1 << 30
    for dtype in (BF16, F32):
        out = prompt_attention(q.to(DEV, dtype), k.to(DEV, dtype), v.to(DEV, dtype), ends.to(DEV), 0.1)
        torch.cuda.synchronize()
        assert out.shape == q.shape


@pytest.mark.parametrize("dtype", TYPES)
def test_a_large_launch_of_few_sequences(dtype):
    # more than 2048 workgroups: the tiles sequence after sequence
    _check(dtype, 128, 128, 64, [300, 0, 1100], seed=22, before=300, behind=200)


def test_long_sequences():
    _check(BF16, 4, 1, 128, [3500, 100], seed=5)
    _check(F16, 2, 2, 64, [4100], seed=6)


@pytest.mark.parametrize("dtype", TYPES)
def test_scales_and_logits_that_outgrow_the_first_block(dtype):
    for scale in (-0.2, 0.0, 2.0, 1e-30):
        _check(dtype, 4, 2, 64, [300, 40], seed=7, scale=scale)
    # keys whose logits grow along the sequence, by hundreds
    g = torch.Generator().manual_seed(8)
    for d in (64, 128):
        q, k, v = _make(g, 400, 400, 4, 2, d, dtype)
        k = (k * torch.linspace(0.01, 12, 400)[:, None, None]).to(dtype)
        got = prompt_attention(q.to(DEV), k.to(DEV), v.to(DEV), torch.tensor([0, 400]), 1.0)
        _compare(got, q, k, v, [0, 400], [0, 400], 1.0, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_what_a_row_does_not_see_may_be_anything(dtype, value):
    g = torch.Generator().manual_seed(9)
    for d, hq in ((64, 4), (128, 8)):
        q, k, v = (t.to(DEV) for t in _make(g, 300, 300, hq, 2, d, dtype))
        ends = torch.tensor([0, 150, 260], device=DEV)
        want = prompt_attention(q, k, v, ends, 0.1)
        k2, v2, q2 = k.clone(), v.clone(), q.clone()
        k2[149], v2[149] = value, value  # the first sequence's last token: its own row alone
        k2[260:], v2[260:], q2[260:] = value, value, value  # padding
        got = prompt_attention(q2, k2, v2, ends, 0.1)
        same = torch.ones(300, dtype=torch.bool, device=DEV)
        same[149] = False
        # rows of a workgroup that is redone may be rounded another way
        tol = 4 * torch.finfo(dtype).eps * (1 + want[same].float().abs())
        assert bool(((got[same].float() - want[same].float()).abs() <= tol).all()), (d, dtype)
        assert not bool(got[149].isfinite().all())
        # a query that is not finite: its own row and head
        q3 = q.clone()
        q3[60, 1, 3] = value
        got = prompt_attention(q3, k, v, ends, 0.1)
        other = torch.ones(300, hq, dtype=torch.bool, device=DEV)
        other[60, 1] = False
        tol = 4 * torch.finfo(dtype).eps * (1 + want[other].float().abs())
        assert bool(((got[other].float() - want[other].float()).abs() <= tol).all())
        assert bool(got[60, 1].isnan().any())


@pytest.mark.parametrize("d", [64, 128])
def test_float32_workgroups_of_128_rows(d):
    # rows x KV heads from 1536 x 64 on
    _check(F32, 64, 64, d, [700, 1, 0, 95, 850], seed=23, behind=10)
    _check(F32, 96, 32, d, [400, 129, 600], [500, 100, 601], seed=24, before=5)
    g = torch.Generator().manual_seed(25)
    q, k, v = (t.to(DEV) for t in _make(g, 1600, 1600, 64, 64, d, F32))
    ends = torch.tensor([0, 150, 1560], device=DEV)
    want = prompt_attention(q, k, v, ends, 0.1)
    k2, v2 = k.clone(), v.clone()
    k2[149], v2[149] = float("nan"), float("inf")  # the first sequence's last token: its own row alone
    k2[1560:], v2[1560:] = float("nan"), float("nan")
    got = prompt_attention(q, k2, v2, ends, 0.1)
    same = torch.ones(1600, dtype=torch.bool, device=DEV)
    same[149] = False
    # Rows of a masked block with such a value are summed one by one, in another
    # order: both results hold to _bound (a dot product of d terms in 24 bits is off
    # by up to (d + 8) 2^-24 of its absolute terms' sum, 1e-5 and more of a logit
    # here, and the weights by that relative to themselves), so that they are apart by
    # twice that at most. 4 eps (1 + |want|), as first written, leaves that out.
    ends = [0, 150, 1560]
    qn, kn, vn = (t.double().cpu().numpy() for t in (q, k, v))
    clean, mass = R.prompt_attention(qn, kn, vn, ends, ends, 0.1)
    tol = 2 * torch.from_numpy(_bound(qn, kn, vn, ends, ends, 0.1, F32, clean, mass)).to(DEV)[same]
    assert bool(((got[same] - want[same]).abs() <= tol).all())
    assert bool(((got[same] - torch.from_numpy(clean).to(DEV)[same]).abs() <= tol).all())
    assert not bool(got[149].isfinite().any())


def test_strides_and_alignment():
    g = torch.Generator().manual_seed(10)
    qkv = torch.randn(200, 8 + 2 + 2, 128, generator=g).to(BF16).to(DEV)
    q, k, v = qkv.split([8, 2, 2], dim=1)
    ends = torch.tensor([0, 77, 200])
    want = prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), ends, 0.1)
    assert torch.equal(prompt_attention(q, k, v, ends, 0.1), want)
    assert torch.equal(prompt_attention(q.transpose(0, 1).contiguous().transpose(0, 1), k, v, ends.to(DEV), 0.1), want)
    raw = torch.zeros(200 * 2 * 128 + 1, dtype=BF16, device=DEV)
    odd = raw[1:].view(200, 2, 128)
    odd.copy_(v)
    assert torch.equal(prompt_attention(q, k, odd, ends, 0.1), want)
    wide = torch.zeros(200, 8, 131, dtype=BF16, device=DEV)
    out = prompt_attention(q, k, v, ends, 0.1, out=wide[..., 2:130])
    assert torch.equal(out, want) and not wide[..., :2].any() and not wide[..., 130:].any()
    spread = torch.zeros(200, 16, 128, dtype=BF16, device=DEV)
    prompt_attention(q, k, v, ends, 0.1, out=spread[:, ::2])
    assert torch.equal(spread[:, ::2], want) and not spread[:, 1::2].any()
    one = k[:1].expand(200, 2, 128)  # one key row for all tokens
    assert torch.equal(prompt_attention(q, one, v, ends, 0.1), prompt_attention(q, one.contiguous(), v, ends, 0.1))


def test_ends_on_the_device_are_clamped():
    g = torch.Generator().manual_seed(11)
    q, k, v = (t.to(DEV) for t in _make(g, 100, 100, 4, 2, 64, BF16))
    want = prompt_attention(q, k, v, torch.tensor([0, 30, 100]), 0.1)
    for bad in ([-5, 30, 1000], [0, 30, 100, 1 << 40]):
        got = prompt_attention(q, k, v, torch.tensor(bad, device=DEV), 0.1)
        assert torch.equal(got, want), bad
    prompt_attention(q, k, v, torch.tensor([90, 10, 70], device=DEV), 0.1)  # falling: nothing out of bounds


def test_graphs_streams_and_repeats():
    g = torch.Generator().manual_seed(12)
    for dtype, hq, d, lens in ((BF16, 8, 128, [500, 30, 700]), (F16, 4, 64, [64]), (F32, 4, 64, [200, 100])):
        total = sum(lens)
        keys = total + 900  # and key ranges
        q, k, v = (t.to(DEV) for t in _make(g, total, keys, hq, 2, d, dtype))
        ends_q = torch.tensor(_ends(lens), device=DEV)
        ends_k = ends_q.clone()
        ends_k[-1] = keys
        want = prompt_attention(q, k, v, ends_q, 0.1, ends_k)
        assert torch.equal(prompt_attention(q, k, v, ends_q, 0.1, ends_k), want)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = prompt_attention(q, k, v, ends_q, 0.1, ends_k)
        side.synchronize()
        assert torch.equal(got, want)
        graphs, outs = [], []
        for _ in range(2):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1]):
                outs.append(prompt_attention(q, k, v, ends_q, 0.1, ends_k))
        for rep in range(3):
            for o in outs:
                o.fill_(float("nan"))
            prompt_attention(q, v, k, ends_q, 0.1, ends_k)
            streams = [torch.cuda.Stream(), torch.cuda.Stream()]
            torch.cuda.synchronize()
            for s, graph in zip(streams, graphs):
                with torch.cuda.stream(s):
                    graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(o, want) for o in outs), rep


def test_prompt_attention_refuses():
    q = torch.zeros(6, 4, 64, dtype=BF16, device=DEV)
    k = torch.zeros(6, 2, 64, dtype=BF16, device=DEV)
    ends = torch.tensor([0, 6])

    def refuse(error, word, q=q, k=k, v=None, ends=ends, **more):
        with pytest.raises(error, match=word):
            prompt_attention(q, k, k if v is None else v, ends, 0.1, **more)

    refuse(RuntimeError, "ROCm device tensor", q=q.cpu())
    refuse(ValueError, "must be", q=q.flatten(1))
    refuse(ValueError, "shapes do not match", v=k[:5])
    refuse(ValueError, "shapes do not match", q=q[..., :32])
    refuse(ValueError, "share a dtype", q=q.half())
    refuse(ValueError, "not supported", q=q.double(), k=k.double())
    refuse(ValueError, "64 or 128", q=q[..., :32], k=k[..., :32])
    refuse(ValueError, "divisible", q=q[:, :3])
    refuse(ValueError, "need cu_seqlens_k", k=k[:5])
    refuse(ValueError, "must be", ends=torch.zeros(1, 2, dtype=torch.int32))
    refuse(ValueError, "must be", ends=torch.zeros(0, dtype=torch.int32))
    refuse(ValueError, "whole numbers", ends=torch.tensor([0.0, 6.0]))
    refuse(IndexError, "must rise", ends=torch.tensor([0, 7]))
    refuse(IndexError, "must rise", ends=torch.tensor([-1, 6]))
    refuse(IndexError, "must rise", ends=torch.tensor([0, 5, 3, 6]))
    refuse(IndexError, "must rise", k=k[:4], cu_seqlens_k=torch.tensor([0, 6]))
    refuse(ValueError, "ends of keys", cu_seqlens_k=torch.tensor([0, 3, 6]))
    refuse(ValueError, "out must be", out=q[:5])
    refuse(ValueError, "must not overlap", out=q[:1].expand(6, 4, 64))
    with pytest.raises(ValueError, match="finite"):
        prompt_attention(q, k, k, ends, float("nan"))
    assert prompt_attention(q[:0], k[:0], k[:0], torch.tensor([0]), 0.1).shape == (0, 4, 64)
    assert not prompt_attention(q + 1, k, k, torch.tensor([0]), 0.1).any()  # no sequence at all
    assert not prompt_attention(q + 1, k[:0], k[:0], ends, 0.1, torch.tensor([0, 0])).any()  # no keys


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hkv", [(16, 2), (4, 4)])
def test_falling_ends_on_the_device_touch_the_output_only(hq, hkv, dtype):
    # overlapping sequences, more tiles than workgroups, keys that end before they begin:
    # rows of `out` are undefined, what lies around and between them is not
    g = torch.Generator().manual_seed(31)
    q, k, v = (t.to(DEV) for t in _make(g, 300, 900, hq, hkv, 64, dtype))
    held = torch.full((5 + 300 + 5, hq, 96), 7.0, dtype=dtype, device=DEV)
    keep = [t.clone() for t in (q, k, v)]
    for ends_q, ends_k in (([0, 100, 50, 200], [0, 100, 50, 200]), ([200, 0, 300, 100], [0, 900, 0, 900]),
                           ([0, 300] * 40, [0, 900] * 40), ([0, 300] * 100, [0, 300] * 100),
                           ([300, 200, 100, 0], [900, 0, 900, 0]), ([-5, 300, -5, 1 << 30], [-5, 900, -5, 1 << 30])):
        print(dtype, hq, ends_q[:4], len(ends_q), flush=True)
        ends = [torch.tensor(e, dtype=torch.int32, device=DEV) for e in (ends_q, ends_k)]
        prompt_attention(q, k, v, ends[0], 0.125, ends[1], out=held[5:305, :, 16:80])
        got = prompt_attention(q, k, v, ends[0], 0.125, ends[1])
        torch.cuda.synchronize()
        assert got.shape == q.shape
        assert bool((held[:5] == 7).all()) and bool((held[305:] == 7).all())
        assert bool((held[..., :16] == 7).all()) and bool((held[..., 80:] == 7).all())
        assert all(torch.equal(a, b) for a, b in zip((q, k, v), keep))
    # and calls in order are what they were
    _check(dtype, 4, 2, 64, [40, 90], seed=32)
