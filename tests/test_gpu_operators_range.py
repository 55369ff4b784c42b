"""GPU: the prompt and decode attentions where magnitudes lie far apart or near
the ends of float32's range, against 64 bits.

Tolerance over 4-bit pages. A logit sums, per 32 dims, a query element times a
whole number below 16, then step times that sum and offset times the query's sum:
fewer than 67 float32 roundings of at most 2^-24 of the sum of the absolute terms
OF EACH GROUP of 32 dims, whatever the other groups hold. Beside that a 16-bit
query element may be off by 2^-36 of its row's largest, and, where products lie
below float32's normal range, by an absolute 2^-149 that the row's unit scales
up (`tiny`, given by the test that goes there). Weights: 2^-15 (two bf16 parts,
and their sum's roundings; float32 2^-22); a relative change e of every weight
moves an output by at most 2 e sum p |v|. The values' products hold step * 144 (float32: step * 16) +
|offset| and round at most once a key of a lane; last comes the type's half step."""

import numpy as np
import pytest
import torch

from cacheblend_vllm import kv_layout as KL
from cacheblend_vllm.attention import paged_attention_int4, prompt_attention
from oracle import operators as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _held(rows, d):
    """|steps| and |offsets| [.., groups] of 4-bit rows."""
    words = np.ascontiguousarray(rows[..., d // 2:]).view(np.uint16).astype(np.uint32) << 16
    both = np.abs(words.view(np.float32).astype(np.float64)).reshape(*rows.shape[:-1], d // 32, 2)
    return both[..., 0], both[..., 1]


def _decode(dtype, q, k, v, scale, tiny=0.0, size=16):
    """One sequence whose pages hold k, v [tokens, heads, d] (64 bits); q [rows, hq, d]."""
    n, heads, d = k.shape
    rows, hq = q.shape[:2]
    blocks = (n + size - 1) // size
    held = np.zeros((2, blocks * size, heads, KL.int4_row_bytes(d)), dtype=np.uint8)
    held[:, :n] = R.int4_encode(np.stack([k, v]))
    pages = torch.from_numpy(held).reshape(2, blocks, size, heads, -1).to(DEV)
    tables = torch.arange(blocks, dtype=torch.int32)[None]
    got = paged_attention_int4(q[None].to(DEV), pages, tables.to(DEV), torch.tensor([n], device=DEV), size, scale)
    torch.cuda.synchronize()
    qn = q.double().numpy()
    want, mass = R.paged_attention_int4(qn[None], *pages.cpu().numpy(), tables.numpy(), [n], scale)
    (ks, ko), (vs, vo) = (_held(p[:n], d) for p in held)
    group = hq // heads
    qg = np.abs(qn).reshape(rows, hq, d // 32, 32)
    # [rows, hq, keys, groups] -> the largest sum over the groups of any key
    terms = np.einsum("rhg,nhg->rhn", qg.sum(-1), (16 * ks + ko).repeat(group, axis=1)).max(-1)
    exact = dtype == F32
    e = 67 * 2.0 ** -24 * abs(scale) * terms + tiny + (2.0 ** -22 if exact else 2.0 ** -15) + (n / 16 + 64) * 2.0 ** -24
    if not exact:
        e = e + abs(scale) * 2.0 ** -36 * np.abs(qn).max(-1) * 32 * 15 * ks.sum(-1).max(0).repeat(group)
    values = ((16 if exact else 144) * vs + vo).max(0).repeat(group, axis=0).repeat(32, axis=1)
    tol = 2 * e[..., None] * mass[0] + (n / 16 + 64) * 2.0 ** -24 * values
    tol = tol + torch.finfo(dtype).eps / 2 * np.abs(want[0]) + (2.0 ** -25 if dtype == F16 else 1e-38)
    err = np.abs(got[0].double().cpu().numpy() - want[0])
    print(f"decode {dtype} {hq}/{heads}x{d} of {n}: worst {float((err / tol).max()):.3f} of the bound", flush=True)
    assert np.all(err <= tol)
    return got[0]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("outlier,rest,step", [(200.0, 0.1, 5.0), (200.0, 0.03, 15.0), (1000.0, 0.1, 5.0)])
def test_an_outlier_of_the_query_beside_small_elements(outlier, rest, step, dtype):
    # a large element of q over keys that are small there: the other groups' elements
    # keep their bits
    g = np.random.default_rng(int(outlier + step))
    for d, hq, heads, n in ((128, 8, 2, 300), (64, 4, 4, 90), (128, 32, 2, 700)):
        q = g.standard_normal((1, hq, d)) * rest
        q[..., 5] = outlier
        k = g.standard_normal((n, heads, d)) * step
        k[..., :32] *= 0.004 / step
        v = g.standard_normal((n, heads, d))
        _decode(dtype, torch.from_numpy(q).to(dtype), k, v, d ** -0.5)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_an_outlier_within_a_group_of_the_query(dtype):
    # its keys are the group's lowest: code 0, all in the offset
    g = np.random.default_rng(3)
    for d, hq, heads, n in ((128, 8, 2, 300), (64, 4, 4, 90)):
        q = g.standard_normal((1, hq, d)) * 0.1
        q[..., 5] = 200.0
        k = g.standard_normal((n, heads, d)) * 5
        k[..., 5] = -32.0
        v = g.standard_normal((n, heads, d))
        _decode(dtype, torch.from_numpy(q).to(dtype), k, v, d ** -0.5)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("big", [1.6e35, 1e36, 1e38, 1e-36])
def test_queries_near_the_ends_of_the_range(big, dtype):
    g = np.random.default_rng(4)
    for d, hq, heads, n in ((128, 8, 2, 300), (64, 4, 4, 90), (128, 32, 2, 33)):
        q = g.uniform(0.5, 2, (1, hq, d)) * big
        k = g.standard_normal((n, heads, d)) / big
        v = g.standard_normal((n, heads, d))
        # a row's unit is at most 2^24 * 2^(127 - 14) * scale * log2 e: 12 products that may lie
        # below 2^-126 round by 2^-150 each
        _decode(dtype, torch.from_numpy(q).to(dtype), k, v, d ** -0.5,
                tiny=12 * 2.0 ** -150 * 2.0 ** 137 * d ** -0.5 if big > 1 else 0.0)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("big", [1e33, 1e34, 1e36, 2e37])
def test_values_near_the_end_of_the_range(big, dtype):
    g = np.random.default_rng(5)
    for d, hq, heads, n in ((128, 8, 2, 300), (64, 4, 4, 90), (128, 32, 2, 33), (64, 8, 1, 1000)):
        q = g.standard_normal((1, hq, d))
        k = g.standard_normal((n, heads, d))
        v = g.standard_normal((n, heads, d)) * big
        got = _decode(dtype, torch.from_numpy(q).to(dtype), k, v, d ** -0.5)
        assert bool(got.isfinite().all())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_small_values(dtype):
    g = np.random.default_rng(6)
    for d, hq, heads, n in ((128, 8, 2, 300), (64, 4, 4, 90)):
        q = g.standard_normal((1, hq, d))
        k = g.standard_normal((n, heads, d))
        v = g.standard_normal((n, heads, d)) * 1e-25
        _decode(dtype, torch.from_numpy(q).to(dtype), k, v, d ** -0.5)


def _one_dim(n, heads, d, at):
    """Keys [n, heads, d]: `at` in dim 0, nothing elsewhere."""
    k = np.zeros((n, heads, d))
    k[..., 0] = np.asarray(at)[:, None]
    return k


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_logits_past_the_range_in_log2_units_over_pages(dtype):
    # 2.4e38 .. 3.3e38: finite, but not times log2 e. One key leads by 1e37 and
    # more, a thousand times a logit's rounding: its value alone is left
    g = np.random.default_rng(7)
    for d, heads, n in ((128, 2, 300), (64, 1, 90), (128, 1, 5000)):
        for sign, rest in ((1, 2.4e18), (-1, 3.2e18), (1, -3.0e18)):
            lead = int(g.integers(n))
            at = np.full(n, rest)
            at[lead] = 3.2e18 if sign > 0 else 2.5e18
            q = torch.zeros(1, 4 * heads, d, dtype=dtype)
            q[..., 0] = sign * 1e20
            v = g.standard_normal((n, heads, d))
            size = 16
            blocks = (n + size - 1) // size
            held = np.zeros((2, blocks * size, heads, KL.int4_row_bytes(d)), dtype=np.uint8)
            held[:, :n] = R.int4_encode(np.stack([_one_dim(n, heads, d, at), v]))
            pages = torch.from_numpy(held).reshape(2, blocks, size, heads, -1).to(DEV)
            got = paged_attention_int4(q.to(DEV), pages, torch.arange(blocks, device=DEV)[None],
                                       torch.tensor([n], device=DEV), size, 1.0)
            want = R.int4_decode(held[1, lead]).repeat(4, axis=0)
            _, offset = _held(held[1, lead], d)
            step, _ = _held(held[1, lead], d)
            room = (144 * step + offset).repeat(4, axis=0).repeat(32, axis=-1)
            tol = (2.0 ** -14 if dtype == BF16 else 2.0 ** -21) * room + torch.finfo(dtype).eps / 2 * np.abs(want)
            assert np.all(np.abs(got[0].double().cpu().numpy() - want) <= tol), (d, n, sign, rest)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("largest", [3.2e38, 2.3e38, 1e30, 1e12, 3e9, 1e8])
def test_large_logits_of_prompts(largest, dtype):
    # past float32's range in log2 units, and past what a multiply-add's exponent holds:
    # rows whose keys hold one leading logit, or many equal ones
    top = 3.2e4
    scale = largest / top
    g = torch.Generator().manual_seed(8)
    for d, lens, keys in ((128, [70, 3], [300, 3]), (64, [200], [200]), (128, [20], [3000])):
        q = torch.zeros(sum(lens), 4, d)
        q[..., 0] = 1.0
        k = torch.zeros(sum(keys), 2, d)
        k[..., 0] = -top * 0.75
        v = torch.randn(sum(keys), 2, d, generator=g)
        ends_q, ends_k = np.concatenate([[0], np.cumsum(lens)]), np.concatenate([[0], np.cumsum(keys)])
        for c in ends_k[:-1]:
            k[c, :, 0] = top       # every row's leading key
        q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)

        def run():
            got = prompt_attention(q.to(DEV), k.to(DEV), v.to(DEV), torch.tensor(ends_q, device=DEV), scale,
                                   torch.tensor(ends_k, device=DEV))
            return got.double().cpu()

        got = run()
        for a, b, c in zip(ends_q[:-1], ends_q[1:], ends_k[:-1]):
            want = v[c].double().repeat_interleave(2, dim=0)[None].expand(int(b - a), -1, -1)
            assert torch.equal(got[a:b], want), (d, lens, keys)
        # all keys alike: the mean of what a row sees
        k[..., 0] = float(k[0, 0, 0])
        got = run()
        want, mass = R.prompt_attention(*(t.double().numpy() * f for t, f in ((q, 0.0), (k, 0.0), (v, 1.0))), ends_q, ends_k, 1.0)
        tol = (2.0 ** -23 * sum(keys) + torch.finfo(dtype).eps) * mass + 2.0 ** -24
        assert np.all(np.abs(got.numpy() - want) <= tol), (d, lens, keys)
