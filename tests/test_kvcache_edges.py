"""The paged key-value cache where values, lengths and layouts are at their limits.  Bounds as in test_kvcache.py, unless a test
says otherwise."""
import math

import pytest
import torch

import tritonformer_b200._lib as L

from test_kvcache import U, Cache, _attend_reference, _check_mass, _gen, _mass_reference
from tritonformer_b200 import kvcache

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("group", [1, 4, 5, 8, 9, 16, 24])
def test_attention_is_rounded_once_whatever_the_group(group, hd, dtype):
    """The weights enter the second product in two parts, so u^2 of them is lost and not u; 32-bit sums of a few tiles lose 2^-17."""
    c = Cache([129, 40, 700], 2, hd, 32, dtype)
    q = (2 * torch.randn((3, 2 * group, hd), device="cuda", generator=_gen(1))).to(dtype)
    ref, _, weights = _attend_reference(q, c.copy(), None)
    bound = []
    for b, n in enumerate(c.lengths):
        p, r = c.at(b, torch.arange(n, device="cuda"))
        v = c.v[p, :, r].double().abs().repeat_interleave(group, 1)  # (n, heads, hd)
        scale = torch.einsum("hn,nhd->hd", weights[b], v)
        bound.append(U[dtype] * ref[b].abs() + (1e-5 + 2.0 ** -17 + U[dtype] ** 2) * scale + n * 2.0 ** -29 * v.amax() + 1e-7)
    out = kvcache.paged_attention(q, c.k, c.v, c.tables, c.len)
    assert ((out.double() - ref).abs() <= torch.stack(bound)).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("group", [1, 4, 5, 8, 16])
def test_attention_of_an_infinite_value_is_infinite(group, hd, dtype):
    """A weight times infinity is infinity, in this value's column alone; equal weights, in tiles before and behind it as well."""
    n = 600
    c = Cache([n], 1, hd, 16, dtype)
    p, r = c.at(0, torch.tensor([7, 300], device="cuda"))
    c.v[p, 0, r, 3] = torch.tensor([math.inf, 1.0], device="cuda", dtype=dtype)
    c.v[p, 0, r, 9] = torch.tensor([1.0, -math.inf], device="cuda", dtype=dtype)
    q = torch.zeros((1, group, hd), device="cuda", dtype=dtype)
    out = kvcache.paged_attention(q, c.k, c.v, c.tables, c.len)[0].double()
    p, r = c.at(0, torch.arange(n, device="cuda"))
    v = c.v[p, 0, r].double()
    want = v.mean(0)
    plain = want.isfinite()
    assert torch.equal(out[:, ~plain], want[~plain].expand(group, -1)) and int((~plain).sum()) == 2
    bound = 2 * U[dtype] * v.abs().mean(0) + 1e-5  # the rests of the finite columns may go with the infinite one
    assert ((out - want).abs() <= bound)[:, plain].all()


# ------------------------------------------------------------------------------------------------------- prompt mass


@gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("T", [100, 256, 640, 1300])
def test_mass_of_heads_that_follow_one_another(T, hd):
    """Runs of one tile, or of an odd number, each with the log-sum-exps of another query head: none sees its neighbour's."""
    q = (2 * torch.randn((2, 6, T, hd), device="cuda", generator=_gen(T))).half()
    q *= torch.tensor([0.1, 1.5, 1.0, 2.0, 0.2, 1.0], device="cuda").half()[:, None, None]  # sums far apart
    k = torch.randn((2, 2, T, hd), device="cuda", generator=_gen(T + 1)).half()
    slopes = torch.rand((6,), device="cuda", generator=_gen(0)) * 0.3
    first = _check_mass(2, 2, 3, T, hd, torch.float16, slopes=slopes, q=q, k=k)
    lse = _mass_reference(q, k, None, slopes)[1]
    for _ in range(20):
        assert torch.equal(first, kvcache.prompt_mass(q, k, lse, attn_bias=slopes))


@gpu
@pytest.mark.parametrize("alibi", [False, True])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("T,counts", [(200, [150, 1, 0]), (512, [300, 256, 511]), (700, [129, 640, 500])])
def test_mass_does_not_see_what_lies_behind_a_prompt(T, counts, hd, alibi):
    """Padding may be NaN or infinite, in the queries, the keys and the log-sum-exps; so may a query whose row gives no weight."""
    q = (2 * torch.randn((3, 4, T, hd), device="cuda", generator=_gen(T))).to(torch.bfloat16)
    k = torch.randn((3, 2, T, hd), device="cuda", generator=_gen(T + 1)).to(torch.bfloat16)
    slopes = torch.rand((4,), device="cuda", generator=_gen(0)) * 0.3 if alibi else None
    clean = _check_mass(3, 2, 2, T, hd, torch.bfloat16, counts=counts, slopes=slopes, q=q, k=k)
    lse = _mass_reference(q, k, counts, slopes)[1]
    n = torch.tensor(counts, dtype=torch.int32, device="cuda")
    for value in (math.nan, math.inf, -math.inf):
        bad = q.clone(), k.clone(), lse.clone()
        for b, count in enumerate(counts):
            for x in bad:
                x[b, :, count:] = value
        assert torch.equal(clean, kvcache.prompt_mass(*bad, n, attn_bias=slopes))
    lse[:, :, 40:60] = -math.inf
    want = kvcache.prompt_mass(q, k, lse, n, attn_bias=slopes)
    for value in (math.nan, math.inf):
        bad = q.clone()
        bad[:, :, 40:60] = value
        assert torch.equal(want, kvcache.prompt_mass(bad, k, lse, n, attn_bias=slopes))
    assert want.isfinite().all() and L.device_status() == 0
