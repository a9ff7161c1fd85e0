"""The paged key-value cache where values, lengths and layouts are at their limits.  Bounds as in test_kvcache.py, unless a test
says otherwise."""
import ctypes
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


# --------------------------------------------------------------------------------------------------- append and evict


def _pool(c):
    return [x.clone() for x in (c.k, c.v, c.mass, c.positions)]


def _equal(a, b):
    return all(torch.equal(x.nan_to_num(7), y.nan_to_num(7)) for x, y in zip(a, b))


@gpu
@pytest.mark.parametrize("hd,off", [(32, 0), (64, 1), (128, 0)])
def test_append_of_more_keys_than_there_is_room_for(hd, off):
    """Those that fit are written, nothing else is, and it is reported; the other sequence gets all of its own."""
    c = Cache([46, 10], 2, hd, 16, torch.float16, room=2)
    c.tables = torch.arange(6, dtype=torch.int32, device="cuda").view(2, 3).flip(0).contiguous()  # two full tables of 48 slots
    flat = torch.randn((2 * 2 * 9 * hd + 8,), device="cuda", generator=_gen(1)).half()
    keys = flat[off:off + 2 * 2 * 9 * hd].view(2, 2, 9, hd)
    want = c.copy()
    for b, n in ((0, 2), (1, 9)):
        p, r = c.at(b, c.lengths[b] + torch.arange(n, device="cuda"))
        want.k[p, :, r], want.v[p, :, r] = keys[b, :, :n].transpose(0, 1), -keys[b, :, :n].transpose(0, 1)
        want.mass[p, :, r] = 0.0
        want.positions[p, :, r] = (c.lengths[b] + torch.arange(n, device="cuda", dtype=torch.int32))[:, None]
    kvcache.cache_append(c.k, c.v, c.tables, c.len, keys, -keys, mass=c.mass, positions=c.positions)
    assert L.device_status(reset=True) == 0x7201
    assert _equal(_pool(c), _pool(want))
    for counts, lengths in (([0, 0], [-3, 10]), ([-1, 0], [46, 10]), ([0, 0], [49, 10])):
        kvcache.cache_append(c.k, c.v, c.tables, torch.tensor(lengths, dtype=torch.int32, device="cuda"), keys, -keys,
                             torch.tensor(counts, dtype=torch.int32, device="cuda"), c.mass, c.positions)
        assert L.device_status(reset=True) == 0x7201
        assert _equal(_pool(c), _pool(want))
    tables = c.tables.clone()
    tables[0, 2] = c.pages
    kvcache.cache_append(c.k, c.v, tables, c.len, keys[:, :, :2], keys[:, :, :2], torch.tensor([2, 0], dtype=torch.int32, device="cuda"),
                         c.mass, c.positions)
    assert L.device_status(reset=True) == 0x7200
    assert _equal(_pool(c), _pool(want))


@gpu
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("lengths,keep", [([100, 100], 50), ([9000, 9000], 3000)])  # one block a head, and clusters
def test_evict_leaves_the_others_alone(lengths, keep, in_place):
    """A bad page or length of one sequence is reported; the other one is cut as ever, and no row of anybody else changes."""
    def evict(c, tables, n):
        out = None if in_place else tuple(torch.zeros_like(x) for x in (c.k, c.v, c.mass, c.positions))
        left = kvcache.cache_evict(c.k, c.v, c.mass, c.positions, tables, n, keep, 0, out=out, out_tables=None if in_place else c.tables)
        return left, _pool(c) if in_place else [x.clone() for x in out]

    good = Cache(lengths, 2, 64, 16, torch.float16)
    clean = _pool(good)
    own = torch.zeros(good.pages, dtype=torch.bool, device="cuda")
    own[good.tables[0].long()] = True  # pages of the sequence with the fault
    left, want = evict(good, good.tables, good.len)
    assert L.device_status() == 0 and left.tolist() == [keep, keep]
    for bad in (-1, good.pages, 2 ** 31 - 1):
        c = Cache(lengths, 2, 64, 16, torch.float16)
        tables = c.tables.clone()
        tables[0, 2] = bad
        left, got = evict(c, tables, c.len)
        assert L.device_status(reset=True) == 0x7200 and left.tolist() == [keep, keep]
        assert _equal([x[~own] for x in got], [x[~own] for x in want])
    c = Cache(lengths, 2, 64, 16, torch.float16)
    n = c.len.clone()
    n[0] = -1
    left, got = evict(c, c.tables, n)
    assert L.device_status(reset=True) == 0x7201 and left.tolist() == [0, keep]
    assert _equal([x[~own] for x in got], [x[~own] for x in want])
    untouched = clean if in_place else [torch.zeros_like(x) for x in clean]
    assert _equal([x[own] for x in got], [x[own] for x in untouched])


def test_evict_in_place_is_slot_by_slot():
    """The input's own buffers under another shape are no output: their slots are not the input's."""
    def strides(*s):
        return (ctypes.c_int64 * len(s))(*s)

    one, two, three = ctypes.c_void_p(256), ctypes.c_void_p(512), strides(1024, 1024, 64)

    def evict(page=16, pages=4, width=2, out=three, k_out=one, mass_out=one):
        return L.lib.tfb_cache_evict(one, one, one, None, one, one, None, k_out, k_out, mass_out, None, one, two, 1, 1, 64, 4, 0, 16, 4,
                                     2, 2, three, page, pages, width, 2, out, one, 8, 0, None)

    assert evict() == -1 and b"scratch" in L.lib.tfb_last_error()  # looked at last: nothing is launched here
    for bad in (dict(page=32, pages=2), dict(out=strides(2048, 1024, 64)), dict(out=strides(1024, 1024, 128)), dict(page=8, mass_out=two),
                dict(page=8, k_out=two)):
        assert evict(**bad) == -1 and b"other shape" in L.lib.tfb_last_error(), bad
    for good in (dict(page=8, k_out=two, mass_out=two), dict(out=strides(2048, 1024, 64), k_out=two), dict(out=strides(1024, 7 * 8, 64)),
                 dict(pages=3)):  # buffers of their own, a stride that says nothing, fewer of the pages
        assert evict(**good) == -1 and b"scratch" in L.lib.tfb_last_error(), good
