"""The paged key-value cache: decode attention, prompt mass, append and eviction against their definitions in 64 bits.

Tolerances.  u is the rounding of the 16-bit type (2^-11, 2^-8).  An output o = sum w v is rounded once, the weights once before
the second product (u sum w |v|); scores of up to some 20 (in log2 units) carry an absolute error of some 1e-6 from 32-bit sums,
taken as 1e-5 of the weights; a weight below 2^-18 of the largest rounds to fp16's subnormal grid, 2^-29 of the largest a key.
A mass is a sum of weights in 32 bits: 2e-5 of the weights and 2^-22 of the sum.  Rows that are moved are equal."""
import ctypes
import math

import pytest
import torch

import tritonformer_b200._lib as L
from tritonformer_b200 import kvcache
from tritonformer_b200.transformer import generate_alibi_mask

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
gpu = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


class Cache:
    """A pool with the pages of `lengths` (plus `room`) keys dealt out in random order; what no slot in use holds is NaN."""

    def __init__(self, lengths, heads, hd, page, dtype, seed=0, room=1, spare=3):
        g = _gen(seed)
        self.lengths, self.page = lengths, page
        need = [-(-(n + room) // page) for n in lengths]
        ids = torch.randperm(sum(need) + spare, generator=g, device="cuda").tolist()
        self.pages, width = len(ids), max(need + [1])
        self.tables = torch.full((len(lengths), width), -7, dtype=torch.int32)  # never read where nothing is
        for b, n in enumerate(need):
            self.tables[b, :n] = torch.tensor([ids.pop() for _ in range(n)], dtype=torch.int32)
        self.tables = self.tables.cuda()
        shape = (self.pages, heads, page)
        self.k = torch.full((*shape, hd), math.nan, device="cuda", dtype=dtype)
        self.v = self.k.clone()
        self.mass = torch.full(shape, math.nan, device="cuda")
        self.positions = torch.full(shape, -12345, device="cuda", dtype=torch.int32)
        for b, n in enumerate(lengths):
            p, r = self.at(b, torch.arange(n, device="cuda"))
            self.k[p, :, r] = torch.randn((n, heads, hd), generator=g, device="cuda").to(dtype)
            self.v[p, :, r] = torch.randn((n, heads, hd), generator=g, device="cuda").to(dtype)
            self.mass[p, :, r] = torch.rand((n, heads), generator=g, device="cuda")
            order = torch.rand((n, heads), generator=g, device="cuda").argsort(0)
            self.positions[p, :, r] = (3 * order + 1).to(torch.int32)
        self.len = torch.tensor(lengths, dtype=torch.int32, device="cuda")

    def at(self, b, slots):
        return self.tables[b].long()[slots // self.page], slots % self.page

    def copy(self):
        other = Cache.__new__(Cache)
        other.__dict__.update({k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in self.__dict__.items()})
        return other


def _rounded_bias(slopes, dist, kind):
    """-slope * distance as a table of that type holds it (transformer.generate_alibi_mask), or exactly."""
    if kind is None:
        return -slopes.double()[:, None] * dist.double()
    return (-dist.to(kind) * slopes.to(kind)[:, None]).double()


def _attend_reference(q, c, new, slopes=None, rounded=None, query_positions=None, use_positions=False):
    """Per sequence: output, error bound of the output, weights (heads, n), in 64 bits; writes the new rows into c."""
    B, heads, hd = q.shape
    kv = c.k.shape[1]
    outs, bounds, weights = [], [], []
    for b in range(B):
        n = c.lengths[b]
        here = int(query_positions[b]) if query_positions is not None else (n if new else n - 1)
        if new:
            p, r = c.at(b, torch.tensor(n, device="cuda"))
            c.k[p, :, r], c.v[p, :, r] = new[0][b], new[1][b]
            c.positions[p, :, r] = here
            n += 1
        slots = torch.arange(n, device="cuda")
        p, r = c.at(b, slots)
        o, bound, ws = [], [], []
        for h in range(heads):
            k, v = c.k[p, h // (heads // kv), r].double(), c.v[p, h // (heads // kv), r].double()
            s = k @ q[b, h].double() / math.sqrt(hd)
            if slopes is not None:
                pos = c.positions[p, h // (heads // kv), r] if use_positions else slots
                s = s + _rounded_bias(slopes[h:h + 1], here - pos, rounded)[0]
            w = torch.softmax(s, 0) if n else s
            u, scale = U[q.dtype], (w @ v.abs() if n else torch.zeros(hd, device="cuda", dtype=torch.double))
            o.append(w @ v if n else torch.zeros(hd, device="cuda", dtype=torch.double))
            top = v.abs().amax() if n else 0.0
            bound.append(u * (o[-1].abs() + scale) + 1e-5 * scale + n * 2.0 ** -29 * top + 1e-7)
            ws.append(w)
        outs.append(torch.stack(o))
        bounds.append(torch.stack(bound))
        weights.append(torch.stack(ws))
    return torch.stack(outs), torch.stack(bounds), weights


def _check_attention(lengths, heads, group, hd, page, dtype, new=True, mode=None, stats=False, seed=0, q_scale=2.0):
    c = Cache(lengths, heads, hd, page, dtype, seed)
    g = _gen(seed + 1)
    B = len(lengths)
    q = (q_scale * torch.randn((B, heads * group, hd), generator=g, device="cuda")).to(dtype)
    kv = [torch.randn((B, heads, hd), generator=g, device="cuda").to(dtype) for _ in range(2)] if new else None
    slopes = torch.rand((heads * group,), generator=g, device="cuda") * 0.3 if mode is not None else None
    at = torch.tensor([3 * n + 7 for n in lengths], dtype=torch.int32, device="cuda") if stats else None
    want = c.copy()
    ref, bound, weights = _attend_reference(q, want, kv, slopes, None, at, stats)
    mass_out = torch.full_like(c.mass, -1.0) if stats else None
    out = kvcache.paged_attention(q, c.k, c.v, c.tables, c.len, *(kv or (None, None)), attn_bias=slopes, query_positions=at,
                                  mass=c.mass if stats else None, positions=c.positions if stats else None, mass_out=mass_out)
    assert L.device_status() == 0
    excess = ((out.double() - ref).abs() - bound).max().item() if B else 0.0
    assert excess <= 0, excess
    assert torch.equal(c.k.nan_to_num(7), want.k.nan_to_num(7)) and torch.equal(c.v.nan_to_num(7), want.v.nan_to_num(7))
    if stats:
        assert torch.equal(c.positions, want.positions)
        untouched = torch.ones_like(c.mass, dtype=torch.bool)
        for b, w in enumerate(weights):
            n = w.shape[1]
            p, r = c.at(b, torch.arange(n, device="cuda"))
            got = mass_out[p, :, r].double()
            w = w.view(heads, group, n).sum(1).T
            had = c.mass[p, :, r].double()
            if new:
                had[-1] = 0
            assert ((got - had - w).abs() <= 2e-5 * w + 2.0 ** -22 * (had + w) + 1e-9).all()
            untouched[p, :, r] = False
        assert (mass_out[untouched] == -1).all()
    return out


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("lengths,page", [([0], 16), ([1], 1), ([5, 0, 17], 7), ([63, 64, 65, 31, 32, 33], 48), ([300, 2], 64),
                                          ([2500], 128), ([15, 16, 4000, 1], 16)])
def test_attention_lengths_and_pages(lengths, page, hd, dtype):
    _check_attention(lengths, 2, 1, hd, page, dtype)
    _check_attention(lengths, 2, 1, hd, page, dtype, new=False, stats=True, mode="exact", seed=5)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,group", [(1, 1), (3, 2), (2, 7), (2, 8), (1, 9), (2, 16), (1, 17), (1, 40), (1, 128), (12, 1)])
def test_attention_head_layouts(heads, group, dtype):
    for hd in (64, 128):
        _check_attention([129, 40, 700], heads, group, hd, 32, dtype, stats=True, mode="exact")


@gpu
def test_attention_many_sequences():
    """More sequences than a block has threads, most of them without keys or with one."""
    g = torch.Generator().manual_seed(3)
    lengths = [int(n) for n in torch.randint(0, 40, (600,), generator=g) * (torch.rand((600,), generator=g) < 0.4)]
    _check_attention(lengths, 2, 1, 64, 16, torch.float16, new=False, stats=True)
    _check_attention(lengths, 1, 2, 32, 16, torch.float16, new=True)
    _check_attention([0] * 5, 1, 2, 32, 16, torch.float16, new=False, stats=True)


@gpu
def test_attention_long():
    """One row shared by every warp of the grid, and a long row among short ones."""
    _check_attention([70001], 1, 3, 128, 64, torch.bfloat16, stats=True)
    _check_attention([3, 90000, 1, 257, 0], 2, 1, 64, 256, torch.float16, stats=True, mode="exact")


@gpu
def test_attention_bit_equal_runs_and_other_stream():
    c = Cache([3000, 17, 900], 4, 64, 32, torch.float16)
    q = torch.randn((3, 8, 64), device="cuda", generator=_gen(1)).half()
    mass = [torch.zeros_like(c.mass) for _ in range(3)]
    base = c.mass.nan_to_num(0)
    outs = [kvcache.paged_attention(q, c.k, c.v, c.tables, c.len, mass=base, mass_out=m) for m in mass[:2]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs.append(kvcache.paged_attention(q, c.k, c.v, c.tables, c.len, mass=base, mass_out=mass[2]))
    side.synchronize()
    for o, m in zip(outs[1:], mass[1:]):
        assert torch.equal(outs[0], o) and torch.equal(mass[0], m)


@gpu
def test_attention_in_a_graph():
    c = Cache([100, 30], 2, 64, 16, torch.float16)
    q = torch.randn((2, 2, 64), device="cuda").half()
    eager = kvcache.paged_attention(q, c.k, c.v, c.tables, c.len)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kvcache.paged_attention(q, c.k, c.v, c.tables, c.len)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, eager)
    c.len.copy_(torch.tensor([7, 0]))  # the lengths are read where they lie
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, kvcache.paged_attention(q, c.k, c.v, c.tables, c.len)) and (out[1] == 0).all()


@gpu
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16])
def test_attention_with_the_models_table(kind):
    """An ALiBi table: slopes and rounding are taken from it, as the training attention does."""
    heads, n, hd = 6, 900, 64
    table = generate_alibi_mask(1024, heads, dtype=kind)[0]
    slopes = -table[:, 1, 0].float()
    c = Cache([n, 33], heads, hd, 64, torch.float16)
    q = torch.randn((2, heads, hd), device="cuda", generator=_gen(2)).half()
    new = [torch.randn((2, heads, hd), device="cuda", generator=_gen(s)).half() for s in (3, 4)]
    ref, bound, _ = _attend_reference(q, c.copy(), new, slopes, kind)
    out = kvcache.paged_attention(q, c.k, c.v, c.tables, c.len, *new, attn_bias=table)
    assert ((out.double() - ref).abs() <= bound).all()


@gpu
def test_attention_strides_and_alignment():
    """Views of one projection's output, rows at odd addresses, pages of a pool that holds other layers too."""
    B, heads, hd, page = 2, 3, 64, 16
    c = Cache([50, 21], heads, hd, page, torch.float16)
    pool = torch.full((c.pages, 4, 2, page, heads, hd), math.nan, device="cuda", dtype=torch.float16)
    k, v = (pool[:, 1, i].permute(0, 2, 1, 3) for i in (0, 1))  # (pages, heads, page, hd), heads inside the slots
    k.copy_(c.k)
    v.copy_(c.v)
    for off in (0, 1, 2, 8):
        flat = torch.randn((B * 9 * hd * heads + 64,), device="cuda", generator=_gen(off)).half()
        qkv = flat[off:off + B * 9 * hd * heads].view(B, 9 * heads, hd)
        q, kn, vn = qkv[:, 0:heads], qkv[:, heads:2 * heads], qkv[:, 4 * heads:7 * heads:3]
        ref, bound, _ = _attend_reference(q, c.copy(), (kn, vn))
        out = kvcache.paged_attention(q, k, v, c.tables, c.len, kn, vn)
        assert ((out.double() - ref).abs() <= bound).all(), off
        transposed = q.transpose(1, 2).contiguous().transpose(1, 2)  # no unit stride on head_dim
        assert torch.equal(out, kvcache.paged_attention(transposed, k, v, c.tables, c.len, kn, vn))
    assert pool[:, [0, 2, 3]].isnan().all()
    wide = torch.full((B, 40), -3, dtype=torch.int32, device="cuda")
    wide[:, 5:5 + c.tables.shape[1]] = c.tables
    assert torch.equal(out, kvcache.paged_attention(q, k, v, wide[:, 5:5 + c.tables.shape[1]], c.len, kn, vn))


@gpu
def test_attention_offsets_beyond_32_bits():
    """Pages whose elements lie beyond 2^31 of the pool's first, and beyond 2^32 bytes."""
    page, heads, hd = 256, 2, 128
    pages = 2 ** 31 // (page * heads * hd) + 5
    k = torch.zeros((pages, heads, page, hd), device="cuda", dtype=torch.float16)
    v = torch.zeros_like(k)
    small = Cache([600], heads, hd, page, torch.float16)
    ids = torch.tensor([pages - 1, pages - 4, pages - 2, pages - 3], device="cuda")[: small.tables.shape[1]]
    k[ids], v[ids] = small.k[small.tables[0].long()], small.v[small.tables[0].long()]
    q = torch.randn((1, 2, hd), device="cuda", generator=_gen(0)).half()
    new = [torch.randn((1, 2, hd), device="cuda", generator=_gen(s)).half() for s in (3, 4)]
    want = kvcache.paged_attention(q, small.k, small.v, small.tables, small.len, *new)
    got = kvcache.paged_attention(q, k, v, ids[None].to(torch.int32), small.len, *new)
    assert torch.equal(want, got)
    assert torch.equal(k[ids[600 // page], :, 600 % page], new[0][0])
    keys = torch.randn((1, heads, 5, hd), device="cuda").half()
    kvcache.cache_append(k, v, ids[None].to(torch.int32), small.len, keys, keys)
    assert torch.equal(k[ids[600 // page], :, 600 % page:600 % page + 5], keys[0])


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_special_values(dtype):
    """Large scores, a maximum that keeps rising, keys at -inf, and NaN that stays with its sequence."""
    _check_attention([400, 3], 2, 2, 64, 16, dtype, q_scale=60.0, stats=True)
    c = Cache([500, 500, 500, 40], 1, 64, 16, dtype)
    q = torch.zeros((4, 1, 64), device="cuda", dtype=dtype)
    q[:, 0, 0] = 8.0
    slots = torch.arange(500, device="cuda")
    for b in (0, 1, 2):
        p, r = c.at(b, slots)
        c.k[p, 0, r] = 0
        # 0: rises by a unit every few keys; 1: the type's lowest value for all but ten keys; 2: all keys at -inf
        c.k[p, 0, r, 0] = (slots / 5 if b == 0 else torch.where(slots >= 490, 0.0, float(torch.finfo(dtype).min)) if b == 1
                           else torch.full_like(slots, -math.inf, dtype=torch.float)).to(dtype)
    p, r = c.at(3, torch.tensor(20, device="cuda"))
    c.k[p, 0, r, 0] = math.nan
    out = kvcache.paged_attention(q, c.k, c.v, c.tables, c.len)
    p, r = c.at(0, slots)
    w = torch.softmax(c.k[p, 0, r, 0].double(), 0)
    v = c.v[p, 0, r].double()
    scale = w @ v.abs()
    assert ((out[0, 0].double() - w @ v).abs() <= U[dtype] * ((w @ v).abs() + scale) + 2e-5 * scale + 1e-6).all()
    p, r = c.at(1, slots[490:])
    v = c.v[p, 0, r].double()
    assert ((out[1, 0].double() - v.mean(0)).abs() <= 3 * U[dtype] * v.abs().mean(0) + 1e-5).all()
    assert (out[2] == 0).all() and out[3].isnan().all()


@gpu
def test_attention_reports_bad_tables_and_lengths():
    c = Cache([40, 40, 40], 2, 64, 16, torch.float16)
    q = torch.randn((3, 2, 64), device="cuda").half()
    want = kvcache.paged_attention(q, c.k, c.v, c.tables, c.len)
    before = c.k.clone(), c.v.clone()
    for bad in (-1, c.pages, 2 ** 31 - 1):
        tables = c.tables.clone()
        tables[1, 1] = bad
        out = kvcache.paged_attention(q, c.k, c.v, tables, c.len)
        assert L.device_status(reset=True) == 0x7200
        assert torch.equal(out[[0, 2]], want[[0, 2]]) and out[1].isfinite().all()
    room = c.tables.shape[1] * 16
    for n in (-5, room, 2 ** 31 - 1):  # with a new key there is no slot for it either
        lengths = c.len.clone()
        lengths[1] = n
        tables = c.tables.clone()
        out = kvcache.paged_attention(q, c.k.nan_to_num(0), c.v.nan_to_num(0), tables, lengths, q, q)
        assert L.device_status(reset=True) == 0x7201
        assert out.isfinite().all()
    with pytest.raises(RuntimeError, match="length"):
        kvcache.paged_attention(q, c.k.nan_to_num(0), c.v.nan_to_num(0), c.tables, lengths)
        L.check_status()
    assert L.device_status(reset=True) == 0x7201
    assert all(torch.equal(a.nan_to_num(7), b.nan_to_num(7)) for a, b in zip(before, (c.k, c.v)))


# ------------------------------------------------------------------------------------------------------- prompt mass


def _mass_reference(q, k, counts, slopes=None, rounded=None):
    """(masses, log-sum-exp) in 64 bits."""
    B, heads, T, hd = q.shape
    kv = k.shape[1]
    at = torch.arange(T, device="cuda")
    dist = at[:, None] - at
    mass, lses = torch.zeros((B, kv, T), device="cuda", dtype=torch.double), torch.zeros((B, heads, T), device="cuda", dtype=torch.double)
    for b in range(B):
        for h in range(heads):
            s = q[b, h].double() @ k[b, h // (heads // kv)].double().T / math.sqrt(hd)
            if slopes is not None:
                s = s + _rounded_bias(slopes[h:h + 1], dist.reshape(-1), rounded).view(T, T)
            s = s.masked_fill(dist < 0, -math.inf)
            lses[b, h] = s.logsumexp(-1)
            w = (s - lses[b, h].float().double()[:, None]).exp()
            n = T if counts is None else counts[b]
            mass[b, h // (heads // kv)] += w[:n].sum(0)
    return mass, lses.float()


def _check_mass(B, kv, group, T, hd, dtype, counts=None, slopes=None, rounded=None, bias=None, q=None, k=None):
    g = _gen(T + hd)
    if q is None:
        q = (2 * torch.randn((B, kv * group, T, hd), generator=g, device="cuda")).to(dtype)
        k = torch.randn((B, kv, T, hd), generator=g, device="cuda").to(dtype)
    want, lse = _mass_reference(q, k, counts, slopes, rounded)
    n = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    got = kvcache.prompt_mass(q, k, lse, n, attn_bias=bias if bias is not None else slopes)
    assert L.device_status() == 0
    assert ((got.double() - want).abs() <= 2e-5 * want + 1e-9).all(), (got.double() - want).abs().max()
    return got


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("T", [1, 2, 31, 127, 128, 129, 257, 700])
def test_mass_lengths(T, hd, dtype):
    _check_mass(2, 2, 1, T, hd, dtype, counts=[T, T // 2])
    _check_mass(1, 2, 3, T, hd, dtype)


@gpu
def test_mass_reports_bad_counts():
    q, k = (torch.randn((2, 2, 40, 64), device="cuda", generator=_gen(s)).half() for s in (1, 2))
    lse = _mass_reference(q, k, None)[1]
    for bad in (-1, 41):
        counts = torch.tensor([bad, 40], dtype=torch.int32, device="cuda")
        kvcache.prompt_mass(q, k, lse, counts)
        assert L.device_status(reset=True) == 0x7201
    assert torch.equal(kvcache.prompt_mass(q, k, lse), kvcache.prompt_mass(q, k, lse, torch.full((2,), 40, dtype=torch.int32, device="cuda")))


@gpu
def test_mass_prompts_of_all_lengths():
    _check_mass(7, 2, 2, 400, 64, torch.float16, counts=[0, 400, 1, 128, 129, 0, 256])
    _check_mass(3, 1, 1, 40, 64, torch.float16, counts=[0, 0, 0])
    B = 500  # more prompts than a block has threads
    _check_mass(B, 1, 1, 20, 32, torch.float16, counts=[b % 21 for b in range(B)])
    _check_mass(1, 1, 2, 3000, 128, torch.bfloat16)  # key tiles that several SMs share


@gpu
def test_mass_with_slopes_and_tables():
    slopes = torch.rand((6,), device="cuda", generator=_gen(0)) * 0.3
    for hd in (64, 128):
        _check_mass(2, 3, 2, 600, hd, torch.float16, counts=[600, 333], slopes=slopes)
    for kind in (torch.float16, torch.bfloat16):
        table = generate_alibi_mask(640, 6, dtype=kind)[0]
        _check_mass(2, 6, 1, 600, 64, torch.float16, slopes=-table[:, 1, 0].float(), rounded=kind, bias=table)


@gpu
def test_mass_layouts():
    """Views of a projection's output, one head for all by a stride of zero, rows at odd addresses; equal bits throughout."""
    B, H, T, hd = 2, 3, 200, 64
    qkv = torch.randn((B, T, 3, H, hd), device="cuda", generator=_gen(4)).half()
    q, k = (qkv[:, :, i].permute(0, 2, 1, 3) for i in (0, 1))
    base = _check_mass(B, H, 1, T, hd, torch.float16, q=q, k=k)
    lse = _mass_reference(q, k, None)[1]
    flat = torch.zeros((q.numel() + 8,), device="cuda", dtype=torch.float16)
    for off in (1, 4):
        odd = flat[off:off + q.numel()].view(B, H, T, hd)
        odd.copy_(q)
        assert torch.equal(base, kvcache.prompt_mass(odd, k, lse))
    turned = k.transpose(2, 3).contiguous().transpose(2, 3)
    strided = torch.zeros((B, H, T, 2), device="cuda")
    strided[..., 0] = lse
    assert torch.equal(base, kvcache.prompt_mass(q, turned, strided[..., 0]))
    one = k[:, :1].expand(B, H, T, hd)
    _check_mass(B, H, 1, T, hd, torch.float16, q=q, k=one)
    _check_mass(1, H, 1, T, hd, torch.float16, q=q[:1], k=k[:1])


@gpu
def test_mass_from_the_training_attention():
    """The forward's log-sum-exp: every query spreads a weight of one, so the masses of a prompt add up to its tokens."""
    B, H, T, hd = 2, 4, 320, 64
    q, k, v = (torch.randn((B, H, T, hd), device="cuda", generator=_gen(s)).half() for s in (1, 2, 3))
    out, lse = kvcache.prompt_attention(q, k, v)
    mass = kvcache.prompt_mass(q, k, lse)
    assert (mass.sum(-1) - T).abs().max().item() <= 1e-3 * T
    want, _ = _mass_reference(q, k, None)
    assert ((mass.double() - want).abs() <= 1e-3 * want + 1e-6).all()
    minus = lse.clone()
    minus[:, :, 100:] = -math.inf  # rows without any weight give none
    assert torch.equal(kvcache.prompt_mass(q, k, minus), kvcache.prompt_mass(q, k, lse, torch.full((B,), 100, dtype=torch.int32, device="cuda")))


# ------------------------------------------------------------------------------------------------------------ append


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("page", [1, 7, 64])
def test_append(page, hd, dtype):
    heads, T = 3, 150
    start, counts = [0, 5, 33, 12], [150, 0, 77, 1]
    for stats in (True, False):
        c = Cache(start, heads, hd, page, dtype, room=T)
        want = c.copy()
        qkv = torch.randn((4, T, 3, heads, hd), device="cuda", generator=_gen(1)).to(dtype)
        key, value = (qkv[:, :, i].permute(0, 2, 1, 3) for i in (1, 2))
        key_mass = torch.rand((4, heads, T), device="cuda", generator=_gen(2)) if stats else None
        first = torch.tensor([4, 9, 100, 7], dtype=torch.int32, device="cuda") if stats else None
        kvcache.cache_append(c.k, c.v, c.tables, c.len, key, value, torch.tensor(counts, dtype=torch.int32, device="cuda"),
                             c.mass, c.positions, key_mass, first)
        for b, n in enumerate(counts):
            p, r = want.at(b, start[b] + torch.arange(n, device="cuda"))
            want.k[p, :, r], want.v[p, :, r] = key[b, :, :n].transpose(0, 1), value[b, :, :n].transpose(0, 1)
            want.mass[p, :, r] = key_mass[b, :, :n].T if stats else 0.0
            want.positions[p, :, r] = ((int(first[b]) if stats else start[b]) + torch.arange(n, device="cuda", dtype=torch.int32))[:, None]
        assert L.device_status() == 0
        for a, b in zip((c.k, c.v, c.mass, c.positions), (want.k, want.v, want.mass, want.positions)):
            assert torch.equal(a.nan_to_num(7), b.nan_to_num(7))


@gpu
def test_append_layouts_and_limits():
    c = Cache([3, 0], 2, 64, 16, torch.float16, room=60)
    keys = torch.randn((2, 2, 40, 64), device="cuda", generator=_gen(1)).half()
    kvcache.cache_append(c.k, c.v, c.tables, c.len, keys, -keys)
    for off in (1, 2, 8):  # rows at odd addresses, rows of another order, one head's rows for both
        flat = torch.zeros((keys.numel() + 8,), device="cuda", dtype=torch.float16)
        odd = flat[off:off + keys.numel()].view(keys.shape)
        odd.copy_(keys)
        d = Cache([3, 0], 2, 64, 16, torch.float16, room=60)
        kvcache.cache_append(d.k, d.v, d.tables, d.len, odd, (-keys).transpose(2, 3).contiguous().transpose(2, 3))
        assert torch.equal(c.k.nan_to_num(7), d.k.nan_to_num(7)) and torch.equal(c.v.nan_to_num(7), d.v.nan_to_num(7))
    kvcache.cache_append(c.k, c.v, c.tables, c.len, keys[:, :1].expand(2, 2, 40, 64), keys[:, :1].expand(2, 2, 40, 64))
    p, r = c.at(1, torch.arange(40, device="cuda"))
    assert torch.equal(c.k[p, 1, r], keys[1, 0])
    assert L.device_status() == 0
    # more keys than there is room for: those that fit are written, and it is reported
    room = c.tables.shape[1] * 16
    before = c.k.clone()
    kvcache.cache_append(c.k, c.v, c.tables[1:], torch.tensor([room - 2], dtype=torch.int32, device="cuda"), keys[1:], keys[1:])
    # the second sequence's table is full length only in its used part: its last page may be none
    assert L.device_status(reset=True) in (0x7200, 0x7201)
    kvcache.cache_append(c.k, c.v, c.tables[:1], torch.tensor([-3], dtype=torch.int32, device="cuda"), keys[:1], keys[:1],
                         torch.tensor([0], dtype=torch.int32, device="cuda"))
    assert L.device_status(reset=True) == 0x7201
    assert c.k.shape == before.shape


# ------------------------------------------------------------------------------------------------------------- evict


def _evict_reference(c, keep, recent, nxt, use_positions=True):
    """The source slot of every slot that is left, per sequence and head."""
    maps = []
    for b, n in enumerate(c.lengths):
        p, r = c.at(b, torch.arange(n, device="cuda"))
        oldest = (n if nxt is None else int(nxt[b])) - recent
        per_head = []
        for h in range(c.k.shape[1]):
            mass = c.mass[p, h, r].tolist()
            pos = c.positions[p, h, r].tolist() if use_positions else list(range(n))
            worth = [math.inf if x >= oldest else -math.inf if m != m else m for m, x in zip(mass, pos)]
            best = set(sorted(range(n), key=lambda i: (-worth[i], i))[:keep])
            spare = iter(sorted(i for i in best if i >= keep))
            per_head.append([i if i in best else next(spare) for i in range(min(n, keep))])
        maps.append(per_head)
    return maps


def _check_evict(c, keep, recent, nxt=None, use_positions=True, in_place=True, out=None):
    want_maps = _evict_reference(c, keep, recent, nxt, use_positions)
    old = c.copy()
    pos = c.positions if use_positions else None
    if in_place:
        left = kvcache.cache_evict(c.k, c.v, c.mass, pos, c.tables, c.len, keep, recent, nxt)
        dst = c
    else:
        dst = out
        left = kvcache.cache_evict(c.k, c.v, c.mass, pos, c.tables, c.len, keep, recent, nxt,
                                   out=(dst.k, dst.v, dst.mass, dst.positions if use_positions else None), out_tables=dst.tables)
        for a, b in zip((c.k, c.v, c.mass, c.positions), (old.k, old.v, old.mass, old.positions)):
            assert torch.equal(a.nan_to_num(7), b.nan_to_num(7))
    assert L.device_status() == 0
    assert left.tolist() == [min(n, keep) for n in c.lengths]
    for b, per_head in enumerate(want_maps):
        for h, src in enumerate(per_head):
            p, r = old.at(b, torch.tensor(src, device="cuda", dtype=torch.long))
            p2, r2 = dst.at(b, torch.arange(len(src), device="cuda"))
            for x, y in ((old.k, dst.k), (old.v, dst.v), (old.mass, dst.mass)) + (((old.positions, dst.positions),) if use_positions else ()):
                assert torch.equal(x[p, h, r].nan_to_num(7), y[p2, h, r2].nan_to_num(7)), (b, h)
    return left


@gpu
@pytest.mark.parametrize("hd,dtype", [(32, torch.float16), (64, torch.bfloat16), (128, torch.float16)])
@pytest.mark.parametrize("lengths,keep,recent,page", [([0, 1, 2, 3], 2, 1, 1), ([65, 64, 63, 130], 64, 0, 16), ([300, 1000], 300, 300, 48),
                                                      ([2000, 31, 700], 128, 40, 64), ([5000], 4999, 10, 128), ([33], 1, 0, 7),
                                                      ([100, 40], 200, 50, 32)])
def test_evict(lengths, keep, recent, page, hd, dtype):
    nxt = torch.tensor([3 * n + 1 for n in lengths], dtype=torch.int32, device="cuda")
    _check_evict(Cache(lengths, 3, hd, page, dtype), keep, recent, nxt)
    _check_evict(Cache(lengths, 2, hd, page, dtype), keep, recent, use_positions=False)
    out = Cache([min(n, keep) for n in lengths], 3, hd, 24, dtype, seed=9, room=keep)
    _check_evict(Cache(lengths, 3, hd, page, dtype), keep, recent, nxt, in_place=False, out=out)


@gpu
def test_evict_ties_and_odd_masses():
    """Equal masses, zeros of both signs, negative, infinite and no numbers."""
    values = torch.tensor([0.0, -0.0, 1.0, 1.0, math.inf, -1.0, math.nan, 1e-40, 2.0, 1.0, -math.inf], device="cuda")
    for keep in (1, 7, 100, 255, 256, 257, 399):
        c = Cache([400, 300], 2, 64, 16, torch.float16, seed=keep)
        for b, n in enumerate(c.lengths):
            p, r = c.at(b, torch.arange(n, device="cuda"))
            c.mass[p, :, r] = values[torch.randint(0, 11, (n, 2), device="cuda", generator=_gen(keep))]
        # an infinite mass ties with the recent ones, by the slot
        _check_evict(c, keep, min(keep, 20), torch.tensor([1201, 901], dtype=torch.int32, device="cuda"))
    c = Cache([500], 2, 64, 16, torch.float16)
    c.mass.fill_(0.25)
    _check_evict(c, 200, 0)


@gpu
def test_evict_more_worths_than_fit_shared_memory():
    for in_place in (True, False):
        c = Cache([60000, 51201, 100], 1, 32, 64, torch.float16)
        out = None if in_place else Cache([20000, 20000, 100], 1, 32, 64, torch.float16)
        nxt = torch.tensor([180001, 3 * 51201, 301], dtype=torch.int32, device="cuda")
        _check_evict(c, 20000, 500, nxt, in_place=in_place, out=out)


@gpu
def test_evict_statistics_elsewhere_and_repeated():
    """Keys in place with the statistics in buffers of their own: a second call finds what the first one found."""
    c = Cache([700, 90], 2, 64, 16, torch.float16)
    out = torch.full_like(c.mass, -1.0), torch.full_like(c.positions, -1)
    first = None
    for _ in range(2):
        left = kvcache.cache_evict(c.k, c.v, c.mass, c.positions, c.tables, c.len, 256, 30,
                                   torch.tensor([2101, 271], dtype=torch.int32, device="cuda"), out=(c.k, c.v, *out))
        got = [left, c.k, c.v, *out]
        if first is not None:
            assert all(torch.equal(a.nan_to_num(7), b.nan_to_num(7)) for a, b in zip(first, got))
        first = [x.clone() for x in got]
    d = Cache([700, 90], 2, 64, 16, torch.float16)
    kvcache.cache_evict(d.k, d.v, d.mass, d.positions, d.tables, d.len, 256, 30,
                        torch.tensor([2101, 271], dtype=torch.int32, device="cuda"))
    assert torch.equal(c.k.nan_to_num(7), d.k.nan_to_num(7))
    for b, n in enumerate((256, 90)):
        p, r = d.at(b, torch.arange(n, device="cuda"))
        assert torch.equal(d.mass[p, :, r], out[0][p, :, r]) and torch.equal(d.positions[p, :, r], out[1][p, :, r])


@gpu
def test_evict_reports_bad_tables_and_lengths():
    c = Cache([100, 100], 2, 64, 16, torch.float16)
    tables = c.tables.clone()
    tables[0, 2] = c.pages
    kvcache.cache_evict(c.k, c.v, c.mass, c.positions, tables, c.len, 50, 0)
    assert L.device_status(reset=True) == 0x7200
    c = Cache([100, 100], 2, 64, 16, torch.float16)
    left = kvcache.cache_evict(c.k, c.v, c.mass, c.positions, c.tables, torch.tensor([-1, 100], dtype=torch.int32, device="cuda"), 50, 0)
    assert L.device_status(reset=True) == 0x7201 and left.tolist() == [0, 50]


# ---------------------------------------------------------------------------------------------------------- refusals


@gpu
def test_refusals():
    c = Cache([20, 30], 2, 64, 16, torch.float16)
    q = torch.zeros((2, 4, 64), device="cuda", dtype=torch.float16)
    kv = q[:, :2]
    att = kvcache.paged_attention
    cases = [
        (lambda: att(q.float(), c.k, c.v, c.tables, c.len), "pages' type"),
        (lambda: att(q[:, :3], c.k, c.v, c.tables, c.len), "multiple of the cache's heads"),
        (lambda: att(q[:, :, :32], c.k, c.v, c.tables, c.len), "head_dim"),
        (lambda: att(q, c.k, c.v[:, :1], c.tables, c.len), "one shape"),
        (lambda: att(q, c.k, c.v.transpose(1, 2).contiguous().transpose(1, 2), c.tables, c.len), "same strides"),
        (lambda: att(q, c.k.float(), c.v.float(), c.tables, c.len), "fp16/bf16"),
        (lambda: att(q, c.k, c.v, c.tables.long(), c.len), "int32"),
        (lambda: att(q, c.k, c.v, c.tables[:1], c.len), "tables"),
        (lambda: att(q, c.k, c.v, c.tables, c.len.long()), "lengths"),
        (lambda: att(q, c.k, c.v, c.tables, c.len[:1]), "lengths"),
        (lambda: att(q, c.k, c.v, c.tables, c.len, kv), "comes with a value"),
        (lambda: att(q, c.k, c.v, c.tables, c.len, q, q), "cache heads"),
        (lambda: att(q, c.k, c.v, c.tables, c.len, mass_out=c.mass), "without mass"),
        (lambda: att(q, c.k, c.v, c.tables, c.len, mass=c.mass[:1]), "pages, heads, page"),
        (lambda: att(q, c.k, c.v, c.tables, c.len, mass=c.mass.double()), "fp32"),
        (lambda: att(q, c.k, c.v, c.tables, c.len, attn_bias=torch.zeros(3, device="cuda")), "number of heads"),
        (lambda: att(q, c.k, c.v, c.tables, c.len, attn_bias=torch.randn((4, 64, 64), device="cuda")), "no other bias"),
        (lambda: att(q.cpu(), c.k, c.v, c.tables, c.len), "CUDA"),
        (lambda: att(q.clone().requires_grad_(), c.k, c.v, c.tables, c.len), "no gradients"),
        (lambda: att(q[..., ::2], c.k[..., ::2], c.v[..., ::2], c.tables, c.len), "unit stride"),
        (lambda: kvcache.cache_append(c.k, c.v, c.tables, c.len, q[:, :, None], q[:, :, None]), "cache heads"),
        (lambda: kvcache.cache_append(c.k, c.v, c.tables, c.len, kv[:, :, None], kv[:, :, None],
                                      key_mass=torch.zeros((2, 2, 1), device="cuda")), "has none"),
        (lambda: kvcache.cache_append(c.k, c.v, c.tables, c.len, kv[:, :, None].float(), kv[:, :, None].float()), "pages' type"),
        (lambda: kvcache.prompt_mass(q[:, :, None], kv[:, :, None], torch.zeros((2, 4, 2), device="cuda")), "log-sum-exp"),
        (lambda: kvcache.prompt_mass(q[:, :3, None], kv[:, :, None], torch.zeros((2, 3, 1), device="cuda")), "multiple of the key heads"),
        (lambda: kvcache.prompt_mass(q[:, :, None, :48], kv[:, :, None, :48], torch.zeros((2, 4, 1), device="cuda")), "head_dims"),
        (lambda: kvcache.cache_evict(c.k, c.v, None, None, c.tables, c.len, 4), "no masses"),
        (lambda: kvcache.cache_evict(c.k, c.v, c.mass, None, c.tables, c.len, 0), "keep"),
        (lambda: kvcache.cache_evict(c.k, c.v, c.mass, None, c.tables, c.len, 4, 5), "recent"),
        (lambda: kvcache.cache_evict(c.k, c.v, c.mass, None, c.tables, c.len, 4, out_tables=c.tables.clone()), "pages of their own"),
        (lambda: kvcache.cache_evict(c.k, c.v, c.mass, None, c.tables, c.len, 4, out=(c.k.clone(), c.v, c.mass, None)), "in place"),
        (lambda: kvcache.cache_evict(c.k, c.v, c.mass, c.positions, c.tables, c.len, 4,
                                     out=(c.k.clone(), c.v.clone(), c.mass.clone(), c.positions)), "positions not"),
        (lambda: kvcache.cache_evict(c.k, c.v, c.mass, None, c.tables, c.len, 20, out=(c.k.clone(), c.v.clone(), c.mass.clone(), None),
                                     out_tables=c.tables[:, :1].contiguous()), "room for"),
    ]
    before = [x.clone() for x in (c.k, c.v, c.mass, c.positions)]
    for i, (call, message) in enumerate(cases):
        with pytest.raises(AssertionError, match=message):
            call()
            raise RuntimeError("case %d was accepted" % i)
    assert all(torch.equal(a.nan_to_num(7), b.nan_to_num(7)) for a, b in zip(before, (c.k, c.v, c.mass, c.positions)))
    empty = torch.zeros((0, 4, 64), device="cuda", dtype=torch.float16)
    assert att(empty, c.k, c.v, c.tables[:0], c.len[:0]).shape == (0, 4, 64)
    assert kvcache.prompt_mass(q[:, :, None][:, :, :0], kv[:, :, None][:, :, :0], torch.zeros((2, 4, 0), device="cuda")).shape == (2, 2, 0)


def _strides(*s):
    return (ctypes.c_int64 * len(s))(*s)


def test_argument_checks_without_device():
    pg, two, three, one = _strides(2048, 1024, 64), _strides(128, 64), _strides(4096, 2048, 64), ctypes.c_void_p(256)

    def attention(hd=64, group=1, pages=4, page=16, width=2, ld=2, k_new=None, mass=None, mass_out=None, scratch=None, nbytes=0,
                  dtype=0, strides=pg, k_pages=one, workspace=None, wbytes=0):
        return L.lib.tfb_paged_attention(one, k_new, None, one, k_pages, one, one, one, None, None, mass, mass_out, None, 0, 2, 2, group,
                                         hd, pages, page, width, ld, strides, two, two, two, two, workspace, wbytes, scratch, nbytes,
                                         dtype, None)

    def said(rc, code, text):
        assert rc == code and text in L.lib.tfb_last_error(), (rc, L.lib.tfb_last_error())

    said(attention(hd=48), -2, b"head_dims")
    said(attention(dtype=2), -1, b"fp16 or bf16")
    said(attention(group=129), -1, b"query heads")
    said(attention(page=0), -1, b"page")
    said(attention(width=2 ** 29), -1, b"2^30 slots")
    said(attention(ld=1), -1, b"overlap")
    said(attention(strides=_strides(2048, 1024, 63)), -1, b"16-byte")
    said(attention(k_pages=ctypes.c_void_p(260)), -1, b"16-byte")
    said(attention(k_new=one), -1, b"without a value")
    said(attention(mass_out=one), -1, b"come together")
    said(attention(), -1, b"workspace")
    said(attention(workspace=one, wbytes=16), -1, b"workspace")
    said(attention(mass=one, mass_out=one, workspace=one, wbytes=1 << 30, scratch=one, nbytes=16), -1, b"scratch")
    assert L.lib.tfb_paged_attention_scratch_bytes(2, 2, 1, 32) == 256 + 2 * 2 * 32 * 4
    said(L.lib.tfb_cache_append(one, one, one, one, one, one, None, None, None, None, one, 1, 2, 5, 64, 4, 16, 2, 2, pg, three, three,
                                two, 0, None), -1, b"masses")
    assert L.lib.tfb_cache_append(one, one, one, one, one, one, None, None, None, None, None, 1, 2, 0, 64, 4, 16, 2, 2, pg, three, three,
                                  two, 0, None) == 0  # no keys
    said(L.lib.tfb_prompt_mass(one, one, one, None, None, 0, one, 1, 2, 1, 8, 64, _strides(0, 64, 64), three, two, one, 1 << 30, 0, None),
         -1, b"positive multiples")
    said(L.lib.tfb_prompt_mass(one, one, one, None, None, 0, one, 1, 2, 1, 8, 64, three, three, two, None, 0, 0, None), -1, b"workspace")
    assert L.lib.tfb_prompt_mass(one, one, one, None, None, 0, one, 1, 2, 1, 0, 64, three, three, two, None, 0, 0, None) == 0

    def evict(keep=4, recent=0, k_out=one, out_tables=one, mass_out=one, out_width=2, nbytes=1 << 20):
        return L.lib.tfb_cache_evict(one, one, one, None, one, one, None, k_out, k_out, mass_out, None, out_tables, two, 1, 2, 64, keep,
                                     recent, 16, 4, 2, 2, pg, 16, 4, out_width, 2, pg, one, nbytes, 0, None)

    other = ctypes.c_void_p(1 << 20)
    rc = L.lib.tfb_cache_evict(one, one, one, None, one, one, None, one, one, one, None, one, one, 1, 2, 64, 4, 0, 16, 4, 2, 2, pg, 16, 4,
                               2, 2, pg, one, 1 << 20, 0, None)
    said(rc, -1, b"array of their own")
    said(evict(keep=0), -1, b"at least 1")
    said(evict(recent=5), -1, b"0 to keep")
    said(evict(out_tables=other), -1, b"pages of their own")
    said(evict(mass_out=None), -1, b"no masses")
    said(evict(keep=20, k_out=other, mass_out=other, out_tables=other, out_width=1), -1, b"room for")
    said(evict(nbytes=8), -1, b"scratch")
