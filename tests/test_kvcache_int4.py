"""The paged key-value cache in 4 bits: attention and append against their definitions in 64 bits.

Tolerances.  u is the rounding of the 16-bit type (2^-11, 2^-8): an output o = sum w v is rounded once, u |o|.  The weights enter the second
product in two parts of bf16, 2^-17 of each, and scores of up to some 20 (in log2 units) carry an absolute error of some 1e-6 from 32-bit sums:
2e-5 sum w |v| bounds both.  What is stored, and what a stored value stands for, is equal."""
import ctypes
import math

import pytest
import torch

import tritonformer_b200._lib as L
from tritonformer_b200 import PagedKVCache, cache_append, cache_evict, kvcache, paged_attention
from tritonformer_b200.transformer import generate_alibi_mask

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
gpu = pytest.mark.gpu
LARGEST = {torch.float16: 9352.0, torch.bfloat16: 36.25 * 2.0 ** 120}  # the scales whose sevenfold is not above the largest value


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(*shape, seed, dtype, scale=1.0):
    return (scale * torch.randn(shape, generator=_gen(seed), device="cuda")).to(dtype)


def _quantized(x):
    """(codes, scales) of the rows of x in 64 bits."""
    top = x.double().abs().amax(-1, keepdim=True)
    scales = torch.where(top.isfinite(), top / 7, math.nan).to(x.dtype).double().clamp(max=LARGEST[x.dtype])
    return torch.where(scales > 0, x.double() / scales, 0.0).round().clamp(-7, 7), scales[..., 0]


def _pack(codes):
    """Bytes of rows: dim 8 w + 2 n + e at bits 4 n + 16 e of the word w."""
    c = (codes + 8).long().unflatten(-1, (codes.shape[-1] // 8, 8))
    words = sum(c[..., d] << (4 * (d // 2) + 16 * (d % 2)) for d in range(8))
    return torch.stack([words >> 8 * i & 255 for i in range(4)], -1).to(torch.uint8).flatten(-2)


def _unpack(rows):
    b = rows.long().unflatten(-1, (rows.shape[-1] // 4, 4))
    words = sum(b[..., i] << 8 * i for i in range(4))
    return torch.stack([(words >> (4 * (d // 2) + 16 * (d % 2)) & 15) - 8 for d in range(8)], -1).flatten(-2).double()


class Cache:
    """A pool with the pages of `lengths` (plus `room`) keys dealt out in random order; what no slot in use holds has a scale of NaN."""

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
        self.k, self.v = (torch.randint(0, 256, (*shape, hd // 2), generator=g, device="cuda", dtype=torch.uint8) for _ in range(2))
        self.scales = torch.full((*shape, 2), math.nan, device="cuda", dtype=dtype)
        for b, n in enumerate(lengths):
            p, r = self.at(b, torch.arange(n, device="cuda"))
            for i, pages in enumerate((self.k, self.v)):
                codes, scales = _quantized(torch.randn((n, heads, hd), generator=g, device="cuda").to(dtype))
                pages[p, :, r], self.scales[p, :, r, i] = _pack(codes), scales.to(dtype)
        self.len = torch.tensor(lengths, dtype=torch.int32, device="cuda")

    def at(self, b, slots):
        return self.tables[b].long()[slots // self.page], slots % self.page

    def copy(self):
        other = Cache.__new__(Cache)
        other.__dict__.update({k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in self.__dict__.items()})
        return other

    def same(self, other):
        return (torch.equal(self.k, other.k) and torch.equal(self.v, other.v)
                and torch.equal(self.scales.nan_to_num(7), other.scales.nan_to_num(7)))

    def rows(self, b, n, head):
        """Keys and values of a sequence's first n slots, in 64 bits."""
        p, r = self.at(b, torch.arange(n, device="cuda"))
        scales = self.scales[p, head, r].double()
        return _unpack(self.k[p, head, r]) * scales[:, :1], _unpack(self.v[p, head, r]) * scales[:, 1:]

    def write(self, b, slot, key, value):
        p, r = self.at(b, torch.tensor(slot, device="cuda"))
        for i, (pages, x) in enumerate(((self.k, key), (self.v, value))):
            codes, scales = _quantized(x)
            pages[p, :, r], self.scales[p, :, r, i] = _pack(codes), scales.to(x.dtype)


def _reference(q, c, new=None, slopes=None, rounded=None):
    """(outputs, their bounds) in 64 bits; writes the new rows into c."""
    B, heads, hd = q.shape
    group = heads // c.k.shape[1]
    out = torch.zeros((B, heads, hd), device="cuda", dtype=torch.double)
    bound = torch.full_like(out, 1e-7)
    for b in range(B):
        n = c.lengths[b]
        if new:
            c.write(b, n, new[0][b], new[1][b])
            n += 1
        if n == 0:
            continue
        for h in range(heads):
            k, v = c.rows(b, n, h // group)
            s = k @ q[b, h].double() / math.sqrt(hd)
            if slopes is not None:
                back = n - 1 - torch.arange(n, device="cuda")
                s = s - (back.double() * slopes[h].double() if rounded is None else (back.to(rounded) * slopes[h].to(rounded)).double())
            w = torch.softmax(s, 0)
            out[b, h] = w @ v
            bound[b, h] += U[q.dtype] * out[b, h].abs() + 2e-5 * (w @ v.abs())
    return out, bound


def _check_attention(lengths, heads, group, hd, page, dtype, new=True, alibi=False, seed=0, q_scale=2.0):
    c = Cache(lengths, heads, hd, page, dtype, seed)
    B = len(lengths)
    q = _randn(B, heads * group, hd, seed=seed + 1, dtype=dtype, scale=q_scale)
    kv = [_randn(B, heads, hd, seed=seed + s, dtype=dtype) for s in (2, 3)] if new else None
    slopes = 0.3 * torch.rand((heads * group,), generator=_gen(seed + 4), device="cuda") if alibi else None
    want = c.copy()
    ref, bound = _reference(q, want, kv, slopes)
    out = paged_attention(q, c.k, c.v, c.tables, c.len, *(kv or (None, None)), attn_bias=slopes, scales=c.scales)
    assert L.device_status() == 0
    if B:
        excess = ((out.double() - ref).abs() - bound).max().item()
        assert excess <= 0, excess
    assert c.same(want)
    return out


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("lengths,page", [([0], 16), ([1], 1), ([5, 0, 17], 7), ([63, 64, 65, 31, 32, 33], 48), ([300, 2], 64),
                                          ([2500], 128), ([15, 16, 4000, 1], 16)])
def test_attention_lengths_and_pages(lengths, page, hd, dtype):
    _check_attention(lengths, 2, 1, hd, page, dtype)
    _check_attention(lengths, 2, 1, hd, page, dtype, new=False, alibi=True, seed=5)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,group", [(1, 1), (3, 2), (2, 7), (2, 8), (1, 9), (2, 16), (1, 17), (1, 40), (1, 128), (12, 1)])
def test_attention_head_layouts(heads, group, dtype):
    for hd in (32, 64, 128):
        _check_attention([129, 40, 700], heads, group, hd, 32, dtype, alibi=hd != 64)


@gpu
def test_attention_many_sequences_and_long_ones():
    g = torch.Generator().manual_seed(3)
    lengths = [int(n) for n in torch.randint(0, 40, (600,), generator=g) * (torch.rand((600,), generator=g) < 0.4)]
    _check_attention(lengths, 2, 1, 64, 16, torch.float16, new=False)
    _check_attention(lengths, 1, 2, 32, 16, torch.float16)
    _check_attention([0] * 5, 1, 2, 32, 16, torch.float16, new=False)
    _check_attention([70001], 1, 3, 128, 64, torch.bfloat16)
    _check_attention([3, 90000, 1, 257, 0], 2, 1, 64, 256, torch.float16, alibi=True)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_special_values(dtype):
    """Large scores, rows of zeros, a new row that is not finite: NaN, in its own sequence."""
    _check_attention([400, 3], 2, 2, 64, 16, dtype, q_scale=60.0)
    c = Cache([50, 20, 33], 2, 64, 16, dtype)
    q = _randn(3, 4, 64, seed=1, dtype=dtype)
    key, value = _randn(3, 2, 64, seed=2, dtype=dtype), _randn(3, 2, 64, seed=3, dtype=dtype)
    key[0], value[0], value[1, 1, 5], key[2, 0, 9] = 0.0, 0.0, math.inf, math.nan
    want = c.copy()
    ref, bound = _reference(q, want, (key, value))
    out = paged_attention(q, c.k, c.v, c.tables, c.len, key, value, scales=c.scales)
    assert c.same(want)
    clean = [(0, slice(0, 4)), (1, slice(0, 2)), (2, slice(2, 4))]
    for b, h in clean:
        assert ((out[b, h].double() - ref[b, h]).abs() <= bound[b, h]).all()
    assert out[1, 2:].isnan().all() and out[2, :2].isnan().all() and ref[1, 2:].isnan().all()
    again = paged_attention(q, c.k, c.v, c.tables, c.len + 1, scales=c.scales)  # the new row from its page
    assert torch.equal(out.nan_to_num(7), again.nan_to_num(7))


@gpu
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16])
def test_attention_with_the_models_table(kind):
    heads, hd = 6, 64
    table = generate_alibi_mask(1024, heads, dtype=kind)[0]
    c = Cache([900, 33], heads, hd, 64, torch.float16)
    q, new = _randn(2, heads, hd, seed=2, dtype=torch.float16), [_randn(2, heads, hd, seed=s, dtype=torch.float16) for s in (3, 4)]
    ref, bound = _reference(q, c.copy(), new, -table[:, 1, 0].float(), kind)
    out = paged_attention(q, c.k, c.v, c.tables, c.len, *new, attn_bias=table, scales=c.scales)
    assert ((out.double() - ref).abs() <= bound).all()


@gpu
def test_attention_strides_alignment_streams_and_graphs():
    B, heads, hd, page = 2, 3, 64, 16
    c = Cache([50, 21], heads, hd, page, torch.float16)
    pool = torch.full((c.pages, 4, 2, page, heads, hd // 2), 17, device="cuda", dtype=torch.uint8)
    k, v = (pool[:, 1, i].permute(0, 2, 1, 3) for i in (0, 1))  # (pages, heads, page, hd / 2), heads inside the slots
    k.copy_(c.k)
    v.copy_(c.v)
    for off in (0, 1, 2, 8):
        flat = _randn(B * 9 * hd * heads + 64, seed=off, dtype=torch.float16)
        qkv = flat[off:off + B * 9 * hd * heads].view(B, 9 * heads, hd)
        q, kn, vn = qkv[:, 0:heads], qkv[:, heads:2 * heads], qkv[:, 4 * heads:7 * heads:3]
        ref, bound = _reference(q, c.copy(), (kn, vn))
        out = paged_attention(q, k, v, c.tables, c.len, kn, vn, scales=c.scales)
        assert ((out.double() - ref).abs() <= bound).all(), off
        transposed = q.transpose(1, 2).contiguous().transpose(1, 2)
        assert torch.equal(out, paged_attention(transposed, k, v, c.tables, c.len, kn, vn, scales=c.scales))
    assert (pool[:, [0, 2, 3]] == 17).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(out, paged_attention(q, k, v, c.tables, c.len, kn, vn, scales=c.scales))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache_append(c.k, c.v, c.tables, c.len, kn[:, :, None], vn[:, :, None], scales=c.scales)
        got = paged_attention(q, c.k, c.v, c.tables, c.len, scales=c.scales)
    c.len.copy_(torch.tensor([7, 0]))  # read where they lie
    graph.replay()
    assert torch.equal(got, paged_attention(q, c.k, c.v, c.tables, c.len, scales=c.scales)) and (got[1] == 0).all()


@gpu
def test_offsets_beyond_32_bits():
    page, heads, hd = 256, 2, 128
    pages = 2 ** 32 // (page * heads * hd // 2) + 5
    k = torch.zeros((pages, heads, page, hd // 2), device="cuda", dtype=torch.uint8)
    v = torch.zeros_like(k)
    scales = torch.zeros((pages, heads, page, 2), device="cuda", dtype=torch.float16)
    small = Cache([600], heads, hd, page, torch.float16)
    ids = torch.tensor([pages - 1, pages - 4, pages - 2, pages - 3], device="cuda")[: small.tables.shape[1]]
    at = small.tables[0].long()
    k[ids], v[ids], scales[ids] = small.k[at], small.v[at], small.scales[at]
    q, new = _randn(1, 2, hd, seed=0, dtype=torch.float16), [_randn(1, 2, hd, seed=s, dtype=torch.float16) for s in (3, 4)]
    want = paged_attention(q, small.k, small.v, small.tables, small.len, *new, scales=small.scales)
    assert torch.equal(want, paged_attention(q, k, v, ids[None].to(torch.int32), small.len, *new, scales=scales))
    assert torch.equal(k[ids], small.k[at]) and torch.equal(scales[ids].nan_to_num(7), small.scales[at].nan_to_num(7))
    keys = _randn(1, heads, 5, hd, seed=9, dtype=torch.float16)
    cache_append(k, v, ids[None].to(torch.int32), small.len, keys, keys, scales=scales)
    assert torch.equal(k[ids[600 // page], :, 600 % page:600 % page + 5], _pack(_quantized(keys[0])[0]))


@gpu
def test_bad_tables_and_lengths_are_reported():
    c = Cache([40, 40, 40], 2, 64, 16, torch.float16)
    q = _randn(3, 2, 64, seed=1, dtype=torch.float16)
    want, before = paged_attention(q, c.k, c.v, c.tables, c.len, scales=c.scales), c.copy()
    for bad in (-1, c.pages, 2 ** 31 - 1):
        tables = c.tables.clone()
        tables[1, 1] = bad
        out = paged_attention(q, c.k, c.v, tables, c.len, scales=c.scales)
        assert L.device_status(reset=True) == 0x7200
        assert torch.equal(out[[0, 2]], want[[0, 2]]) and out[1].isfinite().all()
        tables = c.tables.clone()
        tables[1, 2] = bad
        cache_append(c.k, c.v, tables, torch.where(torch.arange(3, device="cuda") == 1, c.len, c.tables.shape[1] * 16).int(),
                     q[:, :, None], q[:, :, None], torch.tensor([0, 1, 0], device="cuda", dtype=torch.int32), scales=c.scales)
        assert L.device_status(reset=True) == 0x7200
    room = c.tables.shape[1] * 16
    for n in (-5, room, 2 ** 31 - 1):
        lengths = c.len.clone()
        lengths[1] = n
        other = c.copy()
        other.scales.nan_to_num_(0)
        assert paged_attention(q, other.k, other.v, c.tables, lengths, q, q, scales=other.scales).isfinite().all()
        assert L.device_status(reset=True) == 0x7201
        if n > 0:
            cache_append(c.k, c.v, c.tables, torch.where(torch.arange(3, device="cuda") == 1, lengths, room).int(), q[:, :, None],
                         q[:, :, None], torch.tensor([0, 1, 0], device="cuda", dtype=torch.int32), scales=c.scales)
            assert L.device_status(reset=True) == 0x7201
    assert c.same(before)


def _check_append(lengths, counts, T, heads, hd, page, dtype, k=None, v=None, seed=0):
    B = len(lengths)
    c = Cache(lengths, heads, hd, page, dtype, seed, room=max(counts + [1]))
    k = _randn(B, heads, T, hd, seed=seed + 1, dtype=dtype) if k is None else k
    v = _randn(B, heads, T, hd, seed=seed + 2, dtype=dtype, scale=3.0) if v is None else v
    want, also = c.copy(), c.copy()
    stored = [torch.zeros((B, heads, T, hd), device="cuda", dtype=torch.double) for _ in range(2)]
    for b, n in enumerate(counts):
        for x, y in zip((k, v), stored):
            codes, scales = _quantized(x[b, :, :n])
            y[b, :, :n] = codes * scales[..., None]
        for t in range(n):
            want.write(b, lengths[b] + t, k[b, :, t], v[b, :, t])
    count = torch.tensor(counts, dtype=torch.int32, device="cuda") if counts != [T] * B else None
    got = cache_append(c.k, c.v, c.tables, c.len, k, v, count, scales=c.scales, stored=True)
    assert cache_append(also.k, also.v, also.tables, also.len, k, v, count, scales=also.scales) is None
    assert L.device_status() == 0 and c.same(want) and also.same(want)
    for x, y in zip(got, stored):
        assert x.dtype is dtype and x.shape == y.shape and torch.equal(x.nan_to_num(7), y.to(dtype).nan_to_num(7))


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("lengths,counts,T,page", [([0], [1], 1, 16), ([0, 5, 31], [20, 0, 7], 20, 7), ([10, 0], [130, 130], 130, 48),
                                                   ([63, 1], [1, 1], 1, 64), ([3], [65], 70, 1)])
def test_append(lengths, counts, T, page, hd, dtype):
    _check_append(lengths, counts, T, 3, hd, page, dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_special_values_and_strides(dtype):
    k, v = _randn(2, 2, 9, 64, seed=1, dtype=dtype), _randn(2, 2, 9, 64, seed=2, dtype=dtype)
    k[0, 0, 0], v[0, 1, 3, 7], v[1, 0, 2, 0], k[1, 1, 4] = 0.0, math.inf, math.nan, torch.finfo(dtype).max
    k[1, 0, 5] = torch.finfo(dtype).smallest_normal / 64  # scales below what the type holds, or only just
    v[1, 1, 6] *= torch.finfo(dtype).smallest_normal
    _check_append([4, 0], [9, 8], 9, 2, 64, 16, dtype, k, v)
    qkv = _randn(2, 9, 3 * 2 * 64 + 1, seed=3, dtype=dtype)
    for off in (0, 1):
        x = qkv[:, :, off:off + 384].reshape(2, 9, 3, 2, 64) if off == 0 else qkv[:, :, 1:].unflatten(2, (3, 2, 64))
        _check_append([4, 0], [9, 8], 9, 2, 64, 16, dtype, x[:, :, 1].transpose(1, 2), x[:, :, 2].transpose(1, 2))
    _check_append([4, 0], [9, 8], 9, 2, 64, 16, dtype, k.transpose(2, 3).contiguous().transpose(2, 3), v[:, :1].expand(2, 2, 9, 64))


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_run_of_the_operators(dtype):
    """A prompt, then tokens one by one, on the class: every step's output is that of the rows that a prompt of all of them stores."""
    heads, group, hd, n, more = 2, 2, 64, 37, 30
    k, v = _randn(1, heads, n + more, hd, seed=1, dtype=dtype), _randn(1, heads, n + more, hd, seed=2, dtype=dtype)
    q = _randn(more, heads * group, hd, seed=3, dtype=dtype, scale=2.0)
    cache, whole = (PagedKVCache(8, heads, hd, 16, dtype, statistics=False, bits=4) for _ in range(2))
    tables = torch.tensor([[3, 0, 7, 1, 5]], device="cuda", dtype=torch.int32)
    length = torch.zeros(1, device="cuda", dtype=torch.int32)
    all_k, all_v = whole.append(tables, length, k, v, stored=True)
    cache.append(tables, length, k[:, :, :n], v[:, :, :n])
    for t in range(more):
        out = cache.attend(q[t:t + 1], tables, length + n + t, k[:, :, n + t], v[:, :, n + t])
        for h in range(heads * group):
            kk, vv = all_k[0, h // group, : n + t + 1].double(), all_v[0, h // group, : n + t + 1].double()
            w = torch.softmax(kk @ q[t, h].double() / math.sqrt(hd), 0)
            # the stored rows are rounded to the type once more, in the scores too: by u sum |q| |k| / sqrt(hd) each
            shift = U[dtype] * (kk.abs() @ q[t, h].double().abs()).max() / math.sqrt(hd)
            assert ((out[0, h].double() - w @ vv).abs() <= 2 * (U[dtype] + shift) * (w @ vv.abs()) + 1e-5).all()
    assert torch.equal(cache.k, whole.k) and torch.equal(cache.v, whole.v) and torch.equal(cache.scales, whole.scales)


@gpu
def test_refusals():
    c = Cache([5], 2, 64, 16, torch.float16)
    q, kv = _randn(1, 2, 64, seed=1, dtype=torch.float16), _randn(1, 2, 3, 64, seed=2, dtype=torch.float16)
    mass, at = torch.zeros((c.pages, 2, 16), device="cuda"), torch.zeros((1,), device="cuda", dtype=torch.int32)
    attend = lambda q=q, k=c.k, v=c.v, scales=c.scales, **more: paged_attention(q, k, v, c.tables, c.len, scales=scales, **more)  # noqa: E731
    append = lambda k=kv, v=kv, **more: cache_append(c.k, c.v, c.tables, c.len, k, v, scales=c.scales, **more)  # noqa: E731
    for call, text in ((lambda: attend(mass=mass), "no masses"), (lambda: attend(query_positions=at), "no masses"),
                       (lambda: append(mass=mass), "no masses"), (lambda: append(first_positions=at), "no masses"),
                       (lambda: attend(q=q.bfloat16()), "scales' type"), (lambda: attend(q=q[:, :, :32]), "head_dim"),
                       (lambda: attend(k=c.k.to(torch.int8)), "uint8"), (lambda: attend(scales=c.scales[..., :1]), "scales"),
                       (lambda: attend(scales=c.scales.float()), "scales"), (lambda: attend(key=q), "comes with a value"),
                       (lambda: attend(key=q.bfloat16(), value=q.bfloat16()), "scales' type"), (lambda: append(k=kv.bfloat16(), v=kv.bfloat16()), "scales' type"),
                       (lambda: attend(k=c.k[..., :24], v=c.v[..., :24]), "head_dims"), (lambda: append(v=kv[:, :1]), "keys and values"),
                       (lambda: paged_attention(q, c.k, c.v, c.tables, c.len), "fp16/bf16"),
                       (lambda: attend(q=q.clone().requires_grad_()), "no gradients"),
                       (lambda: cache_append(kv, kv, c.tables, c.len, kv, kv, stored=True), "16 bits"),
                       (lambda: PagedKVCache(4, 2, 64, bits=4), "no masses"), (lambda: PagedKVCache(4, 2, 64, statistics=False, bits=8), "16 or 4"),
                       (lambda: PagedKVCache(4, 2, 64, statistics=False, bits=4).evict(c.tables, c.len, 3), "no masses"),
                       (lambda: cache_evict(c.k, c.v, mass, None, c.tables, c.len, 3), "fp16/bf16")):
        with pytest.raises(AssertionError, match=text):
            call()


def test_refusals_without_a_device():
    one = ctypes.c_void_p(16)  # never dereferenced
    s3, s2 = (ctypes.c_int64 * 3)(1024, 512, 32), (ctypes.c_int64 * 2)(128, 64)
    odd = (ctypes.c_int64 * 3)(1024, 512, 40)
    wide = (ctypes.c_int64 * 3)(64, 64, 64)

    def attend(hd=64, group=1, strides=s3, dtype=0, scales=one, B=1):
        return L.lib.tfb_paged_attention_int4(one, None, None, one, one, one, scales, one, one, None, 0, B, 2, group, hd, 4, 16, 2, 2, strides,
                                              s2, s2, s2, s2, None, 0, dtype, None)

    def append(hd=64, T=1, strides=s3, stored=None, B=1):
        return L.lib.tfb_cache_append_int4(one, one, one, one, one, one, one, None, stored, None, B, 2, T, hd, 4, 16, 2, 2, strides, wide,
                                           wide, wide, 0, None)

    for call, text in ((lambda: attend(hd=48), b"head_dims"), (lambda: attend(group=129), b"query heads"), (lambda: attend(strides=odd), b"aligned"),
                       (lambda: attend(dtype=2), b"dtype"), (lambda: attend(scales=ctypes.c_void_p(2)), b"4-byte"), (attend, b"workspace"),
                       (lambda: append(hd=16), b"head_dims"), (lambda: append(strides=odd), b"aligned"), (lambda: append(T=1 << 23), b"more than"),
                       (lambda: append(stored=one), b"stored keys without")):
        assert call() < 0 and text in L.lib.tfb_last_error(), L.lib.tfb_last_error()
    assert attend(B=0) == 0 and append(B=0) == 0 and append(T=0) == 0
    with pytest.raises(AssertionError, match="CUDA"):
        kvcache.cache_append(torch.zeros((1, 1, 16, 32), dtype=torch.uint8), torch.zeros((1, 1, 16, 32), dtype=torch.uint8),
                             torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros((1, 1, 1, 64)).half(),
                             torch.zeros((1, 1, 1, 64)).half(), scales=torch.zeros((1, 1, 16, 2)).half())
