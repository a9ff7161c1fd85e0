"""Weights in 4 bits and products with them against their definitions.

Tolerances.  u is the rounding of the 16-bit type (2^-11, 2^-8): the output is rounded once, u |y|.  With S = sum |x| |w| + |bias| + |addend|, the
sums: an mma adds 16 exact products to its accumulator within 2^-22 of the largest addend each, K / 16 of them in a chain at most, then the groups'
scales, the warps and the epilogue, some 32 roundings of 2^-24: (K / 16 + 32) 2^-22 S bounds both.  Above 64 rows the weights are
rounded to the type before the product: u S more."""
import ctypes

import pytest
import torch

import tritonformer_b200._lib as L
from tritonformer_b200 import Int4Weight, int4, linear_int4, quantize_int4

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LARGEST = {torch.float16: 9352.0, torch.bfloat16: 36.25 * 2.0 ** 120}  # the scales whose sevenfold is not above the largest value
gpu = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(*shape, seed, dtype, scale=1.0):
    return (scale * torch.randn(shape, generator=_gen(seed), device="cuda")).to(dtype)


def _definition(w, group):
    """(codes, scales) of (K, N) in 64 bits, the scales repeated along the rows."""
    k, n = w.shape
    groups = -(-k // group)
    padded = torch.zeros((groups * group, n), dtype=torch.float64, device=w.device)
    padded[:k] = w.double()
    blocks = padded.view(groups, group, n)
    top = blocks.abs().amax(1)
    scales = torch.where(top.isfinite(), top / 7, torch.nan).to(w.dtype).double().clamp(max=LARGEST[w.dtype])
    codes = torch.where(scales[:, None] > 0, blocks / scales[:, None], 0.0).round().clamp(-7, 7)
    return codes.view(-1, n)[:k], scales.repeat_interleave(group, 0)[:k]


def _unpacked(q):
    """(codes, scales) as the header says they lie, (K, N) each."""
    strips, units = q.codes.shape[:2]
    codes = torch.empty((units * 64, strips * 16), dtype=torch.float64)
    scales = torch.empty_like(codes)
    words, packed = q.codes.cpu().long() & 0xffffffff, q.scales.cpu().double()
    for unit in range(units):
        for lane in range(32):
            r, j = lane // 4, lane % 4
            for t in range(4):
                for p in range(2):
                    for e in range(2):
                        row = unit * 64 + 32 * (t // 2) + 8 * j + 4 * (t % 2) + 2 * p + e
                        for c in range(2):
                            bits = words[:, unit, lane, t] >> (4 * (c + 2 * p) + 16 * e) & 15
                            codes[row, r + 8 * c::16] = (bits - 8).double()
                            scales[row, r + 8 * c::16] = packed[:, row // q.group, r, c]
    return codes, scales


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("k,n,columns_first", [(1, 1, False), (64, 16, False), (65, 17, True), (200, 70, False), (129, 33, True)])
def test_quantize_is_its_definition(k, n, columns_first, group, dtype):
    w = _randn(k, n, seed=k, dtype=dtype, scale=0.05)
    if columns_first:
        w = w.t().contiguous().t()
    q = quantize_int4(w, group)
    want, want_scales = _definition(w, group)
    codes, scales = _unpacked(q)
    assert torch.equal(codes[:k, :n], want.cpu()) and torch.equal(scales[:k, :n], want_scales.cpu())
    assert not codes[k:].any() and not codes[:, n:].any() and not scales[:, n:].any()
    back = q.dequantize()
    assert back.shape == w.shape and torch.equal(back, (want * want_scales).to(dtype))
    assert (back.double() - w.double()).abs().max() <= (0.5 + 1e-2) * want_scales.max()


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_quantize_of_zeros_infinities_and_tiny_weights(dtype):
    w = _randn(128, 40, seed=1, dtype=dtype)
    w[:64, 3] = 0.0
    w[70, 5] = float("inf")
    w[0, 6] = float("nan")
    w[64:, 7] = torch.finfo(dtype).smallest_normal / 2 ** 6
    q = quantize_int4(w, 64)
    want, scales = _definition(w, 64)
    back = q.dequantize()
    assert torch.equal(back.nan_to_num(9.0), (want * scales).nan_to_num(9.0).to(dtype))
    assert back[64:, 5].isnan().all() and back[:64, 6].isnan().all() and back.isnan().sum() == 128 and not back[:64, 3].any()
    x = torch.ones((1, 128), device="cuda", dtype=dtype)
    assert linear_int4(x, q).isnan().nonzero()[:, 1].tolist() == [5, 6]


def _check_linear(m, k, n, group, dtype, bias=False, relu=False, addend=False, x=None, seed=0):
    w = _randn(k, n, seed=seed, dtype=dtype, scale=0.1)
    x = _randn(m, k, seed=seed + 1, dtype=dtype) if x is None else x
    b = _randn(n, seed=seed + 2, dtype=dtype) if bias else None
    a = _randn(*x.shape[:-1], n, seed=seed + 3, dtype=dtype) if addend else None
    q = quantize_int4(w, group)
    codes, scales = _definition(w, group)
    full, rows = codes * scales, x.reshape(-1, k).double()
    y, s = rows @ full, rows.abs() @ full.abs()
    if bias:
        y, s = y + b.double(), s + b.double().abs()
    if relu:
        y = y.clamp(min=0)
    if addend:
        y, s = y + a.reshape(-1, n).double(), s + a.reshape(-1, n).double().abs()
    got = linear_int4(x, q, b, relu, a)
    assert got.shape == (*x.shape[:-1], n) and got.dtype is dtype
    bound = U[dtype] * y.abs() + (k / 16 + 32) * 2.0 ** -22 * s + (U[dtype] * s if m > 64 else 0) + 1e-7
    excess = ((got.reshape(-1, n).double() - y).abs() - bound).max().item()
    assert excess <= 0, excess


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m", [1, 3, 8, 9, 16, 17, 32, 33, 64, 65, 200])
@pytest.mark.parametrize("k,n,group", [(64, 16, 64), (200, 130, 32), (1024, 1000, 64), (1000, 24, 128), (33, 5, 128)])
def test_linear(m, k, n, group, dtype):
    _check_linear(m, k, n, group, dtype, seed=m)


@gpu
@pytest.mark.parametrize("m", [1, 20, 100])
@pytest.mark.parametrize("bias,relu,addend", [(True, False, False), (False, True, False), (True, True, True), (True, False, True)])
def test_linear_epilogues(m, bias, relu, addend):
    _check_linear(m, 320, 210, 64, torch.float16, bias, relu, addend)
    _check_linear(m, 321, 211, 32, torch.bfloat16, bias, relu, addend)


@gpu
@pytest.mark.parametrize("n", [16, 2000, 6000, 20000])  # one, two and four strips to a block, blocks of one and of several warps
@pytest.mark.parametrize("m", [1, 12])
def test_linear_splits(m, n):
    _check_linear(m, 512, n, 64, torch.float16)
    _check_linear(m, 1088, n, 32, torch.bfloat16, bias=True)


@gpu
def test_linear_of_many_rows_and_long_contractions():
    _check_linear(2, 16384, 48, 128, torch.float16)
    _check_linear(1500, 256, 100, 64, torch.bfloat16, True, True, True)


@gpu
@pytest.mark.parametrize("m", [5, 70])
def test_linear_of_strided_inputs(m):
    base = _randn(m, 3 * 192 + 1, seed=4, dtype=torch.float16)
    for x in (base[:, :192], base[:, 1:193], base[:, 192:384:1], base[:, :384:2], base[:1, :192].expand(m, 192),
              _randn(192, m, seed=5, dtype=torch.float16).t(), _randn(m, 1, 192, seed=6, dtype=torch.float16)):
        _check_linear(m, 192, 80, 64, torch.float16, x=x)
    assert linear_int4(base[:0, :192], quantize_int4(_randn(192, 80, seed=7, dtype=torch.float16))).shape == (0, 80)


@gpu
@pytest.mark.parametrize("m", [10, 100])
def test_linear_of_repeated_and_transposed_rows(m):
    """The same numbers in another layout: the same bits."""
    q = quantize_int4(_randn(200, 130, seed=1, dtype=torch.float16))
    for x in (_randn(1, 200, seed=2, dtype=torch.float16).expand(m, 200), _randn(200, m, seed=3, dtype=torch.float16).t(),
              _randn(m, 1, seed=4, dtype=torch.float16).expand(m, 200)):
        assert torch.equal(linear_int4(x, q), linear_int4(x.contiguous(), q))
    assert linear_int4(_randn(m, 200, seed=5, dtype=torch.float16)[:0], q).shape == (0, 130)


@gpu
def test_quantize_of_repeated_rows_and_columns():
    for w in (_randn(1, 70, seed=1, dtype=torch.float16).expand(33, 70), _randn(33, 1, seed=2, dtype=torch.float16).expand(33, 70)):
        a, b = quantize_int4(w), quantize_int4(w.contiguous())
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)


@gpu
def test_linear_addend_and_bias_of_any_layout():
    w, x = _randn(128, 96, seed=1, dtype=torch.float16), _randn(4, 128, seed=2, dtype=torch.float16)
    q = quantize_int4(w)
    a, b = _randn(96, 4, seed=3, dtype=torch.float16).t(), _randn(96, 2, seed=4, dtype=torch.float16)[:, 0]
    assert torch.equal(linear_int4(x, q, b, False, a), linear_int4(x, q, b.contiguous(), False, a.contiguous()))


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_the_largest_weights_stay_finite(dtype):
    """7 LARGEST, rounded to the type, is what the type's largest value becomes.  Powers of two of it round alike."""
    w = torch.zeros((64, 17), device="cuda", dtype=dtype)
    w[3, 2], w[5, 16], w[6, 16] = torch.finfo(dtype).max, -torch.finfo(dtype).max, torch.finfo(dtype).max / 2
    q = quantize_int4(w)
    codes, scales = _definition(w, 64)
    assert torch.equal(q.dequantize(), (codes * scales).to(dtype)) and q.dequantize().isfinite().all()
    for m in (1, 70):
        x = torch.zeros((m, 64), device="cuda", dtype=dtype)
        x[0, 3], x[-1, 5] = 0.5, 0.25  # one row or two: the columns have one weight in each
        got = linear_int4(x, q)
        want = (codes * scales)[[3, 5], [2, 16]] * torch.tensor([0.5, 0.25], device="cuda")
        assert torch.equal(torch.stack((got[0, 2], got[-1, 16])), want.to(dtype))


@gpu
@pytest.mark.parametrize("m", [1, 9, 30, 70, 300])
def test_the_relu_of_nan_is_that_of_the_other_linears(m):
    from tritonformer_b200.linear import LinearNoBiasReLU
    w = _randn(128, 64, seed=1, dtype=torch.float16)
    w[5, 7] = float("nan")
    x = _randn(m, 128, seed=2, dtype=torch.float16)
    q = quantize_int4(w)
    got, plain = linear_int4(x, q, relu=True), linear_int4(x, q)
    assert plain[:, 7].isnan().all() and not got[:, 7].any() and torch.equal(got[:, :7], plain[:, :7].clamp(min=0))
    with torch.no_grad():
        assert not LinearNoBiasReLU.apply(x, w)[:, 7].any()


@gpu
def test_linear_infinities_in_the_input_stay_in_their_rows():
    q = quantize_int4(_randn(256, 64, seed=1, dtype=torch.float16))
    x = _randn(10, 256, seed=2, dtype=torch.float16)
    want = linear_int4(x, q)
    x[4, 100], x[7, 3] = float("inf"), float("nan")
    got = linear_int4(x, q)
    keep = [i for i in range(10) if i not in (4, 7)]
    assert torch.equal(got[keep], want[keep]) and not got[4].isfinite().any() and got[7].isnan().all()


@gpu
def test_linear_in_graphs_and_on_other_streams():
    q = quantize_int4(_randn(1024, 1024, seed=1, dtype=torch.bfloat16))
    xs = [_randn(m, 1024, seed=m, dtype=torch.bfloat16) for m in (1, 30, 300)]
    want = [linear_int4(x, q) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert all(torch.equal(linear_int4(x, q), y) for x, y in zip(xs, want))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [linear_int4(x, q) for x in xs]
    for y in got:
        y.zero_()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_linear_refusals():
    w = _randn(128, 64, seed=1, dtype=torch.float16)
    q, x = quantize_int4(w), torch.ones((2, 128), device="cuda", dtype=torch.float16)
    for call, text in ((lambda: linear_int4(x[:, :64], q), "last dimension"), (lambda: linear_int4(x.bfloat16(), q), "type of the weight"),
                       (lambda: linear_int4(x, q, x[0, :63]), "bias"), (lambda: linear_int4(x, q, None, False, x[:, :32]), "addend"),
                       (lambda: quantize_int4(w.float()), "fp16/bf16"), (lambda: quantize_int4(w, 48), "32, 64 or 128"),
                       (lambda: quantize_int4(w[:0]), "weight"),
                       (lambda: linear_int4(x, Int4Weight(q.codes[:2], q.scales, 128, 64, 64)), "codes"),
                       (lambda: linear_int4(x, Int4Weight(q.codes, q.scales, 128, 64, 32)), "scales"),
                       (lambda: linear_int4(x.clone().requires_grad_(), q), "no gradients"),
                       (lambda: linear_int4(x.cpu(), q), "CUDA")):
        with pytest.raises(AssertionError, match=text):
            call()


def test_refusals_without_a_device():
    one = ctypes.c_void_p(16)  # never dereferenced
    for args, text in (((0, 1, 8, 8, 48), b"groups of 48"), ((8, 1, 0, 8, 64), b"bad shape")):
        assert L.lib.tfb_int4_quantize(one, *args, one, one, 0, None) == -1 and text in L.lib.tfb_last_error()
    assert L.lib.tfb_int4_quantize(one, 8, 1, 8, 8, 64, one, one, 2, None) == -1  # fp32
    assert L.lib.tfb_int4_linear(one, 8, ctypes.c_void_p(8), one, None, None, 0, one, 8, 1, 8, 8, 64, 0, 0, None) == -1
    assert b"aligned" in L.lib.tfb_last_error()
    assert L.lib.tfb_int4_linear(one, 8, one, one, None, None, 0, one, 4, 2, 8, 8, 64, 0, 0, None) == -1
    assert L.lib.tfb_int4_linear(None, 8, None, None, None, None, 0, None, 8, 0, 8, 8, 64, 0, 0, None) == 0  # no rows
    assert L.lib.tfb_int4_codes(65, 17) == 2 * 2 * 128 and L.lib.tfb_int4_scales(65, 17, 32) == 4 * 32
    w = torch.zeros((64, 16), dtype=torch.float16)
    with pytest.raises(AssertionError, match="CUDA"):
        int4.quantize_int4(w)
