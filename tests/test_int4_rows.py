"""Products with 4-bit weights give a row the same answer however many rows share the call: no weight is rounded for many of them either.

The numbers are chosen so that nothing but the output's rounding can happen, and results are equal to the definition's, not near."""
import ctypes

import pytest
import torch

import tritonformer_b200._lib as L
from tritonformer_b200 import linear_int4, quantize_int4

gpu = pytest.mark.gpu
ROWS = [1, 16, 65, 96, 97, 300]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _weight(k, n, group, dtype, seed):
    """Weights whose scales all lie in [2^-7, 2^-6): their codes times scales are multiples of 2^-17."""
    w = 0.05 * (2 * torch.rand((k, n), generator=_gen(seed), device="cuda") - 1)
    for g in range(0, k, group):  # the largest of each group, over 7: 0.0086 to 0.0143
        w[g] = 0.06 + 0.04 * torch.rand((n,), generator=_gen(seed + g + 1), device="cuda")
    return w.to(dtype)


def _exact(w, group):
    """codes times scales in 64 bits, unrounded."""
    k, n = w.shape
    groups = -(-k // group)
    blocks = torch.zeros((groups * group, n), dtype=torch.float64, device=w.device)
    blocks[:k] = w.double()
    blocks = blocks.view(groups, group, n)
    scales = (blocks.abs().amax(1, keepdim=True) / 7).to(w.dtype).double()
    return ((blocks / scales).round().clamp(-7, 7) * scales).view(-1, n)[:k]


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("k,n,group", [(64, 16, 64), (128, 200, 32), (77, 50, 128)])
def test_whole_numbers_times_weights_are_rounded_once(k, n, group, m, dtype):
    """Whole numbers up to 4 times multiples of 2^-17 of at most 7 * 2^-6: a sum of 128 is a multiple of 2^-17 below 56, 23 bits, and exact in any order."""
    w = _weight(k, n, group, dtype, k)
    full = _exact(w, group)
    assert (full * 2.0 ** 17 == (full * 2.0 ** 17).round()).all() and (full != full.to(dtype).double()).any()
    x = torch.randint(-4, 5, (m, k), generator=_gen(m), device="cuda").to(dtype)
    q = quantize_int4(w, group)
    assert torch.equal(linear_int4(x, q), (x.double() @ full).to(dtype))
    assert torch.equal(linear_int4(x, q, relu=True), (x.double() @ full).clamp(min=0).to(dtype))


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m", ROWS)
def test_what_rounding_a_weight_would_lose_is_there(m, dtype):
    """One weight less what it is in 16 bits."""
    k, n, group = 200, 40, 64
    w = _weight(k, n, group, dtype, 3)
    q = quantize_int4(w, group)
    full, rounded = _exact(w, group), q.dequantize()
    at = torch.arange(m, device="cuda") * 7 % k
    x = torch.zeros((m, k), device="cuda", dtype=dtype)
    x[torch.arange(m, device="cuda"), at] = 1
    want = (full - rounded.double())[at]
    assert want.any() and torch.equal(linear_int4(x, q, addend=-rounded[at]).double(), want)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m", ROWS)
def test_infinities_and_nan_are_those_of_the_weights(m, dtype):
    """An infinity times a weight is infinite, times a weight of zero NaN, and nothing else of the call changes."""
    k, n, group = 128, 64, 64
    w = _weight(k, n, group, dtype, 5)
    w[:, 9] = w[:, 9].masked_fill(torch.arange(k, device="cuda") == 70, float("nan"))
    q = quantize_int4(w, group)
    x = torch.randint(-4, 5, (m, k), generator=_gen(m), device="cuda").to(dtype)
    want = linear_int4(x, q)
    x[0, 17] = float("inf")
    full = _exact(w, group)[17]
    inf = torch.where(full == 0, float("nan"), full.sign() * float("inf"))
    inf[9] = float("nan")
    assert (full == 0).any() and (full > 0).any() and (full < 0).any()
    got = linear_int4(x, q)
    assert torch.equal(got[0].double().nan_to_num(7.0, 8.0, 9.0), inf.nan_to_num(7.0, 8.0, 9.0))
    assert torch.equal(got[1:].nan_to_num(7.0), want[1:].nan_to_num(7.0)) and got[:, 9].isnan().all()


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m", [3, 100])
def test_rows_at_any_address(m, dtype):
    """Rows that no vector load can read, and the same numbers where one can: the same bits."""
    q = quantize_int4(_weight(100, 48, 32, dtype, 6), 32)
    flat = torch.randint(-4, 5, (m * 205 + 9,), generator=_gen(7), device="cuda").to(dtype)
    for first in (0, 1, 8):
        for pitch in (100, 104, 205):
            x = flat[first:].as_strided((m, 100), (pitch, 1))
            assert torch.equal(linear_int4(x, q), linear_int4(x.clone(), q))


@gpu
def test_in_a_graph_beside_an_eager_call():
    q, x = quantize_int4(_weight(256, 100, 64, torch.float16, 8), 64), torch.randn((130, 256), generator=_gen(9), device="cuda").half()
    want = linear_int4(x, q)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        got = linear_int4(x, q)
    torch.cuda.synchronize()
    for _ in range(10):
        got.zero_()
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            again = linear_int4(x, q)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(again, want)


def test_refusals_without_a_device():
    one, odd = ctypes.c_void_p(16), ctypes.c_void_p(18)  # never dereferenced

    def split(codes=one, out=one, x=one, ld=8, m=3, x_out=one, dtype=0, k=8, group=64):
        return L.lib.tfb_int4_split(codes, one, k, 8, group, out, x, ld, m, x_out, dtype, None)

    for call, text in (((lambda: split(group=48)), b"groups of 48"), ((lambda: split(k=0)), b"bad shape"), ((lambda: split(codes=odd)), b"aligned"),
                       ((lambda: split(out=None)), b"aligned"), ((lambda: split(x_out=odd)), b"aligned"), ((lambda: split(x=None)), b"aligned"),
                       ((lambda: split(m=-1)), b"row count"), ((lambda: split(ld=-8)), b"row stride"), ((lambda: split(dtype=2)), b"dtype")):
        assert call() == -1 and text in L.lib.tfb_last_error()
