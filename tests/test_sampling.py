"""Drawing tokens against the definition, which sorts each row in 64 bits.  Tokens are equal, not near: the kernel's sums are in 64 bits too, and
the chance that a border between two tokens lies between the two sums is below 1e-8 for all draws here together."""
import ctypes
import math

import pytest
import torch

import tritonformer_b200._lib as L
from tritonformer_b200 import sample_tokens

gpu = pytest.mark.gpu


def definition(row, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The token of one row of logits, on the CPU."""
    x = row.double().nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    best, order = torch.sort(x, descending=True, stable=True)
    if best[0] == -math.inf:
        return -1
    if temperature == 0:
        return int(order[0])
    w = torch.where(best == best[0], 1.0, ((best - best[0]) / float(torch.tensor(temperature))).exp())
    count = len(w) if top_k == 0 else min(top_k, len(w))
    if top_p < 1:
        ahead = w[:count].cumsum(0) - w[:count]
        ahead[1:] = w[:count].cumsum(0)[:-1]
        count = max(1, int((ahead < float(torch.tensor(top_p)) * w[:count].sum()).sum()))
    count = min(count, int((w >= float(torch.tensor(min_p))).sum()), int((w > 0).sum()))
    chosen, back = torch.sort(order[:count])
    line = w[:count][back].cumsum(0)
    return int(chosen[min(int(torch.searchsorted(line, u * float(line[-1]), right=True)), count - 1)])


SETTINGS = [{}, {"temperature": 0.0}, {"temperature": 0.6}, {"top_k": 1}, {"top_k": 5}, {"top_k": 40, "top_p": 0.9}, {"top_p": 0.95},
            {"top_p": 0.3, "temperature": 1.7}, {"min_p": 0.1}, {"top_k": 100, "top_p": 0.8, "min_p": 0.02, "temperature": 0.9},
            {"top_p": 0.999, "temperature": 3.0}, {"top_k": 2000, "temperature": 2.0}, {"min_p": 1.0}, {"top_p": 1e-6}]


def _check(logits, settings, seed=0, u=None):
    batch = logits.shape[0]
    if u is None:
        u = torch.rand((batch,), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")
    got = sample_tokens(logits, u, **settings)
    rows, lines = logits.cpu(), u.tolist()
    pick = lambda v, i: v[i].item() if isinstance(v, torch.Tensor) else v  # noqa: E731
    want = [definition(rows[i], lines[i], **{k: pick(v, i) for k, v in settings.items()}) for i in range(batch)]
    assert got.dtype is torch.int64 and got.tolist() == want
    return got


def _logits(batch, vocab, dtype, seed=0, scale=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn((batch, vocab), generator=g, device="cuda")).to(dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("batch,vocab", [(3, 1), (4, 2), (5, 7), (9, 33), (3, 1000), (40, 5001), (300, 777), (2, 50304)])
def test_draws_are_the_definition(batch, vocab, dtype):
    for i, settings in enumerate(SETTINGS):
        _check(_logits(batch, vocab, dtype, i), settings, i)


@gpu
@pytest.mark.parametrize("dtype,vocab", [(torch.bfloat16, 131071), (torch.float32, 131072), (torch.float16, 262145), (torch.float32, 300001)])
def test_large_vocabularies(dtype, vocab):
    for i, settings in enumerate(({}, {"top_k": 50, "top_p": 0.9}, {"top_p": 0.99}, {"min_p": 0.01})):
        _check(_logits(2, vocab, dtype, i), settings, i)
    _check(_logits(150, 20000, dtype, 9), {"top_p": 0.9})


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_equal_logits(dtype):
    """Many logits share a value, the border's among them; all may be one."""
    for i, settings in enumerate(SETTINGS):
        _check(_logits(12, 4099, dtype, i).round(), settings, i)
        _check(torch.full((12, 3000), -2.5, device="cuda", dtype=dtype), settings, i)
        _check(torch.zeros((4, 50304), device="cuda", dtype=dtype) * torch.where(torch.arange(50304, device="cuda") % 2 == 0, 1, -1).to(dtype),
               settings, i)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("batch,vocab", [(3, 65272), (2, 65535), (40, 65536), (40, 130544), (40, 130545), (40, 131056), (2, 522176 - 150000)])
def test_more_equal_logits_than_a_short_counter_holds(batch, vocab, dtype):
    """Equal weights: the kept ones are the first ones, and the token is the whole part of u times their number.  (i + 1/2) / n in 32 bits, times n
    again, is within n 2^-24 < 1/32 of i + 1/2."""
    x = torch.zeros((batch, vocab), device="cuda", dtype=dtype)  # weights of 1: exact sums
    for settings, kept in (({}, vocab), ({"top_k": 30000}, 30000), ({"top_p": 0.5}, (vocab + 1) // 2), ({"min_p": 1.0}, vocab),
                           ({"top_k": 50000, "top_p": 0.25}, 12500)):
        want = torch.linspace(0, kept - 1, batch, dtype=torch.float64).round().long()
        u = ((want + 0.5) / kept).float().cuda()
        assert sample_tokens(x, u, **settings).tolist() == want.tolist()


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("batch,vocab", [(1, 50304), (3, 2049), (150, 1500), (17, 131071), (2, 300)])
def test_few_and_many_candidates(batch, vocab, dtype):
    """Numbers of candidates around those at which they are found in another way, alone and with many equal logits among them."""
    for i, k in enumerate((2, 31, 32, 33, 64, 200, 255, 256, 257, 1023, 1024, 1025)):
        for x in (_logits(batch, vocab, dtype, i), _logits(batch, vocab, dtype, i, 2.0).round()):
            _check(x[:5] if i % 3 else x, {"top_k": k, "top_p": (1.0, 0.9)[i % 2], "min_p": (0.0, 0.0, 0.01)[i % 3]}, i)
    for i, least in enumerate((0.9, 0.3, 0.01, 1e-3, 1e-5, 1e-8)):
        _check(_logits(batch, vocab, dtype, i)[:5], {"min_p": least, "temperature": (0.5, 1.0, 4.0)[i % 3]}, i)
    # all that is left of a row is few: the rest is ruled out, in one place or all over
    x = _logits(batch, vocab, dtype)
    x[:, 40:] = -math.inf
    _check(x[:5], {"top_k": 39}), _check(x[:5], {"top_k": 40, "top_p": 0.8}), _check(x[:5], {"top_k": 41}), _check(x[:5], {"min_p": 1e-4})
    x = _logits(batch, vocab, dtype).masked_fill(torch.rand((batch, vocab), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") < 0.97, -math.inf)
    _check(x[:5], {"top_k": 20}), _check(x[:5], {"top_p": 0.7}), _check(x[:5], {"top_k": 100, "min_p": 0.1})


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_what_is_not_finite(dtype):
    for i, settings in enumerate(SETTINGS):
        x = _logits(8, 2500, dtype, i)
        x[0] = -math.inf
        x[1] = math.nan
        x[2, 100:] = -math.inf
        x[3, ::3] = math.nan
        x[4, [5, 900, 2000]] = math.inf
        x[5] = math.inf
        x[6] = torch.finfo(dtype).min
        x[7, 17:] = torch.finfo(dtype).min
        got = _check(x, settings, i)
        assert got[0] == -1 and got[1] == -1


@gpu
def test_one_logit_far_below_or_above():
    for dtype in (torch.float16, torch.float32):
        x = _logits(6, 3001, dtype)
        x[0, 3], x[1, 3], x[2, 3000], x[3, 0] = -60000.0, 60000.0, 50.0, 1e-7
        for i, settings in enumerate(SETTINGS):
            _check(x, settings, i)
    big = _logits(4, 1001, torch.float32) * 1e37
    for i, settings in enumerate(SETTINGS):
        _check(big, settings, i)


@gpu
def test_uniform_numbers_at_their_ends():
    x = _logits(6, 1234, torch.float16)
    for settings in SETTINGS:
        _check(x, settings, u=torch.zeros(6, device="cuda"))
        _check(x, settings, u=torch.full((6,), 1 - 2.0 ** -24, device="cuda"))
    # outside of them: the nearest
    near = sample_tokens(x[:3], torch.tensor([0.0, 0.0, 1 - 2.0 ** -24], device="cuda"))
    assert torch.equal(sample_tokens(x[:3], torch.tensor([-1.0, math.nan, 7.0], device="cuda")), near)


@gpu
def test_settings_of_each_row():
    n = len(SETTINGS)
    x = _logits(n, 6007, torch.float16)
    each = {k: torch.tensor([s.get(k, d) for s in SETTINGS], device="cuda", dtype=torch.int32 if k == "top_k" else torch.float32)
            for k, d in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))}
    got = _check(x, each)
    u = torch.rand((n,), generator=torch.Generator(device="cuda").manual_seed(0), device="cuda")
    for i, settings in enumerate(SETTINGS):  # whatever a row shares the call with
        assert sample_tokens(x[i:i + 1], u[i:i + 1], **settings)[0] == got[i]
    # numbers out of range count as the nearest
    odd = {"temperature": torch.tensor([-1.0, math.nan] + [1.0] * (n - 2)), "top_k": torch.tensor([0, 0, -5, 1 << 30] + [0] * (n - 4)),
           "top_p": torch.tensor([1.0] * 4 + [math.nan, 2.0, -1.0] + [1.0] * (n - 7)),
           "min_p": torch.tensor([0.0] * 7 + [math.nan, -1.0, 3.0] + [0.0] * (n - 10))}
    odd = {k: v.to(device="cuda", dtype=each[k].dtype) for k, v in odd.items()}
    got, plain = sample_tokens(x, u, **odd), sample_tokens(x, u)
    first = x.float().argmax(1)
    for i in range(n):
        assert got[i] == (first[i] if i in (0, 1, 6, 9) else plain[i]), i


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_rows_of_any_layout(dtype):
    base = _logits(7, 2003, dtype)
    for x in (base[:, 1:], base[:, 3:1900], base[::2], base[:1].expand(7, 2003), base[:, ::2], base.t()[:500], base[:, :1]):
        for settings in ({}, {"top_k": 20, "top_p": 0.8}):
            _check(x, settings)
    assert sample_tokens(base[:0], torch.zeros(0, device="cuda")).shape == (0,)


@gpu
def test_the_shares_are_the_weights():
    """Evenly spaced uniform numbers: each token gets its weight's share of them, to one of them at each border."""
    x = torch.tensor([0.5, -1.0, 2.0, 0.0, -math.inf, 1.0], device="cuda", dtype=torch.float32)
    n = 4096
    u = (torch.arange(n, device="cuda") + 0.5) / n
    got = torch.bincount(sample_tokens(x.expand(n, 6), u.float(), temperature=0.7), minlength=6)
    assert (got.double() - n * torch.softmax(x.double() / 0.7, 0)).abs().max() <= 1.001


@gpu
def test_in_graphs_and_on_other_streams():
    x, u = _logits(5, 50304, torch.float16), torch.rand(5, device="cuda")
    settings = {"top_k": 30, "top_p": 0.9}
    want = sample_tokens(x, u, **settings)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(sample_tokens(x, u, **settings), want)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sample_tokens(x, u, **settings)
    for seed in range(3):
        x.copy_(_logits(5, 50304, torch.float16, seed))
        u.uniform_()
        graph.replay()
        assert torch.equal(got, sample_tokens(x, u, **settings))


@gpu
def test_refusals():
    x, u = _logits(3, 100, torch.float16), torch.zeros(3, device="cuda")
    for call, text in ((lambda: sample_tokens(x[0], u), r"\(batch, vocab\)"), (lambda: sample_tokens(x, u[:2]), "uniform"),
                       (lambda: sample_tokens(x, u.double()), "uniform"), (lambda: sample_tokens(x.long(), u), "fp16, bf16 or fp32"),
                       (lambda: sample_tokens(x, u, temperature=-0.1), "temperature"), (lambda: sample_tokens(x, u, temperature=math.inf), "temperature"),
                       (lambda: sample_tokens(x, u, top_k=-1), "top_k"), (lambda: sample_tokens(x, u, top_k=2.5), "whole number"), (lambda: sample_tokens(x, u, top_p=0.0), "top_p"),
                       (lambda: sample_tokens(x, u, top_p=1.1), "top_p"), (lambda: sample_tokens(x, u, min_p=1.5), "min_p"),
                       (lambda: sample_tokens(x, u, top_k=u), "int32"), (lambda: sample_tokens(x, u, temperature=u[:1]), "fp32"),
                       (lambda: sample_tokens(x.cpu(), u), "CUDA"), (lambda: sample_tokens(x.clone().requires_grad_(), u), "no gradients")):
        with pytest.raises(AssertionError, match=text):
            call()
    with pytest.raises(AssertionError, match="cluster"):
        sample_tokens(torch.zeros((1, 1 << 20), device="cuda"), u[:1])


def test_refusals_without_a_device():
    one = ctypes.c_void_p(16)  # never dereferenced
    rest = (one, None, 1.0, None, 0, None, 1.0, None, 0.0, one)
    assert L.lib.tfb_sample(one, 8, *rest, 2, 0, 0, None) == -1 and b"bad shape" in L.lib.tfb_last_error()
    assert L.lib.tfb_sample(None, 8, *rest, 2, 8, 0, None) == -1 and b"null" in L.lib.tfb_last_error()
    assert L.lib.tfb_sample(one, 8, *rest, 2, 8, 7, None) == -1 and b"dtype" in L.lib.tfb_last_error()
    assert L.lib.tfb_sample(None, 8, *rest, 0, 8, 0, None) == 0
    with pytest.raises(AssertionError, match="CUDA"):
        sample_tokens(torch.zeros((2, 8)), torch.zeros(2))
