"""Drawing tokens at the borders of what is kept."""
import os
import re

import pytest
import torch

import tritonformer_b200
from test_sampling import SETTINGS, _check, _logits
from tritonformer_b200 import sample_tokens

gpu = pytest.mark.gpu


def test_a_border_that_is_being_read_is_not_written():
    """In the kernel of 16-bit logits all warps read the border that top-k or top-p has left behind the same barrier that lets one warp look for min-p's.
    That one has to leave its result in another place: by reading, as no run shows it for certain."""
    path = os.path.join(os.path.dirname(tritonformer_b200.__file__), "csrc", "sampling.cu")
    with open(path) as f:
        kernel = re.search(r"sample_hist_kernel\(const SampleParams p\) \{.*?\n\}\n", f.read(), re.S).group(0)
    block = re.search(r"\n  if \(min_p > 0\.f\) \{.*?\n  \}\n", kernel, re.S).group(0)
    search = block[:block.index("__syncthreads()")]
    written = set(re.findall(r"sh\.(\w+) = ", search))
    before = kernel[:kernel.index(block)]
    assert written and not any(re.search(rf"sh\.{name}\b", before) for name in written)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("batch,vocab", [(100, 3001), (3, 20000), (2, 131071)])
def test_min_p_behind_another_cut(batch, vocab, dtype):
    """min-p's border above the other one and below it, behind top-k, top-p and both, for more candidates than are listed."""
    for i, settings in enumerate(({"top_p": 0.9, "min_p": 0.3}, {"top_p": 0.5, "min_p": 1e-4}, {"top_k": 1000, "min_p": 0.2}, {"top_k": 300, "min_p": 1e-6},
                                  {"top_k": 1000, "top_p": 0.97, "min_p": 0.1}, {"top_k": 2000, "top_p": 0.6, "min_p": 1e-3})):
        _check(_logits(batch, vocab, dtype, i, 1.0), settings, i)
        _check(_logits(batch, vocab, dtype, i, 2.0).round(), settings, i)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("value", [-2.5, 0.375, 1.125, 1.375, 4.0, 30.0])
@pytest.mark.parametrize("n", [4, 6, 12, 40, 200, 300, 1000, 5000])
def test_equal_logits_at_an_exact_border(n, value, dtype):
    """n logits share a row's weight and weigh 1 each, so that every sum is a whole number: the share of top_p is a prefix, and the uniform number's of
    that its token.  Both products are exact: n and the shares are whole numbers over powers of two."""
    vocab = 3 * n + 7
    x = torch.full((64, vocab), -float("inf"), device="cuda", dtype=dtype)
    columns = 3 * torch.arange(n, device="cuda") + 2
    x[:, columns] = value
    u = (torch.arange(64, device="cuda") * 2 + 1) / 128
    ends = torch.tensor([0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24] * 12 + [0.125] * 4, device="cuda")
    for numbers in (u.float(), ends):
        for p in (0.25, 0.5, 0.75, 1.0):
            for k in {0, n, n - 1, n // 2, n + 3}:
                among = min(k, n) if k else n
                kept = max(-(-int(4 * p) * among // 4), 1)
                for least, t in ((0.0, 1.0), (1.0, 0.7), (0.5, 3.0)):
                    got = sample_tokens(x, numbers, temperature=t, top_k=k, top_p=p, min_p=least)
                    want = columns[(numbers.double() * kept).long()]
                    assert torch.equal(got, want), (p, k, least, t)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_the_same_logits_in_another_type_give_the_same_tokens(dtype):
    """Weights depend on the values alone; the three ways to a token have one rule for ties."""
    u = torch.rand((150,), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    for i, settings in enumerate(SETTINGS):
        for x in (_logits(150, 4001, dtype, i).round(), _logits(150, 300, dtype, i, 0.4).round() + 1.375):
            assert torch.equal(sample_tokens(x, u, **settings), sample_tokens(x.float(), u, **settings))


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [5, 900, 70000])
def test_the_smallest_numbers_do_not_draw_what_weighs_nothing(vocab, dtype):
    """At temperature 0.05 a logit of -30 below ten weighs e^-800, zero in 64 bits: not even u = 0 draws it, the first of its row and of many."""
    x = _logits(6, vocab, dtype, 1, 0.5).clamp(-2, 2) + 8
    x[:, 0] = -30.0
    x[1::2, 1:vocab // 2] = -30.0
    x[2, :-1], x[3, -1] = -30.0, -30.0
    for u in (torch.zeros(6, device="cuda"), torch.full((6,), 2.0 ** -149, device="cuda"), torch.full((6,), 2.0 ** -24, device="cuda")):
        for settings in ({}, {"top_k": 4}, {"top_k": 600}, {"top_p": 0.9}, {"min_p": 1e-30}, {"top_k": 200, "top_p": 0.999}):
            got = _check(x, {"temperature": 0.05, **settings}, u=u)
            assert (x.gather(1, got[:, None]) > 0).all()
