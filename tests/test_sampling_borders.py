"""Drawing tokens at the borders of what is kept."""
import os
import re

import pytest
import torch

import tritonformer_b200
from test_sampling import _check, _logits

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
