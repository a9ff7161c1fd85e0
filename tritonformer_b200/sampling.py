"""Drawing tokens from logits.  The reference has no counterpart: it trains only."""
import torch

from . import _host


def _setting(value):
    return (value, 0.0) if isinstance(value, torch.Tensor) else (None, value)


def _positive(value):
    return (value, 1.0) if isinstance(value, torch.Tensor) else (None, value)


def sample_tokens(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(batch,) int64: one token per row of `logits` (batch, vocab), fp16, bf16 or fp32, from `uniforms` (batch,) fp32 in [0, 1).

    With w = exp((logit - largest) / temperature), larger logits first and equal ones by index, kept are the first `top_k` tokens (0: all),
    of those the ones before which less than `top_p` of their weight lies, and of those the ones with at least `min_p` of the largest
    weight; the first is always kept.  The token is the first, in the order of the vocabulary, at which the kept weight reaches `uniforms`
    of its sum.  Temperature 0 takes the largest logit, of equal ones the first.  Each setting is a number (taken in 32 bits) or a (batch,)
    tensor with one for each row: int32 for top_k, fp32 for the others; of a tensor's values those out of range count as the nearest.
    A logit that is NaN or -infinity is never drawn; a row without any other gives -1.  Weights and sums are in 64 bits and in a fixed
    order: the same numbers give the same token, also in a captured graph.  A row has at most 522176 logits of 16 bits, or some 434000 of 32; longer
    ones are refused.  No gradients."""
    return _host.sample(logits, uniforms, *_positive(temperature), *_setting(top_k), *_positive(top_p), *_setting(min_p))
