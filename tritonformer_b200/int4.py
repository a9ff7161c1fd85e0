"""Linear weights in 4 bits, for generating text: a token of one or a few sequences reads every weight once, so that its time is the
weights' bytes.  The reference has no counterpart: it trains only.

A weight (in, out) is a 16-bit scale for each group of 32, 64 or 128 rows of a column, times a whole number from -7 to 7: the scale
is the group's largest magnitude over 7 (at most the largest number whose sevenfold the type holds), the number the nearest to weight / scale.  4.5, 4.25 or 4.125 bits a weight.

  * `quantize_int4`  packs a weight
  * `linear_int4`    act(x W + bias) + addend with a packed weight, any number of rows
  * `Int4Weight`     a packed weight; `dequantize()` gives what it stands for

No product rounds a weight a second time.  Up to 96 rows read the packed weights as they are; for more (a prompt) each becomes the sum of two
numbers of the 16-bit type, and the tensor-core product of the training takes both along a contraction of twice the length.  That call has
two buffers beside its output: twice the weight in 16 bits, and twice its rows.  `dequantize` rounds, to give one number for a weight.  No gradients.
"""
from . import _host


class Int4Weight:
    """A weight of `in_features` rows and `out_features` columns in 4 bits.  `codes` (strips of 16 columns, units of 64 rows, 32, 4)
    int32 and `scales` (strips, groups, 8, 2), as `quantize_int4` lays them out (tritonformer_b200.h has the places of the bits)."""

    __slots__ = ("codes", "scales", "in_features", "out_features", "group")

    def __init__(self, codes, scales, in_features, out_features, group):
        self.codes, self.scales, self.in_features, self.out_features, self.group = codes, scales, in_features, out_features, group

    def dequantize(self):
        """(in, out) in the scales' type, a view of a transposed and padded buffer."""
        return _host.int4_expand(self.codes, self.scales, self.in_features, self.out_features, self.group)

    def nbytes(self):
        return self.codes.numel() * 4 + self.scales.numel() * 2


def quantize_int4(weight, group=64):
    """The fp16 or bf16 `weight` (in, out), of any strides, with a scale for each `group` rows of a column.  A group with a weight that is not
    finite becomes NaN as a whole."""
    codes, scales = _host.int4_quantize(weight, group)
    return Int4Weight(codes, scales, weight.shape[0], weight.shape[1], group)


def linear_int4(x, weight, bias=None, relu=False, addend=None):
    """act(x W + bias) + addend: x (.., in) of the type of the weight's scales, bias (out,), addend (.., out); sums in 32 bits, one rounding.  The ReLU
    of a NaN is 0, as in the other linears."""
    return _host.int4_linear(x, weight.codes, weight.scales, weight.in_features, weight.out_features, weight.group, bias, relu, addend)
