"""Newton-Schulz orthogonalisation and the Muon step: the largest tiles in every result type, lists that take more than
one set of launches, and what the optimiser does before, during and instead of a step.

Tolerance, relative in the Frobenius norm, u = 2^-24.  An operand is a pair of fp16 values, off by 2 u at most and by
2 u / sqrt 12 or so in the mean; the product of the two low halves, left out, is below 4 u and 0.7 u in the mean where
both factors are the same value (the diagonal of X X^T); a sum over K values in one 32-bit accumulator is rounded three
times for 16 of them, with errors that add up at random: sqrt(3 K / 16) u.  Together u (4 + sqrt(K) / 2) covers a step's
products.  x -> a x + b x^3 + c x^5 passes an error on with a factor between 0 and max |p'| = 4, about 2 in the mean:
five steps collect 1 + 2 + ... + 16 = 31 of them."""
import pytest
import torch

DEV = "cuda"
U = 2.0 ** -24
A, B, C = 3.4445, -4.775, 2.0315


def test_sizes_that_32_bits_cannot_hold_are_refused():
    from mmsa_amd import _lib, ops
    for shape in ((2 ** 32 + 64, 64), (64, 2 ** 32 + 64), (2 ** 16, 2 ** 16), (2 ** 20 + 1, 2), (1, 2 ** 20 + 1)):
        with pytest.raises(_lib.MmsaError, match="limit"):
            ops._sizes([torch.empty(4, 4, device="meta"), torch.empty(shape, device="meta")])
    rows, cols = ops._sizes([torch.empty(2 ** 20, 2 ** 11, device="meta"), torch.empty(8, 4, 3, 3, device="meta")])
    assert list(rows) == [2 ** 20, 8] and list(cols) == [2 ** 11, 36]
