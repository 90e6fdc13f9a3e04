"""The weights of attention over the 4-bit cache, as the second product takes
them: what is lost of them, in every type and at every number of heads.

Tolerances as in test_gpu_cache4bit.py, with two 16-bit parts for all types
(2^-21 of a weight, twice, and what the sums lose: 2^-18 in all).
"""
import pytest
import torch

from .test_gpu_cache4bit import HALF, TINY, TYPES, fill, gen, randn, reference, within

pytestmark = pytest.mark.gpu
WEIGHT = 2.0 ** -18


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [16, 7])
@pytest.mark.parametrize("each", [1, 3, 4, 5, 8, 9])
@pytest.mark.parametrize("lens", [[2, 5, 40, 300], [20011, 3, 0, 150]])
def test_weights_have_two_parts(dtype, page, each, lens):
    """Scores of a few hundredths: the weights are near to one another and not short numbers, and nothing else rounds
    as much.  Outputs near 0 beside their terms, of which there are many, show what a weight has lost."""
    g = gen(page + each + len(lens))
    c, table, n = fill(g, lens, page, 2, 64, 32, dtype)
    q = randn(g, len(lens), 2 * each, 64, dtype=dtype)
    out, lse, errs, mags = reference(c, q, table, n, 2.0 ** -9, 0)
    got = c.attend(q, table, n, scale=2.0 ** -9)
    within(got, out, HALF[dtype] * out.abs() + TINY[dtype] + (2 * errs[..., None] + WEIGHT) * mags)
    c.check()
