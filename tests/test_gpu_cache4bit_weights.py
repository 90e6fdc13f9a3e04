"""The weights of attention over the 4-bit cache, as the second product takes
them: what is lost of them, in every type and at every number of heads.

Tolerances as in test_gpu_cache4bit.py, with two 16-bit parts for all types
(2^-21 of a weight, twice, and what the sums lose: 2^-18 in all).
"""
import pytest
import torch

import pyflame_b200 as pf

from .test_gpu_cache4bit import BF16, F16, F32, HALF, TINY, TYPES, check_attend, fill, gen, randn, reference, within

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


def far_apart(g, dtype, n, heads, page, values, order):
    """A cache of one sequence of n keys whose first value alone makes scores: 0 for most keys, up to 1/32 for the
    others; `order`: where a key of -60 and one of 60 stand (None: none).  values: [n, 1, 64]."""
    c = pf.PagedKVCache4bit(-(-n // page), page, 1, 64, group_size=32)
    k = randn(g, n, 1, 64) * 2.0 ** -9
    for at, score in order:
        k[at] = 0
        k[at, 0, 0] = score
    c.append(k.to(dtype), values.to(dtype), torch.arange(n, device="cuda"))
    table = torch.arange(-(-n // page), dtype=torch.int32, device="cuda")[None]
    q = randn(g, 1, heads, 64) * 0.5
    q[..., 0] = torch.where(torch.arange(heads, device="cuda") % 2 == 0, 1.0, -1.0)
    return c, q.to(dtype), table, torch.tensor([n], dtype=torch.int32, device="cuda")


def check_far_apart(c, q, table, n):
    """As check_attend, with the errors of the scores that have any weight."""
    dtype, heads, keys = q.dtype, q.shape[1], int(n)
    k, v = (x.double()[:, 0] for x in c.read(torch.arange(keys, device="cuda")))
    s = q[0].double() @ k.T
    p = torch.softmax(s, -1)
    bound = lambda x: 2 * ((p2 := x.unflatten(-1, (-1, 32))).amax(-1) - p2.amin(-1) + p2.abs().amax(-1)).repeat_interleave(32, -1)
    errs = torch.where(p > 2.0 ** -60, q[0].double().abs() @ bound(k).T * 2.0 ** -18, 0.0).amax(-1)
    out, mags = p @ v, p @ bound(v)
    got = c.attend(q, table, n, scale=1.0)[0]
    within(got, out, HALF[dtype] * out.abs() + TINY[dtype] + (2 * errs[..., None] + WEIGHT) * mags)
    c.check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [16, 5])
@pytest.mark.parametrize("n,heads", [(5, 2), (70, 1), (300, 3), (9000, 4), (9000, 8)])
@pytest.mark.parametrize("place", ["first", "last", "before"])
def test_large_values_without_weight(dtype, page, n, heads, place):
    """One key has values a thousand million times the others' (float16: 2^22 times) and, for every second head, a score 60 below or above theirs:
    where it is below, the others keep their digits.  "before": a key of the score 60 comes after it, so that it had
    weight when it was read."""
    g = gen(n + heads)
    size, big = (2.0 ** -8, 2.0 ** 14) if dtype == F16 else (1.0, 1e9)
    v = size * randn(g, n, 1, 64)
    at = n - 1 if place == "last" else n // 2 if place == "before" else 0
    v[at] = big * torch.rand(1, 64, generator=g, device="cuda")
    order = [(at, -60.0)]
    if place == "before":
        order = [(at, -30.0), (n - 2, 60.0)]
    check_far_apart(*far_apart(g, dtype, n, heads, page, v, order))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ratio", [1e-3, 1e-6, 1e-9])
@pytest.mark.parametrize("n,heads", [(70, 1), (9000, 4), (9000, 8)])
def test_groups_of_different_sizes(dtype, ratio, n, heads):
    """The values of one group far smaller than the other's, in all keys: they keep their digits too."""
    g = gen(n)
    if dtype == F16:
        ratio = max(ratio, 2.0 ** -20)
    v = randn(g, n, 1, 64) * (2.0 ** 12 if dtype == F16 else 1.0)
    v[..., 32:] *= ratio
    check_far_apart(*far_apart(g, dtype, n, heads, 16, v, []))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,heads", [(70, 2), (9000, 4), (9000, 8)])
def test_values_at_both_ends_of_the_type(dtype, n, heads):
    """Values next to the largest that are kept, 2^126, and next to the smallest steps."""
    g = gen(n + 1)
    for size in (2.0 ** 14,) if dtype == F16 else (2.0 ** 122, 2.0 ** -100):
        v = size * (torch.rand(n, 1, 64, generator=g, device="cuda") - 0.5)
        check_far_apart(*far_apart(g, dtype, n, heads, 16, v, []))
    if dtype != F16:  # both: the large ones without weight
        v = 2.0 ** -60 * randn(g, n, 1, 64)
        v[3] = 2.0 ** 120 * torch.rand(1, 64, generator=g, device="cuda")
        c, q, table, lens = far_apart(g, dtype, n, 1, 16, v, [(3, -200.0)])
        check_far_apart(c, q, table, lens)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("each,lens", [(2, [70]), (4, [9000, 5]), (8, [9000, 5])])
def test_queries_next_to_the_largest_numbers(dtype, each, lens):
    """Queries of 2^118 and a scale that brings their scores back."""
    g = gen(each)
    c, table, n = fill(g, lens, 16, 1, 64, 64, dtype)
    q = (2.0 ** 118 * randn(g, len(lens), each, 64)).to(dtype)
    check_attend(c, q, table, n, scale=2.0 ** -121)
