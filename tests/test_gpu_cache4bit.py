"""The 4-bit paged cache on the GPU: what it keeps against the definition, and
attention over it against 64 bits from what it keeps.

Tolerances count roundings and truncations.  eps(t)/2 of the result is the
output's own.  A score is a sum of exact products in the tensor cores, of at
most 16 instructions for a group, each of which may lose 2^-23 of what has been
added, and a few fp32 operations (2^-24 each): below 2^-18 of M, the sum of
|q| times the largest numbers that a key's codes stand for, which is below
15 step + |low|.  A relative error of a weight is one of its share in the
output twice (numerator and sum).  Weights enter the second product in two
16-bit parts (2^-22) or, for bfloat16, in one (2^-12), its sums lose what the
first's lose, and exp2 2^-22.
"""
import ctypes as C
import math

import pytest
import torch

import pyflame_b200 as pf
from pyflame_b200 import _native as N

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
HALF = {t: torch.finfo(t).eps / 2 for t in TYPES}
TINY = {F32: 0.0, F16: 2.0 ** -25, BF16: 0.0}  # half a step of fp16's subnormals
WEIGHT = {F32: 2.0 ** -18, F16: 2.0 ** -18, BF16: 2.0 ** -11}


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def within(got, want, tol, what=""):
    got = got.double()
    assert got.shape == want.shape, (got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    bad &= ~((got == want) | (got.isnan() & want.isnan()))  # infinities and NaN in the same places
    if bad.any():
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; first {i}: {got[i]} for {want[i]}, "
                             f"tolerance {torch.broadcast_to(torch.as_tensor(tol), got.shape)[i]}")


def kept(x, group):
    """(value, step, |low|) of the definition, x in float32, one operation at a time."""
    d, value, steps, lows = x.shape[-1], torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    for at in range(0, d, group):
        p = x[..., at:at + group]
        low = p.amin(-1, keepdim=True).bfloat16().float()
        step = ((p.amax(-1, keepdim=True) - low) * torch.tensor(1 / 15, dtype=F32, device=x.device)).bfloat16().float()
        step = torch.where(step < 2.0 ** -126, 0.0, step)
        code = ((p - low) * torch.where(step > 0, 1 / step, 0.0)).round().clamp(0, 15)
        value[..., at:at + group] = low + step * code
        steps[..., at:at + group] = step
        lows[..., at:at + group] = low.abs()
    return value, steps, lows


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=-12345.0), torch.nan_to_num(b, nan=-12345.0))


# ---------------------------------------------------------------------------
# what is kept
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,group,page,heads,tokens", [(128, 64, 16, 8, 37), (64, 32, 1, 3, 5), (8, 32, 7, 1, 1), (40, 64, 2, 2, 9),
                                                         (72, 32, 13, 5, 33), (80, 64, 16, 3, 8), (96, 128, 5, 2, 7), (104, 32, 32, 1, 65),
                                                         (128, 128, 3, 12, 4), (256, 32, 16, 2, 19), (200, 128, 4, 1, 3), (64, 128, 8, 2, 2)])
def test_append_and_read(dtype, dim, group, page, heads, tokens):
    g = gen(dim + group + tokens)
    pages = -(-tokens // page) + 2
    c = pf.PagedKVCache4bit(pages, page, heads, dim, group_size=group)
    k, v = (3 * randn(g, tokens, heads, dim, dtype=dtype) + 1 for _ in range(2))
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    if tokens > 2:
        slots[tokens // 2] = -1
    before = [t.clone() for t in (c.k, c.v, c.k_scales, c.v_scales)]
    c.append(k, v, slots)
    live = slots >= 0
    for got, x in zip(c.read(slots), (k, v)):
        want, step, low = kept(x.float(), group)
        assert same(got[live], want[live])
        assert not got[~live].any()
        # half a step, the scales' own rounding (2^-9 of 15 steps, 2^-9 of low), and fp32's
        within(got[live], x[live].double(), (0.53 * step + 2.0 ** -9 * low + 2.0 ** -20 * (low + 15 * step)).double()[live])
    for t in TYPES:  # rounded once
        for got, x in zip(c.read(slots, t), (k, v)):
            assert same(got[live], kept(x.float(), group)[0].to(t)[live])
    others = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    others[slots[live]] = False
    rest = others.nonzero()[:, 0]
    assert not any(t.any() for t in c.read(rest))  # what was not named is as it was
    assert all(a.shape == b.shape for a, b in zip(before, (c.k, c.v, c.k_scales, c.v_scales)))
    c.check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rot,heads,q_heads,tokens", [(128, 128, 8, 32, 9), (64, 64, 12, 12, 1), (80, 40, 3, 6, 33), (72, 36, 5, 5, 6),
                                                          (96, 96, 2, 0, 40), (256, 250, 1, 7, 3), (8, 2, 3, 3, 4), (64, 0, 2, 4, 5), (128, 24, 1, 40, 300)])
def test_append_rotated(dtype, layout, dim, rot, heads, q_heads, tokens):
    g = gen(dim + rot + tokens)
    r = pf.RotaryEmbedding(dim, rot, layout=layout, factor=1.25)
    qkv = randn(g, tokens, (q_heads + 2 * heads) * dim, dtype=dtype)
    q, k, v = (x.unflatten(1, (-1, dim)) if x.numel() else x.view(tokens, 0, dim)
               for x in qkv.split([q_heads * dim, heads * dim, heads * dim], 1))
    pos = torch.randint(0, 30000, (tokens,), generator=g, device="cuda")
    slots = torch.arange(tokens, device="cuda") + 3
    a = pos.double()[:, None] * r.inv_freq
    cos, sin = (f(a)[:, None] * r.factor for f in (torch.cos, torch.sin))

    def turned(x):
        y, x = x.double().clone(), x.double()
        i, j = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
        y[..., i] = x[..., i] * cos - x[..., j] * sin
        y[..., j] = x[..., i] * sin + x[..., j] * cos
        return y

    c = pf.PagedKVCache4bit(tokens + 9, 1, heads, dim, group_size=32)
    out = c.append(k, v, slots, positions=pos, rotary=r, q=q)
    got_k, got_v = c.read(slots)
    assert same(got_v, kept(v.float(), 32)[0])
    # in 64 bits up to the rounding to fp32: the same fp32 keys, the same codes
    assert same(got_k, kept(turned(k).float(), 32)[0])
    if q_heads:
        y = turned(q)
        # cosine and sine rounded to fp32, two products and a sum: 4 roundings of the magnitudes
        within(out, y, HALF[dtype] * y.abs() + 2.0 ** -21 * 1.25 * 2 * q.double().abs().amax() + TINY[dtype])


def test_the_factor_counts_in_64_bits():
    """Many keys, rotated with a factor that fp32 does not hold: one rounding to fp32, and so the same codes."""
    g = gen(31)
    r = pf.RotaryEmbedding(128, scaling={"type": "yarn", "factor": 8.0, "original_max_position": 4096})
    k, pos = randn(g, 6000, 8, 128, dtype=F16), torch.randint(0, 32768, (6000,), generator=g, device="cuda")
    c = pf.PagedKVCache4bit(375, 16, 8, 128)
    slots = torch.randperm(6000, generator=g, device="cuda")
    c.append(k, k, slots, positions=pos, rotary=r)
    a, x = pos.double()[:, None] * r.inv_freq, k.double()
    cos, sin = (f(a)[:, None] * r.factor for f in (torch.cos, torch.sin))
    turned = torch.cat((x[..., :64] * cos - x[..., 64:] * sin, x[..., :64] * sin + x[..., 64:] * cos), -1)
    # angles of up to 32768 in one 64-bit number are off by 2^-38: one key in 10^4 rounds to another fp32
    # number, and one in 10^5 of those to another code
    assert same(c.read(slots)[0], kept(turned.float(), 64)[0])


def test_queries_in_place_and_skipped_rows():
    g = gen(3)
    r = pf.RotaryEmbedding(64)
    for layout_width in (64, 68):  # rows of 16 bytes, and rows that are not
        c = pf.PagedKVCache4bit(4, 16, 2, 64)
        wide = randn(g, 7, 4, layout_width, dtype=BF16)
        q = wide[..., :64]
        k, v = randn(g, 7, 2, 64, dtype=BF16), randn(g, 7, 2, 64, dtype=BF16)
        slots = torch.tensor([5, -1, 6, 7, -3, 8, 9], device="cuda")
        pos = torch.arange(7, device="cuda") * 77
        apart = torch.full_like(q, 9.0)
        c.append(k, v, slots, positions=pos, rotary=r, q=q, q_out=apart)
        assert (apart[[1, 4]] == 9).all()
        keep = q.clone()
        assert c.append(k, v, slots, positions=pos, rotary=r, q=q, q_out=q) is q
        assert torch.equal(q[[1, 4]], keep[[1, 4]]) and torch.equal(q[[0, 2, 3, 5, 6]], apart[[0, 2, 3, 5, 6]])
        new = c.append(k, v, slots, positions=pos, rotary=r, q=keep)
        assert not new[[1, 4]].any() and torch.equal(new[0], q[0])


@pytest.mark.parametrize("dtype", TYPES)
def test_values_at_the_edges_of_the_types(dtype):
    """Constant groups, zeros, the smallest and the largest numbers, infinities and NaN."""
    top = {F32: 2.0 ** 126, BF16: 2.0 ** 126, F16: 65504.0}[dtype]
    x = torch.zeros(12, 1, 64, device="cuda")
    x[1] = 1.7  # constant
    x[2, 0, :32] = -top
    x[2, 0, 32:] = top
    x[3, 0, 5] = float("inf")
    x[4, 0, 40] = float("nan")
    x[5] = torch.linspace(-1e-30, 1e-30, 64)
    x[6, 0, 0] = 2.0 ** -130
    x[7] = 1000 + torch.linspace(0, 1, 64)  # far from 0: low's rounding counts
    x[8, 0, 63] = -float("inf")
    x[9] = -5.0
    x[10] = torch.linspace(-top, -top / 2, 64)
    if dtype == F32:
        x[11, 0, 3] = 1.5 * 2.0 ** 126  # above what a group may hold
    x = x.to(dtype)
    c = pf.PagedKVCache4bit(1, 16, 1, 64, group_size=32)
    slots = torch.arange(12, device="cuda")
    c.append(x, x.flip(0), slots)
    want = kept(x.float(), 32)[0]
    for row, group in [(3, 0), (4, 1), (8, 1)] + ([(11, 0)] if dtype == F32 else []):
        want[row, 0, 32 * group:32 * group + 32] = float("nan")
    k, v = c.read(slots)
    assert same(k, want) and same(v, want.flip(0))


def test_append_twice_and_moved_pages():
    g = gen(4)
    c = pf.PagedKVCache4bit(6, 5, 3, 96, group_size=32)
    a, b = randn(g, 30, 3, 96), randn(g, 30, 3, 96)
    slots = torch.arange(30, device="cuda")
    c.append(a, b, slots)
    c.append(b[3:9], a[3:9], slots[3:9])  # overwritten, neighbours in the same words too
    k, v = c.read(slots)
    want_k, want_v = a.clone(), b.clone()
    want_k[3:9], want_v[3:9] = b[3:9], a[3:9]
    assert same(k, kept(want_k, 32)[0]) and same(v, kept(want_v, 32)[0])
    for t in (c.k, c.v, c.k_scales, c.v_scales):
        t[5].copy_(t[1])
    k2, v2 = c.read(torch.arange(25, 30, device="cuda"))
    assert same(k2, k[5:10]) and same(v2, v[5:10])


def test_slots_outside_are_skipped_and_reported():
    c = pf.PagedKVCache4bit(2, 4, 1, 64)
    x = torch.ones(3, 1, 64, device="cuda")
    c.append(x, x, torch.tensor([0, 8, 1 << 40], device="cuda"))
    with pytest.raises(N.PfcError, match="4-bit"):
        c.check()
    c.check()
    k, _ = c.read(torch.tensor([0, 9, -5, -(1 << 60)], device="cuda"))
    assert k[0].all() and not k[1:].any()
    with pytest.raises(N.PfcError):
        c.check()
    assert not c.read(torch.arange(1, 8, device="cuda"))[0].any()


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def fill(g, lens, page, heads, dim, group, dtype, outliers=True):
    """A cache of sequences of these lengths with shuffled pages, and its block table."""
    need = [-(-n // page) for n in lens]
    pages, most = sum(need) + 2, max(1, max(need))
    c = pf.PagedKVCache4bit(pages, page, heads, dim, group_size=group)
    k, v = (randn(g, pages * page, heads, dim, dtype=dtype) for _ in range(2))
    if outliers:
        k[..., ::17] += 3
    c.append(k, v, torch.arange(pages * page, device="cuda"))
    table = torch.full((len(lens), most), 1 << 30, dtype=torch.int32)  # entries behind the length are not looked at
    order, at = torch.randperm(pages, generator=g, device="cuda").int().cpu(), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return c, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")


def reference(c, q, table, lens, scale, window):
    """(out, lse, tolerances' parts) in 64 bits from what the cache holds."""
    b, h, d = q.shape
    each, page = h // c.num_heads, c.page_size
    out = torch.zeros(b, h, d, dtype=torch.float64, device="cuda")
    lse = torch.full((b, h), -math.inf, dtype=torch.float64, device="cuda")
    errs, mags = torch.zeros(b, h, dtype=torch.float64, device="cuda"), torch.zeros(b, h, d, dtype=torch.float64, device="cuda")

    def bound(x):  # 15 step + |low| of each value is at most twice the range and the least of its group
        p = torch.nn.functional.pad(x, (0, -d % c.group_size)).unflatten(-1, (-1, c.group_size))
        return (2 * (p.amax(-1) - p.amin(-1)) + 2 * p.abs().amax(-1)).repeat_interleave(c.group_size, -1)[..., :d]

    for i, n in enumerate(lens.tolist()):
        j = torch.arange(max(0, n - window) if window else 0, n, device="cuda")
        if not len(j):
            continue
        slots = table[i, j // page].long() * page + j % page
        k, v = (x.double().transpose(0, 1) for x in c.read(slots))  # [heads, keys, dim]
        qi = q[i].double().view(c.num_heads, each, d)
        s = qi @ k.transpose(1, 2) * scale
        lse[i] = torch.logsumexp(s, -1).flatten()
        p = torch.softmax(s, -1)
        out[i] = (p @ v).flatten(0, 1)
        e = abs(scale) * (qi.abs() @ bound(k).transpose(1, 2)) * 2.0 ** -18
        errs[i] = e.amax(-1).flatten()
        mags[i] = (p @ bound(v)).flatten(0, 1)
    return out, lse, errs, mags


def check_attend(c, q, table, lens, scale=None, window=0, **kw):
    t, real = q.dtype, 1 / math.sqrt(q.shape[-1]) if scale is None else scale
    got, got_lse = c.attend(q, table, lens, scale=scale, window=window, return_lse=True, **kw)
    out, lse, errs, mags = reference(c, q, table, lens, real, window)
    within(got, out, HALF[t] * out.abs() + TINY[t] + (2 * errs[..., None] + WEIGHT[t]) * mags, "out")
    within(got_lse, lse, errs + 2.0 ** -20 + 2.0 ** -22 * lse.abs().nan_to_num(posinf=0.0), "lse")
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,group,page,heads,each,lens", [
    (128, 64, 16, 2, 4, [1, 0, 15, 16, 17, 129, 64]), (64, 32, 16, 3, 1, [333]), (80, 64, 13, 2, 5, [0, 1, 40, 200]), (128, 32, 32, 1, 8, [700, 5]),
    (128, 128, 64, 1, 9, [300, 0, 64]), (96, 128, 1, 2, 2, [31, 33]), (96, 64, 48, 2, 3, [100, 250]), (72, 32, 7, 1, 16, [55]),
    (256, 64, 16, 1, 2, [150, 16]), (256, 32, 5, 2, 1, [77]), (8, 32, 2, 4, 3, [9, 64, 1]), (40, 64, 80, 1, 40, [90]), (200, 128, 16, 1, 1, [130]),
    (64, 64, 3, 12, 1, [64, 65, 127, 128])])
def test_attend(dtype, dim, group, page, heads, each, lens):
    g = gen(dim + group + page)
    c, table, n = fill(g, lens, page, heads, dim, group, dtype)
    q = randn(g, len(lens), heads * each, dim, dtype=dtype)
    check_attend(c, q, table, n)
    c.check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page,window", [(16, 1), (16, 100), (13, 64), (32, 1000), (1, 7), (16, 17), (7, 1 << 40)])
def test_window(dtype, page, window):
    g = gen(page)
    c, table, n = fill(g, [0, 1, 64, 100, 333], page, 2, 64, 32, dtype)
    check_attend(c, randn(g, 5, 6, 64, dtype=dtype), table, n, window=window)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [16, 10])
def test_many_sequences_share_ctas(dtype, page):
    """More sequences than a CTA has threads, and lengths from 0 on: units begin and end inside CTAs' runs."""
    g = gen(9)
    lens = [(i * 37) % 300 for i in range(150)]
    c, table, n = fill(g, lens, page, 2, 64, 64, dtype)
    check_attend(c, randn(g, 150, 4, 64, dtype=dtype), table, n)


@pytest.mark.parametrize("dtype", TYPES)
def test_long_sequence(dtype):
    g = gen(10)
    c, table, n = fill(g, [40000, 3], 64, 1, 128, 64, dtype)
    check_attend(c, randn(g, 2, 8, 128, dtype=dtype), table, n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,group,page,heads,each,lens", [
    (128, 64, 7, 1, 2, [20011, 0, 696]), (64, 32, 16, 2, 1, [0, 17001]), (96, 64, 48, 1, 9, [9000, 1, 0, 12345]),
    (256, 64, 5, 1, 1, [8000]), (8, 32, 1, 3, 1, [9000, 8999]), (128, 64, 16, 21, 1, [9001, 0, 12000]), (128, 64, 16, 22, 1, [9001, 0, 12000]),
    (128, 64, 16, 16, 1, [9001, 700]), (128, 64, 16, 11, 1, [9001, 0, 7000])])
def test_few_sequences_of_many_shares(dtype, dim, group, page, heads, each, lens):
    """Units that most of the device's CTAs share, empty sequences among them."""
    g = gen(dim + page + heads)
    c, table, n = fill(g, lens, page, heads, dim, group, dtype)
    q = randn(g, len(lens), heads * each, dim, dtype=dtype)
    assert torch.equal(check_attend(c, q, table, n), c.attend(q, table, n))
    c.check()


@pytest.mark.parametrize("dtype", TYPES)
def test_sharp_scores_and_scales(dtype):
    """Weights of one key alone, maxima that rise all the way, negative and zero scales."""
    g = gen(11)
    c, table, n = fill(g, [500, 130], 16, 2, 64, 32, dtype)
    q = randn(g, 2, 4, 64, dtype=dtype)
    for scale in (3.0, -0.125, 0.0, 1e-3):
        check_attend(c, q, table, n, scale=scale)
    ramp = torch.linspace(-20, 20, 512, device="cuda").flip(0)
    for order in (ramp, ramp.flip(0)):
        c = pf.PagedKVCache4bit(32, 16, 1, 64, group_size=64)
        k = order[:, None, None] * torch.ones(512, 1, 64, device="cuda") + randn(g, 512, 1, 64) * 0.1
        c.append(k.to(dtype), randn(g, 512, 1, 64, dtype=dtype), torch.arange(512, device="cuda"))
        table = torch.arange(32, dtype=torch.int32, device="cuda")[None]
        check_attend(c, torch.ones(1, 3, 64, device="cuda", dtype=dtype), table, torch.tensor([512], dtype=torch.int32, device="cuda"), scale=0.05)


@pytest.mark.parametrize("dtype", TYPES)
def test_steps_of_very_different_sizes(dtype):
    """A step of values is scaled by the largest so far: keys with small ones still count in their own dimensions' sums."""
    g = gen(12)
    c = pf.PagedKVCache4bit(16, 16, 1, 64, group_size=32)
    size = torch.logspace(-3, 3, 256, device="cuda").flip(0)[:, None, None]
    if dtype == F16:
        size = size.clamp(max=900)
    c.append(randn(g, 256, 1, 64, dtype=dtype), (randn(g, 256, 1, 64) * size).to(dtype), torch.arange(256, device="cuda"))
    table = torch.randperm(16, generator=g, device="cuda").int()[None]
    check_attend(c, randn(g, 1, 2, 64, dtype=dtype), table, torch.tensor([256], dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("dtype", TYPES)
def test_large_and_small_queries(dtype):
    g = gen(13)
    c, table, n = fill(g, [70], 16, 1, 64, 64, dtype)
    q = randn(g, 1, 4, 64, dtype=dtype)
    q[0, 1] *= 3e4 if dtype == F16 else 1e20
    q[0, 2] *= 1e-4 if dtype == F16 else 1e-30
    q[0, 3] = 0
    q = q.clamp(-65504, 65504) if dtype == F16 else q
    big = 1.0 if dtype == F16 else 1e-16
    check_attend(c, q, table, n, scale=big * 1e-4)


@pytest.mark.parametrize("page", [16, 5])
def test_what_is_not_seen_has_no_effect(page):
    """NaN and infinities in unseen slots of seen pages, in other pages, and in other sequences."""
    g = gen(14)
    lens = [37, 0, 16, 50]
    for dtype in TYPES:
        c, table, n = fill(g, lens, page, 2, 64, 32, dtype)
        q = randn(g, 4, 4, 64, dtype=dtype)
        for window in (0, 9):
            want, lse = c.attend(q, table, n, window=window, return_lse=True)
            seen = torch.zeros(c.num_pages * page, dtype=torch.bool, device="cuda")
            for i, m in enumerate(lens):
                j = torch.arange(max(0, m - window) if window else 0, m, device="cuda")
                seen[table[i, j // page].long() * page + j % page] = True
            rest = (~seen).nonzero()[:, 0]
            bad = torch.full((len(rest), 2, 64), float("nan"), device="cuda", dtype=dtype)
            keep = [t.clone() for t in (c.k, c.v, c.k_scales, c.v_scales)]
            c.append(bad, bad, rest)
            got, got_lse = c.attend(q, table, n, window=window, return_lse=True)
            assert torch.equal(got, want) and torch.equal(got_lse, lse)
            for t, o in zip((c.k, c.v, c.k_scales, c.v_scales), keep):
                t.copy_(o)
        c.check()


@pytest.mark.parametrize("page", [16, 6])
def test_bad_pages_and_lengths(page):
    """They are skipped and reported; the rest of the sequence counts."""
    g = gen(15)
    c, table, n = fill(g, [4 * page, 40], page, 1, 64, 64, F16)
    q = randn(g, 2, 2, 64, dtype=F16)
    bad = table.clone()
    bad[0, 1] = c.num_pages
    bad[0, 2] = -1
    got = c.attend(q, bad, n)
    with pytest.raises(N.PfcError):
        c.check()
    slots = torch.cat([table[0, i].long() * page + torch.arange(page, device="cuda") for i in (0, 3)])
    k, v = (x[:, 0].double() for x in c.read(slots))
    want = torch.softmax(q[0].double() @ k.T / 8, -1) @ v
    within(got[0], want, HALF[F16] * want.abs() + 2.0 ** -14 * v.abs().amax())
    for wrong in (-1, 1 << 30):
        c.attend(q, table, torch.tensor([page, wrong], dtype=torch.int32, device="cuda"))
        with pytest.raises(N.PfcError):
            c.check()


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(dtype):
    g = gen(16)
    c, table, n = fill(g, [100, 7, 300], 16, 2, 64, 64, dtype)
    q = randn(g, 3, 4, 64, dtype=dtype)
    want = c.attend(q, table, n)
    wide = torch.zeros(5, 3, 4, 96, device="cuda", dtype=dtype)
    view = wide.permute(1, 2, 0, 3)[:, :, 2, 3:67]  # neither dense nor aligned
    view.copy_(q)
    assert torch.equal(c.attend(view, table, n), want)
    out = torch.empty_like(wide)[:, :, :, :64].permute(1, 2, 0, 3)[:, :, 1]
    assert c.attend(q, table, n, out=out) is out and torch.equal(out, want)
    padded = torch.full((3, table.shape[1] + 9), -7, dtype=torch.int32, device="cuda")
    padded[:, :table.shape[1]] = table
    assert torch.equal(c.attend(q, padded[:, :table.shape[1]], n), want)
    inside = q.clone()
    assert torch.equal(c.attend(inside, table, n, out=inside), want)
    assert c.attend(q[:0], table[:0], n[:0]).shape == (0, 4, 64)
    none = c.attend(q, table[:, :0], torch.zeros_like(n))
    assert not none.any()


@pytest.mark.parametrize("page", [16, 15])
def test_places_beyond_32_bits(page):
    """A cache of 9 GB of keys' codes and as much of values': tokens at both ends of it."""
    g = gen(19)
    pages = (1 << 25) // page
    c = pf.PagedKVCache4bit(pages, page, 2, 256, group_size=128)
    assert c.k.numel() * 4 > 1 << 32 and c.v.numel() * 4 > 1 << 32
    table = torch.tensor([[pages - 1, 0, pages - 2, pages // 2]], dtype=torch.int32, device="cuda")
    n = 4 * page - 3
    j = torch.arange(n, device="cuda")
    slots = table[0, j // page].long() * page + j % page
    k, v = randn(g, n, 2, 256, dtype=F16), randn(g, n, 2, 256, dtype=F16)
    c.append(k, v, slots)
    got = c.read(slots)
    assert same(got[0], kept(k.float(), 128)[0]) and same(got[1], kept(v.float(), 128)[0])
    check_attend(c, randn(g, 1, 4, 256, dtype=F16), table, torch.tensor([n], dtype=torch.int32, device="cuda"))
    c.check()


def test_same_bits_streams_and_graphs():
    """The same call gives the same bits: again, on another stream while it runs, captured and replayed with new data."""
    g = gen(17)
    c, table, n = fill(g, [900, 40, 2000, 0], 16, 2, 128, 64, BF16)
    q = [randn(g, 4, 8, 128, dtype=BF16) for _ in range(2)]
    want = [c.attend(x, table, n) for x in q]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = c.attend(q[i], table, n)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs, ins = [], [], [x.clone() for x in q]
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(c.attend(ins[i], table, n))
        graphs.append(graph)
    ins[0].copy_(q[1])
    ins[1].copy_(q[0])
    torch.cuda.synchronize()
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            graphs[i].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[1]) and torch.equal(outs[1], want[0])


def test_append_attend_captured():
    g = gen(18)
    c = pf.PagedKVCache4bit(8, 16, 2, 64)
    r = pf.RotaryEmbedding(64)
    qkv, slots, pos = randn(g, 2, 8 * 64, dtype=F16), torch.tensor([0, 64], device="cuda"), torch.tensor([0, 0], device="cuda")
    table = torch.tensor([[0, 1, 2, 3], [4, 5, 6, 7]], dtype=torch.int32, device="cuda")
    n = torch.tensor([1, 1], dtype=torch.int32, device="cuda")

    def step():
        q, k, v = qkv.unflatten(1, (-1, 64)).split([4, 2, 2], 1)
        q = c.append(k, v, slots, positions=pos, rotary=r, q=q)
        return c.attend(q, table, n)

    for _ in range(3):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(20):
        qkv.copy_(randn(g, 2, 8 * 64, dtype=F16))
        slots.copy_(torch.tensor([i, 64 + i], device="cuda"))
        pos.fill_(i)
        n.fill_(i + 1)
        graph.replay()
        torch.cuda.synchronize()
        q = r.apply(qkv.unflatten(1, (-1, 64))[:, :4], pos)
        want, _, errs, mags = reference(c, q, table, n, 0.125, 0)
        # the queries are rounded once more or less than the call's own: a step of fp16 in each
        within(out, want, HALF[F16] * want.abs() + (2 * errs[..., None] + 2.0 ** -10) * mags)
    c.check()


def test_refusals():
    c = pf.PagedKVCache4bit(4, 16, 2, 64)
    k, slots = torch.zeros(3, 2, 64, device="cuda"), torch.arange(3, device="cuda")
    q, table, n = torch.zeros(1, 4, 64, device="cuda"), torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    r = pf.RotaryEmbedding(64)
    for bad, err in [(dict(k=k.double()), TypeError), (dict(v=k.half()), TypeError), (dict(k=k[:, :1]), ValueError), (dict(v=k[:2]), ValueError),
                     (dict(slots=slots.int()), TypeError), (dict(slots=slots.cpu()), ValueError), (dict(positions=slots), ValueError),
                     (dict(rotary=r), ValueError), (dict(q_out=q), ValueError), (dict(k=k.transpose(1, 2).contiguous().transpose(1, 2)), ValueError),
                     (dict(positions=slots, rotary=pf.RotaryEmbedding(32)), ValueError), (dict(k=k.clone().requires_grad_()), RuntimeError)]:
        with pytest.raises(err):
            c.append(**{**dict(k=k, v=k, slots=slots), **bad})
    x = torch.zeros(3, 4, 64, device="cuda")
    with pytest.raises(ValueError, match="shares memory"):
        c.append(x[:, :2], x[:, 2:], slots, q=x[:, :2], q_out=x[:, 1:3])
    with pytest.raises(ValueError, match="cache"):
        c.attend(q, table, n, out=c.k.view(torch.float32).view(-1)[:256].view(1, 4, 64))
    for bad, err in [(dict(q=q[0]), ValueError), (dict(q=q[:, :3]), ValueError), (dict(q=q[..., :32]), ValueError), (dict(q=q.double()), TypeError),
                     (dict(block_table=table.long()), TypeError), (dict(seq_lens=n.long()), TypeError), (dict(block_table=table[0]), ValueError),
                     (dict(window=-1), ValueError), (dict(scale=float("nan")), N.PfcError), (dict(out=q[:, :2]), ValueError),
                     (dict(out=q.half()), TypeError), (dict(q=q.cpu()), ValueError), (dict(q=q.clone().requires_grad_()), RuntimeError)]:
        with pytest.raises(err):
            c.attend(**{**dict(q=q, block_table=table, seq_lens=n), **bad})
    with pytest.raises(TypeError):
        c.read(slots.int())
    with pytest.raises(TypeError):
        c.read(slots, torch.float64)
    with pytest.raises(N.PfcError):
        pf.PagedKVCache4bit(4, 16, 2, 60)
    with pytest.raises(N.PfcError):
        pf.PagedKVCache4bit(4, 16, 2, 64, group_size=48)
    with torch.inference_mode():
        made = pf.PagedKVCache4bit(4, 16, 2, 64)
    made.append(k, k, slots)
    made.append(k, k, slots + 1000)
    with pytest.raises(N.PfcError):
        made.check()


def test_workspace_is_checked():
    c = pf.PagedKVCache4bit(200, 64, 8, 128)
    L = N.lib()
    q, table = torch.zeros(8, 32, 128, device="cuda"), torch.zeros(8, 50, dtype=torch.int32, device="cuda")
    n, need = torch.full((8,), 3000, dtype=torch.int32, device="cuda"), C.c_size_t(0)
    out = torch.empty_like(q)
    p = N.Cache4AttentionParamsC(c._c, 0, 8, 32, q.data_ptr(), 4096, 128, out.data_ptr(), 4096, 128, None, table.data_ptr(), 50, 50, n.data_ptr(), 0, 0.1)
    assert L.pfk_cache4_attention_workspace(C.byref(p), C.byref(need)) == 0 and need.value > 0
    work = torch.empty(need.value + 16, dtype=torch.uint8, device="cuda")
    for at, size in ((None, need.value), (work.data_ptr(), need.value - 1), (work.data_ptr() + 8, need.value)):
        p.workspace, p.workspace_bytes = at, size
        assert L.pfk_cache4_attention(C.byref(p), None) == -1 and b"workspace" in L.pfc_last_error()
