"""Token-generation operators on the GPU against plain implementations in 64
bits, at the sizes, layouts and masks where they can go wrong.

Tolerances count roundings.  eps(t)/2 of the result is the output's own.  The
rest happens in fp32 (2^-24 a rounding, 2^-23 an addition inside a tensor-core
instruction, which truncates) and is scaled by the sum of the magnitudes that
were added, computed in 64 bits.
"""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import pyflame_b200 as pf

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
HALF = {t: torch.finfo(t).eps / 2 for t in TYPES}
TINY = {F32: 0.0, F16: 2.0 ** -25, BF16: 0.0}  # half a step of fp16's subnormals


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


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------

def turn(x, positions, rot, sign=1):
    """x [..., tokens, heads, dim] rotated in 64 bits, and the sum of magnitudes of each result's terms."""
    x, r = x.double(), rot.rotary_dim
    a = sign * positions.double()[..., None] * rot.inv_freq
    c, s = (f(a).unsqueeze(-2) * rot.factor for f in (torch.cos, torch.sin))
    y, mag = x.clone(), torch.zeros_like(x)
    i, j = (slice(0, r // 2), slice(r // 2, r)) if rot.layout == "half" else (slice(0, r, 2), slice(1, r, 2))
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., i] * s + x[..., j] * c
    mag[..., i] = mag[..., j] = (x[..., i].abs() + x[..., j].abs()) * abs(rot.factor)
    return y, mag


def turn_tol(y, mag, t):
    # the angle rounded to 2^-24 of half a turn (pi 2^-24), cosine and sine to 2 ulp (2^-22 of 1), their factor, two
    # products and a sum (3 2^-24): below 2^-21 of the magnitudes
    return HALF[t] * y.abs() + 2.0 ** -21 * mag + TINY[t]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rot,heads,tokens", [(64, 64, 12, 5), (128, 128, 3, 33), (128, 64, 2, 9), (80, 80, 5, 7), (72, 36, 1, 1),
                                                  (7, 6, 3, 4), (2, 2, 1, 1), (5, 0, 2, 3), (256, 16, 1, 300), (1024, 1024, 2, 3),
                                                  (100, 20, 4, 6), (64, 64, 65, 2)])
def test_rope(dtype, layout, dim, rot, heads, tokens):
    g = gen(dim + heads)
    x = randn(g, tokens, heads, dim, dtype=dtype)
    pos = torch.randint(-1000, 1 << 20, (tokens,), generator=g, device="cuda")
    r = pf.RotaryEmbedding(dim, rot, layout=layout)
    y, mag = turn(x, pos, r)
    got = r.apply(x, pos)
    within(got, y, turn_tol(y, mag, dtype))
    assert torch.equal(got[..., rot:], x[..., rot:])
    dx, mag = turn(x, pos, r, -1)
    within(r.backward(x, pos), dx, turn_tol(dx, mag, dtype), "backward")
    inplace = x.clone()
    assert r.apply(inplace, pos, out=inplace) is inplace and torch.equal(inplace, got)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scaling", [{"type": "linear", "factor": 8}, {"type": "ntk", "factor": 8},
                                     {"type": "yarn", "factor": 8, "original_max_position": 4096}])
def test_rope_scaled_far_positions(dtype, scaling):
    g = gen(3)
    r = pf.RotaryEmbedding(64, scaling=scaling)
    pos = torch.tensor([0, 1, 4095, 4096, 32767, 10 ** 6, 10 ** 7 + 1], device="cuda")
    x = randn(g, len(pos), 3, 64, dtype=dtype)
    y, mag = turn(x, pos, r)
    within(r.apply(x, pos), y, turn_tol(y, mag, dtype))
    assert r.factor == (pytest.approx(0.1 * math.log(8) + 1) if scaling["type"] == "yarn" else 1.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_rope_batches_and_strides(dtype):
    g = gen(4)
    r = pf.RotaryEmbedding(40, 24, layout="interleaved")
    pos = torch.randint(0, 5000, (3, 11), generator=g, device="cuda")
    for x in (randn(g, 3, 11, 5, 40, dtype=dtype), randn(g, 3, 5, 11, 40, dtype=dtype).transpose(1, 2),
              randn(g, 3, 11, 15, 41, dtype=dtype)[:, :, 2::3, 1:], randn(g, 1, 11, 1, 40, dtype=dtype).expand(3, 11, 5, 40)):
        for p in (pos, pos.t().contiguous().t(), pos[0], pos[:, ::1][1]):
            y, mag = turn(x, p, r)
            within(r.apply(x, p), y, turn_tol(y, mag, dtype))
    # an output inside a larger one: what lies around stays as it was
    big = torch.full((3, 13, 5, 44), 7.0, device="cuda", dtype=dtype)
    x = randn(g, 3, 11, 5, 40, dtype=dtype)
    y, mag = turn(x, pos, r)
    r.apply(x, pos, out=big[:, 1:12, :, 3:43])
    within(big[:, 1:12, :, 3:43], y, turn_tol(y, mag, dtype))
    big[:, 1:12, :, 3:43] = 7.0
    assert bool((big == 7).all())


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_gradient_by_differences(layout):
    g = gen(5)
    r = pf.RotaryEmbedding(16, 12, layout=layout, factor=1.5)
    x, d, w = (randn(g, 9, 3, 16) for _ in range(3))
    pos = torch.arange(9, device="cuda") * 977
    grad = r.backward(w, pos).double()
    # the map is linear: the difference over +-d is the derivative along d, up to the roundings of three applications
    f = [(r.apply(x + s * d, pos).double() * w.double()).sum() for s in (1, -1)]
    mag = ((x.abs() + d.abs()).double().sum() * 3 * w.abs().double().amax())
    assert abs((f[0] - f[1]) / 2 - (grad * d.double()).sum()) <= 2.0 ** -20 * mag


def test_rope_nothing_to_do():
    r = pf.RotaryEmbedding(8)
    for shape in ((0, 2, 8), (3, 0, 8), (0, 4, 2, 8), (2, 0, 2, 8)):
        assert r.apply(torch.zeros(shape, device="cuda"), torch.zeros(shape[-3], dtype=torch.int64, device="cuda")).shape == shape


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------

def new_cache(g, pages, page, heads, dim, dtype, tokens_first=True):
    shape = (pages, page, heads, dim) if tokens_first else (pages, heads, page, dim)
    k, v = (randn(g, *shape, dtype=dtype) for _ in range(2))
    return pf.PagedKVCache.from_tensors(*((k, v) if tokens_first else (k.transpose(1, 2), v.transpose(1, 2))))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,page,heads,q_heads,dim,rot,tokens_first", [
    (1, 16, 12, 12, 64, 64, True), (37, 7, 2, 10, 72, 36, True), (130, 1, 1, 1, 128, 128, True), (5, 64, 3, 0, 8, 0, True),
    (64, 16, 8, 32, 128, 64, False), (9, 5, 1, 3, 6, 2, True), (3, 4, 2, 2, 5, 4, False), (1000, 16, 2, 4, 32, 32, True)])
def test_append(dtype, tokens, page, heads, q_heads, dim, rot, tokens_first):
    g = gen(tokens)
    pages = tokens // page + 3
    cache = new_cache(g, pages, page, heads, dim, dtype, tokens_first)
    r = pf.RotaryEmbedding(dim, rot)
    qkv = randn(g, tokens, (q_heads + 2 * heads) * dim, dtype=dtype)
    q, k, v = (x.unflatten(1, (-1, dim)) if x.shape[1] else x.view(tokens, 0, dim)
               for x in qkv.split([q_heads * dim, heads * dim, heads * dim], 1))
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    slots[tokens // 2:: 4] = -1
    pos = torch.randint(0, 100000, (tokens,), generator=g, device="cuda")
    want_k, want_v, live = cache.k.double(), cache.v.clone(), slots >= 0
    (ky, km), (qy, qm) = turn(k, pos, r), turn(q, pos, r)
    at = slots[live]
    tol = torch.zeros_like(want_k)
    want_k[at // page, at % page] = ky[live]
    tol[at // page, at % page] = turn_tol(ky, km, dtype)[live]
    want_v[at // page, at % page] = v[live]
    out = cache.append(k, v, slots, positions=pos, rotary=r, q=q)
    within(cache.k, want_k, tol, "keys")
    assert torch.equal(cache.v, want_v)
    within(out, qy * live[:, None, None], turn_tol(qy, qm, dtype), "queries")
    kept = q.clone()
    kept[live] = out[live]
    cache.append(k, v, slots, positions=pos, rotary=r, q=q, q_out=q)  # in place, inside the projection's output
    assert torch.equal(q, kept)  # rows of skipped tokens stay
    cache.check()


@pytest.mark.parametrize("dtype", TYPES)
def test_append_as_it_is_and_bad_slots(dtype):
    g = gen(1)
    cache = new_cache(g, 4, 16, 2, 24, dtype)
    k, v = randn(g, 5, 2, 24, dtype=dtype), randn(g, 5, 2, 24, dtype=dtype)
    v[0, 0, 0], v[1, 1, 3], k[2, 0, 1] = math.nan, math.inf, -math.inf
    want_k, want_v = cache.k.clone(), cache.v.clone()
    slots = torch.tensor([63, 0, 17, 64, 1 << 40], device="cuda")
    for i in range(3):
        s = int(slots[i])
        want_k[s // 16, s % 16], want_v[s // 16, s % 16] = k[i], v[i]
    assert cache.append(k, v, slots) is None
    bits = torch.int32 if dtype == F32 else torch.int16
    assert torch.equal(cache.k.view(bits), want_k.view(bits)) and torch.equal(cache.v.view(bits), want_v.view(bits))
    with pytest.raises(pf._native.PfcError):
        cache.check()
    cache.check()  # raised once
    cache.append(k[:0], v[:0], slots[:0])
    cache.append(k, v, torch.full((5,), -7, device="cuda"))
    cache.check()
    assert torch.equal(cache.k.view(bits), want_k.view(bits))


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def make_batch(g, lens, page, heads, q_heads, dim, dtype, tokens_first=True, spoil=True):
    """A cache with the sequences' pages in random order.  Everything that no sequence sees is NaN, and the table's
    unused entries name no page."""
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 2
    cache = new_cache(g, pages, page, heads, dim, dtype, tokens_first)
    table = torch.full((len(lens), max(need, default=0) + 2), -1, dtype=torch.int32)
    free = torch.randperm(pages, generator=g, device="cuda").tolist()
    seen = torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for i in range(need[b]):
            p = free.pop()
            table[b, i] = p
            seen[p, :min(page, n - i * page)] = True
    if spoil:
        cache.k[~seen.cuda()] = math.nan
        cache.v[~seen.cuda()] = math.nan
    q = randn(g, len(lens), q_heads, dim, dtype=dtype)
    return cache, q, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")


def attention(cache, q, table, lens, window=0, scale=None):
    """(out, lse) in 64 bits with the tolerance of each."""
    t, page = q.dtype, cache.page_size
    b, h, d = q.shape
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(b, h, d, dtype=torch.float64, device="cuda")
    lse = torch.full((b, h), -math.inf, dtype=torch.float64, device="cuda")
    tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
    for i, n in enumerate(lens.tolist()):
        j = torch.arange(max(0, n - window) if window else 0, n, device="cuda")
        if len(j) == 0:
            continue
        at = table[i, j // page].long()
        k, v = (x[at, j % page].double().transpose(0, 1) for x in (cache.k, cache.v))  # [heads, keys, d]
        qq = q[i].double().unflatten(0, (cache.num_heads, -1))
        s = qq @ k.transpose(1, 2) * scale
        p = torch.softmax(s, -1)
        out[i] = (p @ v).flatten(0, 1)
        lse[i] = torch.logsumexp(s, -1).flatten()
        # a score: d products summed eight or sixteen at a time; in fp32 each also split (3 2^-22)
        es = ((qq.abs() @ k.abs().transpose(1, 2)).amax(-1) * abs(scale) *
              ((d / 8 + 8) * 2.0 ** -23 + (3 * 2.0 ** -22 if t == F32 else 0)))
        ep = es + 2.0 ** -21 * (1 + s.abs().amax(-1))  # the weight: its argument's roundings, and exp2
        add = (len(j) / 64 + 64) * 2.0 ** -23  # a warp adds 16 keys at a time, every fourth 16 of them; then the joins
        split = 3 * 2.0 ** -22 if t == F32 else 2.0 ** -16
        tol[i] = HALF[t] * out[i].abs() + ((2 * ep + add + split)[..., None] * (p @ v.abs())).flatten(0, 1) + TINY[t]
        lse_tol[i] = (ep + add).flatten() + 2.0 ** -22 * lse[i].abs()
    return out, lse, tol, lse_tol


def tables(table, page):
    """The table as it is, and one with room for long sequences: the kernels share their work in another way."""
    wide = torch.full((table.shape[0], table.shape[1] + 100000 // page), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    return table, wide


LENS = {
    "one": [1], "edges": [15, 16, 17, 63, 64, 65, 128, 0, 1], "empty": [0], "empties": [0, 0, 5, 0], "long": [5000],
    "ragged": [3, 700, 0, 129, 2048, 64, 1], "many": [(i * 37) % 90 for i in range(300)],
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,page,heads,q_heads,dim,window", [
    ("one", 16, 2, 2, 64, 0), ("edges", 16, 3, 3, 64, 0), ("edges", 1, 1, 8, 128, 0), ("edges", 13, 2, 10, 80, 0),
    ("edges", 64, 1, 9, 64, 33), ("empty", 16, 2, 4, 64, 0), ("empties", 7, 1, 1, 8, 0), ("long", 16, 2, 16, 128, 0),
    ("long", 32, 1, 17, 128, 0), ("long", 16, 1, 40, 64, 1000), ("ragged", 16, 8, 32, 128, 0), ("ragged", 100, 4, 4, 72, 0),
    ("ragged", 16, 2, 2, 256, 0), ("ragged", 16, 1, 12, 192, 100), ("ragged", 32, 2, 6, 16, 1), ("many", 16, 2, 4, 64, 0),
    ("many", 3, 1, 2, 96, 20)])
def test_attend(dtype, lens, page, heads, q_heads, dim, window):
    g = gen(page + dim)
    cache, q, table, n = make_batch(g, LENS[lens], page, heads, q_heads, dim, dtype)
    out, lse, tol, lse_tol = attention(cache, q, table, n, window)
    for t in tables(table, page):
        got, got_lse = cache.attend(q, t, n, window=window, return_lse=True)
        within(got, out, tol, "out")
        within(got_lse, lse, lse_tol, "lse")
        again = cache.attend(q, t, n, window=window)
        assert torch.equal(again, got)  # shares are joined in one order
    cache.check()


@pytest.mark.parametrize("dtype", TYPES)
def test_attend_strides_and_layouts(dtype):
    g = gen(8)
    cache, q, table, n = make_batch(g, LENS["ragged"], 16, 2, 8, 64, dtype, tokens_first=False)
    wide = torch.zeros(7, 3, 11, 69, device="cuda", dtype=dtype)
    view = wide[:, 1, 2:10, 3:67]  # no 16-byte alignment, two strides
    view.copy_(q)
    out, _, tol, _ = attention(cache, q, table, n, scale=0.3)
    for t in tables(table[:, :-1], 16):
        target = torch.full((9, 10, 70), 5.0, device="cuda", dtype=dtype)
        got = cache.attend(view, t, n, scale=0.3, out=target[1:8, 1:9, 5:69])
        within(got, out, tol)
        target[1:8, 1:9, 5:69] = 5.0
        assert bool((target == 5).all())  # nothing around it was touched
    # a table inside a larger one
    big = torch.full((7, table.shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    big[:, 2:-3] = table
    assert torch.equal(cache.attend(q, big[:, 2:-3], n, scale=0.3), cache.attend(q, table, n, scale=0.3))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,heads,q_heads", [("ragged", 2, 8), ("one", 1, 20), ("edges", 2, 2), ("many", 1, 12), ("long", 2, 6)])
def test_attend_into_the_queries(dtype, lens, heads, q_heads):
    g = gen(13)
    cache, q, table, n = make_batch(g, LENS[lens], 16, heads, q_heads, 64, dtype)
    for t in tables(table, 16):
        want = cache.attend(q, t, n)
        wide = torch.full((len(q), q_heads + 2, 70), 5.0, device="cuda", dtype=dtype)
        view = wide[:, 1:-1, 3:67]
        view.copy_(q)
        assert cache.attend(view, t, n, out=view) is view and torch.equal(view, want)
        view[:] = 5.0
        assert bool((wide == 5).all())
    cache.check()


def test_attend_refuses_queries_with_other_strides():
    cache = pf.PagedKVCache(4, 16, 2, 64)
    q = torch.zeros(2, 2, 64, device="cuda")
    table, n = torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    for _ in range(2):  # checked for the first time, and as a known call
        with pytest.raises(ValueError, match="strides"):
            cache.attend(q, table, n, out=q.transpose(0, 1))


@pytest.mark.parametrize("window", [300, 2 ** 31 - 1, 2 ** 31, 2 ** 63 - 1, 2 ** 64, 2 ** 80])
def test_attend_windows_beyond_all_keys(window):
    g = gen(14)
    cache, q, table, n = make_batch(g, [300, 0, 17], 16, 1, 2, 64, F32)
    out, _, tol, _ = attention(cache, q, table, n)
    for t in tables(table, 16):  # a window may change how the work is shared, and so the order of the sums
        within(cache.attend(q, t, n, window=window), out, tol)


@pytest.mark.parametrize("dtype", TYPES)
def test_attend_bad_pages_and_lengths(dtype):
    g = gen(9)
    cache, q, table, n = make_batch(g, [40, 40, 40], 16, 1, 4, 64, dtype, spoil=False)
    table = table[:, :3].clone()
    for bad in (-1, cache.num_pages, 2 ** 31 - 1):
        t = table.clone()
        t[1, 1] = bad  # its 16 tokens are skipped
        out, _, tol, _ = attention(cache, q, table, n)
        keep = torch.cat((torch.arange(16), torch.arange(32, 40))).cuda()
        k, v = (x[table[1, keep // 16].long(), keep % 16, 0].double() for x in (cache.k, cache.v))
        out[1] = torch.softmax(q[1].double() @ k.T / 8, -1) @ v
        tol[1] = tol[1].amax() * 4  # of the same magnitudes, fewer keys
        for tt in tables(t, 16):
            within(cache.attend(q, tt, n), out, tol)
            with pytest.raises(pf._native.PfcError):
                cache.check()
    for bad, means in ((-5, 0), (1000, 48), (2 ** 31 - 1, 48)):
        m = n.clone()
        m[2] = bad
        want = torch.tensor([40, 40, means], dtype=torch.int32, device="cuda")
        assert torch.equal(cache.attend(q, table, m), cache.attend(q, table, want))
        with pytest.raises(pf._native.PfcError):
            cache.check()


@pytest.mark.parametrize("dtype", TYPES)
def test_attend_extremes(dtype):
    """One key that outweighs all, scores far apart, equal scores, NaN and infinities in a seen row of one sequence."""
    g = gen(10)
    cache, q, table, n = make_batch(g, [300, 300, 300, 64], 16, 1, 2, 64, dtype)
    big = 60.0
    cache.k[table[0, 3].long(), 5, 0] = q[0, 0] * big  # the score of head 0 jumps in the middle of the row
    cache.k[table[1, :19].long()] = 0  # all equal
    cache.v[table[2, 1].long(), 2, 0, 7] = math.nan
    cache.k[table[3, 0].long(), 0, 0, 0] = math.inf
    out, _, tol, _ = attention(cache, q, table, n)
    for t in tables(table, 16):
        got = cache.attend(q, t, n)
        within(got[:2], out[:2], tol[:2])
        assert bool(got[2, :, 7].isnan().all()) and bool(got[2, :, :7].isfinite().all())
        within(got[2, :, :7], out[2, :, :7], tol[2, :, :7].nan_to_num(1e-2))
        assert bool(got[0].isfinite().all())


@pytest.mark.parametrize("q_heads", [12, 24, 48, 96])
def test_attend_fp32_keeps_its_precision(q_heads):
    """Long runs of keys in one accumulator, which a truncating one would lose systematically. In the norm over independent
    keys the relative errors of a weight add in quadrature, rounding errors with their rms (their bound by the square root
    of 3): the argument of its exponential (2^-24 of about 7), exp2 (2^-22), the products of its score (3 2^-22 of about 1),
    its own and the value's splitting (3 2^-23), and 100 additions of 2^-24: 6.3e-7, below 2^-20."""
    g = gen(14)
    cache, q, table, n = make_batch(g, [6000] * 6, 64, 12, q_heads, 64, F32, spoil=False)
    out = attention(cache, q, table, n)[0]
    got = cache.attend(q, table, n).double()
    assert float((got - out).norm() / out.norm()) < 2.0 ** -20


def test_attend_small_weights_in_fp16():
    """A weight below fp16's range still counts: 4000 keys of weight 2^-20 next to one of weight 1."""
    n = 4001
    cache = pf.PagedKVCache(1, n, 1, 64, F16)
    q = torch.zeros(1, 1, 64, device="cuda", dtype=F16)
    q[..., 0] = 1
    cache.k[0, 0, 0, 0] = 20.0
    cache.v[0, 1:] = 1.0
    one = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    want = 4000 * 2.0 ** -20 / (1 + 4000 * 2.0 ** -20)
    for t in tables(one, n):
        got = cache.attend(q, t, torch.tensor([n], dtype=torch.int32, device="cuda"), scale=math.log(2.0))
        within(got, torch.full((1, 1, 64), want, dtype=torch.float64, device="cuda"), want * (HALF[F16] + 2.0 ** -16))


def test_attend_offsets_past_32_bits():
    """Pages more than 2^32 bytes from the cache's start."""
    page, heads, dim = 64, 8, 128
    pages = (5 << 30) // (page * heads * dim * 2)
    k, v = (torch.empty(pages, page, heads, dim, device="cuda", dtype=BF16) for _ in range(2))
    cache = pf.PagedKVCache.from_tensors(k, v)
    g = gen(11)
    chosen = [pages - 1, 0, pages // 2, pages - 2]
    table = torch.tensor([chosen], dtype=torch.int32, device="cuda")
    n = torch.tensor([4 * page - 3], dtype=torch.int32, device="cuda")
    tokens = 4 * page
    new_k, new_v = (randn(g, tokens, heads, dim, dtype=BF16) for _ in range(2))
    slots = (torch.tensor(chosen, device="cuda")[:, None] * page + torch.arange(page, device="cuda")).flatten()
    cache.append(new_k, new_v, slots)
    assert torch.equal(k[chosen].flatten(0, 1), new_k) and torch.equal(v[chosen].flatten(0, 1), new_v)
    q = randn(g, 1, 16, dim, dtype=BF16)
    out, _, tol, _ = attention(cache, q, table, n)
    for t in tables(table, page):
        within(cache.attend(q, t, n), out, tol)
    cache.check()


# ---------------------------------------------------------------------------
# 4-bit weights
# ---------------------------------------------------------------------------

def weights(g, n, k, group, zeros, scale_dtype=F16, size=1.0):
    packed = torch.randint(0, 256, (n, (k + 1) // 2), generator=g, device="cuda", dtype=torch.uint8)
    groups = -(-k // group)
    scales = ((torch.rand((n, groups), generator=g, device="cuda") + 0.5) * (size / 16)).to(scale_dtype)
    z = torch.randint(0, 16, (n, groups), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    q = torch.stack((packed & 15, packed >> 4), -1).flatten(1)[:, :k].double()
    of = torch.arange(k, device="cuda") // group
    w = (q - (z.double()[:, of] if zeros else 8.0)) * scales.double()[:, of]
    return packed, scales, z, w


def linear_tol(x, w, y, t, k, group):
    # a group (at most 128 columns) is summed 16 columns at a time, blocks and warps after it; fp32 x in three parts
    adds = (min(group, 128) / 8 + k / 1024 + 16) * 2.0 ** -23
    return HALF[t] * y.abs() + adds * (x.double().abs() @ w.abs().T) + 2.0 ** -23 * y.abs() + TINY[t]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inner,outer,group,zeros,bias", [
    (1, 4096, 64, 128, False, False), (1, 1, 1, 32, True, True), (2, 2, 15, 64, True, False), (3, 33, 16, 32, False, True),
    (5, 127, 17, 128, True, True), (7, 129, 100, 64, True, False), (8, 1000, 33, 32, True, True), (9, 1024, 48, 256, True, False),
    (16, 2049, 31, 128, False, False), (17, 640, 40, 4096, True, True), (21, 5000, 24, 32, True, False),
    (22, 384, 20, 64, False, True), (33, 4096, 37, 64, True, False), (64, 1536, 16, 128, True, True), (65, 200, 50, 32, True, False),
    (200, 700, 19, 128, False, True), (1, 16384, 200, 256, True, False), (8, 16384, 70, 128, True, True), (5, 9000, 130, 32, True, False),
    (2, 512, 10000, 64, True, False), (48, 9000, 300, 64, True, True), (40, 16384, 129, 512, False, False), (13, 3000, 2000, 32, True, False)])
def test_linear4(dtype, rows, inner, outer, group, zeros, bias):
    g = gen(rows + inner)
    packed, scales, z, w = weights(g, outer, inner, group, zeros)
    b = randn(g, outer, dtype=dtype) if bias else None
    layer = pf.Linear4bit(packed, scales, z, b, in_features=inner, group_size=group)
    x = randn(g, rows, inner, dtype=dtype)
    y = x.double() @ w.T + (b.double() if bias else 0.0)
    tol = linear_tol(x, w, y, dtype, inner, group)
    got = layer(x)
    within(got, y, tol)
    assert torch.equal(layer(x), got)
    # rows of a wider matrix, without 16-byte alignment; an output inside a larger one
    wide = torch.full((rows, inner + 3), math.nan, device="cuda", dtype=dtype)
    wide[:, 1:inner + 1] = x
    big = torch.full((rows + 2, outer + 5), 3.0, device="cuda", dtype=dtype)
    layer(wide[:, 1:inner + 1], out=big[1:-1, 2:-3])
    assert torch.equal(big[1:-1, 2:-3], got)
    big[1:-1, 2:-3] = 3.0
    assert bool((big == 3).all())


def test_linear4_most_rows():
    g = gen(12)
    packed, scales, z, w = weights(g, 8, 32, 32, True)
    layer = pf.Linear4bit(packed, scales, z, group_size=32)
    x = randn(g, 65535 * 16, 32)
    y = x.double() @ w.T
    within(layer(x), y, linear_tol(x, w, y, F32, 32, 32))
    with pytest.raises(pf._native.PfcError, match="rows"):
        layer(x[:1].expand(65535 * 16 + 1, 32))


@pytest.mark.parametrize("scale_dtype", [F16, BF16])
@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("inner,group", [(256, 64), (301, 32), (130, 128)])
def test_linear4_quantize(scale_dtype, symmetric, inner, group):
    g = gen(inner)
    w = randn(g, 40, inner) * 0.1
    w[3] = 0
    w[5, :group] = 0.25
    layer = pf.Linear4bit.quantize(w, group, symmetric=symmetric, scale_dtype=scale_dtype)
    back = layer(torch.eye(inner, device="cuda")).T  # row by row the weights that the layer stands for
    step = layer.scales.float().repeat_interleave(group, 1)[:, :inner]
    # half a step, and what the scale's own rounding moves: up to 15 steps at eps/2 each
    assert bool(((back - w).abs() <= step * (0.5 + 15 * HALF[scale_dtype] + 2.0 ** -20) + 1e-30).all())
    assert bool((back[3] == 0).all())


def test_linear4_quantize_ranges():
    g = gen(13)
    for size in (1e-9, 1e6):  # scales outside float16's range
        w = randn(g, 20, 100) * size
        layer = pf.Linear4bit.quantize(w, 32)
        assert layer.scales.dtype == BF16
        back = layer(torch.eye(100, device="cuda")).T
        step = layer.scales.float().repeat_interleave(32, 1)[:, :100]
        assert bool(((back - w).abs() <= step * (0.5 + 15 * HALF[BF16] + 2.0 ** -20)).all())
    w[1, 1] = math.inf
    for bad in (lambda: pf.Linear4bit.quantize(w, 32), lambda: pf.Linear4bit.quantize(w[0], 32), lambda: pf.Linear4bit.quantize(w, 48),
                lambda: pf.Linear4bit.quantize(randn(g, 4, 64) * 1e8, 32, scale_dtype=F16)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("dtype", TYPES)
def test_linear4_extremes(dtype):
    g = gen(12)
    packed, scales, z, w = weights(g, 32, 256, 64, True, BF16)
    layer = pf.Linear4bit(packed, scales, z, in_features=256, group_size=64)
    x = randn(g, 4, 256, dtype=dtype)
    x[1] *= torch.finfo(dtype).max / 2 ** 12
    x[2, 9], x[3, 200] = math.nan, math.inf
    y = x.double() @ w.T
    got = layer(x)
    assert bool(got[2].isnan().all())
    assert bool((~got[3].isfinite()).all())
    tol = linear_tol(x, w, y, dtype, 256, 64)
    within(got[0], y[0], tol[0])
    if dtype != F16:  # fp16 may overflow to an infinity there, as its rounding says
        within(got[1], y[1], tol[1])
    assert layer(x[:0]).shape == (0, 32)
    assert torch.equal(layer(x.view(2, 2, 256)).view(4, 32).nan_to_num(), got.nan_to_num())
    within(layer(x[0]), y[0], tol[0])  # one row alone is added in another order


# ---------------------------------------------------------------------------
# together, and as a program runs them
# ---------------------------------------------------------------------------

class Layer:
    """A decoder layer's attention for new tokens."""

    def __init__(self, g, dtype, width=256, q_heads=8, heads=2, dim=32, pages=40, page=8):
        self.heads, self.q_heads, self.dim, self.page = heads, q_heads, dim, page
        self.qkv_w = weights(g, (q_heads + 2 * heads) * dim, width, 64, True, size=0.125)  # scores of a few units
        self.out_w = weights(g, width, q_heads * dim, 32, True, size=0.125)
        self.qkv = pf.Linear4bit(*self.qkv_w[:3], in_features=width, group_size=64)
        self.out = pf.Linear4bit(*self.out_w[:3], in_features=q_heads * dim, group_size=32)
        self.rotary = pf.RotaryEmbedding(dim, scaling={"type": "yarn", "factor": 4, "original_max_position": 64})
        self.cache = pf.PagedKVCache(pages, page, heads, dim, dtype)

    def step(self, x, positions, slots, table, lens):
        q, k, v = self.qkv(x).unflatten(1, (-1, self.dim)).split([self.q_heads, self.heads, self.heads], 1)
        q = self.cache.append(k, v, slots, positions=positions, rotary=self.rotary, q=q)
        return self.out(self.cache.attend(q, table, lens).flatten(1))


@pytest.mark.parametrize("dtype", TYPES)
def test_decoding_steps(dtype):
    """Three sequences over 20 steps, one of them joining late; every step against 64 bits from the same inputs."""
    g = gen(20)
    layer = Layer(g, dtype)
    table = torch.randperm(39, generator=g, device="cuda")[:12].view(3, 4).to(torch.int32)
    keys = [[] for _ in range(3)]
    for step in range(20):
        x = randn(g, 3, 256, dtype=dtype)
        pos = torch.tensor([step, step, step - 10], device="cuda")
        slots = torch.where(pos >= 0, table[torch.arange(3), pos.clamp(min=0) // 8].long() * 8 + pos.clamp(min=0) % 8, -1)
        lens = (pos + 1).clamp(min=0).to(torch.int32)
        got = layer.step(x, pos, slots, table, lens)
        q, k, v = (x.double() @ layer.qkv_w[3].T).unflatten(1, (-1, 32)).split([8, 2, 2], 1)
        k, q = turn(k, pos, layer.rotary)[0], turn(q, pos, layer.rotary)[0]
        o = torch.zeros(3, 8, 32, dtype=torch.float64, device="cuda")
        for b in range(3):
            if pos[b] < 0:
                continue
            keys[b].append((k[b], v[b]))
            kk, vv = (torch.stack(c, 1) for c in zip(*keys[b]))  # [heads, keys, dim]
            s = q[b].unflatten(0, (2, 4)) @ kk.transpose(1, 2) / math.sqrt(32)
            o[b] = (torch.softmax(s, -1) @ vv).flatten(0, 1)
        want = o.flatten(1) @ layer.out_w[3].T
        # Each stage rounds to its type once: x W (eps/2 of it), the rotation (eps/2), the attention's output (eps/2), the
        # result (eps/2). q and k are each off by two of these, so a score by 4 eps/2 of scale |q||k| = m eps/2, and a
        # weight, a quotient of two exponentials, by the factor e^(2 m eps/2). The outputs are averages of values.
        m = 4 * float((q.norm(dim=-1).amax() * max(c[0].norm(dim=-1).amax() for r in keys for c in r)) / math.sqrt(32))
        rel = (math.exp(2 * m * HALF[dtype]) - 1) + 4 * HALF[dtype]
        scale = max(float(c[1].abs().amax()) for r in keys for c in r)
        bound = rel * scale * layer.out_w[3].abs().sum(1) + HALF[dtype] * want.abs() + 2.0 ** -18 * scale * layer.out_w[3].abs().sum(1)
        within(got, want, bound, f"step {step}")
    layer.cache.check()


def test_captured_steps_replay():
    """A captured step follows its inputs; two captured graphs replayed at once on two streams do not meet."""
    dtype = BF16
    layers = [Layer(gen(30 + i), dtype) for i in range(2)]
    table = tables(torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4), 8)[1]
    state, graphs, outs = [], [], []
    side = torch.cuda.Stream()
    for layer in layers:
        s = dict(x=torch.zeros(2, 256, device="cuda", dtype=dtype), positions=torch.zeros(2, dtype=torch.int64, device="cuda"),
                 slots=torch.full((2,), -1, dtype=torch.int64, device="cuda"), table=table,
                 lens=torch.zeros(2, dtype=torch.int32, device="cuda"))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer.step(**s)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(layer.step(**s))
        state.append(s)
        graphs.append(graph)
    eager = [Layer(gen(30 + i), dtype) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    g = gen(40)
    for step in range(12):
        wants = []
        for s, layer in zip(state, eager):
            s["x"].copy_(randn(g, 2, 256, dtype=dtype))
            s["positions"].fill_(step)
            s["slots"].copy_(table[:, step // 8].long() * 8 + step % 8)
            s["lens"].fill_(step + 1)
            wants.append(layer.step(**s))
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for out, want in zip(outs, wants):
            assert torch.equal(out, want), step


def test_first_call_captured_after_a_fork():
    """Calls of shapes not seen before, captured where two streams join, after a copy, and followed by another library's
    kernel; replayed on new data."""
    g = gen(45)
    layer = Layer(g, F16, q_heads=6, dim=40)
    x = randn(g, 5, 256, dtype=F16)
    source = torch.zeros_like(x)
    pos, slots = torch.arange(5, device="cuda"), torch.arange(5, device="cuda") * 9
    table, lens = torch.arange(5, dtype=torch.int32, device="cuda")[:, None].contiguous(), torch.ones(5, dtype=torch.int32, device="cuda")
    slots = torch.arange(5, device="cuda") * 8
    other = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            moved = x * 2
        x.copy_(source)
        torch.cuda.current_stream().wait_stream(other)
        got = layer.step(x, pos, slots, table, lens) + moved.sum() * 0
    for _ in range(3):
        source.copy_(randn(g, 5, 256, dtype=F16))
        graph.replay()
        want = layer.step(source, pos, slots, table, lens)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_calls_from_two_threads():
    import threading
    g = gen(46)
    cache, q, table, n = make_batch(g, [700, 90], 16, 2, 8, 64, F16)
    r = pf.RotaryEmbedding(64)
    layer = pf.Linear4bit(*weights(g, 96, 512, 64, True)[:3], in_features=512, group_size=64)
    pos = torch.arange(2, device="cuda")
    xs = [randn(g, i + 1, 512, dtype=F16) for i in range(12)]
    want = [layer(x) for x in xs], cache.attend(q, table, n), r.apply(q, pos)
    torch.cuda.synchronize()
    wrong = []

    def work(stream):
        with torch.cuda.stream(stream):
            for i in range(60):
                ok = (torch.equal(layer(xs[i % 12]), want[0][i % 12]) and torch.equal(cache.attend(q, table, n), want[1])
                      and torch.equal(r.apply(q, pos), want[2]))
                if not ok:
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(torch.cuda.Stream(),)) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    cache.check()


def test_plans_follow_their_arguments():
    """Calls that differ in one argument are not taken for one another."""
    g = gen(47)
    cache, q, table, n = make_batch(g, [300, 200], 16, 2, 8, 64, F32)
    for scale, window in ((None, 0), (0.5, 0), (0.5, 7), (None, 7), (torch.tensor(0.25), 7), (1, 1)):
        out, _, tol, _ = attention(cache, q, table, n, window, None if scale is None else float(scale))
        within(cache.attend(q, table, n, scale=scale, window=window), out, tol)
    scale = torch.tensor(0.25)
    first = cache.attend(q, table, n, scale=scale)
    scale.fill_(0.75)
    out, _, tol, _ = attention(cache, q, table, n, 0, 0.75)
    within(cache.attend(q, table, n, scale=scale), out, tol)
    assert not torch.equal(first, cache.attend(q, table, n, scale=scale))
    x = randn(g, 4, 64, 8, 64)  # the same shape in other strides
    r, pos = pf.RotaryEmbedding(64), torch.arange(64, device="cuda")
    for v in (x, x.transpose(0, 1).contiguous().transpose(0, 1), x.transpose(1, 2).contiguous().transpose(1, 2)):
        y, mag = turn(v, pos, r)
        within(r.apply(v, pos), y, turn_tol(y, mag, F32))
        within(r.backward(v, pos), turn(v, pos, r, -1)[0], turn_tol(y.abs() + mag, mag, F32))


def test_two_streams_at_once():
    g = gen(50)
    cache, q, table, n = make_batch(g, [4000, 3000], 16, 2, 16, 128, BF16)
    q2 = randn(g, 2, 16, 128, dtype=BF16)
    table = tables(table, 16)[1]
    want, want2 = cache.attend(q, table, n), cache.attend(q2, table, n)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    got, got2 = [], []
    for _ in range(20):
        with torch.cuda.stream(a):
            got.append(cache.attend(q, table, n))
        with torch.cuda.stream(b):
            got2.append(cache.attend(q2, table, n))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got) and all(torch.equal(x, want2) for x in got2)


def test_refusals():
    cache = pf.PagedKVCache(4, 16, 2, 64)
    r = pf.RotaryEmbedding(64)
    x, i64 = torch.zeros(3, 2, 64, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    table, lens = torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    layer = pf.Linear4bit(torch.zeros(8, 32, dtype=torch.uint8, device="cuda"), torch.ones(8, 1, device="cuda", dtype=F16), group_size=64,
                          bias=torch.zeros(8, device="cuda"))
    grad = x.clone().requires_grad_()
    value = [
        lambda: r.apply(x.cpu(), i64), lambda: r.apply(x, i64.cpu()), lambda: r.apply(x[0], i64), lambda: r.apply(x[..., :32], i64),
        lambda: r.apply(x, i64[:2]), lambda: r.apply(x.transpose(1, 2).contiguous().transpose(1, 2), i64),
        lambda: r.apply(x, i64, out=x[:1].expand(3, 2, 64)), lambda: r.apply(x, i64, out=x[:, :1]),
        lambda: pf.RotaryEmbedding(64, 65), lambda: pf.RotaryEmbedding(64, layout="other"), lambda: pf.RotaryEmbedding(2000),
        lambda: pf.RotaryEmbedding(64, inv_freq=[1.0]), lambda: pf.PagedKVCache(0, 16, 2, 64),
        lambda: pf.PagedKVCache.from_tensors(cache.k, cache.v[:2]), lambda: pf.PagedKVCache.from_tensors(cache.k, cache.v.transpose(0, 1)),
        lambda: pf.PagedKVCache.from_tensors(cache.k[:1].expand(4, 16, 2, 64), cache.v[:1].expand(4, 16, 2, 64)),
        lambda: cache.append(x, x[:2], i64), lambda: cache.append(x, x, i64[:2]), lambda: cache.append(x, x, i64, positions=i64),
        lambda: cache.append(x, x, i64, rotary=r), lambda: cache.append(x, x, i64, positions=i64, rotary=pf.RotaryEmbedding(32)),
        lambda: cache.append(x, x, i64, q_out=x), lambda: cache.append(x, x, i64, q=x[:2]),
        lambda: cache.attend(x[:, :1], table, lens), lambda: cache.attend(x, table[:2], lens), lambda: cache.attend(x, table, lens[:1]),
        lambda: cache.attend(x, table, lens, window=-1), lambda: cache.attend(x[0], table, lens),
        lambda: layer(torch.zeros(2, 63, device="cuda")), lambda: layer(x[0].view(2, 64), out=x[0].view(16, 8)[:2]),
        lambda: layer(torch.zeros(2, 3, 64, device="cuda"), out=torch.zeros(3, 2, 8, device="cuda").transpose(0, 1)), lambda: layer(torch.zeros(2, 64)),
        lambda: pf.Linear4bit(torch.zeros(8, 32, dtype=torch.uint8, device="cuda"), torch.ones(8, 2, device="cuda", dtype=F16), group_size=64),
        lambda: pf.Linear4bit(torch.zeros(8, 32, dtype=torch.uint8, device="cuda"), torch.ones(8, 1, device="cuda", dtype=F16), group_size=48),
        lambda: pf.Linear4bit(torch.zeros(8, 32, dtype=torch.uint8, device="cuda"), torch.ones(8, 1, device="cuda", dtype=F16),
                              torch.full((8, 1), 16, dtype=torch.uint8, device="cuda"), group_size=64),
    ]
    for i, f in enumerate(value):
        with pytest.raises(ValueError):
            f()
            raise AssertionError(f"call {i} was not refused")
    kind = [
        lambda: r.apply(x.double(), i64), lambda: r.apply(x, i64.int()), lambda: cache.append(x.half(), x, i64),
        lambda: cache.attend(x.half(), table, lens), lambda: cache.attend(x, table.long(), lens), lambda: cache.attend(x, table, lens.long()),
        lambda: layer(torch.zeros(2, 64, device="cuda", dtype=F16)), lambda: pf.PagedKVCache(2, 2, 2, 8, torch.int8),
        lambda: pf.Linear4bit(torch.zeros(8, 32, dtype=torch.uint8, device="cuda"), torch.ones(8, 1, device="cuda"), group_size=64),
    ]
    for i, f in enumerate(kind):
        with pytest.raises(TypeError):
            f()
            raise AssertionError(f"call {i} was not refused")
    with pytest.raises(RuntimeError, match="gradient"):
        r.apply(grad, i64)
    with torch.no_grad():
        r.apply(grad, i64)
    odd = pf.PagedKVCache(2, 4, 1, 12)  # appended to, not attended
    with pytest.raises(pf._native.PfcError, match="head_dim"):
        odd.attend(torch.zeros(1, 1, 12, device="cuda"), table[:1], lens[:1])


def test_workspace_is_checked(native):
    cache, q, table, n = make_batch(gen(60), [40], 16, 1, 4, 64, F32)
    table = tables(table, 16)[1]
    out = torch.zeros_like(q)
    work = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    p = native.PagedAttentionParamsC(cache._c, 1, 4, q.data_ptr(), 256, 64, out.data_ptr(), 256, 64, None, table.data_ptr(),
                                     table.shape[1], table.shape[1], n.data_ptr(), 0, 0.125, work.data_ptr(), 0)
    L, need = native.lib(), C.c_size_t(0)
    assert L.pfk_paged_attention_workspace(C.byref(p), C.byref(need)) == 0 and 0 < need.value <= work.numel()
    for ptr, size in ((work.data_ptr(), need.value - 1), (None, need.value), (work.data_ptr() + 8, need.value)):
        p.workspace, p.workspace_bytes = ptr, size
        assert L.pfk_paged_attention(C.byref(p), None) == -1 and b"workspace" in L.pfc_last_error()
    p.workspace, p.workspace_bytes = work.data_ptr(), need.value
    work.fill_(255)  # what is in it does not matter
    torch.cuda.synchronize()
    assert L.pfk_paged_attention(C.byref(p), None) == 0
    torch.cuda.synchronize()
    assert torch.equal(out, cache.attend(q, table, n, scale=0.125))
