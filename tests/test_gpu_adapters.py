"""Low-rank adapters on the GPU against 64 bits.

Tolerances count roundings.  eps(t)/2 of the result is the output's own.  Sums
in the tensor cores lose at most 2^-23 of what has been added for each of a
step's two instructions (fp32: six, and 2^-21 for the parts of an operand),
and are added up in fp32, at most some hundred times (2^-24 each): below 2^-16
of the sum of magnitudes S = |scale| sum_r |B| sum_k |A| |x|.  What lies between
the products is held to 2^-17 in bfloat16's two parts: 2^-15 of S in all, and
2^-16 in the other types.
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
SUMS = {F32: 2.0 ** -16, F16: 2.0 ** -16, BF16: 2.0 ** -15}


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def within(got, want, tol, what=""):
    got = got.double()
    assert got.shape == want.shape, (got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    if bad.any():
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; first {i}: {got[i]} for {want[i]}, "
                             f"tolerance {torch.broadcast_to(torch.as_tensor(tol), got.shape)[i]}")


def make(g, n, inner, outer, ranks, dtype, most=None):
    layer = pf.LowRankAdapters(n, inner, outer, most or max(ranks), dtype=dtype)
    parts = []
    for i in range(n):
        r = ranks[i % len(ranks)]
        a, b = (randn(g, r, inner) / math.sqrt(inner)).to(dtype), randn(g, outer, r, dtype=dtype)
        parts.append((a, b, 0.5 + 0.25 * i))
        layer.load(i, *parts[-1])
    return layer, parts


def reference(parts, x, index, base, outer):
    x2, i2 = x.reshape(-1, x.shape[-1]).double(), index.reshape(-1)
    out = torch.zeros(len(x2), outer, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(out)
    for i, (a, b, s) in enumerate(parts):
        rows = (i2 == i).nonzero()[:, 0]
        out[rows] = x2[rows] @ a.double().T @ b.double().T * s
        mag[rows] = x2[rows].abs() @ a.double().abs().T @ b.double().abs().T * abs(s)
    out, mag = out.view(*x.shape[:-1], outer), mag.view(*x.shape[:-1], outer)
    return (out if base is None else out + base.double()), mag


def check(layer, parts, x, index, base, **kw):
    t = x.dtype
    got = layer(x, index, base, **kw)
    out, mag = reference(parts, x, index, None if base is None else base.clone() if kw.get("out") is base else base, layer.out_features)
    within(got, out, HALF[t] * out.abs() + SUMS[t] * mag)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inner,outer,ranks,n", [
    (1, 4096, 4096, [16], 3), (1, 60, 77, [4], 1), (5, 64, 64, [8, 16], 2), (8, 1024, 33, [17], 1), (9, 333, 100, [32], 1), (16, 100, 31, [64, 3], 2),
    (17, 768, 768, [16], 1), (32, 256, 512, [48], 1), (33, 128, 1000, [16], 2), (61, 500, 2051, [64], 64), (100, 2048, 96, [100], 5),
    (300, 515, 515, [16, 32, 1], 7), (1000, 96, 200, [128], 3), (2, 16384, 40, [16], 2), (40, 31, 16, [256], 2), (3, 1, 1, [1], 2), (64, 8, 24, [16], 3)])
def test_rows(dtype, rows, inner, outer, ranks, n):
    g = gen(rows + inner + outer)
    layer, parts = make(g, n, inner, outer, ranks, dtype)
    x, base = randn(g, rows, inner, dtype=dtype), randn(g, rows, outer, dtype=dtype)
    mixed = torch.randint(-1, n, (rows,), generator=g, device="cuda", dtype=torch.int32)
    check(layer, parts, x, mixed, base)
    check(layer, parts, x, mixed.sort()[0], base)
    check(layer, parts, x, torch.full_like(mixed, n - 1), None)
    layer.check()


@pytest.mark.parametrize("dtype", TYPES)
def test_groups_of_every_size(dtype):
    """Tiles of 32 rows whose groups have 1, 8, 9, 16, 17 and 32 rows, in runs and mixed."""
    g = gen(1)
    layer, parts = make(g, 6, 200, 130, [16, 32, 5], dtype)
    index = sum(([i] * m for i, m in enumerate((1, 8, 9, 16, 17, 32))), []) + [-1] * 5
    index = torch.tensor(index, dtype=torch.int32, device="cuda")
    for order in (index, index[torch.randperm(len(index), generator=g, device="cuda")], index.flip(0)):
        check(layer, parts, randn(g, len(index), 200, dtype=dtype), order, randn(g, len(index), 130, dtype=dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_without_an_adapter_keep_their_bits(dtype):
    g = gen(2)
    layer, _ = make(g, 2, 64, 70, [16], dtype)
    x, base = randn(g, 40, 64, dtype=dtype), randn(g, 40, 70, dtype=dtype)
    base[3, 5], base[4, 6] = float("inf"), float("nan")
    index = torch.full((40,), -1, dtype=torch.int32, device="cuda")
    index[::3], index[1::3] = -(1 << 31), -7
    out = layer(x, index, base)
    assert torch.equal(out.view(torch.uint8), base.view(torch.uint8))
    assert not layer(x, index).any()
    inside = base.clone()
    assert layer(x, index, inside, out=inside) is inside and torch.equal(inside.view(torch.uint8), base.view(torch.uint8))


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(dtype):
    """Leading axes, slices of wider rows, in place, odd strides and places."""
    g = gen(3)
    layer, parts = make(g, 3, 72, 56, [16, 24], dtype)
    x, base = randn(g, 4, 5, 72, dtype=dtype), randn(g, 4, 5, 56, dtype=dtype)
    index = torch.randint(-1, 3, (4, 5), generator=g, device="cuda", dtype=torch.int32)
    want = check(layer, parts, x, index, base)
    assert torch.equal(layer(x[1, 2], index[1, 2], base[1, 2]), layer(x[1, 2][None], index[1, 2][None], base[1, 2][None])[0])
    wide = randn(g, 4, 5, 200, dtype=dtype)
    wide[..., 3:75], wide[..., 101:157] = x, base
    assert torch.equal(layer(wide[..., 3:75], index, wide[..., 101:157]), want)
    keep = wide.clone()
    view = wide[..., 101:157]
    assert layer(wide[..., 3:75], index, view, out=view) is view
    assert torch.equal(view, want) and torch.equal(wide[..., :101], keep[..., :101]) and torch.equal(wide[..., 157:], keep[..., 157:])
    turned = x.transpose(0, 1).contiguous().transpose(0, 1)  # rows at two strides: copied
    assert torch.equal(layer(turned, index.T.contiguous().T, base), want)
    out = torch.empty(20, 56, device="cuda", dtype=dtype)
    layer(x.view(20, 72), index.view(20), base.view(20, 56), out=out)
    assert torch.equal(out.view(4, 5, 56), want)
    assert layer(x[:0], index[:0], base[:0]).shape == (0, 5, 56)
    thin = torch.stack((index.view(20), index.view(20)), 1)[:, 0]
    assert torch.equal(layer(x.view(20, 72), thin, base.view(20, 56)), out)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inner,outer", [(72, 56), (33, 131), (7, 3), (515, 1025), (1, 1)])
def test_rows_at_every_place(dtype, inner, outer):
    """Rows between NaNs, that begin on no 16 bytes: the bits of packed, aligned ones, and the NaNs stay."""
    g = gen(inner)
    layer, parts = make(g, 4, inner, outer, [16, 48], dtype)
    index = torch.tensor([0] * 40 + [1] * 12 + [-1] * 9 + [2] * 3 + [-1] + [3] * 17, dtype=torch.int32, device="cuda")
    x, base = randn(g, len(index), inner, dtype=dtype), randn(g, len(index), outer, dtype=dtype)
    pad = lambda n: torch.zeros(len(index), (n + 15) // 8 * 8, device="cuda", dtype=dtype)
    ax, ab = pad(inner)[:, :inner].copy_(x), pad(outer)[:, :outer].copy_(base)
    aligned = pad(outer)[:, :outer]
    want = check(layer, parts, ax, index, ab, out=aligned)
    assert torch.equal(layer(x, index, base), want)
    zero = layer(ax, index)
    for place in range(8):
        wide = torch.full((len(index), inner + outer + 23 + place % 3), float("nan"), device="cuda", dtype=dtype)
        wx, wb = wide[:, place:place + inner], wide[:, place + inner + 5:place + inner + 5 + outer]
        wx.copy_(x)
        wb.copy_(base)
        assert torch.equal(layer(wx, index, wb), want) and torch.equal(layer(wx, index), zero)
        layer(wx, index, wb, out=wb)
        assert torch.equal(wb, want) and torch.equal(wx, x)
        wx.fill_(float("nan"))
        wb.fill_(float("nan"))
        assert wide.isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,inner,outer", [(600, 16, 640, 320), (731, 16, 1000, 97), (1200, 5, 512, 1024), (2100, 3, 1025, 65)])
def test_tiles_of_few_and_of_many_groups(dtype, rows, n, inner, outer):
    """Runs, mixed rows and both beside each other: groups that several CTAs share and groups that one has."""
    g = gen(rows)
    layer, parts = make(g, n, inner, outer, [16, 40], dtype)
    x, base = randn(g, rows, inner, dtype=dtype), randn(g, rows, outer, dtype=dtype)
    mixed = torch.randint(-1, n, (rows,), generator=g, device="cuda", dtype=torch.int32)
    runs = mixed.sort()[0]
    both = torch.where(torch.arange(rows, device="cuda") // 100 % 2 == 0, mixed, runs)
    for index in (runs, mixed, both):
        got = check(layer, parts, x, index, base)
        inside = base.clone()
        assert torch.equal(layer(x, index, inside, out=inside), got)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inner,outer,rank", [(1, 4096, 200, 16), (7, 96, 130, 40), (16, 333, 65, 16), (70, 512, 96, 64), (40, 64, 33, 256)])
def test_between_the_products(dtype, rows, inner, outer, rank):
    """scale A x far from 1, which B brings back: sizes from 1e-6 to 1e8, both in one adapter, and zeros of B
    beside them.  The tolerance is that of any other call, with half a step of float16's subnormals (2^-25), and
    for float16 what its two parts lose of a row's small values: half of 2^-24 on a scale where the largest is
    2^14 at least, so 2^-39 of that for each rank."""
    g = gen(rows + rank)
    x, base = randn(g, rows, inner, dtype=dtype), randn(g, rows, outer, dtype=dtype)
    layer = pf.LowRankAdapters(4, inner, outer, rank, dtype=dtype)
    parts = []
    for i, (size, scale) in enumerate([(300.0, 350.0), (100.0, 1e6), (1e-4, 1e-2), (30.0, 4000.0)]):
        a = (size * randn(g, rank, inner) / math.sqrt(inner)).to(dtype)  # scale a x: 1e5, 1e8, 1e-6, 1e5
        b = (randn(g, outer, rank) * min(1e3, max(1e-7, 1 / (size * scale)))).to(dtype)
        if i == 3:
            a[rank // 2:] = (1e-7 * a[rank // 2:].float()).to(dtype)
            b[:, rank // 2:] = (1e3 * randn(g, outer, rank - rank // 2)).to(dtype)
        b[outer // 2] = 0
        parts.append((a, b, scale))
        layer.load(i, *parts[-1])
    mixed = torch.arange(rows, device="cuda", dtype=torch.int32) % 4
    for index in (mixed, mixed.sort()[0], *(torch.full_like(mixed, i) for i in range(4))):
        got = layer(x, index, base)
        out, mag = reference(parts, x, index, base, outer)
        lost = torch.zeros_like(mag)
        if dtype == F16:
            for i, (a, b, s) in enumerate(parts):
                hit = index == i
                lost[hit] = 2.0 ** -39 * abs(s) * (x[hit].double() @ a.double().T).abs().amax(1, keepdim=True) * b.double().abs().sum(1)
        within(got, out, HALF[dtype] * out.abs() + SUMS[dtype] * mag + lost + 2.0 ** -25)
        assert got.isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 3, 20, 70])
@pytest.mark.parametrize("inner", [64, 100, 333])
def test_rows_of_a_wider_than_x(dtype, rows, inner):
    """The C entry point takes rows of a at any distance: what lies behind their zeros, here NaN, is not read."""
    g, outer, rank = gen(rows + inner), 48, 16
    layer, parts = make(g, 2, inner, outer, [rank], dtype)
    x, base = randn(g, rows, inner, dtype=dtype), randn(g, rows, outer, dtype=dtype)
    index = torch.arange(rows, device="cuda", dtype=torch.int32) % 2
    want = check(layer, parts, x, index, base)
    per = 16 // x.element_size()
    real = -(-inner // per) * per
    a = torch.full((2, rank, real + 40 * per), float("nan"), device="cuda", dtype=dtype)
    a[..., :real] = layer._a[..., :real]
    out = torch.empty_like(base)
    p = N.AdaptersParamsC.from_buffer_copy(layer._base)
    p.rows, p.x, p.x_st, p.index, p.base, p.base_st = rows, x.data_ptr(), inner, index.data_ptr(), base.data_ptr(), outer
    p.out, p.out_st, p.a, p.a_st = out.data_ptr(), outer, a.data_ptr(), a.shape[-1]
    N.check(N.lib().pfk_adapters(C.byref(p), torch.cuda.current_stream().cuda_stream))
    within(out, want.double(), HALF[dtype] * 2 * want.double().abs() + 2 * SUMS[dtype] * reference(parts, x, index, base, outer)[1])


@pytest.mark.parametrize("dtype", TYPES)
def test_adapters_are_replaced(dtype):
    g = gen(4)
    layer, parts = make(g, 2, 64, 64, [32], dtype)
    x, base = randn(g, 6, 64, dtype=dtype), randn(g, 6, 64, dtype=dtype)
    index = torch.tensor([0, 1, 0, 1, 1, -1], dtype=torch.int32, device="cuda")
    check(layer, parts, x, index, base)
    parts[1] = (randn(g, 3, 64, dtype=dtype), randn(g, 64, 3, dtype=dtype), -2.0)  # a lower rank: nothing of the old one remains
    layer.load(1, *parts[1])
    check(layer, parts, x, index, base)
    fresh = pf.LowRankAdapters(2, 64, 64, 8, dtype=dtype)
    assert torch.equal(fresh(x, index, base), base)


def test_bad_index_is_reported():
    g = gen(5)
    layer, parts = make(g, 2, 64, 64, [16], F16)
    x, base = randn(g, 3, 64, dtype=F16), randn(g, 3, 64, dtype=F16)
    out = layer(x, torch.tensor([1, 2, 1 << 30], dtype=torch.int32, device="cuda"), base)
    assert torch.equal(out[1:], base[1:]) and not torch.equal(out[0], base[0])
    with pytest.raises(N.PfcError, match="adapter"):
        layer.check()
    layer.check()


def test_a_row_does_not_depend_on_other_rows():
    """NaN and infinities of one request stay in its rows."""
    g = gen(6)
    for dtype in TYPES:
        layer, parts = make(g, 3, 100, 60, [16], dtype)
        x, base = randn(g, 24, 100, dtype=dtype), randn(g, 24, 60, dtype=dtype)
        index = torch.tensor([0, 1] * 12, dtype=torch.int32, device="cuda")
        want = layer(x, index, base)
        x[3], x[4, 7] = float("nan"), float("inf")
        got = layer(x, index, base)
        rest = torch.tensor([i for i in range(24) if i not in (3, 4)], device="cuda")
        assert torch.equal(got[rest], want[rest]) and got[3].isnan().all() and not got[4].isfinite().any()
        layer.load(2, torch.full((16, 100), float("nan"), device="cuda", dtype=dtype), torch.zeros(60, 16, device="cuda", dtype=dtype))
        index[5] = 2
        again = layer(x, index, base)
        assert torch.equal(again[rest[rest != 5]], want[rest[rest != 5]]) and again[5].isnan().all()


def test_same_bits_streams_and_graphs():
    g = gen(7)
    layer, parts = make(g, 4, 512, 2048, [16, 64], BF16)
    x, base = randn(g, 50, 512, dtype=BF16), randn(g, 50, 2048, dtype=BF16)
    index = torch.randint(-1, 4, (50,), generator=g, device="cuda", dtype=torch.int32)
    want = layer(x, index, base)
    for _ in range(3):
        assert torch.equal(layer(x, index, base), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = layer(x, index, base)
    assert torch.equal(layer(x, index, base), want)
    torch.cuda.synchronize()
    assert torch.equal(other, want)
    graph, i2 = torch.cuda.CUDAGraph(), index.clone()
    with torch.cuda.graph(graph):
        out = layer(x, i2, base)
    i2.copy_(index.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, layer(x, index.flip(0), base))


def test_refusals():
    layer = pf.LowRankAdapters(2, 64, 48, 16, dtype=F16)
    x, index, base = (torch.zeros(3, 64, device="cuda", dtype=F16), torch.zeros(3, dtype=torch.int32, device="cuda"),
                      torch.zeros(3, 48, device="cuda", dtype=F16))
    for bad, err in [(dict(x=x.float()), TypeError), (dict(x=x[:, :63]), ValueError), (dict(x=x.cpu()), ValueError), (dict(index=index.long()), TypeError),
                     (dict(index=index[:2]), ValueError), (dict(base=base[:, :47]), ValueError), (dict(base=base.float()), TypeError),
                     (dict(out=base[:2]), ValueError), (dict(out=base.bfloat16()), TypeError), (dict(x=x.clone().requires_grad_()), RuntimeError),
                     (dict(out=base[:1].expand(3, 48)), ValueError), (dict(x=x.T.contiguous().T), ValueError)]:
        with pytest.raises(err):
            layer(**{**dict(x=x, index=index, base=base), **bad})
    memory = torch.zeros(3, 64 + 48, device="cuda", dtype=F16)
    with pytest.raises(ValueError, match="shares memory with x"):
        layer(memory[:, :64], index, base, out=memory[:, 32:80])
    with pytest.raises(ValueError, match="base"):
        layer(x, index, memory[:, :48], out=memory[:, 1:49])
    flat = torch.zeros(200, device="cuda", dtype=F16)
    with pytest.raises(ValueError, match="base"):
        layer(x, index, flat[:144].view(3, 48), out=flat.as_strided((3, 48), (50, 1)))
    layer(memory[:, :64], index, base, out=memory[:, 64:])  # between each other's rows is no overlap
    a, b = torch.zeros(4, 64, device="cuda", dtype=F16), torch.zeros(48, 4, device="cuda", dtype=F16)
    for args, err in [((2, a, b), IndexError), ((-1, a, b), IndexError), ((0, a.float(), b), TypeError), ((0, a, b[:, :3]), ValueError),
                      ((0, a[:, :3], b), ValueError), ((0, torch.zeros(17, 64, device="cuda", dtype=F16), b), ValueError), ((0, a.cpu(), b), ValueError)]:
        with pytest.raises(err):
            layer.load(*args)
    layer.load(0, a.T.contiguous().T, b.clone().requires_grad_())  # any strides; values are copied
