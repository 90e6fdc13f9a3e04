"""Token-generation operators on the GPU where precision, ranges and memory
come to an edge, and next to the graph executor.
"""
import numpy as np
import pytest
import torch

import pyflame_b200 as pf
from tests.test_gpu_decoding import (BF16, F16, F32, HALF, TYPES, Layer, attention, gen, linear_tol, make_batch, randn, turn,
                                     turn_tol, weights, within)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("w", [1.0, 0.75, 2.0 ** -9 * 5])
def test_rope_cosines_next_to_quarter_turns(w):
    """Each cosine and sine is right in relation to itself, however small, at any position: next to quarter turns (11, 33,
    355 and 103993 are numerators of approximations of pi) and far out. Angles are exact in numpy's long double.
    sinpi and cospi are off by 1 ulp (2^-23) at most, and their argument, rounded to fp32 within an eighth of a turn of
    0, by 2^-24, which a sine passes on at most whole and a cosine at most pi/4 of: below 2^-22 in all."""
    positions = [0, 1, 11, 22, 33, 355, 710, 104348, 103993, 10 ** 6 + 1, 2 ** 31 - 1, 5419351, 80143857, 2 ** 40 + 12345, 2 ** 52 + 1]
    r = pf.RotaryEmbedding(2, inv_freq=[w])
    x = torch.tensor([[[1.0, 0.0], [0.0, 1.0]]], device="cuda").expand(len(positions), 2, 2).contiguous()
    pos = torch.tensor(positions, device="cuda")
    angle = np.array(positions, dtype=np.longdouble) * np.longdouble(w)
    c, s = (torch.from_numpy(f(angle).astype(np.float64)).cuda() for f in (np.cos, np.sin))
    for got, sign in ((r.apply(x, pos), 1), (r.backward(x, pos), -1)):
        want = torch.stack((torch.stack((c, sign * s), -1), torch.stack((-sign * s, c), -1)), 1)
        within(got, want, 2.0 ** -22 * want.abs())
    assert torch.equal(r.apply(x, -pos), r.backward(x, pos))


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("q_heads,dim", [(1, 64), (8, 128), (16, 128), (8, 256)])
def test_attend_long_rows_keep_their_precision(dtype, q_heads, dim):
    """Values around 1 in the first half of a row and around -1 in the second: the running output climbs to half of the
    weights' sum and comes back, so what each addition loses shows beside a small result. 131072 keys make 2048 additions
    in each of four warps, to a running output of half the sum at most. Rounded to nearest, an addition is off by an ulp
    / sqrt(12) in the root mean square, so a warp by sqrt(2048) 2^-23 / 2 / sqrt(12) = 7.8e-7 and the mean of four by
    3.9e-7; a step's own sum of 16 products, which the instruction truncates, adds at most 2^-22. Six times the first
    and the second are below 2^-18. Cut off instead, the additions would lose about 6e-5."""
    g = gen(70)
    page, n, rows = 64, 131072, 300  # rows for every CTA of one wave; they share the pages
    cache = pf.PagedKVCache.from_tensors(*(randn(g, n // page, page, 1, dim, dtype=dtype) for _ in range(2)))
    cache.v.copy_(torch.rand(cache.v.shape, generator=g, device="cuda") + 0.5)
    cache.v[n // page // 2:].neg_()
    q = randn(g, rows, q_heads, dim, dtype=dtype)
    table = torch.arange(n // page, dtype=torch.int32, device="cuda").expand(rows, -1)
    got = cache.attend(q, table, torch.full((rows,), n, dtype=torch.int32, device="cuda"))
    k, v = (x.view(n, dim).double() for x in (cache.k, cache.v))
    for i in range(0, rows, 37):
        want = torch.softmax(q[i].double() @ k.T * dim ** -0.5, -1) @ v
        within(got[i], want, HALF[dtype] * want.abs() + 2.0 ** -18, f"row {i}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,heads,q_heads,dim,page,window", [
    (24, 1, 4, 64, 16, 777), (24, 2, 8, 128, 13, 1500), (10, 2, 32, 128, 32, 4999), (20, 1, 1, 256, 16, 333), (24, 2, 10, 80, 1, 601)])
def test_attend_windows_shared_by_ctas(dtype, rows, heads, q_heads, dim, page, window):
    """Windows of many tiles, that begin inside a tile and inside a page, with more units than clusters take: the work list,
    whose units several CTAs share."""
    g = gen(71)
    lens = [(i * 1397) % 6001 for i in range(rows)]
    cache, q, table, n = make_batch(g, lens, page, heads, q_heads, dim, dtype)
    out, lse, tol, lse_tol = attention(cache, q, table, n, window)
    got, got_lse = cache.attend(q, table, n, window=window, return_lse=True)
    within(got, out, tol, "out")
    within(got_lse, lse, lse_tol, "lse")
    cache.check()


# ---------------------------------------------------------------------------
# 4-bit weights
# ---------------------------------------------------------------------------

SHAPES = [(1, 256, 32, 32), (1, 512, 40, 64), (2, 384, 17, 128), (3, 4096, 10000, 128), (20, 512, 40, 32), (40, 256, 300, 256)]


@pytest.mark.parametrize("rows,inner,outer,group", SHAPES)
def test_linear4_largest_numbers_in_fp32(rows, inner, outer, group):
    """Single values of a row at fp32's largest, which is above bf16's largest."""
    g = gen(80)
    packed, scales, z, w = weights(g, outer, inner, group, True, BF16, 2.0 ** -8)
    x = torch.zeros(rows, inner, device="cuda")
    most = torch.finfo(F32).max
    x[:, 7] = most
    x[0, inner - 1] = -most
    x[rows - 1, 20] = 3.395e38  # between the two largest
    w = w.clone()
    y = x.double() @ w.T
    layer = pf.Linear4bit(packed, scales, z, in_features=inner, group_size=group)
    within(layer(x), y, linear_tol(x, w, y, F32, inner, group))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,inner,outer,group", SHAPES)
def test_linear4_sums_beyond_the_largest_number(dtype, rows, inner, outer, group):
    """Groups whose sum of x (q - z) is above the type's largest number, and comes back with the scale."""
    g = gen(81)
    packed, scales, z, w = weights(g, outer, inner, group, True, BF16, 2.0 ** -16)
    x = (torch.rand(rows, inner, generator=g, device="cuda") * 1e38 + 2e38).to(dtype)
    y = x.double() @ w.T
    assert float(y.abs().max()) < 1e38
    layer = pf.Linear4bit(packed, scales, z, in_features=inner, group_size=group)
    within(layer(x), y, linear_tol(x, w, y, dtype, inner, group))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,inner,outer,group", SHAPES)
@pytest.mark.parametrize("size", [2.0 ** -100, 2.0 ** -118])
def test_linear4_smallest_numbers(dtype, rows, inner, outer, group, size):
    """Rows of tiny numbers, of which no bit may be lost where scales bring the result back to the middle. (fp32 values above
    2^-110 split into three normal bf16 numbers; smaller ones lose what is below 2^-134, half of bf16's smallest step.)"""
    g = gen(82)
    packed, scales, z, w = weights(g, outer, inner, group, True, BF16, 2.0 ** 40)
    x = (randn(g, rows, inner) * size).to(dtype)
    y = x.double() @ w.T
    layer = pf.Linear4bit(packed, scales, z, in_features=inner, group_size=group)
    lost = 2.0 ** -134 * w.abs().sum(1) if dtype == F32 else 0.0
    within(layer(x), y, linear_tol(x, w, y, dtype, inner, group) + lost)


@pytest.mark.parametrize("bits", [0x7f800001, 0x7f80ffff, 0x7fc00000, 0x7fffffff])
@pytest.mark.parametrize("rows,inner,outer,group", SHAPES[:5:2])
def test_linear4_any_nan_in_fp32(rows, inner, outer, group, bits):
    """Also a NaN whose only bits are below bf16's, of either sign, makes its row NaN and no other."""
    g = gen(83)
    packed, scales, z, w = weights(g, outer, inner, group, True, BF16)
    x = torch.cat((randn(g, rows, inner), randn(g, 2, inner)))
    x.view(torch.int32)[:2, 9] = torch.tensor([bits, bits - 2 ** 31], dtype=torch.int64, device="cuda").to(torch.int32)
    got = pf.Linear4bit(packed, scales, z, in_features=inner, group_size=group)(x)
    assert bool(got[:2].isnan().all())
    y = x[2:].double() @ w.T
    within(got[2:], y, linear_tol(x[2:], w, y, F32, inner, group))


@pytest.mark.parametrize("dtype,rows,inner,outer,group", [
    (F32, 2, 9000, 19999, 64), (BF16, 5, 9000, 19999, 128), (F16, 7, 8200, 19000, 32), (F32, 1, 16384, 30000, 32), (F16, 1, 4100, 19999, 64)])
def test_linear4_more_row_tiles_than_ctas(dtype, rows, inner, outer, group):
    """CTAs that walk over several tiles of weight rows, with rows of x that are staged again for each, or kept."""
    g = gen(84)
    packed, scales, z, w = weights(g, outer, inner, group, True)
    b = randn(g, outer, dtype=dtype)
    layer = pf.Linear4bit(packed, scales, z, b, in_features=inner, group_size=group)
    x = randn(g, rows, inner, dtype=dtype)
    y = x.double() @ w.T + b.double()
    tol = linear_tol(x, w, y, dtype, inner, group)
    for _ in range(2):
        within(layer(x), y, tol)


# ---------------------------------------------------------------------------
# a layer's calls, each against 64 bits
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
def test_decoding_steps_call_by_call(dtype):
    """Three sequences over 20 steps, one of them joining late: every call of a step against 64 bits from what the call
    before it gave, and tolerances that a swapped row or a wrong slot, page, length or position cannot pass."""
    g = gen(90)
    layer = Layer(g, dtype)
    cache, rotary = layer.cache, layer.rotary
    table = torch.randperm(39, generator=g, device="cuda")[:12].view(3, 4).to(torch.int32)
    stored = [[] for _ in range(3)]  # the keys and values that each sequence's calls were given, rotated in 64 bits

    def close(got, want, tol, what):
        within(got, want, tol, what)
        if bool((want != 0).any()):
            assert float(tol.double().mean()) < 0.02 * float(want.abs().mean()), (what, "a loose tolerance")

    for step in range(20):
        x = randn(g, 3, 256, dtype=dtype)
        pos = torch.tensor([step, step, step - 10], device="cuda")
        live = pos >= 0
        at = pos.clamp(min=0)
        slots = torch.where(live, table[torch.arange(3), at // 8].long() * 8 + at % 8, -1)
        lens = (pos + 1).clamp(min=0).to(torch.int32)
        qkv = layer.qkv(x)
        w = layer.qkv_w[3]
        y = x.double() @ w.T
        close(qkv, y, linear_tol(x, w, y, dtype, 256, 64), f"step {step}: qkv")
        q, k, v = qkv.unflatten(1, (-1, 32)).split([8, 2, 2], 1)
        turned = cache.append(k, v, slots, positions=pos, rotary=rotary, q=q)
        for got, of, heads in ((turned, q, 8), (cache.k.flatten(0, 1)[slots.clamp(min=0)], k, 2)):
            want, mag = turn(of, pos, rotary)
            close(got[live], want[live], turn_tol(want, mag, dtype)[live], f"step {step}: rotated")
        assert torch.equal(cache.v.flatten(0, 1)[slots[live]], v[live]) and bool((turned[~live] == 0).all())
        out = cache.attend(turned, table, lens)
        want, _, tol, _ = attention(cache, turned, table, lens)
        close(out, want, tol, f"step {step}: attention")
        # the cache itself holds what the calls were given, in the order of the positions
        kk = turn(k, pos, rotary)[0]
        for b in range(3):
            if bool(live[b]):
                stored[b].append((kk[b], v[b].double()))
                n = len(stored[b])
                place = table[b, torch.arange(n, device="cuda") // 8].long() * 8 + torch.arange(n, device="cuda") % 8
                want = torch.stack([c[0] for c in stored[b]])
                within(cache.k.flatten(0, 1)[place], want, (HALF[dtype] + 2.0 ** -20) * (want.abs() + want.abs().amax()), "keys")
                assert torch.equal(cache.v.flatten(0, 1)[place].double(), torch.stack([c[1] for c in stored[b]]))
        got = layer.out(out.flatten(1))
        w = layer.out_w[3]
        y = out.flatten(1).double() @ w.T
        close(got, y, linear_tol(out.flatten(1), w, y, dtype, 256, 32), f"step {step}: out")
    cache.check()


# ---------------------------------------------------------------------------
# what a call may not be given
# ---------------------------------------------------------------------------

def _calls(dtype=F32):
    """One call of each kind: (name of the tensor, the call with that tensor, the tensor)."""
    cache, r = pf.PagedKVCache(4, 16, 2, 64, dtype), pf.RotaryEmbedding(64)
    layer = pf.Linear4bit(*weights(gen(95), 64, 64, 64, True)[:3], group_size=64)
    x, pos = randn(gen(96), 3, 2, 64, dtype=dtype), torch.arange(3, device="cuda")
    table, lens = torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    out = torch.empty_like(x)
    return x, [
        ("x", lambda t: r.apply(t, pos)), ("x", lambda t: r.backward(t, pos)), ("out", lambda t: r.apply(x, pos, out=t)),
        ("k", lambda t: cache.append(t, x, pos)), ("v", lambda t: cache.append(x, t, pos)),
        ("q", lambda t: cache.append(x, x, pos, q=t)), ("q_out", lambda t: cache.append(out, out, pos, q=x, q_out=t)),
        ("q", lambda t: cache.attend(t, table, lens)), ("out", lambda t: cache.attend(x, table, lens, out=t)),
        ("x", lambda t: layer(t)), ("x", lambda t: layer(t.flatten(0, 1)[:2])), ("out", lambda t: layer(x, out=t))]


def test_tangents_are_refused():
    """A forward-mode tangent would be lost in silence: refused at the first call and at a known one."""
    import torch.autograd.forward_ad as forward
    x, calls = _calls()
    for known in (False, True):
        for name, call in calls:
            t = torch.empty_like(x)
            if known:
                call(t.copy_(x))
            with forward.dual_level():
                dual = forward.make_dual(t, torch.ones_like(t))
                with pytest.raises(RuntimeError, match="tangent"):
                    call(dual)
                call(t)  # without a tangent it runs there too
    r, pos = pf.RotaryEmbedding(64), torch.arange(3, device="cuda")
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: r.apply(t, pos), (x,), (torch.ones_like(x),))
    bias = torch.zeros(64, device="cuda")
    with forward.dual_level(), pytest.raises(RuntimeError, match="tangent"):
        pf.Linear4bit(*weights(gen(95), 64, 64, 64, True)[:3], bias=forward.make_dual(bias, torch.ones_like(bias)), group_size=64)


def test_overlapping_outputs_are_refused():
    cache, r = pf.PagedKVCache(4, 16, 2, 64), pf.RotaryEmbedding(64)
    layer = pf.Linear4bit(*weights(gen(95), 64, 64, 64, True)[:3], group_size=64)
    pos = torch.arange(3, device="cuda")
    table, lens = torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    buf = torch.zeros(1000, device="cuda")
    at = lambda o: buf[o:o + 384].view(3, 2, 64)
    wide = torch.zeros(3, 6, 64, device="cuda")  # heads of one projection, interleaved in memory with their neighbours
    other = torch.zeros(3, 2, 64, device="cuda")
    for _ in range(2):  # checked for the first time, and as a known call
        for call in (
                lambda: r.apply(at(0), pos, out=at(4)), lambda: r.backward(at(64), pos, out=at(0)),
                lambda: r.apply(wide[:, 0:2], pos, out=wide[:, 1:3]),
                lambda: cache.append(other, other, pos, q=at(0), q_out=at(383)),
                lambda: cache.append(at(0), other, pos, q=other, q_out=at(0)),
                lambda: cache.append(other, at(0), pos, q=other, q_out=at(128)),
                lambda: cache.append(wide[:, 2:4], other, pos, q=wide[:, :2], q_out=wide[:, 1:3]),
                lambda: cache.attend(at(0), table, lens, out=at(64)), lambda: cache.attend(wide[:, 2:4], table, lens, out=wide[:, 3:5]),
                lambda: cache.attend(other, table, lens, out=cache.v[:3, 0]), lambda: cache.attend(other, table, lens, out=cache.k[1:, 3]),
                lambda: layer(buf[:128].view(2, 64), out=buf[127:255].view(2, 64)),
                lambda: layer(buf[64:192].view(2, 64), out=buf[:128].view(2, 64))):
            with pytest.raises(ValueError, match="memory"):
                call()
    for shared in (pf.PagedKVCache.from_tensors(cache.k, cache.k), pf.PagedKVCache.from_tensors(cache.k[:3], cache.k[1:])):
        shared.attend(other, table, lens)
        with pytest.raises(ValueError, match="memory"):
            shared.append(other, other, pos)
    bias = torch.zeros(64, device="cuda")
    biased = pf.Linear4bit(*weights(gen(95), 64, 64, 64, True)[:3], bias=bias, group_size=64)
    with pytest.raises(ValueError, match="memory"):
        biased(torch.zeros(1, 64, device="cuda"), out=bias[None])


def test_neighbouring_outputs_are_taken():
    """Outputs between the inputs' rows in one buffer, and in place of an input, are no overlap."""
    g = gen(97)
    r, pos = pf.RotaryEmbedding(64), torch.arange(3, device="cuda")
    layer = pf.Linear4bit(*weights(g, 64, 64, 64, True)[:3], group_size=64)
    cache, q, table, lens = make_batch(g, [20, 0, 33], 16, 2, 2, 64, F32)
    wide = torch.zeros(3, 8, 64, device="cuda")
    for run in (lambda x, out: r.apply(x, pos, out=out), lambda x, out: cache.attend(x, table, lens, out=out),
                lambda x, out: cache.append(wide[:, 4:6], wide[:, 6:8], torch.full((3,), -1, device="cuda"), q=x, q_out=out)):
        for x, out in ((wide[:, 0:2], wide[:, 2:4]), (wide[:, 2:4], wide[:, 0:2]), (wide[:, 1:3], wide[:, 1:3]), (wide[:, 0:4:2], wide[:, 1:4:2])):
            x.copy_(q)
            out_of = run(q.clone(), None)
            keep = out.clone()
            run(x, out)
            want = out_of if bool((out_of != 0).any()) else keep  # skipped tokens: the rows stay
            assert torch.equal(out, want)
    both = torch.zeros(2, 4, 16, 2, 64, device="cuda").transpose(0, 1)  # keys and values of a page next to each other
    k = randn(g, 3, 2, 64)
    pf.PagedKVCache.from_tensors(both[:, 0], both[:, 1]).append(k, -k, torch.arange(3, device="cuda") * 20)
    for i in range(3):
        assert torch.equal(both[i * 20 // 16, 0, i * 20 % 16], k[i]) and torch.equal(both[i * 20 // 16, 1, i * 20 % 16], -k[i])
    rows = torch.zeros(5, 192, device="cuda")
    rows[:, :64] = randn(g, 5, 64)
    want = layer(rows[:, :64].clone())
    assert torch.equal(layer(rows[:, :64], out=rows[:, 64:128]), want) and torch.equal(layer(rows[::2, :64], out=rows[::2, 128:]), want[::2])


def test_handles_made_in_inference_mode():
    """Made in torch's inference mode and used outside, made outside and used inside."""
    def make():
        cache, r = pf.PagedKVCache(4, 16, 2, 64), pf.RotaryEmbedding(64)
        return cache, r, pf.Linear4bit(*weights(gen(95), 64, 64, 64, True)[:3], group_size=64)

    def use(cache, r, layer):
        x, pos = randn(gen(96), 3, 2, 64), torch.arange(3, device="cuda")
        table, lens = torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
        outs = []
        for _ in range(2):
            q = cache.append(x, x, pos, positions=pos, rotary=r, q=x)
            out, lse = cache.attend(q, table, lens, return_lse=True)
            outs.append((layer(out), lse, r.backward(q, pos)))
        cache.check()
        cache.append(x, x, pos + 1000)
        with pytest.raises(pf._native.PfcError):
            cache.check()
        cache.check()
        return outs

    want = use(*make())
    with torch.inference_mode():
        made = make()
        inside = use(*make())
    outside = use(*made)
    made = make()
    with torch.inference_mode():
        mixed = use(*made)
    for got in (inside, outside, mixed):
        for a, b in zip(sum(got, ()), sum(want, ())):
            assert torch.equal(a, b)


def test_calls_of_no_rows():
    """Nothing to do, with and without a bias, a given output, queries: the first time and as a known call."""
    cache, r = pf.PagedKVCache(4, 16, 2, 64), pf.RotaryEmbedding(64)
    bias = torch.ones(64, device="cuda")
    none, pos = torch.zeros(0, 2, 64, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda")
    table, lens = torch.zeros(0, 3, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    for b in (None, bias):
        layer = pf.Linear4bit(*weights(gen(95), 64, 64, 64, True)[:3], bias=b, group_size=64)
        for out in (None, torch.empty_like(none), none):
            for _ in range(2):
                assert layer(none, out=out).shape == (0, 2, 64) and layer(none[:, 0]).shape == (0, 64)
                assert r.apply(none, pos, out=out).shape == r.backward(none, pos, out=out).shape == (0, 2, 64)
                assert cache.attend(none, table, lens, out=out).shape == (0, 2, 64)
                assert cache.attend(none, table, lens, out=out, return_lse=True)[1].shape == (0, 2)
                assert cache.append(none, none, pos, q=none, q_out=out).shape == (0, 2, 64)
                assert cache.append(none, none, pos, positions=pos, rotary=r) is None
    cache.check()


def test_known_calls_hold_no_memory():
    """What a handle keeps of the calls it knows is of no consequence beside them: no memory for each shape."""
    g = gen(98)
    layer = pf.Linear4bit(*weights(g, 1024, 64, 64, True)[:3], group_size=64)
    cache, q, table, lens = make_batch(g, [1] * 60, 16, 2, 64, 64, F32)
    r = pf.RotaryEmbedding(64)

    def calls():
        for n in range(1, 60):
            layer(torch.zeros(n, 64, device="cuda"))
            cache.attend(q[:n], table[:n], lens[:n], return_lse=True)
            r.apply(q[:n], lens[:n].long())

    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    calls()
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() <= before


# ---------------------------------------------------------------------------
# next to the graph executor
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["default", "side"])
def test_executor_on_torchs_stream(kind):
    """A graph between two of these calls, all in the order of torch's current stream (its default one has the handle 0,
    which names the executor's own stream). Long work goes before each, so that what does not wait reads old data."""
    g = gen(99)
    layer = pf.Linear4bit(*weights(g, 64, 256, 64, True, size=0.1)[:3], group_size=64)
    rotary, pos = pf.RotaryEmbedding(64), torch.arange(8, device="cuda")
    pf.reset_graph()
    shape = [8, 1, 64]
    a = pf.from_numpy(np.random.default_rng(0).standard_normal(shape, np.float32))
    y = pf.relu(a) * pf.from_numpy(np.full(shape, 2.0, np.float32))
    graph, ids, leaf = y.graph(), [y.node().id()], a.node().id()
    ex = pf.CudaExecutor(pf.CudaExecutor.Config())
    stream = torch.cuda.current_stream() if kind == "default" else torch.cuda.Stream()
    hidden, doubled = torch.zeros(8, 64, device="cuda"), torch.zeros(8, 1, 64, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for i in range(5):  # the first as a plan is made, the later ones as a replayed graph
            x = randn(g, 8, 256)
            want = rotary.apply(torch.relu(layer(x)).view(8, 1, 64) * 2, pos)
            hidden.zero_()
            doubled.zero_()
            torch.cuda._sleep(20_000_000)
            layer(x, out=hidden)
            ex.execute_device(graph, {leaf: hidden.data_ptr()}, ids, [doubled.data_ptr()], stream=torch.cuda.current_stream())
            got = rotary.apply(doubled, pos)
            assert torch.equal(got, want), i
    torch.cuda.synchronize()
    ex.close()
