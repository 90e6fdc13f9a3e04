"""The mixture-of-experts layer on the GPU against 64 bits.

Tolerances count roundings.  eps(t)/2 of the result is the output's own.  A
sum in the tensor cores loses at most 2^-23 of what has been added for each
instruction, a piece's few, and pieces are added up in fp32, at most some
hundred times (2^-24 each); fp32 operands come in parts that lose 2^-21: below
2^-17 of the sum of magnitudes.  Gate and up enter act(g) u with their errors
(|act'| below 1.2), which is held to 2^-17 in bfloat16's two parts.  The
weights' exponentials and their sum: 2^-19.  2^-15 of all magnitudes covers
the sum of these.
"""
import math

import pytest
import torch

import pyflame_b200 as pf

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
HALF = {t: torch.finfo(t).eps / 2 for t in TYPES}
TINY = {F32: 0.0, F16: 2.0 ** -25, BF16: 0.0}


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


def weights(g, e, d, f, dtype):
    return (randn(g, e, d) / math.sqrt(d)).to(dtype), (randn(g, e, 2 * f, d) / math.sqrt(d)).to(dtype), (randn(g, e, d, f) / math.sqrt(f)).to(dtype)


def routing(x, router, top, renormalize):
    """Chosen experts and their weights in 64 bits; ties to the lower expert."""
    logits = x.double() @ router.double().T
    values, chosen = torch.sort(logits, dim=-1, descending=True, stable=True)
    chosen = chosen[:, :top]
    p = torch.softmax(logits, -1).gather(-1, chosen)
    return chosen, p / p.sum(-1, keepdim=True) if renormalize else p


def reference(x, router, gate_up, down, top, renormalize, activation):
    chosen, part = routing(x, router, top, renormalize)
    x, f = x.double(), down.shape[-1]
    y, mag = torch.zeros_like(x), torch.zeros_like(x)
    for e in chosen.unique().tolist():
        n, j = (chosen == e).nonzero(as_tuple=True)
        w, both = gate_up[e].double(), x[n] @ gate_up[e].double().T
        size = x[n].abs() @ w.abs().T
        gate, up = both[:, :f], both[:, f:]
        act = torch.nn.functional.silu(gate) if activation == "silu" else torch.nn.functional.gelu(gate, approximate="tanh")
        h, hm = act * up, (act * up).abs() + 1.2 * size[:, :f] * up.abs() + act.abs() * size[:, f:] + 2.0 ** -17 * size[:, :f] * size[:, f:]
        share = part[n, j][:, None]
        y.index_add_(0, n, share * (h @ down[e].double().T))
        mag.index_add_(0, n, share * (hm @ down[e].double().abs().T))
    return y, mag, chosen, part


def check(layer, x, ws, **kw):
    t = x.dtype
    keep = x.clone()
    y, chosen, part = layer(x, return_routing=True, **kw)
    rows = keep.reshape(-1, layer.width)
    want, mag, c, p = reference(rows, *ws, layer.top_k, layer.renormalize, layer.activation)
    assert chosen.dtype == torch.int32 and torch.equal(chosen.reshape(-1, layer.top_k).long(), c)
    # (below 2^-126 fp32 comes in steps of 2^-149: an exponential's two and the quotient's half)
    within(part.reshape(-1, layer.top_k), p, 2.0 ** -18 * p + 2.5 * 2.0 ** -149)
    within(y.reshape(-1, layer.width), want, HALF[t] * want.abs() + 2.0 ** -15 * mag + TINY[t])
    return y


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,e,top,d,f", [(1, 8, 2, 768, 256), (1, 64, 6, 512, 96), (1, 1, 1, 64, 64), (3, 4, 4, 100, 60), (4, 16, 1, 65, 33), (5, 16, 2, 2100, 40),
                                              (8, 8, 3, 256, 512), (9, 8, 2, 128, 256), (17, 4, 1, 96, 72), (33, 128, 8, 160, 48), (64, 16, 2, 333, 77),
                                              (100, 2, 2, 64, 40), (128, 60, 4, 72, 24), (129, 8, 2, 64, 32), (300, 5, 3, 40, 17), (2, 1024, 32, 32, 16),
                                              (7, 1000, 5, 24, 8), (6, 100, 7, 1, 1), (20, 33, 32, 8, 9)])
def test_layer(dtype, tokens, e, top, d, f):
    g = gen(tokens + e + d)
    ws = weights(g, e, d, f, dtype)
    x = randn(g, tokens, d, dtype=dtype)
    for renormalize, activation in ((True, "silu"), (False, "gelu")):
        layer = pf.MixtureOfExperts(*ws, top, renormalize=renormalize, activation=activation)
        y = check(layer, x, ws)
        assert torch.equal(layer(x), y)


@pytest.mark.parametrize("dtype", TYPES)
def test_all_tokens_choose_the_same(dtype):
    """Every pair of one expert: parts of 8 and of 16 pairs, also not full ones."""
    g = gen(2)
    router, gate_up, down = weights(g, 8, 64, 48, dtype)
    router[3] = 40 * router[3].abs()
    layer = pf.MixtureOfExperts(router, gate_up, down, 1)
    for tokens in (1, 4, 7, 8, 9, 16, 17, 31, 33, 128):
        x = randn(g, tokens, 64, dtype=dtype).abs()
        y = check(layer, x, (router, gate_up, down))
        assert (layer(x, return_routing=True)[1] == 3).all()


def test_ties_and_a_router_in_fp32():
    g = gen(3)
    router, gate_up, down = weights(g, 12, 64, 16, BF16)
    router = torch.randn(12, 64, generator=g, device="cuda")
    router[7] = router[2]
    router[9] = router[2]
    router[0] = -0.0 * router[0]
    router[11] = 0.0
    x = randn(g, 10, 64, dtype=BF16)
    layer = pf.MixtureOfExperts(router, gate_up, down, 5)
    check(layer, x, (router, gate_up, down))
    x[4] = 0  # every logit equal
    y, chosen, part = layer(x, return_routing=True)
    assert chosen[4].tolist() == [0, 1, 2, 3, 4] and torch.allclose(part[4], torch.full_like(part[4], 0.2)) and not y[4].any()


def test_nan_stays_in_its_token():
    g = gen(4)
    for dtype in TYPES:
        ws = weights(g, 8, 96, 40, dtype)
        layer = pf.MixtureOfExperts(*ws, 3)
        for tokens in (3, 20):
            x = randn(g, tokens, 96, dtype=dtype)
            _, chosen, part = layer(x, return_routing=True)
            x[1, 5] = float("nan")
            y, c, p = layer(x, return_routing=True)
            rest = torch.arange(tokens, device="cuda") != 1
            assert torch.equal(c[rest], chosen[rest]) and y[1].isnan().all()
            # not the same bits: token 1 chooses others, and the sums over all pieces of the experts in
            # use are shared out among warps at other places, each share rounded by itself
            exact, mag, _, _ = reference(x[rest], *ws, 3, True, "silu")
            within(y[rest], exact, HALF[dtype] * exact.abs() + 2.0 ** -15 * mag + TINY[dtype])
            assert ((c >= 0) & (c < 8)).all() and c[1].unique().numel() == 3
        bad = ws[1].clone()
        bad[2] = float("nan")
        x = randn(g, 20, 96, dtype=dtype)
        y, c, _ = pf.MixtureOfExperts(ws[0], bad, ws[2], 3)(x, return_routing=True)
        hit = (c == 2).any(-1)
        assert y[hit].isnan().all() and torch.equal(y[~hit], layer(x)[~hit])


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(dtype):
    g = gen(5)
    ws = weights(g, 6, 72, 36, dtype)
    layer = pf.MixtureOfExperts(*ws, 2)
    x = randn(g, 3, 4, 72, dtype=dtype)
    want = check(layer, x, ws)
    wide = randn(g, 3, 4, 100, dtype=dtype)
    wide[..., 5:77] = x
    assert torch.equal(layer(wide[..., 5:77]), want)
    view, keep = wide[..., 5:77], wide.clone()
    assert layer(view, out=view) is view and torch.equal(view, want)
    assert torch.equal(wide[..., :5], keep[..., :5]) and torch.equal(wide[..., 77:], keep[..., 77:])
    assert torch.equal(layer(x.transpose(0, 1)), layer(x.transpose(0, 1).contiguous()))
    one, c, p = layer(x[0, 0], return_routing=True)
    assert one.shape == (72,) and c.shape == (2,) and torch.equal(one, layer(x[0, 0][None])[0])
    empty = layer(x[:0], return_routing=True)
    assert empty[0].shape == (0, 4, 72) and empty[1].shape == (0, 4, 2)
    # weights in other places: slices, transposed, not aligned
    big = torch.zeros(6, 72, 80, device="cuda", dtype=dtype)
    big[..., 3:75] = ws[1]
    turned = ws[2].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(pf.MixtureOfExperts(ws[0], big[..., 3:75], turned, 2)(x), want)


def test_weights_are_used_where_they_are():
    g = gen(6)
    ws = weights(g, 4, 64, 32, F16)
    layer = pf.MixtureOfExperts(*ws, 2)
    assert layer.gate_up.data_ptr() == ws[1].data_ptr() and layer.down.data_ptr() == ws[2].data_ptr()
    ws[2].mul_(2)
    x = randn(g, 3, 64, dtype=F16)
    check(layer, x, ws)


def test_a_token_does_not_depend_on_the_others_choices():
    """Its bits are the same whichever tokens are beside it, as long as the kernels are."""
    g = gen(7)
    ws = weights(g, 16, 128, 64, BF16)
    layer = pf.MixtureOfExperts(*ws, 2)
    x = randn(g, 40, 128, dtype=BF16)
    want = layer(x)
    order = torch.randperm(40, generator=g, device="cuda")
    got = layer(x[order])
    # the pieces of the output's rows are shared out by the experts in use, which stay the same
    assert torch.equal(got, want[order])


def test_same_bits_streams_and_graphs():
    g = gen(8)
    ws = weights(g, 32, 256, 128, BF16)
    layer = pf.MixtureOfExperts(*ws, 4)
    for tokens in (1, 6, 50):
        x = [randn(g, tokens, 256, dtype=BF16) for _ in range(2)]
        want = [layer(v) for v in x]
        torch.cuda.synchronize()
        streams, got = [torch.cuda.Stream() for _ in range(2)], [None, None]
        for _ in range(5):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[i] = layer(x[i])
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        graphs, outs, ins = [], [], [v.clone() for v in x]
        for i in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(layer(ins[i], return_routing=True))
            graphs.append(graph)
        ins[0].copy_(x[1])
        ins[1].copy_(x[0])
        torch.cuda.synchronize()
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0][0], want[1]) and torch.equal(outs[1][0], want[0])
        assert torch.equal(outs[0][1], layer(x[1], return_routing=True)[1])


@pytest.mark.parametrize("dtype", TYPES)
def test_large_intermediate_values(dtype):
    """Products of gate and up far from 1; in float16 an infinity above 65504, as in a layer of float16."""
    g = gen(9)
    router, gate_up, down = weights(g, 4, 64, 32, dtype)
    gate_up = (gate_up.float() * 40).to(dtype)
    layer = pf.MixtureOfExperts(router, gate_up, down, 2)
    check(layer, randn(g, 5, 64, dtype=dtype), (router, gate_up, down))
    big = (randn(g, 5, 64) * 100).to(dtype)
    y = layer(big)
    if dtype == F16:
        assert not y.isfinite().all()
    else:
        check(layer, big, (router, gate_up, down))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,e,top,d,f", [(1, 8, 4, 64, 100), (6, 4, 2, 2048, 33), (8, 8, 3, 72, 256), (9, 4, 2, 128, 64), (40, 6, 3, 96, 200), (130, 3, 2, 40, 24),
                                              (64, 16, 2, 333, 77)])
@pytest.mark.parametrize("mixed", [False, True])
def test_between_the_products(dtype, tokens, e, top, d, f, mixed):
    """Products of gate and up from 1e-7 to 1e8 in size, which down brings back: by expert, and, `mixed`, also from one
    value to the next.  In float16 the parts of 8 values, which come in steps of 2^-24, have a power of two that leaves
    the largest at 2^-8 at least: they lose 2^-17 of it, and so does what makes the powers of 32 values the same:
    2^-16 of the largest of 32 for each."""
    g = gen(tokens + f)
    router, gate_up, down = (w.float() for w in weights(g, e, d, f, dtype))
    size = torch.tensor([1.0, 3e3, 1e-3, 40.0, 0.05], device="cuda")[torch.arange(e, device="cuda") % 5]
    size = size[:, None].expand(e, f).clone()
    if mixed:
        size *= 2.0 ** torch.randint(-4, 3, (e, f), generator=g, device="cuda")
    gate_up = (gate_up * torch.cat([size, size], 1)[..., None]).clamp(-6e4, 6e4).to(dtype)
    if mixed:
        gate_up[:, :f:5] = 0
    down = (down / (size * size).clamp(1e-7, 1e5)[:, None]).clamp(-6e4, 6e4).to(dtype)
    x = randn(g, tokens, d, dtype=dtype)
    ws = router.to(dtype), gate_up, down
    layer = pf.MixtureOfExperts(*ws, top)
    y, chosen, part = layer(x, return_routing=True)
    want, mag, c, p = reference(x, *ws, top, True, "silu")
    assert torch.equal(chosen.long(), c)
    lost = torch.zeros_like(mag)
    if dtype == F16:
        for i in range(e):
            n, j = (c == i).nonzero(as_tuple=True)
            both = x[n].double() @ gate_up[i].double().T
            h = torch.nn.functional.silu(both[:, :f]) * both[:, f:] * p[n, j][:, None]
            pad = lambda t: torch.nn.functional.pad(t.abs(), (0, -f % 32)).unflatten(-1, (-1, 32))
            lost.index_add_(0, n, 2.0 ** -16 * pad(h).amax(-1) @ pad(down[i].double()).sum(-1).T)
    within(y, want, HALF[dtype] * want.abs() + 2.0 ** -15 * mag + TINY[dtype] + lost)
    assert y.isfinite().all() and torch.equal(layer(x), y)


def test_refusals():
    g = gen(10)
    r, u, d = weights(g, 4, 64, 32, F16)
    for args, err in [((r, u, d, 0), ValueError), ((r, u, d, 5), ValueError), ((r[:3], u, d, 2), ValueError), ((r, u[:, :63], d, 2), ValueError),
                      ((r, u, d.float(), 2), TypeError), ((r, u, d[:, :, :31], 2), ValueError), ((r.double(), u, d, 2), TypeError),
                      ((r, u.cpu(), d, 2), ValueError), ((r.cpu(), u, d, 2), ValueError), ((r, u.double(), d.double(), 2), TypeError)]:
        with pytest.raises(err):
            pf.MixtureOfExperts(*args)
    with pytest.raises(ValueError, match="activation"):
        pf.MixtureOfExperts(r, u, d, 2, activation="relu")
    layer = pf.MixtureOfExperts(r, u, d, 2)
    x = torch.zeros(3, 64, device="cuda", dtype=F16)
    for bad, err in [(dict(x=x.float()), TypeError), (dict(x=x[:, :63]), ValueError), (dict(x=x.cpu()), ValueError), (dict(out=x[:2]), ValueError),
                     (dict(out=x.float()), TypeError), (dict(x=x.clone().requires_grad_()), RuntimeError), (dict(out=x[:1].expand(3, 64)), ValueError)]:
        with pytest.raises(err):
            layer(**{**dict(x=x), **bad})
    memory = torch.zeros(3, 100, device="cuda", dtype=F16)
    with pytest.raises(ValueError, match="shares memory"):
        layer(memory[:, :64], out=memory[:, 36:])
