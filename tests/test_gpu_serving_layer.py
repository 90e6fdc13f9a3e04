"""A decoder layer of a serving step, its calls one behind the other: 4-bit
projections with the adapters of each request beside them, the 4-bit cache,
and a mixture of experts, while sequences grow.  Each call is checked against
64 bits from what the call before it gave."""
import pytest
import torch

import pyflame_b200 as pf

from . import test_gpu_adapters as adapters
from . import test_gpu_cache4bit as cache4
from . import test_gpu_experts as experts

pytestmark = pytest.mark.gpu
WIDTH, HEADS, KV, DIM, PAGE = 256, 8, 2, 64, 16


class Layer:
    def __init__(self, dtype, requests=4):
        g = self.g = adapters.gen(21)
        self.dtype = dtype
        qkv_width = (HEADS + 2 * KV) * DIM
        self.qkv = pf.Linear4bit.quantize(adapters.randn(g, qkv_width, WIDTH) / 16, group_size=64)
        self.out = pf.Linear4bit.quantize(adapters.randn(g, WIDTH, HEADS * DIM) / 23, group_size=64)
        self.qkv_adapters, self.qkv_parts = adapters.make(g, 3, WIDTH, qkv_width, [16, 8], dtype)
        self.out_adapters, self.out_parts = adapters.make(g, 3, HEADS * DIM, WIDTH, [8], dtype, most=16)
        self.weights = experts.weights(g, 8, WIDTH, 96, dtype)
        self.experts = pf.MixtureOfExperts(*self.weights, 2)
        self.rotary = pf.RotaryEmbedding(DIM)
        self.cache = pf.PagedKVCache4bit(64, PAGE, KV, DIM, group_size=32)
        self.index = torch.tensor([2, -1, 0, 1], dtype=torch.int32, device="cuda")[:requests]
        self.table = torch.randperm(64, generator=g, device="cuda").int()[:requests * 8].view(requests, 8)
        self.lens = torch.zeros(requests, dtype=torch.int32, device="cuda")
        self.slots = torch.zeros(requests, dtype=torch.int64, device="cuda")
        self.positions = torch.zeros(requests, dtype=torch.int64, device="cuda")

    def place(self, lens):
        """Where the sequences' newest tokens go."""
        at = torch.tensor(lens, device="cuda") - 1
        self.lens.copy_(at + 1)
        self.positions.copy_(at)
        self.slots.copy_(self.table.gather(1, (at // PAGE)[:, None]).long()[:, 0] * PAGE + at % PAGE)

    def step(self, x, seen=None):
        seen = {} if seen is None else seen
        qkv = seen["qkv"] = self.qkv(x)
        qkv = seen["qkv2"] = self.qkv_adapters(x, self.index, qkv)
        q, k, v = qkv.unflatten(1, (-1, DIM)).split([HEADS, KV, KV], 1)
        q = seen["q"] = self.cache.append(k, v, self.slots, positions=self.positions, rotary=self.rotary, q=q)
        o = seen["o"] = self.cache.attend(q, self.table, self.lens)
        y = self.out(o.flatten(1))
        y = seen["y"] = self.out_adapters(o.flatten(1), self.index, y, out=y)
        return self.experts(y)


@pytest.mark.parametrize("dtype", cache4.TYPES)
def test_every_call_of_growing_sequences(dtype):
    layer = Layer(dtype)
    lens = [1, 14, 15, 60]
    for s, n in enumerate(lens):  # the prompts but for their last tokens
        for i in range(n - 1):
            slots = (layer.table[s, i // PAGE].long() * PAGE + i % PAGE)[None]
            k, v = (adapters.randn(layer.g, 1, KV, DIM, dtype=dtype) for _ in range(2))
            layer.cache.append(k, v, slots, positions=torch.tensor([i], device="cuda"), rotary=layer.rotary)
    for _ in range(5):
        layer.place(lens)
        x, seen = adapters.randn(layer.g, 4, WIDTH, dtype=dtype), {}
        z = layer.step(x, seen)
        want, mag = adapters.reference(layer.qkv_parts, x, layer.index, seen["qkv"], layer.qkv.out_features)
        adapters.within(seen["qkv2"], want, adapters.HALF[dtype] * want.abs() + adapters.SUMS[dtype] * mag, "qkv")
        out, _, errs, mags = cache4.reference(layer.cache, seen["q"], layer.table, layer.lens, DIM ** -0.5, 0)
        cache4.within(seen["o"], out, cache4.HALF[dtype] * out.abs() + cache4.TINY[dtype] + (2 * errs[..., None] + cache4.WEIGHT[dtype]) * mags, "o")
        flat = seen["o"].flatten(1)
        want, mag = adapters.reference(layer.out_parts, flat, layer.index, layer.out(flat), WIDTH)
        adapters.within(seen["y"], want, adapters.HALF[dtype] * want.abs() + adapters.SUMS[dtype] * mag, "y")
        want, mag, _, _ = experts.reference(seen["y"], *layer.weights, 2, True, "silu")
        experts.within(z, want, experts.HALF[dtype] * want.abs() + 2.0 ** -15 * mag + experts.TINY[dtype], "z")
        lens = [n + 1 for n in lens]
    for c in (layer.cache, layer.qkv_adapters, layer.out_adapters):
        c.check()


def test_captured_steps_give_the_same_bits():
    """The whole step in one graph, replayed while an eager copy of the layer takes the same steps."""
    a, b = Layer(cache4.BF16), Layer(cache4.BF16)
    x = torch.zeros(4, WIDTH, device="cuda", dtype=cache4.BF16)
    b.place([1, 1, 1, 1])
    for _ in range(3):
        b.step(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = b.step(x)
    for n in range(1, 40):
        lens = [n, n + 3, 1 + n // 2, n]
        new = adapters.randn(a.g, 4, WIDTH, dtype=cache4.BF16)
        a.place(lens)
        b.place(lens)
        x.copy_(new)
        want = a.step(new)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), n
    b.cache.check()
