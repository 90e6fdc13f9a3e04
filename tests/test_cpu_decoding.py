"""Token generation without a GPU: what the entry points refuse (before they
touch a device), and the rotary frequencies."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import pyflame_b200 as pf

FAKE = 1 << 20  # never dereferenced: every call here is refused, or has nothing to do, before a launch


def rotary(native, dim=64, inv=FAKE, interleaved=0):
    return native.RotaryC(inv, dim, interleaved, 1.0)


def cache(native, **kw):
    v = dict(dtype=0, k=FAKE, v=FAKE, num_pages=4, page_size=16, heads=2, head_dim=64, page_stride=2048, token_stride=128,
             head_stride=64, err=None)
    v.update(kw)
    return native.PagedCacheC(*v.values())


def refused(native, rc, word):
    assert rc == -1, rc
    assert word in native.lib().pfc_last_error().decode(), native.lib().pfc_last_error()


@pytest.mark.parametrize("change,word", [
    (dict(dtype=3), "dtype"), (dict(batch=-1), "negative"), (dict(head_dim=0), "head_dim"), (dict(head_dim=1025), "head_dim"),
    (dict(tokens=1 << 31), "2^31"), (dict(batch=1 << 20, tokens=1 << 20), "2^31"), (dict(heads=65537), "heads"),
    (dict(inverse=2), "inverse"), (dict(rot=63), "rotary_dim"), (dict(rot=130), "rotary_dim"), (dict(rot=-2), "rotary_dim"),
    (dict(inv=None), "inv_freq"), (dict(interleaved=5), "interleaved"), (dict(positions=None), "positions"), (dict(x=None), "null"),
])
def test_rope_refusals(native, change, word):
    v = dict(x=FAKE, dtype=0, inverse=0, batch=1, tokens=4, heads=2, head_dim=64, positions=FAKE, rot=64, inv=FAKE, interleaved=0)
    v.update(change)
    p = native.RopeParamsC(v["dtype"], v["inverse"], v["batch"], v["tokens"], v["heads"], v["head_dim"], 0, 128, 64, 0, 128, 64,
                           v["positions"], 0, 1, rotary(native, v["rot"], v["inv"], v["interleaved"]))
    refused(native, native.lib().pfk_rope(v["x"], FAKE, C.byref(p), None), word)
    refused(native, native.lib().pfk_rope(FAKE, FAKE, None, None), "null")


def test_nothing_to_do_needs_no_device(native):
    L = native.lib()
    p = native.RopeParamsC(0, 0, 1, 0, 2, 64, 0, 128, 64, 0, 128, 64, None, 0, 1, rotary(native))
    assert L.pfk_rope(None, None, C.byref(p), None) == 0
    a = native.PagedAppendParamsC(cache(native), 0)
    assert L.pfk_paged_append(C.byref(a), None) == 0
    t = native.PagedAttentionParamsC(cache(native), 0, 4)
    assert L.pfk_paged_attention(C.byref(t), None) == 0
    n = C.c_size_t(7)
    assert L.pfk_paged_attention_workspace(C.byref(t), C.byref(n)) == 0 and n.value == 0
    w = native.LinearW4ParamsC(0, 0, 64, 64, 64)
    assert L.pfk_linear_w4(C.byref(w), None) == 0
    r = native.W4ArrangeParamsC(64, 0, 64, None, None, 1)
    assert L.pfk_w4_arrange(C.byref(r), None) == 0


@pytest.mark.parametrize("change,word", [
    (dict(dtype=8), "dtype"), (dict(k=None), "null"), (dict(num_pages=0), "positive"), (dict(page_size=0), "positive"),
    (dict(head_dim=0), "positive"), (dict(num_pages=1 << 20, page_size=1 << 12), "2^31"), (dict(heads=1 << 17), "heads"),
    (dict(token_stride=-1), "negative"),
])
def test_cache_refusals(native, change, word):
    c = cache(native, **change)
    a = native.PagedAppendParamsC(c, 1, FAKE, 1, 1, FAKE, 1, 1)
    a.slots = FAKE
    refused(native, native.lib().pfk_paged_append(C.byref(a), None), word)
    t = native.PagedAttentionParamsC(c, 1, 2, FAKE, 1, 1, FAKE, 1, 1, None, FAKE, 1, 1, FAKE, 0, 1.0)
    refused(native, native.lib().pfk_paged_attention(C.byref(t), None), word)


@pytest.mark.parametrize("change,word", [
    (dict(tokens=-1), "tokens"), (dict(k=None), "null"), (dict(slots=None), "null"), (dict(q=FAKE), "q_out"),
    (dict(q=FAKE, q_out=FAKE, q_heads=-1), "q_heads"), (dict(rotary=65), "rotary_dim"), (dict(rotary=64), "positions"),
])
def test_append_refusals(native, change, word):
    v = dict(tokens=3, k=FAKE, slots=FAKE, q=None, q_out=None, q_heads=2, rotary=0)
    v.update(change)
    p = native.PagedAppendParamsC(cache(native), v["tokens"], v["k"], 128, 64, FAKE, 128, 64, v["q"], v["q_out"], v["q_heads"])
    p.slots, p.rotary = v["slots"], rotary(native, v["rotary"])
    refused(native, native.lib().pfk_paged_append(C.byref(p), None), word)


@pytest.mark.parametrize("change,word", [
    (dict(head_dim=60), "head_dim"), (dict(head_dim=264), "head_dim"), (dict(k=FAKE + 8), "16 bytes"),
    (dict(token_stride=130), "16 bytes"), (dict(dtype=1, head_stride=68), "16 bytes"), (dict(q_heads=3), "q_heads"),
    (dict(q_heads=0), "q_heads"), (dict(batch=-1), "q_heads"), (dict(batch=1 << 30), "2^31"), (dict(window=-1), "window"),
    (dict(scale=math.nan), "scale"), (dict(width=-1), "table"), (dict(q=None), "null"), (dict(table=None), "null"),
    (dict(lens=None), "null"),
])
def test_attention_refusals(native, change, word):
    v = dict(batch=2, q_heads=4, q=FAKE, table=FAKE, width=4, lens=FAKE, window=0, scale=0.125)
    c = cache(native, **{k: x for k, x in change.items() if k not in v})
    v.update({k: x for k, x in change.items() if k in v})
    p = native.PagedAttentionParamsC(c, v["batch"], v["q_heads"], v["q"], 256, 64, FAKE, 256, 64, None, v["table"], 4, v["width"],
                                     v["lens"], v["window"], v["scale"])
    refused(native, native.lib().pfk_paged_attention(C.byref(p), None), word)
    refused(native, native.lib().pfk_paged_attention(None, None), "null")


@pytest.mark.parametrize("strides", [(128, 64), (256, 128)])
def test_attention_into_queries_with_other_strides(native, strides):
    p = native.PagedAttentionParamsC(cache(native), 2, 4, FAKE, 256, 64, FAKE, *strides, None, FAKE, 4, 4, FAKE, 0, 0.125)
    refused(native, native.lib().pfk_paged_attention(C.byref(p), None), "strides")


@pytest.mark.parametrize("change,word", [
    (dict(dtype=7), "dtype"), (dict(rows=-1), "rows"), (dict(rows=(1 << 20) + 1), "rows"),
    (dict(inner=0), "inner"), (dict(outer=0), "inner"), (dict(group=16), "group"), (dict(group=96), "group"), (dict(group=192), "group"),
    (dict(x=None), "null"), (dict(weight=None), "null"), (dict(weight=FAKE + 4), "aligned"), (dict(meta=None), "null"),
    (dict(meta=FAKE + 8), "aligned"),
])
def test_linear_refusals(native, change, word):
    v = dict(dtype=0, rows=1, inner=256, outer=32, group=128, x=FAKE, x_st=256, y=FAKE, y_st=32, weight=FAKE, meta=FAKE,
             bias=None)
    v.update(change)
    p = native.LinearW4ParamsC(*v.values())
    refused(native, native.lib().pfk_linear_w4(C.byref(p), None), word)
    refused(native, native.lib().pfk_linear_w4(None, None), "null")


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_linear_rows_of_one_grid(native, dtype):
    p = native.LinearW4ParamsC(dtype, 65535 * 16 + 1, 256, 32, 128, FAKE, 256, FAKE, 32, FAKE, FAKE, None)
    refused(native, native.lib().pfk_linear_w4(C.byref(p), None), "rows")


@pytest.mark.parametrize("args,word", [
    ((64, 4, 64, None, FAKE, 1, None, FAKE, FAKE), "null"), ((64, 4, 64, FAKE, FAKE, 1, None, FAKE, None), "null"),
    ((64, -4, 64, FAKE, FAKE, 1, None, FAKE, FAKE), "size"), ((64, 4, 48, FAKE, FAKE, 1, None, FAKE, FAKE), "group"),
    ((64, 4, 64, FAKE, FAKE, 0, None, FAKE, FAKE), "scale_dtype")])
def test_arrange_refusals(native, args, word):
    p = native.W4ArrangeParamsC(*args)
    refused(native, native.lib().pfk_w4_arrange(C.byref(p), None), word)
    refused(native, native.lib().pfk_w4_arrange(None, None), "null")


def test_host_tensors_are_refused(native):
    x = torch.zeros(1, 2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        pf.RotaryEmbedding(64, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        pf.PagedKVCache(2, 4, 1, 8, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        pf.PagedKVCache.from_tensors(x[None], x[None])
    with pytest.raises(ValueError, match="CUDA"):
        pf.Linear4bit(torch.zeros(4, 64, dtype=torch.uint8), torch.ones(4, 1))


def test_rotary_frequencies():
    inv, f = pf.rotary_frequencies(64, 10000.0)
    np.testing.assert_allclose(inv, [10000.0 ** (-i / 32) for i in range(32)], rtol=1e-15)
    assert f == 1.0 and inv.dtype == np.float64
    lin, f = pf.rotary_frequencies(64, scaling={"type": "linear", "factor": 4})
    np.testing.assert_allclose(lin, inv / 4, rtol=1e-15)
    ntk, f = pf.rotary_frequencies(64, scaling={"type": "ntk", "factor": 4})
    assert ntk[0] == 1.0 and f == 1.0
    np.testing.assert_allclose(ntk[-1], inv[-1] / 4, rtol=1e-12)  # base^(-(d-2)/d) * f^(-1)
    yarn, f = pf.rotary_frequencies(64, scaling={"type": "yarn", "factor": 4, "original_max_position": 4096})
    assert f == pytest.approx(0.1 * math.log(4) + 1)
    turns = 4096 * inv / (2 * math.pi)
    assert (yarn[turns > 33] == inv[turns > 33]).all() and np.allclose(yarn[turns < 0.5], inv[turns < 0.5] / 4, rtol=1e-15)
    assert ((yarn <= inv) & (yarn >= inv / 4 * (1 - 1e-15))).all() and (np.diff(yarn) < 0).all()
    assert pf.rotary_frequencies(0)[0].shape == (0,)


@pytest.mark.parametrize("args", [
    (63,), (-2,), (64, 0.0), (64, 1.0), (64, math.inf), (64, 1e4, {"type": "spiral", "factor": 2}), (64, 1e4, {"type": "linear"}),
    (64, 1e4, {"type": "linear", "factor": 0.5}), (64, 1e4, {"type": "linear", "factor": 2, "beta": 1}),
    (2, 1e4, {"type": "ntk", "factor": 2}), (64, 1e4, {"type": "yarn", "factor": 2}),
    (64, 1e4, {"type": "yarn", "factor": 2, "original_max_position": 64, "beta_fast": 1, "beta_slow": 1}),
])
def test_rotary_frequencies_refusals(args):
    with pytest.raises(ValueError):
        pf.rotary_frequencies(*args)
