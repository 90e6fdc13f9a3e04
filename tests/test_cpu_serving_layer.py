"""The 4-bit cache, adapters and experts without a GPU: what the entry points
refuse (before they touch a device), and calls that have nothing to do."""
import ctypes as C

import pytest
import torch

import pyflame_b200 as pf

FAKE = 1 << 20  # never dereferenced: every call here is refused, or has nothing to do, before a launch


def refused(native, rc, word):
    assert rc == -1, rc
    assert word in native.lib().pfc_last_error().decode(), native.lib().pfc_last_error()


def cache(native, **kw):
    v = dict(k=FAKE, v=FAKE, k_scales=FAKE, v_scales=FAKE, num_pages=4, page_size=16, heads=2, head_dim=64, group=64, err=None)
    v.update({k: x for k, x in kw.items() if k in v})
    return native.Cache4C(*v.values())


CACHE = [(dict(num_pages=0), "positive"), (dict(page_size=0), "positive"), (dict(heads=0), "positive"), (dict(head_dim=0), "head_dim"),
         (dict(head_dim=60), "head_dim"), (dict(head_dim=264), "head_dim"), (dict(group=16), "group"), (dict(group=96), "group"),
         (dict(num_pages=1 << 20, page_size=1 << 11), "2^31"), (dict(num_pages=1 << 26, heads=65), "2^32"), (dict(heads=65537), "2^32"),
         (dict(k=None), "null"), (dict(v=None), "null"), (dict(k_scales=None), "null"), (dict(v_scales=None), "null"),
         (dict(k=FAKE + 8), "aligned"), (dict(v_scales=FAKE + 4), "aligned")]


@pytest.mark.parametrize("change,word", CACHE + [
    (dict(dtype=3), "dtype"), (dict(tokens=-1), "tokens"), (dict(tokens=1 << 31), "tokens"), (dict(q_heads=65537), "q_heads"),
    (dict(q=None), "together"), (dict(q_out=None), "together"), (dict(rot=63), "rotary_dim"), (dict(rot=66), "rotary_dim"),
    (dict(rot=-2), "rotary_dim"), (dict(inv=None), "inv_freq"), (dict(interleaved=2), "interleaved"), (dict(tk=None), "null"),
    (dict(tv=None), "null"), (dict(slots=None), "null"), (dict(positions=None), "positions"), (dict(k_st=-1), "negative"),
    (dict(q=FAKE, q_out=FAKE, qo_st=999), "strides"),
])
def test_append_refusals(native, change, word):
    v = dict(dtype=0, tokens=4, tk=FAKE, k_st=128, tv=FAKE, q=FAKE, q_out=2 * FAKE, q_heads=4, qo_st=256, slots=FAKE, positions=FAKE,
             rot=64, inv=FAKE, interleaved=0)
    v.update(change)
    p = native.Cache4AppendParamsC(cache(native, **change), v["dtype"], v["tokens"], v["tk"], v["k_st"], 64, v["tv"], 128, 64, v["q"], v["q_out"],
                                   v["q_heads"], 256, 64, v["qo_st"], 64, v["slots"], v["positions"],
                                   native.RotaryC(v["inv"], v["rot"], v["interleaved"], 1.0), 1.0)
    refused(native, native.lib().pfk_cache4_append(C.byref(p), None), word)


@pytest.mark.parametrize("change,word", CACHE + [
    (dict(dtype=7), "dtype"), (dict(tokens=-1), "tokens"), (dict(slots=None), "null"), (dict(ok=None), "null"), (dict(ov=None), "null"),
    (dict(ok=FAKE + 8), "aligned")])
def test_read_refusals(native, change, word):
    v = dict(dtype=1, tokens=4, slots=FAKE, ok=FAKE, ov=FAKE)
    v.update(change)
    p = native.Cache4ReadParamsC(cache(native, **change), v["dtype"], v["tokens"], v["slots"], v["ok"], v["ov"])
    refused(native, native.lib().pfk_cache4_read(C.byref(p), None), word)


@pytest.mark.parametrize("change,word", CACHE + [
    (dict(dtype=5), "dtype"), (dict(batch=-1), "q_heads"), (dict(q_heads=3), "multiple"), (dict(q_heads=0), "multiple"),
    (dict(q_heads=65538), "65536"), (dict(batch=1 << 28), "too many"), (dict(table_width=-1), "table"), (dict(table_stride=-1), "table"),
    (dict(window=-1), "window"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(q=None), "null"),
    (dict(out=None), "null"), (dict(lens=None), "null"), (dict(table=None), "null"), (dict(o_sb=-1), "negative"),
    (dict(out=FAKE, o_sb=999), "strides")])
def test_attention_refusals(native, change, word):
    v = dict(dtype=0, batch=2, q_heads=4, q=FAKE, out=2 * FAKE, o_sb=256, table=FAKE, table_stride=8, table_width=8, lens=FAKE, window=0, scale=0.1)
    v.update(change)
    p = native.Cache4AttentionParamsC(cache(native, **change), v["dtype"], v["batch"], v["q_heads"], v["q"], 256, 64, v["out"], v["o_sb"], 64, None,
                                      v["table"], v["table_stride"], v["table_width"], v["lens"], v["window"], v["scale"], None, 0)
    refused(native, native.lib().pfk_cache4_attention(C.byref(p), None), word)


def test_words(native):
    L, a, b = native.lib(), C.c_int64(0), C.c_int64(0)
    for dim, group, codes, scales in [(8, 32, 8, 2), (64, 32, 8, 2), (64, 128, 8, 1), (72, 32, 12, 4), (96, 64, 12, 2), (96, 128, 12, 1),
                                      (128, 32, 16, 4), (128, 64, 16, 2), (136, 32, 32, 8), (256, 128, 32, 2)]:
        assert L.pfk_cache4_words(dim, group, C.byref(a), C.byref(b)) == 0 and (a.value, b.value) == (codes, scales)
    refused(native, L.pfk_cache4_words(12, 32, C.byref(a), C.byref(b)), "head_dim")
    refused(native, L.pfk_cache4_words(64, 48, C.byref(a), C.byref(b)), "group")
    refused(native, L.pfk_cache4_words(64, 64, None, C.byref(b)), "null")


@pytest.mark.parametrize("change,word", [
    (dict(dtype=3), "dtype"), (dict(rows=-1), "rows"), (dict(rows=(1 << 31) - 1), "rows"), (dict(inner=0), "inner"), (dict(outer=0), "outer"),
    (dict(inner=1 << 25), "inner"), (dict(adapters=0), "number"), (dict(rank=0), "rank"), (dict(rank=8), "rank"), (dict(rank=24), "rank"),
    (dict(rank=272), "rank"), (dict(x_st=-1), "negative"), (dict(out_st=-1), "negative"), (dict(a_st=60), "padded"), (dict(a_st=66), "padded"),
    (dict(x=None), "null"), (dict(index=None), "null"), (dict(out=None), "null"), (dict(a=None), "null"), (dict(b=None), "null"),
    (dict(scales=None), "null"), (dict(a=FAKE + 8), "aligned"), (dict(b=FAKE + 4), "aligned"), (dict(out=FAKE, base=FAKE, out_st=65), "stride")])
def test_adapters_refusals(native, change, word):
    v = dict(dtype=0, rows=4, inner=64, outer=64, adapters=2, rank=16, x=FAKE, x_st=64, index=FAKE, base=FAKE, base_st=64, out=2 * FAKE, out_st=64,
             a=FAKE, a_st=64, b=FAKE, scales=FAKE, err=None)
    v.update(change)
    p = native.AdaptersParamsC(*v.values())
    refused(native, native.lib().pfk_adapters(C.byref(p), None), word)


@pytest.mark.parametrize("change,word", [
    (dict(dtype=3), "dtype"), (dict(activation=2), "activation"), (dict(renormalize=3), "renormalize"), (dict(tokens=-1), "tokens"),
    (dict(tokens=1 << 27), "tokens"), (dict(width=0), "width"), (dict(inner=65537), "inner"), (dict(experts=0), "number"),
    (dict(experts=1025), "number"), (dict(top=0), "top"), (dict(top=9), "top"), (dict(experts=64, top=33), "top"), (dict(x_st=-1), "negative"),
    (dict(router_st=62), "padded"), (dict(router_st=66), "padded"), (dict(up_st=66), "padded"), (dict(down_st=28), "padded"),
    (dict(x=None), "null"), (dict(y=None), "null"), (dict(router=None), "null"), (dict(up=None), "null"), (dict(down=None), "null"),
    (dict(up=FAKE + 4), "aligned"), (dict(work=None), "workspace"), (dict(work_bytes=100), "workspace"), (dict(work=FAKE + 8), "workspace")])
def test_experts_refusals(native, change, word):
    v = dict(dtype=0, activation=0, renormalize=1, tokens=4, width=64, inner=32, experts=8, top=2, x=FAKE, x_st=64, router=FAKE, router_st=64, up=FAKE,
             up_st=64, down=FAKE, down_st=32, y=FAKE, y_st=64, chosen=None, weights=None, work=FAKE, work_bytes=1 << 20)
    v.update(change)
    p = native.ExpertsParamsC(*v.values())
    refused(native, native.lib().pfk_experts(C.byref(p), None), word)


def test_experts_in_place_at_another_stride(native):
    """Refused: rows of a later pass would be written before they are read."""
    p = native.ExpertsParamsC(0, 0, 1, 300, 64, 32, 8, 2, FAKE, 64, FAKE, 64, FAKE, 64, FAKE, 32, FAKE, 72, None, None, FAKE, 1 << 30)
    refused(native, native.lib().pfk_experts(C.byref(p), None), "stride")


def test_null_parameters(native):
    L, n = native.lib(), C.c_size_t(0)
    for f in (L.pfk_cache4_append, L.pfk_cache4_read, L.pfk_cache4_attention, L.pfk_adapters, L.pfk_experts):
        refused(native, f(None, None), "null")
    refused(native, L.pfk_cache4_attention_workspace(None, C.byref(n)), "null")
    refused(native, L.pfk_experts_workspace(None, C.byref(n)), "null")


def test_nothing_to_do_needs_no_device(native):
    L, n = native.lib(), C.c_size_t(7)
    a = native.Cache4AppendParamsC(cache(native), 0, 0)
    assert L.pfk_cache4_append(C.byref(a), None) == 0
    r = native.Cache4ReadParamsC(cache(native), 0, 0)
    assert L.pfk_cache4_read(C.byref(r), None) == 0
    t = native.Cache4AttentionParamsC(cache(native), 0, 0, 4)
    assert L.pfk_cache4_attention(C.byref(t), None) == 0
    assert L.pfk_cache4_attention_workspace(C.byref(t), C.byref(n)) == 0 and n.value == 0
    d = native.AdaptersParamsC(0, 0, 64, 64, 2, 16)
    d.a_st = 64
    assert L.pfk_adapters(C.byref(d), None) == 0
    e = native.ExpertsParamsC(0, 0, 1, 0, 64, 32, 8, 2)
    e.router_st = e.gate_up_st = 64
    e.down_st = 32
    assert L.pfk_experts(C.byref(e), None) == 0
    assert L.pfk_experts_workspace(C.byref(e), C.byref(n)) == 0 and n.value == 0


def test_handles_need_a_cuda_device(native):
    with pytest.raises(ValueError, match="CUDA"):
        pf.PagedKVCache4bit(4, 16, 2, 64, device="cpu")
    with pytest.raises(ValueError, match="positive"):
        pf.PagedKVCache4bit(0, 16, 2, 64)
    with pytest.raises(ValueError, match="2\\^31"):
        pf.PagedKVCache4bit(1 << 20, 1 << 11, 2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        pf.LowRankAdapters(2, 64, 64, 16, device="cpu")
    with pytest.raises(ValueError, match="256"):
        pf.LowRankAdapters(2, 64, 64, 257)
    with pytest.raises(TypeError, match="dtype"):
        pf.LowRankAdapters(2, 64, 64, 16, dtype=torch.float64)
    with pytest.raises(ValueError, match="CUDA"):
        pf.MixtureOfExperts(torch.zeros(4, 8), torch.zeros(4, 8, 8), torch.zeros(4, 8, 4), 2)
