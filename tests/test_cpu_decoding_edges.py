"""Token generation without a GPU: tangents, which tensors share memory and are
refused for it, what handles keep, and the order of a cache's check."""
import ctypes as C

import pytest
import torch

import pyflame_b200 as pf
from pyflame_b200 import decoding
from tests.test_cpu_decoding import FAKE, cache, refused, rotary


def test_tangents(native):
    import torch.autograd.forward_ad as forward
    decoding._Bound.load()
    x = torch.zeros(3)
    decoding._no_tangents(x=x, y=None)
    with forward.dual_level():
        dual = forward.make_dual(x, torch.ones(3))
        decoding._no_tangents(x=x, y=None)
        with pytest.raises(RuntimeError, match="y: .*tangent"):
            decoding._no_tangents(x=x, y=dual)
        decoding._no_tangents(x=dual.detach())


@pytest.mark.parametrize("strides,refuse", [((256, 128, 64), False), ((256, 64, 128), True), ((512, 128, 64), True)])
def test_rope_in_place_with_other_strides(native, strides, refuse):
    p = native.RopeParamsC(0, 0, 2, 2, 2, 64, 256, 128, 64, *strides, None, 0, 1, rotary(native))
    if refuse:
        refused(native, native.lib().pfk_rope(FAKE, FAKE, C.byref(p), None), "strides")
    else:  # as far as the next check
        refused(native, native.lib().pfk_rope(FAKE, FAKE, C.byref(p), None), "positions")


@pytest.mark.parametrize("sizes", [(1, 1, 1), (1, 1, 2), (1, 2, 1), (2, 1, 1)])
def test_rope_in_place_strides_of_single_axes(native, sizes):
    """A stride matters where its axis has more than one entry."""
    x, y = [7, 5, 3], [8 if n == 1 else s for n, s in zip(sizes, (7, 5, 3))]
    p = native.RopeParamsC(0, 0, *sizes, 64, *x, *y, None, 0, 1, rotary(native))
    refused(native, native.lib().pfk_rope(FAKE, FAKE, C.byref(p), None), "positions")


@pytest.mark.parametrize("strides,word", [((128, 64), "positions"), ((64, 128), "strides"), ((256, 64), "strides")])
def test_append_in_place_with_other_strides(native, strides, word):
    p = native.PagedAppendParamsC(cache(native), 3, FAKE, 128, 64, FAKE, 128, 64, FAKE, FAKE, 2, 128, 64, *strides)
    p.slots, p.rotary = FAKE, rotary(native, 64)
    refused(native, native.lib().pfk_paged_append(C.byref(p), None), word)


def test_which_tensors_share_memory():
    buf = torch.zeros(600)
    wide = torch.zeros(4, 6, 8)
    for a, b, share in [
            (buf[:100], buf[100:], False), (buf[:101], buf[100:], True), (buf[100:200], buf[:101], True), (buf, buf, True),
            (wide[:, :2], wide[:, 2:4], False), (wide[:, :2], wide[:, 1:3], True), (wide[:, 0:4:2], wide[:, 1:4:2], False),
            (wide[:2], wide[2:], False), (wide[..., :4], wide[..., 4:], False), (wide[..., :5], wide[..., 4:], True),
            (wide.transpose(0, 1), wide[3], True), (buf[0:0], buf, False), (buf, buf[5:5], False),
            (buf[:8].view(torch.uint8)[:5], buf[1:2], True), (buf[:8].view(torch.uint8)[:4], buf[1:2], False),
            (wide[0, 0, :1].expand(3, 8), wide[1], False), (wide[0, 0, :1].expand(3, 8), wide[0], True)]:
        assert decoding._share(a, b) == share and decoding._share(b, a) == share
        size = [decoding._extent(x) for x in (a, b)]  # what the calls look at first
        meet = a.data_ptr() < b.data_ptr() + size[1] and b.data_ptr() < a.data_ptr() + size[0]
        assert meet or not share
        if share:
            with pytest.raises(ValueError, match="out: shares memory with the other"):
                decoding._apart("out", a, the_other=b)
        else:
            decoding._apart("out", a, the_other=b)


@pytest.mark.parametrize("shape", [(5,), (1, 7), (7, 1), (4, 1, 5), (0, 9), (2, 3, 1, 8), (1, 1, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_outputs_like_one_element(shape, dtype):
    memory = torch.zeros((2, 3), dtype=torch.int32)
    model = decoding._model(memory, shape, dtype)
    out = torch.empty_like(model)
    assert model.untyped_storage().data_ptr() == memory.untyped_storage().data_ptr() and out.shape == shape and out.dtype == dtype and out.is_contiguous()
    assert out.untyped_storage().nbytes() == out.numel() * out.element_size()


def test_check_leaves_no_write_in_flight(monkeypatch):
    """The flag is cleared before check() returns: cleared later, it would take the error of a call on another stream."""
    did = []

    class Flag:
        def item(self):
            did.append("read")
            return -1

        def zero_(self):
            did.append("clear")

    class Torch:
        class cuda:
            synchronize = staticmethod(lambda device: did.append("wait"))

    monkeypatch.setattr(decoding._Bound, "torch", Torch)
    c = pf.PagedKVCache.__new__(pf.PagedKVCache)
    c._err, c.device = Flag(), "cuda:0"
    with pytest.raises(pf._native.PfcError):
        c.check()
    assert did == ["wait", "read", "clear", "wait"]
