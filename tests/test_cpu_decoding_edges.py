"""Token generation without a GPU, beside its refusals: tangents."""
import pytest
import torch

from pyflame_b200 import decoding


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
