"""Token-generation operators on the GPU where precision, ranges and memory
come to an edge.
"""
import numpy as np
import pytest
import torch

import pyflame_b200 as pf
from tests.test_gpu_decoding import within

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
