"""`model.rope_angles` with YaRN's two ramps against each one's definition, pair by pair."""
import math

import pytest
import torch

import model as M

THETA, N, F = 1e6, 32768, 4.0


def frequencies(rot, **scaling):
    """The angle of position 1 of every pair, from the tables."""
    cos, sin = M.rope_angles(2, rot, THETA, "cpu", {"type": "yarn", "factor": F, "original_max_position": N, "attention_factor": 1.0, **scaling})
    return torch.atan2(sin[1].double(), cos[1].double())


@pytest.mark.parametrize("rot", [16, 64, 128])
@pytest.mark.parametrize("fast,slow", [(32.0, 1.0), (16.0, 2.0), (1e6, 1e-6)])
def test_ramps(rot, fast, slow):
    def turns(i):                                    # of pair i (any real index) over the trained positions
        return N * THETA ** (-2 * i / rot) / (2 * math.pi)

    def index(t):                                    # the real index of the pair that turns t times
        lo, hi = -float(rot), 2.0 * rot
        for _ in range(200):
            mid = (lo + hi) / 2
            lo, hi = (mid, hi) if turns(mid) > t else (lo, mid)
        return lo

    first, last = max(0, math.floor(index(fast))), min(rot - 1, math.ceil(index(slow)))
    by_turns, by_dims = (frequencies(rot, beta_fast=fast, beta_slow=slow, ramp=r) for r in ("turns", "dims"))
    for i in range(rot // 2):
        w = THETA ** (-2 * i / rot)
        keep = min(1.0, max(0.0, (turns(i) - slow) / (fast - slow)))
        assert abs(by_turns[i].item() / (w * keep + w / F * (1 - keep)) - 1) < 1e-6
        keep = 1 - min(1.0, max(0.0, (i - first) / (last - first)))
        assert abs(by_dims[i].item() / (w * keep + w / F * (1 - keep)) - 1) < 1e-6


def test_the_two_ramps_differ_between_their_corners():
    """128 dims, theta 1e6, factor 4 from 32,768 (Qwen3's): pairs 24 to 39, where one ramp has down to 0.58 of the other's."""
    a, b = frequencies(128), frequencies(128, ramp="dims")
    assert torch.equal(a, frequencies(128, ramp="turns"))
    differ = ((a / b - 1).abs() > 1e-6).nonzero().flatten().tolist()
    assert differ == list(range(24, 40))
    assert abs((a / b)[32].item() - 0.58) < 0.005


@pytest.mark.parametrize("bad", [dict(ramp="steps"), dict(ramp=None), dict(original_max_position=None), dict(original_max_position=0),
                                 dict(beta_fast=1.0, beta_slow=1.0), dict(beta_slow=0.0), dict(attention_factor=None),
                                 dict(original_max_position_embeddings=N)], ids=str)
def test_refusals(bad):
    """A configuration in other words is refused, not served by another formula."""
    good = {"type": "yarn", "factor": F, "original_max_position": N}
    M.rope_angles(2, 128, THETA, "cpu", good)
    with pytest.raises(ValueError):
        M.rope_angles(2, 128, THETA, "cpu", {**good, **bad})
    with pytest.raises(ValueError):
        M.rope_angles(2, 128, THETA, "cpu", {"type": "yarn", "factor": F, "original_max_position_embeddings": N})
