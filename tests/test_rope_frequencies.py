"""rope.frequencies on the CPU: which pairs a scaling stretches, and by how much."""
import math

import pytest
import torch

from e2e_browser_voice_agent_b200 import rope


def plain(n, base):
    return torch.tensor([base ** (-2 * j / n) for j in range(n // 2)], dtype=torch.float64)


def test_yarn_goes_linearly_with_the_pair():
    # 128 wide, base 1e6, 32,768 positions: pair 23.6 turns 32 times, pair 39.7 once; so pairs to 23 stay, from 40 on they are divided
    f = rope.frequencies(128, 1e6, "yarn", 4.0, original=32768, device="cpu")
    share = torch.tensor([1.0] * 24 + [1 - (j - 23) / 17 for j in range(24, 40)] + [0.0] * 24, dtype=torch.float64)
    assert torch.allclose(f, plain(128, 1e6) * (share + (1 - share) / 4), rtol=1e-14, atol=0)
    # 64 wide, base 1e4, 4,096 positions, other borders: pair 8.1 turns 64 times, pair 20.1 twice
    f = rope.frequencies(64, 1e4, "yarn", 8.0, original=4096, fast=64, slow=2, device="cpu")
    low, high = 8, 21
    assert 64 * math.log(4096 / (2 * math.pi * 64)) / (2 * math.log(1e4)) > low and 64 * math.log(4096 / (4 * math.pi)) / (2 * math.log(1e4)) < high
    share = torch.tensor([min(1.0, max(0.0, 1 - (j - low) / (high - low))) for j in range(32)], dtype=torch.float64)
    assert torch.allclose(f, plain(64, 1e4) * (share + (1 - share) / 8), rtol=1e-14, atol=0)


def test_yarn_whose_pairs_all_turn_often_or_seldom():
    assert torch.equal(rope.frequencies(64, 1e4, "yarn", 4.0, original=10**9, device="cpu"), plain(64, 1e4))
    f = rope.frequencies(64, 1e4, "yarn", 4.0, original=4, device="cpu")
    assert torch.allclose(f[1:], plain(64, 1e4)[1:] / 4, rtol=1e-14, atol=0)
    f = rope.frequencies(2, 1e4, "yarn", 4.0, original=2048, device="cpu")      # one pair, which turns 326 times
    assert torch.equal(f, plain(2, 1e4))


def test_turns_goes_linearly_with_the_turns():
    f = rope.frequencies(128, 5e5, "turns", 8.0, original=8192, fast=4.0, slow=1.0, device="cpu")
    p = plain(128, 5e5)
    share = ((p * 8192 / (2 * math.pi) - 1) / 3).clamp(0, 1)
    assert torch.allclose(f, p * (share + (1 - share) / 8), rtol=1e-14, atol=0)


def test_refusals():
    for name in ("yarn", "turns"):
        for kw in ({"original": 0}, {"original": 4096, "fast": 1.0, "slow": 1.0}, {"original": 4096, "slow": 0.0}):
            with pytest.raises(ValueError):
                rope.frequencies(64, 1e4, name, 4.0, device="cpu", **kw)
