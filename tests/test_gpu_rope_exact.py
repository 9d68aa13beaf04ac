"""How exact rope.rotate's float32 results are, near and far out, against angles from exact fractions."""
import math
from fractions import Fraction

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
TWO_PI = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494459")


def turned(x, position, f):
    """x turned (halves), in 64 bits with angles that are rounded once from the exact ones less their whole turns."""
    u = torch.tensor([[float((int(p) * Fraction(v) / TWO_PI + Fraction(1, 2)) % 1 - Fraction(1, 2)) * 2 * math.pi for v in f.tolist()]
                      for p in position.tolist()], dtype=torch.float64, device=DEV)[:, None]
    a, b = x.double().chunk(2, -1)
    return torch.cat([a * u.cos() - b * u.sin(), b * u.cos() + a * u.sin()], -1)


@pytest.mark.parametrize("first", [0, 100_000, 2**24, 2**31 - 64])
@pytest.mark.parametrize("lowest,highest", [(1e-4, 1.0), (0.5, 1.0), (3.0, 6.0)])
def test_float32_is_as_exact_far_out_as_near(first, lowest, highest):
    """A rounding is off by 2^-24 of the value at most, by its third in the mean square. A pair (a, b) of length L turned by cosine and sine that
    are rounded once: (a^2 + b^2) (c^2 + s^2) / 3 from those, (a^2 + b^2) s^2 / 3 from the product that is rounded (the other is exact within the
    sum), L^2 / 3 from the sums; s^2 is a half on average: 5/6 L^2 in units of 2^-48, so 0.92 2^-24. An angle that is a float32 gives some 0.95, one
    of a single rounded 64-bit product near position 2^31 up to 14."""
    from e2e_browser_voice_agent_b200 import rope
    gen = torch.Generator(device=DEV)
    gen.manual_seed(first % 1000 + int(lowest * 10))
    x = torch.randn(64, 8, 64, generator=gen, device=DEV)
    position = torch.arange(first, first + 64, device=DEV).int()
    f = lowest * (highest / lowest) ** torch.rand(32, generator=gen, device=DEV, dtype=torch.float64)
    want = turned(x, position, f)
    for kw in ({}, {"interleaved": True}):
        mix = torch.arange(64, device=DEV).view(2, 32).t().reshape(-1) if kw else torch.arange(64, device=DEV)
        got = rope.rotate(x[..., mix].contiguous(), position, f, **kw).double()
        assert float((got - want[..., mix]).norm() / want.norm()) < 0.92 * 2.0**-24
