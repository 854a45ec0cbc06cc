"""Rotary angles of positions up to 2^31 against exact arithmetic."""
import math
from fractions import Fraction

import pytest
import torch

pytestmark = pytest.mark.gpu
TWO_PI = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")


def _exact(positions, freqs):
    """cos and sin of position * frequency: the angle as a fraction, less whole turns."""
    ang = [[float(Fraction(f) * p % TWO_PI) for f in freqs] for p in positions]
    return torch.tensor([[math.cos(a) for a in r] for r in ang], dtype=torch.float64), torch.tensor([[math.sin(a) for a in r] for r in ang], dtype=torch.float64)


@pytest.mark.parametrize("inter", [True, False])
def test_angles_far_out(dev, inter):
    """Pairs (1, 0) become (cos, sin). The quarter turns' distance from a whole one (at most 1/2) rounds to 32 bits, so does pi
    / 2 and so does their product: 0.79 * 2.5 * 2^-24 = 2^-23 of angle. The series and their two last roundings add 2^-28 +
    1.5 * 2^-24: below 2^-22 in all."""
    from arcagi2_flashnext_dots3_amd import kernels
    g = torch.Generator().manual_seed(3)
    pos = torch.cat((2 ** 31 - 1 - torch.randint(0, 100000, (40,), generator=g), torch.tensor([0, 1, 2 ** 24 + 1, 163840])))
    freqs = torch.cat((0.5 + 0.5 * torch.rand(24, generator=g, dtype=torch.float64),
                       10000.0 ** (-torch.arange(8, dtype=torch.float64) / 8), torch.tensor([1.0, math.pi / 4, 0.0, 2.0 ** -40], dtype=torch.float64)))
    n = freqs.shape[0]
    x = torch.zeros(len(pos), 2 * n)
    a, b = (x[:, 0::2], x[:, 1::2]) if inter else (x[:, :n], x[:, n:])
    a.fill_(1.0)
    y = kernels.rope(x.to(dev), pos.to(dev), freqs.to(dev), interleaved=inter).cpu().double()
    torch.cuda.synchronize()
    c, s = _exact(pos.tolist(), freqs.tolist())
    got = (y[:, 0::2], y[:, 1::2]) if inter else (y[:, :n], y[:, n:])
    err = max(float((got[0] - c).abs().max()), float((got[1] - s).abs().max()))
    print(f"[rope] largest error 2^{math.log2(err):.2f}", flush=True)
    assert err <= 2.0 ** -22
    back = kernels.rope(y.float().to(dev), pos.to(dev), freqs.to(dev), interleaved=inter, inverse=True).cpu().double()
    assert float((back - x.double()).abs().max()) <= 2.0 ** -20          # two rotations of sizes below 2^1/2, two components each
