"""Rotary positions of the query and the cache's rope part: the frequencies, plain or scaled for long contexts, and the
calls that use them (kernels.rope, kernels.latent_write).
"""
import math

import torch

from . import kernels


# keys of a scaling's types beside "type", "factor" and "original"
KEYS = {"linear": set(), "ntk": set(), "yarn": {"beta_fast", "beta_slow", "attention_factor", "mscale", "mscale_all_dim"}}


def frequencies(dim, base=10000.0, scaling=None):
    """(radians a position, float64 [dim / 2] on the CPU; the factor of cosine and sine). scaling: None or a dict with
    "type" and "factor" s (the stretch of the context); keys that a type does not know are refused, but for "original":
      "linear"  every frequency / s
      "ntk"     base * s^(dim / (dim - 2)) as the base
      "yarn"    frequencies that turn at least "beta_fast" (32) times within the "original" context kept, those that
                turn at most "beta_slow" (1) times divided by s, a linear ramp over the index between; the factor is
                "attention_factor", else m("mscale" (1)) / m("mscale_all_dim" (0)) with m(a) = 0.1 a ln s + 1 (1 for
                s <= 1). A model with "mscale_all_dim" scales its softmax by m("mscale_all_dim")^2 itself: equal ones
                leave cosine and sine as they are, and the columns of a head that do not turn keep their weight."""
    if dim <= 0 or dim % 2:
        raise ValueError("rotary dim: a positive even number")
    i = torch.arange(dim // 2, dtype=torch.float64)
    if scaling is None:
        return base ** (-2.0 * i / dim), 1.0
    given = {k: v for k, v in scaling.items() if v is not None}
    kind, s = given.get("type"), float(given.get("factor", 1.0))
    if kind not in KEYS:
        raise ValueError(f"rotary scaling type {kind!r}: linear, ntk or yarn")
    other = sorted(set(given) - {"type", "factor", "original"} - KEYS[kind])
    if other:
        raise ValueError(f"rotary scaling {kind!r}: {', '.join(other)} is not known")
    if not s > 0.0:
        raise ValueError("rotary scaling: factor > 0")
    if kind == "linear":
        return base ** (-2.0 * i / dim) / s, 1.0
    if kind == "ntk":
        if dim < 4:
            raise ValueError("rotary scaling 'ntk': dim of at least 4")
        return (base * s ** (dim / (dim - 2))) ** (-2.0 * i / dim), 1.0
    length = given.get("original")
    if not length:
        raise ValueError("rotary scaling 'yarn': original (the context length before the stretch)")
    if "attention_factor" in given and {"mscale", "mscale_all_dim"} & set(given):
        raise ValueError("rotary scaling 'yarn': attention_factor, or mscale and mscale_all_dim")
    f = base ** (-2.0 * i / dim)
    index = lambda turns: dim * math.log(length / (2.0 * math.pi * turns)) / (2.0 * math.log(base))  # noqa: E731
    lo = max(math.floor(index(given.get("beta_fast", 32.0))), 0)
    hi = min(math.ceil(index(given.get("beta_slow", 1.0))), dim - 1)
    ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
    m = lambda a: 0.1 * float(a) * math.log(s) + 1.0 if s > 1.0 else 1.0  # noqa: E731
    factor = given.get("attention_factor", m(given.get("mscale", 1.0)) / m(given.get("mscale_all_dim", 0.0)))
    return f / s * ramp + f * (1.0 - ramp), float(factor)


class Rotary:
    """The rotation of `dim` columns: frequencies on a device, the layout of the pairs and the factor."""

    def __init__(self, dim, base=10000.0, scaling=None, interleaved=True, device="cuda"):
        f, self.factor = frequencies(dim, base, scaling)
        self.dim, self.interleaved, self.freqs = dim, interleaved, f.to(device)

    def rotate(self, x, positions, out=None, start=0, inverse=False):
        """kernels.rope of columns start .. start + dim of x [T, H, W] or [T, W]."""
        return kernels.rope(x, positions, self.freqs, out=out, start=start, interleaved=self.interleaved,
                            factor=self.factor, inverse=inverse)

    def write_latent(self, kv, weight, eps, positions, slots, cache, **kw):
        """kernels.latent_write: the cache rows of the down projection's latents kv [n, 576]."""
        kernels.latent_write(kv, weight, eps, positions, self.freqs, slots, cache, interleaved=self.interleaved,
                             factor=self.factor, **kw)
