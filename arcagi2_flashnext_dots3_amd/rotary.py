"""Rotary positions of the query and the cache's rope part: the frequencies, plain or scaled for long contexts, and the
calls that use them (kernels.rope, kernels.latent_write).
"""
import math

import torch

from . import kernels


def frequencies(dim, base=10000.0, scaling=None):
    """(radians a position, float64 [dim / 2] on the CPU; the factor of cosine and sine). scaling: None or a dict with
    "type" and "factor" s (the stretch of the context):
      "linear"  every frequency / s
      "ntk"     base * s^(dim / (dim - 2)) as the base
      "yarn"    frequencies that turn at least "beta_fast" (32) times within the "original" context kept, those that
                turn at most "beta_slow" (1) times divided by s, a linear ramp over the index between; the factor is
                "attention_factor", else 0.1 ln s + 1 (1 for s <= 1)"""
    if dim <= 0 or dim % 2:
        raise ValueError("rotary dim: a positive even number")
    i = torch.arange(dim // 2, dtype=torch.float64)
    if scaling is None:
        return base ** (-2.0 * i / dim), 1.0
    kind, s = scaling.get("type"), float(scaling.get("factor", 1.0))
    if not s > 0.0:
        raise ValueError("rotary scaling: factor > 0")
    if kind == "linear":
        return base ** (-2.0 * i / dim) / s, 1.0
    if kind == "ntk":
        if dim < 4:
            raise ValueError("rotary scaling 'ntk': dim of at least 4")
        return (base * s ** (dim / (dim - 2))) ** (-2.0 * i / dim), 1.0
    if kind == "yarn":
        length = scaling.get("original")
        if not length:
            raise ValueError("rotary scaling 'yarn': original (the context length before the stretch)")
        f = base ** (-2.0 * i / dim)
        index = lambda turns: dim * math.log(length / (2.0 * math.pi * turns)) / (2.0 * math.log(base))  # noqa: E731
        lo = max(math.floor(index(scaling.get("beta_fast", 32.0))), 0)
        hi = min(math.ceil(index(scaling.get("beta_slow", 1.0))), dim - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        factor = scaling.get("attention_factor")
        return f / s * ramp + f * (1.0 - ramp), float(factor if factor is not None else
                                                      0.1 * math.log(s) + 1.0 if s > 1.0 else 1.0)
    raise ValueError(f"rotary scaling type {kind!r}: linear, ntk or yarn")


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
