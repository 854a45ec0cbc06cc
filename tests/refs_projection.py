"""64-bit references of the norm, quantization, rotary, latent-row and projection operators, and the bounds their outputs
meet. Roundings count half a step each: 2^-8 of the value for bf16, 2^-11 for fp16, 2^-24 for fp32."""
import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -149}   # half the smallest step
# fp32 inside a norm: a thread adds up to 64 squares, a tree of 6 and up to 16 partial sums follow: 90 roundings of the
# sum, half of that in its root, then mean, root, division, two products: below 64 roundings of 2^-24
NORM_REL = 2.0 ** -18


def normed(x, weight, eps, residual=None):
    """(y, z) in float64; z is the stored sum, rounded as fp32 sums are to the type."""
    z = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    d = z.double()
    w = 1.0 if weight is None else weight.double()
    return d * w / (d.square().mean(1, keepdim=True) + eps).sqrt(), z


def e4m3_step(q):
    """Distance of the e4m3 values around q."""
    _, e = torch.frexp(q.abs())
    return torch.ldexp(torch.ones_like(q), (e - 4).clamp(min=-9))


def check_codes(codes, scales, y, ue8m0=False, rel=NORM_REL):
    """codes [T, D] e4m3 and scales [T, G] of y (float64): scales to rel (powers of two: the next one, or its neighbour
    where y's error can pass it), every code within half a step of the quotient, plus rel of it."""
    T, D = y.shape
    G = -(-D // 128)
    assert codes.shape == (T, D) and scales.shape == (T, G)
    pad = torch.nn.functional.pad(y, (0, G * 128 - D)).view(T, G, 128)
    want = (pad.abs().amax(2) / 448.0).clamp_min(1e-12)
    sc = scales.double()
    if ue8m0:
        lo, hi = want * (1 - rel), want * (1 + rel)
        assert ((sc == torch.exp2(torch.ceil(torch.log2(lo)))) | (sc == torch.exp2(torch.ceil(torch.log2(hi))))).all()
    else:
        assert ((sc - want).abs() <= rel * want).all()
        sc = want
    q = (pad / sc[:, :, None]).reshape(T, -1)[:, :D]
    got = codes.float().double()
    assert torch.isfinite(got).all()
    assert ((got - q).abs() <= 0.5 * e4m3_step(q) + rel * q.abs()).all()


def turned(x, positions, freqs, start, interleaved, factor=1.0, inverse=False):
    """The rotation of x [T, H, W] in float64 and the bound of its fp32 computation: the sizes of a pair times 2^-22 (cos,
    sin, two products, their sum and the factor round, the angle's distance from a quarter turn too), and the angle's own
    64-bit rounding."""
    x = x.double()
    n = freqs.shape[0]
    ang = positions.double()[:, None] * freqs.double()
    c, s = ang.cos()[:, None] * factor, ang.sin()[:, None] * (-factor if inverse else factor)
    i = torch.arange(n)
    ia, ib = (start + 2 * i, start + 2 * i + 1) if interleaved else (start + i, start + n + i)
    y, tol = x.clone(), torch.zeros_like(x)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    size = (a.abs() + b.abs()) * abs(factor) * (2.0 ** -22 + 2.0 ** -51 * ang.abs()[:, None])
    tol[..., ia], tol[..., ib] = size, size
    return y, tol


def linear(a, sa, w, sw):
    """out and sum of |products| in float64."""
    N, K = w.shape
    A = a.float().double() * sa.double().repeat_interleave(128, 1)[:, :K]
    W = w.float().double() * sw.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    return A @ W.t(), A.abs() @ W.abs().t()
