"""Rotary positions and the cache rows of latents against 64 bits."""
import pytest
import torch

from tests import refs_projection as ref

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _pos(T, seed):
    p = torch.randint(0, 1 << 20, (T,), generator=torch.Generator().manual_seed(seed))
    p[:4] = torch.tensor([0, 1, 2 ** 31 - 1, 163840])[:T]
    return p


def _freqs(n):
    return 10000.0 ** (-torch.arange(n, dtype=torch.float64) / max(n, 1))


# T, H, W, start, pairs: whole heads, the first and last part, odd widths and parts, one head, more units than lanes
SHAPES = [(5, 128, 64, 0, 32), (3, 64, 128, 0, 32), (4, 8, 192, 128, 32), (1, 1, 64, 0, 32), (7, 5, 80, 40, 20),
          (2, 3, 7, 1, 2), (6, 1, 33, 0, 16), (2, 2, 4096, 0, 2048), (300, 2, 16, 8, 4), (2, 4, 24, 8, 0), (3, 300, 8, 0, 4)]


@pytest.mark.parametrize("T,H,W,start,n", SHAPES)
@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_rope(dev, T, H, W, start, n, inter, dt):
    from arcagi2_flashnext_dots3_amd import kernels
    g = torch.Generator().manual_seed(T + W)
    x = torch.randn(T, H, W + 8, generator=g).to(DT[dt])
    pos, f = _pos(T, 3), _freqs(n)
    y, tol = ref.turned(x[..., 8:], pos, f, start, inter, 1.25)
    tol = tol + ref.HALF[x.dtype] * (y.abs() + tol) + ref.TINY[x.dtype]
    out = torch.full((T, H, W + 16), 9.0, dtype=x.dtype, device=dev)
    xd = x.to(dev)
    for p in (pos, pos.to(torch.int32)):
        out.fill_(9.0)
        kernels.rope(xd[..., 8:], p.to(dev), f.to(dev), out=out[..., :W], start=start, interleaved=inter, factor=1.25)
        torch.cuda.synchronize()
        got = out.cpu()
        assert ((got[..., :W].double() - y).abs() <= tol).all()
        assert bool((got[..., W:] == 9.0).all()) and torch.equal(got[..., :start], x[..., 8:8 + start])
        assert torch.equal(got[..., start + 2 * n:W], x[..., 8 + start + 2 * n:])
    kernels.rope(xd[..., 8:], pos.to(dev), f.to(dev), out=xd[..., 8:], start=start, interleaved=inter, factor=1.25)
    torch.cuda.synchronize()
    assert torch.equal(xd[..., 8:].cpu(), got[..., :W]) and torch.equal(xd[..., :8].cpu(), x[..., :8])


@pytest.mark.parametrize("inter", [True, False])
def test_inverse_is_the_gradient(dev, inter):
    """The rotation's transpose is the rotation by the negative angle: <rope(x), g> = <x, inverse(g)>, and a difference
    quotient along one direction (the map is linear: exact but for rounding)."""
    from arcagi2_flashnext_dots3_amd import kernels
    gen = torch.Generator().manual_seed(1)
    x, g = torch.randn(9, 4, 64, generator=gen), torch.randn(9, 4, 64, generator=gen)
    pos, f = _pos(9, 2), _freqs(16)
    kw = dict(start=32, interleaved=inter, factor=0.75)
    y = kernels.rope(x.to(dev), pos.to(dev), f.to(dev), **kw).cpu().double()
    gx = kernels.rope(g.to(dev), pos.to(dev), f.to(dev), inverse=True, **kw).cpu()
    torch.cuda.synchronize()
    want, tol = ref.turned(g, pos, f, 32, inter, 0.75, inverse=True)
    assert ((gx.double() - want).abs() <= tol + 2.0 ** -24 * want.abs()).all()
    lhs, rhs = (y * g.double()), (x.double() * gx.double())
    assert abs(float(lhs.sum() - rhs.sum())) <= 2.0 ** -21 * float(lhs.abs().sum() + rhs.abs().sum())
    h = 2.0 ** -4
    y2 = kernels.rope((x + h * g).to(dev), pos.to(dev), f.to(dev), **kw).cpu().double()
    diff, along = (y2 - y) / h, ref.turned(g, pos, f, 32, inter, 0.75)[0]
    size = ref.turned(x.abs() + g.abs(), pos, f, 32, inter, 0.75)[1].amax() + 2.0 ** -22 * y.abs().amax()
    assert float((diff - along).abs().max()) <= 4.0 * float(size) / h


def test_two_dimensional_and_frequencies(dev):
    from arcagi2_flashnext_dots3_amd import rotary
    r = rotary.Rotary(64, scaling={"type": "yarn", "factor": 40.0, "original": 4096}, interleaved=False, device=dev)
    x = torch.randn(50, 128, generator=torch.Generator().manual_seed(6)).to(torch.bfloat16)
    pos = _pos(50, 5)
    y, tol = ref.turned(x[:, None], pos, r.freqs.cpu(), 0, False, r.factor)
    got = r.rotate(x.to(dev), pos.to(dev))
    torch.cuda.synchronize()
    assert ((got.cpu().double() - y[:, 0]).abs() <= (tol + ref.HALF[x.dtype] * (y.abs() + tol))[:, 0]).all()
    assert r.rotate(x.to(dev)[:0], pos.to(dev)[:0]).shape == (0, 128)


# ---- cache rows of latents
def _latent(n, seed):
    g = torch.Generator().manual_seed(seed)
    kv = (torch.randn(n, 640, generator=g) * torch.exp(torch.randn(n, 1, generator=g))).to(torch.bfloat16)
    w = (1 + 0.2 * torch.randn(512, generator=g)).to(torch.bfloat16)
    return kv[:, 64:], w


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("n,paged", [(1, False), (70, False), (333, True)])
def test_latent_write(dev, fmt, inter, n, paged):
    from arcagi2_flashnext_dots3_amd import kernels
    rowb, R, scale = kernels._ROWB[fmt], 640, 0.03
    kv, w = _latent(n, n + fmt)
    pos, f = _pos(n, 7), _freqs(32)
    slots = torch.randperm(R, generator=torch.Generator().manual_seed(4))[:n]
    if n > 1:
        slots[::9] = -1
        slots[1] = R                                          # beyond the cache: skipped too
    on = (slots >= 0) & (slots < R)
    lat, _ = ref.normed(kv[:, :512], w, 1e-6)
    pe, ptol = ref.turned(kv[:, None, 512:], pos, f, 0, inter, 1.1)
    pe, ptol = pe[:, 0], ptol[:, 0]
    kvd = kv.to(dev)
    kvd[~on.to(dev)] = float("nan")                           # padding: not read
    back = torch.full((10, 64 * rowb + 64), 0x5A, dtype=torch.uint8, device=dev)
    cache = back.as_strided((10, 64, rowb), (64 * rowb + 64, rowb, 1)) if paged else \
        torch.full((R, rowb), 0x5A, dtype=torch.uint8, device=dev)
    kernels.latent_write(kvd, w.to(dev), 1e-6, pos.to(dev), f.to(dev), slots.to(dev), cache, fmt=fmt, kv_scale=scale,
                         interleaved=inter, factor=1.1)
    torch.cuda.synchronize()
    rows = cache.cpu().reshape(R, rowb)
    idle = torch.ones(R, dtype=torch.bool)
    idle[slots[on]] = False
    assert bool((rows[idle] == 0x5A).all()) and (not paged or bool((back[:, 64 * rowb:] == 0x5A).all()))
    rows, lat, pe, ptol = rows[slots[on]].contiguous(), lat[on], pe[on], ptol[on]
    if fmt == 0:
        ref.check_codes(rows[:, :512].view(torch.float8_e4m3fn), rows[:, 512:528].contiguous().view(torch.float32), lat)
        got = rows[:, 528:].contiguous().view(torch.bfloat16).double()
        assert ((got - pe).abs() <= ptol + 2.0 ** -8 * (pe.abs() + ptol)).all()
        return
    q, qt = (lat / scale).clamp(-448, 448), None
    p = (pe / scale).clamp(-448, 448)
    rope_codes = rows[:, 512:] if fmt == 1 else rows[:, 336:]
    got = rope_codes.contiguous().view(torch.float8_e4m3fn).float().double()
    assert ((got - p).abs() <= 0.5 * ref.e4m3_step(p) + ptol / scale + 2.0 ** -22 * p.abs()).all()
    if fmt == 1:
        got = rows[:, :512].contiguous().view(torch.float8_e4m3fn).float().double()
        assert ((got - q).abs() <= 0.5 * ref.e4m3_step(q) + ref.NORM_REL * q.abs()).all()
        return
    # Row400: k the smallest exponent with 7 2^k >= the block's largest magnitude; steps of 1/4, 1/2, 1 in units of 2^k
    from oracle import spmla_ref as oracle
    code, k, _ = oracle.row400_unpack(rows.numpy())
    k = torch.as_tensor(k).double()
    am = q.view(-1, 16, 32).abs().amax(2)
    lo, hi = (torch.ceil(torch.log2(am * (1 + s * ref.NORM_REL) / 7.0)) for s in (-1, 1))
    assert ((k >= lo) & (k <= hi)).all()
    unit = torch.exp2(k)[..., None].expand(-1, 16, 32).reshape(q.shape)
    deq = torch.as_tensor(oracle.row400_dequant(code, k.numpy().astype("int8"))).double()
    size = q.abs() / unit
    step = torch.where(size < 2, 0.25, torch.where(size < 4, 0.5, 1.0)) * unit
    assert ((deq - q).abs() <= 0.5 * step + ref.NORM_REL * q.abs()).all()


def test_latent_write_equals_the_calls_it_joins_where_nothing_rounds_between(dev):
    """Positions 0 (no turn) and latents of +-2^e per row, whose norm is +-1 before the weight (powers of two): the norm
    is exact in bf16, so the joined call writes the bytes of rms_norm, rope and cache_write."""
    from arcagi2_flashnext_dots3_amd import kernels
    g = torch.Generator().manual_seed(8)
    n = 40
    kv = torch.where(torch.rand(n, 576, generator=g) < 0.5, -1.0, 1.0) * 2.0 ** torch.randint(-4, 5, (n, 1), generator=g)
    kv = kv.to(torch.bfloat16).to(dev)
    w = (2.0 ** torch.randint(-3, 4, (512,), generator=g)).to(torch.bfloat16).to(dev)
    pos, f = torch.zeros(n, dtype=torch.int64, device=dev), _freqs(32).to(dev)
    slots = torch.randperm(64, generator=g)[:n].to(dev)
    for fmt in (0, 1, 2):
        a, b = (torch.zeros(64, kernels._ROWB[fmt], dtype=torch.uint8, device=dev) for _ in range(2))
        kernels.latent_write(kv, w, 0.0, pos, f, slots, a, fmt=fmt, kv_scale=0.5)
        kernels.cache_write(kernels.rms_norm(kv[:, :512], w, 0.0), kernels.rope(kv[:, 512:], pos, f), slots, b, fmt=fmt,
                            kv_scale=0.5)
        torch.cuda.synchronize()
        assert torch.equal(a, b)
