"""Attention of whole prompts against 64 bits."""
import pytest
import torch

from tests import refs_dense as ref

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _inputs(lens, H, Hk, D, Dv, dtype, seed, tail=0):
    g = torch.Generator().manual_seed(seed)
    T = sum(lens) + tail
    q, k, v = torch.randn(T, H, D, generator=g), torch.randn(T, Hk, D, generator=g), torch.randn(T, Hk, Dv, generator=g)
    q[:, :, 0] *= 4.0                                          # some heads with peaks
    start = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32)
    return q.to(dtype), k.to(dtype), v.to(dtype), start


def _check(out, lse, q, k, v, lens, scale, causal):
    H, Hk, D, dtype = q.shape[1], k.shape[1], q.shape[2], q.dtype
    t0 = 0
    for b, n in enumerate(lens):
        if n == 0:
            continue
        qs, ks, vs = (x[t0:t0 + n].double().transpose(0, 1) for x in (q, k, v))
        ks, vs = (x.repeat_interleave(H // Hk, 0) for x in (ks, vs))
        seen = torch.ones(n, n, dtype=torch.bool)
        r = ref.softmax_product(qs, ks, vs, seen.tril() if causal else seen, scale)
        # fp16 weights: the largest of a query is 2^7 at least, a subnormal one loses 2^-25 at most
        floor = 0.0 if dtype == torch.bfloat16 else n * 2.0 ** -32 * float(vs.abs().max()) + 2.0 ** -25
        ref.check(out[t0:t0 + n].transpose(0, 1), lse[t0:t0 + n].transpose(0, 1), r, D, n, dtype, ref.HALF[dtype], floor, f"sequence {b} of {n}")
        t0 += n


SIZES = [  # lengths around the tiles of 64 keys and 128 / 256 queries, heads, widths
    ([1], 1, 1, 64, 64), ([2, 1, 63], 4, 2, 64, 64), ([64, 65, 1, 127], 3, 1, 128, 128), ([256, 257, 255], 2, 2, 192, 128),
    ([700], 2, 1, 192, 128), ([130, 3, 90], 16, 8, 128, 128), ([33, 129], 5, 1, 72, 40), ([100, 28], 2, 2, 256, 256),
    ([200], 2, 2, 96, 96), ([50, 0, 77], 2, 1, 8, 8), ([300, 20], 2, 2, 64, 128), ([150], 2, 1, 192, 192), ([1] * 70, 2, 2, 128, 64),
    ([300, 2, 130], 32, 4, 128, 128), ([130, 40], 64, 64, 64, 64), ([170], 24, 8, 192, 128),
]


@pytest.mark.parametrize("lens,H,Hk,D,Dv", SIZES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_against_64_bits(dev, lens, H, Hk, D, Dv, causal, dt):
    from arcagi2_flashnext_dots3_amd import kernels
    q, k, v, start = _inputs(lens, H, Hk, D, Dv, DT[dt], D + len(lens))
    out, lse = kernels.attend_prompt(q.to(dev), k.to(dev), v.to(dev), start.to(dev), D ** -0.5, causal=causal)
    torch.cuda.synchronize()
    _check(out.cpu(), lse.cpu(), q, k, v, lens, D ** -0.5, causal)


@pytest.mark.parametrize("causal", [True, False])
def test_many_sequences(dev, causal):
    """More sequences than the kernel sorts, many of them empty."""
    from arcagi2_flashnext_dots3_amd import kernels
    lens = [(7 * b * b + b) % 11 % 6 for b in range(300)] + [140, 0, 0]
    q, k, v, start = _inputs(lens, 3, 1, 64, 64, torch.bfloat16, 13)
    out, lse = kernels.attend_prompt(q.to(dev), k.to(dev), v.to(dev), start.to(dev), 0.125, causal=causal)
    torch.cuda.synchronize()
    _check(out.cpu(), lse.cpu(), q, k, v, lens, 0.125, causal)


@pytest.mark.parametrize("D,Dv", [(128, 128), (192, 128), (120, 104)])
@pytest.mark.parametrize("causal", [True, False])
def test_long_prompts_of_many_heads(dev, D, Dv, causal):
    """Enough work for workgroups of eight waves: some heads against 64 bits; a value that is no number reaches those behind
    it only."""
    from arcagi2_flashnext_dots3_amd import kernels
    lens, H, Hk, at = [2100, 1], 128, 8, 1333
    q, k, v, start = _inputs(lens, H, Hk, D, Dv, torch.bfloat16, D)
    args = (q.to(dev), k.to(dev), v.to(dev), start.to(dev), D ** -0.5)
    out, lse = kernels.attend_prompt(*args, causal=causal)
    torch.cuda.synchronize()
    for h in (0, 37, 127):
        g = h // (H // Hk)
        _check(out[:, h:h + 1].cpu(), lse[:, h:h + 1].cpu(), q[:, h:h + 1], k[:, g:g + 1], v[:, g:g + 1], lens, D ** -0.5, causal)
    args[2][at, 3, 5] = float("inf")
    o2, z2 = kernels.attend_prompt(*args, causal=causal)
    torch.cuda.synchronize()
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[at if causal else 0:2100, 3 * 16:4 * 16, 5] = True
    assert bool((o2[hit] == float("inf")).all()) and torch.equal(o2[~hit], out[~hit]) and torch.equal(z2, lse)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 3.0])
def test_scales(dev, scale):
    """A negative scale turns the order, zero makes all weights equal, a large one leaves a few."""
    from arcagi2_flashnext_dots3_amd import kernels
    lens = [90, 140]
    q, k, v, start = _inputs(lens, 2, 1, 128, 128, torch.bfloat16, 5)
    out, lse = kernels.attend_prompt(q.to(dev), k.to(dev), v.to(dev), start.to(dev), scale)
    torch.cuda.synchronize()
    _check(out.cpu(), lse.cpu(), q, k, v, lens, scale, True)


def test_strides_padding_and_rows_of_no_sequence(dev):
    """Slices of wider tensors with NaN around them; tokens before the first and behind the last sequence stay."""
    from arcagi2_flashnext_dots3_amd import kernels
    lens, H, Hk, D, Dv = [37, 129, 64], 4, 2, 192, 128
    q, k, v, start = _inputs(lens, H, Hk, D, Dv, torch.bfloat16, 9)
    T = sum(lens)

    def wide(x, by, axis):
        pad = [0, 0] * (2 - axis) + [8 * by, 8]
        y = torch.nn.functional.pad(x, pad, value=float("nan"))
        y = torch.nn.functional.pad(y, (0, 0, 0, 0, 3, 5), value=float("nan")).to(dev)
        return y.narrow(axis, 8 * by, x.shape[axis]) if axis else y
    qd, kd = wide(q, 1, 2), wide(k, 2, 2)
    kv = torch.nn.functional.pad(torch.cat((k, v), 2), (0, 0, 0, 0, 3, 5), value=float("nan")).to(dev)
    vd = kv[..., D:]                                           # the values of a joint tensor
    out = torch.full((T + 8, H, Dv + 8), 7.0, dtype=torch.bfloat16, device=dev)
    lse = torch.full((T + 8, H + 1), 7.0, device=dev)
    kernels.attend_prompt(qd, kd, vd, (start + 3).to(dev), D ** -0.5, out=out[..., :Dv], lse=lse[:, :H])
    torch.cuda.synchronize()
    o, z = out.cpu(), lse.cpu()
    _check(o[3:3 + T, :, :Dv], z[3:3 + T, :H], q, k, v, lens, D ** -0.5, True)
    for x in (o[:3], o[3 + T:], o[..., Dv:], z[:3], z[3 + T:], z[:, H:]):
        assert bool((x == 7.0).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_no_numbers_in_masked_places(dev, bad, dt):
    """Keys and values that are no numbers are not seen by the tokens before them; those behind get them."""
    from arcagi2_flashnext_dots3_amd import kernels
    lens = [200, 90]
    q, k, v, start = _inputs(lens, 2, 1, 128, 128, DT[dt], 11)
    at, col = 130, 77
    v[at, 0, col] = bad
    k2 = k.clone()
    k2[at] = bad
    out, lse = kernels.attend_prompt(q.to(dev), k.to(dev), v.to(dev), start.to(dev), 0.1)
    o2, z2 = kernels.attend_prompt(q.to(dev), k2.to(dev), v.to(dev), start.to(dev), 0.1)
    torch.cuda.synchronize()
    out, lse, o2, z2 = out.cpu(), lse.cpu(), o2.cpu(), z2.cpu()
    hit = out[at:200, :, col].float()
    assert bool((hit.isnan() if bad != bad else hit == bad).all())
    clean = out.clone()
    clean[at:200, :, col] = 0
    assert bool(clean.isfinite().all())
    assert bool(o2[:at].isfinite().all()) and bool(o2[200:].isfinite().all()) and bool(z2[:at].isfinite().all())
    v[at, 0, col] = 0.0
    _check(torch.cat((out[:at], out[200:])), torch.cat((lse[:at], lse[200:])), torch.cat((q[:at], q[200:])), torch.cat((k[:at], k[200:])),
           torch.cat((v[:at], v[200:])), [at, 90], 0.1, True)
    assert torch.equal(o2[:at], out[:at]) and torch.equal(z2[:at], lse[:at])


def test_large_scores_move_the_maximum(dev):
    """Scores that climb along the keys: the reference maximum moves in many tiles."""
    from arcagi2_flashnext_dots3_amd import kernels
    lens = [600]
    q, k, v, start = _inputs(lens, 2, 2, 64, 64, torch.bfloat16, 3)
    k = (k.float() + torch.linspace(0, 30, 600)[:, None, None] * q[300:301].float().sign()).to(torch.bfloat16)
    out, lse = kernels.attend_prompt(q.to(dev), k.to(dev), v.to(dev), start.to(dev), 0.125, causal=False)
    torch.cuda.synchronize()
    _check(out.cpu(), lse.cpu(), q, k, v, lens, 0.125, False)


def test_streams_and_graph(dev):
    from arcagi2_flashnext_dots3_amd import kernels
    lens = [129, 300]
    q, k, v, start = (x.to(dev) for x in _inputs(lens, 4, 2, 192, 128, torch.bfloat16, 4))
    want, wl = kernels.attend_prompt(q, k, v, start, 0.07)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        o, z = kernels.attend_prompt(q, k, v, start, 0.07)
    s.synchronize()
    assert torch.equal(o, want) and torch.equal(z, wl)
    g = torch.cuda.CUDAGraph()
    qs, o2, z2 = q.clone(), torch.zeros_like(want), torch.zeros_like(wl)
    with torch.cuda.graph(g):
        kernels.attend_prompt(qs, k, v, start, 0.07, out=o2, lse=z2)
    for i in range(4):
        qs.copy_(q.roll(i, 0))
        g.replay()
        e, ez = kernels.attend_prompt(qs, k, v, start, 0.07)
        torch.cuda.synchronize()
        assert torch.equal(o2, e) and torch.equal(z2, ez)


def test_empty(dev):
    from arcagi2_flashnext_dots3_amd import kernels
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=dev)  # noqa: E731
    out, lse = kernels.attend_prompt(z(0, 4, 64), z(0, 4, 64), z(0, 4, 64), torch.zeros(1, dtype=torch.int32, device=dev), 1.0)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
