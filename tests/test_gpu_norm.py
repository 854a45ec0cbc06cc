"""RMS norm with residual and 8-bit output, and the quantization alone, against 64 bits."""
import pytest
import torch

from tests import refs_projection as ref

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _x(T, D, dtype, seed, stride=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, D + stride, generator=g) * torch.exp(torch.randn(T, 1, generator=g))
    return x.to(dtype)[:, :D]


# one value, one short of and one over a group, sizes on both sides of each kernel's row length, odd ones
SIZES = [(1, 1), (3, 127), (2, 128), (5, 129), (4, 512), (7, 520), (3, 1536), (2, 2048), (3, 2056), (2, 4096),
         (2, 4104), (1, 7168), (2, 16384), (1, 16392), (1, 65536), (300, 576)]


@pytest.mark.parametrize("T,D", SIZES)
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_rms_norm_all_outputs(dev, T, D, dt):
    from arcagi2_flashnext_dots3_amd import kernels
    dtype = DT[dt]
    x, r = _x(T, D, dtype, D, 24), _x(T, D, dtype, D + 1)
    w = (1 + 0.3 * torch.randn(D, generator=torch.Generator().manual_seed(3))).to(dtype)
    y, z = ref.normed(x, w, 1e-5, r)
    xb = torch.nn.functional.pad(x, (0, 24), value=float("nan")).to(dev)[:, :D]      # NaNs behind the rows
    rd = r.to(dev)
    out = torch.full((T, D + 16), 7.0, dtype=dtype, device=dev)
    codes, scales = kernels.rms_norm_fp8(xb, w.to(dev), 1e-5, residual=rd, out=out[:, :D])
    torch.cuda.synchronize()
    assert torch.equal(rd.cpu(), z)                                                  # updated in place
    got = out.cpu()
    assert ((got[:, :D].double() - y).abs() <= y.abs() * (ref.HALF[dtype] + ref.NORM_REL) + ref.TINY[dtype]).all()
    assert bool((got[:, D:] == 7.0).all())
    ref.check_codes(codes.cpu(), scales.cpu(), y)


@pytest.mark.parametrize("T,D", [(1, 4096), (4, 1536), (9, 130)])
@pytest.mark.parametrize("ue8m0", [False, True])
def test_rms_norm_plain_and_ue8m0(dev, T, D, ue8m0):
    from arcagi2_flashnext_dots3_amd import kernels
    x = _x(T, D, torch.bfloat16, 5)
    w = 1 + 0.3 * torch.randn(D, generator=torch.Generator().manual_seed(4))        # fp32 weight of a bf16 norm
    for weight in (w, None):
        wd = None if weight is None else weight.to(dev)
        y, _ = ref.normed(x, weight, 1e-6)
        out = kernels.rms_norm(x.to(dev), wd)
        codes, scales = kernels.rms_norm_fp8(x.to(dev), wd, ue8m0=ue8m0)
        torch.cuda.synchronize()
        assert ((out.cpu().double() - y).abs() <= y.abs() * (ref.HALF[x.dtype] + ref.NORM_REL) + ref.TINY[x.dtype]).all()
        ref.check_codes(codes.cpu(), scales.cpu(), y, ue8m0)


def test_out_in_place_and_separate_residual(dev):
    from arcagi2_flashnext_dots3_amd import kernels
    x, r = _x(6, 2048, torch.bfloat16, 8), _x(6, 2048, torch.bfloat16, 9)
    w = torch.ones(2048, dtype=torch.bfloat16)
    want = kernels.rms_norm(x.to(dev), w.to(dev), residual=r.to(dev))
    xd, rd, ro = x.to(dev), r.to(dev), torch.empty(6, 2048, dtype=torch.bfloat16, device=dev)
    got = kernels.rms_norm(xd, w.to(dev), residual=rd, residual_out=ro, out=xd)
    torch.cuda.synchronize()
    assert got is xd and torch.equal(xd, want) and torch.equal(rd.cpu(), r)
    assert torch.equal(ro.cpu(), (x.float() + r.float()).to(torch.bfloat16))


@pytest.mark.parametrize("T,D", [(1, 1), (3, 100), (2, 128), (5, 2048), (3, 2056), (2, 16384), (1, 70000)])
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("ue8m0", [False, True])
def test_quant(dev, T, D, dt, ue8m0):
    from arcagi2_flashnext_dots3_amd import kernels
    x = _x(T, D, DT[dt], D + T)
    codes, scales = kernels.quant_fp8(x.to(dev), ue8m0=ue8m0)
    torch.cuda.synchronize()
    # the largest magnitude over 448 and the quotient round once or twice in fp32
    ref.check_codes(codes.cpu(), scales.cpu(), x.double(), ue8m0, rel=2.0 ** -22)


def test_quotients_halfway_between_codes(dev):
    """Values whose quotient by their group's scale lies exactly halfway between two codes take the even one: amax 7 v and
    values m v, m whole 16ths, so that the quotients are whole multiples of 4, at sizes from the smallest to the largest a scale takes."""
    from arcagi2_flashnext_dots3_amd import kernels
    m = torch.arange(1, 112).float() / 16.0
    rows = torch.zeros(12, 128)
    rows[:, 0] = 7.0
    rows[:, 1:1 + len(m)] = m
    rows *= 2.0 ** torch.tensor([-20, -10, -3, 0, 1, 5, 20, 40, 60, 90, 100, 118])[:, None].float()
    x = rows.to(torch.bfloat16)
    assert torch.equal(x.float(), rows)
    codes, _ = kernels.quant_fp8(x.to(dev))
    torch.cuda.synchronize()
    q = x.double() * 448.0 / x.double().abs().amax(1, keepdim=True)
    step = ref.e4m3_step(q)
    assert int((((q / step) % 1) == 0.5).sum()) > 100
    assert torch.equal(codes.cpu().float().double(), torch.round(q / step) * step)


def test_zero_tiny_and_not_finite_values(dev):
    from arcagi2_flashnext_dots3_amd import kernels
    inf, nan = float("inf"), float("nan")
    x = torch.randn(6, 256, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    x[0] = 0
    x[1, 128:] = 0
    x[2] = 1e-30
    x[3, 5], x[4, 200], x[5, 3] = nan, inf, -inf
    codes, scales = kernels.quant_fp8(x.to(dev))
    out = kernels.rms_norm(x.to(dev), None)
    c2, s2 = kernels.rms_norm_fp8(x.to(dev), None)
    torch.cuda.synchronize()
    v, s = codes.cpu().float(), scales.cpu()
    assert s[0].tolist() == [torch.tensor(1e-12).item()] * 2 and not v[0].any() and not v[1, 128:].any() and not v[2].any()
    ref.check_codes(codes.cpu()[:3], s[:3], x[:3].double(), rel=2.0 ** -22)
    assert torch.isnan(v[3, 5]) and torch.isfinite(v[3, 128:]).all() and int(torch.isnan(v[3]).sum()) == 1
    assert s[4, 1] == inf and torch.isnan(v[4, 200]) and not v[4, 128:200].any() and torch.isfinite(v[4, :128]).all()
    assert s[5, 0] == inf and torch.isnan(v[5, 3])
    y, _ = ref.normed(x, None, 1e-6)
    assert not out[0].any() and torch.isfinite(out[:3]).all()
    assert torch.isnan(out[3]).all()                       # a NaN is in every value's mean
    assert torch.isnan(out[4, 200]) and not out[4, :200].any()   # inf / inf, and finite / inf
    ref.check_codes(c2.cpu()[:3], s2.cpu()[:3], y[:3])
    assert torch.isnan(c2[3].float()).all() and torch.isnan(c2[4, 200].float())


def test_empty_batches(dev):
    from arcagi2_flashnext_dots3_amd import kernels
    x = torch.empty(0, 256, dtype=torch.bfloat16, device=dev)
    assert kernels.rms_norm(x, None).shape == (0, 256)
    c, s = kernels.quant_fp8(x)
    assert c.shape == (0, 256) and s.shape == (0, 2)
