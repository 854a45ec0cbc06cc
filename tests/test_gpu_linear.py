"""The projection on FP8 block-scaled weights against 64 bits."""
import pytest
import torch

from tests import refs_projection as ref

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _whole(T, N, K, seed):
    """Codes of -4 .. 4 and power-of-two scales: every sum is a whole multiple of 2^-4 below 2^20, so it is exact in fp32
    and in the matrix core, and only the output rounds."""
    g = torch.Generator().manual_seed(seed)
    kb, nb = -(-K // 128), -(-N // 128)
    a = torch.randint(-4, 5, (T, K), generator=g).float().to(torch.float8_e4m3fn)
    w = torch.randint(-4, 5, (N, K), generator=g).float().to(torch.float8_e4m3fn)
    p = lambda *s: 2.0 ** torch.randint(-2, 3, s, generator=g).float()  # noqa: E731
    return a, p(T, kb), w, p(nb, kb)


def _wide(t, extra, dev, nan=False):
    """t's rows inside a wider buffer of NaN codes (or values)."""
    T, K = t.shape
    if t.dtype == torch.float8_e4m3fn:
        b = torch.full((T, K + extra), 0x7F, dtype=torch.uint8, device=dev)
        b[:, :K] = t.view(torch.uint8).to(dev)
        return b.view(torch.float8_e4m3fn)[:, :K]
    b = torch.full((T, K + extra), float("nan"), device=dev)
    b[:, :K] = t.to(dev)
    return b[:, :K]


# one token and output, ends inside every tile, k ends inside a block, row counts on both sides of each kernel's choice
SHAPES = [(1, 1, 16), (1, 64, 128), (2, 17, 112), (3, 130, 144), (16, 16, 1024), (17, 129, 400), (33, 576, 512), (64, 300, 272),
          (65, 257, 272), (100, 100, 4096), (128, 256, 1536), (130, 200, 1152), (200, 300, 2064), (257, 513, 640),
          (300, 1100, 256), (1, 2112, 4096), (5, 24576, 256), (32, 128, 16384), (700, 1030, 384), (1100, 2112, 272)]


@pytest.mark.parametrize("T,N,K", SHAPES)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_whole_numbers_exact(dev, T, N, K, dt):
    from arcagi2_flashnext_dots3_amd import kernels
    a, sa, w, sw = _whole(T, N, K, T + N + K)
    want = ref.linear(a, sa, w, sw)[0]
    assert float(want.abs().max()) < 2 ** 20
    out = torch.full((T, N + 5), 3.0, dtype=dt, device=dev)
    print(f"[linear] T={T} N={N} K={K}", flush=True)
    kernels.linear_fp8(_wide(a, 48, dev), _wide(sa, 3, dev), _wide(w, 16, dev), _wide(sw, 2, dev), out=out[:, :N])
    torch.cuda.synchronize()
    assert torch.equal(out[:, :N].cpu(), want.float().to(dt))
    assert bool((out[:, N:] == 3.0).all())


@pytest.mark.parametrize("T,N,K", [(1, 512, 7168), (16, 300, 1040), (48, 2112, 4096), (150, 384, 2048), (600, 1536, 4096)])
def test_normal_values(dev, T, N, K):
    """Normally distributed codes: the matrix core's sum of 128 products is within 2^-11 of the sum of their sizes (the
    largest error found over all its inputs tried is 2.6e-4), the fp32 sums of the blocks below 2^-16 of it, the output
    rounds once. The error over all outputs stays below twice the output's own rounding (2^-8 / sqrt(3) at most)."""
    from arcagi2_flashnext_dots3_amd import kernels
    g = torch.Generator().manual_seed(K)
    a = (100 * torch.randn(T, K, generator=g)).clamp(-448, 448).to(torch.float8_e4m3fn)
    w = (100 * torch.randn(N, K, generator=g)).clamp(-448, 448).to(torch.float8_e4m3fn)
    sa = 1e-2 * torch.exp(torch.randn(T, -(-K // 128), generator=g))
    sw = 1e-3 * torch.exp(torch.randn(-(-N // 128), -(-K // 128), generator=g))
    want, size = ref.linear(a, sa, w, sw)
    got = kernels.linear_fp8(a.to(dev), sa.to(dev), w.to(dev), sw.to(dev))
    torch.cuda.synchronize()
    err = (got.cpu().double() - want).abs()
    assert (err <= (2.0 ** -11 + 2.0 ** -16) * size + 2.0 ** -8 * want.abs()).all()
    assert float(err.norm() / want.norm()) <= 2.0 * 2.0 ** -8 / 3 ** 0.5


def test_same_bits_every_time(dev):
    from arcagi2_flashnext_dots3_amd import kernels
    for T, N, K in ((7, 640, 4096), (64, 4096, 2048), (300, 700, 2048)):
        g = torch.Generator().manual_seed(T)
        a = torch.randn(T, K, generator=g).to(torch.float8_e4m3fn).to(dev)
        w = torch.randn(N, K, generator=g).to(torch.float8_e4m3fn).to(dev)
        sa, sw = torch.rand(T, K // 128, generator=g).to(dev), torch.rand(-(-N // 128), K // 128, generator=g).to(dev)
        first = kernels.linear_fp8(a, sa, w, sw)
        for _ in range(5):
            assert torch.equal(kernels.linear_fp8(a, sa, w, sw), first)


@pytest.mark.parametrize("T,N,K", [(5, 200, 272), (80, 200, 272), (300, 300, 272)])
def test_nan_codes_stay_in_their_row(dev, T, N, K):
    from arcagi2_flashnext_dots3_amd import kernels
    a, sa, w, sw = _whole(T, N, K, 2)
    want = ref.linear(a, sa, w, sw)[0].to(BF)
    a.view(torch.uint8)[T - 2, K - 1] = 0x7F
    w.view(torch.uint8)[N - 3, 1] = 0xFF
    got = kernels.linear_fp8(a.to(dev), sa.to(dev), w.to(dev), sw.to(dev)).cpu()
    torch.cuda.synchronize()
    bad = torch.zeros(T, N, dtype=torch.bool)
    bad[T - 2], bad[:, N - 3] = True, True
    assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], want[~bad])


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_from_activations(dev, dt):
    """mla_fp8.linear_fp8 of 16-bit activations is quant_fp8 and the product; of codes it takes them as they are."""
    from arcagi2_flashnext_dots3_amd import kernels, mla_fp8
    g = torch.Generator().manual_seed(1)
    x = torch.randn(20, 1040, generator=g).to(dt).to(dev)
    w = torch.randn(260, 1040, generator=g).to(torch.float8_e4m3fn).to(dev)
    sw = torch.rand(3, 9, generator=g).to(dev)
    a, sa = kernels.quant_fp8(x)
    got = mla_fp8.linear_fp8(x, (w, sw))
    assert got.dtype == dt and torch.equal(got, kernels.linear_fp8(a, sa, w, sw, dtype=dt))
    assert torch.equal(mla_fp8.linear_fp8((a, sa), (w.view(torch.uint8), sw)), kernels.linear_fp8(a, sa, w, sw))
    assert mla_fp8.linear_fp8(x[:0], (w, sw)).shape == (0, 260)
