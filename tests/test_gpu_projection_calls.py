"""Calls of the norm, projection, rotary and latent-row entry points that their documentation allows beside the usual ones."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def _column(row):
    """The values of row [1, D] as a tensor of that shape with strides (1, 1): a transposed column."""
    t = torch.empty(row.shape[1], 1, dtype=row.dtype, device=row.device).t()
    t.view(torch.uint8 if row.dtype == F8 else row.dtype).copy_(row.view(torch.uint8 if row.dtype == F8 else row.dtype))
    assert t.stride() == (1, 1) and t.shape == row.shape
    return t


def test_strides_of_single_rows(dev):
    """The stride of a dimension of one element is never used, whatever a view left there."""
    from arcagi2_flashnext_dots3_amd import kernels
    g = torch.Generator().manual_seed(1)
    a, w = (torch.randn(n, 272, generator=g).to(F8).to(dev) for n in (1, 300))
    sa, sw = torch.rand(1, 3, generator=g).to(dev), torch.rand(3, 3, generator=g).to(dev)
    want = kernels.linear_fp8(a, sa, w, sw)
    out = torch.empty(300, 1, dtype=torch.bfloat16, device=dev).t()
    kernels.linear_fp8(_column(a), _column(sa), w, sw, out=out)
    assert torch.equal(out, want)
    assert torch.equal(kernels.linear_fp8(w, torch.ones(300, 3, device=dev), _column(a), _column(sa)),
                       kernels.linear_fp8(w, torch.ones(300, 3, device=dev), a, sa))
    x = torch.randn(1, 272, generator=g).to(torch.bfloat16).to(dev)
    assert torch.equal(kernels.linear_quant(_column(x), w, sw), kernels.linear_quant(x, w, sw))
    c, s = kernels.rms_norm_fp8(x, None)
    c2, s2 = kernels.rms_norm_fp8(_column(x), None, codes=_column(c), scales=_column(s))
    assert torch.equal(c2.view(torch.uint8), c.view(torch.uint8)) and torch.equal(s2, s)
    torch.cuda.synchronize()


def test_strides_of_a_single_token_or_head_turned_in_place(dev):
    from arcagi2_flashnext_dots3_amd import kernels
    g = torch.Generator().manual_seed(2)
    f = (10000.0 ** (-torch.arange(8, dtype=torch.float64) / 8)).to(dev)
    for shape, strides, pos in (((1, 6, 16), (5, 16, 1), [77]), ((6, 1, 16), (16, 3, 1), [3, 1, 4, 1, 5, 9])):
        x = torch.randn(96, generator=g).to(dev)
        p = torch.tensor(pos, device=dev)
        want = kernels.rope(x.view(shape), p, f)
        kernels.rope(x.view(shape), p, f, out=x.as_strided(shape, strides))
        torch.cuda.synchronize()
        assert torch.equal(x.view(shape), want)


@pytest.mark.parametrize("fmt", [0, 1, 2])
def test_strides_of_a_single_latent_and_block(dev, fmt):
    from arcagi2_flashnext_dots3_amd import kernels
    g = torch.Generator().manual_seed(3)
    rowb = kernels._ROWB[fmt]
    kv = torch.randn(1, 576, generator=g).to(torch.bfloat16).to(dev)
    f = (10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)).to(dev)
    args = None, 1e-6, torch.tensor([9], device=dev), f, torch.tensor([2], device=dev)
    a, b = (torch.zeros(4, rowb, dtype=torch.uint8, device=dev) for _ in range(2))
    kernels.latent_write(kv, *args, a, fmt=fmt, kv_scale=0.1)
    kernels.latent_write(_column(kv), *args, b.as_strided((1, 4, rowb), (1, rowb, 1)), fmt=fmt, kv_scale=0.1)
    torch.cuda.synchronize()
    assert torch.equal(a, b) and bool(a[2].any())
