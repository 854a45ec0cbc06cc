"""Latents written into an offloaded layer's rows: pinned host memory, and the cached copies of the rows written."""
import pytest
import torch

pytestmark = pytest.mark.gpu
R, C = 600, 160


def _inputs(n, seed, dev):
    g = torch.Generator().manual_seed(seed)
    kv = torch.randn(n, 640, generator=g).to(torch.bfloat16).to(dev)[:, 64:]
    w = (1 + 0.2 * torch.randn(512, generator=g)).to(torch.bfloat16).to(dev)
    pos = torch.randint(0, 100000, (n,), generator=g).to(dev)
    slots = torch.randperm(R, generator=g)[:n]
    slots[::7] = -1
    return kv, w, pos, slots.to(dev)


def _rows(fmt, kv, w, pos, slots, scale, dev):
    from arcagi2_flashnext_dots3_amd import kernels, rotary
    rows = torch.zeros(R, kernels._ROWB[fmt], dtype=torch.uint8, device=dev)
    rotary.Rotary(64, device=dev).write_latent(kv, w, 1e-6, pos, slots, rows, fmt=fmt, kv_scale=scale)
    return rows


@pytest.mark.parametrize("fmt", [0, 1, 2])
def test_rows_in_pinned_memory(dev, fmt):
    """The bytes that a cache on the GPU gets; rows that no slot names are left."""
    from arcagi2_flashnext_dots3_amd import kernels, rotary
    kv, w, pos, slots = _inputs(333, fmt, dev)
    want = _rows(fmt, kv, w, pos, slots, 0.05, dev)
    host = torch.zeros(R, kernels._ROWB[fmt], dtype=torch.uint8, pin_memory=True)
    rotary.Rotary(64, device=dev).write_latent(kv, w, 1e-6, pos, slots, host, fmt=fmt, kv_scale=0.05)
    torch.cuda.synchronize()
    assert torch.equal(host, want.cpu()) and bool(host.any())
    with pytest.raises(ValueError, match="pinned"):
        rotary.Rotary(64, device=dev).write_latent(kv, w, 1e-6, pos, slots, torch.zeros_like(want, device="cpu"), fmt=fmt)


@pytest.mark.parametrize("row_fmt,mode,cache_fmt", [("row656", "static", "row656"), ("e2m2", "static", "row656"),
                                                    ("e2m2", "static", "e2m2"), ("row656", "ways", "row656"), ("e2m2", "ways", "e2m2")])
def test_store_latent_keeps_the_cached_rows(dev, row_fmt, mode, cache_fmt):
    """A layer with cached rows, rewritten: host rows are latent_write's, and the attention over a step that had them cached is
    that of a layer which never cached any."""
    from arcagi2_flashnext_dots3_amd import rotary
    from arcagi2_flashnext_dots3_amd.sparse_offload import LayerOffload
    scale, fmt = (0.05, 2) if row_fmt == "e2m2" else (1.0, 0)
    rot = rotary.Rotary(64, device=dev)
    lo = LayerOffload(R, dev, cache_rows=C, row_fmt=row_fmt, cache_mode=mode, ways=8, cache_fmt=cache_fmt, spill_rows=4096)
    plain = LayerOffload(R, dev, row_fmt=row_fmt)
    g = torch.Generator().manual_seed(5)
    q = torch.randn(2, 32, 576, generator=g).to(torch.bfloat16).to(dev)
    idx = torch.stack([torch.randperm(R, generator=g)[:128] for _ in range(2)]).to(torch.int32).to(dev)
    for step in range(3):
        kv, w, pos, slots = _inputs(R if step == 0 else 200, step, dev)
        if step == 0:
            slots = torch.arange(R, device=dev)
        rows = _rows(fmt, kv, w, pos, slots, scale, dev)
        for layer in (lo, plain):
            layer.store_latent(kv, w, 1e-6, rot, pos, slots, kv_scale=scale)
        torch.cuda.synchronize()
        on = slots[slots >= 0].cpu()
        assert torch.equal(lo.host[on], rows.cpu()[on]) and torch.equal(lo.host, plain.host)
        if step == 0 and mode == "static":
            lo.set_hot_rows(idx[0].to(torch.int64))
        if mode == "static" and cache_fmt == row_fmt:
            hot = lo.tag[lo.tag >= 0]
            assert torch.equal(lo.cache[:hot.numel()].cpu(), lo.host[hot.cpu()])
        a, b = (layer.attend(q, idx, 192 ** -0.5, scale, return_lse=True) for layer in (lo, plain))
        torch.cuda.synchronize()
        # the same rows over other tiers: the order of the fp32 sums, and the outputs' rounding to bf16 on each side (2^-8 of
        # a value: 2^-7 = 0.0078 together, 0.0022 for the sums)
        err = (a[0].float() - b[0].float()).abs() / b[0].float().abs().clamp_min(1.0)
        assert float(err.max()) <= 1e-2 and float((a[1] - b[1]).abs().max()) <= 1e-4


def test_store_latent_refusals(dev):
    from arcagi2_flashnext_dots3_amd import rotary
    from arcagi2_flashnext_dots3_amd.sparse_offload import LayerOffload
    kv, w, pos, slots = _inputs(4, 1, dev)
    lo = LayerOffload(R, dev)
    with pytest.raises(ValueError, match="kv_scale"):
        lo.store_latent(kv, w, 1e-6, rotary.Rotary(64, device=dev), pos, slots, kv_scale=0.5)
    lo.store_latent(kv[:0], w, 1e-6, rotary.Rotary(64, device=dev), pos[:0], slots[:0])
    lo.store(kv[:0, :512], kv[:0, 512:], slots[:0])
    assert not lo.host.any()
