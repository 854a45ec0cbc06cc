"""The norm, projection, rotary and latent-row calls as callers may make them: every kernel of the projection's rule, rows at
any alignment, two streams at once, replayed graphs, repeated and mixed arguments."""
import pytest
import torch

from tests import refs_projection as ref
from tests.test_gpu_linear import _whole, _wide
from tests.test_linear_choice import REACHES

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.mark.parametrize("kernel,T,N,K", REACHES)
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_every_projection_kernel(dev, kernel, T, N, K, dt):
    """Whole numbers: exact in the matrix core and in fp32, so that only the output rounds."""
    from arcagi2_flashnext_dots3_amd import kernels
    a, sa, w, sw = _whole(T, N, K, T + N + K)
    want = ref.linear(a, sa, w, sw)[0].float().to(DT[dt])
    out = torch.full((T, N + 3), 5.0, dtype=DT[dt], device=dev)
    print(f"[linear] kernel {kernel} T={T} N={N} K={K}", flush=True)
    args = _wide(a, 16, dev), sa.to(dev), _wide(w, 16, dev), sw.to(dev)
    kernels.linear_fp8(*args, out=out[:, :N])
    whole = kernels.linear_fp8(*args, dtype=DT[dt])           # rows that begin on 64 bytes where N allows it
    torch.cuda.synchronize()
    assert torch.equal(out[:, :N].cpu(), want) and bool((out[:, N:] == 5.0).all())
    assert torch.equal(whole.cpu(), want)


@pytest.mark.parametrize("T,D", [(3, 256), (2, 1536), (5, 1500), (2, 4096), (3, 3268), (2, 6578), (70, 15), (2, 16385)])
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_norm_rows_at_any_alignment(dev, T, D, dt):
    """Rows that begin at each place inside 16 bytes: the bytes of the call on aligned rows, nothing written beside them."""
    from arcagi2_flashnext_dots3_amd import kernels
    g = torch.Generator().manual_seed(D)
    x, r = (torch.randn(T, D, generator=g).to(DT[dt]).to(dev) for _ in range(2))
    w = (1 + 0.1 * torch.randn(D, generator=g)).to(DT[dt]).to(dev)
    base = [torch.empty(T, D, dtype=x.dtype, device=dev) for _ in range(2)]
    codes, scales = kernels.rms_norm_fp8(x, w, residual=r, residual_out=base[0], out=base[1])
    for off in (1, 2, 3, 5, 7):
        def moved(t, fill=0.0):
            b = torch.full((T, D + 9 + off), fill, dtype=t.dtype, device=dev)
            b[:, off:off + D] = t
            return b
        xs, rs, ws = moved(x, float("nan")), moved(r, float("nan")), torch.cat((w[:1].expand(off), w))[off:]
        outs = [torch.full((T, D + 9 + off), 3.0, dtype=x.dtype, device=dev) for _ in range(2)]
        c8 = torch.full((T, D + 9 + off), 0x2A, dtype=torch.uint8, device=dev)
        sl = slice(off, off + D)
        _, sc = kernels.rms_norm_fp8(xs[:, sl], ws, residual=rs[:, sl], residual_out=outs[0][:, sl], out=outs[1][:, sl],
                                     codes=c8[:, sl])
        torch.cuda.synchronize()
        assert torch.equal(sc, scales) and torch.equal(c8[:, sl], codes.view(torch.uint8))
        for o, b in zip(outs, base):
            assert torch.equal(o[:, sl], b) and bool((o[:, :off] == 3.0).all()) and bool((o[:, off + D:] == 3.0).all())
        assert bool((c8[:, :off] == 0x2A).all()) and bool((c8[:, off + D:] == 0x2A).all())


@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_rope_rows_at_any_alignment(dev, inter, dt):
    from arcagi2_flashnext_dots3_amd import kernels
    T, H, W = 6, 3, 64
    g = torch.Generator().manual_seed(1)
    x = torch.randn(T, H, W, generator=g).to(DT[dt]).to(dev)
    pos = torch.arange(100, 100 + T, device=dev)
    f = (10000.0 ** (-torch.arange(16, dtype=torch.float64) / 16)).to(dev)
    want = kernels.rope(x, pos, f, start=24, interleaved=inter)
    for off, pitch in ((1, 67), (2, 66), (3, 75), (4, 72)):
        xs, o = (torch.full((T, H, pitch + 8), 8.0, dtype=x.dtype, device=dev) for _ in range(2))
        xs[..., off:off + W] = x
        kernels.rope(xs[..., off:off + W], pos, f, out=o[..., off:off + W], start=24, interleaved=inter)
        torch.cuda.synchronize()
        assert torch.equal(o[..., off:off + W], want)
        o[..., off:off + W] = 8.0
        assert bool((o == 8.0).all())


def test_two_streams_at_once(dev):
    """The same calls on two streams, a hundred deep: each call has its own outputs and workspace."""
    from arcagi2_flashnext_dots3_amd import kernels, mla_fp8
    g = torch.Generator().manual_seed(3)
    f = (torch.randn(700, 1024, generator=g).to(torch.float8_e4m3fn).to(dev), torch.rand(6, 8, generator=g).to(dev))
    xs = [torch.randn(T, 1024, generator=g).to(torch.bfloat16).to(dev) for T in (5, 90)]
    want = [mla_fp8.linear_fp8(x, f) for x in xs]
    norms = [kernels.rms_norm_fp8(x, None) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(100):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((mla_fp8.linear_fp8(xs[i], f), *kernels.rms_norm_fp8(xs[i], None)))
    torch.cuda.synchronize()
    for i in range(2):
        for y, c, s in got[i]:
            assert torch.equal(y, want[i])
            assert torch.equal(c.view(torch.uint8), norms[i][0].view(torch.uint8)) and torch.equal(s, norms[i][1])


@pytest.mark.parametrize("fmt", [0, 1, 2])
def test_graphs_of_every_call(dev, fmt):
    """A graph of the quantized projection, the rotation in place and a latent row, beside a second graph of the same calls;
    both replayed with eager calls between."""
    from arcagi2_flashnext_dots3_amd import kernels, mla_fp8
    g = torch.Generator().manual_seed(4)
    rowb, R, T = kernels._ROWB[fmt], 128, 21
    f = (torch.randn(576, 512, generator=g).to(torch.float8_e4m3fn).to(dev), torch.rand(5, 4, generator=g).to(dev))
    w = torch.ones(512, device=dev)
    freqs = (10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)).to(dev)

    def calls(b):
        b["kv"].copy_(mla_fp8.linear_fp8(b["x"], f))
        kernels.latent_write(b["kv"], w, 1e-6, b["pos"], freqs, b["slots"], b["cache"], fmt=fmt, kv_scale=0.05)
        kernels.rope(b["q"], b["pos"], freqs, out=b["q"])

    def bufs(seed):
        g = torch.Generator().manual_seed(seed)
        return {"x": torch.randn(T, 512, generator=g).to(torch.bfloat16).to(dev), "kv": torch.empty(T, 576, dtype=torch.bfloat16, device=dev),
                "pos": torch.randint(0, 9999, (T,), generator=g).to(torch.int32).to(dev), "slots": torch.randperm(R, generator=g)[:T].to(dev),
                "cache": torch.zeros(R, rowb, dtype=torch.uint8, device=dev), "q": torch.randn(T, 4, 64, generator=g).to(dev)}

    held = [bufs(0), bufs(1)]
    for b in held:
        calls(b)
    torch.cuda.synchronize()
    graphs = []
    for b in held:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            calls(b)
    for seed in range(2, 6):
        eager = [bufs(seed), bufs(seed + 50)]
        for b, e in zip(held, eager):
            for k in b:
                b[k].copy_(e[k])
        for gr in graphs:
            gr.replay()
        for e in eager:
            calls(e)
        torch.cuda.synchronize()
        for b, e in zip(held, eager):
            assert all(torch.equal(b[k], e[k]) for k in ("kv", "cache", "q"))


def test_quantized_product_in_pieces(dev):
    """linear_quant is quant_fp8 and linear_fp8: the same bits, scales of powers of two included, out given or not."""
    from arcagi2_flashnext_dots3_amd import kernels, mla_fp8
    g = torch.Generator().manual_seed(6)
    for T, N, K in ((1, 70, 16), (5, 223, 9328), (33, 300, 1040)):
        x = torch.randn(T, K + 8, generator=g).to(torch.float16).to(dev)[:, 3:K + 3]
        f = (torch.randn(N, K, generator=g).to(torch.float8_e4m3fn).to(dev), torch.rand(-(-N // 128), -(-K // 128), generator=g).to(dev))
        for ue8m0 in (False, True):
            want = kernels.linear_fp8(*kernels.quant_fp8(x, ue8m0=ue8m0), *f, dtype=torch.float16)
            out = torch.empty(T, N, dtype=torch.bfloat16, device=dev)
            got = mla_fp8.linear_fp8(x, f, ue8m0=ue8m0)
            assert got.dtype == torch.float16 and torch.equal(got, want)
            assert mla_fp8.linear_fp8(x, f, out=out, ue8m0=ue8m0) is out
            assert torch.equal(out, kernels.linear_fp8(*kernels.quant_fp8(x, ue8m0=ue8m0), *f))


@pytest.mark.parametrize("T,D", [(4100, 2056), (4097, 4001), (1030, 4104), (1025, 7001), (600, 1000), (2, 5), (1, 9)])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_norm_of_many_rows_and_of_few_values(dev, T, D, dt):
    """Sizes on the other side of the norm's choices by rows, and rows around eight values, against 64 bits; the sums in place."""
    from arcagi2_flashnext_dots3_amd import kernels
    g = torch.Generator().manual_seed(T)
    x, r = (torch.randn(T, D, generator=g).to(DT[dt]) for _ in range(2))
    w = 1 + 0.2 * torch.randn(D, generator=g)
    y, z = ref.normed(x, w, 1e-6, r)
    xd, rd = x.to(dev), r.to(dev)
    codes, scales = kernels.rms_norm_fp8(xd, w.to(dev), residual=rd, out=xd)
    torch.cuda.synchronize()
    assert torch.equal(rd.cpu(), z)
    assert ((xd.cpu().double() - y).abs() <= y.abs() * (ref.HALF[x.dtype] + ref.NORM_REL) + ref.TINY[x.dtype]).all()
    ref.check_codes(codes.cpu(), scales.cpu(), y)
