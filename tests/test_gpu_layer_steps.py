"""The steps of a layer together, as a serving program runs them: hidden state -> norm -> down projection -> query norm, up
projection and rotary, cache row -> attention -> output projection; eagerly on a side stream and replayed from a graph."""
import pytest
import torch

pytestmark = pytest.mark.gpu
HID, QL, H, R, K = 512, 256, 16, 256, 64


class _Layer:
    def __init__(self, dev, seed=0):
        from arcagi2_flashnext_dots3_amd import mla_fp8, rotary
        g = torch.Generator().manual_seed(seed)

        def fp8(n, k):
            w = (100 * torch.randn(n, k, generator=g)).clamp(-448, 448).to(torch.float8_e4m3fn)
            return w.to(dev), (0.01 / k ** 0.5 * torch.ones(-(-n // 128), -(-k // 128))).to(dev)

        self.n_in, self.n_q, self.n_kv = ((1 + 0.1 * torch.randn(n, generator=g)).to(torch.bfloat16).to(dev)
                                          for n in (HID, QL, 512))
        self.down, self.up, self.o = fp8(QL + 576, HID), fp8(H * 192, QL), fp8(HID, H * 128)
        self.uk = (torch.randn(H, 512, 128, generator=g).to(torch.float8_e4m3fn).view(torch.uint8).to(dev),
                   torch.full((H, 128, 4), 0.09).to(dev), False)
        self.uv = (torch.randn(H, 128, 512, generator=g).to(torch.float8_e4m3fn).view(torch.uint8).to(dev),
                   torch.full((H, 128, 4), 0.04).to(dev), True)
        self.rot = rotary.Rotary(64, device=dev)
        self.mla = mla_fp8

    def step(self, hidden, residual, residual_out, positions, slots, cache, idx):
        from arcagi2_flashnext_dots3_amd import kernels
        T = hidden.shape[0]
        x = kernels.rms_norm_fp8(hidden, self.n_in, residual=residual, residual_out=residual_out)
        down = self.mla.linear_fp8(x, self.down)
        q = self.mla.linear_fp8(kernels.rms_norm_fp8(down[:, :QL], self.n_q), self.up).view(T, H, 192)
        q_pe = self.rot.rotate(q[..., 128:], positions)
        self.rot.write_latent(down[:, QL:], self.n_kv, 1e-6, positions, slots, cache)
        query = self.mla.build_query(q[..., :128], q_pe, self.uk)
        o, _ = kernels.attend(query, cache, idx, 192 ** -0.5)
        y = torch.empty(T, H, 128, dtype=torch.bfloat16, device=hidden.device)
        self.mla.bmm_fp8(o.transpose(0, 1), self.uv, y.transpose(0, 1))
        return self.mla.linear_fp8(y.view(T, H * 128), self.o)

    def plain(self, hidden, residual, positions, slots, cache, idx):
        """The same step in float64 on the CPU from the same weights, quantized where the step quantizes."""
        c = lambda t: t.cpu()  # noqa: E731

        def q8(y):                                            # through e4m3 with a scale per 128 values
            T, D = y.shape
            p = y.view(T, -1, 128)
            s = (p.abs().amax(2, keepdim=True) / 448).clamp_min(1e-12)
            return ((p / s).float().to(torch.float8_e4m3fn).double() * s).view(T, D)

        def lin(x, f):
            N, Kd = f[0].shape
            s = c(f[1]).double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :Kd]
            return x @ (c(f[0]).double() * s).t()

        def norm(x, w):
            return x / (x.square().mean(1, keepdim=True) + 1e-6).sqrt() * c(w).double()

        def turn(x):                                          # [..., 64] interleaved
            ang = positions.double().view(-1, *[1] * (x.dim() - 1)) * c(self.rot.freqs)
            a, b = x[..., 0::2], x[..., 1::2]
            return torch.stack((a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()), -1).flatten(-2)

        T = hidden.shape[0]
        z = (hidden.float() + residual.float()).to(torch.bfloat16).double()
        down = lin(q8(norm(z, self.n_in)), self.down)
        q = lin(q8(norm(down[:, :QL], self.n_q)), self.up).view(T, H, 192)
        lat, pe = q8(norm(down[:, QL:QL + 512], self.n_kv)), turn(down[:, QL + 512:])
        rows = torch.cat((cache[:, :512].view(torch.float8_e4m3fn).double() *
                          cache[:, 512:528].contiguous().view(torch.float32).double().repeat_interleave(128, 1),
                          cache[:, 528:].contiguous().view(torch.bfloat16).double()), 1)
        rows[slots] = torch.cat((lat, pe), 1)
        uk = c(self.uk[0]).view(torch.float8_e4m3fn).double() * 0.09
        uv = c(self.uv[0]).view(torch.float8_e4m3fn).double() * 0.04
        query = torch.cat((torch.stack([q[:, h, :128] @ uk[h].t() for h in range(H)], 1), turn(q[..., 128:])), 2)
        out = []
        for t in range(T):
            kv = rows[idx[t].long()]
            p = torch.softmax(query[t] @ kv.t() * 192 ** -0.5, 1)
            o = p @ kv[:, :512]
            out.append(torch.stack([uv[h] @ o[h] for h in range(H)]).flatten())
        return lin(q8(torch.stack(out)), self.o), z


def _inputs(T, seed):
    g = torch.Generator().manual_seed(seed)
    hid, res = (torch.randn(T, HID, generator=g).to(torch.bfloat16) for _ in range(2))
    pos = torch.randint(0, 5000, (T,), generator=g)
    slots = torch.randperm(R, generator=g)[:T]
    idx = torch.stack([torch.cat((slots[t:t + 1], torch.randperm(R, generator=g)[:K - 1])) for t in range(T)])
    cache = torch.zeros(R, 656, dtype=torch.uint8)
    cache[:, :512] = torch.randn(R, 512, generator=g).to(torch.float8_e4m3fn).view(torch.uint8)
    cache[:, 512:528] = torch.full((R, 4), 1.0).view(torch.uint8)
    cache[:, 528:] = torch.randn(R, 64, generator=g).to(torch.bfloat16).view(torch.uint8)
    return hid, res, pos, slots, idx.to(torch.int32), cache


@pytest.mark.parametrize("T", [1, 37])
def test_steps_of_a_layer(dev, T):
    """Relative error (2-norm) of the whole step: some ten roundings to bf16 (2^-8 / sqrt(3) each at most) and e4m3 codes
    that a value's bf16 rounding moved to the neighbour (a code's step is 2^-3 of it, a bf16 rounding crosses a border for
    one value in 16: 2^-3 / 4 each time, at three quantizations) stay below sqrt(10 / 3) 2^-8 + 3 * 2^-5 = 0.1."""
    layer = _Layer(dev)
    hid, res, pos, slots, idx, cache = _inputs(T, T)
    want, z = layer.plain(hid, res, pos, slots, cache, idx)
    side = torch.cuda.Stream()
    d = [t.to(dev) for t in (hid, res, torch.empty_like(res), pos, slots, cache, idx)]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = layer.step(*d)
    side.synchronize()
    assert torch.equal(d[2].cpu().double(), z) and torch.equal(d[1].cpu(), res)
    assert float((got.cpu().double() - want).norm() / want.norm()) <= 0.1


def test_replayed_from_a_graph(dev):
    """Captured once, replayed on new inputs in the same buffers, with eager steps between: the eager step's bits."""
    from arcagi2_flashnext_dots3_amd import kernels
    T = 8
    layer = _Layer(dev)
    kernels.reserve_workspace(dev, H)
    bufs = [t.to(dev) for t in (lambda i: (i[0], i[1], torch.empty_like(i[1]), *i[2:4], i[5], i[4]))(_inputs(T, 0))]
    layer.step(*bufs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer.step(*bufs)
    for seed in (1, 2, 3, 4):
        hid, res, pos, slots, idx, cache = _inputs(T, seed)
        eager = [t.to(dev) for t in (hid, res, torch.empty_like(res), pos, slots, cache, idx)]
        for b, t in zip(bufs, eager):
            b.copy_(t)
        want = layer.step(*eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(bufs[5], eager[5]) and torch.equal(bufs[2], eager[2])
