"""Row656 scales of any size in the attention over all cached rows: zero, the smallest, far apart between the groups of 128."""
import pytest
import torch

from tests import refs_dense as ref
from tests.test_gpu_chunk import SM, _case, _device

pytestmark = pytest.mark.gpu
# rows of few heads; a tile of one token; 128 rows of several tokens; gathered first
SHAPES = [([300], [1], 16), ([700, 90], [2, 1], 24), ([700], [1], 128), ([300], [20], 64), ([700], [12], 128), ([1500, 40], [1, 1], 128)]


def _scales(cache, table, b, x, bs):
    """The four scales of request b's positions x, as a copy, and how to put them back."""
    page, off = table[b].long()[x // bs], x % bs
    old = cache[page, off]

    def put(scales, codes=None):
        old[:, 512:528] = scales.contiguous().view(torch.uint8).view(-1, 16)
        if codes is not None:
            old[:, :512] = codes
        cache[page, off] = old
    return old[:, 512:528].contiguous().view(torch.float32).clone(), put


def _check(out, lse, q, cache, table, seqs, start, bs):
    """The bounds of test_gpu_chunk, but for what subnormal weights lose: 2^-29 of the largest latent of the same group a position."""
    for b in range(len(seqs)):
        t0, t1, L = int(start[b]), int(start[b + 1]), int(seqs[b])
        x = torch.arange(L)
        raw = cache[table[b].long()[x // bs], x % bs]
        rows = ref.rows64(raw)
        seen = x <= (L - (t1 - t0) + torch.arange(t1 - t0))[:, None]
        r = ref.softmax_product(q[t0:t1].double().transpose(0, 1), rows[None], rows[None, :, :512], seen, SM)
        top = raw[:, 512:528].contiguous().view(torch.float32).double().abs().amax(0).repeat_interleave(128) * 448.0
        ref.check(out[t0:t1].transpose(0, 1), lse[t0:t1].transpose(0, 1), r, 576, L, torch.bfloat16, ref.HALF[torch.float16],
                  L * 2.0 ** -29 * top, f"request {b}")


def _run(dev, case, bs, **kw):
    from arcagi2_flashnext_dots3_amd import kernels
    q, cache, table, seqs, start = case
    args = q.to(dev), _device(cache, dev), table.to(dev), seqs.to(dev), start.to(dev), SM
    for items in (None, 0):
        out, lse = kernels.attend_chunk(*args, items=items, **kw)
        torch.cuda.synchronize()
        assert bool(out.isfinite().all()) and bool(lse.isfinite().all())
        _check(out.cpu(), lse.cpu(), q, cache, table, seqs, start, bs)
    return out, lse


@pytest.mark.parametrize("seqs,lens,heads", SHAPES)
@pytest.mark.parametrize("scale", [0.0, 2.0 ** -126, 2.0 ** -115, 2.0 ** -101, 2.0 ** -60])
@pytest.mark.parametrize("where", ["all", "first", "odd tiles", "one group"])
def test_small_scales(dev, seqs, lens, heads, scale, where):
    """Zero-filled rows and rows of the smallest scales: everywhere, before ordinary ones, in every second tile, in a group."""
    q, cache, table, s, start = case = _case(seqs, lens, heads, 656, 16, heads)
    for b, L in enumerate(seqs):
        x = torch.arange(L)
        x = x[:70] if where == "first" else x[x // 32 % 2 == 1] if where == "odd tiles" else x
        if len(x):
            old, put = _scales(cache, table, b, x, 16)
            old[:, 1 if where == "one group" else slice(None)] = scale
            put(old)
    out, lse = _run(dev, case, 16)
    if scale == 0.0 and where in ("all", "one group"):
        assert bool((out[..., slice(128, 256) if where == "one group" else slice(None)] == 0).all())


@pytest.mark.parametrize("seqs,lens,heads", SHAPES)
@pytest.mark.parametrize("apart", [12, 24, 50, 100])
def test_groups_far_apart(dev, seqs, lens, heads, apart):
    """Latents of one group 2^-apart of the others': its part of the output keeps its precision."""
    q, cache, table, s, start = case = _case(seqs, lens, heads, 656, 16, heads + apart)
    for b, L in enumerate(seqs):
        old, put = _scales(cache, table, b, torch.arange(L), 16)
        old[:, 2] *= 2.0 ** -apart
        put(old)
    _run(dev, case, 16)


@pytest.mark.parametrize("seqs,lens,heads", [([300], [5], 16), ([300], [20], 128), ([700], [12], 128)])
def test_large_scales_behind_a_token(dev, seqs, lens, heads):
    """A later token's row of 2^60 times the others' latents takes nothing from the tokens before it."""
    from arcagi2_flashnext_dots3_amd import kernels
    q, cache, table, s, start = _case(seqs, lens, heads, 656, 16, 3)
    i = lens[0] - 2
    at = seqs[0] - lens[0] + i
    far = cache.clone()
    old, put = _scales(far, table, 0, torch.tensor([at]), 16)
    put(old * 2.0 ** 60)
    for items in (None, 0):
        out, lse = kernels.attend_chunk(q.to(dev), far.to(dev), table.to(dev), s.to(dev), start.to(dev), SM, items=items)
        torch.cuda.synchronize()
        _check(out[:i].cpu(), lse[:i].cpu(), q[:i], cache, table, torch.tensor([at]), torch.tensor([0, i]), 16)


@pytest.mark.parametrize("seqs,lens,heads,items", [([150], [150], 1, None), ([40], [40], 4, None), ([300], [130], 2, 0), ([300], [130], 2, 30),
                                                   ([330], [300], 16, None), ([700], [200], 8, 40), ([1000, 200], [100, 50], 16, None),
                                                   ([64, 30], [5, 30], 6, None), ([25], [25], 128, None)])
@pytest.mark.parametrize("spread", [2, 20, 60])
def test_scales_of_every_size_in_a_chunk(dev, seqs, lens, heads, items, spread):
    """Scales from 2^-spread to 2^spread of the ordinary ones at random, by position and group, under weights that do not depend on
    them (rope alone): each token's output keeps the precision that the largest scale of the group among the rows it sees leaves."""
    from arcagi2_flashnext_dots3_amd import kernels
    q, cache, table, s, start = _case(seqs, lens, heads, 656, 16, heads + spread)
    q[..., :512] = 0
    g = torch.Generator().manual_seed(spread)
    for b, L in enumerate(seqs):
        old, put = _scales(cache, table, b, torch.arange(L), 16)
        put(old * 2.0 ** (spread * (2 * torch.rand(L, 4, generator=g) - 1)))
    out, lse = kernels.attend_chunk(q.to(dev), cache.to(dev), table.to(dev), s.to(dev), start.to(dev), SM, items=items)
    torch.cuda.synchronize()
    out, lse = out.cpu(), lse.cpu()
    assert bool(out.isfinite().all())
    for b, L in enumerate(seqs):
        t0, t1 = int(start[b]), int(start[b + 1])
        x = torch.arange(L)
        raw = cache[table[b].long()[x // 16], x % 16]
        rows = ref.rows64(raw)
        last = L - (t1 - t0) + torch.arange(t1 - t0)
        r = ref.softmax_product(q[t0:t1].double().transpose(0, 1), rows[None], rows[None, :, :512], x <= last[:, None], SM)
        top = raw[:, 512:528].contiguous().view(torch.float32).double().abs().cummax(0).values[last].repeat_interleave(128, 1) * 448.0
        ref.check(out[t0:t1].transpose(0, 1), lse[t0:t1].transpose(0, 1), r, 576, L, torch.bfloat16, ref.HALF[torch.float16],
                  L * 2.0 ** -29 * top, f"request {b}")
