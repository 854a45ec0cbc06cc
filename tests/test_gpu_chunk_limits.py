"""Calls at the limits that kernels.attend_chunk documents."""
import pytest
import torch

from tests.test_gpu_chunk import SM, _case, _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("row,heads,lens,seqs,items", [
    (656, 16, [0] * 100 + [1] + [0] * 155, [0] * 100 + [80000] + [0] * 155, 767),      # 511 beyond the 256 counted tiles, one tile alone
    (656, 32, [1] * 256, [64] * 200 + [60000] + [64] * 55, 895),
    (656, 64, [2], [51000], 513), (576, 8, [1], [51000], 512), (576, 128, [1], [51000], 512)])
def test_as_many_workgroups_as_may_be(dev, row, heads, lens, seqs, items):
    """511 workgroups beyond one a tile, where requests without tokens or short ones leave them to one long request."""
    from arcagi2_flashnext_dots3_amd import kernels
    q, cache, table, s, start = _case(seqs, lens, heads, row, 64, items)
    T = q.shape[0]
    out = torch.full((T, heads, 512), 7.0, dtype=torch.bfloat16, device=dev)
    lse = torch.full((T, heads), 7.0, device=dev)
    kernels.attend_chunk(q.to(dev), cache.to(dev), table.to(dev), s.to(dev), start.to(dev), SM, out=out, lse=lse, items=items)
    torch.cuda.synchronize()
    _check(out.cpu(), lse.cpu(), q, cache, table, s, start, 1.0, 64)
    with pytest.raises(Exception, match="limit"):
        kernels.attend_chunk(q.to(dev), cache.to(dev), table.to(dev), s.to(dev), start.to(dev), SM, items=items + 300)


@pytest.mark.parametrize("row", [656, 576])
@pytest.mark.parametrize("heads,lens,seqs,T", [(16, [2, 9], [300, 150], 7), (128, [1, 3], [300, 400], 3), (128, [4, 30], [700, 900], 20),
                                               (24, [5, 6, 7], [300, 200, 100], 8), (16, [60], [90], 1)])
def test_fewer_places_than_tokens(dev, row, heads, lens, seqs, T):
    """A step cut to T places (page_step: tokens beyond have none): the tokens that are there see what they would see in the
    whole step."""
    from arcagi2_flashnext_dots3_amd import kernels
    q, cache, table, s, start = _case(seqs, lens, heads, row, 16, T)
    args = [x.to(dev) for x in (q[:T], cache, table, s, start)] + [SM]
    short = start.clamp(max=T)
    cut = (start[1:] - start[:-1]) - (short[1:] - short[:-1])
    for items in (None, 0, 40):
        out, lse = kernels.attend_chunk(*args, items=items)
        torch.cuda.synchronize()
        _check(out.cpu(), lse.cpu(), q[:T], cache, table, s - cut, short, 1.0, 16)


@pytest.mark.parametrize("row", [656, 576])
@pytest.mark.parametrize("heads,lens,seqs,items", [(16, [2] * 40, [100] * 40, 0), (32, [2] * 60, [70] * 60, 0), (40, [1] * 30, [150] * 30, None),
                                                   (128, [1, 2, 1], [2000, 500, 60], None), (128, [9, 10], [700, 800], None)])
def test_same_bits_again(dev, row, heads, lens, seqs, items):
    """The same inputs give the same bits, whatever the waves' order (tiles of 32, 64 and 128 rows, splits, gathered rows)."""
    from arcagi2_flashnext_dots3_amd import kernels
    q, cache, table, s, start = case = _case(seqs, lens, heads, row, 16, heads)
    args = [x.to(dev) for x in case] + [SM]
    out, lse = kernels.attend_chunk(*args, items=items)
    torch.cuda.synchronize()
    _check(out.cpu(), lse.cpu(), q, cache, table, s, start, 1.0, 16)
    more = [kernels.attend_chunk(*args, items=items) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, out) and torch.equal(z, lse) for o, z in more)
