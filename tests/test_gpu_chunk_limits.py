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
