"""Cached rows behind a token, whatever they hold, take no part in its attention (kernels.attend_chunk), in every kernel."""
import pytest
import torch

from tests.test_gpu_chunk import SM, _case, _check, _device

pytestmark = pytest.mark.gpu


def _behind(dev, case, i, spoil, bs, **kw):
    """Attention with the row of the only request's new token i spoiled: tokens before it as if it were not there."""
    from arcagi2_flashnext_dots3_amd import kernels
    q, cache, table, seqs, start = case
    at = int(seqs[0]) - int(start[1]) + i
    page, off = int(table[0, at // bs]), at % bs
    bad = cache.clone()
    spoil(bad[page, off])
    out, lse = kernels.attend_chunk(q.to(dev), _device(bad, dev), table.to(dev), seqs.to(dev), start.to(dev), SM, **kw)
    torch.cuda.synchronize()
    _check(out[:i].cpu(), lse[:i].cpu(), q[:i], cache, table, torch.tensor([at]), torch.tensor([0, i]), 1.0, bs)
    return out, lse


def nan_code(row):
    row[300] = 0x7F


def infinite_scale(row):
    row[516:520] = torch.tensor([float("inf")]).view(torch.uint8)


def nan_scale(row):
    row[512:516] = torch.tensor([float("nan")]).view(torch.uint8)


@pytest.mark.parametrize("heads,tokens", [(128, 12), (256, 5), (64, 20), (40, 30)])
@pytest.mark.parametrize("row,spoil", [(576, nan_code), (656, nan_code), (656, infinite_scale), (656, nan_scale)])
@pytest.mark.parametrize("items", [None, 0, 60])
def test_rows_gathered_first(dev, heads, tokens, row, spoil, items):
    """Requests of 1024 (token, head) rows or more, whose tiles are gathered with the rows of later tokens among them."""
    case = _case([700], [tokens], heads, row, 16, heads)
    for i in (1, tokens - 1):
        out, lse = _behind(dev, case, i, spoil, 16, items=items)
        if spoil is not infinite_scale:                        # (of scores that may be -inf)
            assert bool(out[i:].isnan().any(2).all())


def nan_rope(row):
    row[-64:] = 0x7F if len(row) == 576 else 0xFF


def infinite_rope(row):
    row[-64:] = 0x7F if len(row) == 576 else torch.tensor([float("inf")], dtype=torch.bfloat16).view(torch.uint8).repeat(32)


@pytest.mark.parametrize("seqs,heads,tokens,longest", [(300, 16, 5, 300), (300, 128, 3, 300), (300, 4, 70, None), (900, 128, 5, None), (900, 16, 9, None),
                                                       (40, 40, 40, None), (900, 1, 200, None), (700, 64, 20, None)])
@pytest.mark.parametrize("row,spoil", [(576, nan_code), (576, nan_rope), (656, nan_code), (656, infinite_scale), (656, nan_scale), (656, nan_rope),
                                       (656, infinite_rope)])
def test_every_kernel(dev, seqs, heads, tokens, longest, row, spoil):
    """Tiles of 32, 64 and 128 rows, of one token and of several, split or not."""
    case = _case([seqs], [tokens], heads, row, 16, heads + tokens)
    for items in (None, 0):
        _behind(dev, case, max(1, tokens // 2), spoil, 16, items=items, max_seq_len=longest)
