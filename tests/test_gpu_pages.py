"""Block tables and slot maps built on the GPU against the same steps on Python lists."""
import random

import pytest
import torch

from tests.refs_dense import Pages

pytestmark = pytest.mark.gpu


def _ints(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _step(pool, ref, new, n, dev):
    from arcagi2_flashnext_dots3_amd import kernels
    got = kernels.page_step(pool, _ints(new, dev), n)
    want = ref.step(new, n)
    for g, w, name in zip(got, want, ("start", "req", "positions", "slots")):
        assert g.cpu().tolist() == w, name
    ref.same_as(pool)


def _trim(pool, ref, keep, dev):
    from arcagi2_flashnext_dots3_amd import kernels
    kernels.page_trim(pool, _ints(keep, dev))
    ref.trim(keep)
    ref.same_as(pool)


# one request; more than a workgroup's; many workgroups of tokens; odd pages, pages of one row
@pytest.mark.parametrize("M,bs,W,pages,most", [(1, 64, 8, 8, 200), (5, 1, 40, 120, 12), (17, 48, 30, 400, 300),
                                               (300, 16, 12, 2500, 40), (1500, 64, 6, 9000, 9), (40, 7, 4000, 60000, 9000),
                                               (8192, 16, 3, 20000, 7)])
def test_steps_and_trims(dev, M, bs, W, pages, most):
    from arcagi2_flashnext_dots3_amd.paging import PagePool
    rng = random.Random(M * bs)
    pool, ref = PagePool(pages, bs, M, W, dev), Pages(pages, bs, M, W)
    ref.same_as(pool)
    for k in range(4):
        new = [rng.choice([0, 1, 1, rng.randrange(most)]) for _ in range(M)]
        total = sum(new)
        _step(pool, ref, new, [total, total + 13, max(0, total - 5), total][k], dev)
        _trim(pool, ref, [rng.choice([0, x, x + 9, rng.randrange(x + 1)]) for x in ref.lens], dev)


def test_stack_runs_out_and_refills(dev):
    from arcagi2_flashnext_dots3_amd.paging import PagePool
    pool, ref = PagePool(10, 16, 4, 20, dev), Pages(10, 16, 4, 20)
    _step(pool, ref, [40, 100, 16, 1], 157, dev)               # 12 pages wanted, 10 there
    assert ref.missing == 2
    _step(pool, ref, [0, 0, 0, 0], 0, dev)
    _trim(pool, ref, [0, 200, 200, 200], dev)
    _step(pool, ref, [0, 1, 1, 1], 3, dev)                     # what was missing is filled in
    assert ref.missing == 0
    _trim(pool, ref, [0, 0, 0, 0], dev)
    assert sorted(ref.free) == list(range(10))


def test_table_width_ends(dev):
    """Tokens behind the table's last column have no slot; the request goes on holding W pages."""
    from arcagi2_flashnext_dots3_amd.paging import PagePool
    pool, ref = PagePool(100, 4, 2, 3, dev), Pages(100, 4, 2, 3)
    _step(pool, ref, [20, 5], 25, dev)
    _step(pool, ref, [3, -7], 3, dev)                          # (a negative count is none)
    _trim(pool, ref, [9, -1], dev)


def test_step_then_trim_is_the_identity(dev):
    from arcagi2_flashnext_dots3_amd import kernels
    from arcagi2_flashnext_dots3_amd.paging import PagePool
    pool = PagePool(500, 16, 30, 40, dev)
    g = torch.Generator().manual_seed(1)
    pool.free.copy_(torch.randperm(500, generator=g))
    kernels.page_step(pool, torch.randint(0, 90, (30,), generator=g).int().to(dev), 3000)
    before = [t.clone() for t in (pool.table, pool.lens, pool.held, pool.free, pool.state[:1])]
    kernels.page_step(pool, torch.randint(0, 90, (30,), generator=g).int().to(dev), 3000)
    kernels.page_trim(pool, before[1])
    for a, b in zip((pool.table, pool.lens, pool.held, pool.free, pool.state[:1]), before):
        assert torch.equal(a, b)


def test_captured_decode_loop(dev):
    """A captured step and trim, replayed: each replay as the eager calls."""
    from arcagi2_flashnext_dots3_amd import kernels
    from arcagi2_flashnext_dots3_amd.paging import PagePool
    M, n = 40, 90
    pool, ref = PagePool(600, 4, M, 60, dev), Pages(600, 4, M, 60)
    new, keep = _ints([0] * M, dev), _ints([0] * M, dev)
    out = dict(start=torch.zeros(M + 1, dtype=torch.int32, device=dev), req=torch.zeros(n, dtype=torch.int32, device=dev),
               positions=torch.zeros(n, dtype=torch.int64, device=dev), slots=torch.zeros(n, dtype=torch.int64, device=dev))
    kernels.page_step(pool, new, n, **out)
    kernels.page_trim(pool, keep)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kernels.page_step(pool, new, n, **out)
        kernels.page_trim(pool, keep)
    rng = random.Random(3)
    for _ in range(6):
        cnt = [rng.randrange(4) for _ in range(M)]
        kp = [max(0, x + c - rng.randrange(3)) for x, c in zip(ref.lens, cnt)]
        new.copy_(_ints(cnt, dev))
        keep.copy_(_ints(kp, dev))
        g.replay()
        want = ref.step(cnt, n)
        ref.trim(kp)
        torch.cuda.synchronize()
        for k, w in zip(("start", "req", "positions", "slots"), want):
            assert out[k].cpu().tolist() == w, k
        ref.same_as(pool)
