"""The page tables, the attention of whole prompts and that of new tokens over the cached rows as a serving loop uses them
together: a prompt step, decode steps with drafts of which some are rejected, a request that ends and one that enters."""
from types import SimpleNamespace

import pytest
import torch

from tests import refs_dense as ref

pytestmark = pytest.mark.gpu
SM, H, BS = 192 ** -0.5, 16, 16


def _impl(row):
    from arcagi2_flashnext_dots3_amd.dsa import PortableSparseImpl
    return PortableSparseImpl(H, 576, SM, 1, None, None, "fp8_ds_mla" if row == 656 else "fp8", None, "decoder", None,
                              topk_indices_buffer=torch.zeros(1, 8, dtype=torch.int32))


def _latents(n, g):
    return torch.randn(n, 512, generator=g).to(torch.bfloat16), torch.randn(n, 1, 64, generator=g).to(torch.bfloat16)


def _check(out, lse, q, start, seqs, rows, scale):
    """rows[b]: request b's cached rows in order, bytes [L, row]."""
    for b in range(len(seqs)):
        t0, t1, L = int(start[b]), int(start[b + 1]), int(seqs[b])
        n = t1 - t0
        if n == 0:
            continue
        kv = ref.rows64(rows[b]) * scale
        assert kv.shape[0] == L
        seen = torch.arange(L) <= (L - n + torch.arange(n))[:, None]
        r = ref.softmax_product(q[t0:t1].double().transpose(0, 1), kv[None], kv[None, :, :512], seen, SM)
        floor = L * 2.0 ** -29 * float(kv.abs().max())
        ref.check(out[t0:t1].transpose(0, 1), lse[t0:t1].transpose(0, 1), r, 576, L, torch.bfloat16, 2.0 ** -11, floor, f"request {b}")


@pytest.mark.parametrize("row", [656, 576])
def test_a_serving_loop(dev, row):
    from arcagi2_flashnext_dots3_amd import kernels
    from arcagi2_flashnext_dots3_amd.paging import PagePool
    g, ks = torch.Generator().manual_seed(row), 1.0 if row == 656 else 0.03
    impl, layer = _impl(row), SimpleNamespace(_k_scale_float=ks)
    M, W = 4, 12
    pool, book = PagePool(30, BS, M, W, dev), ref.Pages(30, BS, M, W)
    cache = torch.full((30, BS, row), 0x7F, dtype=torch.uint8, device=dev)         # what nobody wrote is no number
    steps = [([70, 33, 1, 0], None),                        # prompts enter
             ([1, 1, 1, 90], None),                         # decoding beside a prompt
             ([4, 4, 4, 4], [73, 36, 5, 91]),               # drafts, some rejected
             ([1, 1, 1, 1], [0, 37, 6, 92]),                # the first request ends
             ([40, 3, 3, 3], None)]                         # another one takes its place
    seen_lens = [0] * M
    for new, keep in steps:
        n, T = sum(new), sum(new) + 3                       # a padded batch
        longest = max(a + b for a, b in zip(seen_lens, new))
        md, req, pos = pool.step(torch.tensor(new, dtype=torch.int32, device=dev), n, max(new), longest, n=T)
        start, breq, bpos, bslots = book.step(new, T)
        assert md.query_start_loc.cpu().tolist() == start and req.cpu().tolist() == breq and pos.cpu().tolist() == bpos
        assert md.slot_mapping.cpu().tolist() == bslots
        kv, pe = _latents(T, g)
        impl.do_kv_cache_update(kv.to(dev), pe.to(dev), cache, md.slot_mapping, "", ks)
        q = torch.randn(T, H, 576, generator=g).to(torch.bfloat16)
        out, lse = impl.forward_dense(q.to(dev), cache, md, layer)
        torch.cuda.synchronize()
        c = cache.cpu()
        rows = [torch.stack([c[book.table[b][x // BS], x % BS] for x in range(L)]) if L else torch.zeros(0, row, dtype=torch.uint8)
                for b, L in enumerate(book.lens)]
        _check(out.cpu(), lse.cpu(), q, start, book.lens, rows, ks)
        if not any(seen_lens):                              # nothing cached before: the prompts alone give the same
            lat = torch.zeros(n, 1, 576, dtype=torch.float64)
            for b in range(M):
                lat[start[b]:start[b + 1], 0] = ref.rows64(rows[b]) * ks
            o2, z2 = impl.forward_mha(q[:n, :, :256].to(dev), lat[..., :256].to(torch.bfloat16).to(dev),
                                      lat[..., 256:512].to(torch.bfloat16).to(dev), md)
            torch.cuda.synchronize()
            for b in range(M):
                t0, t1 = start[b], start[b + 1]
                if t1 == t0:
                    continue
                k = lat[t0:t1, :, :256].to(torch.bfloat16).double().transpose(0, 1)
                v = lat[t0:t1, :, 256:512].to(torch.bfloat16).double().transpose(0, 1)
                r = ref.softmax_product(q[t0:t1, :, :256].double().transpose(0, 1), k, v, torch.ones(t1 - t0, t1 - t0, dtype=torch.bool).tril(), SM)
                ref.check(o2[t0:t1].cpu().transpose(0, 1), z2[t0:t1].cpu().transpose(0, 1), r, 256, t1 - t0, torch.bfloat16, 2.0 ** -8, 0.0, f"prompt {b}")
        if keep is not None:
            pool.trim(torch.tensor(keep, dtype=torch.int32, device=dev))
            book.trim(keep)
        book.same_as(pool)
        seen_lens = list(book.lens)


@pytest.mark.parametrize("heads,most", [(16, 600), (128, 600), (128, 700)])
def test_a_captured_decode_step(dev, heads, most):
    """A decode step with a draft (tables, rows written, attention, one draft rejected) captured once and replayed: every replay
    is the eager step over a copy of the pool and the cache, while eager calls run between."""
    from arcagi2_flashnext_dots3_amd import kernels
    from arcagi2_flashnext_dots3_amd.paging import PagePool
    M, W = 3, 48
    g = torch.Generator().manual_seed(heads)
    pools = [PagePool(100, BS, M, W, dev) for _ in range(2)]
    caches = [torch.zeros(100, BS, 656, dtype=torch.uint8, device=dev) for _ in range(2)]
    first = torch.tensor([300, 17, 150], dtype=torch.int32, device=dev)
    kv, pe = (x.to(dev) for x in _latents(467, g))
    for p, c in zip(pools, caches):
        _, _, _, slots = kernels.page_step(p, first, 467)
        kernels.cache_write(kv, pe, slots, c)
    new, cut = torch.full((M,), 2, dtype=torch.int32, device=dev), torch.zeros(M, dtype=torch.int32, device=dev)
    kv, pe, q = kv[:2 * M].clone(), pe[:2 * M].clone(), torch.zeros(2 * M, heads, 576, dtype=torch.bfloat16, device=dev)
    keep = [torch.zeros(M, dtype=torch.int32, device=dev) for _ in range(2)]

    def step(i):
        p, c = pools[i], caches[i]
        start, req, pos, slots = kernels.page_step(p, new, 2 * M)
        kernels.cache_write(kv, pe, slots, c)
        out, lse = kernels.attend_chunk(q, c, p.table, p.lens, start, SM, max_seq_len=most)
        keep[i].copy_(p.lens)
        keep[i].sub_(cut)
        kernels.page_trim(p, keep[i])
        return out, lse, slots, pos

    before = [[x.clone() for x in (p.table, p.lens, p.held, p.free, p.state)] for p in pools]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(0)
    torch.cuda.synchronize()
    for p, s in zip(pools, before):                          # capture ran nothing
        assert all(torch.equal(a, b) for a, b in zip((p.table, p.lens, p.held, p.free, p.state), s))
    for i in range(6):
        cut.copy_(torch.tensor([i % 2, (i + 1) % 2, 0], dtype=torch.int32))
        a, b = (x.to(dev) for x in _latents(2 * M, g))
        kv.copy_(a)
        pe.copy_(b)
        q.copy_(torch.randn(2 * M, heads, 576, generator=g).to(torch.bfloat16))
        graph.replay()
        want = step(1)
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y), i
        for x, y in zip((pools[0].table, pools[0].lens, pools[0].held, pools[0].free, pools[0].state),
                        (pools[1].table, pools[1].lens, pools[1].held, pools[1].free, pools[1].state)):
            assert torch.equal(x, y), i
        assert torch.equal(caches[0], caches[1])
