"""Arguments that the page, prompt and chunk calls refuse, on the CPU: by the wrappers (ValueError before the library) and by
the library (its codes before a launch); sizes of the chunk call's workspace."""
import pytest
import torch

from arcagi2_flashnext_dots3_amd import _lib, kernels
from arcagi2_flashnext_dots3_amd.paging import PagePool

BF, U8, I32, I64 = torch.bfloat16, torch.uint8, torch.int32, torch.int64


def _t(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def _refused(match, f, *a, **k):
    with pytest.raises(ValueError, match=match):
        f(*a, **k)


def test_page_step_and_trim():
    p = PagePool(10, 16, 3, 4, "cpu")
    new = _t(3, dtype=I32)
    _refused("one GPU", kernels.page_step, p, new, 5)
    _refused("one GPU", kernels.page_trim, p, new)
    _refused("n, or req", kernels.page_step, p, new)
    _refused("new \\[requests\\]", kernels.page_step, p, new[:2], 5)
    _refused("new \\[requests\\]", kernels.page_step, p, new.long(), 5)
    _refused("start", kernels.page_step, p, new, 5, start=_t(3, dtype=I32))
    _refused("req \\[n\\]", kernels.page_step, p, new, 5, req=_t(4, dtype=I32))
    _refused("positions", kernels.page_step, p, new, 5, positions=_t(5, dtype=I32))
    _refused("slots", kernels.page_step, p, new, 5, slots=_t(6, dtype=I64))
    _refused("keep", kernels.page_trim, p, _t(4, dtype=I32))

    def over(**k):
        f = dict(table=p.table, lens=p.lens, held=p.held, free=p.free, state=p.state, block_size=16)
        return PagePool.over(**{**f, **k})
    for match, pool in (("lens", over(lens=p.lens[:2])), ("held", over(held=p.held.long())), ("free", over(free=p.free[None])),
                        ("state", over(state=p.state[:3])), ("table", over(table=p.table[0])), ("at least one", over(table=p.table[:0])),
                        ("block_size", over(block_size=0)), ("overlap", over(table=p.table[:1].expand(3, 4))),
                        ("requests", over(table=_t(8193, 1, dtype=I32)))):
        _refused(match, kernels.page_trim, pool, new)


def test_attend_prompt():
    q, k, v, start = _t(6, 4, 64), _t(6, 2, 64), _t(6, 2, 32), _t(3, dtype=I32)
    f = kernels.attend_prompt
    _refused("one GPU", f, q, k, v, start, 1.0)
    _refused("q \\[T, H, D\\]", f, q[0], k, v, start, 1.0)
    _refused("fp16 / bf16", f, q.float(), k.float(), v.float(), start, 1.0)
    _refused("q's type", f, q, k.half(), v, start, 1.0)
    _refused("q's type", f, q, k, v.half(), start, 1.0)
    _refused("multiple of k's", f, _t(6, 3, 64), k, v, start, 1.0)
    _refused("multiple of k's", f, q, k[:, :0], v[:, :0], start, 1.0)
    _refused("multiples of 8", f, _t(6, 4, 60), _t(6, 2, 60), v, start, 1.0)
    _refused("multiples of 8", f, _t(6, 4, 264), _t(6, 2, 264), v, start, 1.0)
    _refused("multiples of 8", f, q, k, v[..., :0], start, 1.0)
    _refused("k \\[T, Hk, D\\]", f, q, k[:5], v, start, 1.0)
    _refused("v \\[T, Hk, Dv\\]", f, q, k, v[:, :1], start, 1.0)
    _refused("contiguous heads", f, _t(6, 4, 128)[..., ::2], k, v, start, 1.0)
    _refused("16", f, _t(6, 4, 68)[..., :64], k, v, start, 1.0)
    _refused("start", f, q, k, v, start.long(), 1.0)
    _refused("start", f, q, k, v, start[:0], 1.0)
    _refused("finite", f, q, k, v, start, float("nan"))
    _refused("out", f, q, k, v, start, 1.0, out=_t(6, 4, 64))
    _refused("out", f, q, k, v, start, 1.0, out=_t(6, 4, 32).half())
    _refused("overlap", f, q, k, v, start, 1.0, out=_t(6, 1, 32).expand(6, 4, 32))
    _refused("lse", f, q, k, v, start, 1.0, lse=_t(6, 4))


def test_attend_chunk():
    q, cache, table = _t(4, 2, 576), _t(5, 16, 656, dtype=U8), _t(3, 7, dtype=I32)
    seqs, start = _t(3, dtype=I32), _t(4, dtype=I32)
    f = kernels.attend_chunk
    _refused("one GPU", f, q, cache, table, seqs, start, 1.0)
    _refused("q \\[T, H, 576\\]", f, q[0], cache, table, seqs, start, 1.0)
    _refused("q \\[T, H, 576\\]", f, q.half(), cache, table, seqs, start, 1.0)
    _refused("q \\[T, H, 576\\]", f, _t(4, 2, 512), cache, table, seqs, start, 1.0)
    _refused("cache", f, q, cache[..., :600], table, seqs, start, 1.0)
    _refused("cache", f, q, cache.to(torch.int8), table, seqs, start, 1.0)
    _refused("contiguous", f, q, _t(5, 32, 656, dtype=U8)[:, ::2], table, seqs, start, 1.0)
    _refused("whole number of rows", f, q, _t(5 * 11000, dtype=U8).as_strided((5, 16, 656), (11000, 656, 1)), table, seqs, start, 1.0)
    _refused("whole number of rows", f, q, cache[:1].expand(5, 16, 656), table, seqs, start, 1.0)
    _refused("block_table", f, q, cache, table[:2], seqs, start, 1.0)
    _refused("block_table", f, q, cache, table.long(), seqs, start, 1.0)
    _refused("seq_lens", f, q, cache, table, seqs[:2], start, 1.0)
    _refused("seq_lens", f, q, cache, table, seqs.long(), start, 1.0)
    _refused("start", f, q, cache, table, seqs, start.long(), 1.0)
    _refused("finite", f, q, cache, table, seqs, start, float("inf"))
    _refused("items", f, q, cache, table, seqs, start, 1.0, items=-1)
    _refused("items", f, q, cache, table, seqs, start, 1.0, items=65537)
    _refused("out", f, q, cache, table, seqs, start, 1.0, out=_t(4, 2, 576))
    _refused("overlap", f, q, cache, table, seqs, start, 1.0, out=_t(1, 2, 512).expand(4, 2, 512))
    _refused("lse", f, q, cache, table, seqs, start, 1.0, lse=_t(4, 2))
    _refused("cache \\[blocks", f, q, cache[0], table, seqs, start, 1.0)


@pytest.mark.parametrize("name,args,code", [
    # (256 ...: placeholder addresses that the checks reject before anything is launched)
    ("spmla_page_step", (256, 0, 256, 256, 256, 4, 4, 256, 9, 256, 16, 5, 256, 256, 256, 256, None), -2),
    ("spmla_page_step", (256, 3, 256, 256, 256, 3, 4, 256, 9, 256, 16, 5, 256, 256, 256, 256, None), -2),
    ("spmla_page_step", (256, 3, 256, 256, 256, 4, 4, 256, 9, 256, 0, 5, 256, 256, 256, 256, None), -2),
    ("spmla_page_step", (256, 3, 256, 256, 256, 4, 4, 256, 9, 256, 16, -1, 256, 256, 256, 256, None), -2),
    ("spmla_page_step", (256, 3, 256, 256, 256, 4, 4, 256, 9, 256, 16, 5, 256, None, 256, 256, None), -2),
    ("spmla_page_step", (256, 8193, 256, 256, 256, 4, 4, 256, 9, 256, 16, 5, 256, 256, 256, 256, None), -5),
    ("spmla_page_trim", (256, 3, 256, 256, None, 4, 4, 256, 9, 256, 16, None), -2),
    ("spmla_page_trim", (256, 8193, 256, 256, 256, 4, 4, 256, 9, 256, 16, None), -5),
    ("spmla_attn_prompt", (256, 64, 64, 256, 64, 64, 256, 64, 64, 256, 1, 4, 3, 2, 64, 64, 1.0, 1, 2, 256, 64, 64, None, 0, None), -2),
    ("spmla_attn_prompt", (256, 64, 64, 256, 64, 64, 256, 64, 64, 256, 1, 4, 2, 2, 64, 64, 1.0, 1, 3, 256, 64, 64, None, 0, None), -2),
    ("spmla_attn_prompt", (256, 64, 64, 256, 64, 64, 256, 64, 64, 256, 1, 4, 2, 2, 264, 64, 1.0, 1, 2, 256, 64, 64, None, 0, None), -5),
    ("spmla_attn_prompt", (256, 64, 64, 256, 64, 64, 256, 64, 64, 256, 1, 4, 2, 2, 60, 64, 1.0, 1, 2, 256, 64, 64, None, 0, None), -3),
    ("spmla_attn_prompt", (256, 64, 64, 264, 64, 64, 256, 64, 64, 256, 1, 4, 2, 2, 64, 64, 1.0, 1, 2, 256, 64, 64, None, 0, None), -3),
    ("spmla_attn_prompt", (256, 64, 68, 256, 64, 64, 256, 64, 64, 256, 1, 4, 2, 2, 64, 64, 1.0, 1, 2, 256, 64, 64, None, 0, None), -3),
    ("spmla_attn_prompt", (None, 64, 64, 256, 64, 64, 256, 64, 64, 256, 1, 4, 2, 2, 64, 64, 1.0, 1, 2, 256, 64, 64, None, 0, None), -2),
    ("spmla_attn_prompt", (256, 64, 64, 256, 64, 64, 256, 64, 64, 256, 1, 0, 2, 2, 64, 64, 1.0, 1, 2, 256, 64, 64, None, 0, None), 0),
    ("spmla_attn_chunk", (256, 576, 576, 256, 80, 600, 16, 16, 256, 5, 5, 256, 256, 3, 4, 2, 1.0, 1.0, 80, 0, 256, 512, 512, None, 0, None, 0, None), -2),
    ("spmla_attn_chunk", (256, 576, 576, 256, 80, 656, 16, 15, 256, 5, 5, 256, 256, 3, 4, 2, 1.0, 1.0, 80, 0, 256, 512, 512, None, 0, None, 0, None), -2),
    ("spmla_attn_chunk", (256, 576, 576, 256, 80, 656, 16, 16, 256, 5, 5, 256, 256, 3, 4, 2, 1.0, 1.0, -1, 0, 256, 512, 512, None, 0, None, 0, None), -2),
    ("spmla_attn_chunk", (256, 576, 576, 256, 80, 656, 16, 16, 256, 5, 5, 256, None, 3, 4, 2, 1.0, 1.0, 80, 0, 256, 512, 512, None, 0, None, 0, None), -2),
    ("spmla_attn_chunk", (256, 576, 576, 264, 80, 656, 16, 16, 256, 5, 5, 256, 256, 3, 4, 2, 1.0, 1.0, 80, 0, 256, 512, 512, None, 0, None, 0, None), -3),
    ("spmla_attn_chunk", (256, 580, 576, 256, 80, 656, 16, 16, 256, 5, 5, 256, 256, 3, 4, 2, 1.0, 1.0, 80, 0, 256, 512, 512, None, 0, None, 0, None), -3),
    # splits without a workspace, with one that is too small or off its alignment; more of them than the join takes
    ("spmla_attn_chunk", (256, 576, 576, 256, 80, 656, 16, 16, 256, 5, 5, 256, 256, 3, 4, 2, 1.0, 1.0, 80, 64, 256, 512, 512, None, 0, None, 0, None), -2),
    ("spmla_attn_chunk", (256, 576, 576, 256, 80, 656, 16, 16, 256, 5, 5, 256, 256, 3, 4, 2, 1.0, 1.0, 80, 64, 256, 512, 512, None, 0, 256, 4096, None), -2),
    ("spmla_attn_chunk", (256, 576, 576, 256, 80, 656, 16, 16, 256, 5, 5, 256, 256, 3, 4, 2, 1.0, 1.0, 80, 64, 256, 512, 512, None, 0, 264, 1 << 40, None), -3),
    ("spmla_attn_chunk", (256, 576, 576, 256, 80, 656, 16, 16, 256, 5, 5, 256, 256, 3, 4, 2, 1.0, 1.0, 80, 1000, 256, 512, 512, None, 0, 256, 1 << 40, None), -5),
    ("spmla_attn_chunk", (256, 576, 576, 256, 1 << 31, 656, 16, 16, 256, 5, 5, 256, 256, 3, 4, 2, 1.0, 1.0, 80, 0, 256, 512, 512, None, 0, None, 0, None), -5),
    ("spmla_attn_chunk", (256, 576, 576, 256, 80, 656, 16, 16, 256, 5, 5, 256, 256, 0, 4, 2, 1.0, 1.0, 80, 0, 256, 512, 512, None, 0, None, 0, None), 0),
])
def test_codes_before_a_launch(name, args, code):
    assert getattr(_lib.lib(), name)(*args) == code


def test_chunk_workgroups_and_workspace():
    items, ws = kernels.chunk_items, kernels.chunk_ws_bytes
    assert items(1, 128, 1, 656, 65536) == 256                    # one tile of query rows: the whole chip
    assert items(64, 128, 64, 656, 6000) == 256
    assert items(250, 128, 250, 656, 6000) == 256 + 64            # few beyond one a tile: some for the longest requests
    assert items(1024, 128, 1, 576, 16384) == 0                   # four rounds and more: no splits
    assert items(257, 128, 257, 656, 6000) == 0                   # more requests than the shares are formed for
    assert items(1, 128, 1, 656, 192) == 0 and items(1, 128, 1, 656, 193) == 256 and items(0, 128, 1, 656, 9999) == 0
    assert ws(1, 128, 1, 656, 65536, 0) == 0 and ws(1, 128, 1, 656, 0, 256) == 0
    assert ws(1, 128, 1, 656, 65536, 1) == 0                      # no more workgroups than tiles
    assert ws(1, 128, 1, 656, 65536, 256) == 128 * 8 + 16 + 256 * 128 * 513 * 4
    images = 512 * (9 * 4096 + 1024)                              # 16384 rows, gathered first
    assert ws(1024, 128, 1, 576, 16384, 0) == images
    assert ws(7, 128, 1, 576, 16384, 0) == 0 and ws(8, 128, 1, 576, 16384, 0) == images
    assert ws(1024, 128, 8, 656, 1 << 20, 0) == 0                 # beyond 4 GiB: rows are converted where they are used


def test_forward_dense_refuses(monkeypatch):
    from arcagi2_flashnext_dots3_amd.dsa import CommonAttentionMetadata, PortableSparseImpl
    impl = PortableSparseImpl(8, 576, 0.1, 1, None, None, "fp8_ds_mla", None, "decoder", None, topk_indices_buffer=_t(4, 64, dtype=I32))
    md = CommonAttentionMetadata(query_start_loc=_t(2, dtype=I32), num_reqs=1, num_actual_tokens=4, max_query_len=4, max_seq_len=16,
                                 slot_mapping=_t(4, dtype=I64), block_table_tensor=_t(1, 1, dtype=I32))
    cache = _t(2, 16, 656, dtype=U8)
    _refused("seq_lens", impl.forward_dense, _t(4, 8, 576), cache, md)
    md.seq_lens = _t(1, dtype=I32)
    _refused("one GPU", impl.forward_dense, _t(4, 8, 576), cache, md)
    _refused("one GPU", impl.forward_dense, (_t(4, 8, 512), _t(4, 8, 64)), cache, md)
    monkeypatch.setattr(impl, "_offload", True)
    with pytest.raises(NotImplementedError):
        impl.forward_dense(_t(4, 8, 576), cache, md)
