"""The plugin's vLLM sparse-MLA attention backend (reference dotsnote/engine/arcstats_pkg/arcstats/dsa_sm89.py:216-530)
on libspmla_gfx950.so, without vLLM: the same class names, methods, arguments and metadata fields, with the metadata
objects duck-typed (the dataclasses below carry exactly the fields the backend reads).

  PortableSparseBackend   get_name / get_impl_cls / get_builder_cls / get_metadata_cls / get_supported_head_sizes
  PortableXPUBuilder      build(common_prefix_len, common_attn_metadata) -> SparseMetadata (req_id_per_token by
                          searchsorted over query_start_loc, dsa_sm89.py:484-499)
  PortableSparseImpl      do_kv_cache_update (quantize-and-pack into the paged cache, or into the host pool of the
                          offload layer) and forward_mqa (paged: top-k positions -> cache rows -> attention; offload:
                          LayerOffload.attend for decode tokens, staged rows for prefill chunks)

Cache rows: the paged cache is [num_blocks, block_size, 656] uint8 Row656 ("fp8_ds_mla": 512 e4m3 codes, 4 fp32
scales, 64 bf16 rope) or [num_blocks, block_size, 576] uint8 Row576 ("fp8", the reference's deployed per-tensor
rows, dsa_sm89.py:551-562): do_kv_cache_update writes either; forward_mqa attends either in place, Row576 rows with
the layer's kv_scale (dsa_sm89.py:379-391).
"""
import dataclasses
import os
from typing import Any, List, Optional

import torch

from . import kernels
from .diagnostics import verify_outputs
from .sparse_offload import LayerOffload


# ------------------------------------------------------------------------------------------------ index helpers
def convert_req_index_to_global_index(req_id, block_table, token_indices, BLOCK_SIZE=64, NUM_TOPK_TOKENS=2048,
                                      BLOCK_STRIDE_ROWS=None, return_valid_counts=False):
    """vLLM's triton_convert_req_index_to_global_index (called at dsa_sm89.py:314-315, :460-462, :467-469):
    row = block_table[req_id[t], p // BLOCK_SIZE] * BLOCK_STRIDE_ROWS + p % BLOCK_SIZE for p = token_indices[t, k]
    >= 0 inside the table, else -1 -> int32 [T, NUM_TOPK_TOKENS] (and the per-token count of valid rows)."""
    T = token_indices.shape[0]
    tk = token_indices if token_indices.shape[1] <= NUM_TOPK_TOKENS else token_indices[:, :NUM_TOPK_TOKENS]
    tk = tk if tk.dtype == torch.int32 else tk.to(torch.int32)
    bt = block_table if block_table.dtype == torch.int32 else block_table.to(torch.int32)
    rid = req_id if req_id.dtype == torch.int32 else req_id.to(torch.int32)
    counts = torch.empty(T, dtype=torch.int32, device=tk.device) if return_valid_counts else None
    rows = kernels.rows_from_topk(tk, (rid if rid.shape[0] == T else rid[:T]).contiguous(), bt, BLOCK_SIZE,
                                  stride_rows=BLOCK_STRIDE_ROWS if BLOCK_STRIDE_ROWS is not None else BLOCK_SIZE,
                                  counts=counts)
    return (rows, counts) if return_valid_counts else rows


def compact_stage(rows, sidx):
    """rows [tot] int64 host rows of a prefill chunk's context, sidx [M, K] int32 positions into them (-1 = none)
    -> (sel [U] int64 rows of the distinct selected positions in ascending order, sidx2 [M, K] int32 into sel)
    (reference compact_stage, dsa_sm89.py:27-35). Reads U back to the host once, as the reference does."""
    sel, U, sidx2 = kernels.compact_stage(rows.to(torch.int64).contiguous(), sidx.to(torch.int32).contiguous())
    return sel[:int(U.item())], sidx2


# ------------------------------------------------------------------------------------------------ metadata
@dataclasses.dataclass
class CommonAttentionMetadata:
    """The fields of vLLM's CommonAttentionMetadata that the builder reads."""
    query_start_loc: torch.Tensor        # [num_reqs + 1] int32
    num_reqs: int
    num_actual_tokens: int
    max_query_len: int
    max_seq_len: int
    slot_mapping: torch.Tensor           # [num_actual_tokens] int64
    block_table_tensor: torch.Tensor     # [num_reqs, max_blocks] int32
    seq_lens: Optional[torch.Tensor] = None


@dataclasses.dataclass
class SparseMetadata:
    """XPUMLASparseMetadata fields used by forward_mqa (paged path)."""
    num_reqs: int
    max_query_len: int
    max_seq_len: int
    num_actual_tokens: int
    query_start_loc: torch.Tensor
    slot_mapping: torch.Tensor
    block_table: torch.Tensor
    req_id_per_token: torch.Tensor
    block_size: int
    topk_tokens: int
    num_decodes: int = 0
    num_prefills: int = 0
    num_decode_tokens: int = 0
    num_prefill_tokens: int = 0


@dataclasses.dataclass
class DecodeMetadata:
    """Indexer decode metadata fields read by the offload path (dsa_sm89.py:299-316)."""
    block_table: torch.Tensor            # [num_decodes (or decode tokens), max_blocks] int32
    seq_lens: torch.Tensor
    decode_lens: torch.Tensor
    requires_padding: bool = False


@dataclasses.dataclass
class PrefillChunk:
    """One prefill chunk (dsa_sm89.py:320-331): tokens [token_start, token_end) over total_seq_lens context rows."""
    token_start: int
    token_end: int
    total_seq_lens: int
    token_to_seq: torch.Tensor           # [total_seq_lens] int32: request of each context position
    cu_seq_lens: torch.Tensor            # [num_seqs + 1] int32: first context position of each request
    block_table: torch.Tensor            # [num_seqs, max_blocks] int32
    cu_seqlen_ks: torch.Tensor           # [tokens] int32: first context position of each query token's request
    cu_seqlen_ke: torch.Tensor


@dataclasses.dataclass
class PrefillMetadata:
    chunks: List[PrefillChunk]


@dataclasses.dataclass
class IndexerMetadata:
    """The indexer's metadata as the offload path reads it (num_decode_tokens, num_decodes, num_prefill_tokens,
    decode, prefill)."""
    num_decode_tokens: int
    num_decodes: int
    num_prefill_tokens: int
    decode: Optional[DecodeMetadata] = None
    prefill: Optional[PrefillMetadata] = None


class PortableXPUBuilder:
    """Metadata builder (reference PortableXPUBuilder, dsa_sm89.py:484-499): the request of every query token is
    produced on the device, with no host round trip -- here by expanding the request ids over their query lengths
    (repeat_interleave with the output size given, which needs no device-to-host read); buffer entries past the step's
    tokens hold the last request."""

    def __init__(self, block_size, topk_tokens, max_num_tokens, device):
        self.block_size = int(block_size)
        self.topk_tokens = int(topk_tokens)
        self.req_id_per_token_buffer = torch.zeros(max_num_tokens, dtype=torch.int32, device=device)

    def _request_of_token(self, qsl, num_reqs, n):
        buf = self.req_id_per_token_buffer
        last = max(num_reqs - 1, 0)
        if n and num_reqs:
            bounds = qsl[: num_reqs + 1].to(device=buf.device, dtype=torch.int64)
            per_req = bounds[1:] - bounds[:-1]
            ids = torch.arange(num_reqs, device=buf.device, dtype=torch.int32)
            buf[:n] = torch.repeat_interleave(ids, per_req, output_size=n)
        buf[n:].fill_(last)
        return buf[:n]

    def build(self, common_prefix_len, common_attn_metadata, fast_build=False):
        cam = common_attn_metadata
        n = cam.num_actual_tokens
        fields = dict(num_reqs=cam.num_reqs, max_query_len=cam.max_query_len, max_seq_len=cam.max_seq_len,
                      num_actual_tokens=n, query_start_loc=cam.query_start_loc, slot_mapping=cam.slot_mapping,
                      block_table=cam.block_table_tensor, block_size=self.block_size, topk_tokens=self.topk_tokens)
        # every token is treated as a decode token of the paged path (the indexer's own metadata splits decode and
        # prefill for the offload path)
        fields.update(req_id_per_token=self._request_of_token(cam.query_start_loc, cam.num_reqs, n),
                      num_decodes=cam.num_reqs, num_prefills=0, num_decode_tokens=n)
        return SparseMetadata(**fields)


# ------------------------------------------------------------------------------------------------ impl
class PortableSparseImpl:
    """Sparse-MLA attention layer implementation (reference PortableSparseImpl, dsa_sm89.py:216-470).

    head_size = 576 (512 latent + 64 rope), scale = softmax scale, kv_lora_rank = 512 (from mla_args, default 512).
    topk_indices_buffer [max_tokens, topk] int32: request-local positions chosen by the indexer (-1 = none).
    offload: keep the rows in pinned host memory behind an HBM hot-row cache (reference ARC_DOTS3_OFFLOAD=1; also
    read from that variable when not given); cache_rows: HBM cache lines of the offload layer.
    """
    masked_mha_available = False

    def __init__(self, num_heads, head_size, scale, num_kv_heads, alibi_slopes, sliding_window, kv_cache_dtype,
                 logits_soft_cap, attn_type, kv_sharing_target_layer_name, topk_indices_buffer=None, indexer=None,
                 offload=None, cache_rows=0, verify=None, **mla_args):
        self.num_heads = int(num_heads)
        self.head_size = int(head_size)
        self.softmax_scale = float(scale)
        self.num_kv_heads = num_kv_heads
        self.kv_cache_dtype = kv_cache_dtype
        self.kv_lora_rank = int(mla_args.get("kv_lora_rank", kernels.D_LAT))
        self.topk_indices_buffer = topk_indices_buffer
        self._indexer_mod = indexer
        self._offload = (os.environ.get("ARC_DOTS3_OFFLOAD") == "1") if offload is None else bool(offload)
        # offload mode checked against the paged path every step (ARC_OFFLOAD_VERIFY): both caches are written and the
        # paged output is returned; verify_stats counts calls, tokens, bad tokens and the largest relative error
        self._verify = (os.environ.get("ARC_OFFLOAD_VERIFY") == "1") if verify is None else bool(verify)
        self.verify_stats = {}
        self._cache_rows = int(cache_rows)
        self._off = None
        self._off_key = None
        if self.head_size != kernels.D_QK or self.kv_lora_rank != kernels.D_LAT:
            raise ValueError(f"PortableSparseImpl: head_size 576 / kv_lora_rank 512 required, got "
                             f"{self.head_size} / {self.kv_lora_rank}")
        if alibi_slopes is not None or sliding_window is not None or logits_soft_cap is not None:
            raise NotImplementedError("PortableSparseImpl: alibi, sliding window and soft cap are not supported")

    # ---- cache layout helpers
    @staticmethod
    def _rows_view(kv_cache):
        """(pointer tensor, number of addressable rows, rows between block starts, row bytes) of a paged or flat
        cache of uint8 rows."""
        c = kv_cache.view(torch.uint8) if kv_cache.dtype != torch.uint8 else kv_cache
        rb = c.shape[-1]
        if c.dim() == 3:
            if c.stride(0) % rb or c.stride(1) != rb:
                raise ValueError("paged cache: block stride must be a whole number of rows")
            sr = c.stride(0) // rb
            return c, (c.shape[0] - 1) * sr + c.shape[1], sr, rb
        return c, c.shape[0], None, rb

    def _off_state(self, kv_cache):
        c = kv_cache if kv_cache.dim() == 3 else kv_cache.view(-1, 1, kv_cache.shape[-1])
        key = (c.data_ptr(), c.shape[0], c.shape[1])
        if self._off is None or self._off_key != key:
            self._off = LayerOffload(c.shape[0] * c.shape[1], c.device, cache_rows=self._cache_rows)
            self._off_key = key
            self._block_size = c.shape[1]
        return self._off

    # ---- KV write
    def do_kv_cache_update(self, kv_c_normed, k_pe, kv_cache, slot_mapping, kv_cache_dtype, k_scale):
        """Quantize-and-pack kv_c_normed [n, 512] bf16 + k_pe [n, 1, 64] bf16 into the rows slot_mapping[i] of
        kv_cache ([num_blocks, block_size, 656 or 576] uint8): 656-byte rows get per-128 scales (Row656), 576-byte
        rows clamp(x / k_scale) (Row576). Offload mode writes the layer's host pool (and cached copies) instead
        (reference dsa_sm89.py:281-290, LayerOffload.store)."""
        slots = slot_mapping if slot_mapping.dtype == torch.int64 else slot_mapping.to(torch.int64)
        if self._offload:
            self._off_state(kv_cache).store(kv_c_normed, k_pe, slots, 1.0)
            if not self._verify:
                return
        c = kv_cache.view(torch.uint8) if kv_cache.dtype != torch.uint8 else kv_cache
        fmt = 0 if c.shape[-1] == kernels.ROW656 else 1
        ks = float(k_scale.item() if torch.is_tensor(k_scale) else (k_scale if k_scale is not None else 1.0))
        kernels.cache_write(kv_c_normed, k_pe, slots, c, fmt=fmt, kv_scale=ks)

    # ---- attention
    def forward_mqa(self, q, kv_c_and_k_pe_cache, attn_metadata, layer=None):
        """q [T, H, 576] bf16 (or the pair (q_nope [T, H, 512], q_pe [T, H, 64])) -> (out [T, H, 512] bf16, None).
        Row576 caches are attended with the layer's per-tensor scale (layer._k_scale_float, 1.0 without a layer)."""
        if isinstance(q, tuple):
            q = torch.cat(q, dim=-1)
        if not kernels.query_ok(q):
            q = q.contiguous()
        kv_scale = float(getattr(layer, "_k_scale_float", 1.0)) if layer is not None else 1.0
        if self._offload and not self._verify:
            return self._forward_offload(q, kv_c_and_k_pe_cache, attn_metadata), None
        if self._offload:                          # dsa_sm89.py:396-424: offload output checked, paged one returned
            o_off = self._forward_offload(q, kv_c_and_k_pe_cache, attn_metadata)
            o_ref = self._forward_paged(q, kv_c_and_k_pe_cache, attn_metadata, kv_scale)
            verify_outputs(o_off, o_ref, self.verify_stats, label=str(getattr(self._indexer_mod, "prefix", "")))
            return o_ref, None
        return self._forward_paged(q, kv_c_and_k_pe_cache, attn_metadata, kv_scale), None

    def forward_dense(self, q, kv_c_and_k_pe_cache, attn_metadata, layer=None):
        """forward_mqa without a selection (layers without an indexer, or contexts of at most topk rows): every token of
        q [T, H, 576] bf16 (or the pair (q_nope, q_pe)) attends all cached rows of its request up to its own -> (out [T, H,
        512] bf16, lse [T, H] fp32). attn_metadata: CommonAttentionMetadata (with seq_lens, none of them beyond
        max_seq_len). Tokens of no request (a padded batch) get no output. The rows are in the paged cache: not for an
        offloaded layer."""
        if self._offload:
            raise NotImplementedError("forward_dense: the rows of an offloaded layer are not in the paged cache")
        if isinstance(q, tuple):
            q = torch.cat(q, dim=-1)
        if not kernels.query_ok(q):
            q = q.contiguous()
        md = attn_metadata
        if md.seq_lens is None:
            raise ValueError("forward_dense: attn_metadata.seq_lens")
        c = kv_c_and_k_pe_cache
        c = c.view(torch.uint8) if c.dtype != torch.uint8 else c
        kv_scale = float(getattr(layer, "_k_scale_float", 1.0)) if layer is not None else 1.0
        return kernels.attend_chunk(q, c, md.block_table_tensor, md.seq_lens, md.query_start_loc, self.softmax_scale, kv_scale,
                                    max_seq_len=md.max_seq_len)

    def forward_mha(self, q, k, v, attn_metadata):
        """Prompts of which nothing is cached yet, on expanded heads: q, k [T, H, 192], v [T, H, 128] (any widths that
        kernels.attend_prompt takes) -> (out [T, H, 128], lse [T, H] fp32), causal within each request of
        attn_metadata.query_start_loc."""
        return kernels.attend_prompt(q, k, v, attn_metadata.query_start_loc, self.softmax_scale)

    def _run(self, q, kvc, gidx, kv_scale=1.0):
        """Attention of q over cache rows gidx [n, K] (-1 or out of range: none) of a paged or flat cache."""
        c, num_rows, _, rb = self._rows_view(kvc)
        if gidx.dtype != torch.int32:
            gidx = gidx.to(torch.int32)
        if rb == kernels.ROW656:
            if not torch.cuda.is_current_stream_capturing():    # the split merge's workspace, found by later captures
                kernels.reserve_workspace(q.device, q.shape[1], K=gidx.shape[1])
            out, _ = kernels.attend(q, c, gidx, self.softmax_scale, kv_scale, R=num_rows)
        elif rb == kernels.ROW576:
            # per-tensor fp8 rows attended in place (spmla_attn576): every code times the tensor's scale
            out, _ = kernels.attend(q, c, gidx, self.softmax_scale, kv_scale, R=num_rows, row_bytes=kernels.ROW576)
        else:
            raise NotImplementedError(f"attention reads Row656 or Row576 rows, not {rb}-byte rows")
        return out if out.shape[1] <= self.num_heads else out[:, :self.num_heads]

    def _forward_paged(self, q, kv_c_and_k_pe_cache, md, kv_scale=1.0):
        n = q.shape[0]
        topk = self.topk_indices_buffer if self.topk_indices_buffer.shape[0] == n else self.topk_indices_buffer[:n]
        c, num_rows, stride_rows, rb = self._rows_view(kv_c_and_k_pe_cache)
        if rb in (kernels.ROW656, kernels.ROW576):     # rows formed in the attention kernel
            if rb == kernels.ROW656 and not torch.cuda.is_current_stream_capturing():
                kernels.reserve_workspace(q.device, q.shape[1], K=topk.shape[1])
            req = md.req_id_per_token if md.req_id_per_token.shape[0] == n else md.req_id_per_token[:n]
            out = kernels.attend_paged(q, c, topk, req, md.block_table, md.block_size,
                                       stride_rows if stride_rows is not None else md.block_size, self.softmax_scale,
                                       kv_scale, R=num_rows, row_bytes=rb)
            if out is not None:
                return out if out.shape[1] <= self.num_heads else out[:, :self.num_heads]
        gidx = convert_req_index_to_global_index(md.req_id_per_token[:n], md.block_table, topk,
                                                 BLOCK_SIZE=md.block_size, BLOCK_STRIDE_ROWS=stride_rows,
                                                 NUM_TOPK_TOKENS=topk.shape[1])
        return self._run(q, c, gidx, kv_scale)

    def _decode_rows(self, im, topk, nd, device):
        """(host rows [nd, K] of the decode tokens' selections, query tokens per request). The indexer's decode block
        table holds a row per request, or -- for a speculative-decode batch that the indexer flattened -- a row per
        token (dsa_sm89.py:299-316); consecutive tokens of a request are packed for the attention either way."""
        dec = im.decode
        if dec.requires_padding:
            raise NotImplementedError("offload decode: speculative batches with padded (unequal) query lengths are "
                                      "not supported")
        per_req = max(1, nd // max(1, im.num_decodes))
        tok = torch.arange(nd, device=device, dtype=torch.int32)
        owner = tok if dec.block_table.shape[0] >= nd else torch.div(tok, per_req, rounding_mode="floor")
        rows = convert_req_index_to_global_index(owner, dec.block_table, topk[:nd], BLOCK_SIZE=self._block_size,
                                                 NUM_TOPK_TOKENS=topk.shape[1])
        return rows, per_req

    def _prefill_rows(self, ch, device):
        """Host rows of a prefill chunk's context [total_seq_lens] int64: context position i belongs to request
        token_to_seq[i] at request-local position i - cu_seq_lens[request]; the paged rows kernel maps it through the
        chunk's block table (one position per context row)."""
        tot = ch.total_seq_lens
        owner = ch.token_to_seq[:tot].to(torch.int32).contiguous()
        first = ch.cu_seq_lens.to(torch.int64).index_select(0, owner.long())
        local = (torch.arange(tot, device=device, dtype=torch.int64) - first).to(torch.int32).view(tot, 1)
        table = ch.block_table.to(torch.int32).contiguous()
        rows = kernels.rows_from_topk(local.contiguous(), owner, table, self._block_size, stride_rows=self._block_size)
        return rows.view(-1).to(torch.int64)

    def _forward_offload(self, q, kv_cache, md):
        """Decode tokens: top-k positions -> host rows -> LayerOffload.attend; prefill chunks: the chunk's context
        rows (or only the selected ones, compact_stage) gathered into HBM and attended there
        (reference _forward_offload, dsa_sm89.py:292-378)."""
        im = getattr(md, "indexer", md)
        n = q.shape[0]
        st = self._off_state(kv_cache)
        topk = self.topk_indices_buffer[:n]
        out = torch.empty((n, self.num_heads, kernels.D_LAT), dtype=q.dtype, device=q.device)
        nd = im.num_decode_tokens
        if nd:
            rows, per_req = self._decode_rows(im, topk, nd, q.device)
            o = st.attend(q[:nd], rows, self.softmax_scale, 1.0, self.num_heads, ql=per_req, out=out[:nd])
            if o.data_ptr() != out.data_ptr():      # the layer wrote a buffer of its own (q with extra heads)
                out[:nd].copy_(o[:, :self.num_heads])
        for ch in (im.prefill.chunks if im.num_prefill_tokens else ()):
            rows = self._prefill_rows(ch, q.device)
            chosen = topk[ch.token_start:ch.token_end]
            base = ch.cu_seqlen_ks[: chosen.shape[0]].to(chosen.dtype).unsqueeze(1)
            sidx = (chosen + base).masked_fill_(chosen < 0, -1)      # positions in the chunk's context
            if rows.shape[0] > chosen.numel():   # fewer selections than context rows: stage only the selected rows
                rows, sidx = compact_stage(rows, sidx)
                if rows.shape[0] == 0:
                    rows = torch.full((1,), -1, dtype=torch.int64, device=q.device)
            staged = torch.empty((rows.shape[0], kernels.ROW656), dtype=torch.uint8, device=q.device)
            st.gather(rows, staged)
            o, _ = kernels.attend(q[ch.token_start:ch.token_end], staged, sidx.to(torch.int32).contiguous(),
                                  self.softmax_scale, 1.0)
            out[ch.token_start:ch.token_end] = o[:, :self.num_heads]
        return out


class PortableSparseBackend:
    """Backend descriptor (reference PortableSparseBackend, dsa_sm89.py:501-530)."""

    @classmethod
    def supported_kv_cache_layouts(cls):
        return ["NHD"]

    @staticmethod
    def get_name():
        return "DOTS3_PORTABLE_MLA_SPARSE"

    @staticmethod
    def get_impl_cls():
        return PortableSparseImpl

    @staticmethod
    def get_builder_cls():
        return PortableXPUBuilder

    @staticmethod
    def get_metadata_cls():
        return SparseMetadata

    @classmethod
    def get_supported_head_sizes(cls):
        return []
