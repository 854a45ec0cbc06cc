"""Pages of the paged cache and the tables of a serving step, kept and built on the GPU (kernels.page_step / page_trim): which
request holds which pages, and for each token of a step its request, position and cache slot. What a scheduler forms on the
host and copies over (the fields of dsa.CommonAttentionMetadata), without the copy: a decode loop, with drafts that are
rejected and requests that end, can be captured whole.
"""
import torch

from . import kernels
from .dsa import CommonAttentionMetadata


class PagePool:
    """`pages` pages of block_size cache rows for up to `requests` requests of up to `columns` pages each.

    table [requests, columns] int32: the pages of each request (-1: none); lens [requests]: its tokens; held [requests]: its
    pages; free [pages]: the stack of pages that nobody holds; state [4]: their number, the pages that the last step
    lacked, two of the kernels' own. Calls on a pool run in order: on one stream, or with events between."""

    def __init__(self, pages, block_size, requests, columns, device="cuda"):
        z = dict(dtype=torch.int32, device=device)
        self._set(torch.full((requests, columns), -1, **z), torch.zeros(requests, **z), torch.zeros(requests, **z),
                  torch.arange(pages - 1, -1, -1, **z), torch.tensor([pages, 0, 0, 0], **z), block_size)

    def _set(self, table, lens, held, free, state, block_size):
        self.table, self.lens, self.held, self.free, self.state = table, lens, held, free, state
        self.block_size = int(block_size)

    @classmethod
    def over(cls, table, lens, held, free, state, block_size):
        """A pool over tensors that exist."""
        p = cls.__new__(cls)
        p._set(table, lens, held, free, state, block_size)
        return p

    def step(self, new, num_tokens, max_query_len, max_seq_len, n=None):
        """Enter new [requests] int32 tokens of each request (num_tokens in all; n places, default num_tokens) -> (the step's
        CommonAttentionMetadata, req [n] int32, positions [n] int64). The block table and the lengths are the pool's own
        tensors: they change with the next step."""
        start, req, positions, slots = kernels.page_step(self, new, num_tokens if n is None else n)
        md = CommonAttentionMetadata(query_start_loc=start, num_reqs=self.table.shape[0], num_actual_tokens=num_tokens,
                                     max_query_len=max_query_len, max_seq_len=max_seq_len, slot_mapping=slots,
                                     block_table_tensor=self.table, seq_lens=self.lens)
        return md, req, positions

    def trim(self, keep):
        """kernels.page_trim: rejected drafts (keep: the accepted lengths), finished requests (keep 0)."""
        kernels.page_trim(self, keep)
