"""A paged key-value cache for several decoder layers: the holder of the tensors that ``ops.paged_plan`` / ``paged_kv_write`` / ``paged_attention`` work on.

    cache = PagedKVCache(layers=12, rows=64, heads=12, head_dim=64, max_tokens=514, dtype=torch.bfloat16, device="cuda")
    slots, positions, cu, granted = cache.plan(new_tokens, max_tokens)      # once per step: pages, slots, positions (device only)
    for layer in range(12):
        cache.write(layer, k, v, slots)                                     # [T, heads, head_dim] of the new tokens
        out = cache.attend(layer, q)                                        # [rows, query heads, head_dim], one new token per row

``new_tokens`` int32 [rows]: tokens to append to each row, 0 for none, -1 to release the row.  The pool is shared by the rows: with ``pages`` fewer than
rows x ceil(max_tokens / page_size) a row whose tokens find no page is refused (``granted`` 0) and keeps its state.  The tensors keep their
addresses, so steps can be captured into HIP graphs."""
import torch

from . import ops


class PagedKVCache:
    def __init__(self, layers, rows, heads, head_dim, max_tokens, *, pages=None, page_size=16, dtype=torch.bfloat16, device="cuda"):
        if layers < 1 or rows < 1 or max_tokens < 1:
            raise ValueError(f"PagedKVCache: at least one layer, row and token, got {layers}, {rows}, {max_tokens}")
        if page_size < 16 or page_size & (page_size - 1):
            raise ValueError(f"PagedKVCache: page_size must be a power of two from 16 on, got {page_size}")
        self.columns = -(-int(max_tokens) // page_size)
        pages = rows * self.columns if pages is None else int(pages)
        if pages < 1:
            raise ValueError(f"PagedKVCache: at least one page, got {pages}")
        self.page_size = page_size
        # one allocation for all layers; what a page holds before its first write is never read into a result
        self.pages = torch.empty(layers, 2, pages, heads, page_size, head_dim, dtype=dtype, device=device)
        self.block_table = torch.full((rows, self.columns), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(rows, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(pages, dtype=torch.int32, device=device)
        self.free_ring = torch.tensor([0, pages], dtype=torch.int32, device=device)

    def reset(self):
        """every row empty, every page free"""
        self.block_table.fill_(-1)
        self.lengths.zero_()
        self.free_pages.copy_(torch.arange(self.free_pages.shape[0], dtype=torch.int32, device=self.free_pages.device))
        self.free_ring[0] = 0
        self.free_ring[1] = self.free_pages.shape[0]

    def plan(self, new_tokens, max_tokens):
        return ops.paged_plan(self.lengths, new_tokens, self.block_table, self.free_pages, self.free_ring, self.page_size, max_tokens)

    def write(self, layer, k, v, slots):
        pages = self.pages[layer]
        ops.paged_kv_write(k, v, pages[0], pages[1], slots)

    def attend(self, layer, q, scale=None):
        pages = self.pages[layer]
        return ops.paged_attention(q, pages[0], pages[1], self.block_table, self.lengths, scale)
