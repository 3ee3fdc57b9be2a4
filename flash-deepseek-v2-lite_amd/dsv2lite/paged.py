"""Paged MLA latent cache held in 4 bits: requests share one pool of pages.

Where ``CompressedKVCache`` gives every row a fixed capacity of bf16 rows (1,152 bytes per token and
layer), this cache hands pages of ``page_size`` tokens to the requests as they grow and takes them back
as they shrink or end, all on the GPU, and holds a token in 400 bytes per layer: the latent as e2m1
codes in blocks of 32 with power-of-two scales, the rotary key in bf16.  The kernels and their
functions are in ``triton_kernels.paged_cache``; this class keeps their tensors together.

A serving step, which may be captured in a graph (``delta`` and the rows then keep their tensors):

    slots, positions, rows = cache.step(delta, max_tokens)     # lengths, pages, where the tokens go
    for each layer:
        cache.write(layer, new_rows, slots)                    # [max_tokens, 576], as dsv2_mla_prepare writes them
        latent = cache.attend(layer, q, softmax_scale, cache.cu_q, max_q)  # [max_tokens, heads, 512], what W_UV takes

``new_rows`` and ``q`` are the new tokens', in the order of ``slots``: one request after the other, none of a
request whose length does not grow; ``cache.cu_q`` says which are whose.

The reference keeps one expanded bf16 tensor of fixed length instead (src/run.py:81-99)."""

from __future__ import annotations

import torch

from triton_kernels import paged_cache as ops


class PagedLatentCache:
    def __init__(self, n_layers: int, requests: int, max_len: int, n_pages: int, page_size: int = 64, device="cuda"):
        """Room for ``requests`` requests of up to ``max_len`` tokens (whole pages: the next multiple of
        ``page_size``), ``n_pages * page_size`` tokens in all."""
        if min(n_layers, requests, max_len, n_pages) <= 0:
            raise ValueError("n_layers, requests, max_len and n_pages must be positive")
        if requests > ops.MAX_REQUESTS:
            raise ValueError(f"at most {ops.MAX_REQUESTS} requests, not {requests}")
        if page_size < 1 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two up to 1024, not {page_size}")
        if n_pages * page_size >= 2 ** 31:
            raise ValueError(f"{n_pages} pages of {page_size} tokens: slots are int32")
        self.n_layers, self.requests, self.max_len = n_layers, requests, max_len
        self.n_pages, self.page_size = n_pages, page_size
        self.pages = torch.zeros(n_layers, n_pages, page_size * ops.TOKEN_BYTES, dtype=torch.uint8, device=device)
        self.block_table = torch.full((requests, -(-max_len // page_size)), -1, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(n_pages, dtype=torch.int32, device=device)
        # the lengths, then head and count of the ring of free pages
        self.state = torch.zeros(requests + 2, dtype=torch.int32, device=device)
        self.state[-1] = n_pages
        self.lens = self.state[:requests]
        # attend's cu_q for a query of each new token of the last step: request b's are cu_q[b] .. cu_q[b + 1], at
        # most max(delta) many.  One that the step refused keeps its places; what comes out there means nothing, as
        # rows[i] = -1 tells
        self.cu_q = torch.zeros(requests + 1, dtype=torch.int32, device=device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)  # what this cache's calls had to skip

    def step(self, delta: torch.Tensor, max_tokens: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Change every request's length by ``delta`` (int32 [requests]; negative: tokens dropped from its end, at
        most all, which ends it) and give the new tokens, requests in order, their (slots, positions, rows), -1
        behind the last one.  A request that does not fit keeps its length (``check_status``), and those behind it
        that need what it asked for are refused with it."""
        after, slots, positions, rows = ops.paged_cache_step(self.state, delta, self.block_table, self.free_pages,
                                                             self.page_size, max_tokens, self.status, self.cu_q)
        self.state.copy_(after)
        return slots, positions, rows

    def slots_of(self, starts: torch.Tensor, counts: torch.Tensor, max_tokens: int) -> tuple[torch.Tensor, ...]:
        """(slots, positions, rows) of the cached tokens [starts[b], starts[b] + counts[b]) of every request."""
        return ops.paged_slot_map(starts, counts, self.block_table, self.page_size, max_tokens, self.status)

    def write(self, layer: int, rows: torch.Tensor, slots: torch.Tensor) -> None:
        """Round cache rows [n, 576] (normalised latent | rotated key) into a layer's slots."""
        ops.paged_cache_write_fp4(rows, slots, self.pages[layer], self.status)

    def read(self, layer: int, slots: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """The bf16 rows [n, 576] that a layer's slots hold."""
        return ops.paged_cache_read_fp4(self.pages[layer], slots, out, self.status)

    def attend(self, layer: int, q: torch.Tensor, softmax_scale: float, cu_q: torch.Tensor | None = None,
               max_q: int = 1, out: torch.Tensor | None = None) -> torch.Tensor:
        """Latent attention outputs [tokens, heads, 512] of absorbed queries [tokens, heads, 576] over a layer: the
        requests' last cached tokens, ``cu_q[b]`` .. ``cu_q[b + 1]`` of them request b's (``self.cu_q`` after a step),
        or without it row b for request b, idle requests included.  Rows past ``cu_q[-1]`` are not written."""
        return ops.attention_decode_paged_fp4(q, self.pages[layer], self.block_table, self.lens, softmax_scale, cu_q,
                                              max_q, out, self.status)

    def snapshot(self) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Lengths, block table and free pages; the tokens themselves stay where they are, so a snapshot holds until
        a page that it names is written again."""
        return self.state.clone(), self.block_table.clone(), self.free_pages.clone()

    def restore(self, snap: tuple[torch.Tensor, torch.Tensor, torch.Tensor]) -> None:
        for t, saved in zip((self.state, self.block_table, self.free_pages), snap):
            t.copy_(saved)

    def free_tokens(self) -> int:
        """Tokens that the free pages hold (synchronises)."""
        return int(self.state[-1].item()) * self.page_size

    def check_status(self) -> None:
        """Raise if a call of this cache skipped tokens since the last check (waits for the device)."""
        ops.check_paged_status(status=self.status)
