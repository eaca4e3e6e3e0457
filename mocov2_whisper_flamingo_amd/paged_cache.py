"""A key / value cache in pages, for requests of different lengths that come and go: what ``WhisperDecoder.new_cache`` holds for
sequences of one length (HF ``DynamicCache``, modeling_whisper.py:649-797), shared out to a server's requests.

All state lives on the GPU and moves on by one ``plan`` per step; nothing here waits for the GPU except :meth:`PagedKVCache.check`,
so a step can be recorded in a HIP graph (``new`` is read when it is replayed)."""
import torch

from . import _lib, ops

STATUS = ((1, "the pool has too few free pages"), (2, "a request outgrows its row of the block table"),
          (4, "more new tokens than max_tokens"), (8, "a negative length, or an inconsistent pool"))


class PagedKVCache:
    """``layers`` caches of ``heads`` heads over one pool of ``pages`` pages of ``page_size`` tokens, for up to ``requests`` requests of
    at most ``max_tokens`` tokens each (rounded up to whole pages).  A request is a row index; it holds pages for the tokens it has."""

    def __init__(self, layers, requests, heads, head_dim=64, *, pages, max_tokens, page_size=64, dtype=torch.bfloat16, device="cuda"):
        if page_size not in ops.PAGE_SIZES or min(layers, requests, heads, pages, max_tokens) < 1:
            raise ValueError(f"a paged cache needs positive sizes and a page size of {ops.PAGE_SIZES}")
        self.page_size, self.requests, self.dtype = page_size, requests, dtype
        self.kv = [torch.empty((pages, 2, heads, page_size, head_dim), dtype=dtype, device=device) for _ in range(layers)]
        self.table = torch.zeros((requests, -(-max_tokens // page_size)), dtype=torch.int32, device=device)
        self.lens = torch.zeros(requests, dtype=torch.int32, device=device)
        self.ring = torch.arange(pages, dtype=torch.int32, device=device)
        self.pool = torch.tensor([0, pages], dtype=torch.int32, device=device)

    def plan(self, new, max_tokens):
        """One step: ``new`` int32 [requests] on the GPU (tokens to add, 0, or negative: the request ends) -> ``ops.PagedPlan`` for the
        step's ``max_tokens`` rows.  A step that does not fit changes nothing (see :meth:`check`)."""
        return ops.paged_plan(self.lens, new, self.table, self.ring, self.pool, self.page_size, max_tokens)

    def write(self, layer, k, v, plan):
        """The step's keys and values [rows, heads, head_dim] of one layer into their slots."""
        kv, slots = self.kv[layer], plan.slots
        ops.paged_write(k, v, kv[:, 0], kv[:, 1], slots if slots.shape[0] == k.shape[0] else slots[:k.shape[0]])

    def attend(self, layer, q, q_start, *, max_q=None, scale=1.0, causal=True):
        """Attention of q [rows, query heads, head_dim], the requests' rows as ``q_start`` (of a plan) says, over the cache."""
        kv = self.kv[layer]
        return ops.paged_attn(q, kv[:, 0], kv[:, 1], self.table, self.lens, q_start, max_q=max_q, scale=scale, causal=causal)

    @staticmethod
    def check(plan):
        """Waits for the plan and raises if the step did not fit."""
        status = int(plan.status.item())
        if status:
            raise _lib.AvsrHipError("paged cache: " + "; ".join(text for bit, text in STATUS if status & bit))
