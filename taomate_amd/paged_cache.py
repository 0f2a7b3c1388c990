"""A KV cache in blocks for requests of different lengths (no counterpart in the reference, whose caches
hold one length a batch: ltx_causal/transformer/kv_cache.py:321-358).

The arena cache (``kv_cache``) keeps one sequence of spans for a whole batch.  ``PagedKVCache`` keeps a
table of blocks for every request, so that requests come, grow and go by themselves in one pool of
memory.  Tables, lengths and the stack of free blocks lie on the device and every step is a few
launches without a wait, so a decoding step can be captured into a graph:

    cache = PagedKVCache(layers=48, requests=64, blocks=4096, heads=8, dim_head=128, max_tokens=8192)
    plan = cache.grow(new, tokens)                          # int32 [64]: new tokens of each request
    for i, (q, k, v) in enumerate(...):                     # packed rows [tokens, heads, D] of each layer
        cache.append(i, k, v, plan)
        out = cache.attend_prompts(i, q, k, v, plan)        # or cache.attend(i, q): one token a request
    cache.release(done)                                     # bool [64]
    cache.check()                                           # raises if a call did not fit (waits)

A call of ``grow`` that does not fit gives no request anything and is noted in ``status``: its tokens
have no slots, so ``append`` writes nothing, and the lengths stay.
"""
from __future__ import annotations

from typing import Optional, Sequence, Union

import torch

from . import _native as N
from . import kernels
from .kv_cache import KVArenaFull

_ROWS = N.MAX_REQUESTS   # rows of one paged_attn call


class PagedKVCache:
    """Pools of ``blocks`` blocks of ``block_size`` tokens for each of ``layers`` layers, shared by up to ``requests``
    requests of at most ``max_tokens`` tokens.  ``heads`` counts key heads.  A head's tokens of a block lie
    together in memory; ``pool(layer)`` gives the [blocks, block_size, heads, dim_head] views."""

    def __init__(self, layers: int, requests: int, blocks: int, heads: int, dim_head: int, max_tokens: int,
                 block_size: int = 64, kv_dtype: str = "bf16", device="cuda"):
        if kv_dtype not in ("bf16", "fp8"):
            raise ValueError(f"kv_dtype must be 'bf16' or 'fp8', got {kv_dtype!r}")
        if dim_head not in (64, 128):
            raise ValueError(f"dim_head must be 64 or 128, got {dim_head}")
        if block_size not in (16, 32, 64, 128, 256):
            raise ValueError(f"block_size must be 16, 32, 64, 128 or 256, got {block_size}")
        if not 1 <= requests <= N.MAX_REQUESTS:
            raise ValueError(f"requests must lie in [1, {N.MAX_REQUESTS}], got {requests}")
        if min(layers, blocks, heads, max_tokens) < 1:
            raise ValueError("layers, blocks, heads and max_tokens must be positive")
        self.layers, self.requests, self.blocks = int(layers), int(requests), int(blocks)
        self.block_size, self.kv_dtype, self.device = int(block_size), kv_dtype, torch.device(device)
        store = torch.uint8 if kv_dtype == "fp8" else torch.bfloat16
        shape = (self.layers, 2, self.blocks, int(heads), self.block_size, int(dim_head))
        # never read before it is written: a request's keys are its first lens tokens
        self._store = torch.empty(shape, dtype=store, device=self.device)
        self._scales = torch.empty(shape[:-1], device=self.device) if kv_dtype == "fp8" else None
        i32 = dict(dtype=torch.int32, device=self.device)
        self.tables = torch.full((self.requests, -(-int(max_tokens) // self.block_size)), -1, **i32)
        self.lens = torch.zeros(self.requests, **i32)
        self.free = torch.arange(self.blocks - 1, -1, -1, **i32)
        self.top = torch.full((1,), self.blocks, **i32)
        self.status = torch.zeros(1, **i32)

    def pool(self, layer: int):
        """(k, v, k_scales, v_scales) of a layer: pools [blocks, block_size, heads, dim_head] and, for fp8, their
        float32 scales [blocks, block_size, heads] (else None)."""
        k, v = self._store[layer].permute(0, 1, 3, 2, 4)
        if self._scales is None:
            return k, v, None, None
        ks, vs = self._scales[layer].permute(0, 1, 3, 2)
        return k, v, ks, vs

    def _vector(self, values, dtype) -> torch.Tensor:
        if isinstance(values, torch.Tensor):
            return values
        return torch.tensor(list(values), dtype=dtype, device=self.device)

    def grow(self, new: Union[torch.Tensor, Sequence[int]], tokens: int) -> kernels.BlockPlan:
        """Blocks and slots for ``new`` (int32 [requests]) more tokens of each request; ``tokens`` rows in all, of
        which those behind the last token belong to nobody.  Updates ``lens`` in place."""
        return kernels.kv_block_grow(self.tables, self.lens, self._vector(new, torch.int32), self.free, self.top,
                                     self.status, self.block_size, tokens, self.lens, self.top)

    def release(self, done: Union[torch.Tensor, Sequence[bool]]) -> None:
        """The blocks of the requests with ``done`` (bool [requests]) are free again, and the requests empty."""
        kernels.kv_block_release(self.tables, self.lens, self._vector(done, torch.bool), self.free, self.top,
                                 self.status, self.block_size, self.lens, self.top)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, plan: kernels.BlockPlan) -> None:
        """K and V rows [tokens, heads, dim_head] of a plan's tokens into their slots."""
        kp, vp, ks, vs = self.pool(layer)
        kernels.kv_paged_append(k, v, kp, vp, plan.slots, ks, vs)

    def attend(self, layer: int, q: torch.Tensor, scale: Optional[float] = None) -> torch.Tensor:
        """One row a request, q [requests, query heads, dim_head], over all its tokens; empty requests: zeros."""
        kp, vp, ks, vs = self.pool(layer)
        return kernels.paged_attn(q, kp, vp, self.tables, self.lens, ks, vs, scale=scale)

    def attend_prompts(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, plan: kernels.BlockPlan,
                       continued: bool = False, scale: Optional[float] = None) -> torch.Tensor:
        """Causal attention of a plan's rows, q [tokens, query heads, dim_head].  The rows' own ``k`` and ``v`` are all
        that they see, as for requests that were empty before the plan; with ``continued`` they see everything
        that their request holds up to themselves, read from the cache after ``append`` (every row as a token of
        its own: for a few rows a request).  Rows without a slot are zero.  Without ``continued``, rows of a request
        that held tokens before do not see them and nothing says so: the lengths lie on the device."""
        if not continued:
            return kernels.prompt_attn(q, k, v, plan.starts, scale=scale)
        kp, vp, ks, vs = self.pool(layer)
        rows = torch.arange(q.shape[0], dtype=torch.int32, device=q.device)
        request = torch.searchsorted(plan.starts[1:], rows, right=True).clamp_(max=self.requests - 1)
        lens = torch.where(plan.slots >= 0, plan.positions + 1, torch.zeros_like(plan.positions))
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        for a in range(0, q.shape[0], _ROWS):
            part = slice(a, a + _ROWS)
            # table rows of thousands of entries: gathered for one part, and gone before the next one's
            kernels.paged_attn(q[part], kp, vp, self.tables[request[part]], lens[part], ks, vs, scale=scale,
                               out=out[part])
        return out

    def check(self) -> None:
        """Waits for the device and raises if a call since the last ``check`` did not fit."""
        status = int(self.status.item())
        self.status.zero_()
        if status & (N.BLOCKS_TOKENS | N.BLOCKS_LENGTH):
            raise ValueError("PagedKVCache: a plan had more tokens than rows, or a negative number of them")
        if status & N.BLOCKS_WIDTH:
            raise KVArenaFull(f"PagedKVCache: a request outgrew {self.tables.shape[1] * self.block_size} tokens")
        if status & N.BLOCKS_FREE:
            raise KVArenaFull(f"PagedKVCache: not enough of {self.blocks} blocks were free")
