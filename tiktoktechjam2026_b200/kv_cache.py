"""Paged K/V cache: the tensors of the paged-cache operators (``ops.cache_*``, ``ops.paged_attention``) kept together.

``B200Transformer.extend`` runs a model over it token by token or in chunks.
The reference has no cache: each of its calls recomputes the whole sequence
(mixed_precision/transformer.py:480-699).
"""

from __future__ import annotations

from typing import Optional

import torch

from . import ops


class PagedKVCache:
    """K and V of up to ``slots`` sequences of at most ``max_len`` tokens, in pages of ``page`` tokens.

    Attributes (all on ``device``): ``k``, ``v`` [layers, pages, kv_heads, page, stored head_dim],
    ``tables`` [slots, ceil(max_len / page)] (-1: no page), ``lens`` [slots], ``refs`` [pages] (table
    entries that name a page; 0: free) and ``status`` [1], the result of the last ``reserve`` or
    ``fork``.  Bookkeeping stays on the device: no method but ``check`` waits for it.
    """

    def __init__(self, layers: int, pages: int, kv_heads: int, head_dim: int, *, slots: int, max_len: int, page: int = 64,
                 dtype: torch.dtype = torch.float16, device="cuda") -> None:
        if page not in ops.PAGE_SIZES:
            raise ValueError(f"page must be one of {ops.PAGE_SIZES}")
        if min(layers, pages, kv_heads, slots, max_len) <= 0:
            raise ValueError("layers, pages, kv_heads, slots and max_len must be positive")
        if head_dim not in ops.HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {ops.HEAD_DIMS}")
        if dtype not in ops.PAGED_DTYPES:
            raise ValueError("dtype must be torch.float16 or torch.bfloat16")
        dev = torch.device(device)
        if dev.type != "cuda":
            raise ValueError("the cache lives on a CUDA device")
        self.page, self.head_dim = page, head_dim
        shape = (layers, pages, kv_heads, page, ops.stored_head_dim(head_dim))
        self.k = torch.empty(shape, dtype=dtype, device=dev)
        self.v = torch.empty(shape, dtype=dtype, device=dev)
        self.tables = torch.full((slots, -(-max_len // page)), -1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(slots, dtype=torch.int32, device=dev)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=dev)
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)

    @classmethod
    def for_model(cls, model, *, slots: int, max_len: int, pages: Optional[int] = None, page: int = 64) -> "PagedKVCache":
        """A cache for ``model`` on its device; without ``pages`` every slot can reach ``max_len``."""
        cfg = model.config
        return cls(cfg.num_layers, slots * -(-max_len // page) if pages is None else pages, cfg.num_heads,
                   cfg.d_model // cfg.num_heads, slots=slots, max_len=max_len, page=page,
                   device=next(model.parameters()).device)

    @property
    def device(self) -> torch.device:
        return self.k.device

    def check(self, status: Optional[torch.Tensor] = None) -> None:
        """Waits for the ``reserve`` or ``fork`` that returned ``status`` (the last one without it) and raises if it
        was refused (it then changed nothing)."""
        status = int((self.status if status is None else status).item())
        if status > 0:
            raise RuntimeError(f"the page pool is {status} page(s) short")
        if status < 0:
            raise RuntimeError({-1: "a sequence would outgrow its table row, or lacks its last page",
                                -2: "a slot outside the table, or a cu_q that decreases",
                                -3: "a child slot that is not empty or occurs twice"}[status])

    def reserve(self, cu_q: torch.Tensor, slots: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Pages for the new tokens cu_q describes, which ``lens`` counts from then on; see ``ops.cache_reserve``.

        Returns the reservation's status, which every ``append`` of these tokens takes.
        """
        self.status = ops.cache_reserve(self.tables, self.lens, self.refs, cu_q, self.page, slots)
        return self.status

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor,
               slots: Optional[torch.Tensor] = None, *, status: torch.Tensor) -> None:
        """Writes one layer's K and V of the tokens whose ``reserve`` returned ``status`` (nothing if it was refused:
        the lengths do not count them, and the positions they would take hold other tokens)."""
        ops.cache_append(k, v, self.k[layer], self.v[layer], self.tables, self.lens, cu_q, slots, status=status)

    def attend(self, layer: int, q: torch.Tensor, cu_q: torch.Tensor, slots: Optional[torch.Tensor] = None, *,
               scale: Optional[float] = None, window: int = 0, sinks: int = 0,
               max_q_len: Optional[int] = None) -> torch.Tensor:
        """Attention of the new tokens over one layer's pages; see ``ops.paged_attention``."""
        return ops.paged_attention(q, self.k[layer], self.v[layer], self.tables, self.lens, cu_q, slots=slots, scale=scale,
                                   window=window, sinks=sinks, head_dim=self.head_dim, max_q_len=max_q_len)

    def fork(self, parents: torch.Tensor, children: torch.Tensor) -> torch.Tensor:
        """Makes each empty slot of ``children`` a copy of its parent; full pages are shared."""
        self.status = ops.cache_fork(self.k, self.v, self.tables, self.lens, self.refs, parents, children)
        return self.status

    def release(self, slots: Optional[torch.Tensor] = None) -> None:
        """Empties the slots (all without ``slots``)."""
        ops.cache_release(self.tables, self.lens, self.refs, self.page, slots)

    def trim(self, window: int, sinks: int = 0, slots: Optional[torch.Tensor] = None) -> None:
        """Frees the pages that no later query can see under the window."""
        if window <= 0:
            raise ValueError("window must be positive (release empties a slot)")
        ops.cache_release(self.tables, self.lens, self.refs, self.page, slots, window, sinks)

    def compact(self) -> torch.Tensor:
        """Moves the live pages to the front of the pool; returns their number, int32 [1]."""
        return ops.cache_compact(self.k, self.v, self.tables, self.lens, self.refs)

    def copy_pages(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Copies pages src[i] -> dst[i] of every layer (tables and counts are the caller's)."""
        ops.cache_copy_pages(self.k, self.v, self.tables, self.lens, src, dst)
