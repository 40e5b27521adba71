"""Key / value cache in pages: what ``MHACache`` is to one batch of equal length, this is to sequences of any lengths that come,
branch and end (beam search, serving).  Which row holds which page lives on the device (``ops/paged.py``), so a step of decoding
needs nothing from the host."""
from __future__ import annotations

from typing import List, Optional, Sequence

import torch

from .. import ops as F


class PagedLayer:
    """One layer's pages, in place of an ``MHACache``: the attention module hands it its projection output."""

    def __init__(self, cache: "PagedCache", index: int):
        self.cache = cache
        self.k_pages, self.v_pages = cache.pool[index, 0], cache.pool[index, 1]

    @property
    def seq_len(self) -> int:
        """Tokens of the longest row (of no row there are more)."""
        return self.cache.longest

    def attend(self, qkv: torch.Tensor, batch: int, n: int, heads: int, rope=None) -> torch.Tensor:
        """Appends the keys and values of ``qkv [batch * n, (heads + 2 kv_heads) hd]``, the tokens that the cache was last
        extended by, and attends: a token of every row over the row's pages, or the tokens of prompts over one another (causal).
        Returns ``[batch * n, heads * hd]``.  Angles are of 64 bits here and of 32 in ``ops.rope``, which turns a contiguous cache's
        tokens: at position 100000 the two are up to 0.005 radians apart."""
        c = self.cache
        if c.positions is None:
            raise ValueError("PagedCache: nothing to attend with: prompts and fork extend the cache")
        if c.rows is None and (n != 1 or batch != c.table.shape[0]) or c.rows is not None and batch * n != c.positions.numel():
            raise ValueError(f"PagedCache: {batch} x {n} tokens, the cache was extended by {c.positions.numel()}")
        kw = dict(rows=c.rows, rotary_dim=0 if rope is None else rope.rotary_dim, rope_base=1.0 if rope is None else rope.base)
        if c.rows is None:
            q = F.paged_append(qkv, self.k_pages, self.v_pages, c.table, c.positions, heads, **kw)
            return F.paged_attention(q, self.k_pages, self.v_pages, c.table, c.lens).view(batch, -1)
        hkv, hd = self.k_pages.shape[1], self.k_pages.shape[3]
        q, k = F.paged_append(qkv, self.k_pages, self.v_pages, c.table, c.positions, heads, keys=True, **kw)
        v = qkv[:, (heads + hkv) * hd:]
        if qkv.is_cuda:
            from ..ops import flash
            return flash.attention_tokens(q.view(batch * n, -1), k.view(batch * n, -1), v, batch, n, n, heads, hkv, hd, True)
        q, k, v = (t.reshape(batch, n, -1, hd).transpose(1, 2) for t in (q, k, v))
        return F.attention(q, k, v, causal=True).transpose(1, 2).reshape(batch * n, heads * hd)


class PagedCache:
    """Pages of ``num_layers`` layers for up to ``rows`` sequences of up to ``max_len`` tokens.  ``layers[i]`` goes where a layer's
    ``MHACache`` goes.

    ``prompts`` starts rows, ``fork`` makes rows copies of others and gives each room for a token, ``free`` ends them,
    ``compact`` packs the pages that are left.  A model's step follows each of the first two.  ``num_pages`` is every row's own share
    unless given; a pool that runs out raises at the next ``_native.raise_on_device_error``."""

    def __init__(self, num_layers: int, num_kv_heads: int, head_dim: int, rows: int, max_len: int, page_size: int = 16,
                 num_pages: Optional[int] = None, dtype=torch.float32, device=None):
        if min(num_layers, num_kv_heads, head_dim, rows, max_len, page_size) <= 0:
            raise ValueError("PagedCache: sizes must be positive")
        width = -(-max_len // page_size)
        self.max_len, self.page_size = max_len, page_size
        self.num_pages = rows * width if num_pages is None else num_pages
        # (a page of a head is one piece of memory: 16 tokens of 128 bf16 features are 4 KB)
        self.pool = torch.zeros(num_layers, 2, self.num_pages, num_kv_heads, page_size, head_dim, dtype=dtype, device=device)
        self.table = torch.full((rows, width), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(rows, dtype=torch.int32, device=device)
        self.longest = 0                                   # no row is longer (one that has ended may have been as long)
        self.positions: Optional[torch.Tensor] = None      # of the tokens that the cache was last extended by
        self.rows: Optional[torch.Tensor] = None           # and their rows; None: one token of every row
        self.layers: List[PagedLayer] = [PagedLayer(self, i) for i in range(num_layers)]

    def longer_by(self, grow: int, parents=None) -> int:
        """``longest`` of the rows after ``fork(parents)`` by ``grow`` tokens.  Rows that have ended, or that no row goes on from, may have
        been the longest: where the bound kept here does not fit, the lengths themselves are looked at."""
        longest = self.longest + grow
        if longest > self.max_len:
            lens = self.lens
            if parents is not None:
                lens = torch.where(parents >= 0, lens[parents.long().clamp(0, lens.shape[0] - 1)], 0)
            longest = int(lens.max())
            longest += grow if longest > 0 else 0
        if longest > self.max_len:
            raise ValueError(f"PagedCache: a row of {longest} tokens in a cache of {self.max_len}")
        return longest

    def check_window(self, what: str, max_ctx: int) -> None:
        """Raises if a row is longer than ``max_ctx``."""
        if self.longest > max_ctx:
            self.longest = int(self.lens.max())
        if self.longest > max_ctx:
            raise ValueError(f"{what}: sequence of {self.longest} tokens exceeds maxCtx {max_ctx}")

    def _fork(self, parents, grow, longest: int) -> None:
        self.table, self.lens, src, dst = F.fork_pages(self.table, self.lens, self.num_pages, self.page_size, parents, grow)
        F.copy_pages(self.pool, src, dst)
        self.longest = longest

    def prompts(self, lengths: Sequence[int], rows: Sequence[int]) -> None:
        """Room for prompts of ``lengths`` tokens in ``rows``, which hold nothing; the model's step takes them as one batch,
        padded behind to the longest."""
        count, n = self.table.shape[0], max(lengths, default=0)
        if len(lengths) != len(rows) or len(set(rows)) != len(rows) or not all(0 <= r < count for r in rows):
            raise ValueError(f"PagedCache: {len(lengths)} prompts for rows {list(rows)} of {count}")
        if min(lengths, default=0) <= 0:
            raise ValueError("PagedCache: prompts must not be empty")
        dev, grow = self.table.device, [0] * count
        parents = list(range(count))
        for r, m in zip(rows, lengths):
            parents[r], grow[r] = -1, m
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        if n > self.max_len:
            raise ValueError(f"PagedCache: a prompt of {n} tokens in a cache of {self.max_len}")
        self._fork(ints(parents), ints(grow), max(min(self.longest, self.max_len), n))
        self.rows = ints([r for r in rows for _ in range(n)])
        self.positions = ints([t if t < m else -1 for m in lengths for t in range(n)])

    def fork(self, parents: Optional[torch.Tensor] = None) -> None:
        """Every row becomes a copy of row ``parents[r]`` (int32; itself without ``parents``; -1: empty) with room for a token,
        which the model's step brings; rows that hold nothing stay empty."""
        self._fork(parents, 1, self.longer_by(1, parents))
        self.rows, self.positions = None, self.lens - 1

    def free(self, rows: Sequence[int]) -> None:
        """Ends ``rows``; pages that nobody else lists are free again."""
        count, ended = self.table.shape[0], set(rows)
        if not all(0 <= r < count for r in ended):
            raise ValueError(f"PagedCache: rows {list(rows)} of {count} to end")
        keep = [-1 if r in ended else r for r in range(count)]
        self._fork(torch.tensor(keep, dtype=torch.int32, device=self.table.device), 0, self.longest)
        self.rows = self.positions = None

    def compact(self) -> torch.Tensor:
        """Moves the pages that are listed to the front of the pool; returns their number, int32 ``[1]`` on the device."""
        self.table, src, dst, live = F.compact_pages(self.table, self.num_pages)
        F.copy_pages(self.pool, src, dst)
        return live


