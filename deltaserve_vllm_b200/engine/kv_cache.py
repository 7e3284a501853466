"""Paged KV cache: page allocator and the per-layer cache tensors.

Each layer owns ``k`` and ``v`` tensors of shape ``[num_blocks, Hkv_local,
block_size, head_dim]`` (bf16): one (page, head) is a contiguous
``block_size x head_dim`` tile, the unit the attention kernels load. A request
holds a list of page ids; token ``t`` of the request lives in page
``block_ids[t // block_size]`` at offset ``t % block_size``.

With ``kv_group`` the cache holds 4-bit codes instead: one uint8 tensor per layer
(``ops.kv4_cache_shape``) with K and V side by side, in ``k``; ``v`` is empty.

A request can be forked (full pages shared by reference, the partly filled one
copied) and the pool compacted (live pages moved to its front); both move pages of
every layer with one kernel on the current stream, which has to be the one that the
forwards use (or ordered with it on both sides).

Pages are sized from the HBM left after weights, LoRA buffers and the
activation-capture buffers (``gpu_memory_utilization`` of the total).
"""

from __future__ import annotations

import hashlib
from collections import OrderedDict

import torch

from .. import ops


class BlockAllocator:
    """LIFO free list of page ids (recently freed pages are reused first, which
    keeps the working set of the cache warm in L2)."""

    def __init__(self, num_blocks: int):
        self.num_blocks = num_blocks
        self._free = list(range(num_blocks - 1, -1, -1))
        self._shared: dict[int, int] = {}       # page -> holders beside the first

    @property
    def num_free(self) -> int:
        return len(self._free)

    def allocate(self, n: int) -> list[int]:
        if n > len(self._free):
            raise MemoryError(f"KV cache out of pages: need {n}, have {len(self._free)}")
        out = self._free[-n:] if n else []
        del self._free[len(self._free) - n:]
        return out[::-1]

    def free(self, ids: list[int]) -> None:
        if self._shared:
            ids = [p for p in ids if not self._drop_share(p)]
        self._free.extend(reversed(ids))

    def share(self, ids: list[int]) -> None:
        """One more holder of each page: it returns to the pool with its last ``free``."""
        for p in ids:
            self._shared[p] = self._shared.get(p, 0) + 1

    def _drop_share(self, page: int) -> bool:
        n = self._shared.get(page, 0)
        if n > 1:
            self._shared[page] = n - 1
        elif n:
            del self._shared[page]
        return n > 0

    def compact(self) -> list[tuple[int, int]]:
        """Renumber the pages in use to ``[0, pages in use)``. Returns the moves
        (page, new page); no new page is a moved one, and everything that names
        a page outside the allocator has to follow them."""
        free = set(self._free)
        used = self.num_blocks - len(free)
        moves = list(zip((p for p in range(used, self.num_blocks) if p not in free),
                         (p for p in range(used) if p in free)))
        self._free = list(range(self.num_blocks - 1, used - 1, -1))
        self._renumber(dict(moves))
        return moves

    def _renumber(self, to: dict[int, int]) -> None:
        self._shared = {to.get(p, p): n for p, n in self._shared.items()}

    def usage(self) -> float:
        return 1.0 - len(self._free) / max(1, self.num_blocks)


def blocks_needed(num_tokens: int, block_size: int) -> int:
    return -(-num_tokens // block_size)


def block_hash(parent: bytes, tokens, extra: tuple = ()) -> bytes:
    """Hash of a full page given its parent page's hash, its token ids and the
    identity of whatever else shaped its KV (the LoRA slot and its version)."""
    h = hashlib.blake2b(digest_size=16)
    h.update(parent)
    h.update(repr(tuple(extra)).encode())
    h.update(b",".join(str(int(t)).encode() for t in tokens))
    return h.digest()


class PrefixCachingAllocator(BlockAllocator):
    """Page allocator with automatic prefix caching (vLLM's semantics): every
    full page of a request is registered under a chained hash of its tokens
    (and the LoRA slot version that produced its K/V); a later request whose
    prompt starts with the same pages reuses them instead of recomputing.
    Pages are reference counted; a released page that holds a registered
    prefix stays cached (evictable, least recently used first) until its id
    is needed for a new allocation."""

    def __init__(self, num_blocks: int):
        super().__init__(num_blocks)
        self.ref = [0] * num_blocks
        self.hash_of: dict[int, bytes] = {}     # page -> registered hash
        self.page_of: dict[bytes, int] = {}     # hash -> page
        self.evictable: OrderedDict[int, None] = OrderedDict()  # cached pages with ref 0, LRU first
        self.hits = 0
        self.queries = 0

    @property
    def num_free(self) -> int:
        return len(self._free) + len(self.evictable)

    def _evict(self, page: int) -> None:
        del self.evictable[page]
        h = self.hash_of.pop(page)
        if self.page_of.get(h) == page:
            del self.page_of[h]

    def allocate(self, n: int) -> list[int]:
        if n > self.num_free:
            raise MemoryError(f"KV cache out of pages: need {n}, have {self.num_free}")
        take = min(n, len(self._free))
        out = super().allocate(take)
        while len(out) < n:                      # reuse the least recently used cached pages
            page = next(iter(self.evictable))
            self._evict(page)
            out.append(page)
        for p in out:
            self.ref[p] = 1
        return out

    def free(self, ids: list[int]) -> None:
        plain = []
        for p in ids:
            self.ref[p] -= 1
            if self.ref[p] > 0:
                continue
            if p in self.hash_of:
                self.evictable[p] = None         # most recently used at the end
            else:
                plain.append(p)
        super().free(plain)

    def lookup(self, hashes: list[bytes]) -> list[int]:
        """Pages holding the longest cached run of ``hashes`` (each gets a
        reference)."""
        out = []
        self.queries += len(hashes)
        for h in hashes:
            p = self.page_of.get(h)
            if p is None:
                break
            if self.ref[p] == 0:
                del self.evictable[p]
            self.ref[p] += 1
            out.append(p)
        self.hits += len(out)
        return out

    def share(self, ids: list[int]) -> None:
        for p in ids:
            self.ref[p] += 1

    def _renumber(self, to: dict[int, int]) -> None:
        ref = [0] * self.num_blocks
        for p, n in enumerate(self.ref):
            if n:
                ref[to.get(p, p)] = n
        self.ref = ref
        self.hash_of = {to.get(p, p): h for p, h in self.hash_of.items()}
        self.page_of = {h: to.get(p, p) for h, p in self.page_of.items()}
        self.evictable = OrderedDict((to.get(p, p), None) for p in self.evictable)

    def usage(self) -> float:
        return 1.0 - self.num_free / max(1, self.num_blocks)

    def register(self, page: int, h: bytes) -> None:
        """Record that ``page`` (full) holds the prefix hashed ``h``."""
        if page in self.hash_of:
            return
        if h in self.page_of:                    # the same prefix already lives elsewhere
            return
        self.hash_of[page] = h
        self.page_of[h] = page


class KVCache:
    def __init__(self, num_layers: int, num_blocks: int, num_kv_heads_local: int, block_size: int,
                 head_dim: int, device, dtype=torch.bfloat16, prefix_caching: bool = False,
                 kv_group: int | None = None):
        self.block_size = block_size
        self.num_blocks = num_blocks
        if kv_group:
            if head_dim != 128:
                raise ValueError(f"a 4-bit KV cache needs head_dim 128, got {head_dim}")
            shape = ops.kv4_cache_shape(num_blocks, num_kv_heads_local, block_size, kv_group)
            dtype = torch.uint8
        else:
            shape = (num_blocks, num_kv_heads_local, block_size, head_dim)
        self.k = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(num_layers)]
        self.v = [] if kv_group else [torch.zeros(shape, dtype=dtype, device=device) for _ in range(num_layers)]
        self.allocator = PrefixCachingAllocator(num_blocks) if prefix_caching else BlockAllocator(num_blocks)

    @staticmethod
    def bytes_per_block(num_layers: int, num_kv_heads_local: int, block_size: int, head_dim: int,
                        elem: int = 2, kv_group: int | None = None) -> int:
        if kv_group:
            return num_layers * num_kv_heads_local * (block_size // 16) * 2 * ops.kv4_record_bytes(kv_group)
        return 2 * num_layers * num_kv_heads_local * block_size * head_dim * elem

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self.k + self.v)

    def fork(self, parents: list[tuple[list[int], int]]) -> list[list[int]]:
        """Pages of a copy of each parent, given as (its pages, its cached
        tokens): the full pages are shared by reference, the partly filled last
        ones copied (all of them in one launch). The children own their pages as
        any request does. Raises MemoryError (nothing changed) without room."""
        tails = [i for i, (_, n) in enumerate(parents) if n % self.block_size]
        new = dict(zip(tails, self.allocator.allocate(len(tails))))
        children, src = [], []
        for i, (pages, n) in enumerate(parents):
            full = n // self.block_size
            self.allocator.share(pages[:full])
            children.append(pages[:full] + ([new[i]] if i in new else []))
            if i in new:
                src.append(pages[full])
        ops.copy_pages(self.k + self.v, src, list(new.values()))
        return children

    def compact(self, tables: list[list[int]]) -> int:
        """Move the pages in use to the front of the pool, in one launch, and
        rewrite ``tables`` (every list of page ids that is held, in place).
        Returns the pages in use (cached prefixes are): the rest of the pool is free."""
        moves = self.allocator.compact()
        ops.copy_pages(self.k + self.v, [a for a, _ in moves], [b for _, b in moves])
        to = dict(moves)
        for t in tables:
            t[:] = [to.get(p, p) for p in t]
        return self.num_blocks - len(self.allocator._free)
