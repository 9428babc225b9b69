"""A paged key/value cache for decode loops over the streaming softmax kernels.

``PagedCache`` owns the page pools of every layer, which pages belong to which request, and the lengths; its steps
call ``ops.paged_append``, ``ops.om_paged_fwd`` and ``ops.paged_evict``.  All bookkeeping is host arithmetic on
numbers the host knows, so no step reads anything back from the device:

    cache = PagedCache(n_layers, n_pages, 16, n_kv_heads, head_dim, track_weights=True)
    r = cache.open()
    batch = cache.begin({r: prompt_len})          # pages taken, tables on their way to the device
    for layer in ...:
        q = cache.append(layer, batch, q, k, v, cos=cos, sin=sin)
        o = cache.attend(layer, batch, q)
    cache.evict([r], budget=4096, keep_first=4, keep_last=256)
    cache.close(r)

One cache serves one stream: a page that a request gives back may be written for another one by the next step, which is
ordered after the reads of the last only on the same stream.
"""
from __future__ import annotations

from dataclasses import dataclass, field

import torch

from . import ops
from ._lib import B200Error


@dataclass(frozen=True)
class PagedBatch:
    """The index tensors of one step: ``table [R, pages]``, ``seq_lens [R]`` (new tokens included), ``cu_q [R+1]``,
    ``positions [n_tokens]``, all int32, and the bounds that the kernels take from the host.  Good until one of its
    requests is closed or cut."""
    requests: tuple[int, ...]
    table: torch.Tensor
    seq_lens: torch.Tensor
    cu_q: torch.Tensor
    positions: torch.Tensor
    n_tokens: int
    max_q: int
    max_k: int
    #: the cache that made it (``None``: nobody checks), and how often each request had been given other pages by then
    owner: object = field(default=None, repr=False)
    hands: tuple[int, ...] = ()


class PagedCache:
    def __init__(self, n_layers: int, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cuda", track_weights: bool = False):
        if min(n_layers, n_pages, n_kv_heads) < 1:
            raise B200Error("PagedCache: at least one layer, page and kv head")
        if page_size < 8 or page_size > 1024 or page_size & (page_size - 1):
            raise B200Error(f"PagedCache: page_size {page_size} is not a power of two from 8 to 1024")
        if head_dim < 8 or head_dim > 128 or head_dim % 8:
            raise B200Error(f"PagedCache: head_dim {head_dim} is not a multiple of 8 up to 128")
        if dtype not in (torch.bfloat16, torch.float32):
            raise B200Error(f"PagedCache: unsupported dtype {dtype}")
        self.page_size = page_size
        self.device = torch.device(device)
        shape = (n_pages, n_kv_heads, page_size, head_dim)
        self.k = [torch.zeros(shape, dtype=dtype, device=self.device) for _ in range(n_layers)]
        self.v = [torch.zeros(shape, dtype=dtype, device=self.device) for _ in range(n_layers)]
        #: attention weight that each cached key has received, per layer (``None`` without ``track_weights``)
        self.weights = [torch.zeros(shape[:3], device=self.device) for _ in range(n_layers)] if track_weights else None
        self._free = list(range(n_pages - 1, -1, -1))
        self._pages: dict[int, list[int]] = {}
        self._length: dict[int, int] = {}
        self._position: dict[int, int] = {}
        self._hands: dict[int, int] = {}      # times that an eviction gave the request other pages
        self._owner = object()
        self._next = 0

    # ------------------------------------------------------------------ requests
    def open(self) -> int:
        """A new, empty request."""
        r = self._next
        self._next += 1
        self._pages[r], self._length[r], self._position[r], self._hands[r] = [], 0, 0, 0
        return r

    def close(self, request: int) -> None:
        """Give the request's pages back."""
        self._known(request)
        self._free.extend(reversed(self._pages.pop(request)))
        del self._length[request], self._position[request], self._hands[request]

    def length(self, request: int) -> int:
        """Cached keys."""
        self._known(request)
        return self._length[request]

    def position(self, request: int) -> int:
        """Tokens seen so far: the position of the next one (eviction does not change it)."""
        self._known(request)
        return self._position[request]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _known(self, request: int) -> None:
        if request not in self._length:
            raise B200Error(f"PagedCache: request {request} is not open")

    def _pages_for(self, n: int) -> int:
        return (n + self.page_size - 1) // self.page_size

    def _fresh(self, skip: int, n: int) -> list[int]:
        """The ``n`` free pages that are next once ``skip`` have been taken; they stay on the list."""
        end = len(self._free) - skip
        return self._free[end - n:end][::-1]

    def _to_device(self, *rows: list[int]) -> list[torch.Tensor]:
        """int32 tensors of these values on the device, in one copy that the host does not wait for."""
        flat = torch.tensor([x for r in rows for x in r], dtype=torch.int32)
        if self.device.type == "cuda":
            flat = flat.pin_memory().to(self.device, non_blocking=True)
        return list(torch.split(flat, [len(r) for r in rows]))

    # ------------------------------------------------------------------ a step
    def begin(self, new_tokens: dict[int, int]) -> PagedBatch:
        """Make room for ``new_tokens[request]`` tokens of each request and return the step's index tensors; rows of
        q, k and v follow the order of ``new_tokens``.  Nothing changes if the free pages do not suffice."""
        if not new_tokens:
            raise B200Error("PagedCache.begin: no requests")
        for r, n in new_tokens.items():
            self._known(r)
            if n < 0:
                raise B200Error(f"PagedCache.begin: {n} new tokens for request {r}")
        need = {r: self._pages_for(self._length[r] + n) - len(self._pages[r]) for r, n in new_tokens.items()}
        if sum(need.values()) > len(self._free):
            raise B200Error(f"PagedCache.begin: {sum(need.values())} pages wanted, {len(self._free)} free")
        cu, positions, pages, taken = [0], [], {}, 0
        for r, n in new_tokens.items():
            pages[r] = self._pages[r] + self._fresh(taken, need[r])
            taken += need[r]
            positions.extend(range(self._position[r], self._position[r] + n))
            cu.append(cu[-1] + n)
        requests = tuple(new_tokens)
        lens = [self._length[r] + n for r, n in new_tokens.items()]
        width = max(1, max(map(len, pages.values())))
        table = [p for x in pages.values() for p in x + [-1] * (width - len(x))]
        t, s, c, p = self._to_device(table, lens, cu, positions)
        del self._free[len(self._free) - taken:]      # (nothing has changed before, should the copy raise)
        self._pages.update(pages)
        for r, n in new_tokens.items():
            self._length[r] += n
            self._position[r] += n
        return PagedBatch(requests, t.view(len(requests), width), s, c, p, cu[-1], max(new_tokens.values()), max(1, max(lens)),
                          self._owner, tuple(map(self._hands.get, requests)))

    def _current(self, batch: PagedBatch) -> None:
        """The pages of a batch made by ``begin`` are still its requests' own."""
        if batch.owner is None:
            return
        if batch.owner is not self._owner:
            raise B200Error("PagedCache: a batch of another cache")
        if tuple(map(self._hands.get, batch.requests)) != batch.hands:
            r = next(r for r, n in zip(batch.requests, batch.hands) if self._hands.get(r) != n)
            raise B200Error(f"PagedCache: request {r} has been closed or cut since this batch was made")

    def append(self, layer: int, batch: PagedBatch, q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, *,
               q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
               cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
               interleaved: bool = False) -> torch.Tensor | None:
        """``ops.paged_append`` of the step's tokens into a layer, rotated at their positions if ``cos`` and ``sin``
        are given; returns the normed and rotated ``q``."""
        self._current(batch)
        return ops.paged_append(q, k, v, self.k[layer], self.v[layer], batch.table, batch.seq_lens, batch.cu_q,
                                q_weight=q_weight, k_weight=k_weight, eps=eps, cos=cos, sin=sin,
                                positions=None if cos is None else batch.positions, interleaved=interleaved,
                                weights=self.weights[layer] if self.weights else None)

    def attend(self, layer: int, batch: PagedBatch, q: torch.Tensor, *, scale: float | None = None,
               causal: bool = True) -> torch.Tensor:
        """``ops.om_paged_fwd`` of the step's queries over a layer; the attention weight is added up if the cache
        tracks it."""
        self._current(batch)
        return ops.om_paged_fwd(q, self.k[layer], self.v[layer], batch.table, batch.seq_lens, batch.cu_q, batch.max_q,
                                max_k=batch.max_k, scale=scale, causal=causal,
                                weights=self.weights[layer] if self.weights else None)

    def evict(self, requests: list[int], budget: int, *, keep_first: int = 0, keep_last: int = 0) -> list[torch.Tensor]:
        """Cut the given requests to ``budget`` keys in every layer (``ops.paged_evict``; those that are not longer
        stay as they are).  The kept keys move to fresh pages, as many as the budget fills, and the old pages are free
        afterwards: the free pages have to serve one request, those that it leaves serve the next.  Returns the kept slots
        per layer, ``[cut requests, Hkv, budget]``, in the order of ``requests``."""
        if self.weights is None:
            raise B200Error("PagedCache.evict: the cache does not track attention weights")
        if budget < 1 or keep_first < 0 or keep_last < 0 or keep_first + keep_last > budget:
            raise B200Error(f"PagedCache.evict: budget {budget} with {keep_first} first and {keep_last} last keys")
        if len(set(requests)) != len(requests):
            raise B200Error("PagedCache.evict: a request is named twice")
        cut = [r for r in requests if self.length(r) > budget]
        each = self._pages_for(budget)
        if cut and each > len(self._free):
            raise B200Error(f"PagedCache.evict: {each} pages wanted for a request, {len(self._free)} free")
        groups = []
        while cut:          # as many at a time as the free pages serve: each gives back no fewer than it takes
            n = len(self._free) // each
            groups.append(self._cut(cut[:n], budget, keep_first, keep_last))
            cut = cut[n:]
        return groups[0] if len(groups) == 1 else [torch.cat(x) for x in zip(*groups)]

    def _cut(self, cut: list[int], budget: int, keep_first: int, keep_last: int) -> list[torch.Tensor]:
        each = self._pages_for(budget)
        fresh = [self._fresh(i * each, each) for i in range(len(cut))]
        width = max(len(self._pages[r]) for r in cut)
        table, lens, to = self._to_device([p for r in cut for p in self._pages[r] + [-1] * (width - len(self._pages[r]))],
                                          [self._length[r] for r in cut], [p for f in fresh for p in f])
        max_k = max(self._length[r] for r in cut)
        kept = [ops.paged_evict(self.k[i], self.v[i], self.weights[i], table.view(len(cut), width), lens,
                                to.view(len(cut), each), budget, keep_first=keep_first, keep_last=keep_last, max_k=max_k)[0]
                for i in range(len(self.k))]
        del self._free[len(self._free) - each * len(cut):]      # (nothing has changed before, should a call raise)
        for r, pages in zip(cut, fresh):
            self._free.extend(reversed(self._pages[r]))
            self._pages[r], self._length[r] = pages, budget
            self._hands[r] += 1
        return kept
