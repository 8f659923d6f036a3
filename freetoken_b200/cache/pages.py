"""Free list of fixed-size pages.

Page 0 is never handed out: block-table entries that point nowhere (beyond a request's
length, or pages a window has passed) hold 0, so a stray read lands in memory the pool
owns.  The free list is last-in first-out, so a page given back is the next one handed
out; tests with small pools rely on that to exercise reuse.  The reference keeps its free
list as a device tensor of page base slots (python/freetoken/scheduler/cache.py:38,256-275);
this one lives on the host and block-table changes travel with the step's metadata.
"""

from __future__ import annotations

from typing import Dict, Iterable, List

from ..errors import CacheError

NULL_PAGE = 0


class PagePool:
    def __init__(self, num_pages: int):
        """``num_pages`` counts the usable pages; ids run from 1 to ``num_pages``."""
        if num_pages < 1:
            raise CacheError(f"a page pool needs at least one page, got {num_pages}")
        self.num_pages = num_pages
        self._free: List[int] = list(range(num_pages, 0, -1))
        self._held = [0] * (num_pages + 1)  # holders
        self.shared = 0  # pages of several holders
        self.handed_out = 0  # pages ever handed out (reuse shows as handed_out > num_pages)

    @property
    def free_count(self) -> int:
        return len(self._free)

    def alloc(self, n: int) -> List[int]:
        if n < 0:
            raise CacheError("cannot allocate a negative number of pages")
        if n > len(self._free):
            raise CacheError(f"out of pages: {n} wanted, {len(self._free)} free of {self.num_pages}")
        out = [self._free.pop() for _ in range(n)]
        for p in out:
            self._held[p] = 1
        self.handed_out += n
        return out

    def share(self, pages: Iterable[int]) -> None:
        """One more holder for each of ``pages``, which are held already."""
        pages = list(pages)
        for p in pages:
            if not 1 <= p <= self.num_pages or not self._held[p]:
                raise CacheError(f"page {p} is held by nobody and cannot be shared")
        for p in pages:
            self.shared += self._held[p] == 1
            self._held[p] += 1

    def holders(self, page: int) -> int:
        return self._held[page]

    def free(self, pages: Iterable[int]) -> None:
        for p in pages:
            if not 1 <= p <= self.num_pages:
                raise CacheError(f"page {p} does not belong to this pool")
            if not self._held[p]:
                raise CacheError(f"page {p} freed twice")
            self._held[p] -= 1
            self.shared -= self._held[p] == 1
            if not self._held[p]:
                self._free.append(p)

    def renumber(self, moved: Dict[int, int]) -> None:
        """Held pages ``moved`` (from -> to, the targets free) change their numbers; the lowest free page is handed out next."""
        for a, b in moved.items():
            if not self._held[a] or self._held[b]:
                raise CacheError(f"page {a} cannot become page {b}")
            self._held[b], self._held[a] = self._held[a], 0
        self._free = [p for p in range(self.num_pages, 0, -1) if not self._held[p]]

    def check(self, held_by_requests: Iterable[int]) -> None:
        """Every page is either free or held as often as it has holders.  (``held_by_requests``: pages, once per holder.)"""
        held = list(held_by_requests)
        times: Dict[int, int] = {}
        for p in held:
            times[p] = times.get(p, 0) + 1
        for p, n in times.items():
            if n > max(1, self._held[p]):
                raise CacheError("a page is held twice")
        if len(set(self._free)) != len(self._free):
            raise CacheError("a page is on the free list twice")
        if set(times) & set(self._free):
            raise CacheError("a page is both held and free")
        if len(times) + len(self._free) != self.num_pages:
            raise CacheError(
                f"pages lost: {len(times)} held + {len(self._free)} free != {self.num_pages}")
        for p, n in times.items():
            if not self._held[p]:
                raise CacheError(f"page {p} is in a block table but marked free")
            if self._held[p] != n:
                raise CacheError(f"page {p} is in {n} block tables but has {self._held[p]} holders")
        if self.shared != sum(n > 1 for n in times.values()):
            raise CacheError(f"{self.shared} pages count as shared, {sum(n > 1 for n in times.values())} are")
