"""Host-side work list of attention over shared keys (``ops.shared_attention``).

Requests that continue one prompt, or that begin with the same system prompt, share the pages of it.  A *span* says so: its
members read the same pages for the positions ``[start, end)``.  The keys of a span are worked on once, with the query rows of all
its members together: the members are put into tiles of as many query rows as the kernel takes, and the tiles are cut along the keys
until they keep every SM busy.  What a request reads outside of spans is its own, and the kernel that joins a request's partial
results takes it.  Spans may nest (a system prompt under several users' prompts, each under several answers).

Nothing here depends on the requests' lengths but the ``requests`` array and the number of CTAs that share a request's own keys
(``cluster``, which goes by the longest own part rounded up to a power of two): a decode step replayed from a CUDA graph keeps
its sizes while the requests grow.  The reference reads shared pages once per request
(python/freetoken/kernel/triton/attention.py:147-352).
"""

from __future__ import annotations

import math
from dataclasses import dataclass, field, replace
from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

from ..errors import KernelError

ITEM_INTS = 8     # first member, members, block-table row, first key, one past the last key, first slot, split, 0
REQUEST_INTS = 8  # query row, block-table row, first own key, one past the last, first join, joins, 0, 0
ROWS_TILE = 16    # query rows of a piece on the kernels for few rows
WIDE_TILE = 256   # on the tcgen05 kernel: two tiles of 128
WIDE_KEYS = 128   # keys that kernel works on at a time
MOST_CLUSTER = 8
MOST_SLOT_BYTES = 64 << 20  # of partial results, where fewer and longer pieces can do with less
OWN_CTAS_PER_SM, OWN_BEHIND_US = 4, 9.0  # of the kernel for own keys; what it takes more where it has to wait for the other to end
# what a piece costs the tcgen05 kernel: microseconds per key tile with one and with two query tiles, and per piece; and how fast
# partial results are written and read again
WIDE_ONE_US, WIDE_TWO_US, WIDE_PIECE_US, JOIN_BYTES_PER_US = 1.35, 2.1, 5.0, 2.5e6

ROWS_KEYS = {torch.bfloat16: 64, torch.float32: 32}  # keys the kernels for few rows work on at a time

Span = Tuple[Sequence[int], int, int]  # members (indices of requests), first position, one past the last


def _rounded(n: int) -> int:
    """``n`` up to a power of two or three halves of one."""
    top = 1 << (n - 1).bit_length() if n else 0
    return top // 4 * 3 if top >= 4 and n <= top // 4 * 3 else top


@dataclass
class SharedPlan:
    """int32 arrays of one step's shared and own keys, and what the launch needs beside them."""

    items: np.ndarray     # [n, 8]
    members: np.ndarray   # query rows
    requests: np.ndarray  # [n, 8]
    joins: np.ndarray     # slots of every request's partial results, in the order of its keys
    n_slots: int
    tile_rows: int
    cluster: int
    own_tiles: int        # tiles of keys that one CTA of a cluster has at most
    n_rows: int           # rows of q that the plan reads, from the first on
    n_heads: int
    n_kv_heads: int
    head_dim: int

    def key(self) -> Tuple[int, ...]:
        """What a recorded step's launches depend on."""
        return (self.items.shape[0], self.members.shape[0], self.requests.shape[0], self.joins.shape[0], self.n_slots, self.tile_rows, self.cluster, self.own_tiles)

    def rounded(self) -> "SharedPlan":
        """The same work in lists of few sizes (two to an octave), so that few launches have to be recorded: items behind the last have no
        members, which makes them no pieces, and nobody points to other entries behind the last."""
        def room(arr: np.ndarray) -> np.ndarray:
            out = np.zeros((_rounded(arr.shape[0]), *arr.shape[1:]), dtype=arr.dtype)
            out[:arr.shape[0]] = arr
            return out

        return replace(self, items=room(self.items), members=room(self.members), joins=room(self.joins), n_slots=_rounded(self.n_slots))

    def sections(self) -> List[Tuple[str, np.ndarray]]:
        return [("items", self.items), ("members", self.members), ("requests", self.requests), ("joins", self.joins)]

    def bind(self, tensors: Dict[str, torch.Tensor], part_o: Optional[torch.Tensor], part_ml: Optional[torch.Tensor]) -> "SharedDevicePlan":
        return SharedDevicePlan(tensors["items"], tensors["members"], tensors["requests"], tensors["joins"], part_o, part_ml, self)

    def to(self, device) -> "SharedDevicePlan":
        """On the device, with scratch of its own: for callers without an engine's buffers.  Two calls that may run at once
        need a plan each."""
        tensors = {name: torch.from_numpy(arr).to(device) for name, arr in self.sections()}
        part_o = part_ml = None
        if self.n_slots:
            part_o = torch.empty((self.n_slots, self.n_heads, self.head_dim), dtype=torch.float32, device=device)
            part_ml = torch.empty((self.n_slots, self.n_heads, 2), dtype=torch.float32, device=device)
        return self.bind(tensors, part_o, part_ml)


@dataclass
class SharedDevicePlan:
    items: torch.Tensor
    members: torch.Tensor
    requests: torch.Tensor
    joins: torch.Tensor
    part_o: Optional[torch.Tensor]   # [slots, heads, head_dim] float32
    part_ml: Optional[torch.Tensor]  # [slots, heads, 2] float32
    host: SharedPlan
    fixed: Optional[object] = field(default=None, init=False, compare=False)  # what its launches have in common: made by the first

    def __setattr__(self, name: str, value: object) -> None:
        """Whatever is replaced, the next launch looks at everything again (a launch that did so by itself took 0.6 us longer)."""
        own = self.__dict__
        own["fixed"] = None
        own[name] = value


def tile_members(n: int, most: int) -> List[Tuple[int, int]]:
    """``n`` members in as few tiles of at most ``most`` as there are, of about the same size: (first, members) each."""
    tiles = -(-n // most)
    edges = [n * i // tiles for i in range(tiles + 1)]
    return [(a, b - a) for a, b in zip(edges, edges[1:])]


def own_slots(dtype: torch.dtype, head_dim: int) -> int:
    """CTAs of the kernel for own keys on an SM: by registers, and by shared memory with all of its places for tiles."""
    if dtype == torch.bfloat16:
        smem = (ROWS_TILE + 6 * ROWS_KEYS[dtype]) * (head_dim + 8) * 2
    else:
        smem = (ROWS_TILE * head_dim + 4 * ROWS_KEYS[dtype] * (head_dim + 4)) * 4
    return max(1, min(OWN_CTAS_PER_SM if head_dim <= 128 else 2, 228 * 1024 // (smem + 5 * 1024)))


def own_cluster(longest: int, blocks: int, dtype: torch.dtype, slots: int) -> int:
    """CTAs that share one request's own keys, none with less than two tiles of them.  A CTA takes as long to come and go as for some of its
    tiles (and for one more with every two others it joins with), and clusters beyond the ``slots`` of the GPU (a seventh of them stays
    empty) wait for several at once.  Clusters of 1, 2, 4 and 8, us, own keys of one length: 48 heads on 8 of 128, 20 requests of 600 26,
    35, 47, 78; 8 of 4,000 84, 52, 35, 45; 32 of 1,500 46, 54, 68, 102; 16 on 4 of 64 in 32 bits, 6 of 1,000 91, 50, 29, 20."""
    tile, lost = ROWS_KEYS[dtype], 9.0 if dtype == torch.bfloat16 else 4.0
    best, best_t, cluster = 1, None, 1
    while cluster <= MOST_CLUSTER and (cluster == 1 or longest > cluster * tile):
        t = max(1.0, blocks * cluster / (0.85 * slots)) * (lost + 0.75 * longest / (cluster * tile) + cluster // 2)  # (lengths vary: three quarters)
        if best_t is None or t < 0.95 * best_t:
            best, best_t = cluster, t
        cluster *= 2
    return best


def rows_length(units: Sequence[int], heads: int, dtype: torch.dtype, sm_count: int) -> int:
    """The most tiles of keys a piece of the kernels for few rows may have.  A CTA goes through its piece tile by tile, and every piece's
    result is joined behind it, so both grow with the root of a span; and pieces beyond one wave of CTAs (four, once there are
    that many) only queue.  Measured, pieces of 1, 2 and 4 tiles: two requests of 48 heads on 8 over 256 keys 8.7, 9.5, 11.5 us, over 1,024
    11.3, 10.5, 11.8, over 4,096 29.7, 18.7, 14.6; 16 over 256 15.4, 11.0, 12.0; in 32 bits (16 heads on 4 of 64) two over 256 9.0,
    11.8, 18.2, over 4,096 24.3, 19.7, 21.8."""
    if not units:
        return 1
    total = sum(units) * heads
    root = math.ceil(math.sqrt(max(units)) / (2 if dtype == torch.bfloat16 else 4))
    return max(root, -(-total // (sm_count if total <= 4 * sm_count else 4 * sm_count)))


def takes_wide(dtype: torch.dtype, head_dim: int, page_size: int, group: int) -> bool:
    """Whether the tcgen05 kernel takes these sizes (``csrc/shared_attention_tc.cuh: shared_tc_fits``)."""
    return dtype == torch.bfloat16 and head_dim in (64, 128) and page_size % 16 == 0 and page_size >= 16 and group <= WIDE_TILE // 2


def wide_pays(sets: Sequence[Span], group: int, n_kv_heads: int, head_dim: int) -> bool:
    """Whether the tcgen05 kernel is faster than the one for few rows.  That one reads a set's keys once for every 16 query rows, the
    other has some 5 us more around its pieces: it takes over from 45,000 keys on, counted once per tile of 16 rows and KV head, where those
    tiles are 24 and more, from 100,000 where they are fewer (and hold up each other less), twice as many for heads of 64.  A layer of 48
    heads on 8 of 128, few rows against tcgen05: 3 requests over 4,096 keys 17.7 and 19.7 us, over 8,192 32.0 and 22.0; 5 over 1,024 12.8 and
    13.1, over 2,048 15.4 and 14.8; 48 over 256 20.0 and 14.6.  16 on 4 of 128: 8 over 8,192 20.5 and 22.5, over 16,384 25.9 and 24.8; 48 over
    256 10.3 and 14.3, over 1,024 18.4 and 15.1; of 64: 48 over 1,024 12.3 and 12.5, over 2,048 16.9 and 13.3; 16 over 8,192 16.1 and
    19.2, over 16,384 28.7 and 21.3."""
    tiles = [-(-len(members) // max(1, ROWS_TILE // group)) * max(1, -(-group // ROWS_TILE)) * n_kv_heads for members, _, _ in sets]
    keys = sum(t * (end - start) for t, (_, start, end) in zip(tiles, sets))
    return keys * head_dim >= 128 * (45000 if sum(tiles) >= 24 else 100000)


def piece_lengths(units: np.ndarray, two: np.ndarray, members: np.ndarray, n_kv_heads: int, row_bytes: int, ctas: int, own_ctas: int) -> int:
    """The most key tiles a piece of the tcgen05 kernel may have, by the estimated time of the launches: the kernel deals the sorted
    list out to and fro over its CTAs, the busiest of them decides; partial results are written and read once per piece; and the kernel
    for own keys runs under it where SMs are left that have room for all of its CTAs.  (12 requests of 48 heads on 8 over 4,096 keys, 128 pieces 28.2
    us, 64 pieces 18.9; 16 over 16,384 37.1 and 31.2 with 104.)"""
    best, best_t = 1, None
    longest = int(units.max())
    seen = set()
    for k in range(1, 65):
        most = -(-longest // k)
        if most in seen:
            continue
        seen.add(most)
        n = -(-units // most)
        low, more = units // n, units % n
        # of a tile's n pieces `more` have one unit more than the others
        costs = np.concatenate([np.repeat(low + 1, more), np.repeat(low, n - more)]).astype(np.float64)
        wide = np.concatenate([np.repeat(two, more), np.repeat(two, n - more)])
        costs = WIDE_PIECE_US + costs * np.where(wide, WIDE_TWO_US, WIDE_ONE_US)
        costs = np.sort(np.repeat(costs, n_kv_heads))[::-1]
        g = min(ctas, costs.shape[0])
        rounds = -(-costs.shape[0] // g)
        costs = np.concatenate([costs, np.zeros(rounds * g - costs.shape[0])]).reshape(rounds, g)
        costs[1::2] = costs[1::2, ::-1].copy()
        slots = float((n * members).sum())
        if best_t is not None and slots * row_bytes > 2 * MOST_SLOT_BYTES:
            break  # (row_bytes: written and read)
        t = float(costs.sum(axis=0).max()) + slots * row_bytes / JOIN_BYTES_PER_US
        if own_ctas > OWN_CTAS_PER_SM * (ctas - g):
            t += OWN_BEHIND_US
        if best_t is None or t < best_t * 0.99:
            best, best_t = most, t
        if most == 1:
            break
    return best


@dataclass
class SharedLayout:
    """What a work list has that does not depend on the requests' lengths: it stays while the same requests share the same pages."""

    items: np.ndarray
    members: np.ndarray
    joins: np.ndarray
    fixed: np.ndarray  # [n, 8] requests, without their ends
    n_slots: int
    wide: bool
    n_heads: int
    n_kv_heads: int
    head_dim: int
    dtype: torch.dtype
    blocks: int        # CTAs it has without clusters
    slots: int         # CTAs of it that the GPU takes at once

    def plan(self, kv_lens: Sequence[int]) -> SharedPlan:
        requests = self.fixed.copy()
        requests[:, 3] = kv_lens
        longest = max(1, int((requests[:, 3] - requests[:, 2]).max(initial=0)))
        longest = 1 << (longest - 1).bit_length()
        cluster = own_cluster(longest, self.blocks, self.dtype, self.slots)
        # the longest first: 48 requests of up to 1,500 own keys 66 -> 46 us, 32 of up to 700 beside 32,000 shared ones 66.0 -> 63.5
        requests = requests[np.argsort(requests[:, 2] - requests[:, 3], kind="stable")]
        return SharedPlan(self.items, self.members, requests, self.joins, self.n_slots, WIDE_TILE if self.wide else ROWS_TILE, cluster,
                          -(-longest // (cluster * ROWS_KEYS[self.dtype])), requests.shape[0], self.n_heads, self.n_kv_heads, self.head_dim)


def build_shared_plan(kv_lens: Sequence[int], spans: Sequence[Span], n_heads: int, n_kv_heads: int, head_dim: int, dtype: torch.dtype,
                      page_size: int, table_rows: Optional[Sequence[int]] = None, sm_count: int = 148,
                      tile_rows: Optional[int] = None) -> SharedPlan:
    """The work list of one step: request ``i`` has query row ``i``, ``kv_lens[i]`` keys (its own token's among them) and row
    ``table_rows[i]`` (``i``) of the block table.

    ``spans``: (members, start, end) of keys that the members share: the block-table rows of all of them must name the same pages
    for these positions (the first member's row is read).  ``end`` may lie inside a page.  The spans of one request must not
    overlap and leave no positions out in front of them; a span of a single member is that request's own.

    The tcgen05 kernel takes the shared keys where it takes the sizes, spans begin on multiples of 16 and it is faster
    (:func:`wide_pays`); ``tile_rows`` (16 or 256) asks for one of the two."""
    if any(x < 0 for x in kv_lens):
        raise KernelError("shared_attention: a negative length")
    for members, start, end in spans:
        if any(0 <= int(m) < len(kv_lens) and int(end) > kv_lens[int(m)] for m in members):
            raise KernelError(f"shared_attention: the span [{start}, {end}) does not lie within its members' keys")
    return shared_layout(len(kv_lens), spans, n_heads, n_kv_heads, head_dim, dtype, page_size, table_rows, sm_count, tile_rows).plan(kv_lens)


def shared_layout(n: int, spans: Sequence[Span], n_heads: int, n_kv_heads: int, head_dim: int, dtype: torch.dtype, page_size: int,
                  table_rows: Optional[Sequence[int]] = None, sm_count: int = 148, tile_rows: Optional[int] = None) -> SharedLayout:
    """:func:`build_shared_plan` for ``n`` requests up to their lengths, which must reach the spans' ends."""
    if n_heads < 1 or n_kv_heads < 1 or n_heads % n_kv_heads:
        raise KernelError(f"shared_attention: {n_heads} query heads on {n_kv_heads} KV heads")
    rows = list(range(n)) if table_rows is None else [int(r) for r in table_rows]
    if len(rows) != n:
        raise KernelError("shared_attention: one block-table row per request")
    if dtype not in ROWS_KEYS:
        raise KernelError(f"shared_attention: dtype {dtype} is not supported (float32 or bfloat16)")
    group = n_heads // n_kv_heads
    taken: List[List[Tuple[int, int]]] = [[] for _ in range(n)]
    sets: List[Tuple[List[int], int, int]] = []
    for members, start, end in spans:
        members = [int(m) for m in members]
        start, end = int(start), int(end)
        if len(set(members)) != len(members) or any(not 0 <= m < n for m in members):
            raise KernelError("shared_attention: a span's members are different requests of the step")
        if start < 0:
            raise KernelError(f"shared_attention: the span [{start}, {end}) does not lie within its members' keys")
        if end <= start or len(members) < 2:
            continue
        for m in members:
            if any(a < end and start < b for a, b in taken[m]):
                raise KernelError(f"shared_attention: request {m} is in two spans that overlap")
            taken[m].append((start, end))
        sets.append((members, start, end))

    wide = takes_wide(dtype, head_dim, page_size, group) and all(start % 16 == 0 for _, start, _ in sets) \
        and wide_pays(sets, group, n_kv_heads, head_dim)
    if tile_rows is not None:
        if tile_rows not in (ROWS_TILE, WIDE_TILE) or (tile_rows == WIDE_TILE and (not takes_wide(dtype, head_dim, page_size, group) or any(
                start % 16 for _, start, _ in sets))):
            raise KernelError(f"shared_attention: pieces of {tile_rows} query rows are not taken at these sizes")
        wide = tile_rows == WIDE_TILE
    chunks = -(-group // ROWS_TILE)  # (of the kernels for few rows)
    most = 2 * (WIDE_TILE // 2 // group) if wide else max(1, ROWS_TILE // min(group, ROWS_TILE))
    unit = WIDE_KEYS if wide else ROWS_KEYS[dtype]
    tiles = [(members[a:a + k], start, end) for members, start, end in sets for a, k in tile_members(len(members), most)]
    units = [-(-(end - start) // unit) for _, start, end in tiles]
    own_ctas = max(1, n * n_kv_heads * chunks)
    if wide and tiles:
        length = piece_lengths(np.array(units), np.array([2 * len(m) > most for m, _, _ in tiles]), np.array([len(m) for m, _, _ in tiles]),
                               n_kv_heads, 8 * n_heads * head_dim, sm_count, max(own_ctas, min(2 * own_ctas, sm_count)))  # (clusters of two, often)
    else:
        length = rows_length(units, n_kv_heads * chunks, dtype, sm_count)
    items, member_rows, slots = [], [], [[] for _ in range(n)]
    n_slots = 0
    for (members, start, end), u in zip(tiles, units):
        first = len(member_rows)
        member_rows += members
        for a, k in tile_members(u, length):
            cost = k * (WIDE_TWO_US if 2 * len(members) > most else WIDE_ONE_US) if wide else float(k)
            split = wide and 2 * len(members) <= most and k > 1  # one query tile: both halves of the kernel, half of the key tiles each
            items.append((-cost, first, len(members), rows[members[0]], start + a * unit, min(end, start + (a + k) * unit), n_slots, int(split), 0))
            for half in range(2 if split else 1):
                for i, m in enumerate(members):
                    slots[m].append((start + (a + half) * unit, n_slots + half * len(members) + i))
            n_slots += (2 if split else 1) * len(members)
    items = [it[1:] for it in sorted(items, key=lambda it: it[0])]  # the longest first

    # what is a request's own: one range behind its spans
    requests, joins = [], []
    for i in range(n):
        begin = 0
        for a, b in sorted(taken[i]):
            if a != begin:
                raise KernelError(f"shared_attention: the spans of request {i} leave out positions {begin} to {a}")
            begin = b
        own = [s for _, s in sorted(slots[i])]
        requests.append((i, rows[i], begin, begin, len(joins), len(own), 0, 0))
        joins += own
    as_int = lambda x, w: np.asarray(x, dtype=np.int32).reshape(-1, w) if w else np.asarray(x, dtype=np.int32)  # noqa: E731
    return SharedLayout(as_int(items, ITEM_INTS), as_int(member_rows, 0), as_int(joins, 0), as_int(requests, REQUEST_INTS), n_slots, wide,
                        n_heads, n_kv_heads, head_dim, dtype, own_ctas, sm_count * own_slots(dtype, head_dim))
