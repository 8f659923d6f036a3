"""Work lists of attention over shared keys, played through on the host."""

import random

import numpy as np
import pytest
import torch

from freetoken_b200.engine.shared_plan import build_shared_plan, own_cluster, tile_members
from freetoken_b200.errors import KernelError


def covered(plan, n, rows):
    """Per request: the key ranges of its pieces in the order in which they are joined, then its own."""
    of_slot = {}
    for mem0, k, row, kb, ke, slot0, split, _ in plan.items.tolist():
        assert kb < ke and 0 <= mem0 and mem0 + k <= len(plan.members)
        members = plan.members[mem0:mem0 + k].tolist()
        assert row == rows[members[0]]
        assert not split or (plan.tile_rows == 256 and ke - kb > 128)
        for i, m in enumerate(members * (2 if split else 1)):  # (a split piece: even and odd key tiles, the second without a range of its own)
            assert slot0 + i not in of_slot and slot0 + i < plan.n_slots
            of_slot[slot0 + i] = (m, kb, ke) if i < k else (m, ke, ke)
    assert sorted(of_slot) == list(range(plan.n_slots))
    out = [None] * n
    own = (plan.requests[:, 3] - plan.requests[:, 2]).tolist()
    assert own == sorted(own, reverse=True) and sorted(plan.requests[:, 0].tolist()) == list(range(n))  # (the longest first)
    for i, row, lo, hi, j0, k, *_ in plan.requests.tolist():
        assert row == rows[i]
        pieces = [of_slot[s] for s in plan.joins[j0:j0 + k].tolist()]
        assert all(m == i for m, _, _ in pieces)
        out[i] = [(a, b) for _, a, b in pieces] + [(lo, hi)]
    return out


@pytest.mark.parametrize("seed", range(30))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_every_key_of_every_request_is_taken_once(seed, dtype):
    rng = random.Random(seed)
    heads, kv_heads = rng.choice([(48, 8), (16, 4), (16, 16), (40, 2), (128, 1)])
    n = rng.randint(1, 40)
    system = rng.choice([0, rng.randint(1, 3000)])
    lens, spans, at = [system + rng.randint(0, 400) for _ in range(n)], [], 0
    if system:
        spans.append((list(range(n)), 0, system))
    while at < n:
        k = rng.randint(1, 7)
        members = list(range(at, min(n, at + k)))
        common = min(lens[m] for m in members)
        if common > system:
            spans.append((members, system, rng.randint(system + 1, common)))
        at += k
    rows = rng.sample(range(100), n)
    plan = build_shared_plan(lens, spans, heads, kv_heads, 64, dtype, 16, table_rows=rows, sm_count=rng.choice([1, 16, 148]))
    for i, pieces in enumerate(covered(plan, n, rows)):
        edge = 0
        for a, b in pieces:
            assert a == edge and b >= a
            edge = b
        assert edge == lens[i]


def test_lists_keep_their_sizes_while_requests_grow():
    spans = [([0, 1, 2], 0, 640)]
    plans = [build_shared_plan([700 + t, 660 + t, 690 + t], spans, 16, 4, 64, torch.bfloat16, 16) for t in range(60)]
    # own parts of 20 to 119 tokens: the key changes only where the longest passes a power of two
    assert len({p.key() for p in plans}) <= 2
    assert len({p.items.tobytes() for p in plans}) == 1


def test_members_are_dealt_to_tiles_evenly():
    assert tile_members(64, 21) == [(0, 16), (16, 16), (32, 16), (48, 16)]
    assert tile_members(3, 21) == [(0, 3)]
    assert sum(k for _, k in tile_members(101, 7)) == 101


def test_own_keys_are_split_while_the_gpu_is_not_full():
    bf16, slots = torch.bfloat16, 296
    assert own_cluster(2048, 8, bf16, slots) == 8
    assert own_cluster(128, 8, bf16, slots) <= 2     # two tiles of keys each at least
    assert own_cluster(2048, 512, bf16, slots) == 1  # enough requests
    assert [own_cluster(1 << (x - 1).bit_length(), 8 * n, bf16, slots) for n, x in ((20, 600), (8, 4000), (32, 1500), (16, 2000), (18, 400))] == [1, 4, 1, 2, 1]
    assert own_cluster(1024, 24, torch.float32, 592) == 8


@pytest.mark.parametrize("lens,spans,what", [
    ([10, 10], [([0, 2], 0, 5)], "different requests"),
    ([10, 10], [([0, 0], 0, 5)], "different requests"),
    ([10, 4], [([0, 1], 0, 5)], "within"),
    ([10, 10], [([0, 1], -1, 5)], "within"),
    ([10, 10, 10], [([0, 1], 0, 5), ([1, 2], 4, 6)], "overlap"),
    ([10, 10], [([0, 1], 2, 5)], "leave out"),
    ([-1], [], "negative"),
])
def test_refusals(lens, spans, what):
    with pytest.raises(KernelError, match=what):
        build_shared_plan(lens, spans, 8, 2, 64, torch.float32, 16)


def test_the_wide_form_is_taken_where_it_fits_and_pays():
    def rows(members, keys, heads=16, kv=4, dim=64, dtype=torch.bfloat16, page=16, start=0, **kw):
        spans = ([(list(range(members)), 0, start)] if start else []) + [(list(range(members)), start, keys)]
        return build_shared_plan([keys + 40] * 48, spans, heads, kv, dim, dtype, page, **kw).tile_rows

    # the figures beside the rule: who is faster there
    assert [rows(n, k, 48, 8, 128) for n, k in ((3, 4096), (3, 8192), (5, 1024), (5, 2048), (48, 256), (16, 256), (16, 1024))] == [16, 256, 16, 256, 256, 16, 256]
    assert [rows(n, k, 16, 4, 128) for n, k in ((8, 8192), (8, 16384), (48, 256), (48, 1024), (2, 16384))] == [16, 256, 16, 256, 16]
    assert [rows(n, k) for n, k in ((48, 1024), (48, 2048), (16, 8192), (16, 16384))] == [16, 256, 16, 256]
    # sizes that it does not take
    assert rows(48, 4096) == 256
    assert rows(48, 4096, dtype=torch.float32) == rows(48, 4096, dim=48) == rows(48, 4096, page=8) == rows(48, 4096, heads=516) == rows(48, 4096, start=30) == 16
    assert rows(48, 4096, tile_rows=16) == 16 and rows(2, 64, tile_rows=256) == 256
    for kw in (dict(dim=48), dict(dtype=torch.float32), dict(page=8), dict(start=30)):
        with pytest.raises(KernelError):
            rows(20, 4096, tile_rows=256, **kw)
    with pytest.raises(KernelError):
        rows(20, 4096, tile_rows=64)
    with pytest.raises(KernelError):
        build_shared_plan([1], [], 8, 2, 64, torch.float16, 16)
    assert build_shared_plan([5], [], 8, 2, 64, torch.bfloat16, 16, tile_rows=256).items.shape == (0, 8)


def test_refuses_heads_that_do_not_divide():
    with pytest.raises(KernelError):
        build_shared_plan([1], [], 7, 2, 64, torch.float32, 16)
    with pytest.raises(KernelError):
        build_shared_plan([1, 1], [], 8, 2, 64, torch.float32, 16, table_rows=[0])


def test_recorded_steps_have_lists_of_few_sizes():
    """Prompts of every length under every number of continuations: as many launches to record as there are numbers, times a few."""
    keys = {}
    for members in (2, 7, 8):
        for length in range(640, 4096, 48):
            plan = build_shared_plan([length + 10] * members, [(list(range(members)), 0, length)], 48, 8, 128, torch.bfloat16, 16).rounded()
            keys.setdefault(members, set()).add(plan.key())
    assert max(len(k) for k in keys.values()) <= 14
    rng = random.Random(3)
    for n in (3, 9, 20):
        lens = [rng.randrange(900, 1300) for _ in range(n)]
        spans = [(list(range(n)), 0, 512), (list(range(n // 2)), 512, 864)]
        plan = build_shared_plan(lens, spans, 16, 4, 64, torch.bfloat16, 16)
        round_ = plan.rounded()
        for name in ("items", "members", "joins"):
            a, b = getattr(plan, name), getattr(round_, name)
            assert np.array_equal(b[:len(a)], a) and not b[len(a):].any() and len(a) <= len(b) <= 1.5 * len(a)
        assert plan.n_slots <= round_.n_slots and np.array_equal(plan.requests, round_.requests) and round_.rounded().key() == round_.key()
