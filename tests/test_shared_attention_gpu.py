"""Attention over shared keys against the sums in 64 bits: head layouts, pages, nested spans, lengths from zero on, and how it is called."""

import numpy as np
import pytest
import torch

from freetoken_b200.engine.shared_plan import build_shared_plan
from freetoken_b200.errors import KernelError
from freetoken_b200.kernels import ops

DEV = "cuda:0"


def layout(lens, spans, page, gen):
    """Pages of every request, shared ones where spans say so: a block table, pages used, and per request the pages of its blocks.
    A span that ends inside a page shares the page up to there: the members' rows name pages of their own with equal rows in them."""
    n = len(lens)
    width = max(1, max(-(-x // page) for x in lens)) + 2
    table, owner, count = np.zeros((n, width), dtype=np.int64), {}, 1
    for members, start, end in spans:
        for block in range(start // page, end // page):  # whole pages
            if block * page < start:
                continue
            for m in members:
                table[m, block] = count
            count += 1
    copies = []  # (from page, to page, rows): equal rows in pages of their own
    for i in range(n):
        for block in range(-(-lens[i] // page)):
            if table[i, block] == 0:
                table[i, block] = count
                count += 1
    for members, start, end in spans:
        for block in range(start // page, -(-end // page)):
            for m in members[1:]:
                if table[m, block] != table[members[0], block]:
                    lo, hi = max(start, block * page) - block * page, min(end, block * page + page) - block * page
                    copies.append((table[members[0], block], table[m, block], lo, hi))
    order = torch.randperm(count - 1, generator=gen).numpy() + 1  # places anywhere in the pool
    place = np.concatenate([[0], order])
    return place[table], count, [(place[a], place[b], lo, hi) for a, b, lo, hi in copies]


def case(lens, spans, heads, kv_heads, dim, page, dtype, seed=0, extra_rows=0, spread=1.5):
    gen = torch.Generator().manual_seed(seed)
    table, pages, copies = layout(lens, spans, page, gen)
    k = torch.randn((pages, kv_heads, page, dim), generator=gen).to(dtype)
    v = torch.randn((pages, kv_heads, page, dim), generator=gen).to(dtype)
    for a, b, lo, hi in copies:
        k[b, :, lo:hi] = k[a, :, lo:hi]
        v[b, :, lo:hi] = v[a, :, lo:hi]
    live = torch.zeros((pages, page), dtype=torch.bool)
    for i, x in enumerate(lens):
        pos = np.arange(x)
        live[table[i, pos // page], pos % page] = True
    k.masked_fill_(~live[:, None, :, None], float("nan"))  # fresh pages may hold anything
    v.masked_fill_(~live[:, None, :, None], float("nan"))
    q = (torch.randn((len(lens) + extra_rows, heads, dim), generator=gen) * spread).to(dtype)
    return q, k, v, torch.from_numpy(table.astype(np.int32))


def reference(q, k, v, table, lens, scale, sink=None):
    """(outputs, sum of |weight x value|, largest sum of |q k| scale) in 64 bits."""
    n, (H, D), G, P = len(lens), q.shape[1:], k.shape[1], k.shape[2]
    out, size, reach = torch.zeros((n, H, D), dtype=torch.float64), torch.zeros((n, H, D), dtype=torch.float64), torch.zeros((n, H, 1), dtype=torch.float64)
    for i, x in enumerate(lens):
        if x == 0:
            continue
        pos = torch.arange(x)
        page, at = table[i, pos // P].long(), pos % P
        for h in range(H):
            kk, vv = k[page, h // (H // G), at].double(), v[page, h // (H // G), at].double()
            s = kk @ q[i, h].double() * scale
            m = s.max()
            w = torch.exp(s - m)
            w = w / (w.sum() + (torch.exp(sink[h].double() - m) if sink is not None else 0.0))
            out[i, h], size[i, h] = w @ vv, w @ vv.abs()
            reach[i, h] = (kk.abs() @ q[i, h].double().abs()).max() * scale
    return out, size, reach


def bound(out, size, reach, dtype, dim, keys):
    """What roundings may move an output by.  Scores are sums of `dim` products in 32 bits: each off by at most dim 2^-24 of the sum of the
    products' sizes, an exponential by as much (the maximum's error is common to all and cancels), and by 2^-21 for its own evaluation
    in bfloat16's kernels (ex2.approx: 2^-22.5 and its argument's rounding at sizes up to 64: 2^-24 64 ln 2 / 2^... within 2^-18); sums over `keys` terms in 32 bits.
    bfloat16: probabilities are rounded (2^-8 at most each), and the result (2^-8)."""
    f32 = 2.0 ** -24 * (2 * dim * reach + 2 * keys + 32) * size
    if dtype == torch.float32:
        return f32 + 2.0 ** -23 * out.abs()
    return f32 + (2.0 ** -8 + 2.0 ** -18) * size + 2.0 ** -8 * out.abs() * (1 + 2.0 ** -7)


def run(q, k, v, table, plan, scale, sink=None, fill=7.0):
    d = lambda t: t.to(DEV)  # noqa: E731
    out = torch.full_like(q, fill, device=DEV)
    ops.shared_attention(d(q), d(k), d(v), d(table), plan, out, scale, sink=sink)
    torch.cuda.synchronize()
    ops.check_status()
    return out.cpu()


def check(lens, spans, heads, kv_heads, dim, page, dtype, seed=0, sink=None, spread=1.5, sm_count=148, tile_rows=None):
    q, k, v, table = case(lens, spans, heads, kv_heads, dim, page, dtype, seed, extra_rows=2, spread=spread)
    plan = build_shared_plan(lens, spans, heads, kv_heads, dim, dtype, page, sm_count=sm_count, tile_rows=tile_rows).to(DEV)
    scale = dim ** -0.5
    per_head = sink if sink is None or isinstance(sink, torch.Tensor) else torch.full((heads,), sink)
    got = run(q, k, v, table, plan, scale, sink.to(DEV) if isinstance(sink, torch.Tensor) else sink)
    want, size, reach = reference(q, k, v, table, lens, scale, per_head)
    limit = bound(want, size, reach, dtype, dim, max(lens))
    far = (got[: len(lens)].double() - want).abs()
    assert torch.isfinite(got).all()
    assert (far <= limit).all(), (far - limit).max().item()
    assert (got[len(lens):] == 7.0).all()  # rows that are no request's
    return plan


F32, BF16 = torch.float32, torch.bfloat16
TWO = [([0, 1], 0, 48)]
SIZES = [
    # lens, spans, heads, KV heads, head size, page
    ([50, 49], TWO, 12, 2, 128, 16),
    ([300, 257, 256, 290], [([0, 1, 2, 3], 0, 256)], 12, 2, 128, 16),
    ([300, 257, 256, 290], [([3, 1, 0, 2], 0, 256)], 16, 4, 64, 16),
    ([700] * 25, [(list(range(25)), 0, 640)], 6, 1, 128, 16),          # more members than a tile has room for
    ([200, 201, 330, 331, 90], [([0, 1, 2, 3], 0, 128), ([2, 3], 128, 320)], 16, 4, 64, 16),  # nested, and a request by itself
    ([70, 80, 75], [([0, 2], 0, 61)], 4, 4, 16, 16),                   # one head each; the span ends inside a page
    ([70, 80, 75], [([0, 1, 2], 0, 64)], 32, 1, 64, 16),               # more heads on a KV head than a tile of few rows has
    ([40, 33], [([0, 1], 0, 32)], 40, 2, 48, 4),                       # odd head size, small pages
    ([100, 91], [([0, 1], 0, 91)], 4, 2, 256, 7),                      # large heads, pages of 7; one request has nothing of its own
    ([130, 140, 1], [([0, 1], 0, 128)], 8, 8, 128, 64),
    ([1, 0, 1], [], 8, 2, 128, 16),                                    # nothing shared; a request without keys
    ([1000, 1, 33], [], 8, 2, 64, 16),
    ([2, 2, 2], [([0, 1, 2], 0, 1)], 8, 2, 64, 1),
    ([1, 1], [([0, 1], 0, 1)], 128, 1, 128, 16),                       # 128 heads on one
    ([4000, 4100], [([0, 1], 0, 3968)], 6, 1, 128, 16),                # many pieces of one span
    ([4500], [], 6, 1, 128, 16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("at", range(len(SIZES)))
def test_sizes(at, dtype):
    check(*SIZES[at], dtype, seed=at)


WIDE = [
    # the tcgen05 kernel: one and two query tiles, pieces that end anywhere in a key tile, several pieces a CTA
    ([40, 50], [([0, 1], 0, 16)], 16, 4, 128, 16),
    ([40, 50], [([0, 1], 0, 17)], 4, 4, 64, 16),
    ([150] * 64, [(list(range(64)), 0, 144)], 6, 1, 128, 16),                                       # two tiles of 16 members each
    ([600] * 43, [(list(range(42)), 0, 512)], 12, 2, 64, 32),                                       # 42 members: two full tiles
    ([300] * 5, [(list(range(5)), 0, 272)], 128, 1, 128, 16),                                       # a member a tile
    ([1300, 1400, 1290, 1288, 1500, 1310], [(list(range(6)), 0, 640), ([0, 1, 2], 640, 1280), ([3, 4, 5], 640, 1288)], 24, 2, 128, 64),
    ([3000] * 30, [(list(range(30)), 0, 2900)], 48, 8, 128, 16),
    ([520] * 100, [(list(range(k, 100, 10)), 0, 320 + 16 * k) for k in range(10)], 16, 4, 64, 16),  # many sets of different lengths
]


@pytest.mark.gpu
@pytest.mark.parametrize("tile_rows,sm_count", [(16, 148), (256, 148), (256, 7)])  # (few SMs in the list's eyes: long pieces)
@pytest.mark.parametrize("at", range(len(WIDE)))
def test_both_forms_for_shared_keys(at, tile_rows, sm_count):
    ops.variant_counts(reset=True)
    plan = check(*WIDE[at], BF16, seed=at, tile_rows=tile_rows, sm_count=sm_count)
    assert plan.host.tile_rows == tile_rows
    assert ops.variant_counts()["shared attention: tcgen05, 256 rows" if tile_rows == 256 else "shared attention: bfloat16 mma.sync, 16 rows"] == 1


@pytest.mark.gpu
def test_large_scores_on_tcgen05():
    check([1900, 1950] * 10, [(list(range(20)), 0, 1880)], 12, 2, 128, 16, BF16, spread=12.0, tile_rows=256)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("sink", ["number", "heads"])
def test_sinks(dtype, sink):
    heads = 12
    value = 0.7 if sink == "number" else torch.linspace(-3, 4, heads)
    check([300, 257, 0, 290, 1], [([0, 1, 3], 0, 256)], heads, 2, 128, 16, dtype, sink=value)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_large_scores(dtype):
    """Weights that fall on a few keys, and maxima that move from piece to piece."""
    check([900, 950], [([0, 1], 0, 880)], 12, 2, 128, 16, dtype, spread=12.0)


@pytest.mark.gpu
def test_infinities_and_nan_stay_with_their_request():
    lens, spans = [300, 280, 270], [([0, 1, 2], 0, 256)]
    q, k, v, table = case(lens, spans, 12, 2, 128, 16, BF16)
    scale, plan = 128 ** -0.5, build_shared_plan(lens, spans, 12, 2, 128, BF16, 16).to(DEV)
    clean = run(q, k, v, table, plan, scale)
    page, at = table[1, 270 // 16].long(), 270 % 16  # a key of request 1 alone
    v[page, 0, at, 5] = float("inf")
    k[page, 1, at] = float("nan")
    got = run(q, k, v, table, plan, scale)
    assert torch.equal(got[[0, 2]], clean[[0, 2]])
    assert torch.isinf(got[1, :6, 5]).all() and torch.isnan(got[1, 6:]).all() and torch.isfinite(got[1, :6, :5]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype,tile_rows", [(F32, 16), (BF16, 16), (BF16, 256)])
def test_nan_and_infinite_scores_reach_who_reads_them(dtype, tile_rows, value):
    """Every place of a key tile in turn: as a shared key, and as the only key that a request has of its own."""
    lens, spans = [257, 258, 300], [([0, 1], 0, 256)]
    q, k, v, table = case(lens, spans, 16, 2, 128, 16, dtype)
    q[:, :, 0] = q[:, :, 0].abs() + 0.1  # (an infinite key gives +infinity to every query)
    scale = 128 ** -0.5
    plan = build_shared_plan(lens, spans, 16, 2, 128, dtype, 16, tile_rows=tile_rows).to(DEV)
    clean = run(q, k, v, table, plan, scale)
    assert torch.isfinite(clean).all()
    for pos in list(range(0, 256, 37)) + list(range(128, 160)):
        bad = k.clone()
        bad[table[0, pos // 16].long(), 1, pos % 16, 0] = value
        got = run(q, bad, v, table, plan, scale)
        assert torch.isnan(got[:2, 8:]).all() and torch.equal(got[:2, :8], clean[:2, :8]) and torch.equal(got[2], clean[2]), pos
    k[table[0, 16].long(), 1, 0, 0] = value
    got = run(q, k, v, table, plan, scale)
    assert torch.isnan(got[0, 8:]).all() and torch.equal(got[0, :8], clean[0, :8]) and torch.equal(got[1:], clean[1:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_captured_replayed_and_on_another_stream(dtype):
    lens, spans = [300, 257, 256, 290], [([0, 1, 2, 3], 0, 256)]
    q, k, v, table = [t.to(DEV) for t in case(lens, spans, 16, 4, 64, 16, dtype)]
    scale, plan = 64 ** -0.5, build_shared_plan(lens, spans, 16, 4, 64, dtype, 16).to(DEV)
    want = run(q, k, v, table, plan, scale)
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        ops.shared_attention(q, k, v, table, plan, out, scale)
    side.synchronize()
    assert torch.equal(out.cpu(), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.shared_attention(q, k, v, table, plan, out, scale)
    other = torch.randn_like(q)
    plain = run(other, k, v, table, plan, scale)
    for src, ref in ((q.clone(), want), (other, plain), (other, plain)):
        q.copy_(src)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.cpu(), ref)


@pytest.mark.gpu
def test_two_calls_at_once_with_plans_of_their_own():
    lens, spans = [2000] * 12, [(list(range(12)), 0, 1920)]
    q, k, v, table = [t.to(DEV) for t in case(lens, spans, 12, 2, 128, 16, BF16)]
    scale = 128 ** -0.5
    plans = [build_shared_plan(lens, spans, 12, 2, 128, BF16, 16).to(DEV) for _ in range(2)]
    want = run(q, k, v, table, plans[0], scale)
    outs, streams = [torch.empty_like(q) for _ in range(2)], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for plan, out, stream in zip(plans, outs, streams):
            with torch.cuda.stream(stream):
                ops.shared_attention(q, k, v, table, plan, out, scale)
    torch.cuda.synchronize()
    assert torch.equal(outs[0].cpu(), want) and torch.equal(outs[1].cpu(), want)


@pytest.mark.gpu
def test_pages_outside_the_pool_are_not_read():
    """A block table that names pages that do not exist: those keys are not there."""
    lens, spans = [300, 290], [([0, 1], 0, 256)]
    q, k, v, table = case(lens, spans, 16, 4, 64, 16, BF16)
    plan, scale = build_shared_plan(lens, spans, 16, 4, 64, BF16, 16).to(DEV), 0.125
    bad = table.clone()
    bad[1, 17:] = 1 << 30  # request 1's own keys from position 272 on
    bad[0, 18] = -5        # request 0's from 288 on
    got = run(q, k, v, bad, plan, scale)
    want, size, reach = reference(q, k, v, table, [288, 272], scale)
    assert ((got[:2].double() - want).abs() <= bound(want, size, reach, BF16, 64, 300)).all()


@pytest.mark.gpu
def test_refusals():
    lens, spans = [50, 49], TWO
    q, k, v, table = [t.to(DEV) for t in case(lens, spans, 8, 2, 64, 16, BF16)]
    plan = build_shared_plan(lens, spans, 8, 2, 64, BF16, 16).to(DEV)
    out = torch.empty_like(q)
    ops.shared_attention(q, k, v, table, plan, out, 0.125)
    for args in [
        (q.float(), k, v, table, plan, out), (q, k.float(), v, table, plan, out), (q, k, v, table.long(), plan, out),
        (q[:, :4], k, v, table, plan, out[:, :4]), (q[:1], k, v, table, plan, out[:1]), (q, k, v[:1], table, plan, out),
        (q.cpu(), k, v, table, plan, out), (q, k, v, table, plan, out[:1]), (q, k.transpose(1, 2), v.transpose(1, 2), table, plan, out),
    ]:
        with pytest.raises(KernelError):
            ops.shared_attention(*args, 0.125)
    with pytest.raises(KernelError):
        ops.shared_attention(q, k, v, table, plan, out, 0.125, sink=torch.zeros(3, device=DEV))
    with pytest.raises(KernelError, match="positive scale"):
        ops.shared_attention(q, k, v, table, build_shared_plan(lens, spans, 8, 2, 64, BF16, 16, tile_rows=256).to(DEV), out, -0.125)
    wide = torch.empty((3, 8, 24), dtype=BF16, device=DEV)
    slab = torch.empty((4, 2, 16, 24), dtype=BF16, device=DEV)
    with pytest.raises(KernelError, match="head_dim"):
        ops.shared_attention(wide, slab, slab, table, build_shared_plan(lens, [], 8, 2, 24, BF16, 16).to(DEV), torch.empty_like(wide), 0.125)


@pytest.mark.gpu
@pytest.mark.parametrize("tile_rows", [16, 256])
def test_rounded_lists_give_the_same(tile_rows):
    lens, spans = [700, 650, 644, 300, 701, 0, 650], [([0, 1, 2, 4, 6], 0, 640), ([3, 5], 0, 0)]
    q, k, v, table = case(lens, spans, 16, 4, 64, 16, BF16)
    plan = build_shared_plan(lens, spans, 16, 4, 64, BF16, 16, tile_rows=tile_rows)
    round_ = plan.rounded()
    assert round_.key() != plan.key()
    got = [run(q, k, v, table, p.to(DEV), 0.125) for p in (plan, round_)]
    assert torch.equal(*got)


@pytest.mark.gpu
def test_a_plan_on_another_device_is_refused(monkeypatch):
    lens, spans = [50, 49], TWO
    q, k, v, table = [t.to(DEV) for t in case(lens, spans, 8, 2, 64, 16, BF16)]
    plan, out = build_shared_plan(lens, spans, 8, 2, 64, BF16, 16).to(DEV), torch.empty_like(q)
    ops.shared_attention(q, k, v, table, plan, out, 0.125)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1)  # (of two, the second is current)
    with pytest.raises(KernelError, match="the plan is on"):
        ops.shared_attention(q, k, v, table, plan, out, 0.125)
