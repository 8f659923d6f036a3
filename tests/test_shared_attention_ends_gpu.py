"""Attention over shared keys at its ends: what is not a number in a part that weighs next to nothing, scratch that was replaced, calls at once."""

import dataclasses
import threading

import pytest
import torch

from freetoken_b200.engine.shared_plan import build_shared_plan
from freetoken_b200.kernels import ops
from test_shared_attention_gpu import BF16, DEV, F32, case, run

HEADS, KV, DIM, PAGE = 16, 2, 128, 16
SCALE = DIM ** -0.5


def far_apart(lens, spans, dtype, high):
    """Keys whose first element puts a score some 280 above the others' where ``high(positions)`` says so: e^-280 is zero in 32 bits."""
    q, k, v, table = case(lens, spans, HEADS, KV, DIM, PAGE, dtype)
    q[:, :, 0] = 8.0
    for i, n in enumerate(lens):
        pos = torch.arange(n)
        k[table[i, pos // PAGE].long(), :, pos % PAGE, 0] = torch.where(high(pos), 400.0, 0.0).to(dtype)[:, None]
    return q, k, v, table


FORMS = [(F32, 16), (BF16, 16), (BF16, 256)]


@pytest.mark.gpu
@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("dtype,tile_rows", FORMS)
def test_nan_in_shared_keys_far_below_the_own_ones(dtype, tile_rows, whole):
    """A score that is no number makes the whole row none, however little its piece weighs beside the others."""
    lens, spans = [300, 290, 280], [([0, 1], 0, 256)]
    q, k, v, table = far_apart(lens, spans, dtype, lambda pos: pos >= 256)
    plan = build_shared_plan(lens, spans, HEADS, KV, DIM, dtype, PAGE, tile_rows=tile_rows).to(DEV)
    clean = run(q, k, v, table, plan, SCALE)
    assert torch.isfinite(clean).all()
    for pos in range(256) if whole else (37,):
        k[table[0, pos // PAGE].long(), 1, pos % PAGE, 3] = float("nan")
    got = run(q, k, v, table, plan, SCALE)
    assert torch.isnan(got[:2, 8:]).all() and torch.equal(got[:2, :8], clean[:2, :8]) and torch.equal(got[2], clean[2])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tile_rows", FORMS)
def test_nan_in_one_of_many_pieces(dtype, tile_rows):
    """Pieces beyond one run of the join (32 partial results at a time), the highest scores in the last of them and in the first."""
    for last in (True, False):
        lens, spans = [20000, 19990], [([0, 1], 0, 19904)]
        q, k, v, table = far_apart(lens, spans, dtype, lambda pos: ((19840 <= pos) & (pos < 19904)) if last else pos < 64)
        plan = build_shared_plan(lens, spans, HEADS, KV, DIM, dtype, PAGE, tile_rows=tile_rows).to(DEV)
        assert tile_rows == 256 or plan.host.requests[0, 5] > 32
        clean = run(q, k, v, table, plan, SCALE)
        assert torch.isfinite(clean).all()
        for pos in (100, 10000, 19800, 19989):
            bad = k.clone()
            bad[table[0, pos // PAGE].long(), 0, pos % PAGE, 3] = float("nan")
            got = run(q, bad, v, table, plan, SCALE)
            rows = slice(0, 2) if pos < 19904 else slice(0, 1)
            assert torch.isnan(got[rows, :8]).all() and torch.equal(got[:, 8:], clean[:, 8:]), (last, pos)
            if pos >= 19904:
                assert torch.equal(got[1], clean[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_nan_in_own_keys_of_one_cta_of_a_cluster(dtype):
    lens, spans = [3000], []
    q, k, v, table = far_apart(lens, spans, dtype, lambda pos: pos < 64)
    plan = build_shared_plan(lens, spans, HEADS, KV, DIM, dtype, PAGE).to(DEV)
    assert plan.host.cluster > 1
    clean = run(q, k, v, table, plan, SCALE)
    k[table[0, 2900 // PAGE].long(), 1, 2900 % PAGE, 3] = float("nan")
    got = run(q, k, v, table, plan, SCALE)
    assert torch.isfinite(clean).all() and torch.isnan(got[0, 8:]).all() and torch.equal(got[0, :8], clean[0, :8])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tile_rows", FORMS)
def test_nan_values_of_a_piece_that_weighs_nothing(dtype, tile_rows):
    """0 x NaN is NaN, in a piece of its own as in one tile."""
    lens, spans = [300, 290, 280], [([0, 1], 0, 256)]
    q, k, v, table = far_apart(lens, spans, dtype, lambda pos: pos >= 256)
    plan = build_shared_plan(lens, spans, HEADS, KV, DIM, dtype, PAGE, tile_rows=tile_rows).to(DEV)
    clean = run(q, k, v, table, plan, SCALE)
    v[table[0, 37 // PAGE].long(), 1, 37 % PAGE, 5] = float("nan")
    got = run(q, k, v, table, plan, SCALE)
    assert torch.isnan(got[:2, 8:, 5]).all()
    got[:2, 8:, 5], clean[:2, 8:, 5] = 0, 0
    assert torch.equal(got, clean)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tile_rows", FORMS)
def test_scratch_that_was_replaced_is_used(dtype, tile_rows):
    lens, spans = [300, 290, 280], [([0, 1], 0, 256)]
    q, k, v, table = case(lens, spans, HEADS, KV, DIM, PAGE, dtype)
    plan = build_shared_plan(lens, spans, HEADS, KV, DIM, dtype, PAGE, tile_rows=tile_rows).to(DEV)
    want = run(q, k, v, table, plan, SCALE)
    old = plan.part_o, plan.part_ml
    for t in old:
        t.fill_(5.0)
    plan.part_o, plan.part_ml = (torch.empty_like(t) for t in old)
    assert torch.equal(run(q, k, v, table, plan, SCALE), want)
    assert all((t == 5.0).all() for t in old)


@pytest.mark.gpu
def test_a_copy_of_a_plan_uses_what_it_was_given():
    """``dataclasses.replace`` with scratch of its own: the two may run at once."""
    lens, spans = [300, 290, 280], [([0, 1], 0, 256)]
    q, k, v, table = case(lens, spans, HEADS, KV, DIM, PAGE, BF16)
    plan = build_shared_plan(lens, spans, HEADS, KV, DIM, BF16, PAGE).to(DEV)
    want = run(q, k, v, table, plan, SCALE)
    other = dataclasses.replace(plan, part_o=torch.full_like(plan.part_o, 5.0), part_ml=torch.full_like(plan.part_ml, 5.0))
    plan.part_o.fill_(5.0)
    assert torch.equal(run(q, k, v, table, other, SCALE), want)
    assert (plan.part_o == 5.0).all() and not (other.part_o == 5.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_calls_of_different_sizes_from_two_threads(dtype):
    """A launch with room for many keys beside launches with room for few: none may take the other's room away."""
    sizes = [([2000] * 12, [(list(range(12)), 0, 1600)], DIM), ([40] * 12, [(list(range(12)), 0, 32)], DIM), ([300] * 3, [], 80), ([300] * 3, [], 96)]
    wrong = []
    ops.check_status()  # (the library is there)

    def calls(lens, spans, dim):
        try:
            q, k, v, table = [t.to(DEV) for t in case(lens, spans, HEADS, KV, dim, PAGE, dtype)]
            plan = build_shared_plan(lens, spans, HEADS, KV, dim, dtype, PAGE).to(DEV)
            stream = torch.cuda.Stream()
            stream.wait_stream(torch.cuda.default_stream())
            with torch.cuda.stream(stream):
                want, out = torch.empty_like(q), torch.empty_like(q)
                ops.shared_attention(q, k, v, table, plan, want, dim ** -0.5)
                for _ in range(3000):
                    ops.shared_attention(q, k, v, table, plan, out, dim ** -0.5)
                stream.synchronize()
            assert torch.equal(out, want)
        except Exception as e:
            wrong.append(repr(e))

    threads = [threading.Thread(target=calls, args=s) for s in sizes]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    ops.check_status()
    assert not wrong, wrong
