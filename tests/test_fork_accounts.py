"""What requests that share pages owe and hold, on the host: reservations, names, block-table changes that wait for a step."""

import pytest
import torch

import fork_refs
from freetoken_b200.engine.scheduler import Scheduler
from freetoken_b200.errors import CacheError, SchedulerError
from freetoken_b200.sampling import Sampler, SamplingParams
from helpers import make_engine, model_folder, tokens_for
from tiny_configs import ALL


@pytest.fixture
def cpu(monkeypatch):
    fork_refs.install(monkeypatch)


def scheduler(tmp_path_factory, name="A", reqs=4, pages=20, max_step=16):
    folder = model_folder(tmp_path_factory.getbasetemp(), name, ALL[name])
    eng = make_engine(folder, "float32", "cpu", 4, pages, max_step=max_step, reqs=reqs)
    return Scheduler(eng, Sampler(eng.device, eng.spec.vocab_size, reqs), ())


def held(sched):
    return [g.pool.num_pages - g.pool.free_count for g in sched.engine.cache.paged]


@pytest.mark.parametrize("name", ["A", "B"])
@pytest.mark.parametrize("overlap", [False, True])
@pytest.mark.parametrize("order", [[0, 1, 2], [2, 0, 1], [1, 2, 0]])
@pytest.mark.parametrize("how", ["abort", "end"])
def test_pages_of_a_prompt_stay_reserved_while_a_continuation_holds_them(how, order, overlap, name, cpu, tmp_path_factory):
    """The members of a family end one after the other, the one that read the prompt first, in the middle or last; a request that needs
    most of the pool waits and must not be let in on pages that the others still hold."""
    sched = scheduler(tmp_path_factory, name)
    V = sched.engine.spec.vocab_size
    names = [0, (0, 1), (0, 2)]
    family = [names[i] for i in order]
    # 10 full pages of prompt, 3 more for each: 19 of 20
    sched.add_request(tokens_for(V, 40, 1), SamplingParams(max_tokens=12, temperature=1.0, seed=1, n=3), rid=0)
    sched.add_request(tokens_for(V, 40, 2), SamplingParams(max_tokens=12, temperature=1.0, seed=2), rid="later")
    step = sched.step_overlapped if overlap else sched.step
    ends, wait = iter(family[:2]), None
    while not sched.idle:
        step()
        assert all(h <= r for h, r in zip(held(sched), sched.reserved)), (held(sched), sched.reserved)
        assert all(r <= p for r, p in zip(sched.reserved, sched.pool_pages))
        sched.engine.cache.check()
        live = {r.rid: r for r in sched.running}
        if wait is None and all(n in live and live[n].output for n in names):
            wait = 0
        if wait is not None:
            wait += 1
        if wait in (1, 4):
            rid = next(ends)
            if how == "abort":
                assert sched.abort(rid)
            else:  # (its next token is its last)
                live[rid].max_tokens = len(live[rid].output) + live[rid].in_flight + 1
    sched.drain()
    assert sched.reserved == [0] * len(sched.reserved) and held(sched) == [0] * len(sched.reserved)
    assert sched.done["later"].finish_reason == "length" and all(n in sched.done for n in names)


def test_the_name_of_a_running_continuation_is_refused(cpu, tmp_path_factory):
    sched = scheduler(tmp_path_factory, pages=40)
    V = sched.engine.spec.vocab_size
    several, one = SamplingParams(max_tokens=6, temperature=1.0, seed=1, n=2), SamplingParams(max_tokens=3)
    sched.add_request(tokens_for(V, 5, 1), several, rid="a")
    sched.step()
    assert {r.rid for r in sched.running} == {"a", ("a", 1)}
    for params in (one, several):
        with pytest.raises(SchedulerError, match="name"):
            sched.add_request(tokens_for(V, 5, 2), params, rid=("a", 1))
    sched.run()
    assert sched.reserved == [0]
    sched.add_request(tokens_for(V, 5, 2), one, rid=("a", 1))  # free again
    sched.run()
    assert len(sched.done[("a", 1)].output) == 3 and sched.reserved == [0]


def test_a_request_that_cannot_be_opened_stays_in_line(cpu, tmp_path_factory):
    """Under the name of one that runs: nothing is reserved for it and it is not lost."""
    sched = scheduler(tmp_path_factory, pages=40)
    V = sched.engine.spec.vocab_size
    sched.add_request(tokens_for(V, 5, 1), SamplingParams(max_tokens=6), rid="a")
    sched.step()
    before = list(sched.reserved)
    sched.add_request(tokens_for(V, 5, 2), SamplingParams(max_tokens=3), rid="a")
    with pytest.raises(CacheError, match="already open"):
        sched.step()
    assert sched.reserved == before and len(sched.waiting) == 1
    assert sched.abort("a") and not sched.waiting  # (those in line first)
    sched.run()
    assert len(sched.done["a"].output) == 6 and sched.reserved == [0]
