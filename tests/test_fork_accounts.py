"""What requests that share pages owe and hold, on the host: reservations, names, block-table changes that wait for a step."""

import random
from types import SimpleNamespace

import pytest
import torch

import fork_refs
from freetoken_b200.cache.manager import CacheManager
from freetoken_b200.cache.pages import PagePool
from freetoken_b200.config.spec import PagedKVNeed
from freetoken_b200.engine.engine import StepEntry
from freetoken_b200.engine.scheduler import Scheduler
from freetoken_b200.errors import CacheError, KernelError, SchedulerError
from freetoken_b200.kernels import ops
from freetoken_b200.sampling import Sampler, SamplingParams
from helpers import make_engine, model_folder, tokens_for
from plain.m3_plain import PlainM3
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


def ship(cache):
    for g in cache.paged:
        for at, page in cache.take_updates(g.index):
            g.table_dev.view(-1)[at] = page


def fork(cache, src, copies):
    for g, pairs in zip(cache.paged, cache.fork(src, copies).pages):
        rows = [(cache.requests[src].row, cache.requests[c].row) for c in copies]
        fork_refs.copy_slots([g.table_dev.unsqueeze(0)], torch.tensor(rows))


def grow(cache, rid, n):
    cache.begin_step([(rid, n)])
    ship(cache)
    cache.end_step()


def tables_agree(cache):
    cache.check()
    for r in cache.requests.values():
        blocks = -(-r.length // cache.page_size)
        for g in cache.paged:  # (what is given back is not read, and what waits for a step comes with it)
            wait = dict(g.updates)
            for b in range(blocks):
                page = int(g.table_host[r.row, b])
                assert not page or page == wait.get(r.row * g.width + b, int(g.table_dev[r.row, b]))


def cache_of(pages=40, reqs=4):
    return CacheManager([(0, PagedKVNeed((("k", 1, 2),), None))], 4, pages, reqs, 64, torch.float32, torch.device("cpu"), max_step_tokens=16)


@pytest.mark.parametrize("how", ["a step that did not run", "a fork that ended at once"])
def test_what_a_row_was_to_become_ends_with_its_request(how):
    """Changes of a block-table row that no step has carried yet must not reach the row's next owner, whose row a fork copies on the device."""
    cache = cache_of()
    cache.open("a")
    grow(cache, "a", 14)
    if how == "a step that did not run":
        cache.open("x")
        cache.begin_step([("x", 9)])
        cache.abort_step()
        cache.close("x")
    else:
        cache.open("y")
        grow(cache, "y", 6)
        cache.fork("y", ["x"])
        cache.close("x")
    fork(cache, "a", ["c"])  # on x's row
    ship(cache)
    tables_agree(cache)


def test_a_step_that_is_tried_again_writes_every_place_once():
    cache = cache_of()
    cache.open("a")
    cache.open("b")
    cache.begin_step([("a", 9), ("b", 7)])
    cache.abort_step()
    cache.begin_step([("b", 7), ("a", 9)])  # (other pages)
    updates = cache.take_updates(0)
    assert len({at for at, _ in updates}) == len(updates) == 5
    for at, page in updates:
        cache.paged[0].table_dev.view(-1)[at] = page
    cache.end_step()
    tables_agree(cache)


def test_what_a_failed_step_was_to_carry_goes_with_the_next():
    """A fork's own page waits for a step; where that step fails behind the point at which it took the changes, the next one takes them."""
    cache = cache_of()
    cache.open("a")
    grow(cache, "a", 14)
    fork(cache, "a", ["b"])
    cache.begin_step([("b", 3)])
    assert cache.take_updates(0)
    cache.abort_step()
    cache.begin_step([("a", 1)])
    ship(cache)
    cache.end_step()
    tables_agree(cache)
    grow(cache, "b", 5)
    tables_agree(cache)


def test_a_step_that_fails_before_its_launches_loses_no_pages(cpu, monkeypatch, tmp_path_factory):
    """Through the engine: a fork, a step that fails while its metadata is made, and then the continuation's logits."""
    folder = model_folder(tmp_path_factory.getbasetemp(), "A", ALL["A"])
    plain = PlainM3(folder)
    V = plain.cfg.vocab
    eng = make_engine(folder, "float32", "cpu", 4, pages=40, reqs=4)
    a = tokens_for(V, 14, 1)
    eng.step([StepEntry("a", a)])
    eng.fork("a", ["b"])
    upload = eng.buffers.upload

    def fails(sections):
        raise RuntimeError("no room")

    monkeypatch.setattr(eng.buffers, "upload", fails)
    with pytest.raises(RuntimeError):
        eng.step([StepEntry("b", [5], [0])])
    monkeypatch.setattr(eng.buffers, "upload", upload)
    eng.step([StepEntry("a", [7], [0])])  # (the parent goes on in its last page: the fork must not read that)
    got = eng.step([StepEntry("b", [5], [0])]).logits
    torch.testing.assert_close(got[0], plain.logits(a + [5])[-1], rtol=1e-4, atol=2e-5)
    got = eng.step([StepEntry("b", [6], [0])]).logits
    torch.testing.assert_close(got[0], plain.logits(a + [5, 6])[-1], rtol=1e-4, atol=2e-5)


def test_a_fork_whose_copies_fail_opens_nobody(cpu, monkeypatch, tmp_path_factory):
    folder = model_folder(tmp_path_factory.getbasetemp(), "A", ALL["A"])
    eng = make_engine(folder, "float32", "cpu", 4, pages=40, reqs=4)
    eng.step([StepEntry("a", tokens_for(eng.spec.vocab_size, 14, 1))])
    before = eng.cache.free_pages(), eng.cache.free_request_slots()

    def refused(*args):
        raise KernelError("tensor is on 'cuda:0', the current device is 'cuda:1'")

    for name in ("copy_pages", "copy_slots"):
        with monkeypatch.context() as m:
            m.setattr(ops, name, refused)
            with pytest.raises(KernelError):
                eng.fork("a", ["b", "c"])
        eng.cache.check()
        assert not eng.is_open("b") and not eng.is_open("c") and (eng.cache.free_pages(), eng.cache.free_request_slots()) == before
    eng.fork("a", ["b", "c"])
    eng.cache.check()


class Spied:
    """A table that counts what is taken out of it."""

    def __init__(self, table):
        self.table, self.taken = table, 0

    def __getitem__(self, at):
        out = self.table[at]
        self.taken += out.size
        return out


def test_tables_are_compared_only_while_pages_are_shared_and_only_as_far_as_they_reach():
    cache = cache_of(reqs=6)
    for rid, n in (("a", 9), ("b", 14), ("c", 3)):
        cache.open(rid)
        grow(cache, rid, n)
    group = cache.paged[0]
    table, group.table_host = group.table_host, Spied(group.table_host)
    spy = group.table_host
    assert cache.shared_spans(group, ["a", "b", "c"]) == [] and not spy.taken and not cache.sharing
    group.table_host = table
    fork(cache, "b", ["d"])
    group.table_host = spy
    assert cache.sharing and cache.shared_spans(group, ["a", "b", "c", "d"]) == [([1, 3], 0, 12)]
    assert 0 < spy.taken <= 4 * 3  # (three full pages at most; a row of the table has 16)
    group.table_host = table
    cache.close("b")  # one holder is left
    spy.taken, group.table_host = 0, spy
    assert cache.shared_spans(group, ["a", "c", "d"]) == [] and not spy.taken and not cache.sharing
    group.table_host = table
    cache.check()
    for rid in "acd":
        cache.close(rid)
    cache.check()


def test_pages_of_several_holders_are_counted():
    pool = PagePool(4)
    a, b = pool.alloc(2)
    pool.share([a, b, a])
    assert pool.shared == 2
    pool.free([a])
    assert pool.shared == 2
    pool.free([a, b])
    pool.check([a, b])
    assert pool.shared == 0
    pool.share([b])
    pool.renumber({b: 3})
    assert pool.shared == 1
    pool.free([3, 3, a])
    assert pool.shared == 0 and pool.free_count == 4


class HostEngine:
    """What the scheduler asks of an engine, on block tables alone: full pages, a window, a window that keeps its first tokens."""

    NEEDS = [(0, PagedKVNeed((("k", 1, 2),), None)), (1, PagedKVNeed((("k", 1, 2),), 7)), (2, PagedKVNeed((("k", 1, 2),), 9, 5))]

    def __init__(self, pages, reqs, step):
        self.cache = CacheManager(self.NEEDS, 4, pages, reqs, 96, torch.float32, torch.device("cpu"), max_step_tokens=step)
        self.config = SimpleNamespace(max_running_req=reqs, max_extend_tokens=step, overlap_scheduling=True)
        self.spec = SimpleNamespace(vocab_size=50)
        self.max_step_tokens, self.max_seq_len = step, 96
        self.open, self.close = self.cache.open, self.cache.close

    def fork(self, rid, copies):
        fork(self.cache, rid, copies)

    def step(self, entries):
        self.cache.begin_step([(e.request_id, len(e.tokens)) for e in entries])
        ship(self.cache)
        self.cache.end_step()
        rows = [(e.request_id, w) for e in entries for w in e.want]
        return SimpleNamespace(rows=rows, logits=torch.zeros(len(rows), 1))


class HostSampler:
    def __init__(self, rng, eos):
        self.rng, self.eos = rng, eos

    def launch(self, logits, params, requests, steps, rows=None):
        assert len(params) == len(requests) == len(steps) == (logits.shape[0] if rows is None else len(rows))
        return SimpleNamespace(device_tokens=torch.zeros(1), tokens=[0 if self.rng.random() < self.eos else 5 for _ in params])

    def result(self, ticket):
        return ticket.tokens


@pytest.mark.parametrize("overlap", [False, True])
@pytest.mark.parametrize("seed", range(12))
def test_admitted_requests_always_find_their_pages(seed, overlap):
    """Random prompts, continuations, ends and aborts in a small cache of three kinds of groups."""
    rng = random.Random(seed)
    eng = HostEngine(pages=rng.choice([26, 34, 50]), reqs=rng.choice([4, 6, 9]), step=rng.choice([8, 16]))
    sched = Scheduler(eng, HostSampler(rng, rng.choice([0.0, 0.1, 0.3])), (0,))
    wanted = {}
    for i in range(40):
        n = rng.choice([1, 1, 2, 3, 4])
        wanted[i] = n
        sched.add_request([1] * rng.randint(1, 60), SamplingParams(max_tokens=rng.randint(1, 30), n=n, temperature=1.0), rid=i)
    while not sched.idle:
        sched.step_overlapped() if overlap else sched.step()
        eng.cache.check()
        if rng.random() < 0.1:
            tables_agree(eng.cache)
        assert all(h <= r <= p for h, r, p in zip([g.pool.num_pages - g.pool.free_count for g in eng.cache.paged], sched.reserved, sched.pool_pages))
        assert len(sched.running) <= sched.max_running
        if rng.random() < 0.1 and sched.running:
            sched.abort(rng.choice(sched.running).rid)
    sched.drain()
    assert sched.reserved == [0, 0, 0] and all(g.pool.free_count == g.pool.num_pages for g in eng.cache.paged)
    assert set(wanted) <= set(sched.done) and any(r.continues for r in sched.done.values())
