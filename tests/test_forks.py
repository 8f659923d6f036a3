"""Requests that continue one prompt, on the host: holders of pages, what a fork copies, who shares what, the scheduler's decisions.
Kernels are replaced by their plain statements."""

import random

import pytest
import torch

import fork_refs
from freetoken_b200.cache.manager import CacheManager
from freetoken_b200.cache.pages import PagePool
from freetoken_b200.config.spec import PagedKVNeed, StateNeed
from freetoken_b200.engine.engine import StepEntry
from freetoken_b200.engine.scheduler import Scheduler
from freetoken_b200.errors import CacheError, ConfigError, SchedulerError
from freetoken_b200.kernels import ops
from freetoken_b200.parts.attention import sharing_pays
from freetoken_b200.sampling import Sampler, SamplingParams
from helpers import make_engine, model_folder, tokens_for
from plain.m3_plain import PlainM3
from tiny_configs import ALL, TINY_A


def test_a_page_goes_back_with_its_last_holder():
    pool = PagePool(3)
    a, b = pool.alloc(2)
    pool.share([a])
    pool.share([a, b])
    pool.check([a, a, a, b, b])
    for held, what in ([a, a, b, b], "holders"), ([a, a, a, a, b, b], "twice"), ([a, a, a], "lost"):
        with pytest.raises(CacheError, match=what):
            pool.check(held)
    pool.free([a, a, b])
    assert pool.free_count == 1 and pool.holders(a) == 1
    pool.free([a, b])
    assert pool.free_count == 3
    with pytest.raises(CacheError, match="twice"):
        pool.free([a])
    with pytest.raises(CacheError, match="nobody"):
        pool.share([b])


NEEDS = [(0, PagedKVNeed((("k", 1, 2), ("v", 1, 2)), None)), (1, PagedKVNeed((("k", 1, 2),), 7)), (2, PagedKVNeed((("k", 1, 2),), 9, 5)),
         (3, StateNeed((("s", (2,), "float32"),)))]


def manager(pages=60, reqs=7):
    return CacheManager(NEEDS, 4, pages, reqs, 64, torch.float32, torch.device("cpu"), max_step_tokens=12)


@pytest.mark.parametrize("seed", range(12))
def test_contents_survive_any_order_of_steps_forks_ends_and_moves(seed):
    """Every request's cached tokens are written through its block table and must be read back, whoever shares what."""
    rng = random.Random(seed)
    cache = manager(pages=rng.choice([60, 70]))
    names, written, nth = iter(range(10 ** 6)), {}, iter(range(1, 10 ** 6))

    def write(rid, tokens, plan, t0):
        for g in cache.paged:
            for i, tok in enumerate(tokens):
                slot = int(plan.slot_maps[g.index][t0 + i])
                if slot >= 0:
                    for slab in g.slabs.values():
                        slab[:, slot // 4, :, slot % 4] = tok

    def ship():  # (what steps do with block-table changes)
        for g in cache.paged:
            for at, page in cache.take_updates(g.index):
                g.table_dev.view(-1)[at] = page

    def read_all():
        cache.check()
        for rid, toks in written.items():
            row = cache.requests[rid].row
            for g in cache.paged:
                first = 0 if g.need.window is None else max(0, len(toks) - g.need.window + 1)
                for pos in [p for p in range(len(toks)) if p >= first or p < g.need.keep_first]:
                    page = int(g.table_host[row, pos // 4])
                    assert page and page == int(g.table_dev[row, pos // 4])
                    for slab in g.slabs.values():
                        assert (slab[:, page, :, pos % 4] == toks[pos]).all(), (rid, g.index, pos)
            if toks:  # (a request that has read nothing starts from zeros, whatever its slot holds)
                assert (cache.state[0].tensors["s"][:, cache.requests[rid].state_slot] == sum(toks)).all()

    for _ in range(120):
        what = rng.random()
        if what < 0.45 or not written:
            step = []
            if cache.free_request_slots() and (not written or rng.random() < 0.3):
                rid = next(names)
                cache.open(rid)
                written[rid] = []
            for rid in rng.sample(sorted(written), rng.randint(1, len(written))):
                n = rng.choice([1, 1, 1, 3, 6])
                if len(written[rid]) + n <= 64 and sum(k for _, k in step) + n <= 12:
                    step.append((rid, n))
            if not step:
                continue
            try:
                plan = cache.begin_step(step)
            except CacheError as e:
                assert "out of pages" in str(e)
                cache.check()
                continue
            if rng.random() < 0.1:
                cache.abort_step()
                ship()
                continue
            t0 = 0
            for rid, n in step:
                toks = [next(nth) for _ in range(n)]
                write(rid, toks, plan, t0)
                written[rid] += toks
                cache.state[0].tensors["s"][:, cache.requests[rid].state_slot] = sum(written[rid])
                t0 += n
            ship()
            cache.end_step()
        elif what < 0.7 and written:
            src = rng.choice(sorted(written))
            copies = [next(names) for _ in range(rng.randint(1, 3))]
            before = cache.free_pages(), cache.free_request_slots()
            try:
                made = cache.fork(src, copies)
            except CacheError:
                assert (cache.free_pages(), cache.free_request_slots()) == before
                continue
            for g, pairs in zip(cache.paged, made.pages):
                fork_refs.copy_pages(list(g.slabs.values()), torch.tensor(pairs or [(0, 0, 0)]))
                fork_refs.copy_slots([g.table_dev.unsqueeze(0)], torch.tensor(made.rows))
            fork_refs.copy_slots([cache.state[0].tensors["s"]], torch.tensor(made.slots))
            ship()
            for c in copies:
                written[c] = list(written[src])
        elif what < 0.9 and written:
            rid = rng.choice(sorted(written))
            cache.close(rid)
            del written[rid]
        else:
            for g, pairs in zip(cache.paged, cache.compact()):
                assert not {a for a, _, _ in pairs} & {b for _, b, _ in pairs}
                fork_refs.copy_pages(list(g.slabs.values()), torch.tensor(pairs or [(0, 0, 0)]))
                used = g.pool.num_pages - g.pool.free_count
                assert g.table_host.max(initial=0) <= used  # the lowest numbers
        read_all()
    for rid in list(written):
        cache.close(rid)
    cache.check()
    assert all(g.pool.free_count == g.pool.num_pages for g in cache.paged)


def test_spans_of_nested_forks():
    cache = manager()
    grow = lambda step: (cache.begin_step(step), cache.end_step())  # noqa: E731
    cache.open("a")
    grow([("a", 10)])                 # two full pages
    cache.fork("a", ["b", "c"])
    grow([("b", 5)])                  # 15: a page of its own is full
    cache.fork("b", ["d"])
    cache.open("x")
    grow([("x", 12)])
    full = cache.paged[0]
    spans = cache.shared_spans(full, ["x", "d", "a", "b", "c"])
    assert [(sorted(m), s, e) for m, s, e in spans] == [([1, 2, 3, 4], 0, 8), ([1, 3], 8, 12)]
    assert cache.shared_spans(full, ["x", "d", "a", "b", "c"]) is spans  # kept
    assert cache.shared_spans(full, ["x", "c"]) == [] and cache.shared_spans(full, ["c", "d"]) == [([0, 1], 0, 8)]
    assert cache.shared_spans(cache.paged[1], ["a", "b"]) == []  # a window
    cache.close("b")
    assert cache.shared_spans(full, ["d", "a"]) == [([0, 1], 0, 8)]
    cache.close("d")
    cache.close("a")
    assert cache.shared_spans(full, ["c", "x"]) == []


def test_forks_are_refused_whole():
    cache = manager(pages=8, reqs=4)
    cache.open("a")
    cache.begin_step([("a", 6)])
    with pytest.raises(CacheError, match="in flight"):
        cache.fork("a", ["b"])
    cache.end_step()
    for copies, what in (["b", "b"], "names"), (["a"], "names"), (["b", "c", "d", "e"], "slots"):
        with pytest.raises(CacheError, match=what):
            cache.fork("a", copies)
    with pytest.raises(CacheError, match="not open"):
        cache.fork("z", ["b"])
    cache.open("p")
    cache.begin_step([("p", 12)])
    cache.end_step()
    cache.open("o")
    cache.begin_step([("o", 12)])
    cache.end_step()
    with pytest.raises(CacheError, match="out of pages"):
        cache.fork("a", ["b"])
    cache.check()
    cache.fork("p", ["b"])  # full pages alone: nothing to take
    cache.check()


@pytest.fixture
def cpu(monkeypatch):
    fork_refs.install(monkeypatch)


@pytest.mark.parametrize("name", ["A", "B", "D"])
def test_forked_requests_give_the_plain_models_logits(name, cpu, monkeypatch, tmp_path_factory):
    """A prompt, forks of it, a fork of a fork: every continuation's logits are those of its whole sequence, and steps that share read the
    shared pages through the shared list (block-sparse layers do not)."""
    calls = []
    monkeypatch.setattr("freetoken_b200.parts.attention.SHARED_MIN_KEYS", 1)
    monkeypatch.setattr("freetoken_b200.parts.attention.SHARED_MIN_KEYS_EACH", 0)
    monkeypatch.setattr("freetoken_b200.parts.attention.SHARED_MOST_OWN", 1e9)
    monkeypatch.setattr(ops, "shared_attention", lambda *a, **k: (calls.append(1), fork_refs.shared_attention(*a, **k))[1])
    folder = model_folder(tmp_path_factory.getbasetemp(), name, ALL[name])
    plain = PlainM3(folder)
    V = plain.cfg.vocab
    eng = make_engine(folder, "float32", "cpu", 4, pages=60, reqs=6)
    seqs = {"a": tokens_for(V, 13, 1)}
    eng.step([StepEntry("a", seqs["a"])])
    eng.fork("a", ["b", "c"])
    seqs["b"], seqs["c"] = list(seqs["a"]), list(seqs["a"])
    eng.step([StepEntry("o", tokens_for(V, 5, 9))])
    seqs["o"] = tokens_for(V, 5, 9)
    for t in range(9):
        if t == 5:
            eng.fork("c", ["d"])
            seqs["d"] = list(seqs["c"])
        if t == 7:
            eng.close("a")
            del seqs["a"]
            eng.compact()
        entries = []
        for i, r in enumerate(sorted(seqs)):
            tok = tokens_for(V, 1, 100 * i + t)
            seqs[r] = seqs[r] + tok
            entries.append(StepEntry(r, tok, [0]))
        got = eng.step(entries).logits
        for row, r in zip(got, sorted(seqs)):
            torch.testing.assert_close(row, plain.logits(seqs[r])[-1], rtol=1e-4, atol=2e-5)
    assert calls
    for r in list(seqs):
        eng.close(r)
    assert all(g.pool.free_count == g.pool.num_pages for g in eng.cache.paged)


def scheduler(tmp_path_factory, reqs=4, pages=40, eos=(), **kw):
    folder = model_folder(tmp_path_factory.getbasetemp(), "A", TINY_A)
    eng = make_engine(folder, "float32", "cpu", 4, pages, max_step=16, reqs=reqs, **kw)
    return Scheduler(eng, Sampler(eng.device, eng.spec.vocab_size, reqs), eos), PlainM3(folder)


@pytest.mark.parametrize("overlap", [False, True])
def test_continuations_are_what_requests_of_their_names_give(overlap, cpu, tmp_path_factory):
    """n continuations draw as separate requests with the same names, seed and parameters do."""
    sched, plain = scheduler(tmp_path_factory, reqs=6)
    V = plain.cfg.vocab
    prompts = [tokens_for(V, 11, 1), tokens_for(V, 8, 2), tokens_for(V, 21, 3)]
    sp = [SamplingParams(max_tokens=7, temperature=0.9, top_p=0.95, seed=5, n=3), SamplingParams(max_tokens=5, temperature=0.7, seed=5),
          SamplingParams(max_tokens=6, temperature=1.1, seed=5, min_p=0.02, n=2)]
    for i, (p, s) in enumerate(zip(prompts, sp)):
        sched.add_request(p, s, rid=i)
    while not sched.idle:
        sched.step_overlapped() if overlap else sched.step()
        sched.engine.cache.check()
        assert all(x <= p for x, p in zip(sched.reserved, sched.pool_pages))
        assert len(sched.running) <= 6
    sched.drain()
    assert sched.reserved == [0] and sched.engine.cache.free_request_slots() == 6
    names = {0: [0, (0, 1), (0, 2)], 1: [1], 2: [2, (2, 1)]}
    alone, _ = scheduler(tmp_path_factory, reqs=6)
    for i, group in names.items():
        for rid in group:
            s = sp[i]
            alone.add_request(prompts[i], SamplingParams(max_tokens=s.max_tokens, temperature=s.temperature, top_p=s.top_p, seed=5,
                                                         min_p=s.min_p or (1e-30 if s.n > 1 else 0.0)), rid=rid)
            alone.run(overlap=False)
            assert sched.done[rid].output == alone.done[rid].output, rid
            if i != 1:
                assert sched.done[rid].logprob == pytest.approx(alone.done[rid].logprob, abs=1e-4) and sched.done[rid].logprob < 0
            else:
                assert sched.done[rid].logprob is None
    assert len({tuple(sched.done[r].output) for r in names[0]}) > 1


def test_log_probabilities_are_the_models(cpu, tmp_path_factory):
    sched, plain = scheduler(tmp_path_factory)
    p = tokens_for(plain.cfg.vocab, 9, 4)
    sched.add_request(p, SamplingParams(max_tokens=5, temperature=0.8, top_k=30, seed=1, n=2), rid=0)
    sched.run()
    for rid in (0, (0, 1)):
        out = sched.done[rid].output
        logs = torch.log_softmax(plain.logits(p + out), -1)
        want = sum(float(logs[len(p) - 1 + i, t]) for i, t in enumerate(out))
        assert sched.done[rid].logprob == pytest.approx(want, abs=1e-3)


def test_admission_counts_continuations(cpu, tmp_path_factory):
    sched, plain = scheduler(tmp_path_factory, reqs=4, pages=14)
    V = plain.cfg.vocab
    too_many = sched.add_request(tokens_for(V, 4, 0), SamplingParams(max_tokens=2, n=5))
    assert "continuations" in sched.done[too_many].error
    # prompt of 10 (2 full pages), 6 more tokens: 4 pages, and 2 for each further continuation
    a = sched.add_request(tokens_for(V, 10, 1), SamplingParams(max_tokens=6, temperature=0.5, n=3), rid="a")
    b = sched.add_request(tokens_for(V, 10, 2), SamplingParams(max_tokens=6, temperature=0.5, n=2), rid="b")
    c = sched.add_request(tokens_for(V, 3, 3), SamplingParams(max_tokens=2), rid="c")
    rep = sched.step()
    assert rep.admitted == [a] and sched.reserved == [8]  # two slots more than are free (first in, first out)
    big = sched.add_request(tokens_for(V, 10, 4), SamplingParams(max_tokens=30, n=4), rid="big")  # 10 + 3 * 8 pages
    assert "pages" in sched.done[big].error
    sched.run()
    assert all(sched.done[r].finish_reason == "length" for r in ("a", ("a", 1), ("a", 2), "b", ("b", 1), "c"))
    assert sched.reserved == [0]


def test_ends_and_aborts_of_single_continuations(cpu, tmp_path_factory):
    sched, plain = scheduler(tmp_path_factory, reqs=4)
    V = plain.cfg.vocab
    p = tokens_for(V, 11, 1)
    sched.add_request(p, SamplingParams(max_tokens=8, temperature=1.5, seed=2, n=4), rid=0)
    sched.run()
    outs = {r: sched.done[r].output for r in (0, (0, 1), (0, 2), (0, 3))}
    again, _ = scheduler(tmp_path_factory, reqs=4)
    again.eos = {outs[(0, 2)][3]}
    again.add_request(p, SamplingParams(max_tokens=8, temperature=1.5, seed=2, n=4), rid=0)
    for _ in range(3):
        again.step()
    assert again.abort((0, 1)) and again.done[(0, 1)].finish_reason == "abort"
    again.run()
    for r in (0, (0, 2), (0, 3)):
        cut = next((i + 1 for i, t in enumerate(outs[r]) if t in again.eos), 8)
        assert again.done[r].output == outs[r][:cut]
    assert again.reserved == [0] and all(g.pool.free_count == g.pool.num_pages for g in again.engine.cache.paged)
    waiting, _ = scheduler(tmp_path_factory, reqs=4)
    waiting.add_request(tokens_for(V, 40, 1), SamplingParams(max_tokens=4, temperature=1.0, n=3), rid=0)
    waiting.step()  # a portion of the prompt: not forked yet
    assert waiting.abort(0) and waiting.reserved == [0] and waiting.engine.cache.free_request_slots() == 4


def test_parameters():
    for bad in (dict(n=0), dict(min_p=-0.1), dict(min_p=1.5)):
        with pytest.raises(ConfigError):
            SamplingParams(**bad)
    assert not SamplingParams(temperature=1.0, top_p=0.5).draws and SamplingParams(n=2).draws and SamplingParams(min_p=0.1).draws


def test_the_sampler_keeps_requests_that_do_not_draw_as_they_are(cpu, monkeypatch):
    """Beside draws, the other requests' tokens come from the same call with the same numbers as without them."""
    torch.manual_seed(0)
    logits = torch.randn(4, 50) * 3
    sp = SamplingParams(temperature=0.9, top_p=0.8, top_k=20, seed=3)
    sampler = Sampler(torch.device("cpu"), 50, 4)
    alone = sampler.sample(logits, [sp] * 4, list("abcd"), [0] * 4)
    drawing = SamplingParams(temperature=0.9, seed=3, min_p=0.05)
    seen = []
    monkeypatch.setattr(ops, "sample", lambda *a: (seen.append(1), kernel_refs_sample(*a))[1])
    from kernel_refs import sample as kernel_refs_sample
    mixed = [sp, drawing, sp, drawing]
    ticket = sampler.launch(logits, mixed, list("abcd"), [0] * 4)
    got = sampler.result(ticket)
    assert [got[0], got[2]] == [alone[0], alone[2]] and seen
    logs = torch.log_softmax(logits, -1)
    assert sampler.logprobs(ticket) == [None, pytest.approx(float(logs[1, got[1]]), abs=1e-5), None, pytest.approx(float(logs[3, got[3]]), abs=1e-5)]
    many = sampler.launch(logits[:2], [SamplingParams(temperature=1.0, seed=1, n=3)] * 3 + [SamplingParams()], ["a", "b", "c", "d"], [0] * 4, rows=[0, 0, 0, 1])
    toks = sampler.result(many)
    assert toks[3] == int(logits[1].argmax()) and len(toks) == 4
    for bad in ([0, 0, 5, 1], [0, 0, -1, 1]):
        with pytest.raises(ValueError):
            sampler.launch(logits[:2], [SamplingParams(n=3)] * 4, list("abcd"), [0] * 4, rows=bad)
    with pytest.raises(ValueError):
        sampler.launch(logits[:2], [SamplingParams()] * 2, list("ab"), [0] * 2, rows=[1, 1])


def test_names_of_continuations_are_refused_to_others(cpu, tmp_path_factory):
    sched, _ = scheduler(tmp_path_factory, reqs=6, pages=64)
    several, one = SamplingParams(max_tokens=4, n=3, temperature=1.0, ignore_eos=True), SamplingParams(max_tokens=4, ignore_eos=True)
    sched.add_request([1, 2, 3], several, rid="a")
    for rid, params in ((("a", 2), one), (("a", 1), several)):
        with pytest.raises(SchedulerError, match="name"):
            sched.add_request([5], params, rid=rid)
    sched.add_request([5, 6], one, rid=("a", 3))  # nobody's
    sched.add_request([5, 6], one, rid=("b", 1))
    with pytest.raises(SchedulerError, match="name"):
        sched.add_request([5], several, rid="b")
    sched.run()
    assert all(len(sched.done[r].output) == 4 for r in ("a", ("a", 1), ("a", 2), ("a", 3), ("b", 1)))


def test_sharing_is_used_where_it_pays(cpu, monkeypatch, tmp_path_factory):
    pays = lambda n, shared, own, kv=8, dim=128, dt=torch.bfloat16: sharing_pays((n - 1) * shared, n * own, n, kv, dim, dt)  # noqa: E731
    # the figures beside the rule: who is faster there
    assert [pays(16, x, 60) for x in (64, 1024, 16384)] == [False, True, True] and [pays(48, x, 60) for x in (64, 256, 16384)] == [False, True, True]
    assert [pays(4, 16384, x) for x in (500, 2000, 4000, 16000)] == [True, True, False, False]
    assert [pays(16, 2048, x) for x in (1000, 2000)] == [True, False] and [pays(2, 16384, x) for x in (500, 2000)] == [True, False]
    assert [pays(4, 16384, x, 4, 64) for x in (4000, 16000)] == [True, False] and [pays(4, 2048, x, 4, 64, torch.float32) for x in (1000, 2000)] == [True, False]
    # and what a step says of itself: two of three requests share 8 keys, the third is long
    folder = model_folder(tmp_path_factory.getbasetemp(), "A", TINY_A)
    eng = make_engine(folder, "float32", "cpu", 4, 40, max_step=64, reqs=4)
    eng.step([StepEntry("a", list(range(1, 11)))])
    eng.step([StepEntry("c", list(range(1, 31)))])
    eng.fork("a", ["b"])
    seen = []
    monkeypatch.setattr("freetoken_b200.parts.attention.sharing_pays", lambda *a: seen.append(a) or False)
    eng.step([StepEntry("a", [3], [0]), StepEntry("b", [4], [0]), StepEntry("c", [5], [0])])
    assert seen and all(a[:3] == (8, 3 + 3 + 31, 3) for a in seen)


def test_lists_that_have_no_room_are_not_made(cpu, monkeypatch, tmp_path_factory):
    """A chain of forks, each of the one before: the list over what they share grows with the square of its length."""
    for name, value in (("SHARED_MIN_KEYS", 1), ("SHARED_MIN_KEYS_EACH", 0), ("SHARED_MOST_OWN", 1e9)):
        monkeypatch.setattr(f"freetoken_b200.parts.attention.{name}", value)
    calls = []
    monkeypatch.setattr(ops, "shared_attention", lambda *a, **k: (calls.append(1), fork_refs.shared_attention(*a, **k))[1])
    folder = model_folder(tmp_path_factory.getbasetemp(), "A", TINY_A)
    plain = PlainM3(folder)
    eng = make_engine(folder, "float32", "cpu", 4, 300, max_step=64, reqs=12)
    seqs = {0: tokens_for(plain.cfg.vocab, 4, 1)}
    eng.step([StepEntry(0, seqs[0])])
    for i in range(1, 12):
        more = tokens_for(plain.cfg.vocab, 4, i)
        eng.fork(i - 1, [i])
        seqs[i] = seqs[i - 1] + more
        eng.step([StepEntry(i, more)])
    for room in (eng.plan_ints, 300):
        eng.plan_ints, before = room, len(calls)
        entries = []
        for r in seqs:
            seqs[r] = seqs[r] + [r + 1]
            entries.append(StepEntry(r, [r + 1], [0]))
        got = eng.step(entries).logits
        assert (len(calls) > before) == (room > 300)
        for row, r in zip(got, seqs):
            torch.testing.assert_close(row, plain.logits(seqs[r])[-1], rtol=1e-4, atol=2e-5)
