"""Requests that continue one prompt, through the engine on the GPU: fork, decode steps over shared pages, draws."""

import pytest
import torch

import fork_refs
from freetoken_b200 import LLM, SamplingParams
from freetoken_b200.engine.engine import StepEntry
from freetoken_b200.engine.scheduler import Scheduler
from freetoken_b200.kernels import ops
from freetoken_b200.sampling import Sampler, uniform_for
from helpers import F32_TOL, bf16_tol, make_engine, model_folder, tokens_for
from plain.m3_plain import PlainM3
from tiny_configs import ALL
from tiny_gizulorn import ALL as GIZULORN
from tiny_kekopel import ALL as KEKOPEL
from tiny_nusudra import ALL as NUSUDRA
from tiny_pabavik import ALL as PABAVIK
from tiny_vodatar import ALL as VODATAR

OTHERS = {f"{m}-{n}": raw for m, every in (("gizulorn", GIZULORN), ("kekopel", KEKOPEL), ("nusudra", NUSUDRA), ("pabavik", PABAVIK), ("vodatar", VODATAR))
          for n, raw in list(every.items())[:1]}


@pytest.fixture
def sharing(monkeypatch):
    """Every decode step whose requests share a page takes the shared list; how often that was."""
    monkeypatch.setattr("freetoken_b200.parts.attention.SHARED_MIN_KEYS", 1)
    monkeypatch.setattr("freetoken_b200.parts.attention.SHARED_MIN_KEYS_EACH", 0)
    monkeypatch.setattr("freetoken_b200.parts.attention.SHARED_MOST_OWN", 1e9)
    ops.variant_counts(reset=True)
    return lambda: {k: v for k, v in ops.variant_counts().items() if k.startswith("shared attention")}


def decode(eng, seqs, steps, V, seed, after=None):
    """Random next tokens for every request; logits of every step, per request."""
    got = {r: [] for r in seqs}
    for t in range(steps):
        if after is not None:
            after(t)
        names = sorted(seqs)
        entries = []
        for i, r in enumerate(names):
            got.setdefault(r, [])
            tok = tokens_for(V, 1, seed + 1000 * i + t)
            seqs[r] = seqs[r] + tok
            entries.append(StepEntry(r, tok, [0]))
        logits = eng.step(entries).logits.float().cpu()
        for row, r in zip(logits, names):
            got[r].append(row.clone())
    return {r: torch.stack(v) for r, v in got.items() if v}


@pytest.mark.gpu
@pytest.mark.parametrize("name,page,dtype", [("A", 4, "float32"), ("B", 8, "float32"), ("C", 4, "float32"), ("E", 16, "float32"), ("E", 16, "bfloat16")])
@pytest.mark.parametrize("graphs", [True, False])
def test_continuations_have_the_plain_models_logits(name, page, dtype, graphs, sharing, tmp_path_factory):
    folder = model_folder(tmp_path_factory.getbasetemp(), name, ALL[name])
    plain = PlainM3(folder)
    V = plain.cfg.vocab
    eng = make_engine(folder, dtype, "cuda:0", page, pages=64, reqs=8, cuda_graph=graphs)
    prompt = tokens_for(V, 53, 1)
    eng.step([StepEntry("a", prompt)])
    eng.fork("a", ["b", "c", "d", "e"])
    seqs = {r: list(prompt) for r in "abcde"}
    eng.step([StepEntry("o", prompt[:7])])
    seqs["o"] = list(prompt[:7])

    def after(t):
        if t == 6:
            eng.fork("c", ["f"])
            seqs["f"] = list(seqs["c"])
        if t == 9:
            eng.close("a")
            del seqs["a"]
            eng.compact()

    start = {r: len(s) for r, s in seqs.items()}
    got = decode(eng, seqs, 14, V, 7, after)
    assert sharing()
    tol = F32_TOL if dtype == "float32" else bf16_tol(name)
    for r, rows in got.items():
        if r == "a":
            continue
        ref = plain.logits(seqs[r])[-rows.shape[0]:]
        if dtype == "bfloat16":  # positions whose choice of experts is clear
            sure = plain.router_margins(seqs[r])[-rows.shape[0]:] > 0
            rows, ref = rows[sure], ref[sure]
        torch.testing.assert_close(rows, ref, **tol, msg=lambda m: f"{r}: {m}")
    for r in list(seqs):
        eng.close(r)
    eng.cache.check()
    eng.check_kernels()
    assert all(g.pool.free_count == g.pool.num_pages for g in eng.cache.paged) and start


@pytest.mark.gpu
@pytest.mark.parametrize("name", sorted(OTHERS))
def test_other_designs_fork_states_windows_and_caches(name, sharing, tmp_path_factory):
    """A fork goes on as a request that read the same tokens by itself does: recurrent states, windows, latent rows, blocks with states."""
    folder = model_folder(tmp_path_factory.getbasetemp(), name, OTHERS[name])
    eng = make_engine(folder, "float32", "cuda:0", 4, pages=120, reqs=6)
    V = eng.spec.vocab_size
    prompt = tokens_for(V, 37, 1)
    eng.step([StepEntry("a", prompt)])
    eng.fork("a", ["b", "c"])
    seqs = {r: list(prompt) for r in "abc"}
    got = decode(eng, seqs, 6, V, 3)
    eng.fork("b", ["d"])
    seqs["d"] = list(seqs["b"])
    more = decode(eng, seqs, 5, V, 5)
    for r in list(seqs):
        eng.close(r)
    eng.cache.check()
    for r in seqs:  # the same sequence, by itself
        eng.step([StepEntry("x", prompt)])
        rows = [eng.step([StepEntry("x", [t], [0])]).logits.float().cpu().clone() for t in seqs[r][len(prompt):]]
        eng.close("x")
        want = torch.cat(rows)
        have = torch.cat([got[r], more[r]]) if r in got else more[r]
        torch.testing.assert_close(have, want[-have.shape[0]:], rtol=1e-3, atol=1e-4)


@pytest.mark.gpu
def test_graph_replays_follow_forks_ends_and_moved_pages(sharing, tmp_path_factory):
    """The same calls with and without recorded steps give the same logits, bit for bit."""
    folder = model_folder(tmp_path_factory.getbasetemp(), "E", ALL["E"])
    out = []
    for graphs in (True, False):
        eng = make_engine(folder, "bfloat16", "cuda:0", 16, pages=64, reqs=6, cuda_graph=graphs)
        V = eng.spec.vocab_size
        prompt = tokens_for(V, 70, 2)
        eng.step([StepEntry("a", prompt)])
        eng.fork("a", ["b", "c", "d"])
        seqs = {r: list(prompt) for r in "abcd"}
        rows = decode(eng, seqs, 20, V, 1, lambda t: eng.compact() if t in (3, 11) else None)
        out.append(rows)
        if graphs:
            assert len(eng.graphs) >= 1
    # (steps of recorded engines have fixed splits in what is not shared: the lists over shared keys are the same)
    for r in out[0]:
        assert torch.equal(out[0][r], out[1][r]), r


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_n_continuations_through_the_entry_point(dtype, sharing, tmp_path_factory):
    folder = model_folder(tmp_path_factory.getbasetemp(), "E", ALL["E"])
    plain = PlainM3(folder)
    V = plain.cfg.vocab
    kw = dict(max_running_req=6, num_page_override=64, page_size=16, max_step_tokens=256, max_extend_tokens=256)
    llm = LLM(folder, dtype=dtype, **kw)
    prompts = [tokens_for(V, 45, 1), tokens_for(V, 30, 2)]
    sp = [SamplingParams(max_tokens=8, temperature=0.9, top_p=0.9, seed=4, n=4), SamplingParams(max_tokens=8, temperature=0.9, seed=4, min_p=0.3)]
    res = llm.generate(prompts, sp)
    assert len(res[0]["samples"]) == 4 and "samples" not in res[1]
    assert sharing()
    assert res[0]["token_ids"] == res[0]["samples"][0]["token_ids"]
    assert llm.generate(prompts, sp) == res  # seeded
    for j, s in enumerate(res[0]["samples"]):
        logits = plain.logits(prompts[0] + s["token_ids"])
        logs = torch.log_softmax(logits, -1)
        want = sum(float(logs[len(prompts[0]) - 1 + i, t]) for i, t in enumerate(s["token_ids"]))
        assert s["logprob"] == pytest.approx(want, abs=1e-2 if dtype == "float32" else 0.3)
        if dtype == "float32":  # the tokens are what the rule gives on the plain model's logits
            for i, t in enumerate(s["token_ids"]):
                u = uniform_for(4, 0 if j == 0 else (0, j), i)
                assert t == fork_refs.draw(logits[len(prompts[0]) - 1 + i].numpy(), 0.9, 0, 0.9, 0.0, u)[0]


@pytest.mark.gpu
def test_draws_beside_other_requests_leave_those_alone(tmp_path_factory):
    """A request's tokens do not depend on whether its neighbours draw."""
    folder = model_folder(tmp_path_factory.getbasetemp(), "A", ALL["A"])
    outs = []
    for neighbour in (SamplingParams(max_tokens=6, temperature=0.8, seed=1), SamplingParams(max_tokens=6, temperature=0.8, seed=1, min_p=0.1, n=2)):
        eng = make_engine(folder, "float32", "cuda:0", 4, pages=60, reqs=5)
        sched = Scheduler(eng, Sampler(eng.device, eng.spec.vocab_size, 5))
        V = eng.spec.vocab_size
        sched.add_request(tokens_for(V, 9, 1), SamplingParams(max_tokens=9, temperature=1.1, top_p=0.9, seed=1), rid="x")
        sched.add_request(tokens_for(V, 12, 2), neighbour, rid="y")
        sched.run()
        outs.append(sched.done["x"].output)
    assert outs[0] == outs[1]
