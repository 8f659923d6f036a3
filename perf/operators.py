"""Requests that continue one prompt: what a decode step of such requests needs beside the model's products.

Families (``case["family"]``):

* ``copy``: pages of the cache (the last, partly filled one of a forked request; whole ones that move to other places) or slots of a
  recurrent state, in all layers at once;
* ``attention``: one query token per request over paged keys and values, where requests share the keys of a common prompt, or of
  a prompt all share and one that only some do;
* ``sample``: draws from given random numbers with temperature, top-k, top-p and min-p, several draws from a row of logits where several
  requests continue the same prompt, and the drawn token's log-probability.

Every call is one layer's (``attention``) or one step's (``copy``, ``sample``); the work list of the attention is made once per step, as an
engine does for all of its layers.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = torch.device("cuda:0")
PAGE = 16

# layer sizes of the headline benchmark and of the two smaller ones beside it
LARGE = dict(heads=48, kv_heads=8, dim=128)
MID = dict(heads=16, kv_heads=4, dim=128)
SMALL = dict(heads=16, kv_heads=4, dim=64)


def listed():
    return [
        # four continuations of one short prompt: a partly filled page each, in a small model's four layers
        dict(name="copy_fork_4", family="copy", kind="pages", dtype="bfloat16", entries=4, kv_heads=4, dim=64, pairs=4, whole=False),
        # 63 continuations at once, twelve layers
        dict(name="copy_fork_63", family="copy", kind="pages", dtype="bfloat16", entries=12, kv_heads=8, dim=128, pairs=63, whole=False),
        # a fragmented cache made dense again
        dict(name="copy_compact_1500", family="copy", kind="pages", dtype="bfloat16", entries=4, kv_heads=8, dim=128, pairs=1500, whole=True),
        # a linear attention's matrix states for 7 continuations
        dict(name="copy_states_7", family="copy", kind="slots", dtype="float32", entries=6, kv_heads=16, dim=128, pairs=7, whole=True),
        # two answers to a short question: the smallest step there is
        dict(name="attention_2x500", family="attention", dtype="bfloat16", **MID, groups=1, per=2, system=0, prefix=496, tail=9),
        # eight answers to one prompt of ordinary length
        dict(name="attention_8x2048", family="attention", dtype="bfloat16", **LARGE, groups=1, per=8, system=0, prefix=2048, tail=300),
        # a long document asked about 32 times
        dict(name="attention_32x32000", family="attention", dtype="bfloat16", **LARGE, groups=1, per=32, system=0, prefix=32000, tail=700),
        # a system prompt under all requests, a prompt of their own under every four
        dict(name="attention_16x4_nested", family="attention", dtype="bfloat16", **LARGE, groups=16, per=4, system=4096, prefix=1200, tail=333),
        # a small model's heads, 200 classifications under the same instructions
        dict(name="attention_200_h64", family="attention", dtype="bfloat16", **SMALL, groups=1, per=200, system=0, prefix=4000, tail=65),
        # the true 32-bit path
        dict(name="attention_f32_6", family="attention", dtype="float32", **SMALL, groups=2, per=3, system=160, prefix=640, tail=50),
        # one user's next token, all filters on
        dict(name="sample_1", family="sample", rows=1, draws=1, vocab=200064, filters="all"),
        # a busy step: continuations of 24 prompts, every request with filters of its own
        dict(name="sample_96_of_24", family="sample", rows=24, draws=96, vocab=200064, filters="mixed"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    family = rng.choice(["copy", "attention", "attention", "sample"])
    if family == "copy":
        if rng.random() < 0.3:
            return dict(family=family, kind="slots", dtype="float32", entries=rng.randint(1, 8), kv_heads=rng.choice([4, 16]),
                        dim=rng.choice([64, 128]), pairs=_log(rng, 1, 16), whole=True)
        whole = rng.random() < 0.4
        return dict(family=family, kind="pages", dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), entries=rng.randint(1, 12) if not whole else rng.randint(1, 4),
                    kv_heads=rng.choice([1, 4, 8]), dim=rng.choice([64, 128]), pairs=_log(rng, 1, 700 if whole else 64), whole=whole)
    if family == "attention":
        if rng.random() < 0.2:
            return dict(family=family, dtype="float32", **SMALL, groups=rng.randint(1, 3), per=rng.randint(2, 4),
                        system=PAGE * rng.randint(0, 20), prefix=PAGE * rng.randint(1, 60), tail=_log(rng, 1, 200))
        size = rng.choice([LARGE, MID, SMALL])
        per, groups = _log(rng, 2, 64), rng.choice([1, 1, 2, 5])
        most = 900000 // (per * groups)  # keys per request
        prefix = min(_log(rng, 32, 32000), most * 3 // 4)
        system = rng.choice([0, _log(rng, 32, 4096)]) if groups > 1 else 0
        return dict(family=family, dtype="bfloat16", **size, groups=groups, per=per, system=min(system, most // 8) // PAGE * PAGE,
                    prefix=max(PAGE, prefix // PAGE * PAGE), tail=min(_log(rng, 1, 1500), max(1, most // 8)))
    rows = _log(rng, 1, 48)
    return dict(family=family, rows=rows, draws=rows * rng.choice([1, 1, 2, 4]) if rows <= 24 else rows,
                vocab=rng.choice([32768, 65536, 200064, 32003, 151937]), filters=rng.choice(["none", "all", "mixed", "mixed"]))


# --------------------------------------------------------------------------- inputs, from the seed alone
def _gen(seed, what):
    return torch.Generator(device=DEV).manual_seed((seed * 1000003 + what) & 0x7FFFFFFF)


def _normal(gen, shape, std=1.0, dtype="float32"):
    """Drawn in the type itself: a bfloat16 cache holds bfloat16 numbers."""
    return torch.empty(shape, dtype=getattr(torch, dtype), device=DEV).normal_(0.0, std, generator=gen)


def _own_tokens(case):
    """Tokens that are a request's own: requests began one after the other."""
    n = case["groups"] * case["per"]
    return [max(1, case["tail"] * (i * 7 % n + 1) // n) for i in range(n)]


def _prepare_copy(case, seed):
    gen, rng = _gen(seed, 1), np.random.default_rng([seed, 2])
    n, E, H, D = case["pairs"], case["entries"], case["kv_heads"], case["dim"]
    if case["kind"] == "slots":
        slots = n + 2
        tensors = [_normal(gen, (E, slots, H, D, D)), _normal(gen, (E, slots, H, D))]
        order = rng.permutation(np.arange(1, slots))
        pairs = np.stack([np.full(n, order[0]), order[1:]], axis=1)  # one request's state for all of them
        return dict(tensors=tensors, pairs=torch.from_numpy(pairs.astype(np.int32)).to(DEV))
    pages = 2 * n + 1 if case["whole"] else n + 8
    slabs = [_normal(gen, (E, pages, H, PAGE, D), dtype=case["dtype"]) for _ in "kv"]
    order = rng.permutation(np.arange(1, pages))
    if case["whole"]:  # every page to a place of its own
        pairs = np.stack([order[:n], order[n:2 * n], np.full(n, PAGE)], axis=1)
    else:  # the last page of one prompt for each of its continuations
        pairs = np.stack([np.full(n, order[0]), order[1:n + 1], np.full(n, int(rng.integers(1, PAGE)))], axis=1)
    return dict(tensors=slabs, pairs=torch.from_numpy(pairs.astype(np.int32)).to(DEV))


def _prepare_attention(case, seed):
    gen, rng = _gen(seed, 3), np.random.default_rng([seed, 4])
    H, G, D, dt = case["heads"], case["kv_heads"], case["dim"], case["dtype"]
    groups, per, system, prefix = case["groups"], case["per"], case["system"], case["prefix"]
    n = groups * per
    lens = [system + prefix + t for t in _own_tokens(case)]
    common, each = system // PAGE, prefix // PAGE
    own_blocks = [-(-(x - system - prefix) // PAGE) for x in lens]
    pages = common + groups * each + sum(own_blocks) + 1
    ids = rng.permutation(np.arange(1, pages)).astype(np.int32)
    width = max(-(-x // PAGE) for x in lens) + 3
    table = np.zeros((n, width), dtype=np.int32)
    table[:, :common] = ids[:common]
    table[:, common:common + each] = ids[common:common + groups * each].reshape(groups, 1, each).repeat(per, 1).reshape(n, each)
    at = common + groups * each + np.concatenate([[0], np.cumsum(own_blocks)])
    for i in range(n):
        table[i, common + each:common + each + own_blocks[i]] = ids[at[i]:at[i + 1]]
    slabs = [_normal(gen, (pages, G, PAGE, D), dtype=dt) for _ in "kv"]
    q = _normal(gen, (n, H, D), 1.5, dt)
    spans = [(list(range(n)), 0, system)] if system else []
    spans += [(list(range(g * per, (g + 1) * per)), system, system + prefix) for g in range(groups)]
    state = dict(q=q, k=slabs[0], v=slabs[1], table=torch.from_numpy(table).to(DEV), lens=torch.tensor(lens, device=DEV), most=max(lens),
                 out=torch.empty_like(q), scale=D ** -0.5, plan=None)
    if own:  # a step's work list: made once, for all of the step's layers
        from freetoken_b200.engine.shared_plan import build_shared_plan
        state["plan"] = build_shared_plan(lens, spans, H, G, D, q.dtype, PAGE).to(DEV)
    return state


def _prepare_sample(case, seed):
    gen, rng = _gen(seed, 5), np.random.default_rng([seed, 6])
    N, R, V = case["rows"], case["draws"], case["vocab"]
    # a few likely tokens above a broad floor
    logits = _normal(gen, (N, V), 2.0)
    tops = torch.randint(0, V, (N, 40), device=DEV, generator=gen)
    logits.scatter_add_(1, tops, _normal(gen, (N, 40), 3.0).abs() + 5.0)
    rows = np.sort(np.concatenate([np.arange(N), rng.integers(0, N, R - N)])).astype(np.int32)
    temperature = rng.choice([0.6, 0.8, 1.0, 1.3], R).astype(np.float32)
    top_k = rng.choice([1, 20, 50, 1000], R).astype(np.int32) if R > 1 else np.array([50], dtype=np.int32)
    top_p = rng.choice([0.8, 0.9, 0.95], R).astype(np.float32)
    min_p = rng.choice([0.02, 0.05, 0.1], R).astype(np.float32)
    if case["filters"] == "none":
        top_k[:], top_p[:], min_p[:] = 0, 1.0, 0.0
    elif case["filters"] == "mixed":  # each filter in some requests, and some that take the likeliest token
        top_k[rng.random(R) < 0.6] = 0
        top_p[rng.random(R) < 0.5] = 1.0
        min_p[rng.random(R) < 0.5] = 0.0
        temperature[rng.random(R) < 0.1] = 0.0
    u = rng.random(R, dtype=np.float32)
    put = lambda a: torch.from_numpy(a).to(DEV)  # noqa: E731
    return dict(logits=logits, rows=put(rows), temperature=put(temperature), top_k=put(top_k), top_p=put(top_p), min_p=put(min_p), u=put(u),
                out=torch.empty(R, dtype=torch.int32, device=DEV), logprobs=torch.empty(R, dtype=torch.float32, device=DEV))


def prepare(case, seed):
    state = {"copy": _prepare_copy, "attention": _prepare_attention, "sample": _prepare_sample}[case["family"]](case, seed)
    state["case"] = case
    return state


# --------------------------------------------------------------------------- plain forms
def _copied(t, pairs):
    src, dst = pairs[:, 0].long(), pairs[:, 1].long()
    new = t[:, src]
    if pairs.shape[1] == 3:  # the first rows of a page, the others as they were
        row = torch.arange(t.shape[3], device=t.device)
        new = torch.where((row[None, :] < pairs[:, 2:3])[None, :, None, :, None], new, t[:, dst])
    t[:, dst] = new
    return t


def _attended(s):
    q, table, lens = s["q"], s["table"].long(), s["lens"]
    n, H, D = q.shape
    G = s["k"].shape[1]
    pos = torch.arange(s["most"], device=DEV)
    page, offset = table[:, pos // PAGE], pos % PAGE
    k = s["k"][page, :, offset[None, :]].float()  # [n, keys, KV heads, D]: every request's keys
    scores = torch.einsum("nghd,nkgd->nghk", q.float().view(n, G, H // G, D), k) * s["scale"]
    del k
    scores = torch.softmax(scores.masked_fill((pos[None, :] >= lens[:, None])[:, None, None, :], float("-inf")), dim=-1)
    v = s["v"][page, :, offset[None, :]].float()
    s["out"].copy_(torch.einsum("nghk,nkgd->nghd", scores, v).reshape(n, H, D))
    return s["out"]


def _drawn(s):
    """In 64 bits: a draw is decided by long running sums next to borders."""
    t = s["temperature"].double()[:, None]
    x = s["logits"][s["rows"].long()].double()
    V = x.shape[1]
    top = x.max(dim=1, keepdim=True).values
    greedy = (t <= 0)[:, 0]
    z = (x - top) / torch.where(t > 0, t, torch.ones_like(t))
    e = torch.exp(z)
    ordered = torch.sort(x, dim=1, descending=True).values
    k = s["top_k"].long()[:, None]
    limit = torch.where((k > 0) & (k < V), ordered.gather(1, (k.clamp(1, V) - 1)), torch.full_like(top, float("-inf")))
    kept = torch.where(x >= limit, e, torch.zeros_like(e))
    # top-p: down to the value at which the likeliest kept tokens hold that share
    mass = torch.where(ordered >= limit, torch.exp((ordered - top) / torch.where(t > 0, t, torch.ones_like(t))), torch.zeros_like(e)).cumsum(1)
    p = s["top_p"].double()[:, None]
    at = (mass < p * mass[:, -1:]).sum(dim=1, keepdim=True).clamp(max=V - 1)
    limit = torch.where(p < 1.0, torch.maximum(limit, ordered.gather(1, at)), limit)
    least = torch.log(s["min_p"].double())[:, None]  # (minus infinity: no filter)
    kept = torch.where((x >= limit) & (z >= least), kept, torch.zeros_like(e))
    run = kept.cumsum(1)
    token = (run <= s["u"].double()[:, None] * run[:, -1:]).sum(dim=1).clamp(max=V - 1)
    token = torch.where(greedy, (x == top).int().argmax(dim=1), token)
    s["out"].copy_(token)
    s["logprobs"].copy_(x.gather(1, token[:, None])[:, 0] - torch.logsumexp(x, dim=1))
    return s["out"], s["logprobs"]


def run(state):
    family = state["case"]["family"]
    if own:
        from freetoken_b200.kernels import ops
        if family == "copy":
            (ops.copy_slots if state["case"]["kind"] == "slots" else ops.copy_pages)(state["tensors"], state["pairs"])
            return state["tensors"]
        if family == "attention":
            ops.shared_attention(state["q"], state["k"], state["v"], state["table"], state["plan"], state["out"], state["scale"])
            return state["out"]
        ops.sample_draws(state["logits"], state["rows"], state["temperature"], state["top_k"], state["top_p"], state["min_p"], state["u"],
                         state["out"], state["logprobs"])
        return state["out"], state["logprobs"]
    if family == "copy":
        return [_copied(t, state["pairs"]) for t in state["tensors"]]
    return _attended(state) if family == "attention" else _drawn(state)


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["family"] == "copy":
        E, H, D, n = case["entries"], case["kv_heads"], case["dim"], case["pairs"]
        item = 4 if case["dtype"] == "float32" else 2
        if case["kind"] == "slots":
            return {"bytes": float(E * H * (D * D + D) * item * (n + 1)), "flops": 0.0}
        rows = PAGE if case["whole"] else PAGE // 2  # (about: a prompt ends anywhere in its last page)
        return {"bytes": float(2 * E * H * rows * D * item * (2 * n if case["whole"] else n + 1)), "flops": 0.0}
    if case["family"] == "attention":
        item = 4 if case["dtype"] == "float32" else 2
        own_tokens = _own_tokens(case)
        distinct = case["system"] + case["groups"] * case["prefix"] + sum(own_tokens)
        read = len(own_tokens) * (case["system"] + case["prefix"]) + sum(own_tokens)
        return {"bytes": float(item * case["dim"] * (2 * distinct * case["kv_heads"] + 2 * len(own_tokens) * case["heads"])),
                "flops": 4.0 * case["dim"] * case["heads"] * read}
    return {"bytes": 4.0 * case["rows"] * case["vocab"], "flops": 4.0 * case["draws"] * case["vocab"]}


# --------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    if case["family"] == "copy":
        return None  # (nothing is computed)
    s = prepare(case, seed)
    if case["family"] == "attention":
        lens, table = s["lens"].tolist(), s["table"].long()
        out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
        G = s["k"].shape[1]
        for i, length in enumerate(lens):  # request by request, KV head by KV head
            pages = table[i, :-(-length // PAGE)]
            for g in range(G):
                k = s["k"][pages, g].reshape(-1, s["k"].shape[3])[:length].double()
                v = s["v"][pages, g].reshape(-1, s["v"].shape[3])[:length].double()
                heads = slice(g * (out.shape[1] // G), (g + 1) * (out.shape[1] // G))
                w = (s["q"][i, heads].double() @ k.T) * s["scale"]
                w = torch.exp(w - w.max(dim=1, keepdim=True).values)
                out[i, heads] = (w @ v) / w.sum(dim=1, keepdim=True)
        return out
    tokens, logprobs = [], []
    logits = s["logits"].cpu().numpy()
    get = lambda name: s[name].cpu().numpy()  # noqa: E731
    for r, t, k, p, mp, u in zip(get("rows"), get("temperature"), get("top_k"), get("top_p"), get("min_p"), get("u")):
        x = logits[r].astype(np.float64)
        top = x.max()
        whole = np.exp(x - top)
        if t <= 0:
            token = int(np.flatnonzero(x == top)[0])
        else:
            order = np.argsort(-x, kind="stable")
            z = (x[order] - top) / np.float64(t)
            w = np.exp(z)
            keep = len(w)
            if 0 < k < len(w):
                keep = int(np.searchsorted(-x[order], -x[order[k - 1]], side="right"))  # ties of the k-th stay
            if p < 1:
                held = np.cumsum(w[:keep])
                last = int(np.searchsorted(held, np.float64(p) * held[-1], side="left"))
                keep = int(np.searchsorted(-x[order], -x[order[last]], side="right"))
            if mp > 0:
                keep = min(keep, int((z >= np.log(np.float64(mp))).sum()))
            chosen = np.sort(order[:keep])
            held = np.cumsum(np.exp((x[chosen] - top) / np.float64(t)))
            token = int(chosen[min(keep - 1, np.searchsorted(held, np.float64(u) * held[-1], side="right"))])
        tokens.append(token)
        logprobs.append(x[token] - top - math.log(whole.sum()))
    return torch.tensor(tokens, dtype=torch.int32), torch.tensor(logprobs, dtype=torch.float64)
