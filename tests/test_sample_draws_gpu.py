"""Draws with temperature, top-k, top-p and min-p against the rule in 64 bits."""

import numpy as np
import pytest
import torch

from freetoken_b200.errors import KernelError
from freetoken_b200.kernels import ops

DEV = "cuda:0"


def plain(x, t, k, p, mp, u):
    """(token, log-probability, how near u came to a border of the kept mass, kept tokens)."""
    x = np.where(np.isnan(x), -np.inf, x).astype(np.float64)
    top = x.max()
    if top == -np.inf:
        return 0, -np.inf, 1.0, 0
    with np.errstate(invalid="ignore", divide="ignore"):
        z1 = np.where(x == top, 0.0, x - top)
    whole = np.log(np.exp(z1).sum())
    if not t > 0:
        token = int(np.flatnonzero(x == top)[0])
        return token, z1[token] - whole, 1.0, 1
    z = z1 / np.float64(t)
    w = np.exp(z)
    limit = -np.inf
    if 0 < k < len(x):
        limit = np.sort(x)[::-1][k - 1]
    keep = (x >= limit) & (x > -np.inf)
    if p < 1:
        values = np.unique(x[keep])[::-1]
        held = np.array([w[x >= v].sum() for v in values]) if len(values) < 3000 else None
        if held is None:
            order = np.sort(x[keep])[::-1]
            run = np.cumsum(np.exp(np.where(order == top, 0.0, order - top) / np.float64(t)))
            keep &= x >= order[min(len(order) - 1, np.searchsorted(run, np.float64(p) * run[-1]))]
        else:
            keep &= x >= values[min(len(values) - 1, np.searchsorted(held, np.float64(p) * w[keep].sum()))]
    if mp > 0:
        keep &= (z >= min(0.0, np.log(np.float64(mp)))) | (x == top)
    at = np.flatnonzero(keep)
    held = np.cumsum(w[at])
    target = np.float64(u) * held[-1]
    i = min(len(at) - 1, int(np.searchsorted(held, target, side="right")))
    near = np.abs(held - target).min() / held[-1]
    return int(at[i]), z1[at[i]] - whole, near, len(at)


def draws(logits, rows, t, k, p, mp, u, logprobs=True):
    R = len(u)
    f = lambda a: torch.tensor(np.broadcast_to(a, R).copy(), dtype=torch.float32, device=DEV)  # noqa: E731
    out = torch.full((R,), -7, dtype=torch.int32, device=DEV)
    lp = torch.full((R,), 3.0, dtype=torch.float32, device=DEV) if logprobs else None
    ops.sample_draws(logits, None if rows is None else torch.tensor(rows, dtype=torch.int32, device=DEV), f(t),
                     torch.tensor(np.broadcast_to(k, R).copy(), dtype=torch.int32, device=DEV), f(p), f(mp), f(u), out, lp)
    torch.cuda.synchronize()
    return out.cpu().numpy(), None if lp is None else lp.cpu().numpy()


def check(x, rows, t, k, p, mp, u):
    got, lp = draws(torch.from_numpy(x).to(DEV), rows, t, k, p, mp, u)
    R = len(u)
    b = lambda a: np.broadcast_to(a, R)  # noqa: E731
    for r in range(R):
        args = [np.float32(b(a)[r]) for a in (t, p, mp, u)]
        token, logp, near, kept = plain(x[rows[r] if rows is not None else r], args[0], int(b(k)[r]), args[1], args[2], args[3])
        # sums of up to 2^18 terms in 64 bits are off by 2^-34 of the mass at the very most
        assert got[r] == token or near < 2.0 ** -34, (r, got[r], token, near, kept, [b(a)[r] for a in (t, k, p, mp, u)])
        if got[r] == token:
            assert lp[r] == float(torch.tensor(logp, dtype=torch.float64).float()) or abs(lp[r] - logp) <= 2.0 ** -23 * max(1.0, abs(logp)), (r, lp[r], logp)


def rows_of(kind, n, vocab, rng):
    if kind == "normal":
        return rng.normal(0, 2, (n, vocab)).astype(np.float32)
    if kind == "flat":
        return rng.normal(0, 1e-3, (n, vocab)).astype(np.float32)
    if kind == "peaked":
        x = rng.normal(-5, 1, (n, vocab)).astype(np.float32)
        x[np.arange(n), rng.integers(0, vocab, n)] = 20
        return x
    if kind == "ties":  # few values, each many times
        return (rng.integers(-3, 4, (n, vocab)) / 2).astype(np.float32)
    if kind == "equal":
        return np.full((n, vocab), 1.25, dtype=np.float32)
    x = rng.normal(0, 3, (n, vocab)).astype(np.float32)  # "masked": most tokens ruled out, in several ways
    x[rng.random((n, vocab)) < 0.7] = -np.inf
    x[rng.random((n, vocab)) < 0.05] = np.nan
    x[rng.random((n, vocab)) < 0.05] = np.finfo(np.float32).min
    x[:, vocab // 2] = 0.0
    return x


KINDS = ["normal", "flat", "peaked", "ties", "equal", "masked"]


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1, 2, 31, 257, 1000, 32003])
@pytest.mark.parametrize("kind", KINDS)
def test_filters(kind, vocab):
    rng = np.random.default_rng([vocab, KINDS.index(kind)])
    n = 6
    x = rows_of(kind, n, vocab, rng)
    R = 40
    rows = rng.integers(0, n, R)
    t = rng.choice([0.0, -1.0, 0.05, 0.7, 1.0, 3.0], R)
    k = rng.choice([0, -1, 1, 2, 20, 50, 1000, vocab, vocab + 5], R)
    p = rng.choice([1.0, 0.95, 0.5, 0.1, 1e-6, 0.0, 2.0], R)
    mp = rng.choice([0.0, 0.02, 0.1, 0.5, 1.0, 1.5, -1.0], R)
    u = rng.random(R)
    u[:3] = [0.0, 1.0 - 2.0 ** -24, 0.5]
    check(x, rows, t, k, p, mp, u)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["normal", "flat", "ties"])
def test_a_large_vocabulary(kind):
    rng = np.random.default_rng(KINDS.index(kind))
    x = rows_of(kind, 3, 200064, rng)
    R = 48
    u = rng.random(R)
    check(x, rng.integers(0, 3, R), rng.choice([0.5, 1.0, 1.4], R), rng.choice([0, 0, 40, 5000], R), rng.choice([1.0, 0.9, 0.999], R),
          rng.choice([0.0, 0.05], R), u)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["normal", "masked", "infinite"])
def test_rows_beyond_shared_memory(kind):
    """Longer than a cluster's CTAs hold: read again in every pass."""
    rng = np.random.default_rng(77)
    vocab, R = 460001, 12
    x = rows_of("masked" if kind == "masked" else "normal", 2, vocab, rng)
    if kind == "infinite":
        x[0, [5, 123456, 460000]] = np.inf
        x[1, ::3] = np.inf
        u = rng.random(R).astype(np.float32)
        rows = np.arange(R) % 2
        got, lp = draws(torch.from_numpy(x).to(DEV), rows, 0.7, rng.choice([0, 1, 40], R), rng.choice([1.0, 0.5], R), rng.choice([0.0, 0.1], R), u)
        for r in range(R):  # of equals all stay
            at = np.flatnonzero(x[rows[r]] == np.inf)
            assert got[r] == at[min(int(np.float64(u[r]) * len(at)), len(at) - 1)] and np.isclose(lp[r], -np.log(len(at)), rtol=2e-7, atol=0)
        return
    check(x, rng.integers(0, 2, R), rng.choice([0.5, 1.0, 1.4], R), rng.choice([0, 0, 40, 5000], R), rng.choice([1.0, 0.9, 0.999], R),
          rng.choice([0.0, 0.05], R), rng.random(R))


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [300, 32003])
def test_temperatures_and_logits_at_the_ends_of_32_bits(vocab):
    rng = np.random.default_rng(vocab)
    R = 24
    x = np.stack([rng.normal(0, s, vocab) for s in (1e-30, 1.0, 1e30)]).astype(np.float32)
    x[1, 7] = np.finfo(np.float32).max
    x[1, 9] = np.finfo(np.float32).min
    rows = np.arange(R) % 3
    check(x, rows, rng.choice([1e-38, 1e-30, 1e-3, 1.0, 1e30, 3e38], R), rng.choice([0, 3, 250], R), rng.choice([1.0, 0.9, 0.3], R),
          rng.choice([0.0, 0.05], R), rng.random(R))


@pytest.mark.gpu
def test_rows_of_infinities_and_of_nothing():
    x = np.full((4, 300), -np.inf, dtype=np.float32)
    x[1] = np.nan
    x[2, [7, 200]] = np.inf
    x[2, 50] = 3.0
    x[3, 299] = np.finfo(np.float32).min
    u = np.array([0.3, 0.3, 0.2, 0.9, 0.2, 0.5])
    got, lp = draws(torch.from_numpy(x).to(DEV), [0, 1, 2, 2, 2, 3], [1.0, 1.0, 1.0, 1.0, 0.0, 1.0], 0, 1.0, 0.0, u)
    assert got.tolist() == [0, 0, 7, 200, 7, 299]
    assert lp[0] == lp[1] == -np.inf and np.allclose(lp[2:5], -np.log(2)) and lp[5] == 0.0


@pytest.mark.gpu
def test_strides_missing_rows_and_no_logprobs():
    rng = np.random.default_rng(0)
    wide = torch.from_numpy(rng.normal(0, 2, (5, 1003)).astype(np.float32)).to(DEV)
    view = wide[:, 3:1000]
    u = rng.random(5)
    got, lp = draws(view, None, 0.8, 30, 0.9, 0.01, u)
    want, lp2 = draws(view.contiguous(), [0, 1, 2, 3, 4], 0.8, 30, 0.9, 0.01, u)
    assert (got == want).all() and (lp == lp2).all()
    assert (draws(view, None, 0.8, 30, 0.9, 0.01, u, logprobs=False)[0] == want).all()
    got, lp = draws(view, [4, 5, -1, 0, 1 << 30], 0.8, 30, 0.9, 0.01, u)
    assert (got[[1, 2, 4]] == -1).all() and (lp[[1, 2, 4]] == -np.inf).all() and (got[[0, 3]] >= 0).all()


@pytest.mark.gpu
def test_draws_do_not_depend_on_the_batch():
    rng = np.random.default_rng(1)
    x = torch.from_numpy(rng.normal(0, 2, (8, 50000)).astype(np.float32)).to(DEV)
    R = 64
    rows, u = rng.integers(0, 8, R), rng.random(R)
    t, k, p, mp = rng.choice([0.0, 0.7, 1.0], R), rng.choice([0, 50], R), rng.choice([1.0, 0.9], R), rng.choice([0.0, 0.05], R)
    got, lp = draws(x, rows, t, k, p, mp, u)
    for r in (0, 1, 17, 63):
        one, one_lp = draws(x[rows[r]:rows[r] + 1], None, t[r:r + 1], k[r:r + 1], p[r:r + 1], mp[r:r + 1], u[r:r + 1])
        assert one[0] == got[r] and one_lp[0] == lp[r]


@pytest.mark.gpu
def test_captured_replayed_and_shares():
    """Frequencies of one row over a sweep of u, from a replayed graph."""
    rng = np.random.default_rng(2)
    x = torch.from_numpy(rng.normal(0, 1, (1, 64)).astype(np.float32)).to(DEV)
    R = 1000
    f = lambda v: torch.full((R,), v, dtype=torch.float32, device=DEV)  # noqa: E731
    rows, k = torch.zeros(R, dtype=torch.int32, device=DEV), torch.zeros(R, dtype=torch.int32, device=DEV)
    t, p, mp, u, out = f(1.0), f(1.0), f(0.0), f(0.0), torch.empty(R, dtype=torch.int32, device=DEV)
    ops.sample_draws(x, rows, t, k, p, mp, u, out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.sample_draws(x, rows, t, k, p, mp, u, out)
    u.copy_((torch.arange(R) + 0.5) / R)
    graph.replay()
    torch.cuda.synchronize()
    share = torch.bincount(out.long().cpu(), minlength=64).double() / R
    want = torch.softmax(x[0].double().cpu(), 0)
    assert (share - want).abs().max() <= 1.0 / R + 1e-9  # (evenly spread numbers: a token's share is at most one off)


def test_refusals_without_a_gpu():
    x = torch.zeros((2, 8))
    f, i = torch.zeros(2), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(KernelError, match="device"):
        ops.sample_draws(x, None, f, i, f, f, f, i)


@pytest.mark.gpu
def test_refusals():
    x = torch.zeros((2, 8), device=DEV)
    f, i = torch.zeros(2, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    ops.sample_draws(x, None, f, i, f, f, f, i.clone())
    f3, i3 = torch.zeros(3, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
    for args in [(x.double(), None, f, i, f, f, f, i), (x.t(), None, f, i, f, f, f, i), (x, None, f3, i3, f3, f3, f3, i3), (x, i.float(), f, i, f, f, f, i),
                 (x, None, f[:1], i, f, f, f, i), (x, None, f, f, f, f, f, i), (x, None, f, i, f, f, f, f), (x[0], None, f, i, f, f, f, i),
                 (x[:, :0], None, f, i, f, f, f, i), (x[:0], i, f, i, f, f, f, i), (x[:1].expand(2, 8), None, f, i, f, f, f, i)]:
        with pytest.raises(KernelError):
            ops.sample_draws(*args)
