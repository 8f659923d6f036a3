"""Plain statements of the operators that forked requests need, for CPU tests of the host logic (beside tests/kernel_refs.py)."""

import numpy as np
import torch

import kernel_refs


def copy_pages(slabs, pairs):
    for t in slabs:
        old = t.clone()
        for a, b, rows in pairs.tolist():
            if a != b and min(a, b) >= 0 and max(a, b) < t.shape[1] and rows > 0:
                t[:, b, :, :rows] = old[:, a, :, :rows]


def copy_slots(tensors, pairs):
    for t in tensors:
        old = t.clone()
        for a, b in pairs.tolist():
            t[:, b] = old[:, a]


def shared_attention(q, k_slab, v_slab, block_table, plan, out, scale, sink=None):
    """From the work list itself: every piece's keys once, the requests' own, joined."""
    host = plan.host
    H, G, D, P = host.n_heads, host.n_kv_heads, host.head_dim, k_slab.shape[2]
    parts = {}

    def piece(rows, bt_row, lo, hi):
        pos = torch.arange(lo, hi)
        page = block_table[bt_row][pos // P].long()
        k = k_slab[page, :, pos % P].double().repeat_interleave(H // G, 1)  # [keys, H, D]
        v = v_slab[page, :, pos % P].double().repeat_interleave(H // G, 1)
        s = torch.einsum("rhd,khd->rhk", q[rows].double(), k) * scale
        m = s.max(-1, keepdim=True).values
        w = torch.exp(s - m)
        return m, w.sum(-1, keepdim=True), torch.einsum("rhk,khd->rhd", w, v)

    for mem0, n, bt_row, lo, hi, slot0, split, _ in plan.items.tolist():
        rows = plan.members[mem0:mem0 + n].tolist()
        ranges = [(lo, hi)]
        if split:  # even and odd key tiles
            tiles = list(range(lo, hi, 128))
            ranges = [[(t, min(hi, t + 128)) for t in tiles[half::2]] for half in range(2)]
        for half, r in enumerate(ranges if split else [ranges]):
            got = [piece(rows, bt_row, a, b) for a, b in r]
            for i in range(n):
                parts[slot0 + half * n + i] = [tuple(x[i] for x in g) for g in got]
    for row, bt_row, lo, hi, j0, n, _, _ in plan.requests.tolist():
        mine = [p for s in plan.joins[j0:j0 + n].tolist() for p in parts[s]]
        if hi > lo:
            mine.append(tuple(x[0] for x in piece([row], bt_row, lo, hi)))
        if not mine:
            out[row] = 0
            continue
        M = torch.stack([m for m, _, _ in mine]).max(0).values
        L = sum(l * torch.exp(m - M) for m, l, _ in mine)
        if sink is not None:
            L = L + torch.exp(torch.as_tensor(sink, dtype=torch.float64).reshape(-1, 1) - M)
        out[row] = (sum(o * torch.exp(m - M) for m, _, o in mine) / L).to(out.dtype)


def draw(x, t, k, p, mp, u):
    """(token, log-probability) in 64 bits."""
    x = np.where(np.isnan(x), -np.inf, x).astype(np.float64)
    top = x.max()
    logs = x - top - np.log(np.exp(x - top).sum())
    if not t > 0:
        token = int(np.argmax(x))
        return token, logs[token]
    z = (x - top) / np.float64(t)
    w = np.exp(z)
    keep = x > -np.inf
    if 0 < k < len(x):
        keep &= x >= np.sort(x)[::-1][k - 1]
    if p < 1:
        order = np.sort(x[keep])[::-1]
        run = np.cumsum(np.exp((order - top) / np.float64(t)))
        keep &= x >= order[np.searchsorted(run, np.float64(p) * run[-1])]
    if mp > 0:
        keep &= (z >= np.log(np.float64(mp))) | (x == top)
    at = np.flatnonzero(keep)
    held = np.cumsum(w[at])
    token = int(at[min(len(at) - 1, int(np.searchsorted(held, np.float64(u) * held[-1], side="right")))])
    return token, logs[token]


def sample_draws(logits, rows, temperature, top_k, top_p, min_p, u, out, logprobs=None):
    for r in range(out.numel()):
        x = logits[int(rows[r]) if rows is not None else r].float().numpy()
        token, logp = draw(x, np.float32(temperature[r]), int(top_k[r]), np.float32(top_p[r]), np.float32(min_p[r]), np.float32(u[r]))
        out[r] = token
        if logprobs is not None:
            logprobs[r] = float(logp)


def install(monkeypatch) -> None:
    from freetoken_b200.kernels import ops

    kernel_refs.install(monkeypatch)
    for fn in (copy_pages, copy_slots, shared_attention, sample_draws):
        monkeypatch.setattr(ops, fn.__name__, fn)
