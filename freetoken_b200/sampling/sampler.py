"""Turns logits into tokens.

Greedy requests take the argmax; the others ``softmax(logits / max(T, 1e-6))``, top-k, then
top-p, then an inverse-CDF draw (python/freetoken/engine/sample.py:54-80).  One kernel
handles a whole batch, greedy and sampled rows together; requests with min-p or several continuations go through another
(``ops.sample_draws``: several draws from a row, sums in 64 bits, log-probabilities).  Which one a request's tokens come from
depends on its own parameters alone.  The uniform number of each draw is
made on the host from (seed, request, step) with a counter-based hash, so the same request
gives the same tokens whatever else shares its steps; the reference draws from the device's
global generator (python/freetoken/kernel/triton/sampling.py:398-409).
"""

from __future__ import annotations

import hashlib
from typing import Hashable, List, Optional, Sequence

import numpy as np
import torch

from ..kernels import ops
from .params import SamplingParams

MIN_T = 1e-6
MIN_P = 1e-6


def uniform_for(seed: int, request: Hashable, step: int) -> float:
    """A number in [0, 1) that depends only on its three arguments."""
    h = hashlib.blake2b(f"{seed}|{request!r}|{step}".encode(), digest_size=8).digest()
    return (int.from_bytes(h, "little") >> 40) / float(1 << 24)


class SampleTicket:
    """A launched sampling call: the tokens are on the device (``device_tokens``) and on their way to
    the host; :meth:`Sampler.result` waits for them."""

    def __init__(self, n: int, device_tokens: torch.Tensor, host_tokens: torch.Tensor, event, host_logprobs: Optional[torch.Tensor] = None,
                 drawn: Sequence[int] = ()):
        self.n = n
        self.device_tokens = device_tokens
        self.host_tokens = host_tokens
        self.event = event
        self.host_logprobs = host_logprobs  # of the tokens that were drawn (with their places in `drawn`)
        self.drawn = drawn


class Sampler:
    BUFFERS = 3  # launches that may be in flight before a buffer is used again

    def __init__(self, device: torch.device, vocab_size: int, max_rows: int, default_seed: int = 0):
        self.device = device
        self.vocab_size = vocab_size
        self.default_seed = default_seed
        self.max_rows = max_rows
        pin = device.type == "cuda"
        # per buffer, one packed staging area: temperature, top_p, u (float32 as raw bits) and top_k
        self._host = [torch.empty(4 * max_rows, dtype=torch.int32, pin_memory=pin) for _ in range(self.BUFFERS)]
        self._host_np = [h.numpy() for h in self._host]
        self._dev = [torch.empty(4 * max_rows, dtype=torch.int32, device=device) for _ in range(self.BUFFERS)]
        self._out = [torch.zeros(max_rows, dtype=torch.int32, device=device) for _ in range(self.BUFFERS)]
        self._out_host = [torch.empty(max_rows, dtype=torch.int32, pin_memory=pin) for _ in range(self.BUFFERS)]
        # the same for calls with draws, made by the first
        self._more: Optional[list] = None
        self._turn = 0

    def launch(self, logits: torch.Tensor, params: Sequence[SamplingParams],
               requests: Sequence[Hashable], steps: Sequence[int], rows: Optional[Sequence[int]] = None) -> SampleTicket:
        """Start sampling one token per row of ``logits``, or per entry of ``rows`` from the row that it names; nothing waits for the
        device."""
        if rows is not None or any(p.draws for p in params):
            return self._launch_draws(logits, params, requests, steps, range(len(params)) if rows is None else rows)
        R = logits.shape[0]
        if R > self.max_rows:
            raise ValueError(f"{R} rows to sample, the sampler was built for {self.max_rows}")
        b = self._turn
        self._turn = (self._turn + 1) % self.BUFFERS
        if R == 0:
            return SampleTicket(0, self._out[b], self._out_host[b], None)
        m = self.max_rows
        ints = self._host_np[b]
        f = ints.view(np.float32)
        for i, (p, rid, st) in enumerate(zip(params, requests, steps)):
            greedy = p.is_greedy
            f[i] = 0.0 if greedy else max(p.temperature, MIN_T)
            f[m + i] = 1.0 if greedy else min(max(p.top_p, MIN_P), 1.0)
            seed = p.seed if p.seed is not None else self.default_seed
            f[2 * m + i] = 0.0 if greedy else uniform_for(seed, rid, st)
            ints[3 * m + i] = 0 if (greedy or p.top_k < 1) else min(p.top_k, self.vocab_size)
        dev = self._dev[b]
        dev.copy_(self._host[b], non_blocking=True)
        fd = dev.view(torch.float32)
        ops.sample(logits, fd[0:m], dev[3 * m:4 * m], fd[m:2 * m], fd[2 * m:3 * m], self._out[b])
        self._out_host[b][:R].copy_(self._out[b][:R], non_blocking=True)
        event = None
        if self.device.type == "cuda":
            event = torch.cuda.Event()
            event.record()
        return SampleTicket(R, self._out[b], self._out_host[b], event)

    def _launch_draws(self, logits: torch.Tensor, params: Sequence[SamplingParams], requests: Sequence[Hashable], steps: Sequence[int],
                      rows: Sequence[int]) -> SampleTicket:
        """The requests that draw go to ``ops.sample_draws``, the others to ``ops.sample`` as ever (it takes every row: greedily where nobody
        wants that token); then every token goes to its place."""
        R, N, M = len(params), logits.shape[0], 2 * self.max_rows
        if max(R, N) > self.max_rows:
            raise ValueError(f"{max(R, N)} rows to sample, the sampler was built for {self.max_rows}")
        old, new = [i for i in range(R) if not params[i].draws], [i for i in range(R) if params[i].draws]
        if any(not 0 <= r < N for r in rows) or len({rows[i] for i in old}) != len(old):
            raise ValueError("requests that do not draw take a row each, and every row must be there")
        if self._more is None:
            pin = self.device.type == "cuda"
            self._more = [dict(host=torch.empty(8 * M, dtype=torch.int32, pin_memory=pin), dev=torch.empty(8 * M, dtype=torch.int32, device=self.device),
                               tokens=torch.zeros(M, dtype=torch.int32, device=self.device),
                               logprobs=torch.zeros(M, dtype=torch.float32, device=self.device),
                               host_logprobs=torch.empty(M, dtype=torch.float32, pin_memory=pin)) for _ in range(self.BUFFERS)]
        b = self._turn
        self._turn = (self._turn + 1) % self.BUFFERS
        more = self._more[b]
        ints = more["host"].numpy()
        f = ints.view(np.float32)
        # sections of M: temperature, top_p, u, top_k, min_p, row; the rows' places first, the draws' behind them; then (place, from) pairs
        ints[:] = 0
        f[M:2 * M] = 1.0
        for i, at in [(i, rows[i]) for i in old] + [(i, N + j) for j, i in enumerate(new)]:
            p = params[i]
            if not p.is_greedy:
                seed = p.seed if p.seed is not None else self.default_seed
                f[at] = max(p.temperature, MIN_T)
                f[M + at] = min(max(p.top_p, MIN_P), 1.0)
                f[2 * M + at] = uniform_for(seed, requests[i], steps[i])
                ints[3 * M + at] = 0 if p.top_k < 1 else min(p.top_k, self.vocab_size)
                f[4 * M + at] = p.min_p
            ints[5 * M + at] = rows[i]
            ints[6 * M + 2 * i], ints[6 * M + 2 * i + 1] = i, at
        dev, tokens, logprobs = more["dev"], more["tokens"], more["logprobs"][:len(new)]
        dev.copy_(more["host"], non_blocking=True)
        fd = dev.view(torch.float32)
        if old:
            ops.sample(logits, fd[0:N], dev[3 * M:3 * M + N], fd[M:M + N], fd[2 * M:2 * M + N], tokens)
        if new:
            of = lambda x, section: x[section * M + N:section * M + N + len(new)]  # noqa: E731
            ops.sample_draws(logits, of(dev, 5), of(fd, 0), of(dev, 3), of(fd, 1), of(fd, 4), of(fd, 2), tokens[N:N + len(new)], logprobs)
        ops.copy_tokens(self._out[b], dev[6 * M:], tokens, R, self.vocab_size)
        self._out_host[b][:R].copy_(self._out[b][:R], non_blocking=True)
        more["host_logprobs"][:len(new)].copy_(logprobs, non_blocking=True)
        event = None
        if self.device.type == "cuda":
            event = torch.cuda.Event()
            event.record()
        return SampleTicket(R, self._out[b], self._out_host[b], event, more["host_logprobs"], new)

    def logprobs(self, ticket: SampleTicket) -> List[Optional[float]]:
        """The log-probabilities of a launched call's tokens, None for those of requests that do not draw (waits for the device)."""
        out: List[Optional[float]] = [None] * ticket.n
        if ticket.drawn:
            if ticket.event is not None:
                ticket.event.synchronize()
            for i, x in zip(ticket.drawn, ticket.host_logprobs.tolist()):
                out[i] = x
        return out

    def result(self, ticket: SampleTicket) -> List[int]:
        """The tokens of a launched call (waits for the device)."""
        if ticket.event is not None:
            ticket.event.synchronize()
        return ticket.host_tokens[: ticket.n].tolist()

    def sample(self, logits: torch.Tensor, params: Sequence[SamplingParams],
               requests: Sequence[Hashable], steps: Sequence[int]) -> List[int]:
        """One token per row of ``logits`` (host list; the call waits for the device)."""
        return self.result(self.launch(logits, params, requests, steps))
