"""Draws at their ends: calls of different sizes at once, rows that fill the shared memory of a cluster of sixteen."""

import threading

import numpy as np
import pytest
import torch

from freetoken_b200.kernels import ops
from test_sample_draws_gpu import DEV, check


@pytest.mark.gpu
def test_calls_of_different_sizes_from_two_threads():
    rng = np.random.default_rng(5)
    wrong = []
    ops.check_status()  # (the library is there)

    def calls(vocab, R):
        try:
            x = torch.from_numpy(rng.normal(0, 2, (R, vocab)).astype(np.float32)).to(DEV)
            f = lambda v: torch.full((R,), v, dtype=torch.float32, device=DEV)  # noqa: E731
            args = (x, None, f(1.0), torch.zeros(R, dtype=torch.int32, device=DEV), f(0.9), f(0.0), f(0.5))
            stream = torch.cuda.Stream()
            stream.wait_stream(torch.cuda.default_stream())
            with torch.cuda.stream(stream):
                want, out = (torch.empty(R, dtype=torch.int32, device=DEV) for _ in range(2))
                ops.sample_draws(*args, want)
                for _ in range(3000):
                    ops.sample_draws(*args, out)
                stream.synchronize()
            assert torch.equal(out, want)
        except Exception as e:
            wrong.append(repr(e))

    threads = [threading.Thread(target=calls, args=s) for s in ((400000, 6), (400, 6), (100000, 3), (400, 2), (300, 3), (200000, 1))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong, wrong


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,R", [(440001, 3), (440001, 9), (870001, 3), (900001, 3)])
def test_rows_that_a_cluster_just_holds(vocab, R):
    """Clusters of sixteen for few draws, of eight for more: with as much shared memory as a CTA may have, and a little beyond."""
    rng = np.random.default_rng(vocab)
    x = rng.normal(0, 3, (2, vocab)).astype(np.float32)
    check(x, np.arange(R) % 2, np.resize([1.0, 0.7, 1.0], R), np.resize([0, 50, 0], R), np.resize([1.0, 0.9, 0.95], R),
          np.resize([0.0, 0.0, 1e-4], R), rng.random(R))
