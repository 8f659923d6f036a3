"""Per-request sampling parameters, with the reference's names, defaults and greedy rule
(python/freetoken/core.py:18-31).  ``seed`` is added: draws are a function of (seed, request,
step) only, so they do not depend on what else is in the batch.  ``min_p`` (tokens of less than that share of the likeliest one's
probability are left out) and ``n`` (how many continuations of the prompt are wanted; the prompt is read once) are added too."""

from __future__ import annotations

from dataclasses import dataclass, field
from typing import List, Optional

from ..errors import ConfigError


@dataclass
class SamplingParams:
    temperature: float = 0.0
    top_k: int = -1
    top_p: float = 1.0
    ignore_eos: bool = False
    max_tokens: int = 1024
    stop_strs: List[str] = field(default_factory=list)
    seed: Optional[int] = None
    min_p: float = 0.0
    n: int = 1

    def __post_init__(self) -> None:
        if self.max_tokens < 1:
            raise ConfigError(f"max_tokens must be >= 1, got {self.max_tokens}")
        if not 0.0 < self.top_p <= 1.0:
            raise ConfigError(f"top_p must be in (0, 1], got {self.top_p}")
        if not 0.0 <= self.min_p <= 1.0:
            raise ConfigError(f"min_p must be in [0, 1], got {self.min_p}")
        if self.n < 1:
            raise ConfigError(f"n must be >= 1, got {self.n}")
        if self.stop_strs:
            raise ConfigError("stop_strs need a tokenizer, which this engine does not carry; "
                              "stop on token ids through eos_token_id instead")

    @property
    def is_greedy(self) -> bool:
        return (self.temperature <= 0.0 or self.top_k == 1) and self.top_p == 1.0

    @property
    def draws(self) -> bool:
        """Whether tokens come from ``ops.sample_draws`` (with their log-probabilities) and not from ``ops.sample``."""
        return self.n > 1 or self.min_p > 0.0
