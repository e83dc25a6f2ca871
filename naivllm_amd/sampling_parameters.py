"""Per-request sampling settings, as src/myvllm/sampling_parameters.py:4-13
(same fields, defaults and check): temperature 0 selects greedy decoding,
which the acceptance step treats as temperature <= 1e-6.

``top_k``, ``top_p`` and ``min_p`` are this build's additions: the filters of
rejection_sampler.sample_filtered, off by default."""

from __future__ import annotations

import numbers
from dataclasses import dataclass


@dataclass
class SamplingParams:
    temperature: float = 1.0
    max_tokens: int = 64                  # completion tokens at most
    ignore_eos: bool = False
    max_model_length: int | None = None   # prompt + completion tokens at most
    top_k: int = 0                        # the most likely tokens that stay (0: all)
    top_p: float = 1.0                    # the fewest whose probabilities reach it stay
    min_p: float = 0.0                    # those of at least this share of the largest probability stay

    def __post_init__(self):
        assert self.temperature == 0 or self.temperature >= 1e-6, "temperature must be 0 (greedy) or >= 1e-6"
        if isinstance(self.top_k, bool) or not isinstance(self.top_k, numbers.Integral) or self.top_k < 0:
            raise ValueError(f"top_k must be an integer from 0 on, got {self.top_k!r}")
        if not 0 < self.top_p <= 1:
            raise ValueError(f"top_p must be above 0 and at most 1, got {self.top_p!r}")
        if not 0 <= self.min_p <= 1:
            raise ValueError(f"min_p must be from 0 to 1, got {self.min_p!r}")
