"""Per-request state passed between drafter, verifier and commit.

Same fields, defaults and behaviour as src/myvllm/engine/sequence.py:8-92
(the state type of the reference's drafter/verifier API): drafters append
their drafts with ``append_token`` and record them in ``draft_tokens``; the
commit step truncates ``token_ids`` back to the accepted length.
"""

from __future__ import annotations

import math
from copy import copy
from enum import Enum, auto
from itertools import count

from naivllm_amd.sampling_parameters import SamplingParams


class SequenceStatus(Enum):
    WAITING = auto()
    RUNNING = auto()
    FINISHED = auto()


class Sequence:
    block_size = 256  # tokens per KV page
    counter = count()

    def __init__(self, token_ids: list[int], sampling_params: SamplingParams = SamplingParams()):
        self.seq_id = next(Sequence.counter)
        self.status = SequenceStatus.WAITING
        self.token_ids = copy(token_ids)
        self.last_token = self.token_ids[-1] if self.token_ids else None
        self.num_tokens = len(self.token_ids)
        self.num_prompt_tokens = len(self.token_ids)
        self.num_cached_tokens = 0
        self.block_table: list[int] = []
        self.draft_block_table: list[int] = []
        self.draft_num_cached_tokens = 0
        self.draft_tokens: list[int] = []
        self.temperature = sampling_params.temperature
        self.max_tokens = sampling_params.max_tokens
        self.ignore_eos = sampling_params.ignore_eos
        self.max_model_length = sampling_params.max_model_length
        # (a caller's own settings, of the reference's fields, have no filters)
        self.top_k = max(0, min(int(getattr(sampling_params, "top_k", 0)), 0x7fffffff))
        self.top_p = getattr(sampling_params, "top_p", 1.0)
        self.min_p = getattr(sampling_params, "min_p", 0.0)

    def __len__(self):
        return self.num_tokens

    def __getitem__(self, idx):
        return self.token_ids[idx]

    @property
    def filtered(self):
        """Whether a top-k, top-p or min-p narrows what is sampled."""
        return self.temperature > 1e-6 and (self.top_k > 0 or self.top_p < 1 or self.min_p > 0)

    @property
    def is_finished(self):
        return self.status == SequenceStatus.FINISHED

    @property
    def num_completion_tokens(self):
        return self.num_tokens - self.num_prompt_tokens

    @property
    def prompt_token_ids(self):
        return self.token_ids[:self.num_prompt_tokens]

    @property
    def completion_token_ids(self):
        return self.token_ids[self.num_prompt_tokens:]

    @property
    def num_cached_blocks(self):
        return int(math.ceil(self.num_cached_tokens / self.block_size))

    @property
    def num_blocks(self):
        return int(math.ceil(self.num_tokens / self.block_size))

    @property
    def last_block_num_tokens(self):
        if self.num_tokens == 0:
            return 0
        return self.num_tokens % self.block_size or self.block_size

    def block(self, i):
        assert 0 <= i < self.num_blocks, f"Block index {i} out of range [0, {self.num_blocks})"
        start = i * self.block_size
        return self.token_ids[start:min(start + self.block_size, self.num_tokens)]

    def append_token(self, token_id):
        self.token_ids.append(token_id)
        self.last_token = token_id
        self.num_tokens += 1
