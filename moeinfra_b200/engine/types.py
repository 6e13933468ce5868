"""Engine request/result types (API of the reference's ``engine/types.py``)."""
from __future__ import annotations

import dataclasses
import enum
from typing import Optional

import torch


class PrefetchPolicy(enum.Enum):
    NONE = "none"
    NEXT_LAYER = "next_layer"
    LOOKAHEAD = "lookahead"


@dataclasses.dataclass
class SamplingParams:
    """How tokens are drawn (``kernels.sample_tokens``): each a number, or one per sequence.

    temperature 0 is greedy; top_k 0, top_p 1 and min_p 0 are off.  ``seed``: the same seed, prompts
    and parameters give the same tokens; None draws from torch's global generator.
    """
    temperature: float | list = 1.0
    top_k: int | list = 0
    top_p: float | list = 1.0
    min_p: float | list = 0.0
    seed: Optional[int] = None


@dataclasses.dataclass
class ForwardRequest:
    input_ids: torch.Tensor
    attention_mask: Optional[torch.Tensor] = None
    max_new_tokens: int = 128
    sampling: Optional[SamplingParams] = None  # None: greedy
    num_beams: int = 1  # above 1: beam search (engine.paged_kv)


@dataclasses.dataclass
class ForwardResult:
    logits: torch.Tensor  # [sequences, 1, vocab]: what each sequence's last token was chosen from
    token_ids: list
    ttft_ms: float
    tps: float
    stage_timings: dict
    scores: Optional[list] = None  # beam search: each sequence's sum of log-probabilities
