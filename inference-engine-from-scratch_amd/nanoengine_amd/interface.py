"""Request and event types (same fields as ne/engine/interface.py:8-39) plus the
sampling helpers of ne/engine/sampling.py that stay on the host."""

from __future__ import annotations

import math
import os
from collections.abc import AsyncIterator, Mapping
from dataclasses import dataclass, field
from typing import Protocol

GREEDY_TEMPERATURE = 0.0
FINISH_REASON_STOP = "stop"
FINISH_REASON_LENGTH = "length"


@dataclass(frozen=True)
class SamplingParams:
    max_new_tokens: int
    temperature: float = 0.0
    top_p: float = 1.0
    seed: int | None = None
    ignore_eos: bool = False
    top_k: int = 0  # 0: all tokens
    min_p: float = 0.0  # least probability, relative to the likeliest token's
    # logits of tokens so far: of prompt and output divided (positive ones) or multiplied by
    # repetition_penalty, of output lowered by frequency_penalty a time and presence_penalty once
    repetition_penalty: float = 1.0
    presence_penalty: float = 0.0
    frequency_penalty: float = 0.0
    logit_bias: Mapping[int, float] | None = field(default=None, hash=False)  # added to single tokens' logits

    @property
    def is_penalized(self) -> bool:
        """Whether the logits depend on the tokens so far."""
        return self.repetition_penalty != 1.0 or self.presence_penalty != 0.0 or self.frequency_penalty != 0.0

    def penalty_error(self) -> str | None:
        """Why no logits can be made under these penalties, or None.  (An infinite one bans, or forces, the
        tokens that it is for; of opposite signs two make no sum.)"""
        if not 0.0 < self.repetition_penalty < math.inf:
            return "repetition_penalty must be positive and finite"
        for name in ("presence_penalty", "frequency_penalty"):
            if math.isnan(getattr(self, name)):
                return f"{name} must not be NaN"
        if math.isnan(self.presence_penalty + self.frequency_penalty):
            return "presence_penalty and frequency_penalty must not be infinite in opposite directions"
        return None

    @property
    def is_adjusted(self) -> bool:
        """Whether the request's logits are changed before a token is picked (greedily too)."""
        return self.is_penalized or bool(self.logit_bias)

    @property
    def is_filtered(self) -> bool:
        """Whether a sampled request draws under top-k or min-p, which speculative
        verification does not take."""
        return self.temperature != GREEDY_TEMPERATURE and (self.top_k > 0 or self.min_p > 0.0)


@dataclass(frozen=True)
class GenerationRequest:
    request_id: str
    prompt_token_ids: list[int]
    sampling_params: SamplingParams


@dataclass(frozen=True)
class TokenEvent:
    request_id: str
    token_id: int
    is_finished: bool
    finish_reason: str | None


class InferenceEngine(Protocol):
    async def start(self) -> None: ...

    async def stop(self) -> None: ...

    def submit(self, request: GenerationRequest) -> AsyncIterator[TokenEvent]: ...


@dataclass
class SamplingStream:
    """Per-request randomness (the role of create_sampling_generator, sampling.py:11-18).

    Draws are Philox4x32-10 uniforms keyed by ``seed`` at counter ``step``; one
    step is one sampling event of the request (its first token, then each verify
    step), so a fixed seed always gives the same tokens.
    """

    seed: int
    step: int = 0


def create_sampling_generator(seed: int | None) -> SamplingStream:
    if seed is None:
        seed = int.from_bytes(os.urandom(8), "little") & ((1 << 63) - 1)
    return SamplingStream(seed=int(seed) & ((1 << 63) - 1))


def sampling_uniform(seed: int, step: int) -> float:
    """The uniform in [0, 1) of one draw of a stream: word 3 of Philox4x32-10 (Salmon et al.,
    SC'11) under key ``seed`` at counter (``step``, 15), its 24 leading bits, as the acceptance
    kernel takes it for its draws."""
    mask = 0xFFFFFFFF
    c = [step & mask, step >> 32 & mask, 15, 0]
    k = [seed & mask, seed >> 32 & mask]
    for i in range(10):
        if i:
            k = [(k[0] + 0x9E3779B9) & mask, (k[1] + 0xBB67AE85) & mask]
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & mask, (a >> 32) ^ c[3] ^ k[1], a & mask]
    return (c[3] >> 8) / 16777216.0


def find_finish_reason(token_id: int, num_generated_tokens: int, params: SamplingParams,
                       stop_token_ids: frozenset[int]) -> str | None:
    """sampling.py:54-62: ``stop`` on a stop token unless ignore_eos, ``length`` at the limit."""
    if not params.ignore_eos and token_id in stop_token_ids:
        return FINISH_REASON_STOP
    if num_generated_tokens >= params.max_new_tokens:
        return FINISH_REASON_LENGTH
    return None


def num_guesses(params: SamplingParams, num_generated_tokens: int, k: int) -> int:
    """speculative_generator.py:71-72: never guess past the length limit."""
    return max(0, min(k, params.max_new_tokens - num_generated_tokens - 1))
