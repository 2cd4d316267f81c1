"""Sampling options, with the names and meanings of the reference's
SamplingConfig (src/core/sampler/LLMSampler.h:55-63): ``_type``,
``_temperature``, ``_top_k``, ``_top_p``, ``_min_p``, ``_repetition_penalty``,
``_seed`` there, the same without the underscore here."""
from __future__ import annotations

import math
from dataclasses import dataclass, field
from typing import Callable

import numpy as np

#: strategy names of the reference (src/core/sampler/LLMSampler.h:18-24)
STRATEGIES = ("default", "unknown", "greedy", "random", "top_k", "top_p")

#: the device has the options in float32, where a larger number is infinite: a logit that it makes infinite has no softmax
_FLOAT32_MAX = float(np.finfo(np.float32).max)


@dataclass
class SamplingConfig:
    """``type`` 'greedy' (and 'default', as the reference's ``sample()`` always
    takes the argmax, src/core/sampler/LLMSampler.cpp:13-19) picks the first
    maximum.  'random', 'top_k' and 'top_p' draw from softmax(logits /
    temperature), restricted to the ``top_k`` most likely tokens (0: off), to
    the most likely tokens whose mass reaches ``top_p`` (1: off) and to tokens
    with probability at least ``min_p`` times the largest (0: off).
    ``temperature`` 0 also means greedy.  ``repetition_penalty`` divides the
    positive and multiplies the other logits of tokens already in the prompt or
    the output (LLMSampler.cpp:21-34).  The draw for output token i of a
    request depends only on (seed, i), not on what else is in the batch.

    ``presence_penalty`` comes off the logits of tokens in the output,
    ``frequency_penalty`` as often as they stand there; ``logit_bias`` {token:
    number} is added to single tokens' logits (-inf: never).  ``allowed`` is
    called before every draw with the output so far (int32) and says what may
    come next: int32 or uint32 [ceil(vocabulary / 32)], a bit a token, lowest
    first, or None for all.  It may be called more than once for a place (a
    step that failed runs again).  A mask without a single token leaves token
    0, which it does not allow: the place is listed in the result's
    ``unallowed`` and a warning logged.  A grammar that has come to its end
    allows the stop token, or raises, which leaves the requests where they are.
    """
    type: str = "greedy"
    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0
    repetition_penalty: float = 1.0
    seed: int = 0
    presence_penalty: float = 0.0
    frequency_penalty: float = 0.0
    logit_bias: dict | None = None
    allowed: Callable[[np.ndarray], np.ndarray | None] | None = field(default=None, compare=False)

    def __post_init__(self):
        if self.type not in STRATEGIES or self.type == "unknown":
            raise ValueError(f"unknown sampling strategy '{self.type}'; known: {STRATEGIES}")
        if self.temperature < 0:
            raise ValueError("temperature must not be negative")
        if self.top_k < 0 or not (0 < self.top_p <= 1) or not (0 <= self.min_p <= 1):
            raise ValueError("top_k >= 0, 0 < top_p <= 1 and 0 <= min_p <= 1 are required")
        if self.repetition_penalty <= 0:
            raise ValueError("repetition_penalty must be positive")
        if not (abs(self.presence_penalty) <= _FLOAT32_MAX and abs(self.frequency_penalty) <= _FLOAT32_MAX):
            raise ValueError("presence_penalty and frequency_penalty must be numbers of float32's range")
        if self.allowed is not None and not callable(self.allowed):
            raise ValueError("allowed must be a function of the output so far")
        if self.logit_bias is not None:
            self.logit_bias = {int(t): float(b) for t, b in self.logit_bias.items()}
            if any(not b <= _FLOAT32_MAX for b in self.logit_bias.values()) or any(not 0 <= t < 1 << 31 for t in self.logit_bias):
                raise ValueError("logit_bias: tokens must not be negative, biases numbers of float32's range (or -inf, never again)")
            self.logit_bias = {t: b if b >= -_FLOAT32_MAX else -math.inf for t, b in self.logit_bias.items()}

    @property
    def adjusts(self) -> bool:
        """Whether the logits are changed by more than a repetition penalty."""
        return bool(self.presence_penalty or self.frequency_penalty or self.logit_bias) or self.allowed is not None

    @property
    def needs_output(self) -> bool:
        """Whether a token's choice depends on the tokens before it other than through the model."""
        return bool(self.repetition_penalty != 1.0 or self.presence_penalty or self.frequency_penalty) or self.allowed is not None

    @property
    def greedy(self) -> bool:
        return self.type in ("greedy", "default") or self.temperature == 0

    def effective(self):
        """(temperature, top_k, top_p, min_p) the kernel gets; temperature 0 = argmax."""
        if self.greedy:
            return 0.0, 0, 1.0, 0.0
        return float(self.temperature), int(self.top_k), float(self.top_p), float(self.min_p)
