"""Sampling options of a request.

Names, defaults and checks are the reference's (``engine/sampler.py:7-21``):
``temperature`` 0 means greedy, ``top_k`` 0 and ``top_p`` 1.0 switch the filters off.
What follows ``seed`` is this engine's addition, and applies to the logits in this order before everything else:

* ``repetition_penalty``: a token of the prompt or the answer has its logit divided by it (multiplied where negative); 1 is off;
* ``frequency_penalty``, ``presence_penalty``: the logit of a token that the answer holds ``c > 0`` times loses
  ``frequency_penalty * c + presence_penalty``; 0 is off;
* ``logit_bias``: a number added to the logits of given tokens (minus infinity: never);
* ``allowed_token_ids``: no other token is ever chosen.

``seed`` is an addition too: the reference draws from torch's global generator,
here every request has a seed of its own and token ``n`` of a request is drawn from
``(seed, n)`` alone, so results do not depend on what else is in the batch.
"""

from __future__ import annotations

import dataclasses
import math
from typing import Mapping, Sequence


_FP32_LEAST, _FP32_MOST = 2.0 ** -126, (2.0 - 2.0 ** -23) * 2.0 ** 127


@dataclasses.dataclass(frozen=True)
class SamplingParams:
    temperature: float = 0.0
    top_k: int = 0
    top_p: float = 1.0
    seed: int | None = None
    repetition_penalty: float = 1.0
    frequency_penalty: float = 0.0
    presence_penalty: float = 0.0
    logit_bias: Mapping[int, float] | None = None
    allowed_token_ids: Sequence[int] | None = None

    def __post_init__(self) -> None:
        if self.temperature < 0:
            raise ValueError(f"temperature must be >= 0, got {self.temperature}")
        if self.top_k < 0:
            raise ValueError(f"top_k must be >= 0, got {self.top_k}")
        if not 0.0 <= self.top_p <= 1.0:
            raise ValueError(f"top_p must be in [0, 1], got {self.top_p}")
        if self.seed is not None and not 0 <= self.seed < 2 ** 64:
            raise ValueError(f"seed must fit 64 bits, got {self.seed}")
        # (what the device computes with are fp32 numbers)
        if not _FP32_LEAST <= self.repetition_penalty <= _FP32_MOST:
            raise ValueError(f"repetition_penalty must be positive, got {self.repetition_penalty}")
        for name in ("frequency_penalty", "presence_penalty"):
            if not abs(getattr(self, name)) <= _FP32_MOST:
                raise ValueError(f"{name} must be a number, got {getattr(self, name)}")
        if self.logit_bias is not None:
            items = tuple((int(t), float(b)) for t, b in dict(self.logit_bias).items())
            if any(t < 0 or not (abs(b) <= _FP32_MOST or b == -math.inf) for t, b in items):
                raise ValueError(f"logit_bias gives numbers (or minus infinity) to token ids, got {self.logit_bias}")
            object.__setattr__(self, "logit_bias", items)       # hashable, and nobody's to change
        if self.allowed_token_ids is not None:
            ids = tuple(sorted({int(t) for t in self.allowed_token_ids}))
            if not ids or ids[0] < 0:
                raise ValueError("allowed_token_ids must name at least one token")
            if not set(ids) - set(self.never):
                raise ValueError("logit_bias rules out every token of allowed_token_ids")
            object.__setattr__(self, "allowed_token_ids", ids)

    @property
    def greedy(self) -> bool:
        return self.temperature == 0.0

    @property
    def never(self) -> tuple[int, ...]:
        """The tokens whose bias is minus infinity."""
        return tuple(t for t, b in self.logit_bias or () if b == -math.inf)

    @property
    def penalised(self) -> bool:
        """Whether the logits depend on the tokens so far."""
        return self.repetition_penalty != 1.0 or self.frequency_penalty != 0.0 or self.presence_penalty != 0.0

    @property
    def adjusted(self) -> bool:
        """Whether the logits are changed at all before a token is chosen."""
        return self.penalised or bool(self.logit_bias) or self.allowed_token_ids is not None

    def check_vocabulary(self, vocab_size: int) -> None:
        if len(self.never) == vocab_size:
            raise ValueError("logit_bias rules out every token")
        for t, _ in self.logit_bias or ():
            if t >= vocab_size:
                raise ValueError(f"logit_bias names token {t} of {vocab_size}")
        if self.allowed_token_ids is not None and self.allowed_token_ids[-1] >= vocab_size:
            raise ValueError(f"allowed_token_ids names token {self.allowed_token_ids[-1]} of {vocab_size}")
