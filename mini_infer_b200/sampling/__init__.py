"""Greedy, temperature, top-k and top-p sampling; penalties, biases and masks on the logits before it."""

from .adjust import AdjustedRow, LogitsAdjuster, mask_any, mask_words  # noqa: F401
from .params import SamplingParams  # noqa: F401
from .sampler import DeviceSampler, default_seed  # noqa: F401
