"""What requests ask of their logits before a token is chosen, on the device (the kernels are ``csrc/logits.cu``).

``LogitsAdjuster`` keeps the token histories that penalties read, on the device, one slot per request that asks for one, and on the host the
masks of requests whose tokens are limited for good.  ``apply`` changes a step's logits in place (options, biases and masks go to the device
with every step, in one copy); ``record`` puts the tokens that were chosen into the
histories, on the device and in stream order, so that the next step may be launched before the host has seen them.
"""

from __future__ import annotations

from typing import Hashable, Sequence

import numpy as np
import torch

from ..csrc import ops
from .params import SamplingParams


def mask_words(ids: Sequence[int], vocab_size: int) -> np.ndarray:
    """int32 ``[ceil(V / 32)]`` with bit ``t % 32`` of word ``t / 32`` set for every token ``t``."""
    flags = np.zeros(-(-vocab_size // 32) * 32, dtype=np.uint8)
    at = np.asarray(list(ids), dtype=np.int64)
    if at.size and not (0 <= at.min() and at.max() < vocab_size):
        raise ValueError(f"a mask names a token outside [0, {vocab_size})")
    flags[at] = 1
    return np.packbits(flags.reshape(-1, 32), axis=1, bitorder="little").view("<i4").reshape(-1)


def mask_any(words: np.ndarray, vocab_size: int) -> bool:
    """Whether a mask leaves a token of the vocabulary."""
    whole, rest = divmod(vocab_size, 32)
    return bool(words[:whole].any()) or bool(rest and int(words[whole]) & ((1 << rest) - 1))


class AdjustedRow:
    """One row of a step's logits: the request, its options, its tokens so far, and the words of the mask that its grammar sets for
    this token (None: none; ``LogitsAdjuster.mask_of`` makes them the row's whole mask)."""

    __slots__ = ("rid", "params", "prompt", "generated", "words")

    def __init__(self, rid: Hashable, params: SamplingParams, prompt: Sequence[int], generated: Sequence[int],
                 words: np.ndarray | None = None) -> None:
        self.rid, self.params, self.prompt, self.generated, self.words = rid, params, prompt, generated, words

    @property
    def plain(self) -> bool:
        return self.words is None and not self.params.adjusted


class LogitsAdjuster:
    def __init__(self, device, vocab_size: int, slots: int) -> None:
        self.device = torch.device(device)
        self.vocab_size = int(vocab_size)
        self.slots = int(slots)
        self._free = list(range(self.slots - 1, -1, -1))
        self._slot: dict[Hashable, int] = {}
        self._limits: dict[Hashable, np.ndarray] = {}
        self.counts = self.seen = None

    def forget(self, rid: Hashable) -> None:
        """The request is gone (or comes back later with all its tokens): its slot may be another's from now on."""
        slot = self._slot.pop(rid, None)
        if slot is not None:
            self._free.append(slot)
        self._limits.pop(rid, None)

    def _upload(self, arrays: Sequence[np.ndarray]) -> list[torch.Tensor]:
        """The arrays (4 bytes an element) as device tensors, in one copy; each begins at a multiple of 16 bytes."""
        sizes = [-(-a.size // 4) * 4 for a in arrays]
        host = torch.empty(max(4, sum(sizes)), dtype=torch.int32, pin_memory=True)
        view, at = host.numpy(), 0
        for a, n in zip(arrays, sizes):
            view[at:at + a.size] = np.ascontiguousarray(a).view(np.int32).reshape(-1)
            at += n
        dev, out, at = host.to(self.device, non_blocking=True), [], 0
        for a, n in zip(arrays, sizes):
            t = dev[at:at + a.size]
            out.append(t.view(torch.float32) if a.dtype == np.float32 else t)
            at += n
        return out

    def _admit(self, rows: Sequence[AdjustedRow]) -> None:
        """Histories for requests that have none yet, from their tokens so far."""
        new = [r for r in rows if r.params.penalised and r.rid not in self._slot]
        if not new:
            return
        if self.counts is None:
            self.counts = torch.zeros((self.slots, self.vocab_size), dtype=torch.int32, device=self.device)
            self.seen = torch.zeros((self.slots, -(-self.vocab_size // 32)), dtype=torch.int32, device=self.device)
        for r in new:
            if not self._free:
                raise RuntimeError(f"token histories for {self.slots} requests are all taken")
            self._slot[r.rid] = self._free.pop()
        lengths = [len(r.prompt) + len(r.generated) for r in new]
        tokens = np.concatenate([np.asarray(list(r.prompt) + list(r.generated), dtype=np.int32) for r in new])
        slots, starts, n_prompt, tokens = self._upload([
            np.array([self._slot[r.rid] for r in new], dtype=np.int32), np.cumsum([0] + lengths).astype(np.int32),
            np.array([len(r.prompt) for r in new], dtype=np.int32), tokens])
        ops.record_tokens(self.counts, self.seen, slots, starts, tokens, n_prompt=n_prompt, fresh=True)

    def mask_of(self, row: AdjustedRow) -> np.ndarray | None:
        """The row's mask: what it is limited to for good and what its grammar allows now, without the tokens that a bias rules out (so
        that a mask with a bit has a token that may come)."""
        allowed, never = row.params.allowed_token_ids, row.params.never
        if allowed is None and (row.words is None or not never):
            return row.words
        if row.rid not in self._limits:
            whole = np.full(-(-self.vocab_size // 32), -1, dtype=np.int32) if allowed is None else mask_words(allowed, self.vocab_size)
            self._limits[row.rid] = whole & ~mask_words(never, self.vocab_size)
        return self._limits[row.rid] if row.words is None else self._limits[row.rid] & row.words

    def apply(self, logits: torch.Tensor, rows: Sequence[AdjustedRow]) -> None:
        """What ``rows`` ask for, row by row, on fp32 ``logits [len(rows), V]`` in place."""
        if logits.shape != (len(rows), self.vocab_size):
            raise ValueError(f"logits {tuple(logits.shape)} for {len(rows)} rows of {self.vocab_size}")
        if all(r.plain for r in rows):
            return
        self._admit(rows)
        args: dict = {}
        arrays: list[np.ndarray] = []
        names: list[str] = []

        def put(name: str, values, dtype) -> None:
            names.append(name)
            arrays.append(np.asarray(values, dtype=dtype))

        if any(r.params.penalised for r in rows):
            put("slots", [self._slot[r.rid] if r.params.penalised else -1 for r in rows], np.int32)
            put("repetition", [r.params.repetition_penalty for r in rows], np.float32)
            put("presence", [r.params.presence_penalty for r in rows], np.float32)
            put("frequency", [r.params.frequency_penalty for r in rows], np.float32)
        biases = [r.params.logit_bias or () for r in rows]
        if any(biases):
            put("starts", np.cumsum([0] + [len(b) for b in biases]), np.int32)
            put("ids", [t for b in biases for t, _ in b], np.int32)
            put("values", [v for b in biases for _, v in b], np.float32)
        words = [self.mask_of(r) for r in rows]
        masked = [w for w in words if w is not None]
        if masked:
            number = iter(range(len(masked)))
            put("mask_rows", [-1 if w is None else next(number) for w in words], np.int32)
            put("masks", np.stack(masked), np.int32)
        args = dict(zip(names, self._upload(arrays)))
        if "slots" in args:
            args.update(counts=self.counts, seen=self.seen)
        if "starts" in args:
            args["bias"] = (args.pop("starts"), args.pop("ids"), args.pop("values"))
        if "masks" in args:
            args["masks"] = args["masks"].view(len(masked), -1)
        ops.adjust_logits(logits, logits, **args)

    def record(self, tokens: torch.Tensor, rows: Sequence[AdjustedRow]) -> None:
        """The chosen ``tokens`` (int32 on the device, one per row) into the histories of the rows that have one."""
        if not any(r.params.penalised for r in rows):
            return
        if not isinstance(tokens, torch.Tensor) or not tokens.is_cuda:
            tokens = torch.as_tensor(tokens, dtype=torch.int32).to(self.device)
        slots, = self._upload([np.array([self._slot.get(r.rid, -1) for r in rows], dtype=np.int32)])
        ops.record_tokens(self.counts, self.seen, slots, None, tokens)
