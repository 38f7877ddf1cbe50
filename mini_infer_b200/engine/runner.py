"""``ModelRunner``: a loaded model, its cache and its step function in one object.

``ModelRunner.from_pretrained(model_dir, dtype=..., num_blocks=..., block_size=...)`` follows
the reference's constructor of the same name (``engine/model_runner.py:84-175``; the option
names ``num_blocks`` and ``block_size`` and their defaults 1024 and 16 are the reference's),
reduced to what a single-GPU engine for local model folders needs.
"""

from __future__ import annotations

import os
import threading
from contextlib import contextmanager
from typing import Any, Iterator, Mapping, Sequence

import torch

from ..cache.manager import CacheManager
from ..config.registry import load_config
from ..parts.adapters import AdapterBank
from ..parts.model import DecoderModel
from ..weights.adapters import adapter_scale, pair_matrices, read_adapter
from ..weights.loader import WeightLoadError, bind_state_dict, load_weights
from .step import StepEntry, StepResult, StepRunner

DTYPES = {
    "bfloat16": torch.bfloat16, "bf16": torch.bfloat16,
    "float32": torch.float32, "fp32": torch.float32,
    torch.bfloat16: torch.bfloat16, torch.float32: torch.float32,
}

DEFAULT_NUM_BLOCKS = 1024
DEFAULT_BLOCK_SIZE = 16


def resolve_dtype(dtype) -> torch.dtype:
    try:
        return DTYPES[dtype]
    except KeyError:
        raise ValueError(f"dtype must be bfloat16 or float32, got {dtype!r}") from None


def require_cuda(device) -> torch.device:
    device = torch.device(device)
    if device.type != "cuda":
        raise RuntimeError(f"the engine runs on a CUDA device only, got {device}")
    if not torch.cuda.is_available():
        raise RuntimeError("no CUDA device is available; the engine has no CPU path")
    return device


class ModelRunner:
    def __init__(self, model: DecoderModel, config: Any, *, num_blocks: int = DEFAULT_NUM_BLOCKS,
                 block_size: int = DEFAULT_BLOCK_SIZE, max_requests: int = 64,
                 cuda_graph: bool = False) -> None:
        self.model = model
        self.config = config
        self.dtype = model.dtype
        self.device = model.device
        self.cache = CacheManager(
            model.cache_needs(), page_size=block_size, num_pages=num_blocks,
            max_requests=max_requests, dtype=self.dtype, device=self.device,
            max_request_tokens=model.spec.max_positions,
        )
        self.stepper = StepRunner(model, self.cache, cuda_graph=cuda_graph)
        self.vocab_size = model.spec.vocab_size
        self.max_positions = model.spec.max_positions
        self.num_blocks = num_blocks
        self.block_size = block_size
        self._adapter_names: list[str | None] | None = None      # by index; None: adapters are off
        # Requests come from any thread and never wait for a load: names and users have a lock of their own, held for moments (the
        # innermost one); whoever changes which adapters there are holds the outer one meanwhile.
        self._adapter_lock = threading.RLock()
        self._adapter_changes = threading.RLock()
        # A step, which may be recorded as a graph, or work on the adapters' banks by another thread: one after the other on the
        # host, and in that order on the device whatever streams the two are on.
        self._device_lock = threading.RLock()
        self._step_stream: torch.cuda.Stream | None = None       # of the last step since adapters are on
        self._banks_written: torch.cuda.Event | None = None      # behind work on the banks that no step has waited for yet

    @classmethod
    def from_pretrained(cls, model_dir: str | os.PathLike, *, device="cuda:0", dtype="bfloat16",
                        num_blocks: int = DEFAULT_NUM_BLOCKS, block_size: int = DEFAULT_BLOCK_SIZE,
                        max_requests: int = 64, cuda_graph: bool = False) -> "ModelRunner":
        """Load ``config.json`` and the safetensors of a local model folder.  ``cuda_graph``
        replays decode-only steps as captured CUDA graphs (the reference's option of that name)."""
        device = require_cuda(device)
        tdtype = resolve_dtype(dtype)
        arch, cfg = load_config(model_dir)
        model = DecoderModel(arch.assemble(cfg))
        load_weights(model, model_dir, tdtype, device)
        return cls(model, cfg, num_blocks=num_blocks, block_size=block_size, max_requests=max_requests,
                   cuda_graph=cuda_graph)

    @classmethod
    def from_state_dict(cls, raw_config: Mapping[str, Any], state: Mapping[str, torch.Tensor], *,
                        device="cuda:0", dtype="bfloat16", num_blocks: int = DEFAULT_NUM_BLOCKS,
                        block_size: int = DEFAULT_BLOCK_SIZE, max_requests: int = 64,
                        cuda_graph: bool = False) -> "ModelRunner":
        """Build from a raw configuration mapping and tensors already in memory."""
        device = require_cuda(device)
        tdtype = resolve_dtype(dtype)
        arch, cfg = load_config(raw_config)
        model = DecoderModel(arch.assemble(cfg))
        bind_state_dict(model, dict(state), tdtype, device)
        return cls(model, cfg, num_blocks=num_blocks, block_size=block_size, max_requests=max_requests,
                   cuda_graph=cuda_graph)

    @classmethod
    def from_random(cls, raw_config: Mapping[str, Any], seed: int, *, device="cuda:0", dtype="bfloat16",
                    num_blocks: int = DEFAULT_NUM_BLOCKS, block_size: int = DEFAULT_BLOCK_SIZE,
                    max_requests: int = 64, cuda_graph: bool = False, std: float = 0.02,
                    gain_std: float = 0.1, std_overrides: Mapping[str, float] | None = None) -> "ModelRunner":
        """Build from a raw configuration mapping with the random weights of ``seed`` (the ones
        ``write_random_model`` writes), drawn on the device part by part: a model of tens of
        gigabytes needs neither a file nor host memory, and nothing exists twice."""
        from ..weights.random_init import bind_random

        device = require_cuda(device)
        tdtype = resolve_dtype(dtype)
        arch, cfg = load_config(raw_config)
        model = DecoderModel(arch.assemble(cfg))
        bind_random(model, seed, tdtype, device, std=std, gain_std=gain_std, std_overrides=std_overrides)
        return cls(model, cfg, num_blocks=num_blocks, block_size=block_size, max_requests=max_requests,
                   cuda_graph=cuda_graph)

    # -- adapters -----------------------------------------------------------------------

    @contextmanager
    def _between_steps(self) -> Iterator[None]:
        """Work on the adapters' banks: behind every step before it, and in front of every step behind it."""
        with self._device_lock:
            if self.device.type != "cuda":
                yield
                return
            stream = torch.cuda.current_stream(self.device)
            if self._step_stream is not None:
                stream.wait_stream(self._step_stream)
            if self._banks_written is not None:
                stream.wait_event(self._banks_written)
            try:
                yield
            finally:
                self._banks_written = stream.record_event()

    def enable_adapters(self, count: int = 8, rank: int = 16) -> None:
        """Make room for ``count`` low-rank adapters of rank up to ``rank`` beside every product of the model that takes them
        (``Part.adapted``).  Once, before the first is loaded.  Steps with adapters are recorded when they first occur, or ahead
        where ``capture_decode_steps`` (a scheduler's ``start``) comes behind this."""
        if count <= 0 or rank <= 0:
            raise ValueError(f"room for {count} adapters of rank {rank}")
        if rank > 256:
            raise ValueError(f"adapters of rank {rank}: at most 256")
        if count > 1024:
            raise ValueError(f"{count} adapters: at most 1024")
        with self._adapter_changes:
            if self._adapter_names is not None:
                raise ValueError("adapters are enabled already")
            held = -(-rank // 8) * 8          # whole pieces of 16 bytes
            parts = [p for p in self.model.all_parts() if p.adapted()]
            if not parts:
                raise ValueError("no part of this model takes adapters")
            with self._between_steps():
                # (all of them or, where memory runs out, none)
                banks = [{q.name: AdapterBank(q, count, held, self.dtype, self.device) for q in p.adapted()} for p in parts]
                for p, mine in zip(parts, banks):
                    p.banks = mine
                self.stepper.adapter_count = count
            with self._adapter_lock:
                self._adapter_names = [None] * count
                self._adapter_users = [0] * count
                self._adapter_rank = rank

    def load_adapter(self, name: str, source, config: Mapping[str, Any] | None = None) -> int:
        """Load an adapter under ``name`` and return its index: ``source`` is a folder (``weights.read_adapter``), or the adapter's
        tensors by name with ``config`` (``r``, the rank of all its matrices, and ``lora_alpha``).  Adapters need not be enabled
        before: room for eight of this one's rank is then made.  Any thread may load while requests are served; steps wait while the
        matrices are copied (rank 16 beside all products of an 8B model: 27 to 41 ms)."""
        if isinstance(source, (str, os.PathLike)):
            if config is not None:
                raise ValueError("a folder brings its own configuration")
            config, source = read_adapter(source)
        if config is None:
            raise ValueError("an adapter's tensors need its configuration")
        matrices, scale = pair_matrices(source), adapter_scale(config)
        rank = int(config["r"])
        others = sorted(n for n, (a, _) in matrices.items() if a.shape[0] != rank)
        if others:
            raise WeightLoadError(f"adapter {name!r}: r is {rank}, matrices of other ranks: {others}", mismatched=others)
        takes: dict[str, tuple[int, int]] = {}
        for p in self.model.all_parts():
            for q in p.adapted():
                for local, width in zip(q.tensors, q.widths):
                    takes[p.spec.tensor_name(local)] = (width, q.inputs)
        # (an adapter's files never say whether the tensor's own name ends in ".weight")
        matrices = {n if n in takes else n.removesuffix(".weight") if n.removesuffix(".weight") in takes else n: m for n, m in matrices.items()}
        unknown = sorted(n for n in matrices if n not in takes)
        wrong = sorted((n, takes[n], (b.shape[0], a.shape[1])) for n, (a, b) in matrices.items()
                       if n in takes and takes[n] != (b.shape[0], a.shape[1]))
        if unknown or wrong:
            raise WeightLoadError(f"adapter {name!r} does not fit the model: "
                                  + "; ".join(filter(None, [f"no product that takes adapters: {unknown}" if unknown else "",
                                                            f"sizes (expected, found): {wrong}" if wrong else ""])),
                                  unexpected=unknown, mismatched=wrong)
        with self._adapter_changes:
            if self._adapter_names is None:
                self.enable_adapters(rank=rank)
            if rank > self._adapter_rank:
                raise ValueError(f"adapter {name!r} has rank {rank}, room is for {self._adapter_rank}")
            if name in self._adapter_names:
                raise ValueError(f"an adapter {name!r} is loaded already")
            if None not in self._adapter_names:
                raise ValueError(f"all {len(self._adapter_names)} places for adapters are taken")
            index = self._adapter_names.index(None)
            with self._between_steps(), torch.inference_mode():
                for p in self.model.all_parts():
                    for q in (p.adapted() if p.banks is not None else ()):
                        mine = {local: matrices[p.spec.tensor_name(local)] for local in q.tensors
                                if p.spec.tensor_name(local) in matrices}
                        p.banks[q.name].put(index, mine, scale)
            with self._adapter_lock:
                self._adapter_names[index] = name
            return index

    def unload_adapter(self, name: str) -> None:
        """Give an adapter's place back; refused while requests use it."""
        with self._adapter_changes:
            with self._adapter_lock:
                index = self.adapter_index(name)
                if self._adapter_users[index]:
                    raise ValueError(f"adapter {name!r} is in use by {self._adapter_users[index]} requests")
                self._adapter_names[index] = None         # (nobody may take it up any more; the place is given out behind this)
            with self._between_steps(), torch.inference_mode():
                for p in self.model.all_parts():
                    for bank in (p.banks or {}).values():
                        bank.clear(index)

    def adapter_index(self, name: str) -> int:
        with self._adapter_lock:
            if self._adapter_names is None or name is None or name not in self._adapter_names:
                raise ValueError(f"no adapter {name!r} is loaded")
            return self._adapter_names.index(name)

    def hold_adapter(self, name: str) -> int:
        """The adapter's index, for a request that uses it until ``release_adapter``."""
        with self._adapter_lock:
            index = self.adapter_index(name)
            self._adapter_users[index] += 1
            return index

    def release_adapter(self, index: int) -> None:
        with self._adapter_lock:
            self._adapter_users[index] -= 1

    # -- requests -----------------------------------------------------------------------

    def add_request(self, rid) -> int:
        return self.cache.add_request(rid)

    def free_request(self, rid) -> None:
        self.cache.free_request(rid)

    # a scheduler may feed the sampler's device output to the next step (see StepRunner.step)
    device_token_feedback = True

    def step(self, entries: Sequence[StepEntry], device_tokens: torch.Tensor | None = None) -> StepResult:
        with self._device_lock:
            if self.stepper.adapter_count and self.device.type == "cuda":
                self._step_stream = torch.cuda.current_stream(self.device)
                if self._banks_written is not None:
                    self._step_stream.wait_event(self._banks_written)
                    self._banks_written = None
            return self.stepper.step(entries, device_tokens)

    def capture_decode_steps(self, max_batch: int) -> int:
        """Capture the decode step of every batch size up to ``max_batch`` that has no graph yet
        (a step of a new size otherwise runs kernel by kernel and is captured when it first
        occurs, some 40 ms in the middle of serving).  Uses requests of its own that hold one
        token each and gives their pages back; needs that many free pages and request slots.
        Returns the number of graphs captured; 0 when steps are not captured at all.  Where adapters are enabled, steps with and
        without them are captured."""
        if not self.stepper.cuda_graph:
            return 0
        made = 0
        max_batch = min(max_batch, self.cache.max_requests - self.cache.num_requests)
        kinds = [(-1, ())] if self._adapter_names is None else [(-1, ()), (0, ("adapters",))]
        for b in range(1, max_batch + 1):
            for adapter, kind in kinds:
                slot = self.stepper._graphs.get((b, *kind))
                if slot is not None and slot.graph is not None:
                    continue
                rids = [("__capture__", i) for i in range(b)]
                for r in rids:
                    self.cache.add_request(r)
                try:
                    if not self.cache.can_append([(r, 1) for r in rids]):
                        return made
                    # runs kernel by kernel once, then records
                    self.step([StepEntry(r, [0], [0], adapter) for r in rids])
                    made += 1
                finally:
                    for r in rids:
                        self.cache.free_request(r)
        return made

    # -- health -------------------------------------------------------------------------

    def health_word(self) -> torch.Tensor:
        """An int32 tensor of one element on the device: non-zero once a kernel has given up one
        of its bounded waits (its output, and everything computed from it, is then invalid).  A
        scheduler copies it to the host together with each step's tokens."""
        from ..csrc import ops

        return ops.status_word(self.device)

    def reset_health(self) -> None:
        """Clear the word and whatever the interrupted kernels left behind (synchronises)."""
        from ..csrc import ops

        ops.recover_from_wait_failure(self.device)
