"""Low-rank adapters from a folder or from tensors in memory.

A folder holds ``adapter_config.json`` (``r``, ``lora_alpha``, optional ``use_rslora``) and ``adapter_model.safetensors`` with two
matrices per adapted tensor of the model, ``<tensor>.lora_A.weight [r, inputs]`` and ``<tensor>.lora_B.weight [outputs, r]``, where
``<tensor>`` is the model's name, without ``.weight`` if it ends so, maybe behind ``base_model.model.``.  What is added to a product is
``s B (A x)`` with ``s = lora_alpha / r`` (``lora_alpha / sqrt(r)`` with ``use_rslora``); all matrices have rank ``r``.
"""

from __future__ import annotations

import json
import math
import os
import re
from typing import Mapping

import torch

from .loader import WeightLoadError
from .safetensors_io import SafetensorsFile

_NAME = re.compile(r"^(?:base_model\.model\.)?(?P<tensor>.+)\.lora_(?P<side>[AB])(?:\.default)?\.weight$")
_UNSUPPORTED = ("use_dora", "lora_bias", "rank_pattern", "alpha_pattern", "modules_to_save")


def adapter_scale(config: Mapping) -> float:
    """``s`` of an adapter's configuration."""
    try:
        r, alpha = int(config["r"]), float(config["lora_alpha"])
    except (KeyError, TypeError, ValueError):
        raise WeightLoadError("an adapter's configuration needs the numbers r and lora_alpha") from None
    if r <= 0 or not math.isfinite(alpha):
        raise WeightLoadError(f"an adapter of rank {r} with lora_alpha {alpha}")
    if str(config.get("bias", "none")) != "none":
        raise WeightLoadError("adapters with biases are not supported")
    for key in _UNSUPPORTED:
        if config.get(key):
            raise WeightLoadError(f"adapters with {key} are not supported")
    return alpha / math.sqrt(r) if config.get("use_rslora") else alpha / r


def pair_matrices(state: Mapping[str, torch.Tensor]) -> dict[str, tuple[torch.Tensor, torch.Tensor]]:
    """``{model tensor name: (A, B)}`` from an adapter's tensors; everything that does not fit is named in one error."""
    sides: dict[str, dict[str, torch.Tensor]] = {}
    strange: list[str] = []
    twice: list[str] = []
    for name, t in state.items():
        m = _NAME.match(name)
        if m is None or t.dim() != 2:
            strange.append(name)
        elif m["side"] in sides.get(m["tensor"] + ".weight", ()):
            twice.append(name)
        else:
            sides.setdefault(m["tensor"] + ".weight", {})[m["side"]] = t
    single = sorted(n for n, s in sides.items() if len(s) != 2)
    ranks = sorted(n for n, s in sides.items() if len(s) == 2 and s["A"].shape[0] != s["B"].shape[1])
    if strange or twice or single or ranks or not sides:
        raise WeightLoadError("; ".join(filter(None, [
            "an adapter without matrices" if not sides and not strange else "",
            f"not an adapter's matrices: {sorted(strange)}" if strange else "",
            f"given twice, under other names: {sorted(twice)}" if twice else "",
            f"one matrix of two: {single}" if single else "",
            f"matrices of different ranks: {ranks}" if ranks else ""])), unexpected=strange + twice, missing=single, mismatched=ranks)
    return {n: (s["A"], s["B"]) for n, s in sides.items()}


def read_adapter(folder: str | os.PathLike) -> tuple[dict, dict[str, torch.Tensor]]:
    """``(configuration, tensors)`` of an adapter's folder."""
    folder = os.fspath(folder)
    with open(os.path.join(folder, "adapter_config.json"), "r", encoding="utf-8") as f:
        config = json.load(f)
    file = SafetensorsFile(os.path.join(folder, "adapter_model.safetensors"))
    try:
        return config, {n: file.read(n) for n in file.names()}
    finally:
        file.close()
