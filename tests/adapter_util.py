"""Random low-rank adapters for the tiny models, and the weights that a model with one of them merged in would have."""

import json
import os

import torch

from tiny_configs import SEED, TINY

TARGETS = ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj", "self_attn.o_proj", "mlp.gate_proj", "mlp.up_proj", "mlp.down_proj")


def random_adapter(which, state, rank, salt, targets=TARGETS, layers=None, std=0.6):
    """``(config, tensors)``: matrices that change a product's output by a good part of its size."""
    g = torch.Generator().manual_seed(1000 * SEED[which] + salt)
    tensors = {}
    for i in range(TINY[which]["num_hidden_layers"]):
        if layers is not None and i not in layers:
            continue
        for t in targets:
            name = f"model.layers.{i}.{t}"
            out, inp = state[name + ".weight"].shape
            w = float(state[name + ".weight"].float().std())
            tensors[f"base_model.model.{name}.lora_A.weight"] = torch.randn(rank, inp, generator=g) * inp ** -0.5
            tensors[f"base_model.model.{name}.lora_B.weight"] = torch.randn(out, rank, generator=g) * (std * w * inp ** 0.5 * rank ** -0.5)
    return {"r": rank, "lora_alpha": 1.5 * rank, "bias": "none"}, tensors


def merged(state, config, tensors, dtype=torch.float64):
    """The model's weights with ``s B A`` added, ``s = lora_alpha / r``."""
    out = {n: t.to(dtype) for n, t in state.items()}
    for name, a in tensors.items():
        if ".lora_A." in name:
            w = name.replace("base_model.model.", "").replace(".lora_A.weight", ".weight")
            b = tensors[name.replace(".lora_A.", ".lora_B.")]
            out[w] = out[w] + config["lora_alpha"] / config["r"] * (b.to(dtype) @ a.to(dtype))
    return out


def write_adapter(folder, config, tensors):
    from mini_infer_b200.weights import write_safetensors

    os.makedirs(folder, exist_ok=True)
    with open(os.path.join(folder, "adapter_config.json"), "w", encoding="utf-8") as f:
        json.dump(config, f)
    write_safetensors(os.path.join(folder, "adapter_model.safetensors"), tensors)
    return folder
