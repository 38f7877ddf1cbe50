"""Adapters' places, names and files in a runner whose steps are a stand-in, without a GPU."""

import threading

import pytest
import torch

from adapter_util import random_adapter
from mini_infer_b200.config.registry import load_config
from mini_infer_b200.engine.runner import ModelRunner
from mini_infer_b200.parts.adapters import AdapterBank
from mini_infer_b200.parts.model import DecoderModel
from mini_infer_b200.weights import WeightLoadError, bind_random, pair_matrices, random_state_dict
from tiny_configs import TINY


def cpu_runner(raw):
    arch, cfg = load_config(raw)
    model = DecoderModel(arch.assemble(cfg))
    bind_random(model, 1, torch.float32, torch.device("cpu"))
    return ModelRunner(model, cfg, num_blocks=8, max_requests=2)


class Stepper:
    """A step that lasts until it is let go."""

    def __init__(self):
        self.begun, self.let_go, self.inside = threading.Event(), threading.Event(), False

    def step(self, entries, device_tokens=None):
        self.inside = True
        self.begun.set()
        assert self.let_go.wait(20)
        self.inside = False


def in_thread(f, *args):
    t = threading.Thread(target=f, args=args, daemon=True)
    t.start()
    return t


@pytest.mark.parametrize("what", ["load", "enable", "unload"])
def test_banks_are_not_written_during_a_step(what, monkeypatch):
    """A step may be recorded as a graph, which allocations of another thread spoil, and reads the banks."""
    runner = cpu_runner(TINY["A"])
    config, tensors = random_adapter("A", random_state_dict(TINY["A"], 1), 4, 1)
    if what != "enable":
        runner.enable_adapters(count=2, rank=8)
        runner.load_adapter("first", tensors, config)
    stepper = runner.stepper = Stepper()
    stepper.adapter_count = 2
    seen = []

    def noted(name):
        real = getattr(AdapterBank, name)
        monkeypatch.setattr(AdapterBank, name, lambda self, *a, **kw: (seen.append(stepper.inside), real(self, *a, **kw))[1])

    for name in ("__init__", "put", "clear"):
        noted(name)
    step = in_thread(runner.step, [])
    assert stepper.begun.wait(20)
    work = in_thread(*{"load": (runner.load_adapter, "second", tensors, config), "enable": (runner.enable_adapters, 2, 8),
                       "unload": (runner.unload_adapter, "first")}[what])
    work.join(0.5)
    assert not any(seen)
    stepper.let_go.set()
    step.join(20)
    work.join(20)
    assert not work.is_alive() and seen and not any(seen)


def test_requests_come_and_go_while_an_adapter_is_loaded(monkeypatch):
    runner = cpu_runner(TINY["A"])
    config, tensors = random_adapter("A", random_state_dict(TINY["A"], 1), 4, 1)
    runner.enable_adapters(count=3, rank=8)
    runner.load_adapter("first", tensors, config)
    begun, let_go, real = threading.Event(), threading.Event(), AdapterBank.put

    def slow(self, *a, **kw):
        begun.set()
        assert let_go.wait(20)
        real(self, *a, **kw)

    monkeypatch.setattr(AdapterBank, "put", slow)
    load = in_thread(runner.load_adapter, "second", tensors, config)
    assert begun.wait(20)
    held = []
    user = in_thread(lambda: held.append(runner.hold_adapter("first")))
    user.join(5)
    assert held == [0]
    runner.release_adapter(0)
    with pytest.raises(ValueError, match="no adapter 'second'"):      # not before all of it is there
        runner.hold_adapter("second")
    let_go.set()
    load.join(20)
    assert runner.hold_adapter("second") == 1


def test_a_failed_load_leaves_its_place_free(monkeypatch):
    runner = cpu_runner(TINY["A"])
    config, tensors = random_adapter("A", random_state_dict(TINY["A"], 1), 4, 1)
    runner.enable_adapters(count=1, rank=8)
    real, calls = AdapterBank.put, []

    def fails(self, *a, **kw):
        calls.append(self)
        if len(calls) == 2:
            raise RuntimeError("out of memory")
        real(self, *a, **kw)

    monkeypatch.setattr(AdapterBank, "put", fails)
    with pytest.raises(RuntimeError, match="out of memory"):
        runner.load_adapter("x", tensors, config)
    with pytest.raises(ValueError, match="no adapter"):
        runner.adapter_index("x")
    assert runner.load_adapter("x", tensors, config) == 0


def test_room_that_cannot_be_made_leaves_adapters_off(monkeypatch):
    runner = cpu_runner(TINY["A"])
    real, calls = AdapterBank.__init__, []

    def fails(self, *a, **kw):
        calls.append(self)
        if len(calls) == 3:
            raise RuntimeError("out of memory")
        real(self, *a, **kw)

    monkeypatch.setattr(AdapterBank, "__init__", fails)
    with pytest.raises(RuntimeError, match="out of memory"):
        runner.enable_adapters(count=2, rank=8)
    assert all(p.banks is None for p in runner.model.all_parts()) and runner.stepper.adapter_count == 0
    runner.enable_adapters(count=2, rank=8)
    assert runner.stepper.adapter_count == 2


def gated_mlp_adapter(cfg, rank, salt, prefix=""):
    """``(config, tensors)`` for the dense feed-forwards of a model whose tensors have no ``.weight`` in their names."""
    g = torch.Generator().manual_seed(salt)
    H, tensors = cfg["width"], {}
    for i, layer in enumerate(cfg["layers"]):
        if layer.get("mlp") and layer["mlp"]["kind"] == "dense":
            ff = layer["mlp"]["ff"]
            for name, out, inp in (("gate", ff, H), ("up", ff, H), ("down", H, ff)):
                tensors[f"{prefix}l{i}.mlp.{name}.lora_A.weight"] = torch.randn(rank, inp, generator=g) * inp ** -0.5
                tensors[f"{prefix}l{i}.mlp.{name}.lora_B.weight"] = torch.randn(out, rank, generator=g) * rank ** -0.5
    return {"r": rank, "lora_alpha": 2 * rank}, tensors


@pytest.mark.parametrize("family", ["lilulix", "ruburax"])
def test_an_adapter_finds_tensors_with_plain_names(family):
    import importlib

    for which, raw in importlib.import_module(family + "_configs").CONFIGS.items():
        runner = cpu_runner(raw)
        for name, prefix in (("x", ""), ("y", "base_model.model.")):
            config, tensors = gated_mlp_adapter(raw, 4, 7, prefix)
            index = runner.load_adapter(name, tensors, config)
            found = 0
            for i, block in enumerate(runner.model.blocks):
                ff = block.feed_forward
                if not ff.adapted():
                    continue
                a = tensors[f"{prefix}l{i}.mlp.up.lora_A.weight"]
                assert torch.equal(ff.banks["gate_up"].a[index, 1, :4], a)
                assert torch.equal(ff.banks["down"].b[index, :, :4], tensors[f"{prefix}l{i}.mlp.down.lora_B.weight"])
                found += 3
            assert found and 2 * found == len(tensors)


def test_a_configuration_of_another_rank_is_refused():
    """The scale is lora_alpha / r: with another r than the matrices' it would be another number."""
    runner = cpu_runner(TINY["A"])
    config, tensors = random_adapter("A", random_state_dict(TINY["A"], 1), 8, 1)
    for r in (4, 16):
        with pytest.raises(WeightLoadError, match="r is"):
            runner.load_adapter("x", tensors, {**config, "r": r})
    assert runner.stepper.adapter_count == 0                      # (and no room was made for it)
    assert runner.load_adapter("x", tensors, config) == 0


def test_a_matrix_given_twice_is_refused():
    a, b = torch.zeros(4, 6), torch.zeros(5, 4)
    once = {"x.lora_A.weight": a, "x.lora_B.weight": b}
    assert set(pair_matrices(once)) == {"x.weight"}
    for again in ("x.lora_A.default.weight", "base_model.model.x.lora_A.weight", "base_model.model.x.lora_B.default.weight"):
        with pytest.raises(WeightLoadError, match="given twice"):
            pair_matrices({**once, again: torch.ones(4, 6)})
