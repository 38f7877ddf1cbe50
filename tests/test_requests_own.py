"""What a request may bring of its own, as far as it goes without a GPU: options and their checks, an adapter's files and the banks
they fill, the scheduler's book-keeping of adapters and histories."""

import json
import math

import numpy as np
import pytest
import torch

from mini_infer_b200.engine import Request
from mini_infer_b200.engine.step import StepEntry, StepError, StepRunner
from mini_infer_b200.parts import AdaptedProduct, AdapterBank, PartSpec, build_part
from mini_infer_b200.sampling import SamplingParams, mask_any, mask_words
from mini_infer_b200.sampling.adjust import AdjustedRow, LogitsAdjuster
from mini_infer_b200.weights import SafetensorsError, WeightLoadError, adapter_scale, pair_matrices, read_adapter
from test_scheduler import FakeRunner, FakeSampler, make, prompt


# ----------------------------------------------------------------------------- options


@pytest.mark.parametrize("bad", [dict(repetition_penalty=0.0), dict(repetition_penalty=-1.0), dict(repetition_penalty=math.inf),
                                 dict(repetition_penalty=math.nan), dict(frequency_penalty=math.nan), dict(presence_penalty=math.inf),
                                 dict(logit_bias={3: math.nan}), dict(logit_bias={3: math.inf}), dict(logit_bias={-1: 1.0}),
                                 dict(allowed_token_ids=[]), dict(allowed_token_ids=[-1, 2])])
def test_options_are_checked(bad):
    with pytest.raises(ValueError):
        SamplingParams(**bad)


@pytest.mark.parametrize("bad", [dict(repetition_penalty=1e39), dict(repetition_penalty=1e-40), dict(frequency_penalty=-1e39),
                                 dict(presence_penalty=3.41e38), dict(logit_bias={3: 1e39}), dict(logit_bias={3: -1e39}),
                                 dict(allowed_token_ids=[4, 7], logit_bias={4: -math.inf, 7: -math.inf})])
def test_options_that_fp32_does_not_hold_or_that_leave_no_token(bad):
    with pytest.raises(ValueError):
        SamplingParams(**bad)


def test_biases_that_rule_out_every_token():
    p = SamplingParams(logit_bias={t: -math.inf for t in range(10)})
    p.check_vocabulary(11)
    with pytest.raises(ValueError, match="every token"):
        p.check_vocabulary(10)
    # a mask holds no token that a bias rules out
    adjuster = LogitsAdjuster("cpu", 40, 2)
    never = SamplingParams(logit_bias={5: -math.inf, 6: 2.0})
    row = AdjustedRow("a", never, [1], [], mask_words([5], 40))
    assert not mask_any(adjuster.mask_of(row), 40)
    assert (adjuster.mask_of(AdjustedRow("a", never, [1], [], mask_words([5, 6, 39], 40))) == mask_words([6, 39], 40)).all()
    assert adjuster.mask_of(AdjustedRow("a", never, [1], [])) is None
    both = SamplingParams(logit_bias={5: -math.inf}, allowed_token_ids=[5, 9])
    assert (adjuster.mask_of(AdjustedRow("b", both, [1], [])) == mask_words([9], 40)).all()


def test_a_grammar_that_fails_ends_its_request_alone(monkeypatch):
    from mini_infer_b200.engine import scheduler

    class Adjuster(LogitsAdjuster):
        def apply(self, logits, rows):
            pass

        def record(self, tokens, rows):
            pass

    monkeypatch.setattr(scheduler, "LogitsAdjuster", Adjuster)
    runner = RunnerWithAdapters(64)
    runner.device = "cpu"
    sched = scheduler.ContinuousScheduler(runner, sampler=FakeSampler(), max_tokens_per_step=8)

    def broken(generated):
        if len(generated) == 2:
            raise KeyError("no such state")
        return range(1000)

    handles = [sched.submit(Request(prompt(4), SamplingParams(), 5, token_mask=g))
               for g in (broken, None, lambda said: np.zeros(3, np.int32), lambda said: [1000], lambda said: [] if said else None)]
    with pytest.warns(UserWarning, match="token_mask failed"):
        sched.run_until_done()
    results = [h.wait() for h in handles]
    assert [(r.finish_reason, len(r.tokens)) for r in results] == [("cancelled", 2), ("length", 5), ("cancelled", 0), ("cancelled", 0), ("stop", 1)]
    assert runner.cache.num_requests == 0


def test_options_say_what_they_change():
    assert not SamplingParams().adjusted and not SamplingParams(temperature=1.0, top_k=3).adjusted
    assert not SamplingParams(logit_bias={}).adjusted
    for p in (dict(repetition_penalty=1.1), dict(frequency_penalty=-0.5), dict(presence_penalty=0.5)):
        assert SamplingParams(**p).adjusted and SamplingParams(**p).penalised
    p = SamplingParams(logit_bias={5: -math.inf, 2: 1.5}, allowed_token_ids=[9, 2, 9])
    assert p.adjusted and not p.penalised and p.allowed_token_ids == (2, 9) and dict(p.logit_bias) == {5: -math.inf, 2: 1.5}
    assert hash(p) == hash(SamplingParams(logit_bias={5: -math.inf, 2: 1.5}, allowed_token_ids=[2, 9]))
    p.check_vocabulary(10)
    for V in (9, 5):
        with pytest.raises(ValueError, match="names token"):
            p.check_vocabulary(V)


@pytest.mark.parametrize("V", [1, 31, 32, 33, 100])
def test_masks_as_words(V):
    ids = sorted({0, V // 2, V - 1})
    words = mask_words(ids, V)
    assert words.dtype == np.int32 and words.shape == (-(-V // 32),)
    assert [t for t in range(V) if (int(words[t // 32]) >> (t % 32)) & 1] == ids
    assert mask_any(words, V) and not mask_any(mask_words([], V), V)
    for t in (-1, V):
        with pytest.raises(ValueError, match="outside"):
            mask_words([t], V)
    if V % 32:                            # bits behind the vocabulary are no tokens
        words = mask_words([], V)
        words[-1] = np.int32(-1 << (V % 32)) if V % 32 < 31 else np.int32(-2 ** 31)
        assert not mask_any(words, V)


# ----------------------------------------------------------------------------- adapters


def test_an_adapters_configuration():
    assert adapter_scale({"r": 8, "lora_alpha": 12}) == 1.5
    assert adapter_scale({"r": 16, "lora_alpha": 8, "use_rslora": True, "bias": "none", "rank_pattern": {}}) == 2.0
    for bad in ({}, {"r": 8}, {"r": 0, "lora_alpha": 1}, {"r": "x", "lora_alpha": 1}, {"r": 8, "lora_alpha": math.inf},
                {"r": 8, "lora_alpha": 1, "bias": "all"}, {"r": 8, "lora_alpha": 1, "use_dora": True},
                {"r": 8, "lora_alpha": 1, "rank_pattern": {"q_proj": 4}}):
        with pytest.raises(WeightLoadError):
            adapter_scale(bad)


def test_an_adapters_matrices_are_paired():
    a, b = torch.zeros(4, 6), torch.zeros(5, 4)
    got = pair_matrices({"base_model.model.model.layers.0.mlp.up_proj.lora_A.weight": a, "base_model.model.model.layers.0.mlp.up_proj.lora_B.weight": b,
                         "x.lora_A.default.weight": a, "x.lora_B.default.weight": b})
    assert set(got) == {"model.layers.0.mlp.up_proj.weight", "x.weight"} and got["x.weight"][0] is a
    for bad, message in (({}, "without matrices"), ({"x.lora_A.weight": a}, "one matrix of two"), ({"x.weight": a}, "not an adapter's"),
                         ({"x.lora_A.weight": torch.zeros(3), "x.lora_B.weight": b}, "not an adapter's"),
                         ({"x.lora_A.weight": torch.zeros(3, 6), "x.lora_B.weight": b}, "different ranks")):
        with pytest.raises(WeightLoadError, match=message):
            pair_matrices(bad)


def test_an_adapters_folder(tmp_path):
    from adapter_util import write_adapter

    tensors = {"m.lora_A.weight": torch.randn(4, 6), "m.lora_B.weight": torch.randn(5, 4).to(torch.bfloat16)}
    config, got = read_adapter(write_adapter(str(tmp_path / "a"), {"r": 4, "lora_alpha": 8}, tensors))
    assert adapter_scale(config) == 2.0 and all(torch.equal(got[n], t) for n, t in tensors.items())
    with pytest.raises(FileNotFoundError):
        read_adapter(str(tmp_path / "missing"))
    (tmp_path / "a" / "adapter_model.safetensors").write_bytes(b"short")
    with pytest.raises(SafetensorsError):
        read_adapter(str(tmp_path / "a"))
    (tmp_path / "a" / "adapter_config.json").write_text("{")
    with pytest.raises(json.JSONDecodeError):
        read_adapter(str(tmp_path / "a"))


@pytest.mark.parametrize("pairs", [False, True])
def test_a_bank_lays_an_adapter_out(pairs):
    g = torch.Generator().manual_seed(1)
    widths = (6, 6) if pairs else (6, 4)
    bank = AdapterBank(AdaptedProduct("m", ("u", "v"), widths, 5, pairs), 3, 8, torch.float32, "cpu")
    rnd = lambda *s: torch.randn(*s, generator=g)
    first = {"u": (rnd(3, 5), rnd(6, 3)), "v": (rnd(3, 5), rnd(widths[1], 3))}
    bank.put(1, first, 0.5)
    bank.put(2, {"v": (rnd(8, 5), rnd(widths[1], 8))}, 2.0)      # one of the two alone
    assert bank.ranks.tolist() == [0, 3, 8] and bank.scale.tolist() == [0.0, 0.5, 2.0]
    x = rnd(5)
    for index, which in ((1, "u"), (1, "v"), (2, "u")):
        part = "uv".index(which)
        delta = bank.b[index, bank.columns(part)] @ (bank.a[index, part] @ x)
        want = first[which][1] @ (first[which][0] @ x) if index == 1 else torch.zeros(widths[part])
        assert torch.allclose(delta, want, atol=1e-6)
    bank.put(1, {"u": (rnd(2, 5), rnd(6, 2))}, 1.0)             # nothing of the old one is left
    assert bank.ranks[1] == 2 and not bank.a[1, 0, 2:].any() and not bank.a[1, 1].any() and not bank.b[1, bank.columns(1)].any()
    bank.clear(1)
    assert bank.ranks[1] == 0 and not bank.a[1].any() and not bank.b[1].any()


def test_parts_name_the_products_that_take_adapters():
    mixer = build_part("mixer", PartSpec("gqa_attention", dict(hidden_size=32, num_heads=2, num_kv_heads=1, head_dim=16), ""))
    ffn = build_part("feed_forward", PartSpec("swiglu", dict(hidden_size=32, intermediate_size=48), ""))
    for part in (mixer, ffn):
        decls = part.param_decls()
        for q in part.adapted():
            assert [decls[t].shape for t in q.tensors] == [(w, q.inputs) for w in q.widths]
    norm = build_part("norm", PartSpec("rmsnorm", dict(hidden_size=16, eps=1e-5), ""))
    assert norm.adapted() == ()


# ----------------------------------------------------------------------------- scheduler


class RunnerWithAdapters(FakeRunner):
    vocab_size = 1000

    def __init__(self, *a, **kw):
        super().__init__(*a, **kw)
        self.users, self.seen = [0, 0], []

    def hold_adapter(self, name):
        if name not in ("one", "two"):
            raise ValueError(f"no adapter {name!r} is loaded")
        index = ("one", "two").index(name)
        self.users[index] += 1
        return index

    def release_adapter(self, index):
        self.users[index] -= 1

    def step(self, entries):
        self.seen.append({e.rid: e.adapter for e in entries})
        return super().step(entries)


def test_the_scheduler_hands_adapters_on_and_gives_them_back():
    from mini_infer_b200.engine.scheduler import ContinuousScheduler

    runner = RunnerWithAdapters(64)
    sched = ContinuousScheduler(runner, sampler=FakeSampler(), max_tokens_per_step=8)
    handles = [sched.submit(Request(prompt(n), SamplingParams(), 3, adapter=a)) for n, a in ((9, "two"), (4, None), (5, "one"), (6, "two"))]
    assert runner.users == [1, 2]
    with pytest.raises(ValueError, match="no adapter 'three'"):
        sched.submit(Request(prompt(3), adapter="three"))
    with pytest.raises(ValueError, match="names token 1000"):
        sched.submit(Request(prompt(3), SamplingParams(logit_bias={1000: 1.0}), adapter="one"))
    handles[3].cancel()
    assert runner.users == [1, 1]
    sched.submit(Request([], adapter="one"))                      # ends at once
    sched.run_until_done()
    assert runner.users == [0, 0]
    assert {rid: a for s in runner.seen for rid, a in s.items()} == {0: 1, 1: -1, 2: 0}
    with pytest.raises(ValueError, match="takes none"):
        make()[1].submit(Request(prompt(3), adapter="one"))


def test_a_step_refuses_adapters_that_are_not_there():
    class Cache:
        def __contains__(self, rid):
            return False

    runner = StepRunner.__new__(StepRunner)
    runner.vocab_size, runner.max_positions, runner.cache, runner.adapter_count = 10, None, Cache(), 2
    runner._validate([StepEntry("a", [1], [0], 1), StepEntry("b", [1], [0], -1)])
    for adapter in (2, -2):
        with pytest.raises(StepError, match="adapter"):
            runner._validate([StepEntry("a", [1], [0], adapter)])


def test_history_slots_come_back():
    adjuster = LogitsAdjuster("cpu", 100, 2)
    adjuster._slot = {"a": adjuster._free.pop(), "b": adjuster._free.pop()}
    adjuster.forget("nobody")
    adjuster.forget("a")
    adjuster.forget("a")
    assert adjuster._free == [0] and adjuster._slot == {"b": 1}
