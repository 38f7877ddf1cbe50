"""Requests with adapters, penalties, biases, masks and grammars of their own through the engine, against the plain implementation with the
adapters merged into its weights and the adjustments made on its logits."""

import json
import subprocess
import sys

import numpy as np
import pytest
import torch

import plain_impl as P
import request_ops_plain as Q
import trace_util as T
from adapter_util import merged, random_adapter, write_adapter
from tiny_configs import PAGE_SIZE, TINY, load_state, prompt_ids

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def runner_of(model_dirs, which, dtype="float32", **kw):
    from mini_infer_b200.engine import ModelRunner

    kw.setdefault("num_blocks", 128)
    return ModelRunner.from_pretrained(model_dirs[which], dtype=dtype, block_size=PAGE_SIZE[which], max_requests=8, **kw)


def adapters_of(which, state):
    """Three adapters: all products and an odd rank; attention alone and a high rank; one layer's feed-forward."""
    return {"all": random_adapter(which, state, 5, 1), "attention": random_adapter(which, state, 40, 2, ("self_attn.q_proj", "self_attn.v_proj")),
            "layer": random_adapter(which, state, 8, 3, ("mlp.down_proj", "mlp.up_proj"), layers=(1,))}


def load_all(runner, adapters):
    runner.enable_adapters(count=4, rank=40)
    for name, (config, tensors) in adapters.items():
        runner.load_adapter(name, tensors, config)


# ----------------------------------------------------------------------------- adapters


@pytest.mark.parametrize("cuda_graph", [False, True])
@pytest.mark.parametrize("which", ["A", "B", "C"])
def test_every_request_with_its_own_adapter(which, cuda_graph, model_dirs):
    from mini_infer_b200.engine import ContinuousScheduler, Request
    from mini_infer_b200.sampling import SamplingParams

    state = load_state(model_dirs[which])
    adapters = adapters_of(which, state)
    users = ["all", None, "layer", "attention", "all", None]
    lengths = [17, 9, 150, 1, 70, 33]
    prompts = [prompt_ids(which, n, salt=300 + i) for i, n in enumerate(lengths)]
    weights = {None: state, **{n: merged(state, *a) for n, a in adapters.items()}}
    want = [P.greedy_generate(weights[a], TINY[which], p, 8) for p, a in zip(prompts, users)]
    assert want[0] != P.greedy_generate(state, TINY[which], prompts[0], 8)      # the adapter matters
    runner = runner_of(model_dirs, which, cuda_graph=cuda_graph)
    load_all(runner, adapters)
    sched = ContinuousScheduler(runner, max_tokens_per_step=200, chunk_size=140)
    got = sched.generate([Request(p, SamplingParams(), 8, adapter=a) for p, a in zip(prompts, users)])
    assert [r.tokens for r in got] == want
    assert runner._adapter_users == [0, 0, 0, 0] and runner.cache.num_requests == 0


@pytest.mark.parametrize("which", ["A", "C"])
def test_adapters_in_bfloat16(which, model_dirs):
    """Logits of prompts (long enough for the tensor-core kernels of many rows) and of decoded tokens."""
    from mini_infer_b200.engine import StepEntry

    state = {n: t.to(torch.bfloat16) for n, t in load_state(model_dirs[which]).items()}
    adapters = {n: (c, {k: t.to(torch.bfloat16) for k, t in a.items()}) for n, (c, a) in adapters_of(which, state).items()}
    runner = runner_of(model_dirs, which, dtype="bfloat16")
    load_all(runner, adapters)
    names = [None, "all", "attention", "layer", "all"]
    tokens = {i: prompt_ids(which, n, salt=400 + i) for i, n in enumerate([40, 90, 33, 150, 5])}
    index = {None: -1, **{n: runner.adapter_index(n) for n in adapters}}
    for i in tokens:
        runner.add_request(i)
    rows = {i: [] for i in tokens}

    def step(take):
        entries = [StepEntry(i, tokens[i][a:b], list(range(b - a)), index[names[i]]) for i, (a, b) in take.items()]
        res = runner.step(entries)
        for (rid, _), row in zip(res.rows, res.logits.double().cpu()):
            rows[rid].append(row)

    step({i: (0, len(t) - 3) for i, t in tokens.items()})
    for k in (3, 2, 1):
        step({i: (len(t) - k, len(t) - k + 1) for i, t in tokens.items()})
    for i, t in tokens.items():
        w = merged(state, *adapters[names[i]]) if names[i] else {n: v.double() for n, v in state.items()}
        want = P.llama_logits(w, TINY[which], t)
        got = torch.stack(rows[i])
        # a dozen roundings of 2^-9 (in the mean) a layer in a row, and as many again for what they are multiplied by
        assert (got - want).norm() <= 3e-2 * want.norm(), names[i]
    runner.cache.check()


def test_captured_steps_with_and_without_adapters(model_dirs):
    """Graphs of steps with adapters are others than those without; new adapters in old places are used by them."""
    from mini_infer_b200.engine import ContinuousScheduler, Request
    from mini_infer_b200.sampling import SamplingParams

    state = load_state(model_dirs["C"])
    runner = runner_of(model_dirs, "C", cuda_graph=True)
    prompts = [prompt_ids("C", n, salt=500 + n) for n in (9, 20)]

    def generate(names):
        return [r.tokens for r in ContinuousScheduler(runner).generate(
            [Request(p, SamplingParams(), 7, adapter=a) for p, a in zip(prompts, names)])]

    bare = generate([None, None])
    one = random_adapter("C", state, 16, 7)
    other = random_adapter("C", state, 12, 8)
    assert runner.load_adapter("x", one[1], one[0]) == 0
    assert generate([None, None]) == bare and sorted(runner.stepper._graphs, key=str) == [(2,)]
    with_one = generate(["x", None])
    assert with_one == [P.greedy_generate(merged(state, *one), TINY["C"], prompts[0], 7), bare[1]]
    assert (2, "adapters") in runner.stepper._graphs and generate(["x", None]) == with_one
    runner.unload_adapter("x")
    assert runner.load_adapter("y", other[1], other[0]) == 0
    assert generate(["y", "y"]) == [P.greedy_generate(merged(state, *other), TINY["C"], p, 7) for p in prompts]
    assert generate([None, None]) == bare
    assert runner.capture_decode_steps(3) == 4          # (1,) and (3,), each with and without
    assert generate(["y", None]) == [P.greedy_generate(merged(state, *other), TINY["C"], prompts[0], 7), bare[1]]


def test_adapters_are_refused_where_they_do_not_fit(model_dirs):
    from mini_infer_b200.weights import WeightLoadError

    state = load_state(model_dirs["A"])
    runner = runner_of(model_dirs, "A")
    config, tensors = random_adapter("A", state, 8, 1)
    with pytest.raises(ValueError, match="no adapter"):
        runner.adapter_index("x")
    with pytest.raises(ValueError, match="configuration"):
        runner.load_adapter("x", tensors)
    name = "base_model.model.model.layers.0.self_attn.q_proj.lora_%s.weight"
    wrong = dict(tensors)
    wrong[name % "A"] = torch.zeros(8, 3)
    with pytest.raises(WeightLoadError, match="sizes"):
        runner.load_adapter("x", wrong, config)
    with pytest.raises(WeightLoadError, match="no product"):
        runner.load_adapter("x", {"lm_head.lora_A.weight": torch.zeros(8, 64), "lm_head.lora_B.weight": torch.zeros(512, 8)}, config)
    runner.enable_adapters(count=1, rank=8)
    with pytest.raises(ValueError, match="enabled already"):
        runner.enable_adapters()
    with pytest.raises(ValueError, match="rank 9"):
        runner.load_adapter("x", random_adapter("A", state, 9, 1)[1], {"r": 9, "lora_alpha": 9})
    runner.load_adapter("x", tensors, config)
    with pytest.raises(ValueError, match="loaded already"):
        runner.load_adapter("x", tensors, config)
    with pytest.raises(ValueError, match="places"):
        runner.load_adapter("y", tensors, config)
    runner.hold_adapter("x")
    with pytest.raises(ValueError, match="in use"):
        runner.unload_adapter("x")
    runner.release_adapter(0)
    runner.unload_adapter("x")


# ----------------------------------------------------------------------------- logits


def plain_generate(state, which, prompt, n_new, params, grammar=None):
    """Greedy generation on adjusted plain logits."""
    V = TINY[which]["vocab_size"]
    out = []
    for _ in range(n_new):
        z = P.llama_logits(state, TINY[which], prompt + out)[-1:]
        seen, counts = torch.zeros(1, V, dtype=torch.bool), torch.zeros(1, V, dtype=torch.int32)
        seen[0, prompt + out] = True
        for t in out:
            counts[0, t] += 1
        kw = dict(seen=Q.packed(seen), counts=counts, repetition=torch.tensor([params.repetition_penalty]),
                  presence=torch.tensor([params.presence_penalty]), frequency=torch.tensor([params.frequency_penalty]))
        if params.logit_bias:
            ids, values = zip(*params.logit_bias)
            kw["bias"] = (torch.tensor([0, len(ids)]), torch.tensor(ids), torch.tensor(values))
        allowed = set(range(V)) if params.allowed_token_ids is None else set(params.allowed_token_ids)
        if grammar is not None and grammar(out) is not None:
            allowed &= set(grammar(out))
        if not allowed:
            break
        kw["masks"] = Q.packed(torch.tensor([[v in allowed for v in range(V)]]))
        out.append(int(Q.adjusted(z, **kw)[0][0].argmax()))
    return out


def some_params(which, first):
    from mini_infer_b200.sampling import SamplingParams as S

    V = TINY[which]["vocab_size"]
    return [S(), S(repetition_penalty=1.6), S(frequency_penalty=1.5, presence_penalty=0.4), S(frequency_penalty=-0.7, repetition_penalty=0.8),
            S(logit_bias={first: -float("inf"), 7: 1.0, V - 1: 0.5}), S(allowed_token_ids=range(3, V, 7)),
            S(repetition_penalty=1.3, presence_penalty=1.0, logit_bias={5: 2.0}, allowed_token_ids=range(0, V, 2))]


@pytest.mark.parametrize("which,lookahead,cuda_graph", [("A", True, True), ("A", False, False), ("B", True, False), ("C", True, True)])
def test_penalties_biases_and_masks_through_the_scheduler(which, lookahead, cuda_graph, model_dirs):
    from mini_infer_b200.engine import ContinuousScheduler, Request

    state = load_state(model_dirs[which])
    prompts = [prompt_ids(which, n, salt=600 + n) for n in (12, 25, 7, 31, 18, 40, 3)]
    first = P.greedy_generate(state, TINY[which], prompts[4], 1)[0]
    params = some_params(which, first)
    want = [plain_generate(state, which, p, 10, s) for p, s in zip(prompts, params)]
    assert want[1] != P.greedy_generate(state, TINY[which], prompts[1], 10)
    runner = runner_of(model_dirs, which, cuda_graph=cuda_graph)
    sched = ContinuousScheduler(runner, max_tokens_per_step=50, chunk_size=20, lookahead=lookahead)
    requests = [Request(p, s, 10) for p, s in zip(prompts, params)]
    assert [r.tokens for r in sched.generate(requests)] == want
    assert [r.tokens for r in sched.generate(requests)] == want      # in slots that others have used
    assert len(sched._adjuster._free) == sched.max_concurrent


def test_histories_survive_a_preemption(model_dirs):
    from mini_infer_b200.engine import ContinuousScheduler, Request
    from mini_infer_b200.sampling import SamplingParams

    state = load_state(model_dirs["A"])
    prompts = [prompt_ids("A", n, salt=700 + n) for n in (30, 29, 28)]
    params = SamplingParams(repetition_penalty=1.2, frequency_penalty=0.8)
    want = [plain_generate(state, "A", p, 24, params) for p in prompts]
    runner = runner_of(model_dirs, "A", num_blocks=9)
    sched = ContinuousScheduler(runner, decode_headroom_blocks=0)
    assert [r.tokens for r in sched.generate([Request(p, params, 24) for p in prompts])] == want
    assert sched.preemptions > 0


def test_sampled_tokens_do_not_depend_on_the_look_ahead(model_dirs):
    from mini_infer_b200.engine import ContinuousScheduler, Request
    from mini_infer_b200.sampling import SamplingParams

    prompts = [prompt_ids("B", n, salt=800 + n) for n in (5, 40)]
    params = [SamplingParams(temperature=0.9, top_p=0.95, seed=11, repetition_penalty=1.3, frequency_penalty=0.3),
              SamplingParams(temperature=1.1, top_k=20, seed=12, allowed_token_ids=range(1, 1000, 3), presence_penalty=0.5)]
    runner = runner_of(model_dirs, "B")
    got = [[r.tokens for r in ContinuousScheduler(runner, lookahead=a).generate([Request(p, s, 20) for p, s in zip(prompts, params)])]
           for a in (True, False)]
    assert got[0] == got[1] and all(t % 3 == 1 for t in got[0][1])


def test_a_grammar_says_what_may_come_next(model_dirs):
    """Ids and words; a plain request beside it; a grammar that ends; one with limits of its own that leave nothing."""
    from mini_infer_b200.engine import ContinuousScheduler, Request
    from mini_infer_b200.sampling import SamplingParams, mask_words

    state, V = load_state(model_dirs["A"]), TINY["A"]["vocab_size"]
    prompts = [prompt_ids("A", n, salt=900 + n) for n in (8, 21, 13, 5)]

    def turn(generated):                  # every token lies in another stretch of the vocabulary than the last; five in all
        return [] if len(generated) == 5 else range(100 * (len(generated) % 3), 100 * (len(generated) % 3) + 60)

    def words(generated):
        return None if len(generated) % 2 else mask_words(range(0, V, 5), V)

    params = [SamplingParams(), SamplingParams(repetition_penalty=1.5), SamplingParams(), SamplingParams(allowed_token_ids=[400])]
    grammars = [turn, words, None, turn]
    plain = [turn, lambda g: None if len(g) % 2 else range(0, V, 5), None, turn]
    want = [plain_generate(state, "A", p, 9, s, g) for p, s, g in zip(prompts, params, plain)]
    runner = runner_of(model_dirs, "A", cuda_graph=True)
    got = ContinuousScheduler(runner).generate([Request(p, s, 9, token_mask=g) for p, s, g in zip(prompts, params, grammars)])
    assert [r.tokens for r in got] == want
    assert [len(r.tokens) for r in got] == [5, 9, 9, 0] and [r.finish_reason for r in got] == ["stop", "length", "length", "stop"]


def test_everything_at_once(model_dirs):
    """Adapters, penalties and grammars of different requests in the same steps."""
    from mini_infer_b200.engine import ContinuousScheduler, Request
    from mini_infer_b200.sampling import SamplingParams

    state = load_state(model_dirs["C"])
    adapters = adapters_of("C", state)
    runner = runner_of(model_dirs, "C", cuda_graph=True)
    load_all(runner, adapters)
    names = ["all", "attention", None, "layer"]
    prompts = [prompt_ids("C", n, salt=950 + n) for n in (40, 7, 19, 140)]
    params = [SamplingParams(repetition_penalty=1.4), SamplingParams(), SamplingParams(frequency_penalty=2.0), SamplingParams(logit_bias={3: 4.0})]
    grammars = [None, lambda g: range(len(g), 640, 4), None, None]
    weights = {None: state, **{n: merged(state, *a) for n, a in adapters.items()}}
    want = [plain_generate(weights[a], "C", p, 8, s, g) for p, a, s, g in zip(prompts, names, params, grammars)]
    for budget in (2048, 48):
        got = ContinuousScheduler(runner, max_tokens_per_step=budget).generate(
            [Request(p, s, 8, adapter=a, token_mask=g) for p, s, a, g in zip(prompts, params, names, grammars)])
        assert [r.tokens for r in got] == want


def test_the_command_line_and_the_entry_point_take_them(model_dirs, tmp_path):
    from mini_infer_b200.engine.api import generate
    from mini_infer_b200.sampling import SamplingParams

    state = load_state(model_dirs["A"])
    config, tensors = random_adapter("A", state, 8, 5)
    folder = write_adapter(str(tmp_path / "adapter"), config, tensors)
    prompt = prompt_ids("A", 11, salt=990)
    params = SamplingParams(repetition_penalty=1.5, logit_bias={9: 1.0, 4: -float("inf")}, allowed_token_ids=range(2, 512, 3))
    want = plain_generate(merged(state, config, tensors), "A", prompt, 6, params)
    runner = runner_of(model_dirs, "A")
    runner.load_adapter("x", folder)
    got = generate(runner, [prompt, prompt], max_tokens=6, sampling_params=params, adapters=["x", None])
    assert got[0].tokens == want and got[1].tokens == plain_generate(state, "A", prompt, 6, params)
    out = subprocess.run(
        [sys.executable, "-m", "mini_infer_b200.generate", "--model", model_dirs["A"], "--dtype", "float32", "--num-blocks", "16",
         "--prompt-ids", ",".join(map(str, prompt)), "--max-tokens", "6", "--adapter", folder, "--repetition-penalty", "1.5",
         "--logit-bias", "9:1.0", "--logit-bias", "4:-inf", "--allowed-token-ids", ",".join(map(str, range(2, 512, 3)))],
        capture_output=True, text=True, cwd=T.ROOT, timeout=600)
    assert out.returncode == 0, out.stderr
    assert json.loads(out.stdout.strip().splitlines()[-1])["tokens"] == want
