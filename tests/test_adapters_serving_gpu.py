"""Adapters that come and go while an engine serves."""

import threading

import pytest
import torch

import plain_impl as P
from adapter_util import merged, random_adapter
from tiny_configs import PAGE_SIZE, TINY, load_state, prompt_ids

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def runner_of(model_dirs, which, dtype="float32", **kw):
    from mini_infer_b200.engine import ModelRunner

    return ModelRunner.from_pretrained(model_dirs[which], dtype=dtype, block_size=PAGE_SIZE[which], num_blocks=128, max_requests=8, **kw)


def test_adapters_are_loaded_and_unloaded_while_steps_are_captured(model_dirs):
    """The engine's thread meets batches of new sizes, with and without adapters, while another thread makes room for adapters, loads
    and unloads them, each time with no memory in the allocator's hands."""
    from mini_infer_b200.engine import ContinuousScheduler, Request
    from mini_infer_b200.sampling import SamplingParams

    state = load_state(model_dirs["C"])
    config, tensors = random_adapter("C", state, 8, 1)
    other = random_adapter("C", state, 8, 2)
    prompts = [prompt_ids("C", n, salt=40 + n) for n in (5, 9, 12, 3)]
    weights = {None: state, "x": merged(state, config, tensors)}
    want = {a: [P.greedy_generate(w, TINY["C"], p, 12) for p in prompts] for a, w in weights.items()}
    runner = runner_of(model_dirs, "C", cuda_graph=True)
    sched = ContinuousScheduler(runner)
    sched.start(capture_decode_steps=False)
    stop, failures, rounds = threading.Event(), [], 0

    def churn():
        nonlocal rounds
        try:
            while not stop.is_set():
                with runner._device_lock:                         # (freeing memory spoils a capture as well)
                    torch.cuda.empty_cache()
                runner.load_adapter("other", other[1], other[0])
                runner.unload_adapter("other")
                rounds += 1
        except Exception as e:  # noqa: BLE001
            failures.append(e)

    loader = threading.Thread(target=churn, daemon=True)
    try:
        for b in (1, 2):                                          # before there are adapters
            handles = [sched.submit(Request(p, SamplingParams(), 12)) for p in prompts[:b]]
            assert [h.wait(120).tokens for h in handles] == want[None][:b]
        runner.load_adapter("x", tensors, config)
        loader.start()
        for b in (4, 3, 1, 2, 4):
            for names in (["x"] * b, [None] * b, ["x", None, None, "x"][:b]):
                handles = [sched.submit(Request(p, SamplingParams(), 12, adapter=a)) for p, a in zip(prompts, names)]
                assert [h.wait(120).tokens for h in handles] == [want[a][i] for i, a in enumerate(names)]
    finally:
        stop.set()
        if loader.is_alive():
            loader.join(60)
        sched.stop()
    assert not failures and rounds > 0
    assert any(len(k) == 2 and slot.replays for k, slot in runner.stepper._graphs.items())


def test_a_step_waits_for_banks_written_on_another_stream(model_dirs):
    """An adapter loaded on a stream that is busy for long is there for a step on the engine's stream, and one that is unloaded there
    is not taken away under a step in front of it."""
    from mini_infer_b200.engine import StepEntry

    state = load_state(model_dirs["A"])
    config, tensors = random_adapter("A", state, 8, 1)
    prompt = prompt_ids("A", 40, salt=50)
    want = {a: P.llama_logits(w, TINY["A"], prompt)[-1] for a, w in ((True, merged(state, config, tensors)), (False, state))}
    runner = runner_of(model_dirs, "A")
    runner.enable_adapters(count=2, rank=8)
    side = torch.cuda.Stream()

    def logits(rid, adapter):
        runner.add_request(rid)
        z = runner.step([StepEntry(rid, prompt, [len(prompt) - 1], adapter)]).logits
        runner.free_request(rid)
        return z

    logits("warm", -1)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)                            # a tenth of a second
        index = runner.load_adapter("x", tensors, config)
    first = logits("a", index)
    torch.cuda._sleep(200_000_000)
    second = logits("b", index)
    with torch.cuda.stream(side):
        runner.unload_adapter("x")
    third = logits("c", index)                                    # (an empty place adds nothing)
    torch.cuda.synchronize()
    for got, adapted in ((first, True), (second, True), (third, False)):
        got = got[0].double().cpu()
        near, far = ((got - want[a]).norm() / want[a].norm() for a in (adapted, not adapted))
        assert near < 1e-4 and far > 1e-2


@pytest.mark.parametrize("cuda_graph", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_request_without_an_adapter_beside_one_with(dtype, cuda_graph, model_dirs):
    """Its logits have the same bits in float32 whether or not its neighbour has an adapter.  In bfloat16 they may round otherwise: few
    rows finish a branch, and the gate, in a product's epilogue in fp32, and behind an adapter from its bfloat16 result.  Both are as
    near to the formula as any step, and no further from one another."""
    import numpy as np

    import trace_util as T
    from mini_infer_b200.engine import StepEntry

    state = load_state(model_dirs["C"])
    config, tensors = random_adapter("C", state, 16, 7)
    mine, other = prompt_ids("C", 12, salt=71), prompt_ids("C", 10, salt=72)
    runner = runner_of(model_dirs, "C", dtype=dtype, cuda_graph=cuda_graph)
    runner.enable_adapters(count=2, rank=16)
    runner.load_adapter("x", tensors, config)
    cuts = [slice(0, 3), slice(3, 6), *(slice(i, i + 1) for i in range(6, 12))]
    got = {}
    for adapter in (-1, 0):
        rows = []
        for rid in "ab":
            runner.add_request(rid)
        for c in cuts:
            theirs = (other + other)[c]
            entries = [StepEntry("a", mine[c], list(range(len(mine[c])))), StepEntry("b", theirs, list(range(len(theirs))), adapter)]
            result = runner.step(entries)
            rows += [row.clone() for (rid, _), row in zip(result.rows, result.logits.double()) if rid == "a"]
        for rid in "ab":
            runner.free_request(rid)
        got[adapter] = torch.stack(rows).cpu()
    if dtype == "float32":
        assert torch.equal(got[-1], got[0])
        return
    want = P.llama_logits(state, TINY["C"], mine).numpy()
    tol = T.tolerance(dtype, float(np.abs(want).max()))
    for z in got.values():
        assert T.first_bad(z.numpy(), want, tol) is None
    assert T.first_bad(got[0].numpy(), got[-1].numpy(), tol) is None
