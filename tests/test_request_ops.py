"""What the operators of a request's own refuse, without a GPU: every check of shapes and types comes before the device's."""

import pytest
import torch

from mini_infer_b200.csrc import ops

F, I, BF = torch.float32, torch.int32, torch.bfloat16


def adapter_args(M=3, K=16, N=24, n=2, P=1, R=8, dtype=F):
    return dict(y=torch.zeros(M, N, dtype=dtype), x=torch.zeros(M, K, dtype=dtype), a=torch.zeros(n, P, R, K, dtype=dtype),
                b=torch.zeros(n, N, R, dtype=dtype), plan=ops.AdapterPlan(torch.zeros(M, dtype=I), n))


def adapter_call(**changes):
    args = adapter_args()
    args.update(changes)
    return ops.adapter_add(args.pop("y"), args.pop("x"), args.pop("a"), args.pop("b"), args.pop("plan"), **args)


ADAPTER_REFUSALS = [
    (dict(x=torch.zeros(3, 15)), "do not match"),
    (dict(y=torch.zeros(4, 24)), "do not match"),
    (dict(b=torch.zeros(2, 24, 7)), "do not match"),
    (dict(b=torch.zeros(3, 24, 8)), "do not match"),
    (dict(a=torch.zeros(2, 8, 16)), "a \\[adapters"),
    (dict(x=torch.zeros(3, 16, dtype=torch.float16)), "unsupported dtype"),
    (dict(x=torch.zeros(3, 16, dtype=BF)), "operands of"),
    (dict(a=torch.zeros(2, 1, 16, 8).transpose(2, 3)), "contiguous"),
    (dict(x=torch.zeros(16, 3).t()), "unit inner stride"),
    (dict(plan=ops.AdapterPlan(torch.zeros(4, dtype=I), 2)), "a plan of 4 rows"),
    (dict(plan=ops.AdapterPlan(torch.zeros(3, dtype=I), 5)), "a plan of 3 rows and 5 adapters"),
    (dict(pairs=True), "pairs are two parts"),
    (dict(parts=(12, 12)), "parts"),
    (dict(parts=(23,)), "parts"),
    (dict(a=torch.zeros(2, 2, 8, 16), parts=(25, -1)), "parts"),
    (dict(a=torch.zeros(2, 5, 8, 16), parts=(4, 5, 5, 5, 5)), "at most 4"),
    (dict(a=torch.zeros(2, 2, 8, 16), pairs=True, parts=(10, 14)), "pairs"),
    (dict(scale=torch.zeros(2, dtype=BF)), "scale"),
    (dict(ranks=torch.zeros(3, dtype=I)), "ranks"),
    (dict(out=torch.zeros(3, 24, dtype=BF)), "out must be"),
    (dict(out=torch.zeros(1, 24).expand(3, 24)), "rows apart"),
    (dict(), "CUDA tensors only"),
]


@pytest.mark.parametrize("changes,message", ADAPTER_REFUSALS)
def test_adapter_add_refuses(changes, message):
    with pytest.raises(ops.KernelError, match=message):
        adapter_call(**changes)


def test_adapter_add_refuses_results_over_its_operands():
    flat = torch.zeros(3 * 40)
    y, x = flat[:72].view(3, 24), flat[72:].view(3, 16)
    for out in (flat[1:73].view(3, 24), flat[30:102].view(3, 24)):
        with pytest.raises(ops.KernelError, match="overlaps"):
            adapter_call(y=y, x=x, out=out)
    with pytest.raises(ops.KernelError, match="CUDA tensors only"):      # y itself is fine
        adapter_call(y=y, x=x, out=y)


def test_adapter_plan_refuses():
    for ids in (torch.zeros(3), torch.zeros(3, dtype=torch.int64), torch.zeros(3, 1, dtype=I), torch.zeros(6, dtype=I)[::2]):
        with pytest.raises(ops.KernelError, match="int32 vector"):
            ops.adapter_plan(ids, 2)
    with pytest.raises(ops.KernelError, match="-1 adapters"):
        ops.adapter_plan(torch.zeros(3, dtype=I), -1)
    with pytest.raises(ops.KernelError, match="CUDA tensors only"):
        ops.adapter_plan(torch.zeros(3, dtype=I), 2)
    with pytest.raises(ops.KernelError, match="at most 8000000"):
        ops.adapter_plan(torch.zeros(8_000_001, dtype=I), 2)


B, V, W = 3, 100, 4
LOGITS_REFUSALS = [
    (dict(logits=torch.zeros(B, V, dtype=BF)), "fp32"),
    (dict(logits=torch.zeros(V, B).t()), "unit inner stride"),
    (dict(logits=torch.zeros(1, V).expand(B, V)), "overlap"),
    (dict(counts=torch.zeros(B, V, dtype=I)), "seen bits"),
    (dict(slots=torch.zeros(B, dtype=I)), "seen bits"),
    (dict(repetition=torch.ones(B)), "seen bits"),
    (dict(seen=torch.zeros(B, W, dtype=I), presence=torch.ones(B)), "counts"),
    (dict(seen=torch.zeros(B, W, dtype=I), frequency=torch.ones(B)), "counts"),
    (dict(seen=torch.zeros(B, W - 1, dtype=I)), "seen must be"),
    (dict(seen=torch.zeros(B, W, dtype=torch.int64)), "seen must be"),
    (dict(seen=torch.zeros(B, W, dtype=I), counts=torch.zeros(B + 1, V, dtype=I)), "counts must be"),
    (dict(seen=torch.zeros(B - 1, W, dtype=I)), "without slots"),
    (dict(seen=torch.zeros(B, W, dtype=I), slots=torch.zeros(B + 1, dtype=I)), "slots"),
    (dict(seen=torch.zeros(B, W, dtype=I), repetition=torch.ones(B, dtype=torch.float64)), "repetition"),
    (dict(bias=(torch.zeros(B, dtype=I), torch.zeros(2, dtype=I), torch.zeros(2))), "starts"),
    (dict(bias=(torch.zeros(B + 1, dtype=I), torch.zeros(2, dtype=torch.int64), torch.zeros(2))), "ids"),
    (dict(bias=(torch.zeros(B + 1, dtype=I), torch.zeros(2, dtype=I), torch.zeros(3))), "values"),
    (dict(masks=torch.zeros(B, W + 1, dtype=I)), "masks must be"),
    (dict(masks=torch.zeros(B, W, dtype=torch.uint8)), "masks must be"),
    (dict(masks=torch.zeros(B - 1, W, dtype=I)), "without mask_rows"),
    (dict(mask_rows=torch.zeros(B, dtype=I)), "without masks"),
    (dict(masks=torch.zeros(1, W, dtype=I), mask_rows=torch.zeros(B)), "mask_rows"),
    (dict(), "CUDA tensors only"),
]


@pytest.mark.parametrize("changes,message", LOGITS_REFUSALS)
def test_adjust_logits_refuses(changes, message):
    args = dict(logits=torch.zeros(B, V))
    args.update(changes)
    with pytest.raises(ops.KernelError, match=message):
        ops.adjust_logits(args.pop("logits"), **args)


RECORD_REFUSALS = [
    (dict(counts=torch.zeros(V, dtype=I)), "counts must be"),
    (dict(counts=torch.zeros(B, V)), "counts must be"),
    (dict(seen=torch.zeros(B, W + 1, dtype=I)), "seen must be"),
    (dict(seen=torch.zeros(B + 1, W, dtype=I)), "counts must be"),
    (dict(tokens=torch.zeros(5, dtype=torch.int64)), "tokens"),
    (dict(slots=torch.zeros(3, dtype=I)), "slots"),
    (dict(starts=torch.zeros(3, dtype=torch.int64)), "starts"),
    (dict(starts=torch.zeros(0, dtype=I)), "starts"),
    (dict(n_prompt=torch.zeros(3, dtype=I)), "n_prompt"),
    (dict(starts=None, slots=None), "without slots"),
    (dict(), "CUDA tensors only"),
]


@pytest.mark.parametrize("changes,message", RECORD_REFUSALS)
def test_record_tokens_refuses(changes, message):
    args = dict(counts=torch.zeros(B, V, dtype=I), seen=torch.zeros(B, W, dtype=I), slots=torch.zeros(2, dtype=I),
                starts=torch.zeros(3, dtype=I), tokens=torch.zeros(5, dtype=I), n_prompt=torch.zeros(2, dtype=I), fresh=True)
    args.update(changes)
    with pytest.raises(ops.KernelError, match=message):
        ops.record_tokens(args.pop("counts"), args.pop("seen"), args.pop("slots"), args.pop("starts"), args.pop("tokens"), **args)
