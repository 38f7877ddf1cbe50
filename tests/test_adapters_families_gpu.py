"""Adapters in models whose layers are not Llama's: two branches side by side, branches with the norm behind them, layers run several
times, a GELU in the gate."""

import numpy as np
import pytest
import torch

import lilulix_configs as L
import plain_lilulix as PL
import plain_ruburax as PR
import ruburax_configs as R
import trace_util as T
from test_adapters_cpu import gated_mlp_adapter

pytestmark = pytest.mark.gpu

# every mixer with a dense feed-forward (a router's close calls would be other tests' matter)
DENSE = R.config([R.rglru(32, 4, 3, R.dense(40)), R.attention(R.attn(4, 2, 24, 16, 0.3, R.rot(12, 1000.0)), R.dense(24)),
                  R.attention(R.attn(4, 2, 24, 16, 0.3, kv_from=1), None),
                  R.parallel(R.attn(6, 3, 16, 8, 0.25, R.rot(16, 50.0)), (3, 12, 20, 5.0), (0.6, 0.8), R.dense(56))],
                 vocab=59, width=48, eps=1e-5, mult=0.7, logit_scale=1.3, side=6)
MODELS = {**{"lilulix " + w: (L.CONFIGS[w], L, lambda cfg, st, toks: PL.forward(cfg, st, toks)) for w in L.CONFIGS},
          "ruburax": (DENSE, R, lambda cfg, st, toks: PR.ruburax_logits(st, cfg, toks, torch.float64))}


def with_adapter(state, config, tensors):
    out = {n: t.double() for n, t in state.items()}
    for name, a in tensors.items():
        if ".lora_A." in name:
            b = tensors[name.replace(".lora_A.", ".lora_B.")]
            w = name.replace(".lora_A.weight", "")
            out[w] = out[w] + config["lora_alpha"] / config["r"] * (b.double() @ a.double())
    return out


@pytest.mark.parametrize("cuda_graph", [False, True])
# (in bfloat16 the recurrences' states amplify roundings: this Ruburax model without any adapter is 0.012 and 0.027 of the largest logit
# off in the root mean square, where the bound is 0.01)
@pytest.mark.parametrize("which,dtype", [(w, d) for w in MODELS for d in ("float32", "bfloat16") if w != "ruburax" or d == "float32"])
def test_every_request_with_its_own_adapter(which, dtype, cuda_graph):
    """Prompts in one batch, then their last tokens decoded together, against the model with each adapter merged in."""
    from mini_infer_b200.engine import ModelRunner, StepEntry

    cfg, module, plain = MODELS[which]
    state = module.random_state(cfg, seed=17)
    adapters = {}
    for name, rank in (("x", 4), ("y", 9)):
        config, tensors = gated_mlp_adapter(cfg, rank, 100 + rank)
        config["lora_alpha"] = 0.5 * rank
        adapters[name] = config, {n: t.to(torch.bfloat16) for n, t in tensors.items()}
    weights = {None: {n: t.double() for n, t in state.items()}, **{n: with_adapter(state, *a) for n, a in adapters.items()}}
    users = ["x", None, "y", "x"]
    prompts = [module.prompt(cfg, n, salt=60 + n) for n in (23, 40, 9, 65)]
    runner = ModelRunner.from_state_dict(cfg, state, dtype=dtype, block_size=16, num_blocks=64, max_requests=4, cuda_graph=cuda_graph)
    runner.enable_adapters(count=3, rank=12)
    index = {None: -1, **{n: runner.load_adapter(n, t, c) for n, (c, t) in adapters.items()}}
    rows = [[] for _ in prompts]

    def step(first, last):
        entries = [StepEntry(i, p[len(p) + first if first else 0:len(p) + last if last else None], adapter=index[a]) for i, (p, a) in
                   enumerate(zip(prompts, users))]
        for e in entries:
            e.want = list(range(len(e.tokens)))
        result = runner.step(entries)
        for (rid, _), row in zip(result.rows, result.logits.double().cpu().numpy()):
            rows[rid].append(row)

    for i in range(len(prompts)):
        runner.add_request(i)
    step(0, -6)
    for k in range(6, 0, -1):
        step(-k, 1 - k)
    want = [plain(cfg, weights[a], p).numpy() for p, a in zip(prompts, users)]
    bare = [plain(cfg, weights[None], p).numpy() for p in prompts]
    tol = T.tolerance(dtype, max(float(np.abs(w).max()) for w in want))
    for i, (w, a) in enumerate(zip(want, users)):
        got = np.stack(rows[i])
        bad = T.first_bad(got, w, tol)
        assert bad is None, f"{which} {dtype} request {i}: position {bad} differs by {np.abs(got[bad] - w[bad]).max():.3g} (bound {float(tol):.3g})"
        assert a is None or T.first_bad(bare[i], w, tol) is not None        # the adapter matters
    if cuda_graph:
        assert runner.stepper._graphs[(4, "adapters")].replays == 5
