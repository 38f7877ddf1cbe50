"""What the requests of one batch bring of their own, as operators: low-rank adapters beside the projections that
all requests share, and penalties, biases and masks on the logits with the token histories that the penalties read.

``listed()`` and ``draw(rng)`` give cases, ``prepare(case, seed)`` makes what a program has in hand before the call,
``run(state)`` is one call, ``work(case)`` what it cannot do without, and ``exact(case, seed)`` the same answer in 64
bits from the definition.  With ``own`` set, ``run`` calls this repository's operators; otherwise it computes them from
elementary operations.

The three operators, for a batch of rows:

``adapter``  out[t] = y[t] + s_a B_a (A_a x[t]), a = ids[t]; out[t] = y[t] where ids[t] is negative.  ``y`` is the shared
             projection's output.  Several projections may be merged along the columns ("parts", or two that alternate
             column by column, "pairs"); each has an A of its own, and a column's B acts on its own projection's A x.
``logits``   z / r or z r (z > 0 or not) where the row's history holds the token, minus f times its count and minus p
             where the count is positive, plus the row's biases, and minus infinity where the row's mask has no bit.
``history``  the counts of generated tokens and the bits of all seen tokens, written anew from each request's tokens.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ------------------------------------------------------------------------------- cases


def adapter_case(dtype, singles, prompts, tokens, width, parts, pairs, adapters, rank, mixed, bare):
    """``singles`` requests that bring one token each, then ``prompts`` requests with ``tokens`` tokens between them.
    ``adapters`` are held, of ``rank`` or (``mixed``) of ranks from an eighth of it to all of it; ``bare``: some requests use none."""
    return {"op": "adapter", "dtype": dtype, "singles": singles, "prompts": prompts, "tokens": tokens, "width": width,
            "parts": parts, "pairs": pairs, "adapters": adapters, "rank": rank, "mixed": mixed, "bare": bare}


def logits_case(rows, vocab, history, biases, masks):
    """``history`` tokens behind every row (0: no penalties), ``biases`` given biases a row, ``masks`` different masks (0: none)."""
    return {"op": "logits", "rows": rows, "vocab": vocab, "history": history, "biases": biases, "masks": masks}


def history_case(requests, vocab, longest, generated):
    """``requests`` of up to ``longest`` tokens; ``generated``: some of the tokens are generated ones (a request that comes back)."""
    return {"op": "history", "requests": requests, "vocab": vocab, "longest": longest, "generated": generated}


def listed() -> list[dict]:
    a, z, h = adapter_case, logits_case, history_case
    named = {
        # one user's next token behind the merged q/k/v projection of a 4096-wide model: latency
        "adapter-one-token": a("bfloat16", 1, 0, 0, 4096, "4096,1024,1024", False, 4, 16, False, False),
        # a busy server's decode step at the merged gate/up projection, adapters of several ranks, some requests without
        "adapter-decode-64": a("bfloat16", 64, 0, 0, 4096, "14336,14336", True, 24, 64, True, True),
        # the float32 engine, with which a conversion is checked, at an output projection
        "adapter-float32": a("float32", 3, 2, 128, 2048, "2048", False, 3, 8, False, False),
        # a mixed step: a few requests decode while prompts are read under the step's budget of tokens
        "adapter-mixed-step": a("bfloat16", 12, 3, 2036, 4096, "4096,1024,1024", False, 8, 16, True, True),
        # long documents at the widest projection
        "adapter-documents": a("bfloat16", 0, 2, 8192, 4096, "14336,14336", True, 4, 64, False, False),
        # one request with everything; a batch that only repeats less; a busy server with grammars; odd sizes, masks alone
        "logits-one-row": z(1, 32000, 200, 20, 1),
        "logits-penalties": z(16, 128256, 1500, 0, 0),
        "logits-busy": z(256, 128256, 1000, 100, 32),
        "logits-grammar": z(13, 50021, 0, 0, 5),
        # a short question is admitted; a batch of prompts; long documents that come back with what they had generated
        "history-question": h(1, 32000, 17, False),
        "history-batch": h(16, 128256, 2048, False),
        "history-documents": h(64, 128256, 32768, True),
    }
    return [dict(c, name=n) for n, c in named.items()]


def spread(rng, low, high):
    """A whole number between ``low`` and ``high``, even over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng) -> dict:
    kind = rng.choice(["adapter", "adapter", "logits", "logits", "history"])
    listed_work = [work(c) for c in listed() if c["op"] == kind]
    most = {name: max(w[name] for w in listed_work) for name in ("bytes", "flops")}
    while True:
        if kind == "adapter":
            rank, pairs = rng.choice([3, 8, 16, 24, 32, 64]), rng.random() < 0.3
            half = 8 * spread(rng, 16, 1792)
            parts = [half, half] if pairs else [8 * spread(rng, 16, 1792) for _ in range(rng.choice([1, 1, 2, 3]))]
            singles = rng.choice([0, spread(rng, 1, 128)])
            prompts = 0 if singles and rng.random() < 0.4 else rng.randint(1, 6)
            c = adapter_case(rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"]), singles, prompts,
                             max(prompts, spread(rng, 9, 8192)) if prompts else 0, 8 * spread(rng, 16, 1792),
                             ",".join(map(str, parts)), pairs, spread(rng, 1, 24), rank, rank >= 8 and rng.random() < 0.5,
                             rng.random() < 0.5)
            if c["dtype"] == "float32" and work(c)["flops"] > 4e9:       # the float32 engine reads short prompts
                continue
            if (c["singles"] + c["tokens"]) * c["adapters"] * rank * (len(parts) * c["width"] + sum(parts)) > 8e10:
                continue                                                 # all adapters on all rows, as the plain form has it
        elif kind == "logits":
            c = logits_case(spread(rng, 1, 256), spread(rng, 1000, 160000), rng.choice([0, spread(rng, 1, 4000)]),
                            rng.choice([0, spread(rng, 1, 300)]), rng.choice([0, 0, spread(rng, 1, 32)]))
            if not (c["history"] or c["biases"] or c["masks"]):
                continue
        else:
            c = history_case(spread(rng, 1, 64), spread(rng, 1000, 160000), spread(rng, 1, 32768), rng.random() < 0.5)
        w = work(c)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]:
            return c


# ------------------------------------------------------------------------------- inputs


def widths(case) -> list[int]:
    return [int(n) for n in case["parts"].split(",")]


def shares(case) -> list[int]:
    """The prompts' tokens: one after the other longer, and all of them together ``tokens``."""
    n, left, out = case["prompts"], case["tokens"], []
    for q in range(n):
        take = left if q == n - 1 else max(1, min(left - (n - 1 - q), 2 * case["tokens"] * (q + 1) // (n * (n + 1))))
        out.append(take)
        left -= take
    return out


def ranks_of(case) -> list[int]:
    steps = [8, 4, 2, 1] if case["mixed"] else [1]
    return [max(1, case["rank"] // steps[i % len(steps)]) for i in range(case["adapters"])]


def users(case) -> list[tuple[int, int]]:
    """(tokens, adapter) of every request; -1: none."""
    counts = [1] * case["singles"] + shares(case)
    n = case["adapters"] + (1 if case["bare"] else 0)
    return [(c, i % n if i % n < case["adapters"] else -1) for i, c in enumerate(counts)]


def lengths(case) -> list[int]:
    n, longest = case["requests"], case["longest"]
    return [max(1, longest * (i + 1) // n - (i * 7) % 5) for i in range(n)]


def generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed) + 1)


def tokens_like_text(shape, vocab, gen):
    """Token ids of which a few are frequent and most are rare."""
    u = torch.rand(shape, generator=gen, device=DEVICE)
    return (u.pow(4) * vocab).to(torch.int32).clamp_(max=vocab - 1)


def pack_bits(flags):
    """Bool ``[n, V]`` as int32 words: bit ``v % 32`` of word ``v / 32``."""
    n, vocab = flags.shape
    wide = torch.zeros((n, -(-vocab // 32) * 32), dtype=torch.int64, device=flags.device)
    wide[:, :vocab] = flags
    words = (wide.view(n, -1, 32) << torch.arange(32, device=flags.device)).sum(dim=2)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def prepare(case: dict, seed: int) -> dict:
    return {"adapter": prepare_adapter, "logits": prepare_logits, "history": prepare_history}[case["op"]](case, generator(seed))


def prepare_adapter(case, gen):
    dt, k, n = DTYPES[case["dtype"]], case["width"], case["adapters"]
    parts = widths(case)
    cols, rank = sum(parts), -(-case["rank"] // 8) * 8      # held with whole groups of eight

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=gen, device=DEVICE) * std

    place = torch.randperm(n, generator=gen, device=DEVICE)      # where in the bank an adapter lies
    ranks = torch.empty(n, dtype=torch.int32, device=DEVICE)
    ranks[place] = torch.tensor(ranks_of(case), dtype=torch.int32, device=DEVICE)
    held = torch.arange(rank, device=DEVICE) < ranks[:, None]
    a = (normal(n, len(parts), rank, k, std=k ** -0.5) * held[:, None, :, None]).to(dt)
    b = (normal(n, cols, rank, std=0.5 * case["rank"] ** -0.5) * held[:, None, :]).to(dt)
    who = torch.tensor([u for c, u in users(case) for _ in range(c)], device=DEVICE)
    ids = torch.where(who < 0, who, place[who.clamp(min=0)]).to(torch.int32)
    m = ids.numel()
    scale = 0.5 + 1.5 * torch.rand(n, generator=gen, device=DEVICE)
    return {"op": "adapter", "x": normal(m, k).to(dt), "y": normal(m, cols).to(dt), "a": a, "b": b, "ranks": ranks,
            "scale": scale, "ids": ids, "parts": tuple(parts), "pairs": case["pairs"]}


def prepare_logits(case, gen):
    rows, vocab = case["rows"], case["vocab"]
    st = {"op": "logits", "logits": 3.0 * torch.randn((rows, vocab), generator=gen, device=DEVICE)}
    st["slots"] = torch.randperm(rows, generator=gen, device=DEVICE).to(torch.int32)
    if case["history"]:
        told = tokens_like_text((rows, case["history"]), vocab, gen).long()
        made = torch.rand(told.shape, generator=gen, device=DEVICE) < 0.5          # generated, the others were the prompt's
        st["counts"] = torch.zeros((rows, vocab), dtype=torch.int32, device=DEVICE).scatter_add_(1, told, made.to(torch.int32))
        st["seen"] = pack_bits(torch.zeros((rows, vocab), dtype=torch.bool, device=DEVICE).scatter_(1, told, True))
        st["repetition"] = 1.0 + 0.3 * torch.rand(rows, generator=gen, device=DEVICE)
        st["presence"] = torch.rand(rows, generator=gen, device=DEVICE) - 0.2
        st["frequency"] = 0.6 * torch.rand(rows, generator=gen, device=DEVICE) - 0.1
    if case["biases"]:
        each = min(case["biases"], vocab)
        given = torch.rand((rows, each), generator=gen, device=DEVICE)             # one in every stretch of the vocabulary
        low = torch.arange(each, device=DEVICE) * vocab // each
        high = (torch.arange(each, device=DEVICE) + 1) * vocab // each
        st["bias_ids"] = (low + (given * (high - low)).long().clamp(max=(high - low) - 1)).to(torch.int32).reshape(-1)
        values = 5.0 * torch.randn((rows, each), generator=gen, device=DEVICE)
        values[torch.rand((rows, each), generator=gen, device=DEVICE) < 0.1] = -math.inf   # tokens that are not to come
        st["bias_values"] = values.reshape(-1)
        st["bias_starts"] = (torch.arange(rows + 1, device=DEVICE) * each).to(torch.int32)
    if case["masks"]:
        # what a grammar leaves: a handful of tokens, or nearly all of them
        share = torch.where(torch.arange(case["masks"], device=DEVICE) % 2 == 0, 0.95, 40.0 / vocab)
        st["masks"] = pack_bits(torch.rand((case["masks"], vocab), generator=gen, device=DEVICE) < share[:, None])
        st["mask_rows"] = torch.randint(-1, case["masks"], (rows,), generator=gen, device=DEVICE, dtype=torch.int32)
    return st


def prepare_history(case, gen):
    n, vocab, long = case["requests"], case["vocab"], lengths(case)
    starts = torch.tensor([0] + long, device=DEVICE).cumsum(0).to(torch.int32)
    each = torch.tensor(long, device=DEVICE)
    prompt = each if not case["generated"] else (each * torch.rand(n, generator=gen, device=DEVICE)).long()
    return {"op": "history", "tokens": tokens_like_text((sum(long),), vocab, gen), "starts": starts,
            "prompt": prompt.to(torch.int32), "slots": torch.randperm(n, generator=gen, device=DEVICE).to(torch.int32),
            "counts": torch.full((n, vocab), 7, dtype=torch.int32, device=DEVICE),       # what the slots' last users left
            "seen": torch.full((n, -(-vocab // 32)), -1, dtype=torch.int32, device=DEVICE)}


# ------------------------------------------------------------------------------- one call


def run(state):
    if own:
        return {"adapter": own_adapter, "logits": own_logits, "history": own_history}[state["op"]](state)
    return {"adapter": plain_adapter, "logits": plain_logits, "history": plain_history}[state["op"]](state)


def own_adapter(st):
    from mini_infer_b200.csrc import ops

    plan = ops.adapter_plan(st["ids"], st["a"].shape[0])
    return ops.adapter_add(st["y"], st["x"], st["a"], st["b"], plan, scale=st["scale"], ranks=st["ranks"],
                           parts=st["parts"], pairs=st["pairs"], w_constant=True)


def own_logits(st):
    from mini_infer_b200.csrc import ops

    bias = (st["bias_starts"], st["bias_ids"], st["bias_values"]) if "bias_ids" in st else None
    return ops.adjust_logits(st["logits"], slots=st["slots"] if "seen" in st else None, seen=st.get("seen"),
                             counts=st.get("counts"), repetition=st.get("repetition"), presence=st.get("presence"),
                             frequency=st.get("frequency"), bias=bias, masks=st.get("masks"),
                             mask_rows=st.get("mask_rows"))


def own_history(st):
    from mini_infer_b200.csrc import ops

    ops.record_tokens(st["counts"], st["seen"], st["slots"], st["starts"], st["tokens"], n_prompt=st["prompt"], fresh=True)
    return {"counts": st["counts"], "seen": st["seen"]}


def plain_adapter(st):
    """Every row through every adapter, and all but its own taken out in between."""
    a, b, x, y = (st[name].float() for name in ("a", "b", "x", "y"))
    n, p, r, k = a.shape
    mine = (st["ids"][:, None] == torch.arange(n, device=x.device)) * st["scale"]
    h = (x @ a.reshape(n * p * r, k).t()).reshape(-1, n, p, r) * mine[:, :, None, None]
    of_part = b.reshape(n, -1, 2, r).unbind(2) if st["pairs"] else b.split(st["parts"], dim=1)
    deltas = [h[:, :, i].reshape(-1, n * r) @ w.transpose(1, 2).reshape(n * r, -1) for i, w in enumerate(of_part)]
    delta = torch.stack(deltas, dim=2).reshape(y.shape) if st["pairs"] else torch.cat(deltas, dim=1)
    return torch.where(st["ids"][:, None] >= 0, y + delta, y).to(st["y"].dtype)


def unpack_bits(words, vocab):
    return ((words[:, :, None] >> torch.arange(32, device=words.device)) & 1).reshape(words.shape[0], -1)[:, :vocab] != 0


def plain_logits(st):
    z = st["logits"]
    vocab = z.shape[1]
    if "seen" in st:
        at = st["slots"].long()
        told, count = unpack_bits(st["seen"][at], vocab), st["counts"][at].float()
        r, p, f = (st[name][:, None] for name in ("repetition", "presence", "frequency"))
        z = torch.where(told, torch.where(z > 0, z / r, z * r), z)
        z = z - f * count - p * (count > 0)
    if "bias_ids" in st:
        starts = st["bias_starts"].long()
        row = torch.repeat_interleave(torch.arange(z.shape[0], device=z.device), starts[1:] - starts[:-1],
                                      output_size=st["bias_ids"].numel())
        z = z + torch.zeros_like(z).index_put((row, st["bias_ids"].long()), st["bias_values"])
    if "masks" in st:
        at = st["mask_rows"].long()
        open_ = unpack_bits(st["masks"][at.clamp(min=0)], vocab) | (at < 0)[:, None]
        z = torch.where(open_, z, torch.full_like(z, -math.inf))
    return z


def plain_history(st):
    n, vocab = st["counts"].shape
    starts = st["starts"].long()
    i = torch.arange(st["tokens"].numel(), device=starts.device)
    request = torch.bucketize(i, starts[1:], right=True)
    at = st["slots"].long()[request] * vocab + st["tokens"].long()
    made = (i - starts[request] >= st["prompt"].long()[request]).to(torch.int32)
    counts = torch.zeros(n * vocab, dtype=torch.int32, device=at.device).index_add(0, at, made)
    told = torch.zeros(n * vocab, dtype=torch.bool, device=at.device).index_fill(0, at, True)
    return {"counts": counts.reshape(n, vocab), "seen": pack_bits(told.reshape(n, vocab))}


# ------------------------------------------------------------------------------- work and exact answers


def work(case: dict) -> dict:
    if case["op"] == "adapter":
        size = 4 if case["dtype"] == "float32" else 2
        cols, parts = sum(widths(case)), len(widths(case))
        ranks, who = ranks_of(case), users(case)
        rows = sum(c for c, _ in who)
        used = {u for _, u in who if u >= 0}
        # x of the rows that have an adapter, y and the result of all rows, the adapters in use at their own ranks
        moved = sum(c for c, u in who if u >= 0) * case["width"] + 2 * rows * cols
        moved += sum(ranks[u] * (parts * case["width"] + cols) for u in used)
        flops = sum(2 * c * ranks[u] * (parts * case["width"] + cols) for c, u in who if u >= 0)
        return {"bytes": moved * size + 4 * rows, "flops": flops}
    if case["op"] == "logits":
        rows, vocab = case["rows"], case["vocab"]
        words = -(-vocab // 32)
        # the logits in and out, the bits of history and masks, counts where the history has a token, the biases
        moved = 8 * rows * vocab + 4 * words * (case["masks"] + (rows if case["history"] else 0))
        moved += rows * (4 * min(case["history"], vocab) + 8 * min(case["biases"], vocab) + 20)
        return {"bytes": moved, "flops": 5 * rows * vocab}
    n, vocab = case["requests"], case["vocab"]
    return {"bytes": 4 * n * (vocab + -(-vocab // 32)) + 4 * sum(lengths(case)) + 12 * n, "flops": sum(lengths(case))}


def exact(case: dict, seed: int):
    return {"adapter": exact_adapter, "logits": exact_logits, "history": exact_history}[case["op"]](prepare(case, seed))


def exact_adapter(st):
    """Adapter by adapter, part by part, on the rows that use it."""
    out, ids, offset = st["y"].double(), st["ids"], 0
    for part, width in enumerate(st["parts"]):
        cols = slice(part, None, 2) if st["pairs"] else slice(offset, offset + width)
        offset += width
        for adapter in ids.unique().tolist():
            if adapter < 0:
                continue
            rows = torch.nonzero(ids == adapter)[:, 0]
            r = int(st["ranks"][adapter])
            h = torch.einsum("tk,rk->tr", st["x"][rows].double(), st["a"][adapter, part, :r].double())
            d = torch.einsum("tr,nr->tn", h, st["b"][adapter, cols, :r].double()) * st["scale"][adapter].double()
            whole = out[rows]
            whole[:, cols] += d
            out[rows] = whole
    return out


def exact_logits(st):
    """Row by row, on the tokens that something applies to."""
    out = st["logits"].double()
    vocab = out.shape[1]
    v = torch.arange(vocab, device=out.device)
    for i in range(out.shape[0]):
        z = out[i]
        if "seen" in st:
            slot = int(st["slots"][i])
            told = torch.nonzero((st["seen"][slot][v // 32] >> (v % 32)) & 1)[:, 0]
            r = st["repetition"][i].double()
            z[told] = z[told] * torch.where(z[told] > 0, 1.0 / r, r)
            c = st["counts"][slot].double()
            z -= st["frequency"][i].double() * c + torch.where(c > 0, st["presence"][i].double(), 0.0)
        if "bias_ids" in st:
            given = slice(int(st["bias_starts"][i]), int(st["bias_starts"][i + 1]))
            z[st["bias_ids"][given].long()] += st["bias_values"][given].double()
        if "masks" in st and int(st["mask_rows"][i]) >= 0:
            words = st["masks"][int(st["mask_rows"][i])]
            z[((words[v // 32] >> (v % 32)) & 1) == 0] = -math.inf
    return out


def exact_history(st):
    """Request by request, by counting."""
    n, vocab = st["counts"].shape
    counts, seen = torch.zeros_like(st["counts"]), torch.zeros_like(st["seen"])
    starts, prompt, slots = (st[name].tolist() for name in ("starts", "prompt", "slots"))
    for i, slot in enumerate(slots):
        mine = st["tokens"][starts[i]:starts[i + 1]].long()
        counts[slot] = torch.bincount(mine[prompt[i]:], minlength=vocab).to(torch.int32)
        there = torch.bincount(mine, minlength=seen.shape[1] * 32).clamp(max=1).reshape(-1, 32)
        words = torch.zeros(seen.shape[1], dtype=torch.int64, device=seen.device)
        for bit in range(32):
            words |= there[:, bit] << bit
        seen[slot] = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
    return {"counts": counts, "seen": seen}
