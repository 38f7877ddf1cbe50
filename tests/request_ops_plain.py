"""Plain 64-bit forms of what a request brings of its own (adapters, logit adjustments, token histories), row by row."""

import math

import torch


def adapter_rows(y, x, a, b, ids, scale=None, ranks=None, parts=None, pairs=False):
    """``(result, magnitude, products)`` in float64 on the CPU: the magnitude is the same sum with every term's absolute value,
    the products are the second product alone with the first one's sums as they are and every term's absolute value."""
    y, x, a, b = (t.detach().cpu().double() for t in (y, x, a, b))
    n, P, R, _ = a.shape
    N = y.shape[1]
    parts = list(parts) if parts is not None else [N // P] * P if pairs else [N]
    ends = torch.tensor(parts).cumsum(0)
    part_of = torch.arange(N) % 2 if pairs else torch.bucketize(torch.arange(N), ends, right=True)
    out, mag, products = y.clone(), y.abs(), torch.zeros_like(y)
    for t, i in enumerate(ids.tolist()):
        if not 0 <= i < n:
            continue
        r = R if ranks is None else min(int(ranks[i]), R)
        s = 1.0 if scale is None else float(scale[i])
        if r <= 0:
            continue
        h = a[i, :, :r] @ x[t]                                    # [P, r]
        hm = a[i, :, :r].abs() @ x[t].abs()
        out[t] += s * (b[i, :, :r] * h[part_of]).sum(1)
        mag[t] += abs(s) * (b[i, :, :r].abs() * hm[part_of]).sum(1)
        products[t] += abs(s) * (b[i, :, :r].abs() * h.abs()[part_of]).sum(1)
    return out, mag, products


def unpacked(words, V):
    return (((words.cpu()[:, :, None] >> torch.arange(32)) & 1).reshape(words.shape[0], -1)[:, :V]) != 0


def packed(flags):
    n, V = flags.shape
    wide = torch.zeros(n, -(-V // 32) * 32, dtype=torch.int64)
    wide[:, :V] = flags.cpu()
    words = (wide.view(n, -1, 32) << torch.arange(32)).sum(2)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def adjusted(logits, slots=None, seen=None, counts=None, repetition=None, presence=None, frequency=None, bias=None, masks=None,
             mask_rows=None):
    """``(result, magnitude)`` in float64 on the CPU."""
    z = logits.detach().cpu().double().clone()
    B, V = z.shape
    mag = z.abs()
    for i in range(B):
        slot = -1 if seen is None else int(slots[i]) if slots is not None else i
        if seen is not None and 0 <= slot < seen.shape[0]:
            told = unpacked(seen[slot:slot + 1], V)[0]
            if repetition is not None:
                r = float(repetition[i])
                z[i] = torch.where(told, torch.where(z[i] > 0, z[i] / r, z[i] * r), z[i])
                mag[i] = mag[i] * max(r, 1 / r)
            if counts is not None:
                c = counts[slot].cpu().double() * told
                f = float(frequency[i]) if frequency is not None else 0.0
                p = float(presence[i]) if presence is not None else 0.0
                z[i] -= f * c + p * (c > 0)
                mag[i] += abs(f) * c + abs(p)
        if bias is not None:
            starts, ids, values = (t.cpu().tolist() for t in bias)
            for j in range(max(0, starts[i]), min(len(ids), starts[i + 1])):
                if 0 <= ids[j] < V:
                    z[i, ids[j]] += values[j]
                    mag[i, ids[j]] += abs(values[j])
        m = -1 if masks is None else int(mask_rows[i]) if mask_rows is not None else i
        if masks is not None and 0 <= m < masks.shape[0]:
            z[i] = torch.where(unpacked(masks[m:m + 1], V)[0], z[i], torch.full_like(z[i], -math.inf))
    return z, mag


def recorded(counts, seen, slots, starts, tokens, n_prompt=None, fresh=False):
    counts, V = counts.cpu().clone(), counts.shape[1]
    told = unpacked(seen, V)
    tokens = tokens.tolist()
    n = len(tokens) if starts is None else len(starts) - 1
    for i in range(n):
        slot = i if slots is None else int(slots[i])
        if not 0 <= slot < counts.shape[0]:
            continue
        if fresh:
            counts[slot], told[slot] = 0, False
        first, last = (i, i + 1) if starts is None else (int(starts[i]), int(starts[i + 1]))
        made = first + (0 if n_prompt is None else int(n_prompt[i]))
        for j in range(max(0, first), min(last, len(tokens))):
            v = tokens[j]
            if 0 <= v < V:
                told[slot, v] = True
                counts[slot, v] += int(j >= made)
    return counts, packed(told)
