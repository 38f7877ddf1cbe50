"""Adapters beside a shared projection, adjusted logits and token histories against plain 64-bit forms, at the sizes and
values where they can go wrong."""

import math

import pytest
import torch

import request_ops_plain as P

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F, I, BF = torch.float32, torch.int32, torch.bfloat16
NAN, INF = float("nan"), math.inf


def ops():
    from mini_infer_b200.csrc import ops as o
    return o


def rnd(*shape, dtype=F, seed=0, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).to(DEV)


def ints(values):
    return torch.tensor(values, dtype=I, device=DEV)


# ----------------------------------------------------------------------------- adapters


def adapters(n, widths, R, K, dtype, seed=0):
    return (rnd(n, len(widths), R, K, dtype=dtype, seed=seed + 1, std=K ** -0.5),
            rnd(n, sum(widths), R, dtype=dtype, seed=seed + 2, std=max(R, 1) ** -0.5))


def check_adapter(got, y, x, a, b, ids, **kw):
    want, mag, products = P.adapter_rows(y, x, a, b, ids, **kw)
    K, R = x.shape[1], a.shape[2]
    # fp32 sums of K and of R terms in any order, and the scale: a step of 2^-23 for each; in bfloat16 the first sums may be
    # held as two bfloat16 numbers (2^-16) and the result is rounded once (half a step: 2^-8 of it)
    tol = mag * (K + R + 8) * 2.0 ** -23
    if y.dtype == BF:
        tol = tol + mag * 2.0 ** -16 + want.abs() * 2.0 ** -8
        # many rows of ranks above 32: every first sum h is rounded to bfloat16 once, to h (1 + e) with |e| <= 2^-8 (half a step),
        # so that a result, sum_r s h_r B_r, moves by at most 2^-8 sum_r |s h_r B_r|
        if x.shape[0] > 256 and R > 32:
            tol = tol + products * 2.0 ** -8
    off = (got.cpu().double() - want).abs()
    assert bool((off <= tol).all()), f"off by {(off - tol).max().item():.3g} over the bound at {int((off - tol).argmax())}"


def spread_ids(M, n, seed=0, bare=True):
    """Every adapter somewhere, in no order; some rows with none, and one number too high."""
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(-1 if bare else 0, n, (M,), generator=g)
    if bare and M > 4:
        ids[M // 2] = n
    return ids.to(I).to(DEV)


SHAPES = [   # M, K, widths, pairs, n, R
    (1, 64, (64,), False, 1, 8),
    (1, 4096, (4096, 1024, 1024), False, 4, 16),
    (2, 2048, (2048,), False, 3, 64),
    (7, 264, (40, 8, 24), False, 3, 24),
    (9, 520, (136, 136), True, 5, 16),
    (16, 1032, (72,), False, 2, 8),
    (17, 128, (320, 320), True, 16, 32),
    (33, 96, (200, 16, 64, 8), False, 4, 8),
    (64, 1024, (512, 128), False, 40, 16),
    (65, 176, (264,), False, 2, 40),
    (131, 2048, (256,), False, 3, 8),
    (257, 520, (96, 96), True, 7, 48),
    (600, 264, (328,), False, 5, 16),
    (300, 128, (128,), False, 200, 8),
    (130, 256, (512,), False, 2, 128),
    (40, 256, (264, 264), True, 3, 256),
    (200, 128, (272, 64, 48), False, 3, 16),
    (300, 264, (520, 8, 264), False, 5, 48),
    (280, 200, (64, 512, 128, 320), False, 2, 104),
    (290, 136, (400, 400), True, 4, 16),
    (513, 1024, (272, 272), True, 2, 64),
    (260, 64, (304, 304), True, 3, 128),
    (150, 72, (136,), False, 2, 200),
    (1000, 128, (2048, 512), False, 3, 32),
]


@pytest.mark.parametrize("dtype", [F, BF])
@pytest.mark.parametrize("M,K,widths,pairs,n,R", SHAPES)
def test_adapter_add_against_the_formula(M, K, widths, pairs, n, R, dtype):
    o = ops()
    a, b = adapters(n, widths, R, K, dtype)
    y, x = rnd(M, sum(widths), dtype=dtype, seed=5), rnd(M, K, dtype=dtype, seed=6)
    ids, scale = spread_ids(M, n), rnd(n, seed=8).abs() + 0.25
    parts = None if len(widths) == 1 else widths
    got = o.adapter_add(y, x, a, b, o.adapter_plan(ids, n), scale=scale, parts=parts, pairs=pairs)
    check_adapter(got, y, x, a, b, ids, scale=scale, parts=widths, pairs=pairs)
    bare = (ids < 0) | (ids >= n)
    assert torch.equal(got[bare], y[bare])
    y2 = y.clone()                               # in place, the same bits
    assert o.adapter_add(y2, x, a, b, o.adapter_plan(ids, n), scale=scale, parts=parts, pairs=pairs, out=y2, w_constant=True) is y2
    assert torch.equal(y2, got)


# widths, depths and ranks that are no whole number of 16-byte pieces
@pytest.mark.parametrize("dtype", [F, BF])
@pytest.mark.parametrize("M,K,widths,pairs,n,R", [
    (1, 1, (1,), False, 1, 1), (3, 7, (5,), False, 2, 3), (5, 100, (33, 1, 70), False, 3, 5), (70, 129, (131,), False, 4, 1),
    (9, 4099, (66,), False, 2, 12), (400, 65, (17, 17), True, 3, 2), (300, 36, (41, 8), False, 5, 6), (20, 64, (0, 40, 3), False, 2, 8), (6, 8, (16,), False, 3, 7),
])
def test_adapter_add_at_odd_sizes(M, K, widths, pairs, n, R, dtype):
    o = ops()
    a, b = adapters(n, widths, R, K, dtype)
    y, x = rnd(M, sum(widths), dtype=dtype, seed=5), rnd(M, K, dtype=dtype, seed=6)
    ids = spread_ids(M, n)
    got = o.adapter_add(y, x, a, b, o.adapter_plan(ids, n), parts=widths, pairs=pairs)
    check_adapter(got, y, x, a, b, ids, parts=widths, pairs=pairs)


@pytest.mark.parametrize("dtype", [F, BF])
@pytest.mark.parametrize("M", [6, 350])
def test_adapter_ranks_and_what_lies_behind_them(M, dtype):
    """Ranks from none to all, one over R; NaN behind them and in an adapter that no row uses is not read."""
    o, n, R, K, widths = ops(), 6, 24, 136, (80, 48)
    a, b = adapters(n, widths, R, K, dtype)
    ranks = [0, 1, 8, 15, 24, 99]
    for i, r in enumerate(ranks):
        a[i, :, r:], b[i, :, r:] = NAN, NAN
    ranks, ids = ints(ranks), ints([t % n if t % n != 3 else -1 for t in range(M)])
    a[3], b[3] = NAN, NAN
    y, x = rnd(M, 128, dtype=dtype, seed=5), rnd(M, K, dtype=dtype, seed=6)
    got = o.adapter_add(y, x, a, b, o.adapter_plan(ids, n), ranks=ranks, parts=widths)
    check_adapter(got, y, x, a, b, ids, ranks=ranks, parts=widths)
    assert torch.equal(got[ids == 0], y[ids == 0])


@pytest.mark.parametrize("dtype", [F, BF])
@pytest.mark.parametrize("M", [5, 390])
def test_rows_with_infinities_stay_among_themselves(M, dtype):
    o, n, K = ops(), 2, 64
    a, b = adapters(n, (72,), 8, K, dtype)
    y, x = rnd(M, 72, dtype=dtype, seed=5), rnd(M, K, dtype=dtype, seed=6)
    ids = ints([t % 2 for t in range(M)])
    clean = o.adapter_add(y, x, a, b, o.adapter_plan(ids, n))
    x[1, 3], x[2, 5], y[3, 7] = INF, NAN, -INF
    got = o.adapter_add(y, x, a, b, o.adapter_plan(ids, n))
    rest = [t for t in range(M) if t not in (1, 2, 3)]
    assert torch.equal(got[rest], clean[rest])
    assert not torch.isfinite(got[1]).any() and torch.isnan(got[2]).all() and got[3, 7].item() == -INF


@pytest.mark.parametrize("dtype", [F, BF])
@pytest.mark.parametrize("M", [4, 300])
def test_adapter_add_on_strided_rows(M, dtype):
    """Columns of wider matrices, at 16-byte boundaries and off them, and one row for all."""
    o, n, K, N = ops(), 3, 96, 104
    a, b = adapters(n, (N,), 16, K, dtype)
    ids = spread_ids(M, n)
    plan = o.adapter_plan(ids, n)
    for off in (8, 3):
        xw, yw, ow = (rnd(M, w, dtype=dtype, seed=s) for w, s in ((K + 40, 1), (N + 24, 2), (N + 51, 3)))
        before = ow.clone()
        x, y, out = xw[:, off:off + K], yw[:, off:off + N], ow[:, off:off + N]
        o.adapter_add(y, x, a, b, plan, out=out)
        check_adapter(out, y, x, a, b, ids)
        assert torch.equal(ow[:, :off], before[:, :off]) and torch.equal(ow[:, off + N:], before[:, off + N:])
    x = rnd(1, K, dtype=dtype, seed=9).expand(M, K)
    y = rnd(1, N, dtype=dtype, seed=10).expand(M, N)
    check_adapter(o.adapter_add(y, x, a, b, plan), y, x, a, b, ids)


def test_adapter_add_of_nothing():
    o = ops()
    for M, N, n, K, R in ((0, 8, 2, 16, 8), (3, 0, 2, 16, 8), (3, 8, 0, 16, 8), (3, 8, 2, 0, 8), (3, 8, 2, 16, 0), (70, 8, 0, 16, 8), (300, 8, 0, 16, 8), (300, 8, 2, 0, 8)):
        y, x = rnd(M, N, dtype=BF), rnd(M, K, dtype=BF)
        got = o.adapter_add(y, x, rnd(n, 1, R, K, dtype=BF), rnd(n, N, R, dtype=BF), o.adapter_plan(ints([0] * M), n))
        assert torch.equal(got, y)
    for M in (70, 300):
        y = rnd(M, 40, dtype=BF)
        got = o.adapter_add(y, rnd(M, 16, dtype=BF), *adapters(2, (40,), 8, 16, BF), o.adapter_plan(ints([-1] * M), 2))
        assert torch.equal(got, y)


@pytest.mark.parametrize("M", [9, 300])
def test_rows_beyond_32_bits(M):
    """Rows so far apart that their offsets pass 2^31 elements."""
    o, n, K, N, far = ops(), 2, 64, 72, 2 ** 31 // (M - 1) // 8 * 8 + 64
    a, b = adapters(n, (N,), 8, K, BF)
    room = torch.zeros((M - 1) * far + far, dtype=BF, device=DEV).view(M, far)
    y, x = rnd(M, N, dtype=BF, seed=5), rnd(M, K, dtype=BF, seed=6)
    room[:, :N].copy_(y)
    room[:, 80:80 + K].copy_(x)
    ids = spread_ids(M, n)
    out = torch.empty_like(room)[:, :N] if M < 50 else None
    got = o.adapter_add(room[:, :N], room[:, 80:80 + K], a, b, o.adapter_plan(ids, n), out=out)
    check_adapter(got, y, x, a, b, ids)


@pytest.mark.parametrize("M", [5, 300])
def test_adapters_captured_replayed_and_on_another_stream(M):
    """Two graphs and an eager call between them, with new ids in the same place; results do not depend on the others."""
    o, n, K, N = ops(), 4, 256, 264
    a, b = adapters(n, (N,), 16, K, BF)
    y, x = rnd(M, N, dtype=BF, seed=5), rnd(M, K, dtype=BF, seed=6)
    x2, ids, ids2 = rnd(M, K, dtype=BF, seed=7), spread_ids(M, n, 1), spread_ids(M, n, 2)

    def once(xx, ii):
        return o.adapter_add(y, xx, a, b, o.adapter_plan(ii, n), w_constant=True)

    eager, eager2 = once(x, ids), once(x2, ids2)
    held, held2 = ids.clone(), ids2.clone()
    graphs, outs = [], []
    torch.cuda.synchronize()
    for xx, ii in ((x, held), (x2, held2)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(once(xx, ii))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        assert torch.equal(once(x, ids), eager)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], eager) and torch.equal(outs[1], eager2)
    held.copy_(ids2)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], once(x, ids2))


@pytest.mark.parametrize("M", [8, 64, 320])
def test_a_rows_sum_does_not_depend_on_its_company(M):
    """The same row with the same adapter gives the same bits wherever it stands in a batch of one size."""
    o, n, K, N = ops(), 5, 520, 136
    a, b = adapters(n, (N,), 16, K, BF)
    y, x = rnd(M, N, dtype=BF, seed=5), rnd(M, K, dtype=BF, seed=6)
    ids = spread_ids(M, n, 3, bare=False)
    one = o.adapter_add(y, x, a, b, o.adapter_plan(ids, n))
    turn = torch.randperm(M, generator=torch.Generator().manual_seed(1)).to(DEV)
    other = o.adapter_add(y[turn].contiguous(), x[turn].contiguous(), a, b, o.adapter_plan(ids[turn].contiguous(), n))
    assert torch.equal(other, one[turn])
    assert torch.equal(o.adapter_add(y, x, a, b, o.adapter_plan(ids, n)), one)


def test_a_rows_sum_does_not_depend_on_how_many_share_its_adapter():
    """Items of up to four rows and of more hold the sums' rests elsewhere, and add up in the same order."""
    o, M, n, K, N = ops(), 16, 3, 264, 200
    for R in (16, 24, 64, 104):
        a, b = adapters(n, (N,), R, K, BF, seed=R)
        y, x = rnd(M, N, dtype=BF, seed=5), rnd(M, K, dtype=BF, seed=6)
        alone = ints([0, 1, 0, 1, 1, 0, 2, 2, 2, -1, -1, -1, -1, -1, -1, -1])
        together = ints([0, 1, 0, 1, 1, 0, 2, 2, 2, 0, 1, 0, 1, 0, 1, 2])
        few = o.adapter_add(y, x, a, b, o.adapter_plan(alone, n))
        more = o.adapter_add(y, x, a, b, o.adapter_plan(together, n))
        assert torch.equal(few[:9], more[:9])


@pytest.mark.parametrize("K", [200, 4096])
def test_float32_rows_have_the_same_bits_in_any_company(K):
    """As every sum of the 32-bit path: alone, among few rows, among many, beside more adapters, on strided rows."""
    o, n, N, M = ops(), 6, 136, 700
    a, b = adapters(n, (N,), 12, K, F)
    y, x = rnd(M, N, seed=5), rnd(M, K, seed=6)
    ids = spread_ids(M, n, 3)
    whole = o.adapter_add(y, x, a, b, o.adapter_plan(ids, n))
    for lo, hi in ((0, 1), (5, 6), (0, 9), (100, 300), (300, 699)):
        part = ids[lo:hi].contiguous()
        assert torch.equal(o.adapter_add(y[lo:hi], x[lo:hi], a, b, o.adapter_plan(part, n)), whole[lo:hi])
    wide = torch.empty(M, K + 1, device=DEV)
    wide[:, 1:] = x                              # rows off their 16-byte boundaries
    assert torch.equal(o.adapter_add(y, wide[:, 1:], a, b, o.adapter_plan(ids, n)), whole)


@pytest.mark.parametrize("M,n,R,widths,pairs", [
    (200, 40, 16, (520, 8, 300, 772), False), (256, 3, 24, (2000, 24), False), (130, 130, 64, (1304,), False),
    (256, 64, 16, (1368, 1368), True), (90, 30, 200, (264, 1000), False), (300, 9, 136, (1400, 8, 264), False),
    (700, 3, 200, (900, 900), True)])
def test_tiles_of_many_items_shared_out_over_blocks(M, n, R, widths, pairs):
    """Stretches of tiles that cross parts and items, among them items of rank 0 and rows without an adapter."""
    o, K = ops(), 1040
    a, b = adapters(n, widths, R, K, BF)
    y, x = rnd(M, sum(widths), dtype=BF, seed=5), rnd(M, K, dtype=BF, seed=6)
    ids = spread_ids(M, n, 2)
    ranks = ints([(0, R, 1, 8, R - 3)[i % 5] for i in range(n)])
    plan = o.adapter_plan(ids, n)
    got = o.adapter_add(y, x, a, b, plan, ranks=ranks, parts=widths, pairs=pairs)
    check_adapter(got, y, x, a, b, ids, ranks=ranks, parts=widths, pairs=pairs)
    y2 = y.clone()
    o.adapter_add(y2, x, a, b, plan, ranks=ranks, parts=widths, pairs=pairs, out=y2)
    assert torch.equal(y2, got)


@pytest.mark.parametrize("dtype", [F, BF])
def test_a_plan_read_by_a_kernel_that_starts_early(dtype):
    """Calls that add nothing, behind a fresh plan: rows come out as they were, whatever the memory of the plan held before."""
    o, M = ops(), 2000
    y = rnd(M, 24, dtype=dtype, seed=1)
    for n, R, K in ((0, 8, 16), (3, 0, 16), (3, 8, 0)):
        x, a, b = rnd(M, K, dtype=dtype), rnd(n, 1, R, K, dtype=dtype), rnd(n, 24, R, dtype=dtype)
        for i in range(20):
            ids = spread_ids(M, max(n, 1), i)
            assert torch.equal(o.adapter_add(y, x, a, b, o.adapter_plan(ids, n)), y)


# ----------------------------------------------------------------------------- logits


def histories(slots, V, length, seed=0):
    g = torch.Generator().manual_seed(seed)
    tokens = (torch.rand(slots, length, generator=g).pow(3) * V).long().clamp(max=V - 1)
    made = torch.rand(slots, length, generator=g) < 0.5
    counts = torch.zeros(slots, V, dtype=I).scatter_add_(1, tokens, made.to(I))
    return counts.to(DEV), P.packed(torch.zeros(slots, V, dtype=torch.bool).scatter_(1, tokens, True)).to(DEV)


def check_adjusted(got, logits, **kw):
    want, mag = P.adjusted(logits, **kw)
    got = got.cpu().double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    # up to four rounded operations, each by half a step of its operands at most, and one more for every bias of a token
    n = 4 + (int(kw["bias"][1].numel()) if kw.get("bias") is not None and kw["bias"][1].numel() < 64 else 4)
    assert bool(((got - want).abs()[fine] <= n * 2.0 ** -24 * mag[fine]).all())


def full_set(B, V, seed=0):
    slots = 2 * B
    counts, seen = histories(slots, V, max(1, V // 3), seed)
    g = torch.Generator().manual_seed(seed + 1)
    rows = torch.randperm(slots, generator=g)[:B].to(I)
    each = [min(V, (i * 5) % 40) for i in range(B)]
    ids = torch.cat([torch.randperm(V, generator=g)[:k] for k in each] or [torch.empty(0)]).to(I)
    masks = P.packed(torch.rand(3, V, generator=g) < torch.tensor([[0.5], [0.02], [0.98]]))
    mask_rows = torch.tensor([(i % 5) - 1 for i in range(B)], dtype=I)       # -1 and 3: all tokens
    return dict(slots=rows.to(DEV), seen=seen, counts=counts, repetition=(torch.rand(B, generator=g) + 0.6).to(DEV),
                presence=(torch.rand(B, generator=g) - 0.3).to(DEV), frequency=(torch.rand(B, generator=g) - 0.3).to(DEV),
                bias=(torch.tensor([0] + each).cumsum(0).to(I).to(DEV), ids.to(DEV), rnd(ids.numel(), seed=seed + 2, std=4.0)),
                masks=masks.to(DEV), mask_rows=mask_rows.to(DEV))


@pytest.mark.parametrize("B,V", [(1, 1), (2, 31), (3, 32), (1, 33), (4, 1000), (2, 8192), (3, 8195), (5, 32000), (70, 517), (2, 50021), (1, 128256)])
def test_adjusted_logits_against_the_formula(B, V):
    o = ops()
    z = rnd(B, V, seed=3, std=3.0)
    kw = full_set(B, V)
    before = z.clone()
    got = o.adjust_logits(z, **kw)
    assert torch.equal(z, before)
    check_adjusted(got, z, **kw)
    assert o.adjust_logits(z, z, **kw) is z
    assert torch.equal(z, got)                   # in place, the same bits


PENALTIES, COUNTS = ("slots", "seen", "counts", "repetition", "presence", "frequency"), ("slots", "seen", "counts")


@pytest.mark.parametrize("keys", [(), ("slots", "seen", "repetition"), COUNTS + ("presence",), COUNTS + ("frequency",), PENALTIES, ("bias",),
                                  ("masks", "mask_rows"), ("bias", "masks", "mask_rows"), PENALTIES + ("bias",)])
@pytest.mark.parametrize("B,V", [(3, 1000), (2, 8193)])
def test_each_adjustment_alone(B, V, keys):
    o = ops()
    z, every = rnd(B, V, seed=3, std=3.0), full_set(B, V, 7)
    kw = {k: every[k] for k in keys}
    got = o.adjust_logits(z, **kw)
    check_adjusted(got, z, **kw)
    if not kw:
        assert torch.equal(got, z)
    wide = rnd(B, V + 9, seed=4)                 # rows apart, in and out, at an odd place
    keep = wide.clone()
    view = wide[:, 5:5 + V]
    view.copy_(z)
    out = torch.zeros(B, V + 3, device=DEV)
    assert torch.equal(o.adjust_logits(view, out[:, 1:1 + V], **kw), got)
    assert not out[:, :1].any() and not out[:, 1 + V:].any()
    o.adjust_logits(view, view, **kw)
    assert torch.equal(view, got)
    assert torch.equal(wide[:, :5], keep[:, :5]) and torch.equal(wide[:, 5 + V:], keep[:, 5 + V:])


def test_rows_without_a_history_or_a_mask_and_numbers_outside():
    o, B, V = ops(), 5, 300
    z, kw = rnd(B, V, seed=3), full_set(B, V, 2)
    kw.pop("bias")
    kw["slots"], kw["mask_rows"] = ints([-1, 2, 10, 3, -2 ** 31]), ints([3, -7, 0, 2 ** 31 - 1, -1])
    got = o.adjust_logits(z, **kw)
    check_adjusted(got, z, **kw)
    assert torch.equal(got[0], z[0]) and torch.equal(got[4], z[4])


def test_special_logits():
    """Infinities and NaN, the type's lowest value, both zeros; masked places are minus infinity whatever they held."""
    o, V = ops(), 96
    lowest = torch.finfo(F).min
    z = torch.zeros(2, V, device=DEV)
    for k, v in enumerate((INF, -INF, NAN, lowest, -lowest, 0.0, -0.0, 1e-42)):
        z[:, k::8] = v
    counts, seen = torch.zeros(2, V, dtype=I, device=DEV), torch.full((2, 3), -1, dtype=I, device=DEV)
    counts[:, ::3] = 2
    masks = P.packed(torch.arange(V)[None, :] % 5 != 0).to(DEV)
    rep, zero = torch.tensor([1.25, 0.5], device=DEV), torch.zeros(2, device=DEV)
    got = o.adjust_logits(z, seen=seen, counts=counts, repetition=rep, presence=zero + 1, frequency=zero + 0.5, masks=masks,
                          mask_rows=ints([0, 0]))
    assert bool((got[:, ::5] == -INF).all())
    x = z.clone()
    x = torch.where(x > 0, x / rep[:, None], x * rep[:, None])
    x[:, ::3] = x[:, ::3] - 1.0 - 1.0
    keep = torch.arange(V, device=DEV) % 5 != 0
    assert torch.equal(got[:, keep].nan_to_num(7.0, 8.0, 9.0), x[:, keep].nan_to_num(7.0, 8.0, 9.0))
    nothing = o.adjust_logits(z, masks=torch.zeros(1, 3, dtype=I, device=DEV), mask_rows=ints([0, -1]))
    assert bool((nothing[0] == -INF).all()) and torch.equal(nothing[1].nan_to_num(7.0), z[1].nan_to_num(7.0))
    bias = (ints([0, 2, 4]), ints([0, 1, 0, 1]), torch.tensor([INF, INF, -INF, 2.0], device=DEV))
    both = o.adjust_logits(torch.zeros(2, V, device=DEV), bias=bias, masks=masks, mask_rows=ints([0, -1]))
    assert both[0, 0].item() == -INF and both[0, 1].item() == INF and both[1, 0].item() == -INF and both[1, 1].item() == 2.0


def test_biases_of_one_token_add_up_in_their_order():
    o, V = ops(), 9000
    # 1, 2^25, -2^25 and 1 in this order give 2^25 + 1 -> 2^25, then 0, then 1
    ids, values = [7, 8999, 7, 7, 40, 7] + [8191, 8192] * 50, [1.0, 3.0, 2.0 ** 25, -2.0 ** 25, -1.0, 1.0] + [0.5, 0.25] * 50
    n = len(ids)
    extra = [-1, V, 2 ** 31 - 1, -2 ** 31]                                        # not in the vocabulary
    bias = (ints([0, n, n, 2 * n + 4]), ints(ids + ids + extra), torch.tensor(values + values + [9.0] * 4, device=DEV))
    z = torch.zeros(3, V, device=DEV)
    got = o.adjust_logits(z, bias=bias)
    for row in (0, 2):
        assert got[row, 7].item() == 1.0 and got[row, 8999].item() == 3.0 and got[row, 40].item() == -1.0
        assert got[row, 8191].item() == 25.0 and got[row, 8192].item() == 12.5
        assert int((got[row] != 0).sum()) == 5
    assert not got[1].any()
    wild = (ints([-5, 3, 2, 10 ** 6]), bias[1], bias[2])      # starts that lie outside the lists: what there is of them
    assert torch.isfinite(o.adjust_logits(z, bias=wild)).all()


def test_a_long_list_of_biases():
    o, V, n = ops(), 20000, 5000
    ids = (torch.arange(n) * 3).to(I).to(DEV)
    bias = (ints([0, n]), ids, rnd(n, seed=1))
    z = rnd(1, V, seed=2)
    check_adjusted(o.adjust_logits(z, bias=bias), z, bias=bias)


def test_logits_beyond_32_bits():
    o, V, far = ops(), 40000, 2 ** 30
    room = torch.zeros(3 * far, device=DEV).view(3, far)
    z, kw = rnd(3, V, seed=3), full_set(3, V, 4)
    room[:, :V].copy_(z)
    got = o.adjust_logits(z, **kw)
    o.adjust_logits(room[:, :V], room[:, :V], **kw)
    assert torch.equal(room[:, :V], got)
    slots = 2 ** 31 // 128000 + 2                # histories beyond 2^31 counts
    V = 128000
    counts, seen = torch.zeros(slots, V, dtype=I, device=DEV), torch.zeros(slots, V // 32, dtype=I, device=DEV)
    o.record_tokens(counts, seen, ints([slots - 1]), ints([0, 3]), ints([5, 127999, 127999]), n_prompt=ints([1]), fresh=True)
    o.record_tokens(counts, seen, ints([slots - 1]), None, ints([127999]))
    assert counts[-1, 127999].item() == 3 and counts[-1, 5].item() == 0 and int(counts.view(-1)[:-V].count_nonzero()) == 0
    z = torch.ones(1, V, device=DEV)
    got = o.adjust_logits(z, slots=ints([slots - 1]), seen=seen, counts=counts, repetition=torch.tensor([2.0], device=DEV),
                          frequency=torch.tensor([1.0], device=DEV))
    assert got[0, 5].item() == 0.5 and got[0, 127999].item() == -2.5 and int((got != 1).sum()) == 2


# ----------------------------------------------------------------------------- histories


@pytest.mark.parametrize("V", [1, 31, 32, 1000, 8192, 8193, 20011, 128256])
@pytest.mark.parametrize("fresh", [True, False])
def test_recorded_tokens_against_counting(V, fresh):
    o, g = ops(), torch.Generator().manual_seed(V)
    lengths = [5, 0, 1, 700, 33, 4000]
    B, slots = len(lengths), 9
    starts = torch.tensor([0] + lengths).cumsum(0).to(I)
    tokens = (torch.rand(sum(lengths), generator=g).pow(3) * V).to(I).clamp(max=V - 1)
    tokens[::97] = torch.tensor([-1, V, 2 ** 31 - 1, -2 ** 31], dtype=I).repeat(len(tokens[::97]))[:len(tokens[::97])]
    n_prompt = torch.tensor([5, 0, 0, 300, 99, 0], dtype=I)
    where = torch.tensor([4, 0, 8, 2, 5, 6], dtype=I)
    counts, seen = histories(slots, V, 50, 3)
    want = P.recorded(counts, seen, where, starts, tokens, n_prompt, fresh)
    o.record_tokens(counts, seen, where.to(DEV), starts.to(DEV), tokens.to(DEV), n_prompt=n_prompt.to(DEV), fresh=fresh)
    assert torch.equal(counts.cpu(), want[0]) and torch.equal(seen.cpu(), want[1])
    want = P.recorded(counts, seen, None, None, torch.tensor([0, 0, V - 1]))      # a decode step's tokens
    o.record_tokens(counts, seen, None, None, ints([0, 0, V - 1]))
    assert torch.equal(counts.cpu(), want[0]) and torch.equal(seen.cpu(), want[1])


def test_slots_outside_and_the_same_slot_twice():
    o, V = ops(), 500
    counts, seen = histories(4, V, 20, 1)
    before = (counts.clone(), seen.clone())
    for fresh in (True, False):
        o.record_tokens(counts, seen, ints([-1, 4, 2 ** 31 - 1]), ints([0, 1, 2, 3]), ints([1, 2, 3]), fresh=fresh)
    assert torch.equal(counts, before[0]) and torch.equal(seen, before[1])
    where, starts, tokens = ints([2, 2, 2]), ints([0, 2, 3, 6]), ints([9, 9, 9, 10, 9, 11])
    want = P.recorded(counts, seen, where, starts, tokens)
    o.record_tokens(counts, seen, where, starts, tokens)
    assert torch.equal(counts.cpu(), want[0]) and torch.equal(seen.cpu(), want[1])


def test_histories_through_a_generation_captured():
    """Admission, then steps of adjust, choose, record as a captured graph: each step sees what the last one chose."""
    o, V = ops(), 1000
    counts, seen = (torch.zeros(2, n, dtype=I, device=DEV) for n in (V, 32))
    slots = ints([1, 0])
    z = torch.zeros(2, V, device=DEV)
    z[:, 100:110] = torch.arange(10, 0, -1, device=DEV) * 0.1 + 5.0
    o.record_tokens(counts, seen, slots, ints([0, 2, 3]), ints([100, 101, 100]), n_prompt=ints([2, 1]), fresh=True)
    rep, freq = torch.tensor([2.0, 1.0], device=DEV), torch.tensor([0.0, 0.25], device=DEV)
    chosen = torch.empty(2, dtype=I, device=DEV)

    def step():
        o.sample(o.adjust_logits(z, slots=slots, seen=seen, counts=counts, repetition=rep, frequency=freq), chosen)
        o.record_tokens(counts, seen, slots, None, chosen)

    step()                                       # kernel by kernel, then the same as a graph
    got = [chosen.tolist()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(5):
        graph.replay()
        got.append(chosen.tolist())
    # row 0 (repetition): the prompt's 100, 101 are halved, every token comes once; row 1 (frequency): 0.25 off for every time
    assert [t[0] for t in got] == [102, 103, 104, 105, 106, 107]
    level, want = {v: 5.0 + 0.1 * (110 - v) for v in range(100, 110)}, []
    for _ in range(6):
        want.append(max(level, key=lambda v: (round(level[v], 4), -v)))
        level[want[-1]] -= 0.25
    assert [t[1] for t in got] == want
