"""What becomes of an adapter's first sums on their way into the second product."""

import math

import pytest
import torch

import request_ops_plain as P

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F, I, BF = torch.float32, torch.int32, torch.bfloat16


def ops():
    from mini_infer_b200.csrc import ops as o
    return o


def rnd(*shape, dtype=F, seed=0, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).to(DEV)


@pytest.mark.parametrize("M,widths,pairs,R", [
    (200, (264, 136), False, 64), (256, (136, 136), True, 64), (257, (264, 136), False, 64), (257, (136, 136), True, 64),
    (300, (520,), False, 40), (290, (264, 264), True, 128), (400, (72, 8, 40), False, 128), (270, (136, 136), True, 104),
    (300, (136,), False, 24), (300, (200, 200), True, 32), (300, (137,), False, 48), (300, (136,), False, 200)])
def test_first_sums_keep_two_numbers_at_every_rank(M, widths, pairs, R):
    """A row of x has one number that is not zero, so that a first sum is one product, which fp32 holds exactly; and y takes away
    most of what is added, so that the result's own rounding is small beside an error of the sums."""
    o, n, K, N = ops(), 4, 136, sum(widths)
    a, b = rnd(n, len(widths), R, K, dtype=BF, seed=1), rnd(n, N, R, dtype=BF, seed=2)
    ranks = torch.tensor([R, 8, R - 3, R], dtype=I, device=DEV)        # (a low rank beside high ones)
    ids = torch.tensor([t % (n + 1) - 1 for t in range(M)], dtype=I, device=DEV)
    x = torch.zeros(M, K, dtype=BF, device=DEV)
    x[torch.arange(M), torch.arange(M) * 7 % K] = rnd(M, dtype=BF, seed=3)
    kw = dict(ranks=ranks, parts=widths, pairs=pairs)
    y = -P.adapter_rows(torch.zeros(M, N), x, a, b, ids, **kw)[0].to(BF).to(DEV)
    want, _, products = P.adapter_rows(y, x, a, b, ids, **kw)
    got = o.adapter_add(y, x, a, b, o.adapter_plan(ids, n), **kw)
    # a sum as two bfloat16 numbers: 2^-16 of it; 2 R products and y in fp32: a step of 2^-23 for each; the result: half a step
    tol = (products + y.cpu().double().abs()) * (2 * R + 8) * 2.0 ** -23 + products * 2.0 ** -16 + want.abs() * 2.0 ** -8
    off = (got.cpu().double() - want).abs()
    assert bool((off <= tol).all()), f"off by {(off / tol.clamp(min=2.0 ** -60)).max().item():.3g} times the bound"
    assert math.isfinite(off.max().item())


@pytest.mark.parametrize("M,widths,pairs,R,dtype", [
    (5, (264, 136), False, 8, BF), (40, (136, 136), True, 16, BF), (9, (264,), False, 24, BF), (100, (136, 136), True, 64, BF),
    (30, (72,), False, 200, BF), (300, (264, 136), False, 16, BF), (300, (136, 136), True, 32, BF), (300, (136, 136), True, 64, BF),
    (290, (264, 8), False, 128, BF), (300, (72,), False, 200, BF), (300, (137,), False, 12, BF), (40, (137,), False, 12, F)])
def test_infinite_elements_of_b(M, widths, pairs, R, dtype):
    """As the formula has it: an infinity where one product is infinite, or several of one sign, NaN where two signs meet or a sum is
    zero.  Sums that one bfloat16 number holds, and sums whose rest has their sign or the other one."""
    o, n, K, N = ops(), 3, 136, sum(widths)
    a, b = rnd(n, len(widths), R, K, dtype=dtype, seed=1), rnd(n, N, R, dtype=dtype, seed=2)
    a[:, :, :, ::5] = 0.5                                             # (sums without a rest)
    a[0, 0, 0] = 0                                                    # (one that is zero)
    inf = float("inf")
    b[:, ::3, 0], b[:, 1::5, R // 2], b[:, 2::7, R - 1] = inf, -inf, inf
    ids = torch.tensor([t % (n + 1) - 1 for t in range(M)], dtype=I, device=DEV)
    x = torch.zeros(M, K, dtype=dtype, device=DEV)
    x[torch.arange(M), torch.arange(M) * 7 % K] = rnd(M, dtype=dtype, seed=3)
    x[3, 21] = inf                                                    # an infinite sum: what it meets is infinite or NaN
    y = rnd(M, N, dtype=dtype, seed=4)
    kw = dict(parts=widths, pairs=pairs)
    want, _, products = P.adapter_rows(y, x, a, b, ids, **kw)
    assert bool(torch.isinf(want).any()) and bool(torch.isnan(want).any())
    got = o.adapter_add(y, x, a, b, o.adapter_plan(ids, n), **kw).cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
    fine = torch.isfinite(want)
    tol = (products + y.cpu().double().abs()) * (2 * R + 8) * 2.0 ** -23 + products * 2.0 ** -16 + (want.abs() * 2.0 ** -8 if dtype == BF else 0)
    assert bool(((got - want).abs() <= tol)[fine].all())
