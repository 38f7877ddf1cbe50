"""Low-rank adapters of requests beside the projections of a model's parts.

A part that takes adapters says which of its projections do (``Part.adapted``): the tensors that are merged in one product, how
their columns lie, and how wide they are.  An :class:`AdapterBank` holds, for one such product, the matrices of every adapter of
the engine side by side, so that a step's requests may each use another one; ``add`` is what a part calls behind the product.
The operator is ``csrc/adapters.cu``: ``y + s B (A x)`` with the adapter of each row.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from ..csrc import ops


@dataclass(frozen=True)
class AdaptedProduct:
    """One product of a part that adapters may stand beside: ``tensors`` are the local names of the matrices merged in it, in the order of
    its columns, ``widths`` their columns, ``inputs`` what they read.  ``pairs``: two matrices whose columns alternate."""

    name: str
    tensors: tuple[str, ...]
    widths: tuple[int, ...]
    inputs: int
    pairs: bool = False


class AdapterBank:
    """``count`` adapters of rank up to ``rank`` (a multiple of 8) for one product; empty ones add nothing."""

    def __init__(self, product: AdaptedProduct, count: int, rank: int, dtype: torch.dtype, device) -> None:
        self.product = product
        self.rank = rank
        P, N, K = len(product.tensors), sum(product.widths), product.inputs
        self.a = torch.zeros((count, P, rank, K), dtype=dtype, device=device)
        self.b = torch.zeros((count, N, rank), dtype=dtype, device=device)
        self.scale = torch.zeros(count, dtype=torch.float32, device=device)
        self.ranks = torch.zeros(count, dtype=torch.int32, device=device)

    def columns(self, part: int) -> slice:
        if self.product.pairs:
            return slice(part, None, 2)
        first = sum(self.product.widths[:part])
        return slice(first, first + self.product.widths[part])

    def clear(self, index: int) -> None:
        self.ranks[index] = 0
        self.a[index].zero_()
        self.b[index].zero_()

    def put(self, index: int, matrices: dict[str, tuple[torch.Tensor, torch.Tensor]], scale: float) -> None:
        """The adapter's matrices ``tensor -> (A [r, inputs], B [width, r])``; a tensor that it leaves out gets nothing added."""
        self.clear(index)
        rank = max((a.shape[0] for a, _ in matrices.values()), default=0)
        for part, name in enumerate(self.product.tensors):
            if name in matrices:
                a, b = matrices[name]
                self.a[index, part, :a.shape[0]].copy_(a)
                self.b[index, self.columns(part), :a.shape[0]].copy_(b)
        self.scale[index] = scale
        self.ranks[index] = rank

    def add(self, y: torch.Tensor, x: torch.Tensor, plan: "ops.AdapterPlan") -> torch.Tensor:
        """``y`` (the product of ``x``) with every row's adapter added in place."""
        p = self.product
        return ops.adapter_add(y, x, self.a, self.b, plan, scale=self.scale, ranks=self.ranks, parts=p.widths, pairs=p.pairs, out=y,
                               w_constant=True)
