"""How evenly points spread over the superpoints they may belong to: counts, mean weights, and a loss that is 1 where both are even
and M where one superpoint takes everything. A learned association (`sp_W[N, M]`, LBS_method 'W') or learned neighbour weights collapse
onto few superpoints unless something holds against it; the reference (network.py:498-521) has nothing that does.

    P_m = mean weight of superpoint m over the T points that count
    f_m = its share of all choices (each point chooses the K superpoints of largest logit, or its neighbour of largest weight)
    loss = M * sum_m f_m P_m,  differentiable in the weights through P; the choices carry no gradient
"""
from __future__ import annotations

from typing import Optional, Tuple

from torch import Tensor

from fast_sp_gs_amd.lib import host

__all__ = ['balance_loss', 'neighbour_balance']


def balance_loss(logits: Tensor, K: int = 1, rows: Optional[Tensor] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """(loss [], counts [M] int32, importance P [M]) of association logits [N, M] (float32, float16 or bfloat16; sums in float32 or more),
    whose softmax over the superpoints is the weight. Equal logits are chosen by the lowest index; -inf marks a superpoint that a point
    may not use, and is never chosen. `rows` [N] bool: the points that count; the others' logits are not looked at and get a gradient
    of 0, as do points whose logits are all -inf. K is at most 64, M at most 2^26 - 16, N below 2^31 - 1. loss and importance are differentiable in the
    logits."""
    return host.balance_loss(logits, K, rows)


def neighbour_balance(weights: Tensor, indices: Tensor, M: int, rows: Optional[Tensor] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """`balance_loss` of neighbour weights [N, K] in [0, 1] with their superpoints' indices [N, K] (what `calc_LBS_weight` returns), of
    M superpoints; chosen is a point's neighbour of largest weight, the first of equal ones. An index may be there twice. A weight that
    is negative, above 1.0001 (roundings above 1 pass) or NaN, or an index outside [0, M), in a row that counts makes loss and importance
    NaN. Weights are added in units of 2^-31; N K is below 2^33."""
    return host.neighbour_balance(weights, indices, M, rows)
