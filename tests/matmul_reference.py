"""The segmented matrix product and its gradients in 64 bits, with bounds on
the error of an f32 accumulation; shared by the product's tests.

Bound.  A sum of m products, each exact or rounded to f32 and added in any
order in f32, is off by at most (m + 1) 2^-24 of the sum of the products'
absolute values (a fused or a tensor-core multiply-add rounds no more often;
the tensor cores add groups of products with the alignment of the largest, cut
off below its 2^-24 or finer, which is one more such error for each product).
So |error| <= 2 (m + 1) 2^-24 sum |l| |r|, then one rounding to the output's type.
"""
from __future__ import annotations

import numpy as np

from scan_reference import HALF, TINY


def products(values, weights, offsets, grad_out=None):
    """name -> (value, bound) of out and, with ``grad_out``, the gradients."""
    n, k = values.shape
    b, _, m = weights.shape
    out, bound = np.zeros((n, m)), np.zeros((n, m))
    gv, gv_bound = np.zeros((n, k)), np.zeros((n, k))
    gw, gw_bound = np.zeros((b, k, m)), np.zeros((b, k, m))

    def times(left, right):
        with np.errstate(all="ignore"):
            return left @ right, 2 * (left.shape[1] + 1) * 2.0 ** -24 * (np.abs(left) @ np.abs(right))

    for s in range(b):
        rows = slice(offsets[s], offsets[s + 1])
        out[rows], bound[rows] = times(values[rows], weights[s])
        if grad_out is not None:
            gv[rows], gv_bound[rows] = times(grad_out[rows], weights[s].T)
            gw[s], gw_bound[s] = times(values[rows].T, grad_out[rows])
    found = dict(out=(out, bound))
    if grad_out is not None:
        found.update(grad_values=(gv, gv_bound), grad_weights=(gw, gw_bound))
    return found


def close(actual, pair, dtype):
    expected, bound = pair
    with np.errstate(all="ignore"):
        limit = bound + HALF[dtype] * (np.abs(expected) + bound) + TINY[dtype]
        good = (actual == expected) | (np.isnan(actual) & np.isnan(expected)) | (np.abs(actual - expected) <= limit)
    assert good.all(), (f"{(~good).sum()} of {good.size} values off; first at {tuple(np.argwhere(~good)[0])}: "
                        f"{actual[~good][0]} for {expected[~good][0]}, limit {limit[~good][0]}")
