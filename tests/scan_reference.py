"""The segmented scan in 64 bits, row by row, with bounds on the error of an
f32 evaluation; shared by the scan's CPU and GPU tests.

    h[t] = a[t] h[t-1] + x[t],  u[t] = a[t] g[t],  g[t] = dh[t] + u[t+1]

Bound.  h[t] is a sum of products x[s] a[s+1] ... a[t] over the rows s of its
segment.  However the products and sums are grouped, a term of a segment with
m rows up to t passes at most m multiplications and m additions, plus one of
each where two of the at most 64 pieces of the evaluation tree meet, each off
by at most 2^-24 of its result.  So |error| <= (2 m + 128) 2^-24 (1 + small) times
the same sum over absolute values, which the majorant recurrence
M[t] = |a[t]| M[t-1] + |x[t]| computes.  The same holds for g in the other
direction.  da = g h' adds one rounding to both errors' products.

Below 2^-126 a rounding is off by up to 2^-150 whatever its result.  What it
changes is later multiplied by gates, which the tests keep at or below one in
magnitude where products underflow, and where it is a product of gates, once
by a state, which no majorant is below.  So the same (2 m + 128) roundings add
at most 2^-149 (1 + max M) each.
"""
from __future__ import annotations

import numpy as np

STEP = 2.0 ** -24
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133}


def forward(values, gates, offsets, initial=None):
    """(h, h before each row, final, majorant, rows since the segment's start)"""
    n, d = values.shape
    h, before, major = np.zeros((n, d)), np.zeros((n, d)), np.zeros((n, d))
    count = np.zeros((n, 1))
    b = len(offsets) - 1
    final, final_major = np.zeros((b, d)), np.zeros((b, d))
    with np.errstate(all="ignore"):
        for s in range(b):
            state = initial[s].astype(np.float64) if initial is not None else np.zeros(d)
            bound = np.abs(state)
            for t in range(offsets[s], offsets[s + 1]):
                before[t] = state
                if t == offsets[s] and initial is None:
                    state, bound = values[t], np.abs(values[t])
                else:
                    state = gates[t] * state + values[t]
                    bound = np.abs(gates[t]) * bound + np.abs(values[t])
                h[t], major[t] = state, bound
                count[t] = t - offsets[s] + 1
            final[s], final_major[s] = state, bound
    return dict(out=h, before=before, final=final, major=major, final_major=final_major, count=count)


def backward(values, gates, offsets, grad_out, grad_final=None, initial=None):
    n, d = values.shape
    f = forward(values, gates, offsets, initial)
    b = len(offsets) - 1
    g, gmajor, count = np.zeros((n, d)), np.zeros((n, d)), np.zeros((n, 1))
    gi, gimajor = np.zeros((b, d)), np.zeros((b, d))
    with np.errstate(all="ignore"):
        for s in range(b):
            u = grad_final[s].astype(np.float64) if grad_final is not None else np.zeros(d)
            um = np.abs(u)
            for t in range(offsets[s + 1] - 1, offsets[s] - 1, -1):
                g[t] = grad_out[t] + u
                gmajor[t] = np.abs(grad_out[t]) + um
                u, um = gates[t] * g[t], np.abs(gates[t]) * gmajor[t]
                count[t] = offsets[s + 1] - t
            gi[s], gimajor[s] = u, um
        gate = g * f["before"]
        before_major = np.zeros((n, d))
        for s in range(b):
            lo, hi = offsets[s], offsets[s + 1]
            if hi > lo:
                before_major[lo] = np.abs(initial[s]) if initial is not None else 0
                before_major[lo + 1:hi] = f["major"][lo:hi - 1]
            if initial is None and hi > lo:
                gate[lo] = 0
    return dict(f, grad_values=g, grad_gates=gate, grad_initial=gi, gmajor=gmajor, gcount=count, gimajor=gimajor,
                before_major=before_major)


def close(actual, expected, bound, dtype):
    """Within the evaluation's bound, then one rounding to ``dtype``."""
    with np.errstate(all="ignore"):
        limit = bound + HALF[dtype] * (np.abs(expected) + bound) + TINY[dtype]
        same = (actual == expected) | (np.isnan(actual) & np.isnan(expected))
        good = same | (np.abs(actual - expected) <= limit)
    assert good.all(), (f"{(~good).sum()} of {good.size} values off; first at {tuple(np.argwhere(~good)[0])}: "
                        f"{actual[~good][0]} for {expected[~good][0]}, limit {np.broadcast_to(limit, good.shape)[~good][0]}")


def slack(count, major):
    return (2 * count + 128) * (STEP * major + 2.0 ** -149 * (1 + major.max(initial=0.0)))


def check_forward(ref, out, final, dtype):
    close(out, ref["out"], slack(ref["count"], ref["major"]), dtype)
    if final is not None:
        rows = max(1.0, float(ref["count"].max(initial=0)))
        close(final, ref["final"], slack(rows, ref["final_major"]), "f32")


def check_backward(ref, grad_values, grad_gates, grad_initial, dtype):
    eg = slack(ref["gcount"], ref["gmajor"])
    eh = slack(ref["count"], ref["before_major"])
    close(grad_values, ref["grad_values"], eg, dtype)
    close(grad_gates, ref["grad_gates"], eg * ref["before_major"] + eh * ref["gmajor"] + eg * eh
          + STEP * ref["gmajor"] * ref["before_major"], dtype)
    if grad_initial is not None:
        rows = max(1.0, float(ref["gcount"].max(initial=0)))
        close(grad_initial, ref["grad_initial"], slack(rows, ref["gimajor"]), "f32")
