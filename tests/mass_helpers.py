"""Plain fp64 forms of the operators of a bounded cache (attention that accumulates weights, eviction), one sequence at a time, with
the bounds that their errors may reach."""
from __future__ import annotations

import math

import numpy as np
import torch

from helpers import P

HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}      # the most that a rounding is off, relative to the value


def place(t, sink):
    """Logical page and slot of the token in place t."""
    if sink == 0:
        return t // P, t % P
    return (0, t) if t < sink else (1 + (t - sink) // P, (t - sink) % P)


def attend(q, k, v, n_new, window, scale, dtype):
    """q [n_new, G, D], k, v [n, D] of one kv head, the queries being those of the newest tokens.
    Returns o [n_new, G, D], the bound of its error, the weights [n] that the last `window` of them give, and their bound.

    Scores: products of 16-bit values are exact in fp32, 128 of them are added with at most 2^-23 of the sum of their sizes each
    (tensor cores may truncate: twice a rounding's 2^-24).  fp32 inputs: the product's rounding joins.  A weight is 2^(s - lse): its
    relative error is that of the score times 1 / scale in absolute terms, twice (score and denominator), and one rounding per
    addition that its sums see in a row: bf16 n / 16 pages, fp32 the n keys one by one (2^-24 each), the counted rows, the merges of warps
    and pieces.  The output adds the rounding of every weight to the values' type and its own."""
    q, k, v = q.double(), k.double(), v.double()
    n, (w, G, D) = k.shape[0], q.shape
    z = torch.einsum("wgd,td->gwt", q, k) * scale
    size = (torch.einsum("wgd,td->gwt", q.abs(), k.abs()) * scale).max().item() if n else 0.0
    horizon = torch.arange(n - w, n)
    z = z.masked_fill(torch.arange(n) > horizon[:, None], -math.inf)
    p = torch.softmax(z, -1)
    o = torch.einsum("gwt,td->wgd", p, v)
    counted = horizon >= n - (window or w)
    paid = p[:, counted].sum((0, 1))
    rows = int(counted.sum()) * G
    rel = 2.0 ** -23 * (2 * 132 * size + n / (16 if dtype == torch.bfloat16 else 2) + rows + 64)
    o_bound = HALF[dtype] * (o.abs() + torch.einsum("gwt,td->wgd", p, v.abs())) + rel * torch.einsum("gwt,td->wgd", p, v.abs())
    return o, o_bound, paid, rel * paid + 1e-30


def mass_after(mass, b_of_row, n, n_new, h, decay, paid):
    """New masses of one (row, kv head), and what the rounding of the sum may add to the bound."""
    old = mass[b_of_row, h, :n].double() * decay
    old[n - n_new:] = 0
    return old + paid, 2.0 ** -23 * (old.abs() + paid)


def evict_order(mass, position, seen, keep, sink, recent):
    """Which of n tokens stay, as a boolean array: masses fp32, positions."""
    n = len(mass)
    m = np.asarray(mass, dtype=np.float64)
    safe = (position < sink) | (position >= seen - recent)
    low = np.where(np.isnan(m), 1, 0)                                # NaN behind everything
    order = np.lexsort((np.arange(n), np.where(np.isnan(m), 0, -m), low, ~safe))
    stays = np.zeros(n, dtype=bool)
    stays[order[:keep]] = True
    return stays


def evict_moves(stays, keep):
    """(from, to): the i-th kept token behind place `keep` goes to the i-th hole in front of it."""
    n = len(stays)
    front = np.arange(n) < keep
    return np.flatnonzero(stays & ~front), np.flatnonzero(~stays & front)
