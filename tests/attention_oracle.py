"""Float64 oracle of block selection, block attention and the distance bias, with
elementwise error bounds counted from the roundings of the device kernels.

Everything is dense over one small cloud: weights are zero where a point's block
is not selected.
"""
from __future__ import annotations

import numpy as np
import torch

BLOCK = 64
FAR = float(np.finfo(np.float32).max)
HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def select(points: np.ndarray, order: np.ndarray, queries: np.ndarray, n: int):
    """(blocks, distances) of one cloud from its leaf order, in float32 by definition."""
    first = np.arange(0, len(order), BLOCK)
    leaves = points[order]
    lo, hi = np.minimum.reduceat(leaves, first, axis=0), np.maximum.reduceat(leaves, first, axis=0)
    score = np.zeros((len(queries), len(first)), np.float32)
    with np.errstate(all="ignore"):
        for a in range(points.shape[1]):
            gap = np.maximum(lo[None, :, a] - queries[:, a, None],
                             np.maximum(queries[:, a, None] - hi[None, :, a], np.float32(0)))
            score = score + gap * gap
    blocks = np.full((len(queries), n), -1, np.int64)
    dist = np.full((len(queries), n), FAR, np.float32)
    for i, row in enumerate(score):
        near = [j for j in np.argsort(row, kind="stable") if row[j] < np.float32(FAR)][:n]
        blocks[i, : len(near)] = near
        dist[i, : len(near)] = row[near]
    return blocks, dist


def buckets(d2: torch.Tensor, edges: torch.Tensor) -> torch.Tensor:
    return (d2[..., None] >= edges).sum(-1)


def pair_distances(query_points: torch.Tensor, points: torch.Tensor) -> torch.Tensor:
    """(M, N) float32, every operation rounded, x first."""
    d = torch.zeros((len(query_points), len(points)), dtype=torch.float32)
    for a in range(points.size(1)):
        gap = query_points[:, a, None] - points[None, :, a]
        d = d + gap * gap
    return d


class Attention:
    """One cloud: outputs, gradients and their bounds."""

    def __init__(self, points, order, query_points, chosen, q, k, v, table=None, edges=None, scale=None, grad=None):
        u = HALF_STEP[q.dtype]
        f = 2.0**-24
        m, h, c = q.shape
        n, kv = k.shape[0], k.shape[1]
        group = torch.arange(h) // (h // kv)
        scale = c**-0.5 if scale is None else scale
        block_of = torch.empty(n, dtype=torch.long)
        block_of[torch.as_tensor(order)] = torch.arange(n) // BLOCK
        hit = torch.zeros((m, (n + BLOCK - 1) // BLOCK + 1), dtype=torch.bool)
        hit.scatter_(1, chosen % hit.shape[1], True)  # -1 goes to the spare last column
        hit[:, -1] = False
        seen = hit[:, block_of]  # (m, n)
        Q, K, V = q.double(), k.double()[:, group], v.double()[:, group]
        # Keys and values that a row does not see do not exist for it.
        logit = scale * torch.einsum("mhc,nhc->hmn", Q, K)
        size = abs(scale) * torch.einsum("mhc,nhc->hmn", Q.abs(), K.abs())
        bucket = None
        if table is not None:
            bucket = buckets(pair_distances(query_points, points), edges)
            logit = logit + table.double()[:, bucket]
            size = size + torch.where(table.isfinite(), table, 0).double().abs()[:, bucket]
        logit = torch.where(seen, logit, -torch.inf)
        top = logit.amax(-1, keepdim=True)
        p = torch.exp(logit - torch.where(top == -torch.inf, 0.0, top))
        total = p.sum(-1, keepdim=True)
        p = torch.where(total > 0, p / total, 0.0)

        def over_keys(w, x):  # sum over n of w[h, m, n] x[n, h, c], unseen rows taken as zeros
            x = torch.where(x.isfinite(), x, 0.0)
            return torch.einsum("hmn,nhc->mhc", w, x)

        self.p, self.out = p, over_keys(p, V)
        # Relative error of a probability: the logit's absolute error (c products summed in
        # float32, 2^-21 for each TF32 triple; scaling and bias; the maximum's difference), twice
        # because the row's sum shares it, and the exponential's and the sum's own roundings.
        seen_size = torch.where(seen, size, 0.0)
        rel = 2 * ((c + 8) * 8 * f * seen_size.amax(-1, keepdim=True)) + (n + 64) * 4 * f
        rel16 = u if q.dtype != torch.float32 else 8 * f  # probability as an operand
        # Exponentials below float32's normal range are flushed to zero: each probability that
        # a row sees may also be off by 2^-126 outright (its sum is at least 1, the largest term's).
        flush = torch.where(seen, 2.0**-126, 0.0).expand_as(p)
        weight = over_keys(p * (rel + rel16) + flush, V.abs())
        self.out_bound = weight + u * self.out.abs() * (1 + u) + 1e-30 + tiny(q.dtype)
        if grad is None:
            return
        dO = grad.double()
        dP = torch.einsum("mhc,nhc->hmn", dO, torch.where(V.isfinite(), V, 0.0))
        dP_size = torch.einsum("mhc,nhc->hmn", dO.abs(), torch.where(V.isfinite(), V, 0.0).abs())
        delta = (dO * self.out).sum(-1).T[..., None]  # (h, m, 1)
        # Delta comes from the output as rounded, whose own error is that of its probabilities and
        # of their rounding as operands; or, where a table trains, from the float32 output, whose
        # probabilities are operands in two 16-bit parts.
        kept = weight if table is None else over_keys(p * (rel + u * u + 8 * f) + flush, V.abs())
        delta_err = ((dO.abs() * (kept + (u if table is None else f) * self.out.abs())).sum(-1)
                     + (c + 8) * 4 * f * (dO.abs() * self.out.abs()).sum(-1)).T[..., None]
        ds = p * (dP - delta)
        ds_err = p * ((c + 8) * 8 * f * dP_size + delta_err) + rel * ds.abs() + flush * (dP_size + delta.abs())
        op = ds_err + rel16 * (ds.abs() + ds_err)  # as an operand of the next product
        sums = (n + m + 64) * 4 * f
        self.dq = scale * over_keys(ds, K)
        self.dq_bound = abs(scale) * over_keys(op + sums * ds.abs(), K.abs()) * (1 + u) + u * self.dq.abs() + tiny(q.dtype)

        def over_queries(w, x):  # to key heads
            full = torch.einsum("hmn,mhc->nhc", w, x)
            return torch.zeros((n, kv, c), dtype=torch.float64).index_add_(1, group, full)

        self.dk = scale * over_queries(ds, Q)
        self.dk_bound = abs(scale) * over_queries(op + sums * ds.abs(), Q.abs()) * (1 + u) + u * self.dk.abs() + tiny(q.dtype)
        self.dv = over_queries(p, dO)
        self.dv_bound = over_queries(p * (rel + rel16 + sums) + flush, dO.abs()) * (1 + u) + u * self.dv.abs() + tiny(q.dtype)
        if table is not None:
            flat = bucket.reshape(-1)
            make = lambda w: torch.zeros((h, table.size(1)), dtype=torch.float64).index_add_(1, flat, w.reshape(h, -1))
            self.dt = make(ds)
            self.dt_bound = make(ds_err + sums * ds.abs()) + 1e-30


def tiny(dtype) -> float:
    """Half the spacing of the type's subnormal numbers."""
    return {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134, torch.float32: 2.0**-149}[dtype]


def within(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, what: str) -> None:
    got = got.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert bool(got.isfinite().all()), f"{what}: not finite"
    off = (got - want).abs()
    worst = (off / bound.clamp(min=1e-300)).max() if off.numel() else torch.tensor(0.0)
    assert bool((off <= bound).all()), f"{what}: {float(worst):.3g} of the bound"
