"""Float64 attention of a drafted tree over a cache: what attend_tree's tests compare with.

A node's positions are gathered one node at a time, so that what it does not see takes no part.  With the
output come the bounds' ingredients: `weight` = sum of softmax weights times |V| (what relative errors of
weights scale by) and `score` = the largest sum |scale q_d k_d| of a visible position (what rounding of a
score's sum scales by).
"""

from __future__ import annotations

import torch


def tree_reference(q, k, v, lens, nk, nv, mask, scale):
    """q [B, Hq, T, D]; k, v [B, H, S, D] cached (S >= max lens); nk, nv [B, H, T, D]; mask bool [T, T] or
    [B, T, T] or None (chain).  Returns float64 out [B, Hq, T, D], weight of the same shape, score [B, Hq, T, 1]."""
    q, k, v, nk, nv = (t.detach().double().cpu() for t in (q, k, v, nk, nv))
    B, Hq, T, D = q.shape
    G = Hq // nk.shape[1]
    mask = torch.ones((T, T), dtype=torch.bool).tril() if mask is None else mask.cpu()
    mask = mask.expand(B, T, T)
    out, weight = torch.zeros_like(q), torch.zeros_like(q)
    score = torch.zeros((B, Hq, T, 1), dtype=torch.float64)
    for b in range(B):
        n = int(lens[b])
        keys = torch.cat([k[b, :, :n], nk[b]], dim=1)
        values = torch.cat([v[b, :, :n], nv[b]], dim=1)
        for i in range(T):
            seen = torch.cat([torch.arange(n), n + torch.nonzero(mask[b, i])[:, 0]])
            if not len(seen):
                continue
            for h in range(nk.shape[1]):
                rows = slice(h * G, (h + 1) * G)
                kk, vv, qq = keys[h, seen], values[h, seen], q[b, rows, i]
                p = torch.softmax(qq @ kk.t() * scale, dim=-1)
                out[b, rows, i] = p @ vv
                weight[b, rows, i] = p @ vv.abs()
                score[b, rows, i, 0] = (qq.abs() @ kk.abs().t()).amax(-1) * scale
    return out, weight, score


def tree_bound(out, weight, score, dtype, positions: int, dim: int, pool_dtype=None):
    """How far a kernel with 32-bit sums may be from `out`.  A score's sum of `dim` products rounds by at most
    dim * 2^-24 of the sum of magnitudes, its scaling and the exponent's by a few 2^-24 more of it; a weight's relative
    error is that of its exponent, the weights' sum has it too (twice).  A weight is handed to the second product as two
    16-bit numbers (bf16: half a step each, 2^-18 of it; fp16 loses at most 2^-25 of the largest).  The sums over
    `positions` run in chunks of 16 (positions / 16 + 16 roundings of 2^-24 each, twice for the weights' sum).
    The output is rounded to `dtype` by half a step."""
    half = torch.finfo(dtype).eps / 2
    relative = 2 * (dim + 8) * 2.0**-24 * (score + 1) + 2.0**-18 + positions * 2.0**-25 + 2 * (positions / 16 + 16) * 2.0**-24
    tiny = torch.finfo(dtype).smallest_normal * half * 2  # a subnormal output's half step
    return half * out.abs() * (1 + relative) + weight * relative + tiny
