"""Plain 64-bit forms of the paged 8-bit key/value cache ops (KvAppend, KvRead, KvAttention, KvScore,
KvEvict; formulas in include/bolt_b200.h), sequence by sequence and head by head.

TEST INFRASTRUCTURE ONLY, as the rest of this package.
"""
from __future__ import annotations

import numpy as np
import torch

KV_QMAX = {0: 127.0, 1: 448.0}


def kv_values(codes: torch.Tensor, fmt: int) -> np.ndarray:
    """fp64 values (in units of the scale) of u8 codes."""
    if fmt == 0:
        return codes.numpy().astype(np.float64) - 128
    return codes.view(torch.float8_e4m3fn).double().numpy()


def kv_tokens(cache, scale, table, s, idx, fmt) -> np.ndarray:
    """fp64 values [len(idx), heads, D] of sequence s's positions."""
    T = cache.shape[2]
    page = table[s].long()[torch.as_tensor(idx, dtype=torch.long) // T]
    slot = torch.as_tensor(idx, dtype=torch.long) % T
    return kv_values(cache[page, :, slot], fmt) * scale[page].double().numpy()[..., None]


def kv_visible(pos: int, n: int, window: int, sinks: int) -> np.ndarray:
    j = np.arange(n)
    see = j <= pos
    if window:
        see &= (j > pos - window) | (j < sinks)
    return see


def kv_attention(q, k_cache, v_cache, k_scale, v_scale, table, start, lens, scale, window=0, sinks=0, fmt=0):
    """Returns dict of fp64 arrays: o, lse, and for bounds: av = sum_j p_j |v_j| and ql, the largest
    sum_d |q_d k_jd| * scale of each row."""
    S, R, Hq, D = q.shape
    H = k_cache.shape[1]
    G = Hq // H
    o, av = np.zeros((S, R, Hq, D)), np.zeros((S, R, Hq, D))
    lse, ql = np.full((S, R, Hq), -np.inf), np.zeros((S, R, Hq))
    qd = q.double().numpy()
    for s in range(S):
        n = int(lens[s])
        if n == 0:
            continue
        k = kv_tokens(k_cache, k_scale, table, s, np.arange(n), fmt)
        v = kv_tokens(v_cache, v_scale, table, s, np.arange(n), fmt)
        for r in range(R):
            pos = int(start[s]) + r
            if pos >= n:
                continue
            see = kv_visible(pos, n, window, sinks)
            for i in range(Hq):
                kk, vv = k[see, i // G], v[see, i // G]
                x = kk @ qd[s, r, i] * scale
                m = x.max()
                e = np.exp(x - m)
                lse[s, r, i] = m + np.log(e.sum())
                p = e / e.sum()
                o[s, r, i] = p @ vv
                av[s, r, i] = p @ np.abs(vv)
                ql[s, r, i] = (np.abs(kk) @ np.abs(qd[s, r, i]) * abs(scale)).max()
    return dict(o=o, lse=lse, av=av, ql=ql)


def kv_score(q, k_cache, k_scale, table, start, lens, lse, score, scale, window=0, sinks=0, fmt=0):
    """Returns (score, added) fp64 [S, heads, width]; lse as given."""
    S, R, Hq, D = q.shape
    H = k_cache.shape[1]
    G = Hq // H
    added = np.zeros(score.shape)
    for s in range(S):
        n = int(lens[s])
        if n == 0:
            continue
        k = kv_tokens(k_cache, k_scale, table, s, np.arange(n), fmt)
        for r in range(R):
            pos = int(start[s]) + r
            if pos >= n:
                continue
            see = kv_visible(pos, n, window, sinks)
            for i in range(Hq):
                x = k[:, i // G] @ q[s, r, i].double().numpy() * scale
                added[s, i // G, :n] += np.where(see, np.exp(x - float(lse[s, r, i])), 0.0)
    return score.double().numpy() + added, added


def kv_evict_keep(score, n, keep, sinks, recent) -> np.ndarray:
    """Kept positions of one (sequence, head) of n positions, ascending."""
    if n <= keep:
        return np.arange(n)
    x = np.asarray(score[:n], dtype=np.float64)
    rank = np.where(np.isnan(x), np.inf, x)
    nan = np.isnan(x)
    mid = sorted(range(sinks, n - recent), key=lambda j: (not nan[j], -rank[j], j))[:keep - sinks - recent]
    return np.array(sorted(list(range(sinks)) + mid + list(range(n - recent, n))), dtype=np.int64)
