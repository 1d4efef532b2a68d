"""64-bit restatements of the operators over the paged INT8 cache with grouped heads (numpy).

Plain formulas: what the kernels of paged.hip and pages.hip, and the cache form of heads.hip, are
checked against.  Pages are int8 [NP, Hkv, P, D] with fp32 scales [NP, Hkv, P]; page ids outside
the cache read the last page.
"""
from __future__ import annotations

import numpy as np

from oracle.grouped_oracle import softmax_attend

F32 = np.float32
F64 = np.float64


def quantize(x):
    """Per-row int8 and fp32 scales of fp32 values, in fp32 arithmetic; a NaN makes the row's
    scale NaN, and NaN quotients clamp to -128."""
    x = x.astype(F32)
    with np.errstate(invalid="ignore", over="ignore"):
        amax = np.abs(x).max(-1)
        s = (np.where(amax < F32(1e-8), F32(1e-8), amax) / F32(127)).astype(F32)
        q = (x / s[..., None]).astype(F32)
        q = np.where(np.isnan(q), F32(-128), np.clip(q, F32(-128), F32(127)))
    return np.rint(q).astype(np.int8), s


def page_ids(row, NP):
    t = np.asarray(row, np.int64)
    return np.where((t < 0) | (t >= NP), NP - 1, t)


def rows_of(pages, scales, ids, head, n):
    """The first n rows of a key head along pages `ids`, as float64 values."""
    D = pages.shape[-1]
    return pages[ids, head].reshape(-1, D)[:n].astype(F64) * scales[ids, head].reshape(-1)[:n, None].astype(F64)


def sees(words, i, j):
    return bool(int(words[i, j // 64]) >> (j % 64) & 1)


def tree_attention(Q, Kp, Vp, sQ, sKp, sVp, tables, lens, mask, counts, max_context):
    """Q int8 [B, H, N, D]; mask int64 [B or 1, N, W] or None (j <= i); counts [B] or None
    -> (out, sum p|v|) float64 [B, H, N, D]."""
    B, H, N, D = Q.shape
    NP, Hkv, P, _ = Kp.shape
    G = H // Hkv
    out, mag = np.zeros((B, H, N, D)), np.zeros((B, H, N, D))
    for b in range(B):
        n = min(max(int(lens[b]), 0), max_context)
        c = N if counts is None else min(max(int(counts[b]), 0), N)
        total = min(n + c, max_context)
        if total == 0:
            continue
        seen = np.zeros((c, total), bool)
        seen[:, :n] = True
        for i in range(c):
            for j in range(total - n):
                seen[i, n + j] = j <= i if mask is None else sees(mask[b if len(mask) > 1 else 0], i, j)
        ids = page_ids(tables[b, :-(-total // P)], NP)
        live = seen.any(1)
        for h in range(Hkv):
            k, v = rows_of(Kp, sKp, ids, h, total), rows_of(Vp, sVp, ids, h, total)
            for j in range(h * G, (h + 1) * G):
                q = Q[b, j, :c].astype(F64) * sQ[b, j, :c, None].astype(F64)
                s = np.where(seen, q @ k.T / np.sqrt(D), -np.inf)
                o, m = softmax_attend(s[live], v)
                out[b, j, :c][live], mag[b, j, :c][live] = o, m
    return out, mag


def page_means(pages, scales):
    """Codes and scales of the mean rows of whole pages [n, H, P, D]."""
    m = (pages.astype(F64) * scales[..., None].astype(F64)).sum(2) / pages.shape[2]
    return quantize(m.astype(F32))


def block_scores(q, sq, means, s_means):
    """q int8 [G, D], sq [G]; means int8 [n, D], s_means [n] -> float64 [n], NaN only where all are."""
    dot = q.astype(F64) @ means.astype(F64).T
    with np.errstate(invalid="ignore"):
        s = dot * s_means.astype(F64)[None] * sq.astype(F64)[:, None]
    s = np.where(np.isnan(s).all(0, keepdims=True), np.nan, s)
    return np.nanmax(np.where(np.isnan(s).all(0), -np.inf, s), 0), np.isnan(s).all(0)


def select_blocks(score, nan, n, top):
    """The last of n blocks and the top - 1 best of the others, ascending; ties to the lowest, NaN
    scores last."""
    if n <= top:
        return list(range(n))
    order = sorted(range(n - 1), key=lambda i: (bool(nan[i]), -score[i], i))
    return sorted(order[:top - 1] + [n - 1])


def sparse_decode(Q, Kp, Vp, sQ, sKp, sVp, Km, sKm, tables, lens, max_context, top):
    """Q int8 [B, H, D] -> (out, sum p|v|, selected int32 [B, Hkv, top])."""
    B, H, D = Q.shape
    NP, Hkv, P, _ = Kp.shape
    G = H // Hkv
    out, mag = np.zeros((B, H, D)), np.zeros((B, H, D))
    which = np.full((B, Hkv, top), -1, np.int32)
    for b in range(B):
        length = min(max(int(lens[b]), 0), max_context)
        n = -(-length // P)
        if n == 0:
            continue
        ids = page_ids(tables[b, :n], NP)
        for h in range(Hkv):
            g = slice(h * G, (h + 1) * G)
            score, nan = block_scores(Q[b, g], sQ[b, g], Km[ids, h], sKm[ids, h])
            taken = select_blocks(score, nan, n, top)
            which[b, h, :len(taken)] = taken
            at = (len(taken) - 1) * P + length - (n - 1) * P
            k, v = rows_of(Kp, sKp, ids[taken], h, at), rows_of(Vp, sVp, ids[taken], h, at)
            q = Q[b, g].astype(F64) * sQ[b, g, None].astype(F64)
            out[b, g], mag[b, g] = softmax_attend(q @ k.T / np.sqrt(D), v)
    return out, mag, which
