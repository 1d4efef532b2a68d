"""64-bit restatements of the grouped-query serving operators (numpy).

Plain formulas, no blocking and no running statistics: what the kernels of linear.hip,
heads.hip, packed.hip and kv4.hip are checked against.  The attention functions also return
sum_j p_j |v_j|, the magnitude that their rounding errors scale with.
"""
from __future__ import annotations

import numpy as np

F32 = np.float32
F64 = np.float64


def linear(x, w, sx, sw, bias=None):
    """x int8 [T, K], w int8 [K, N], sx [T] or [1], sw [N] or [1] -> (y, |x w| sx sw) in float64.
    Integer sums in float64 are exact below 2^53."""
    acc = x.astype(F64) @ w.astype(F64)
    y = acc * np.asarray(sx, F64).reshape(-1, 1) * np.asarray(sw, F64).reshape(1, -1)
    return (y if bias is None else y + np.asarray(bias, F64)), np.abs(y)


def norm_rope(y, cos, sin, weight, eps, interleaved):
    """Rows y [..., D] with the angles cos, sin [..., rot/2] of each row -> float64."""
    y = y.astype(F64).copy()
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * weight.astype(F64)
    half = cos.shape[-1]
    a_at = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    b_at = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = y[..., a_at].copy(), y[..., b_at].copy()
    c, s = cos.astype(F64), sin.astype(F64)
    y[..., a_at], y[..., b_at] = a * c - b * s, b * c + a * s
    return y


def qk_norm_rope(x, heads, kv_heads, cos, sin, positions, wq, wk, eps, interleaved):
    """x [B, S, (heads + 2 kv_heads) D] -> q, k, v float64 [B, H, S, D]."""
    B, S, width = x.shape
    D = width // (heads + 2 * kv_heads)
    x = x.reshape(B, S, heads + 2 * kv_heads, D).transpose(0, 2, 1, 3)
    pos = np.clip(positions.reshape(B, S), 0, cos.shape[0] - 1)
    c, s = cos[pos][:, None], sin[pos][:, None]
    return (norm_rope(x[:, :heads], c, s, wq, eps, interleaved),
            norm_rope(x[:, heads:heads + kv_heads], c, s, wk, eps, interleaved),
            x[:, heads + kv_heads:].astype(F64))


def softmax_attend(s, v):
    """softmax(s) v and softmax(s) |v| of scores [M, N] (float64, -inf masked) and v [N, D]."""
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    return p @ v, p @ np.abs(v)


def packed_attention(Q, K, V, sQ, sK, sV, cu, causal):
    """Q int8 [H, T, D], K, V int8 [Hkv, T, D], scales [H or Hkv, T] -> (out, magnitude)
    float64 [H, T, D]; rows of no sequence are zeros."""
    H, T, D = Q.shape
    G = H // K.shape[0]
    out, mag = np.zeros((H, T, D)), np.zeros((H, T, D))
    for a, b in zip(cu[:-1], cu[1:]):
        if b <= a:
            continue
        for h in range(H):
            q = Q[h, a:b].astype(F64) * sQ[h, a:b, None].astype(F64)
            k = K[h // G, a:b].astype(F64) * sK[h // G, a:b, None].astype(F64)
            v = V[h // G, a:b].astype(F64) * sV[h // G, a:b, None].astype(F64)
            s = q @ k.T / np.sqrt(D)
            if causal:
                s[np.triu_indices(b - a, 1)] = -np.inf
            out[h, a:b], mag[h, a:b] = softmax_attend(s, v)
    return out, mag


def kv4_quantize(x):
    """Rows x [..., D] (fp32 values) -> codes int8 in -8..7 and fp32 scales, in fp32 arithmetic
    as the cache defines them; a NaN makes its row's scale NaN."""
    x = x.astype(F32)
    with np.errstate(invalid="ignore", over="ignore"):
        amax = np.abs(x).max(-1)
        s = (np.where(amax < F32(1e-8), F32(1e-8), amax) * (F32(1) / F32(7))).astype(F32)
        q = (x / s[..., None]).astype(F32)
        q = np.where(np.isnan(q), F32(-8), np.clip(q, F32(-8), F32(7)))
    return np.rint(q).astype(np.int8), s


def kv4_pack(codes):
    u = (codes.astype(np.int16) + 8).astype(np.uint8)
    return u[..., 0::2] | (u[..., 1::2] << 4)


def kv4_unpack(packed):
    return np.stack([packed & 15, packed >> 4], -1).reshape(*packed.shape[:-1], -1).astype(np.int16) - 8


def kv4_decode(Q, Kp, Vp, sQ, sKp, sVp, tables, lens):
    """Q int8 [B, H, D], pages uint8 [NP, Hkv, P, D/2] -> (out, magnitude) float64 [B, H, D].
    Page ids outside the cache read the last page."""
    B, H, D = Q.shape
    NP, Hkv, P, _ = Kp.shape
    out, mag = np.zeros((B, H, D)), np.zeros((B, H, D))
    for b in range(B):
        n = int(lens[b])
        if n <= 0:
            continue
        t = tables[b, :-(-n // P)].astype(np.int64)
        t = np.where((t < 0) | (t >= NP), NP - 1, t)
        for j in range(Hkv):
            k = kv4_unpack(Kp[t, j]).reshape(-1, D)[:n] * sKp[t, j].reshape(-1)[:n, None].astype(F64)
            v = kv4_unpack(Vp[t, j]).reshape(-1, D)[:n] * sVp[t, j].reshape(-1)[:n, None].astype(F64)
            g = slice(j * (H // Hkv), (j + 1) * (H // Hkv))
            q = Q[b, g].astype(F64) * sQ[b, g, None].astype(F64)
            out[b, g], mag[b, g] = softmax_attend(q @ k.T / np.sqrt(D), v)
    return out, mag
