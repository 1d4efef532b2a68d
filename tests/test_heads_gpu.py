"""qk_norm_rope and qk_norm_rope_quantize against the 64-bit oracle (GPU)."""
import numpy as np
import pytest
import torch

import int8k_capi as capi
from grouped_helpers import HALF, TINY, assert_within, np64, rows
from oracle import grouped_oracle as G

pytestmark = pytest.mark.gpu

P = 600  # rows of the angle tables


def _tables(half):
    f = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
    a = torch.arange(P, dtype=torch.float64)[:, None] * f
    return a.cos().float(), a.sin().float()


def _case(B, S, Hq, Hkv, D, rot, dt, norm, seed=0):
    g = torch.Generator().manual_seed(seed + B + 10 * S + D + rot)
    x = rows(g, B, S, (Hq + 2 * Hkv) * D).to(dt)
    cos, sin = _tables(rot // 2)
    pos = torch.randint(0, P, (B, S), generator=g, dtype=torch.int32)
    w = [torch.rand(D, generator=g) + 0.5 if norm else None for _ in range(2)]
    return x, cos, sin, pos, w[0], w[1]


def _to(gpu, *ts):
    return [t.to(gpu) if t is not None else None for t in ts]


def _oracle(x, Hq, Hkv, cos, sin, pos, wq, wk, inter, eps=1e-6):
    return G.qk_norm_rope(np64(x), Hq, Hkv, cos.numpy(), sin.numpy(), pos.numpy(),
                          None if wq is None else wq.numpy(), None if wk is None else wk.numpy(),
                          eps, inter)


def _bound(ref, D, half, inter, dt, turned):
    if not turned:
        return np.zeros_like(ref)  # values only pass through
    # the mean of D squares, its root, the quotient and the weight: at most (D / 2 + 8) fp32
    # roundings relative to each normed element; the rotation adds 3 of |a| + |b|
    pair = np.abs(ref).copy()
    a = slice(0, 2 * half, 2) if inter else slice(0, half)
    b = slice(1, 2 * half, 2) if inter else slice(half, 2 * half)
    both = np.sqrt(2) * np.hypot(ref[..., a], ref[..., b])  # |a| + |b| before the turn
    pair[..., a] = pair[..., b] = both
    f32 = (D / 2 + 12) * 2.0 ** -24 * pair
    return f32 + HALF[dt] * (np.abs(ref) + f32) + TINY[dt]


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,S,Hq,Hkv,D,rot,inter", [
    (1, 1, 1, 1, 16, 2, False),      # one token, one pair
    (24, 1, 16, 2, 64, 32, True),    # decode, half of the head in interleaved pairs
    (2, 37, 4, 2, 128, 128, False),
    (1, 130, 6, 3, 80, 80, False),   # 5 lane items of 8
    (1, 65, 3, 1, 80, 40, False),    # rot / 2 = 20: no whole chunks
    (1, 33, 2, 2, 96, 6, False),
    (1, 33, 2, 2, 96, 6, True),
    (3, 11, 5, 5, 256, 256, False),
    (1, 19, 8, 1, 256, 64, True),
    (1, 700, 32, 8, 128, 64, False),
])
@pytest.mark.parametrize("norm", [True, False])
def test_heads(ext, gpu, B, S, Hq, Hkv, D, rot, inter, dt, norm):
    x, cos, sin, pos, wq, wk = _case(B, S, Hq, Hkv, D, rot, dt, norm)
    args = _to(gpu, cos, sin, pos)
    gwq, gwk = _to(gpu, wq, wk)
    got = ext.qk_norm_rope(x.to(gpu), Hq, Hkv, *args, q_weight=gwq, k_weight=gwk, interleaved=inter)
    torch.cuda.synchronize()
    ref = _oracle(x, Hq, Hkv, cos, sin, pos, wq, wk, inter)
    for i, n in enumerate((Hq, Hkv, Hkv)):
        assert got[i].shape == (B, n, S, D) and got[i].dtype == dt
        assert_within(np64(got[i]), ref[i], _bound(ref[i], D, rot // 2, inter, dt, i < 2), "qkv"[i])
    # the int8 form is the per-token quantizer of those rows, byte for byte
    q = ext.qk_norm_rope_quantize(x.to(gpu), Hq, Hkv, *args, q_weight=gwq, k_weight=gwk,
                                  interleaved=inter)
    for i in range(3):
        c, s = ext.quantize_per_token(got[i])
        assert torch.equal(q[2 * i], c) and torch.equal(q[2 * i + 1], s), "qkv"[i]


def test_heads_one_norm_and_eps(ext, gpu):
    x, cos, sin, pos, wq, _ = _case(1, 50, 4, 2, 64, 64, torch.float32, True)
    x = x * 1e-3  # eps weighs in
    got = ext.qk_norm_rope(x.to(gpu), 4, 2, *_to(gpu, cos, sin, pos), q_weight=wq.to(gpu), eps=1e-5)
    ref = _oracle(x, 4, 2, cos, sin, pos, wq, None, False, 1e-5)
    for i in range(3):
        assert_within(np64(got[i]), ref[i], _bound(ref[i], 64, 32, False, torch.float32, i < 2))


def test_heads_packed_tokens(ext, gpu):
    # 2-D x: heads [H, T, D], the layout of packed attention
    x, cos, sin, pos, wq, wk = _case(1, 90, 4, 2, 64, 64, torch.float16, True)
    g = _to(gpu, cos, sin, pos)
    a = ext.qk_norm_rope(x.to(gpu), 4, 2, *g, q_weight=wq.to(gpu), k_weight=wk.to(gpu))
    b = ext.qk_norm_rope(x[0].to(gpu), 4, 2, *g, q_weight=wq.to(gpu), k_weight=wk.to(gpu))
    for u, v in zip(a, b):
        assert v.shape == u.shape[1:] and torch.equal(u[0], v)
    q = ext.qk_norm_rope_quantize(x[0].to(gpu), 4, 2, *g)
    assert q[0].shape == (4, 90, 64) and q[1].shape == (4, 90) and q[2].shape == (2, 90, 64)


def test_heads_views_and_unaligned_input(ext, gpu):
    x, cos, sin, pos, wq, wk = _case(1, 20, 4, 2, 64, 64, torch.bfloat16, True)
    g = _to(gpu, cos, sin, pos)
    want = ext.qk_norm_rope(x.to(gpu), 4, 2, *g)
    base = torch.zeros(x.numel() + 1, dtype=x.dtype)
    base[1:] = x.reshape(-1)
    wide = torch.zeros(1, 20, 1024, dtype=x.dtype)
    wide[..., 512:] = x
    for v in (base.to(gpu)[1:].view_as(x), wide.to(gpu)[..., 512:]):
        for a, b in zip(ext.qk_norm_rope(v, 4, 2, *g), want):
            assert torch.equal(a, b)


def test_heads_positions_outside_the_tables_are_counted(ext, gpu):
    x, cos, sin, pos, _, _ = _case(1, 300, 8, 4, 128, 128, torch.float16, False)
    pos[0, 5], pos[0, 77], pos[0, 299] = -1, P, 2 ** 31 - 1
    before = capi.rope_bad_positions()
    got = ext.qk_norm_rope(x.to(gpu), 8, 4, *_to(gpu, cos, sin, pos))
    assert capi.rope_bad_positions() - before == 3
    ref = _oracle(x, 8, 4, cos, sin, pos, None, None, False)
    assert_within(np64(got[0]), ref[0], _bound(ref[0], 128, 64, False, torch.float16, True))


def test_heads_non_finite_rows_stay_their_own(ext, gpu):
    x, cos, sin, pos, wq, wk = _case(1, 64, 4, 2, 64, 64, torch.float32, True)
    x[0, 9, :64] = float("nan")
    x[0, 10, 70] = float("inf")
    got = ext.qk_norm_rope(x.to(gpu), 4, 2, *_to(gpu, cos, sin, pos), q_weight=wq.to(gpu),
                           k_weight=wk.to(gpu))
    q = got[0][0].cpu()
    assert torch.isnan(q[0, 9]).all() and not torch.isfinite(q[1, 10]).all()
    q[0, 9] = 0
    q[1, 10] = 0
    assert torch.isfinite(q).all() and torch.isfinite(got[1]).all()


def test_heads_graph_replay(ext, gpu):
    x, cos, sin, pos, wq, wk = _to(gpu, *_case(4, 1, 8, 2, 128, 128, torch.bfloat16, True))
    run = lambda: ext.qk_norm_rope_quantize(x, 8, 2, cos, sin, pos, q_weight=wq, k_weight=wk)  # noqa: E731
    run()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = run()
    for i in range(3):
        pos.add_(1).remainder_(P)
        x.mul_(-1)
        want = run()
        for t in held:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), i
