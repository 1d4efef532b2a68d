"""The writer and the upkeep of the paged INT8 cache (GPU): rows appended with the rotation, moved
rows and page means, against the framework's row quantizer and the oracle, bit for bit."""
from fractions import Fraction

import numpy as np
import pytest
import torch

import int8k_capi as capi
from grouped_helpers import quantize_rows, rows
from oracle import paged_oracle as P

pytestmark = pytest.mark.gpu


def _cache(NP, H, page, D, gpu):
    return (torch.full((NP, H, page, D), 77, dtype=torch.int8, device=gpu),
            torch.full((NP, H, page, D), -77, dtype=torch.int8, device=gpu),
            torch.full((NP, H, page), 5.0, device=gpu), torch.full((NP, H, page), 6.0, device=gpu))


# ------------------------------------------------------------------ append


def _append_case(seed, B, S, H, Hkv, D, rot, dt, gpu, flat=False):
    g = torch.Generator().manual_seed(seed)
    x = rows(g, B, S, (H + 2 * Hkv) * D).to(dt).to(gpu)
    a = torch.rand(500, rot // 2, generator=g) * 6.28
    pos = torch.randint(0, 500, (B, S), generator=g, dtype=torch.int32)
    return (x.view(B * S, -1) if flat else x), a.cos().to(gpu), a.sin().to(gpu), pos.to(gpu)


def _append_and_check(ext, gpu, case, H, Hkv, D, page, slots, NP, **kw):
    """The queries and every byte of the cache, against qk_norm_rope_quantize."""
    x, cos, sin, pos = case
    K, V, sK, sV = _cache(NP, Hkv, page, D, gpu)
    sl = torch.tensor(slots, dtype=torch.int32, device=gpu)
    q, sq = ext.qk_norm_rope_append(x, H, Hkv, cos, sin, pos, K, V, sK, sV, sl, **kw)
    ref = [t.cpu() for t in ext.qk_norm_rope_quantize(x, H, Hkv, cos, sin, pos, **kw)]
    assert torch.equal(q.cpu(), ref[0]) and torch.equal(sq.cpu(), ref[1])
    want = [t.cpu() for t in _cache(NP, Hkv, page, D, gpu)]
    if x.dim() == 2:
        ref = [t.unsqueeze(0) for t in ref]
    B, _, S = ref[3].shape
    for t, slot in enumerate(slots):
        if 0 <= slot < NP * page:
            at = (slot // page, slice(None), slot % page)
            for i, (codes, scales) in enumerate(((ref[2], ref[3]), (ref[4], ref[5]))):
                want[i][at] = codes[t // S, :, t % S]
                want[2 + i][at] = scales[t // S, :, t % S]
    for got, w in zip((K, V, sK, sV), want):
        assert torch.equal(got.cpu(), w)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,S,H,Hkv,D,rot,page,interleaved", [
    (1, 1, 1, 1, 64, 64, 16, False), (5, 1, 8, 2, 128, 128, 64, False), (3, 7, 4, 4, 64, 32, 16, True),
    (1, 333, 6, 2, 128, 64, 256, False), (2, 50, 4, 1, 64, 40, 16, False), (1, 1000, 12, 12, 64, 64, 1024, True),
    (48, 1, 32, 8, 128, 128, 64, False)])
def test_append(ext, gpu, B, S, H, Hkv, D, rot, page, interleaved, dt):
    g = torch.Generator().manual_seed(B + S)
    NP = -(-B * S // page) + 2
    slots = torch.randperm(NP * page, generator=g)[:B * S].tolist()
    w = dict(q_weight=(1 + 0.1 * torch.randn(D, generator=g)).to(gpu), k_weight=(1 + 0.1 * torch.randn(D, generator=g)).to(gpu))
    for kw in (dict(interleaved=interleaved), dict(w, interleaved=interleaved, eps=1e-5)):
        _append_and_check(ext, gpu, _append_case(B + D, B, S, H, Hkv, D, rot, dt, gpu), H, Hkv, D, page, slots, NP, **kw)


def test_append_of_flat_tokens_and_strided_projections(ext, gpu):
    x, cos, sin, pos = _append_case(1, 1, 20, 4, 2, 64, 64, torch.float16, gpu, flat=True)
    slots = list(range(40, 20, -1))
    _append_and_check(ext, gpu, (x, cos, sin, pos), 4, 2, 64, 16, slots, 3)
    wide = torch.cat((x, x), 1)[:, :x.shape[1]]
    odd = torch.cat((torch.zeros(3, dtype=x.dtype, device=gpu), x.reshape(-1)))[3:].view(x.shape)
    for y in (wide, odd):
        _append_and_check(ext, gpu, (y, cos.t().contiguous().t(), sin, pos), 4, 2, 64, 16, slots, 3)


def test_append_skips_padding_and_counts_slots_past_the_cache(ext, gpu):
    before = capi.paged_bad_ids()
    _append_and_check(ext, gpu, _append_case(2, 6, 1, 2, 1, 64, 64, torch.bfloat16, gpu), 2, 1, 64, 16,
                      [-1, 47, 48, 0, -2 ** 31, 2 ** 31 - 1], 3)
    assert capi.paged_bad_ids() - before == 2


def test_append_extreme_rows(ext, gpu):
    case = _append_case(3, 1, 8, 1, 1, 64, 64, torch.float32, gpu)
    x = case[0]
    x[0, 1] = 0
    x[0, 2] = 1e-30
    x[0, 3, 130] = 3e38  # a value
    x[0, 4, 70] = float("inf")  # a key
    x[0, 5, 140] = float("-inf")
    _append_and_check(ext, gpu, case, 1, 1, 64, 16, list(range(8)), 1)


def test_append_past_32_bit_offsets(ext, gpu):
    page, Hkv, D = 1024, 8, 128
    NP = (1 << 32) // (Hkv * page * D) + 2
    x, cos, sin, pos = _append_case(4, 1, 5, 8, Hkv, D, 128, torch.bfloat16, gpu)
    K = torch.zeros(NP, Hkv, page, D, dtype=torch.int8, device=gpu)
    V = torch.zeros_like(K)
    sK, sV = torch.zeros(NP, Hkv, page, device=gpu), torch.zeros(NP, Hkv, page, device=gpu)
    slots = torch.arange(NP * page - 5, NP * page, dtype=torch.int32, device=gpu)
    ext.qk_norm_rope_append(x, 8, Hkv, cos, sin, pos, K, V, sK, sV, slots)
    ref = ext.qk_norm_rope_quantize(x, 8, Hkv, cos, sin, pos)
    assert torch.equal(K[-1, :, -5:], ref[2][0]) and torch.equal(V[-1, :, -5:], ref[4][0])
    assert torch.equal(sK[-1, :, -5:], ref[3][0]) and torch.equal(sV[-1, :, -5:], ref[5][0])
    # and moved to the front from there
    ext.kv_cache_move_paged(K, V, sK, sV, slots, torch.arange(5, dtype=torch.int32, device=gpu))
    assert torch.equal(K[0, :, :5], ref[2][0]) and torch.equal(sV[0, :, :5], ref[5][0])
    m, sm = torch.zeros(NP, Hkv, D, dtype=torch.int8, device=gpu), torch.zeros(NP, Hkv, device=gpu)
    ext.kv_page_means(K, sK, torch.tensor([NP - 1], dtype=torch.int32, device=gpu), m, sm)
    want = P.page_means(K[-1:].cpu().numpy(), sK[-1:].cpu().numpy())
    np.testing.assert_array_equal(m[-1:].cpu().numpy(), want[0])
    np.testing.assert_array_equal(sm[-1:].cpu().numpy(), want[1])


# ------------------------------------------------------------------ move


def _filled(seed, NP, H, page, D, gpu):
    g = torch.Generator().manual_seed(seed)
    c = [torch.randint(-128, 128, (NP, H, page, D), generator=g, dtype=torch.int8) for _ in range(2)]
    return [t.to(gpu) for t in c + [torch.rand(NP, H, page, generator=g), torch.rand(NP, H, page, generator=g)]]


def _move_and_check(ext, gpu, cache, src, dst):
    page, cap = cache[0].shape[2], cache[0].shape[0] * cache[0].shape[2]
    want = [t.cpu().clone() for t in cache]
    for s_list, d_list in zip(src, dst) if isinstance(src[0], list) else [(src, dst)]:
        old = [t.clone() for t in want]
        for s, d in zip(s_list, d_list):
            if 0 <= s < cap and 0 <= d < cap:
                for t, o in zip(want, old):
                    t[d // page, :, d % page] = o[s // page, :, s % page]
    i32 = dict(dtype=torch.int32, device=gpu)
    ext.kv_cache_move_paged(*cache, torch.tensor(src, **i32), torch.tensor(dst, **i32))
    for t, w in zip(cache, want):
        assert torch.equal(t.cpu(), w)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,page", [(1, 16), (8, 64), (3, 1024)])
@pytest.mark.parametrize("pairs", [1, 5, 33, 64, 65, 200, 256])
def test_move_within_a_list(ext, gpu, pairs, H, page, D):
    # a random map of a list's rows onto distinct ones, sources among the destinations
    g = torch.Generator().manual_seed(pairs + D)
    NP = -(-2 * pairs // page) + 1
    slots = torch.randperm(NP * page, generator=g)[:pairs + pairs // 2].tolist()
    src = [slots[int(i)] for i in torch.randint(0, len(slots), (pairs,), generator=g)]  # also twice
    _move_and_check(ext, gpu, _filled(pairs, NP, H, page, D, gpu), src, slots[-pairs:])


def test_move_of_accepted_paths(ext, gpu):
    # path nodes to the front, in place, a cycle, one row onto itself
    cache = _filled(1, 8, 4, 16, 64, gpu)
    src = [[0, 2, 3, 7, 12], [40, 41, 42, 43, 44], [64, 65, 66, 67, 68]]
    dst = [[0, 1, 2, 3, 4], [41, 42, 43, 44, 40], [64, 65, 66, 67, 68]]
    _move_and_check(ext, gpu, cache, src, dst)


def test_move_leaves_out_padding_and_counts_slots_past_the_cache(ext, gpu):
    cache = _filled(2, 3, 2, 16, 128, gpu)
    before = capi.paged_bad_ids()
    _move_and_check(ext, gpu, cache, [[-1, 5, 48, 7, 2 ** 31 - 1], [20, 21, -2 ** 31, 30, 31]],
                    [[0, -1, 1, 48, 3], [21, 20, 5, 33, 46]])
    assert capi.paged_bad_ids() - before == 3


# ------------------------------------------------------------------ means


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,page,n", [(1, 16, 1), (3, 32, 7), (8, 64, 40), (2, 256, 5), (1, 1024, 3)])
def test_means(ext, gpu, H, page, n, D):
    g = torch.Generator().manual_seed(n + D)
    k, sk = quantize_rows(rows(g, n + 2, H, page, D) + torch.randn(n + 2, H, 1, D, generator=g))
    m = torch.full((n + 2, H, D), 9, dtype=torch.int8, device=gpu)
    sm = torch.full((n + 2, H), 3.0, device=gpu)
    ids = torch.randperm(n + 2, generator=g)[:n]
    ext.kv_page_means(k.to(gpu), sk.to(gpu), ids.to(torch.int32).to(gpu), m, sm)
    want = P.page_means(k.numpy(), sk.numpy())
    left = [i for i in range(n + 2) if i not in ids.tolist()]
    want[0][left], want[1][left] = 9, 3.0
    np.testing.assert_array_equal(m.cpu().numpy(), want[0])
    np.testing.assert_array_equal(sm.cpu().numpy(), want[1])


def test_means_of_extreme_pages_and_ids(ext, gpu):
    k = torch.randint(-128, 128, (7, 1, 16, 64), generator=torch.Generator().manual_seed(1), dtype=torch.int8)
    sk = torch.full((7, 1, 16), 0.5)
    k[0] = 0                                     # the smallest scale
    k[1], sk[1] = -128, 3e36                     # near fp32's end
    sk[2, 0, :8], sk[2, 0, 8:] = 1e30, 1e-3      # rows of very different sizes that cancel
    k[2, 0, 4:8] = -k[2, 0, :4].clamp(min=-127)
    k[2, 0, :4] = k[2, 0, :4].clamp(min=-127)
    sk[3, 0, 5] = float("nan")
    sk[4] = 1e-30
    m, sm = torch.zeros(7, 1, 64, dtype=torch.int8, device=gpu), torch.full((7, 1), 2.0, device=gpu)
    before = capi.paged_bad_ids()
    ids = torch.tensor([0, 1, -1, 2, 3, 4, 7, 4, -2 ** 31, 2 ** 31 - 1], dtype=torch.int32, device=gpu)
    ext.kv_page_means(k.to(gpu), sk.to(gpu), ids, m, sm)
    assert capi.paged_bad_ids() - before == 2
    want = P.page_means(k.numpy(), sk.numpy())
    assert torch.isnan(sm[3, 0])
    for i in (0, 1, 4):
        np.testing.assert_array_equal(m[i].cpu().numpy(), want[0][i])
        np.testing.assert_array_equal(sm[i].cpu().numpy(), want[1][i])
    # page 2: what the large rows leave depends on the order of the sum.  Each of its 15 additions is
    # off by at most 2^-53 of a partial sum, which is at most sum |x|, so the mean by 2^-53 sum |x|;
    # the code by half a step.  (127e30 * 8 * 2^-53 is far above the small rows: any order is right.)
    x = np.abs(k[2, 0].numpy().astype(np.float64) * sk[2, 0].numpy()[:, None].astype(np.float64)).sum(0)
    exact = np.array([sum(int(k[2, 0, r, d]) * Fraction(float(sk[2, 0, r])) for r in range(16)) / 16 for d in range(64)], dtype=np.float64)
    got = m[2, 0].cpu().numpy().astype(np.float64) * float(sm[2, 0])
    assert (np.abs(got - exact) <= 2.0 ** -53 * x + 0.5001 * float(sm[2, 0])).all()
    assert (m[5:] == 0).all() and (sm[5:] == 2.0).all()
