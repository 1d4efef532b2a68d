"""The paged 4-bit KV cache (GPU): append and read bit for bit, decode attention against the
64-bit oracle."""
import numpy as np
import pytest
import torch

import int8k_capi as capi
from grouped_helpers import assert_within, attention_bound, kv4_case, np64, quantize_rows, rows
from oracle import grouped_oracle as G

pytestmark = pytest.mark.gpu


def _empty(NP, H, page, D, gpu):
    return (torch.full((NP, H, page, D // 2), 0xAB, dtype=torch.uint8, device=gpu),
            torch.full((NP, H, page), 5.0, device=gpu))


def _append_and_check(ext, gpu, k, v, D, H, page, slots, NP, view=lambda t: t):
    K, sK = _empty(NP, H, page, D, gpu)
    V, sV = _empty(NP, H, page, D, gpu)
    ext.kv4_cache_append(view(k.to(gpu)), view(v.to(gpu)), K, V, sK, sV,
                         torch.tensor(slots, dtype=torch.int32, device=gpu))
    torch.cuda.synchronize()
    for x, pages, scales in ((k, K, sK), (v, V, sV)):
        c, s = G.kv4_quantize(x.float().numpy())
        want_p = np.full((NP, H, page, D // 2), 0xAB, np.uint8)
        want_s = np.full((NP, H, page), 5.0, np.float32)
        for t, slot in enumerate(slots):
            if 0 <= slot < NP * page:
                want_p[slot // page, :, slot % page] = G.kv4_pack(c[t])
                want_s[slot // page, :, slot % page] = s[t]
        np.testing.assert_array_equal(pages.cpu().numpy(), want_p)
        np.testing.assert_array_equal(scales.cpu().numpy(), want_s)
    return K, V, sK, sV


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,H,page", [(1, 1, 16), (7, 3, 16), (48, 8, 64), (333, 2, 256), (1000, 5, 1024)])
def test_append_and_read(ext, gpu, T, H, page, D, dt):
    g = torch.Generator().manual_seed(T + H + D)
    k, v = rows(g, T, H, D).to(dt), rows(g, T, H, D).to(dt)
    NP = -(-T // page) + 2
    slots = torch.randperm(NP * page, generator=g)[:T].tolist()
    K, _, sK, _ = _append_and_check(ext, gpu, k, v, D, H, page, slots, NP)
    c, s = G.kv4_quantize(k.float().numpy())
    sl = torch.tensor(slots, dtype=torch.int32, device=gpu)
    for out_t in (torch.float16, torch.bfloat16, torch.float32):
        got = ext.kv4_cache_read(K, sK, sl, dtype=out_t).cpu()
        want = (torch.from_numpy(c).float() * torch.from_numpy(s).unsqueeze(-1)).to(out_t)
        assert torch.equal(got, want)


def test_append_skips_padding_and_counts_slots_past_the_cache(ext, gpu):
    g = torch.Generator().manual_seed(3)
    k, v = rows(g, 6, 2, 64), rows(g, 6, 2, 64)
    before = capi.kv4_bad_ids()
    _append_and_check(ext, gpu, k, v, 64, 2, 16, [-1, 47, 48, 0, -2 ** 31, 2 ** 31 - 1], 3)
    assert capi.kv4_bad_ids() - before == 2


def test_append_strided_rows(ext, gpu):
    # heads [H, T, D] of qk_norm_rope as [T, H, D]; a slice of a wider projection; odd offsets
    g = torch.Generator().manual_seed(4)
    k, v = rows(g, 20, 4, 64).half(), rows(g, 20, 4, 64).half()
    slots = list(range(5, 25))
    for view in (lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),
                 lambda t: torch.cat((t, t), 1)[:, 2:6].roll(2, 1).contiguous(),
                 lambda t: torch.cat((torch.zeros(3, dtype=t.dtype, device=t.device), t.reshape(-1)))[3:].view(t.shape),
                 lambda t: t.transpose(1, 2).contiguous().transpose(1, 2),
                 lambda t: torch.nn.functional.pad(t, (0, 5))[..., :64]):
        _append_and_check(ext, gpu, k, v, 64, 4, 16, slots, 2, view)


def test_append_extreme_rows(ext, gpu):
    k = torch.zeros(8, 1, 64)
    k[1] = 1e-12
    k[2, 0, 3] = 3.4e38
    k[3, 0, 5] = float("nan")
    k[4, 0, 6] = float("inf")
    k[5] = torch.linspace(-1, 1, 64)
    k[6] = 1e-38
    k[7, 0, :2] = torch.tensor([7.0, 3.5])  # a tie: 3.5 rounds to 4
    _append_and_check(ext, gpu, k, k.flip(0), 64, 1, 16, list(range(8)), 1)


def test_read_outside_the_cache_is_zero(ext, gpu):
    K, sK = _empty(2, 3, 16, 64, gpu)
    got = ext.kv4_cache_read(K, sK, torch.tensor([-1, 31, 32], dtype=torch.int32, device=gpu))
    assert (got[0] == 0).all() and (got[2] == 0).all() and (got[1] != 0).any()


# ------------------------------------------------------------------ decode


def _decode(ext, c):
    return ext.int8_decode_attention_forward_kv4_paged(
        c["Q"], c["K"], c["V"], c["sQ"], c["sK"], c["sV"], c["tables"], c["lens"], c["max_context"])


def _check(c, out, label=""):
    ref, mag = G.kv4_decode(*(c[k].cpu().numpy() for k in ("Q", "K", "V", "sQ", "sK", "sV", "tables", "lens")))
    vmax = float(7 * c["sV"][torch.isfinite(c["sV"])].max())
    assert_within(np64(out), ref, attention_bound(ref, mag, c["max_context"], vmax), label)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (4, 4), (8, 2), (6, 2), (16, 1), (32, 1), (20, 1), (32, 8)])
@pytest.mark.parametrize("page", [16, 64, 1024])
def test_decode(ext, gpu, H, Hkv, D, page):
    lens = [1, page - 1, page + 1, 0, 200, 777, 1024]
    c = kv4_case(H + Hkv + D + page, len(lens), H, Hkv, D, page, lens, gpu)
    out = _decode(ext, c)
    assert out.shape == c["Q"].shape and out.dtype == torch.float16
    assert (out[3] == 0).all()
    _check(c, out, f"H{H}/{Hkv} D{D} page{page}")


@pytest.mark.parametrize("B,H,Hkv,D,L", [(1, 8, 1, 128, 20001), (2, 4, 4, 64, 9000), (1, 2, 1, 64, 70000),
                                         (40, 4, 2, 128, 300), (3, 48, 2, 64, 5000)])
def test_decode_long_and_wide(ext, gpu, B, H, Hkv, D, L):
    lens = [max(1, L - 37 * b) for b in range(B)]
    c = kv4_case(L + B, B, H, Hkv, D, 32, lens, gpu)
    _check(c, _decode(ext, c))


def test_decode_max_context_beyond_the_lengths(ext, gpu):
    # the plan follows max_context, the work the lengths; a length past max_context is cut
    c = kv4_case(9, 3, 8, 2, 128, 64, [5, 300, 0], gpu)
    want = _decode(ext, c)
    wide = torch.full((3, 1000), -1, dtype=torch.int32, device=gpu)
    wide[:, :c["tables"].shape[1]] = c["tables"]
    c["tables"], c["max_context"] = wide, 64000
    _check(c, _decode(ext, c))
    c["max_context"] = 200
    c["lens"].copy_(torch.tensor([5, 200, 0]))
    cut = _decode(ext, c)
    c["lens"].copy_(torch.tensor([5, 300, -4]))
    assert torch.equal(_decode(ext, c), cut)
    assert torch.isfinite(want).all()


def test_decode_bad_page_ids_read_the_last_page_and_are_counted(ext, gpu):
    c = kv4_case(5, 2, 4, 2, 64, 16, [100, 50], gpu)
    before = capi.kv4_bad_ids()
    _check(c, _decode(ext, c))  # -1 padding behind the lengths is never read
    assert capi.kv4_bad_ids() == before
    c["tables"][0, 2], c["tables"][1, 0] = -5, 10 ** 6
    _check(c, _decode(ext, c))
    assert capi.kv4_bad_ids() > before


def test_decode_non_finite_scales_behind_the_length(ext, gpu):
    c = kv4_case(6, 2, 8, 2, 128, 64, [70, 33], gpu)
    want = _decode(ext, c)
    for b, n in enumerate((70, 33)):
        for j in range(-(-n // 64)):
            p = int(c["tables"][b, j])
            first = max(0, n - 64 * j)
            if first < 64:
                c["sK"][p, :, first:] = float("nan")
                c["sV"][p, :, first:] = float("inf")
                c["K"][p, :, first:] = 0
                c["V"][p, :, first:] = 255
    assert torch.equal(_decode(ext, c), want)


def test_decode_nan_row_poisons_its_head_only(ext, gpu):
    c = kv4_case(7, 2, 8, 2, 64, 16, [100, 50], gpu)
    c["sK"][int(c["tables"][0, 1]), 1, 3] = float("nan")
    out = _decode(ext, c)
    assert torch.isnan(out[0, 4:]).all()
    assert torch.isfinite(out[0, :4]).all() and torch.isfinite(out[1]).all()


@pytest.mark.parametrize("spread", [1e-6, 1e4])
def test_decode_value_scales_of_very_different_sizes(ext, gpu, spread):
    # fp16 weights times the value scales must not leave fp16's range
    c = kv4_case(8, 2, 8, 2, 128, 32, [500, 900], gpu)
    g = torch.Generator().manual_seed(1)
    c["sV"].mul_((torch.rand(c["sV"].shape, generator=g) ** 4).to(gpu) * spread)
    out = _decode(ext, c).float()
    ref, mag = G.kv4_decode(*(c[k].cpu().numpy() for k in ("Q", "K", "V", "sQ", "sK", "sV", "tables", "lens")))
    # the rounding of the output to fp16 aside, errors scale with sum p |v|; weights that fall
    # 2^-14 below the largest p sV are off by half a subnormal step of it
    biggest = float(7 * c["sV"].max())
    assert_within(np64(out), ref, (3 * 2.0 ** -11 + 2.0 ** -14) * mag + 2.0 ** -11 * np.abs(ref)
                  + 900 * 2.0 ** -24 * biggest + 2.0 ** -25)


def test_decode_large_scores(ext, gpu):
    # one key far above the rest, at the end, at the start, and rising scores
    c = kv4_case(10, 3, 4, 1, 64, 16, [400, 400, 400], gpu)
    pages = c["tables"].cpu()
    for b, at in ((0, 399), (1, 0)):
        c["sK"][int(pages[b, at // 16]), :, at % 16] *= 300
    for j in range(25):
        c["sK"][int(pages[2, j])] *= 1 + j
    _check_large(c, _decode(ext, c))


def _check_large(c, out):
    ref, mag = G.kv4_decode(*(c[k].cpu().numpy() for k in ("Q", "K", "V", "sQ", "sK", "sV", "tables", "lens")))
    # scores of up to 2^12 (3 fp32 roundings each) move a weight by 2^12 * 3 * 2^-24 < 2^-10
    assert_within(np64(out), ref, attention_bound(ref, mag, 400, float(7 * c["sV"].max())) + 2.0 ** -10 * mag)


def test_decode_of_appended_tokens_matches_the_oracle(ext, gpu):
    # tokens appended one step at a time, decoded after each
    g = torch.Generator().manual_seed(11)
    B, H, Hkv, D, page = 3, 8, 2, 128, 16
    NP = 12
    K, sK = torch.zeros(NP, Hkv, page, D // 2, dtype=torch.uint8, device=gpu), torch.zeros(NP, Hkv, page, device=gpu)
    V, sV = torch.zeros_like(K), torch.zeros_like(sK)
    tables = torch.randperm(NP, generator=g).to(torch.int32).view(B, 4).to(gpu)
    for step in range(35):
        k, v = rows(g, B, Hkv, D).to(torch.bfloat16).to(gpu), rows(g, B, Hkv, D).to(torch.bfloat16).to(gpu)
        slots = (tables[:, step // page] * page + step % page).to(torch.int32)
        ext.kv4_cache_append(k, v, K, V, sK, sV, slots)
        if step % 11 == 0 or step == 34:
            q, sq = quantize_rows(torch.randn(B, H, D, generator=g))
            c = dict(Q=q.to(gpu), sQ=sq.to(gpu), K=K, V=V, sK=sK, sV=sV, tables=tables,
                     lens=torch.full((B,), step + 1, dtype=torch.int32, device=gpu), max_context=step + 1)
            _check(c, _decode(ext, c), f"step {step}")


def test_decode_graph_replay_and_streams(ext, gpu):
    c = kv4_case(12, 4, 8, 2, 128, 32, [900, 5, 333, 1000], gpu)
    want = _decode(ext, c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _decode(ext, c)
    side.synchronize()
    assert torch.equal(got, want)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        y1 = _decode(ext, c)
    with torch.cuda.graph(g2):
        y2 = _decode(ext, c)
    for lens in ([900, 5, 333, 1000], [1, 0, 64, 999], [33, 31, 1000, 2]):
        c["lens"].copy_(torch.tensor(lens))
        eager = _decode(ext, c)
        y1.fill_(3)
        y2.fill_(3)
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(y1, eager) and torch.equal(y2, eager), lens


def test_decode_is_the_same_every_time(ext, gpu):
    c = kv4_case(13, 2, 16, 2, 64, 16, [4000, 3000], gpu)
    want = _decode(ext, c)
    for _ in range(5):
        assert torch.equal(_decode(ext, c), want)


def test_decode_offsets_past_32_bits(ext, gpu):
    # a cache side of more than 4 GiB whose used pages lie at its end
    D, page, Hkv = 128, 1024, 8
    NP = (1 << 32) // (Hkv * page * D // 2) + 3
    K = torch.zeros(NP, Hkv, page, D // 2, dtype=torch.uint8, device=gpu)
    V = torch.zeros_like(K)
    sK, sV = torch.zeros(NP, Hkv, page, device=gpu), torch.zeros(NP, Hkv, page, device=gpu)
    g = torch.Generator().manual_seed(14)
    n = 1500
    tables = torch.tensor([[NP - 1, NP - 2]], dtype=torch.int32, device=gpu)
    slots = torch.cat((torch.arange(page) + (NP - 1) * page, torch.arange(n - page) + (NP - 2) * page)).to(torch.int32).to(gpu)
    k, v = rows(g, n, Hkv, D).half(), rows(g, n, Hkv, D).half()
    ext.kv4_cache_append(k.to(gpu), v.to(gpu), K, V, sK, sV, slots)
    back = ext.kv4_cache_read(K, sK, slots).cpu()
    c4, s4 = G.kv4_quantize(k.float().numpy())
    assert torch.equal(back, (torch.from_numpy(c4).float() * torch.from_numpy(s4).unsqueeze(-1)).half())
    q, sq = quantize_rows(torch.randn(1, 16, D, generator=g))
    c = dict(Q=q.to(gpu), sQ=sq.to(gpu), K=K, V=V, sK=sK, sV=sV, tables=tables,
             lens=torch.tensor([n], dtype=torch.int32, device=gpu), max_context=n)
    out = _decode(ext, c)
    small = dict(c, K=K[NP - 2:].clone(), V=V[NP - 2:].clone(), sK=sK[NP - 2:].clone(), sV=sV[NP - 2:].clone(),
                 tables=torch.tensor([[1, 0]], dtype=torch.int32, device=gpu))
    _check(small, out)


def test_decode_of_one_position_rounds_only_its_output(ext, gpu):
    # one key: the weight cancels but for its 22 bits (2^-22) and a few fp32 roundings (2^-21
    # together), and the output rounds once (2^-11)
    c = kv4_case(15, 6, 16, 4, 64, 16, [1] * 6, gpu)
    ref, _ = G.kv4_decode(*(c[k].cpu().numpy() for k in ("Q", "K", "V", "sQ", "sK", "sV", "tables", "lens")))
    assert_within(np64(_decode(ext, c)), ref, (2.0 ** -11 + 2.0 ** -20) * np.abs(ref) + 2.0 ** -25)
