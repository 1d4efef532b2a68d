"""Attention of drafted trees over the paged INT8 cache (GPU) against the 64-bit oracle."""
import numpy as np
import pytest
import torch

import int8k_capi as capi
from grouped_helpers import assert_within, np64, quantize_rows, rows
from oracle import paged_oracle as P
from paged_helpers import attention_bound, tree_case, words_of

pytestmark = pytest.mark.gpu


def _run(ext, c, bshd=False):
    return ext.int8_tree_attention_forward_paged(
        c["Q"], c["K"], c["V"], c["sQ"], c["sK"], c["sV"], c["tables"], c["lens"], c["mask"],
        c["max_context"], node_counts=c["counts"], out_bshd=bshd)


def _oracle(c):
    n = lambda t: None if t is None else t.cpu().numpy()
    m = n(c["mask"])
    return P.tree_attention(*(n(c[k]) for k in ("Q", "K", "V", "sQ", "sK", "sV", "tables", "lens")),
                            m[None] if m is not None and m.ndim == 2 else m, n(c["counts"]), c["max_context"])


def _check(c, out, label=""):
    ref, mag = _oracle(c)
    vmax = float(127 * c["sV"][torch.isfinite(c["sV"])].max())
    assert_within(np64(out), ref, attention_bound(ref, mag, c["max_context"], vmax), label)
    return ref


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (4, 4), (8, 2), (6, 2), (32, 8), (20, 1)])
@pytest.mark.parametrize("N", [1, 3, 8, 17, 64, 65])
def test_trees(ext, gpu, N, H, Hkv, D):
    page = {1: 16, 3: 64, 8: 16, 17: 32, 64: 1024, 65: 16}[N]
    lens = [1, page - 1, 0, page + 1, 200, 333]
    c = tree_case(N + H + D, lens, N, H, Hkv, D, page, gpu)
    out = _run(ext, c)
    assert out.shape == c["Q"].shape and out.dtype == torch.float16
    _check(c, out)
    assert torch.equal(_run(ext, c, True), out.transpose(1, 2))


@pytest.mark.parametrize("N", [1, 7, 130, 256])
@pytest.mark.parametrize("mask", ["each", "shared", None])
def test_masks_and_node_counts(ext, gpu, N, mask):
    counts = [N, 0, 1, max(1, N // 2), N]
    lens = [100, 50, 0, 31, 0]
    c = tree_case(N, lens, N, 4, 2, 64, 16, gpu, counts=counts, mask=mask)
    out = _run(ext, c)
    for b, n in enumerate(counts):
        assert (out[b, :, n:] == 0).all()
    _check(c, out)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,G,N,Hkv,longest", [
    (33, 2, 50, 2, 300), (5, 3, 43, 12, 300), (33, 2, 50, 2, 1500), (3, 8, 50, 2, 4000),
    (33, 3, 43, 4, 300), (12, 2, 130, 8, 300), (33, 8, 50, 1, 1500), (5, 3, 43, 12, 4000),
    (5, 8, 50, 4, 1500), (12, 1, 100, 12, 700), (5, 1, 256, 8, 1500), (20, 3, 43, 8, 1500), (33, 3, 43, 2, 4000),
    (2, 8, 50, 8, 9000), (33, 1, 256, 4, 1000), (33, 3, 43, 2, 6000), (20, 1, 100, 4, 2000), (20, 1, 100, 8, 300),
    (5, 8, 50, 12, 6000)])
def test_many_rows_per_key_head(ext, gpu, B, G, N, Hkv, longest, D):
    # where waves of a block share their keys: whole sequences and cut ones, rows past the last, one
    # long sequence among short and empty ones
    g = torch.Generator().manual_seed(B + N)
    lens = [longest - N] + torch.randint(0, 150, (B - 2,), generator=g).tolist() + [0]
    counts = [N] + torch.randint(0, N + 1, (B - 2,), generator=g).tolist() + [N]
    c = tree_case(B * N + D, lens, N, G * Hkv, Hkv, D, 32, gpu, counts=counts)
    before = capi.paged_bad_ids()
    out = _run(ext, c)
    _check(c, out)
    assert capi.paged_bad_ids() == before
    c["mask"], c["counts"] = None, None
    c["max_context"] = longest
    c["lens"].clamp_(max=100)
    c["lens"][0] = longest - N
    need = (c["lens"] + N + 31) // 32  # entries behind a sequence's pages become page 0
    c["tables"].clamp_(min=0)
    assert int(need.max()) <= c["tables"].shape[1]
    _check(c, _run(ext, c))
    assert torch.equal(_run(ext, c), _run(ext, c))


def test_chain_is_the_mask_of_the_tokens_up_to_itself(ext, gpu):
    c = tree_case(1, [77, 500], 70, 4, 1, 128, 64, gpu, mask=None)
    want = _run(ext, c)
    c["mask"] = words_of([set(range(i + 1)) for i in range(70)], 70).to(gpu)
    assert torch.equal(_run(ext, c), want)


def test_any_mask_bits(ext, gpu):
    # not only trees: rows that see later nodes, no node at all, all of them, bits past the nodes
    N = 66
    g = torch.Generator().manual_seed(2)
    sets = [set(torch.randperm(N, generator=g)[:int(torch.randint(0, N + 1, (1,), generator=g))].tolist()) for _ in range(N)]
    sets[0], sets[1], sets[65] = set(), set(range(N)), {63, 64}
    c = tree_case(3, [0, 90, 0], N, 2, 2, 64, 16, gpu, counts=[66, 66, 40])
    c["mask"] = words_of(sets, N).to(gpu)
    out = _run(ext, c)
    assert (out[0, :, 0] == 0).all() and (out[2, :, 0] == 0).all() and (out[1, :, 0] != 0).any()
    _check(c, out)
    c["mask"][:, 1] |= ~0 << 2  # bits of nodes that do not exist
    assert torch.equal(_run(ext, c), out)


@pytest.mark.parametrize("B,N,H,Hkv,D,L", [(1, 5, 8, 8, 128, 20001), (2, 16, 4, 1, 64, 9000), (1, 1, 2, 1, 64, 70000),
                                           (40, 4, 4, 2, 128, 300), (130, 1, 2, 1, 64, 5000), (70, 2, 3, 3, 128, 2600), (3, 32, 12, 2, 128, 5000), (1, 256, 16, 2, 64, 3000)])
def test_long_and_wide(ext, gpu, B, N, H, Hkv, D, L):
    c = tree_case(L + B, [max(1, L - 37 * b) for b in range(B)], N, H, Hkv, D, 32, gpu)
    _check(c, _run(ext, c))


def test_agrees_with_the_paged_decode(ext, gpu):
    # one node per sequence and a key head per query head: the decode of one position more
    c = tree_case(4, [99, 500, 1], 1, 4, 4, 64, 16, gpu)
    want = ext.int8_decode_attention_forward_paged(
        c["Q"][:, :, 0].contiguous(), c["K"], c["V"], c["sQ"][:, :, 0].contiguous(), c["sK"], c["sV"], c["tables"],
        c["lens"] + 1, c["max_context"])
    out = _run(ext, c)[:, :, 0]
    ref, mag = _oracle(c)
    bound = attention_bound(ref, mag, 501, float(127 * c["sV"].max()))[:, :, 0]
    assert_within(np64(out), np64(want), 2 * bound + 2.0 ** -10 * mag[:, :, 0])


def test_max_context_cuts_the_sequence_then_the_nodes(ext, gpu):
    c = tree_case(5, [100, 300, 40], 8, 4, 2, 64, 16, gpu)
    for top in (303, 300, 200, 44, 40, 3):
        c["max_context"] = top
        _check(c, _run(ext, c), f"max_context {top}")
    c["max_context"] = 308
    c["lens"].copy_(torch.tensor([-7, 2 ** 31 - 1, 40]))
    _check(c, _run(ext, c), "lengths out of range")


def test_max_context_beyond_the_lengths(ext, gpu):
    c = tree_case(6, [5, 300, 0], 6, 8, 2, 128, 64, gpu)
    want = _run(ext, c)
    wide = torch.full((3, 1000), -1, dtype=torch.int32, device=gpu)
    wide[:, :c["tables"].shape[1]] = c["tables"]
    c["tables"], c["max_context"] = wide, 64000
    out = _run(ext, c)
    ref = _check(c, out)
    assert_within(np64(out), np64(want), 2.0 ** -10 * np.abs(ref) + 2.0 ** -12)


def test_bad_page_ids_read_the_last_page_and_are_counted(ext, gpu):
    c = tree_case(7, [100, 50], 5, 4, 2, 64, 16, gpu)
    before = capi.paged_bad_ids()
    _check(c, _run(ext, c))  # -1 padding behind the lengths is never read
    assert capi.paged_bad_ids() == before
    c["tables"][0, 2], c["tables"][1, 0] = -5, 10 ** 6
    _check(c, _run(ext, c))
    assert capi.paged_bad_ids() > before


def test_unseen_rows_may_hold_anything(ext, gpu):
    # behind the last node, and nodes that no row sees
    N = 9
    c = tree_case(8, [70, 33], N, 8, 2, 128, 64, gpu)
    c["mask"] = words_of([{i} for i in range(N)], N).to(gpu)
    c["mask"][4] = 0
    want = _run(ext, c)
    for b, n in enumerate((70, 33)):
        for pos in [n + 4] + list(range(n + N, -(-(n + N) // 64) * 64)):
            p = int(c["tables"][b, pos // 64])
            c["sK"][p, :, pos % 64] = float("nan")
            c["sV"][p, :, pos % 64] = float("inf")
            c["K"][p, :, pos % 64] = -128
            c["V"][p, :, pos % 64] = -128
    assert torch.equal(_run(ext, c), want)
    assert torch.isfinite(want).all()


def test_a_node_reaches_only_the_rows_that_see_it(ext, gpu):
    c = tree_case(9, [40], 6, 4, 2, 64, 16, gpu)
    c["mask"] = words_of([{0}, {0, 1}, {2}, {2, 3}, {4}, {0, 5}], 6).to(gpu)
    p = int(c["tables"][0, 42 // 16])
    c["sK"][p, 1, 42 % 16] = float("nan")  # node 2, key head 1
    out = _run(ext, c)
    assert torch.isnan(out[0, 2:, 2:4]).all()
    assert torch.isfinite(out[0, :2]).all() and torch.isfinite(out[0, 2:, [0, 1, 4, 5]]).all()


def test_scores_of_minus_infinity_weigh_nothing(ext, gpu):
    # the first tiles of a wave hold no other
    c = tree_case(12, [300, 20], 5, 8, 2, 128, 32, gpu)
    c["Q"] = -c["Q"].abs().clamp(min=1)
    for pos in list(range(40)) + list(range(256, 288)):
        p = int(c["tables"][0, pos // 32])
        c["K"][p, :, pos % 32], c["sK"][p, :, pos % 32] = 1, float("inf")
    out = _run(ext, c)
    assert torch.isfinite(out).all()
    with np.errstate(invalid="ignore"):
        _check(c, out)


@pytest.mark.parametrize("spread", [1e-6, 1e4])
def test_value_scales_of_very_different_sizes(ext, gpu, spread):
    c = tree_case(10, [500, 900], 12, 8, 2, 128, 32, gpu)
    g = torch.Generator().manual_seed(1)
    c["sV"].mul_((torch.rand(c["sV"].shape, generator=g) ** 4).to(gpu) * spread)
    _check(c, _run(ext, c))


def test_large_scores(ext, gpu):
    # one key far above the rest, at the end, at the start, and rising scores
    c = tree_case(11, [400, 400, 400], 3, 4, 1, 64, 16, gpu)
    pages = c["tables"].cpu()
    for b, at in ((0, 399), (1, 0)):
        c["sK"][int(pages[b, at // 16]), :, at % 16] *= 300
    for j in range(25):
        c["sK"][int(pages[2, j])] *= 1 + j
    ref, mag = _oracle(c)
    # scores of up to 2^12 (3 fp32 roundings each) move a weight by 2^12 * 3 * 2^-24 < 2^-10
    assert_within(np64(_run(ext, c)), ref, attention_bound(ref, mag, 403, float(127 * c["sV"].max())) + 2.0 ** -10 * mag)


def test_long_flat_tails_add_up(ext, gpu):
    # one key outweighs each of 32768 equal ones by 2^20, so those make 2^-5 of the sum
    L, D = 32768, 64
    c = tree_case(12, [L], 1, 16, 1, D, 64, gpu, mask=None)
    c["Q"].fill_(1), c["sQ"].fill_(1.0)
    c["K"].zero_(), c["V"].fill_(100)
    c["sK"].fill_(1.0), c["sV"].fill_(0.01)
    p = int(c["tables"][0, 3])
    c["K"][p, 0, 5] = 100
    c["sK"][p, 0, 5] = float(20 * np.log(2) * np.sqrt(D) / (100 * D))
    c["V"][p, 0, 5] = 0
    _check(c, _run(ext, c))


def test_strided_and_offset_inputs(ext, gpu):
    c = tree_case(13, [60, 33], 5, 4, 2, 64, 16, gpu)
    want = _run(ext, c)
    d = dict(c)
    d["Q"] = c["Q"].transpose(1, 2).contiguous().transpose(1, 2)
    d["sQ"] = c["sQ"].transpose(1, 2).contiguous().transpose(1, 2)
    d["tables"] = torch.stack((c["tables"], c["tables"]), 2)[..., 0]
    d["lens"] = torch.stack((c["lens"], c["lens"]), 1)[:, 0]
    d["mask"] = torch.stack((c["mask"], c["mask"]), -1)[..., 0]
    assert torch.equal(_run(ext, d), want)
    d["Q"] = torch.cat((torch.zeros(3, dtype=torch.int8, device=gpu), c["Q"].reshape(-1)))[3:].view(c["Q"].shape)
    d["mask"] = c["mask"][:1].expand_as(c["mask"])
    c["mask"] = c["mask"][0]
    assert torch.equal(_run(ext, d), _run(ext, c))


def test_graph_replay_and_streams(ext, gpu):
    c = tree_case(14, [900, 5, 333, 1000], 12, 8, 2, 128, 32, gpu, counts=[12, 12, 12, 12])
    want = _run(ext, c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(ext, c)
    side.synchronize()
    assert torch.equal(got, want)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        y1 = _run(ext, c)
    with torch.cuda.graph(g2):
        y2 = _run(ext, c)
    for lens, counts in (([900, 5, 333, 1000], [12] * 4), ([1, 0, 64, 999], [12, 0, 3, 11]), ([33, 31, 1000, 2], [1, 2, 3, 4])):
        c["lens"].copy_(torch.tensor(lens))
        c["counts"].copy_(torch.tensor(counts))
        eager = _run(ext, c)
        y1.fill_(3)
        y2.fill_(3)
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(y1, eager) and torch.equal(y2, eager), lens


@pytest.mark.parametrize("B,G,N,Hkv,longest", [(33, 2, 50, 2, 300), (33, 3, 43, 4, 300), (5, 3, 43, 12, 4000),
                                                (12, 1, 100, 12, 700), (5, 8, 50, 4, 1500), (33, 1, 256, 4, 1000), (33, 3, 43, 2, 6000)])
def test_replays_of_many_rows_beside_rows_that_hold_anything(ext, gpu, B, G, N, Hkv, longest):
    g = torch.Generator().manual_seed(N)
    lens = [longest - N] + torch.randint(0, 250, (B - 1,), generator=g).tolist()
    c = tree_case(B + N, lens, N, G * Hkv, Hkv, 128, 32, gpu)
    want = _run(ext, c)
    for b, n in enumerate(lens):
        at = torch.arange(n + N, -(-(n + N) // 32) * 32)
        p = c["tables"][b, at // 32].long()
        c["sK"][p, :, at % 32], c["sV"][p, :, at % 32] = float("nan"), float("inf")
        c["K"][p, :, at % 32], c["V"][p, :, at % 32] = -128, -128
    assert torch.isfinite(want).all() and torch.equal(_run(ext, c), want)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = _run(ext, c)
    for shrink in (0, 100, 1):
        c["lens"].copy_((torch.tensor(lens) - shrink).clamp(min=0))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            eager = _run(ext, c)
        y.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager) and (shrink or torch.equal(y, want))


def test_the_same_every_time_and_with_a_larger_workspace(ext, gpu):
    c = tree_case(15, [4000, 3000], 6, 16, 2, 64, 16, gpu)
    want = _run(ext, c)
    for _ in range(3):
        assert torch.equal(_run(ext, c), want)
    n = capi.tree_attention_paged_workspace_bytes(4, 16, 2, 12, 4006, 64)
    ws = torch.full((n,), 0xFF, dtype=torch.uint8, device=gpu)
    got = capi.tree_attention_paged(c["Q"], c["K"], c["V"], c["sQ"], c["sK"], c["sV"], c["tables"], c["lens"], c["mask"],
                                    c["max_context"], workspace=ws)
    assert torch.equal(got, want)


def test_offsets_past_32_bits(ext, gpu):
    # cache sides of more than 4 GiB whose used pages lie at their ends
    D, page, Hkv, N = 128, 1024, 8, 4
    NP = (1 << 32) // (Hkv * page * D) + 3
    K = torch.zeros(NP, Hkv, page, D, dtype=torch.int8, device=gpu)
    V = torch.zeros_like(K)
    sK, sV = torch.zeros(NP, Hkv, page, device=gpu), torch.zeros(NP, Hkv, page, device=gpu)
    g = torch.Generator().manual_seed(16)
    small = {}
    for n, pages, scales in (("K", K, sK), ("V", V, sV)):
        small[n], small["s" + n] = quantize_rows(rows(g, 2, Hkv, page, D))
        pages[NP - 2:], scales[NP - 2:] = small[n].to(gpu), small["s" + n].to(gpu)
    q, sq = quantize_rows(torch.randn(1, 16, N, D, generator=g))
    c = dict(Q=q.to(gpu), sQ=sq.to(gpu), K=K, V=V, sK=sK, sV=sV, mask=None, counts=None, max_context=1504,
             tables=torch.tensor([[NP - 1, NP - 2]], dtype=torch.int32, device=gpu),
             lens=torch.tensor([1500], dtype=torch.int32, device=gpu))
    out = _run(ext, c)
    _check(dict(c, **{n: t.to(gpu) for n, t in small.items()},
                tables=torch.tensor([[1, 0]], dtype=torch.int32, device=gpu)), out)
