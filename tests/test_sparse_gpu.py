"""Decode over selected blocks of the paged INT8 cache (GPU) against the 64-bit oracle."""
import numpy as np
import pytest
import torch

import int8k_capi as capi
from grouped_helpers import assert_within, np64
from oracle import paged_oracle as P
from paged_helpers import attention_bound, sparse_case

pytestmark = pytest.mark.gpu


def _run(ext, c):
    return ext.int8_decode_attention_forward_paged_sparse(
        c["Q"], c["K"], c["V"], c["sQ"], c["sK"], c["sV"], c["M"], c["sM"], c["tables"], c["lens"], c["max_context"],
        c["top"])


def _check(c, got, label=""):
    out, which = got
    ref, mag, want = P.sparse_decode(*(c[k].cpu().numpy() for k in ("Q", "K", "V", "sQ", "sK", "sV", "M", "sM", "tables", "lens")),
                                     c["max_context"], c["top"])
    np.testing.assert_array_equal(which.cpu().numpy(), want)
    vmax = float(127 * c["sV"][torch.isfinite(c["sV"])].max())
    assert_within(np64(out), ref, attention_bound(ref, mag, c["top"] * c["K"].shape[2], vmax), label)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (4, 4), (8, 2), (6, 2), (32, 1), (40, 2)])
@pytest.mark.parametrize("page,top", [(16, 1), (16, 2), (16, 9), (64, 5), (256, 3), (16, 100)])
def test_selection_and_attention(ext, gpu, page, top, H, Hkv, D):
    lens = [1, page - 1, page, page + 1, 0, 7 * page + 3, 40 * page - 1]
    c = sparse_case(H + D + page + top, lens, H, Hkv, D, page, gpu, top)
    out, which = _run(ext, c)
    assert out.shape == c["Q"].shape and out.dtype == torch.float16 and which.dtype == torch.int32
    assert (out[4] == 0).all() and (which[4] == -1).all()
    _check(c, (out, which))


@pytest.mark.parametrize("B,H,Hkv,D,page,L,top", [(1, 8, 2, 128, 16, 70000, 50), (2, 2, 1, 64, 16, 40000, 1500),
                                                  (30, 4, 2, 128, 64, 900, 4), (1, 16, 1, 128, 32, 33000, 1030)])
def test_many_blocks(ext, gpu, B, H, Hkv, D, page, L, top):
    c = sparse_case(L + B, [max(1, L - 37 * b) for b in range(B)], H, Hkv, D, page, gpu, top)
    _check(c, _run(ext, c))


def test_ties_go_to_the_lowest_block(ext, gpu):
    c = sparse_case(1, [16 * 300, 16 * 2500 + 5], 4, 2, 64, 16, gpu, 20)
    c["M"].zero_()  # all scores are equal
    got = _run(ext, c)
    for b, n in enumerate((300, 2501)):
        assert (got[1][b].cpu() == torch.tensor(list(range(19)) + [n - 1])).all()
    _check(c, got)
    # two kinds of blocks, and zeros of either sign
    c["M"][::3] = c["M"].new_tensor(3)
    c["sM"][1::3] = -0.0
    _check(c, _run(ext, c))


def test_scores_next_to_each_other(ext, gpu):
    # scores that differ in the last bits of 64: fp32 products would tie or swap them
    c = sparse_case(2, [16 * 400], 2, 1, 64, 16, gpu, 50)
    g = torch.Generator().manual_seed(3)
    c["M"].copy_(c["M"][:1].expand_as(c["M"]).clone())
    base = torch.full((c["sM"].numel(),), 0.01)
    steps = torch.randint(0, 40, (c["sM"].numel(),), generator=g, dtype=torch.int32)
    c["sM"].copy_((base.view(torch.int32) + steps).view(torch.float32).view(c["sM"].shape))
    c["Q"].copy_(c["M"][0, 0].expand_as(c["Q"]))
    c["sQ"].fill_(0.013)
    _check(c, _run(ext, c))


def test_a_score_is_the_largest_of_its_group(ext, gpu):
    c = sparse_case(4, [16 * 60], 8, 2, 64, 16, gpu, 6)
    c["sQ"][0, :4] *= torch.tensor([1e-3, 1e3, 1.0, 1e-20], device=gpu)
    _check(c, _run(ext, c))
    c["sQ"][0, 0] = 0
    _check(c, _run(ext, c))


def test_nan_scores_come_last(ext, gpu):
    c = sparse_case(5, [16 * 40], 4, 1, 64, 16, gpu, 38)
    t = c["tables"][0].long()
    c["sM"][t[[0, 3, 9]]] = float("nan")
    c["sM"][t[5]] = float("inf")
    out, which = _run(ext, c)
    ref = P.sparse_decode(*(c[k].cpu().numpy() for k in ("Q", "K", "V", "sQ", "sK", "sV", "M", "sM", "tables", "lens")),
                          c["max_context"], 38)[2]
    np.testing.assert_array_equal(which.cpu().numpy(), ref)


def test_the_last_block_and_rows_behind_it_may_hold_anything(ext, gpu):
    c = sparse_case(6, [16 * 30 + 5, 16 * 9], 4, 2, 128, 16, gpu, 4)
    want = _run(ext, c)
    for b, n in enumerate((16 * 30 + 5, 16 * 9)):
        p = int(c["tables"][b, (n - 1) // 16])
        c["sM"][p] = float("nan")
        if n % 16:
            c["sK"][p, :, n % 16:], c["sV"][p, :, n % 16:] = float("nan"), float("inf")
    got = _run(ext, c)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_max_context_cuts_and_widens(ext, gpu):
    c = sparse_case(7, [700, 300, 0], 8, 2, 128, 32, gpu, 5)
    want = _run(ext, c)
    for top in (699, 333, 32, 1):
        c["max_context"] = top
        _check(c, _run(ext, c), f"max_context {top}")
    wide = torch.full((3, 1000), -1, dtype=torch.int32, device=gpu)
    wide[:, :c["tables"].shape[1]] = c["tables"]
    c["tables"], c["max_context"] = wide, 32000
    got = _run(ext, c)
    assert torch.equal(got[1], want[1])
    _check(c, got)
    c["lens"].copy_(torch.tensor([700, 300, -3]))
    again = _run(ext, c)
    assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])


def test_bad_page_ids_read_the_last_page_and_are_counted(ext, gpu):
    c = sparse_case(8, [16 * 20, 16 * 3], 4, 2, 64, 16, gpu, 4)
    before = capi.paged_bad_ids()
    _check(c, _run(ext, c))
    assert capi.paged_bad_ids() == before
    c["tables"][0, 2], c["tables"][1, 0] = -5, 10 ** 6
    _check(c, _run(ext, c))
    assert capi.paged_bad_ids() > before


def test_all_blocks_taken_is_the_whole_decode(ext, gpu):
    c = sparse_case(9, [200, 77], 4, 4, 64, 16, gpu, 50)
    out, which = _run(ext, c)
    want = ext.int8_decode_attention_forward_paged(c["Q"], c["K"], c["V"], c["sQ"], c["sK"], c["sV"], c["tables"], c["lens"], 200)
    assert_within(np64(out), np64(want), 2.0 ** -9 * np.abs(np64(want)) + 2.0 ** -9)
    assert (which[0, 0, :13].cpu() == torch.arange(13)).all() and (which[0, 0, 13:] == -1).all()


def test_graph_replay_and_streams(ext, gpu):
    c = sparse_case(10, [900, 5, 333, 1000], 8, 2, 128, 16, gpu, 7)
    want = _run(ext, c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(ext, c)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        y1 = _run(ext, c)
    with torch.cuda.graph(g2):
        y2 = _run(ext, c)
    for lens in ([900, 5, 333, 1000], [1, 0, 64, 999], [33, 31, 1000, 2]):
        c["lens"].copy_(torch.tensor(lens))
        eager = _run(ext, c)
        for y in (y1, y2):
            y[0].fill_(3), y[1].fill_(3)
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        for y in (y1, y2):
            assert torch.equal(y[0], eager[0]) and torch.equal(y[1], eager[1]), lens


def test_workspace_of_a_larger_call(ext, gpu):
    c = sparse_case(11, [900, 333], 8, 2, 64, 16, gpu, 7)
    want = _run(ext, c)
    n = capi.decode_paged_sparse_workspace_bytes(5, 8, 2, 4000, 16, 11, 64)
    ws = torch.full((n,), 0xFF, dtype=torch.uint8, device=gpu)
    got = capi.decode_attention_paged_sparse(c["Q"], c["K"], c["V"], c["sQ"], c["sK"], c["sV"], c["M"], c["sM"], c["tables"],
                                             c["lens"], c["max_context"], c["top"], workspace=ws)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
