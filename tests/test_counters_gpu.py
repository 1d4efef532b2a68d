"""The counters of bad ids, slots and positions are read with the device synchronised: a call that
still waits on a stream of its own is counted (GPU)."""
import pytest
import torch

import int8k_capi as capi
from grouped_helpers import kv4_case
from paged_helpers import sparse_case, tree_case

pytestmark = pytest.mark.gpu


def _heads(gpu, D=64):
    x = torch.ones(1, 3, 4 * D, device=gpu)
    angles = torch.ones(5, D // 2, device=gpu)
    return x, angles, torch.zeros(3, dtype=torch.int32, device=gpu)


def _append(ext, gpu):
    x, angles, pos = _heads(gpu)
    pages, s = torch.zeros(2, 1, 16, 64, dtype=torch.int8, device=gpu), torch.zeros(2, 1, 16, device=gpu)
    slots = torch.tensor([0, 32, 1], dtype=torch.int32, device=gpu)
    return lambda: ext.qk_norm_rope_append(x, 2, 1, angles, angles, pos, pages, pages.clone(), s, s.clone(), slots)


def _move(ext, gpu):
    pages, s = torch.zeros(2, 1, 16, 64, dtype=torch.int8, device=gpu), torch.zeros(2, 1, 16, device=gpu)
    src, dst = (torch.tensor(i, dtype=torch.int32, device=gpu) for i in ([1, 32], [2, 3]))
    return lambda: ext.kv_cache_move_paged(pages, pages.clone(), s, s.clone(), src, dst)


def _means(ext, gpu):
    pages, s = torch.zeros(2, 1, 16, 64, dtype=torch.int8, device=gpu), torch.zeros(2, 1, 16, device=gpu)
    m, sm = torch.zeros(2, 1, 64, dtype=torch.int8, device=gpu), torch.zeros(2, 1, device=gpu)
    ids = torch.tensor([0, 2], dtype=torch.int32, device=gpu)
    return lambda: ext.kv_page_means(pages, s, ids, m, sm)


def _tree(ext, gpu):
    c = tree_case(1, [40], 3, 4, 2, 64, 16, gpu)
    c["tables"][0, 1] = 10 ** 6
    return lambda: ext.int8_tree_attention_forward_paged(c["Q"], c["K"], c["V"], c["sQ"], c["sK"], c["sV"], c["tables"],
                                                         c["lens"], c["mask"], c["max_context"])


def _sparse(ext, gpu):
    c = sparse_case(1, [320], 4, 2, 64, 16, gpu, 4)
    c["tables"][0, 2] = 10 ** 6
    return lambda: ext.int8_decode_attention_forward_paged_sparse(
        c["Q"], c["K"], c["V"], c["sQ"], c["sK"], c["sV"], c["M"], c["sM"], c["tables"], c["lens"], c["max_context"], 4)


def _rope(ext, gpu):
    x, angles, pos = _heads(gpu)
    pos[1] = 5
    return lambda: ext.qk_norm_rope(x, 2, 1, angles, angles, pos)


def _kv4(ext, gpu):
    c = kv4_case(1, 2, 8, 2, 64, 16, [40, 7], gpu)
    c["tables"][0, 1] = 10 ** 6
    return lambda: ext.int8_decode_attention_forward_kv4_paged(
        c["Q"], c["K"], c["V"], c["sQ"], c["sK"], c["sV"], c["tables"], c["lens"], c["max_context"])


def _paged(ext, gpu):
    c = tree_case(2, [40], 1, 2, 2, 64, 16, gpu)
    c["tables"][0, 1] = 10 ** 6
    q, sq = c["Q"][:, :, 0].contiguous(), c["sQ"][:, :, 0].contiguous()
    return lambda: ext.int8_decode_attention_forward_paged(q, c["K"], c["V"], sq, c["sK"], c["sV"], c["tables"], c["lens"], 40)


@pytest.mark.parametrize("call,count", [
    (_append, capi.paged_bad_ids), (_move, capi.paged_bad_ids), (_means, capi.paged_bad_ids), (_tree, capi.paged_bad_ids),
    (_sparse, capi.paged_bad_ids), (_rope, capi.rope_bad_positions), (_kv4, capi.kv4_bad_ids),
    (_paged, capi.decode_paged_bad_page_ids)], ids=lambda f: f.__name__)
def test_a_call_in_flight_on_another_stream_is_counted(ext, gpu, call, count):
    run = call(ext, gpu)
    run()  # (loads the kernels)
    before = count()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)  # tens of milliseconds before the call's kernels start
        run()
    seen = count()
    torch.cuda.synchronize()
    assert seen > before
    assert count() == seen
