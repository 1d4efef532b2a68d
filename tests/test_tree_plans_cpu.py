"""The sizes of paged_plans.py are those of every kernel that the plan of the attention over the INT8
paged cache picks from, whole and cut, so that the GPU tests run them all."""
import ctypes

import pytest

from paged_plans import CASES, SIZES

INVALID = 1


@pytest.mark.parametrize("kernel,size", CASES)
def test_the_plan_of_a_size(capi, kernel, size):
    B, G, N, Hkv, top = size
    D, rows, share, waves, cut = kernel
    plan = capi.tree_attention_paged_plan(B, G * Hkv, Hkv, N, top, D)
    assert plan[:3] == (rows, share, waves) and (plan[3] > 0) == cut, "take a size that this kernel is chosen for"


def test_every_choice_has_sizes(capi):
    # what the plan picks over a grid of sizes
    seen = set()
    for D in (64, 128):
        for B in (1, 3, 9, 20):
            for G in (1, 4, 8):
                for N in (1, 5, 9, 21, 40, 75, 256):
                    for Hkv in (1, 2, 8, 12):
                        for top in (300, 700, 1500, 3000, 9000, 19000, 100000):
                            plan = capi.tree_attention_paged_plan(B, G * Hkv, Hkv, N, top, D)
                            assert plan[3] == 0 or plan[3] > B
                            seen.add((D,) + plan[:3] + (plan[3] > 0,))
    assert seen <= set(SIZES) and len(SIZES) == 20


def test_a_plan_needs_the_workspace_of_its_pieces(capi):
    for D in (64, 128):
        for B, H, Hkv, N, top in ((4, 32, 8, 64, 16384), (16, 32, 8, 16, 8208), (1, 32, 8, 1, 20000), (13, 12, 12, 9, 3010)):
            pieces = capi.tree_attention_paged_plan(B, H, Hkv, N, top, D)[3]
            need = capi.tree_attention_paged_call_workspace_bytes(B, H, Hkv, N, top, D)
            rows = pieces * H * N
            assert need >= rows * (D + 2) * 4 and need <= rows * (D + 2) * 4 + 512 and (need > 0) == (pieces > 0)


def test_refusals(capi):
    plan = (ctypes.c_int * 4)()
    run = capi.load().int8k_tree_attention_paged_plan
    for a in ((0, 8, 2, 4, 100, 64), (1, 8, 3, 4, 100, 64), (1, 8, 2, 0, 100, 64), (1, 8, 2, 257, 100, 64), (1, 8, 2, 4, 0, 64),
              (1, 8, 2, 4, 100, 96), (1 << 20, 8, 2, 4, 100, 64)):
        assert run(*a, plan) == INVALID
    assert run(1, 8, 2, 4, 100, 64, None) == INVALID
