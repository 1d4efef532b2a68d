"""Workspace sizes of the grouped-query serving entry points, without a GPU."""
import ctypes

import pytest
import torch

PACKED = 1
WORKSPACE, MISALIGNED = 3, 4


@pytest.mark.parametrize("K,N", [(4096, 28672), (4096, 128256), (8192, 28672)])
def test_linear_reads_wide_stored_weights_on_a_route_that_streams_them(capi, K, N):
    # One token against weights as stored: the tiles of 64 columns read 64 bytes a row and are
    # slower than the routes that stream whole lines or split K, which leave partials.
    assert capi.linear_workspace_bytes(1, K, N) >= N * 4


@pytest.mark.parametrize("flags", [0, PACKED])
@pytest.mark.parametrize("K,N", [(4096, 4096), (4096, 6144), (2048, 2560), (14336, 4096), (16384, 16), (131056, 512),
                                 (1024, 1024), (4096, 28672)])
def test_linear_workspace_covers_shorter_calls(capi, K, N, flags):
    # allocated once for the largest batch, used for every one below it
    need, longest = 0, 0
    for T in list(range(1, 700)) + [1000, 1023, 1024, 1025, 1500, 2048, 3000, 4096]:
        need = max(need, capi.linear_call_workspace_bytes(T, K, N, flags))
        if T in (1, 2, 31, 32, 33, 64, 65, 100, 333, 512, 513, 600, 699) or T >= 1000:
            whole = capi.linear_workspace_bytes(T, K, N, flags)
            assert whole >= max(need, longest), T
            longest = whole


def test_linear_workspace_between_the_ranges(capi):
    # past the streamed rows the query steps by 32 rows: every call inside is covered
    for K, N in ((14336, 4096), (131056, 512), (16384, 8192)):
        for T in (545, 800, 1500):
            whole = capi.linear_workspace_bytes(T, K, N)
            assert all(capi.linear_call_workspace_bytes(t, K, N) <= whole for t in range(513, T + 1))


@pytest.mark.parametrize("H,Hkv,D", [(32, 8, 128), (12, 12, 64), (8, 1, 128), (48, 2, 64), (32, 1, 64), (1, 1, 64)])
def test_decode_workspace_covers_smaller_batches(capi, H, Hkv, D):
    sizes = [capi.decode_kv4_paged_workspace_bytes(B, H, Hkv, 16384, D) for B in range(1, 1300)]
    assert sizes == sorted(sizes) and sizes[0] > 0
    assert {capi.decode_kv4_paged_workspace_bytes(7, H, Hkv, n, D) for n in (1, 100, 4096, 1 << 20)} == {sizes[6]}


# The refusals are reached before any launch only where a call does need a workspace: not on a
# machine whose GPU would run the made-up pointers if it did not.
no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up pointers")


@no_gpu
@pytest.mark.parametrize("T,K,N,flags", [(1, 4096, 4096, 0), (300, 14336, 4096, 0), (16, 8192, 1024, PACKED)])
def test_linear_refuses_workspaces_it_cannot_use(capi, T, K, N, flags):
    need = capi.linear_call_workspace_bytes(T, K, N, flags)
    assert need > 0
    P = [ctypes.c_void_p(0x10000 * (i + 1)) for i in range(6)]
    call = lambda ws, n: capi.load().int8k_linear(  # noqa: E731
        P[0], P[1], P[2], 0, P[3], 1, P[4], 1, None, T, K, N, flags, ws, n, None)
    assert call(None, 1 << 40) == WORKSPACE
    assert call(P[5], 0) == WORKSPACE
    assert call(P[5], need - 1) == WORKSPACE
    assert call(ctypes.c_void_p(0x60008), need) == MISALIGNED


@no_gpu
@pytest.mark.parametrize("B,H,Hkv,D,top", [(1, 32, 8, 128, 16384), (2, 12, 12, 64, 4096)])
def test_decode_refuses_workspaces_it_cannot_use(capi, B, H, Hkv, D, top):
    P = [ctypes.c_void_p(0x10000 * (i + 1)) for i in range(10)]
    call = lambda ws, n: capi.load().int8k_decode_attention_forward_kv4_paged(  # noqa: E731
        *P[:9], B, H, Hkv, D, 1000, 64, 256, top, ws, n, None)
    assert call(None, 1 << 40) == WORKSPACE
    assert call(P[9], 0) == WORKSPACE
    assert call(P[9], 1024) == WORKSPACE  # less than any split's states
    assert call(ctypes.c_void_p(0x90008), 1 << 40) == MISALIGNED
