"""Sizes that the grouped-query entry points refuse before any HIP call, without a GPU."""
import ctypes

import pytest
import torch

P = [ctypes.c_void_p(0x10000 * (i + 1)) for i in range(10)]
UNSUPPORTED, MISALIGNED = 2, 4
ODD = ctypes.c_void_p(0x10004)  # refused as misaligned where the sizes are not


@pytest.mark.parametrize("n,status", [(65536, MISALIGNED), (65537, UNSUPPORTED), (2 ** 31 - 1, UNSUPPORTED)])
def test_packed_sequences(capi, n, status):
    assert capi.load().int8k_attention_forward_packed(
        ODD, P[0], P[1], P[2], P[3], P[4], P[5], P[6], n, 1 << 20, 4, 2, 64, 1, None) == status


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up pointers")
@pytest.mark.parametrize("top,status", [((1 << 30) + 1, UNSUPPORTED), (2 ** 31 - 1, UNSUPPORTED)])
def test_decode_positions(capi, top, status):
    assert capi.load().int8k_decode_attention_forward_kv4_paged(
        *P[:9], 1, 8, 2, 64, 1 << 16, 1024, 1 << 21, top, P[9], 1 << 40, None) == status
