"""The C ABI's grouped-query entry points through their ctypes wrappers, with workspaces of exactly
the queried size (GPU): the results of the torch ops, and not a byte written past the size."""
import pytest
import torch

import int8k_capi as capi
from grouped_helpers import kv4_case, quantize_rows, rows
from test_heads_gpu import _case as heads_case
from test_heads_gpu import _to
from test_kv4_gpu import _decode

pytestmark = pytest.mark.gpu

GUARD = 4096


def _workspace(n, gpu):
    """n bytes with a guard behind them; check() tells whether the guard is whole."""
    buf = torch.full((n + GUARD,), 0x5A, dtype=torch.uint8, device=gpu)
    return buf[:n], lambda: bool((buf[n:] == 0x5A).all())


@pytest.mark.parametrize("packed", [0, capi.LINEAR_WEIGHT_PREPACKED])
@pytest.mark.parametrize("K,N", [(4096, 2048), (14336, 1024), (1024, 1040)])
def test_linear_in_one_workspace(ext, gpu, K, N, packed):
    # allocated for 600 rows and used for every shorter call; a call's own size suffices, too
    g = torch.Generator().manual_seed(K + N)
    x, sx = (t.to(gpu) for t in quantize_rows(rows(g, 600, K)))
    w, sw = (t.to(gpu) for t in quantize_rows(torch.randn(N, K, generator=g)))
    w = w if packed else w.t().contiguous()
    b = torch.randn(N, generator=g).to(gpu)
    whole, whole_ok = _workspace(capi.linear_workspace_bytes(600, K, N, packed), gpu)
    for T in (1, 7, 32, 33, 64, 130, 257, 512, 600):
        want = ext.int8_linear(x[:T], w, sx[:T], sw, bias=b, prepacked=bool(packed))
        own, own_ok = _workspace(capi.linear_call_workspace_bytes(T, K, N, packed), gpu)
        for ws in (whole, own):
            y = capi.linear(x[:T], w, sx[:T].contiguous(), sw, bias=b, flags=packed, workspace=ws)
            assert torch.equal(y, want), T
        assert torch.equal(capi.linear(x[:T], w, sx[:T].contiguous(), sw, bias=b, flags=packed), want)
        assert own_ok() and whole_ok(), T


@pytest.mark.parametrize("H,Hkv,D", [(8, 2, 128), (12, 12, 64), (32, 1, 64)])
def test_decode_in_one_workspace(ext, gpu, H, Hkv, D):
    B = 150
    lens = [1 + 37 * b % 3000 for b in range(B)]
    c = kv4_case(H + D, B, H, Hkv, D, 64, lens, gpu)
    size = capi.decode_kv4_paged_workspace_bytes(B, H, Hkv, c["max_context"], D)
    ws, ok = _workspace(size, gpu)
    for n in (1, 2, 3, 5, 17, 40, 85, 86, 127, 128, 150):
        part = dict(c, **{k: c[k][:n].contiguous() for k in ("Q", "sQ", "tables", "lens")})
        want = _decode(ext, part)
        args = (part["Q"], c["K"], c["V"], part["sQ"], c["sK"], c["sV"], part["tables"], part["lens"], c["max_context"])
        assert torch.equal(capi.decode_attention_kv4_paged(*args, workspace=ws), want), n
        assert torch.equal(capi.decode_attention_kv4_paged(*args), want), n
        assert ok(), n


@pytest.mark.parametrize("quantize", [False, True])
def test_heads_wrapper(ext, gpu, quantize):
    x, cos, sin, pos, wq, wk = _to(gpu, *heads_case(2, 21, 4, 2, 64, 32, torch.bfloat16, True))
    got = capi.qk_norm_rope(x, 4, 2, cos, sin, pos, q_weight=wq, k_weight=wk, flags=capi.ROPE_INTERLEAVED,
                            quantize=quantize)
    f = ext.qk_norm_rope_quantize if quantize else ext.qk_norm_rope
    want = f(x, 4, 2, cos, sin, pos, q_weight=wq, k_weight=wk, interleaved=True)
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_cache_wrappers(ext, gpu):
    g = torch.Generator().manual_seed(1)
    k, v = rows(g, 30, 3, 128).half().to(gpu), rows(g, 30, 3, 128).half().to(gpu)
    slots = torch.randperm(64, generator=g)[:30].to(torch.int32).to(gpu)
    sides = [(torch.zeros(4, 3, 16, 64, dtype=torch.uint8, device=gpu), torch.zeros(4, 3, 16, device=gpu)) for _ in range(4)]
    (K, sK), (V, sV), (K2, sK2), (V2, sV2) = sides
    capi.kv4_cache_append(k.transpose(0, 1).contiguous().transpose(0, 1), v, K, V, sK, sV, slots)
    ext.kv4_cache_append(k, v, K2, V2, sK2, sV2, slots)
    assert torch.equal(K, K2) and torch.equal(V, V2) and torch.equal(sK, sK2) and torch.equal(sV, sV2)
    for dt in (torch.float16, torch.float32):
        assert torch.equal(capi.kv4_cache_read(V, sV, slots, dtype=dt), ext.kv4_cache_read(V, sV, slots, dtype=dt))
