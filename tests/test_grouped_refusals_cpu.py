"""What the grouped-query serving entry points refuse, without a GPU: the C ABI before any HIP
call, the torch ops on CPU tensors and wrong types."""
import ctypes

import pytest
import torch

P = [ctypes.c_void_p(0x10000 * (i + 1)) for i in range(20)]
NULL = ctypes.c_void_p(0)
INVALID, UNSUPPORTED, WORKSPACE, MISALIGNED = 1, 2, 3, 4


def _linear(lib, x=P[0], W=P[1], out=P[2], dt=0, sx=P[3], nsx=8, sw=P[4], nsw=64, b=NULL, T=8, K=32,
            N=64, flags=0):
    return lib.int8k_linear(x, W, out, dt, sx, nsx, sw, nsw, b, T, K, N, flags, P[9], 1 << 40, None)


@pytest.mark.parametrize("change,status", [
    (dict(x=NULL), INVALID), (dict(W=NULL), INVALID), (dict(out=NULL), INVALID),
    (dict(sx=NULL), INVALID), (dict(sw=NULL), INVALID), (dict(T=0), INVALID), (dict(K=0), INVALID),
    (dict(N=-16), INVALID), (dict(dt=3), INVALID), (dict(dt=-1), INVALID), (dict(flags=2), INVALID),
    (dict(nsx=7), INVALID), (dict(nsw=63), INVALID), (dict(K=40), UNSUPPORTED),
    (dict(N=72, nsw=72), UNSUPPORTED), (dict(K=131072), UNSUPPORTED),
    (dict(T=1 << 30, nsx=1), UNSUPPORTED), (dict(N=1 << 28, nsw=1), UNSUPPORTED),
    (dict(x=ctypes.c_void_p(0x10008)), MISALIGNED), (dict(W=ctypes.c_void_p(0x10001)), MISALIGNED),
    (dict(out=ctypes.c_void_p(0x10002)), MISALIGNED), (dict(b=ctypes.c_void_p(0x10002)), MISALIGNED)])
def test_linear_refusals(capi, change, status):
    assert _linear(capi.load(), **change) == status


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("change,status", [
    (dict(x=NULL), INVALID), (dict(cos=NULL), INVALID), (dict(pos=NULL), INVALID), (dict(q=NULL), INVALID),
    (dict(dt=5), INVALID), (dict(top=0), INVALID), (dict(rot=0), INVALID), (dict(rot=63), INVALID),
    (dict(rot=66), INVALID), (dict(B=0), INVALID), (dict(S=-1), INVALID), (dict(H=0), INVALID),
    (dict(Hkv=0), INVALID), (dict(flags=2), INVALID), (dict(D=72), UNSUPPORTED), (dict(D=272), UNSUPPORTED),
    (dict(x=ctypes.c_void_p(0x10004)), MISALIGNED), (dict(q=ctypes.c_void_p(0x10004)), MISALIGNED),
    (dict(cos=ctypes.c_void_p(0x10002)), MISALIGNED)])
def test_heads_refusals(capi, change, status, quant):
    a = dict(x=P[0], cos=P[1], pos=P[2], q=P[3], dt=1, top=100, rot=64, B=2, S=3, H=4, Hkv=2, D=64, flags=0)
    a.update(change)
    lib = capi.load()
    head = (a["x"], a["dt"], a["cos"], P[4], a["top"], a["rot"], a["pos"], NULL, NULL, 1e-6)
    tail = (a["B"], a["S"], a["H"], a["Hkv"], a["D"], a["flags"], None)
    if quant:
        st = lib.int8k_qk_norm_rope_quantize(*head, a["q"], *P[5:10], *tail)
    else:
        st = lib.int8k_qk_norm_rope(*head, a["q"], *P[5:7], *tail)
    assert st == status


@pytest.mark.parametrize("change,status", [
    (dict(Q=NULL), INVALID), (dict(cu=NULL), INVALID), (dict(n=0), INVALID), (dict(T=0), INVALID),
    (dict(H=3), INVALID), (dict(Hkv=0), INVALID), (dict(flags=8), INVALID), (dict(D=0), INVALID),
    (dict(D=72), UNSUPPORTED), (dict(D=320), UNSUPPORTED), (dict(T=1 << 26), UNSUPPORTED),
    (dict(Q=ctypes.c_void_p(0x10008)), MISALIGNED), (dict(out=ctypes.c_void_p(0x10004)), MISALIGNED),
    (dict(cu=ctypes.c_void_p(0x10002)), MISALIGNED)])
def test_packed_refusals(capi, change, status):
    a = dict(Q=P[0], out=P[1], cu=P[2], n=3, T=100, H=8, Hkv=2, D=64, flags=1)
    a.update(change)
    assert capi.load().int8k_attention_forward_packed(
        a["Q"], P[3], P[4], a["out"], P[5], P[6], P[7], a["cu"], a["n"], a["T"], a["H"], a["Hkv"],
        a["D"], a["flags"], None) == status


@pytest.mark.parametrize("change,status", [
    (dict(k=NULL), INVALID), (dict(slots=NULL), INVALID), (dict(dt=3), INVALID), (dict(T=0), INVALID),
    (dict(H=0), INVALID), (dict(NP=0), INVALID), (dict(D=96), UNSUPPORTED), (dict(page=8), UNSUPPORTED),
    (dict(page=48), UNSUPPORTED), (dict(page=2048), UNSUPPORTED), (dict(NP=1 << 27, page=16), UNSUPPORTED),
    (dict(st=100), MISALIGNED), (dict(k=ctypes.c_void_p(0x10008)), MISALIGNED),
    (dict(K=ctypes.c_void_p(0x10008)), MISALIGNED)])
def test_kv4_append_and_read_refusals(capi, change, status):
    a = dict(k=P[0], K=P[1], slots=P[2], dt=0, st=128, T=5, H=2, D=64, NP=4, page=16)
    a.update(change)
    lib = capi.load()
    assert lib.int8k_kv4_cache_append(a["k"], P[3], a["dt"], a["st"], 64, 128, 64, a["K"], P[4], P[5], P[6],
                                      a["slots"], a["T"], a["H"], a["D"], a["NP"], a["page"], None) == status
    if not {"k", "st"} & set(change):
        assert lib.int8k_kv4_cache_read(a["K"], P[5], a["slots"], P[7], a["dt"], a["T"], a["H"], a["D"],
                                        a["NP"], a["page"], None) == status


@pytest.mark.parametrize("change,status", [
    (dict(Q=NULL), INVALID), (dict(lens=NULL), INVALID), (dict(B=0), INVALID), (dict(H=5), INVALID),
    (dict(Hkv=0), INVALID), (dict(cols=0), INVALID), (dict(top=0), INVALID), (dict(top=65), INVALID),
    (dict(D=80), UNSUPPORTED), (dict(page=24), UNSUPPORTED), (dict(NP=1 << 28), UNSUPPORTED),
    (dict(Q=ctypes.c_void_p(0x10008)), MISALIGNED), (dict(lens=ctypes.c_void_p(0x10002)), MISALIGNED)])
def test_kv4_decode_refusals(capi, change, status):
    a = dict(Q=P[0], lens=P[1], B=2, H=8, Hkv=2, D=64, NP=4, page=16, cols=4, top=64)
    a.update(change)
    assert capi.load().int8k_decode_attention_forward_kv4_paged(
        a["Q"], P[2], P[3], P[4], P[5], P[6], P[7], P[8], a["lens"], a["B"], a["H"], a["Hkv"], a["D"],
        a["NP"], a["page"], a["cols"], a["top"], P[9], 1 << 40, None) == status


def test_counters_refuse_null(capi):
    lib = capi.load()
    assert lib.int8k_rope_bad_positions(None) == INVALID
    assert lib.int8k_kv4_bad_ids(None) == INVALID


def test_torch_ops_refuse_cpu_tensors(ext):
    i8, f = torch.zeros(4, 32, dtype=torch.int8), torch.ones(4)
    with pytest.raises(RuntimeError, match="CUDA"):
        ext.int8_linear(i8, torch.zeros(32, 16, dtype=torch.int8), f, torch.ones(16))
    with pytest.raises(RuntimeError, match="CUDA"):
        ext.qk_norm_rope(torch.zeros(4, 64), 2, 1, torch.zeros(9, 8), torch.zeros(9, 8),
                         torch.zeros(4, dtype=torch.int32))
    q = torch.zeros(2, 4, 64, dtype=torch.int8)
    with pytest.raises(RuntimeError, match="CUDA"):
        ext.int8_attention_forward_packed(q, q, q, f, f, f, torch.tensor([0, 4], dtype=torch.int32))
    pages, s = torch.zeros(2, 1, 16, 32, dtype=torch.uint8), torch.zeros(2, 1, 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ext.kv4_cache_append(torch.zeros(1, 1, 64), torch.zeros(1, 1, 64), pages, pages, s, s,
                             torch.zeros(1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA"):
        ext.kv4_cache_read(pages, s, torch.zeros(1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA"):
        ext.int8_decode_attention_forward_kv4_paged(q, pages, pages, f, s, s,
                                                    torch.zeros(2, 1, dtype=torch.int32),
                                                    torch.ones(2, dtype=torch.int32), 16)
