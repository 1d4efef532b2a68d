"""What the operators over the paged INT8 cache refuse, without a GPU: the C ABI before any HIP
call, the torch ops on CPU tensors; and what their workspace queries promise."""
import ctypes

import pytest
import torch

P = [ctypes.c_void_p(0x10000 * (i + 1)) for i in range(20)]
NULL = ctypes.c_void_p(0)
OK, INVALID, UNSUPPORTED, WORKSPACE, MISALIGNED = 0, 1, 2, 3, 4
ODD8, ODD2 = ctypes.c_void_p(0x10008), ctypes.c_void_p(0x10002)

CACHE = [(dict(NP=0), INVALID), (dict(Hkv=0), INVALID), (dict(D=96), UNSUPPORTED), (dict(D=32), UNSUPPORTED),
         (dict(page=8), UNSUPPORTED), (dict(page=48), UNSUPPORTED), (dict(page=2048), UNSUPPORTED),
         (dict(NP=1 << 27, page=16), UNSUPPORTED), (dict(K=NULL), INVALID), (dict(K=ODD8), MISALIGNED)]


# (a rotation of 64 dims is past a head of 32 before that head is one the cache does not hold)
@pytest.mark.parametrize("change,status", [(c, INVALID if c == dict(D=32) else st) for c, st in CACHE] + [
    (dict(x=NULL), INVALID), (dict(slots=NULL), INVALID), (dict(q=NULL), INVALID), (dict(pos=NULL), INVALID),
    (dict(dt=3), INVALID), (dict(B=0), INVALID), (dict(S=0), INVALID), (dict(H=0), INVALID), (dict(flags=2), INVALID),
    (dict(rot=66), INVALID), (dict(top=0), INVALID), (dict(x=ctypes.c_void_p(0x10004)), MISALIGNED),
    (dict(slots=ODD2), MISALIGNED)])
def test_append_refusals(capi, change, status):
    a = dict(x=P[0], dt=1, top=100, rot=64, pos=P[1], q=P[2], K=P[3], slots=P[4], B=2, S=3, H=4, Hkv=2, D=64, NP=4,
             page=16, flags=0)
    a.update(change)
    assert capi.load().int8k_qk_norm_rope_append(
        a["x"], a["dt"], P[5], P[6], a["top"], a["rot"], a["pos"], NULL, NULL, 1e-6, a["q"], P[7], a["K"], P[8], P[9],
        P[10], a["slots"], a["B"], a["S"], a["H"], a["Hkv"], a["D"], a["NP"], a["page"], a["flags"], None) == status


def _tree(lib, **change):
    a = dict(Q=P[0], K=P[1], out=P[2], lens=P[3], mask=P[4], words=1, each=0, counts=NULL, B=2, H=8, Hkv=2, N=5, D=64,
             NP=40, page=16, cols=20, top=300, flags=0, ws=P[5], bytes=1 << 40)
    a.update(change)
    return lib.int8k_tree_attention_forward_paged(
        a["Q"], a["K"], P[6], a["out"], P[7], P[8], P[9], P[10], a["lens"], a["mask"], a["words"], a["each"], a["counts"],
        a["B"], a["H"], a["Hkv"], a["N"], a["D"], a["NP"], a["page"], a["cols"], a["top"], a["flags"], a["ws"], a["bytes"], None)


@pytest.mark.parametrize("change,status", CACHE + [
    (dict(Q=NULL), INVALID), (dict(lens=NULL), INVALID), (dict(out=NULL), INVALID), (dict(B=0), INVALID),
    (dict(H=5), INVALID), (dict(H=0), INVALID), (dict(N=0), INVALID), (dict(cols=0), INVALID), (dict(top=0), INVALID),
    (dict(top=321), INVALID), (dict(flags=1), INVALID), (dict(flags=4), INVALID), (dict(words=2), INVALID),
    (dict(words=0), INVALID), (dict(N=65), INVALID), (dict(each=4), INVALID), (dict(each=-5), INVALID),
    (dict(N=257, words=5), UNSUPPORTED), (dict(B=1 << 20, N=4), UNSUPPORTED), (dict(B=1 << 21, H=1, Hkv=1, N=1), UNSUPPORTED),
    (dict(cols=1 << 27, top=(1 << 30) + 1), UNSUPPORTED), (dict(Q=ODD8), MISALIGNED), (dict(lens=ODD2), MISALIGNED),
    (dict(mask=ctypes.c_void_p(0x10004)), MISALIGNED), (dict(counts=ODD2), MISALIGNED),
    (dict(out=ctypes.c_void_p(0x10004)), MISALIGNED),
    (dict(cols=2000, top=30000, ws=NULL), WORKSPACE), (dict(cols=2000, top=30000, bytes=1000), WORKSPACE),
    (dict(cols=2000, top=30000, ws=ODD8), MISALIGNED)])
def test_tree_refusals(capi, change, status):
    assert _tree(capi.load(), **change) == status


@pytest.mark.parametrize("change,status", CACHE + [
    (dict(src=NULL), INVALID), (dict(lists=0), INVALID), (dict(pairs=0), INVALID), (dict(pairs=257), UNSUPPORTED),
    (dict(lists=1 << 22), UNSUPPORTED), (dict(src=ODD2), MISALIGNED)])
def test_move_refusals(capi, change, status):
    a = dict(K=P[0], src=P[1], lists=2, pairs=3, Hkv=2, D=64, NP=4, page=16)
    a.update(change)
    assert capi.load().int8k_kv_cache_move_paged(a["K"], P[2], P[3], P[4], a["src"], P[5], a["lists"], a["pairs"], a["Hkv"],
                                                 a["D"], a["NP"], a["page"], None) == status


@pytest.mark.parametrize("change,status", CACHE + [
    (dict(ids=NULL), INVALID), (dict(n=0), INVALID), (dict(n=1 << 22), UNSUPPORTED), (dict(ids=ODD2), MISALIGNED),
    (dict(M=NULL), INVALID), (dict(M=ODD8), MISALIGNED)])
def test_means_refusals(capi, change, status):
    a = dict(K=P[0], ids=P[1], M=P[2], n=3, Hkv=2, D=64, NP=4, page=16)
    a.update(change)
    assert capi.load().int8k_kv_page_means(a["K"], P[3], a["ids"], a["M"], P[4], a["n"], a["Hkv"], a["D"], a["NP"],
                                           a["page"], None) == status


@pytest.mark.parametrize("change,status", CACHE + [
    (dict(Q=NULL), INVALID), (dict(M=NULL), INVALID), (dict(sel=NULL), INVALID), (dict(B=0), INVALID), (dict(H=5), INVALID),
    (dict(cols=0), INVALID), (dict(top=0), INVALID), (dict(top=321), INVALID), (dict(k=0), INVALID),
    (dict(B=40000), UNSUPPORTED), (dict(B=30000, H=1024), UNSUPPORTED), (dict(k=1 << 30), UNSUPPORTED), (dict(cols=1 << 27, top=(1 << 30) + 1), UNSUPPORTED), (dict(M=ODD8), MISALIGNED),
    (dict(sel=ODD2), MISALIGNED), (dict(ws=NULL), WORKSPACE), (dict(bytes=100), WORKSPACE), (dict(ws=ODD8), MISALIGNED)])
def test_sparse_refusals(capi, change, status):
    a = dict(Q=P[0], K=P[1], M=P[2], sel=P[3], B=2, H=8, Hkv=2, D=64, NP=40, page=16, cols=20, top=300, k=4, ws=P[4],
             bytes=1 << 40)
    a.update(change)
    assert capi.load().int8k_decode_attention_forward_paged_sparse(
        a["Q"], a["K"], P[5], P[6], a["sel"], P[7], P[8], P[9], a["M"], P[10], P[11], P[12], a["B"], a["H"], a["Hkv"], a["D"],
        a["NP"], a["page"], a["cols"], a["top"], a["k"], a["ws"], a["bytes"], None) == status


def test_counter_refuses_null(capi):
    assert capi.load().int8k_paged_bad_ids(None) == INVALID


@pytest.mark.parametrize("H,Hkv", [(1, 1), (8, 2), (32, 8), (40, 1), (48, 48)])
@pytest.mark.parametrize("D", [64, 128])
def test_a_workspace_serves_smaller_calls(capi, H, Hkv, D):
    tree, sparse = capi.tree_attention_paged_workspace_bytes, capi.decode_paged_sparse_workspace_bytes
    tree_call, sparse_call = capi.tree_attention_paged_call_workspace_bytes, capi.decode_paged_sparse_call_workspace_bytes
    for B, N, L in ((8, 16, 4000), (64, 64, 100000), (1, 256, 20)):
        big = tree(B, H, Hkv, N, L, D)
        for b in {1, 2, 3, 5, B // 2, B} - {0}:
            for n in {1, 7, N // 3, N} - {0}:
                for l in (1, 333, 5000, 200000):
                    if b <= B:
                        assert tree(b, H, Hkv, n, l, D) <= big
                        assert tree_call(b, H, Hkv, n, l, D) <= big
    for B, L, top in ((8, 4000, 10), (64, 100000, 64)):
        big = sparse(B, H, Hkv, L, 64, top, D)
        for b in (1, 3, B):
            for l in (1, 333, L):
                for k in (1, 7, top):
                    assert sparse(b, H, Hkv, l, 64, k, D) <= big
                    assert 0 < sparse_call(b, H, Hkv, l, 64, k, D) <= big


def test_workspace_queries_of_bad_arguments_are_0(capi):
    tree, sparse = capi.tree_attention_paged_workspace_bytes, capi.decode_paged_sparse_workspace_bytes
    for a in ((0, 8, 2, 4, 100, 64), (1, 8, 3, 4, 100, 64), (1, 8, 2, 0, 100, 64), (1, 8, 2, 257, 100, 64), (1, 8, 2, 4, 0, 64),
              (1, 8, 2, 4, 100, 96), (1 << 20, 8, 2, 4, 100, 64)):
        assert tree(*a) == 0 and capi.tree_attention_paged_call_workspace_bytes(*a) == 0
    for a in ((0, 8, 2, 100, 16, 4, 64), (1, 8, 3, 100, 16, 4, 64), (1, 8, 2, 0, 16, 4, 64), (1, 8, 2, 100, 24, 4, 64),
              (1, 8, 2, 100, 16, 0, 64), (1, 8, 2, 100, 16, 4, 80)):
        assert sparse(*a) == 0 and capi.decode_paged_sparse_call_workspace_bytes(*a) == 0


def test_torch_ops_refuse_cpu_tensors(ext):
    pages, s = torch.zeros(2, 1, 16, 64, dtype=torch.int8), torch.zeros(2, 1, 16)
    i = torch.zeros(1, dtype=torch.int32)
    q, m, sm = torch.zeros(1, 2, 1, 64, dtype=torch.int8), torch.zeros(2, 1, 64, dtype=torch.int8), torch.zeros(2, 1)
    calls = [lambda: ext.qk_norm_rope_append(torch.zeros(1, 256), 2, 1, torch.zeros(9, 8), torch.zeros(9, 8), i, pages, pages,
                                             s, s, i),
             lambda: ext.int8_tree_attention_forward_paged(q, pages, pages, torch.ones(2), s, s, i.view(1, 1), i, None, 16),
             lambda: ext.kv_cache_move_paged(pages, pages, s, s, i, i),
             lambda: ext.kv_page_means(pages, s, i, m, sm),
             lambda: ext.int8_decode_attention_forward_paged_sparse(q[:, :, 0], pages, pages, torch.ones(2), s, s, m, sm,
                                                                    i.view(1, 1), i, 16, 1)]
    for call in calls:
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
