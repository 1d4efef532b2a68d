"""An infinite value scale in the INT8 paged cache: its key's contribution p v sV is an infinity of
v's sign where v is not zero and a NaN where it is, in every row that sees the key and in no other
(GPU).  With every kernel that a plan picks from, whole sequences and cut ones."""
import pytest
import torch

from paged_helpers import sparse_case, tree_case, words_of
from test_sparse_gpu import _run as _sparse
from test_tree_gpu import _run

pytestmark = pytest.mark.gpu


def _clamp(t):
    return t.double().nan_to_num(nan=0.0, posinf=1.0, neginf=-1.0)


def _holds(rows, v, sign):
    """rows [..., D] that see a key of codes v [D] with the value scale sign * infinity."""
    nan, inf = v == 0, sign * torch.sign(v.double())
    assert rows[..., nan].isnan().all()
    assert (_clamp(rows[..., ~nan]) == inf[~nan]).all()


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,N,H,Hkv,L,at", [
    (2, 1, 4, 4, 1, 0), (3, 5, 8, 2, 333, 40), (3, 5, 8, 2, 333, 332), (2, 16, 4, 1, 9000, 4444), (3, 17, 4, 2, 200, 0),
    (33, 50, 4, 2, 250, 100), (33, 43, 12, 4, 257, 256), (12, 100, 12, 12, 600, 599), (33, 256, 4, 4, 744, 31),
    (5, 50, 32, 4, 1450, 1000), (2, 50, 64, 8, 8950, 0)])
def test_tree(ext, gpu, B, N, H, Hkv, L, at, D, sign):
    lens = [L] + [max(1, L - 40 * b) for b in range(1, B)]
    c = tree_case(N + L, lens, N, H, Hkv, D, 32, gpu)
    p, off = int(c["tables"][0, at // 32]), at % 32
    c["V"][p, :, off, ::5] = 0
    want = _run(ext, c)
    c["sV"][p, :, off] = sign * float("inf")
    out = _run(ext, c)
    assert torch.equal(out[1:], want[1:])
    for h in range(Hkv):
        _holds(out[0, h * (H // Hkv):(h + 1) * (H // Hkv)], c["V"][p, h, off], sign)


@pytest.mark.parametrize("D", [64, 128])
def test_a_node(ext, gpu, D):
    # only the rows that see the node, with one fragment and with two
    for N, H in ((6, 4), (20, 8)):
        c = tree_case(N, [40], N, H, 2, D, 16, gpu)
        sees = [{i} | ({2} if i % 3 == 0 else set()) for i in range(N)]
        c["mask"] = words_of(sees, N).to(gpu)
        p, off = int(c["tables"][0, 42 // 16]), 42 % 16
        c["V"][p, :, off, ::7] = 0
        want = _run(ext, c)
        c["sV"][p, 1, off] = float("inf")
        out = _run(ext, c)
        assert torch.equal(out[:, :H // 2], want[:, :H // 2])
        for i in range(N):
            if 2 in sees[i]:
                _holds(out[0, H // 2:, i], c["V"][p, 1, off], 1.0)
            else:
                assert torch.isfinite(out[0, H // 2:, i]).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("L,top", [(16 * 30, 100), (16 * 2000, 1500)])
def test_sparse(ext, gpu, L, top, D):
    c = sparse_case(L + D, [L, 333], 8, 2, D, 16, gpu, top)
    p = int(c["tables"][0, L // 16 - 1])  # the last block is always taken
    c["V"][p, :, 3, ::5] = 0
    want = _sparse(ext, c)
    c["sV"][p, :, 3] = float("inf")
    out, which = _sparse(ext, c)
    assert torch.equal(which, want[1]) and torch.equal(out[1], want[0][1])
    for h in range(2):
        _holds(out[0, 4 * h:4 * h + 4], c["V"][p, h, 3], 1.0)


@pytest.mark.parametrize("gap", [200.0, 2000.0])
def test_no_component_is_finite_however_small_the_weight(ext, gpu, gap):
    # a weight below fp32's range: the product with infinity is a NaN, never a finite number
    c = tree_case(3, [700], 4, 8, 2, 64, 16, gpu, mask=None)
    c["Q"].fill_(10), c["sQ"].fill_(1.0)
    for at, score in ((300, gap), (10, 0.0), (650, 0.0)):
        p, off = int(c["tables"][0, at // 16]), at % 16
        c["K"][p, :, off], c["sK"][p, :, off] = 1, score * 8 / 640
        if at != 300:
            c["sV"][p, :, off] = float("inf")
    assert not torch.isfinite(_run(ext, c)).any()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,N,H,Hkv,L,at", [(3, 5, 8, 2, 333, 40), (2, 16, 4, 1, 9000, 4444), (33, 43, 12, 4, 257, 256),
                                            (5, 50, 32, 4, 1450, 1000)])
def test_value_scales_of_2_to_64(ext, gpu, B, N, H, Hkv, L, at, D):
    # the largest that are taken: past fp16's range where the code is not zero, finite where it is
    lens = [L] + [max(1, L - 40 * b) for b in range(1, B)]
    c = tree_case(N + L, lens, N, H, Hkv, D, 32, gpu)
    p, off = int(c["tables"][0, at // 32]), at % 32
    c["V"][p, :, off, ::5] = 0
    c["sV"][p, :, off] = 2.0 ** 64
    out = _run(ext, c)
    for h in range(Hkv):
        v = c["V"][p, h, off]
        rows = out[0, h * (H // Hkv):(h + 1) * (H // Hkv)]
        assert torch.isfinite(rows[..., v == 0]).all()
        assert (rows[..., v != 0].double() == torch.sign(v[v != 0].double()) * float("inf")).all()
