"""Dims past the rotation are not rotated, whatever stands in them: an infinity or a NaN there
stays in its own element (GPU)."""
import numpy as np
import pytest
import torch

from grouped_helpers import np64, rows
from oracle import grouped_oracle as G
from test_heads_gpu import _bound, _oracle, _tables, _to

pytestmark = pytest.mark.gpu

# head_dim, rot_dim, interleaved: halves in whole chunks, pairs, halves element by element
LAYOUTS = [(64, 32, False), (128, 64, False), (64, 32, True), (128, 96, True), (80, 40, False),
           (96, 6, False), (96, 6, True), (256, 128, False)]


def _case(D, rot, dt):
    g = torch.Generator().manual_seed(D + rot)
    x = rows(g, 1, 40, 6 * D).to(dt)  # 4 query heads, 1 key head, 1 value head
    cos, sin = _tables(rot // 2)
    pos = torch.arange(40, dtype=torch.int32).unsqueeze(0) * 7
    return x, cos, sin, pos


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,rot,inter", LAYOUTS)
def test_unrotated_dims_pass_through(ext, gpu, D, rot, inter, dt, bad):
    x, cos, sin, pos = _case(D, rot, dt)
    heads = x.view(40, 6, D)
    heads[30:, :, rot:] = -0.0
    at = {(1 + 3 * i): d for i, d in enumerate(range(rot, D, -(-(D - rot) // 10)))}
    for t, d in at.items():
        heads[t, t % 5, d] = bad  # a query or the key head
    args = _to(gpu, x, cos, sin, pos)
    got = ext.qk_norm_rope(args[0], 4, 1, *args[1:], interleaved=inter)
    ref = _oracle(x, 4, 1, cos, sin, pos, None, None, inter)
    for i in range(2):
        out = got[i].cpu()
        # the unrotated dims are x's own bits
        want = heads[:, 4 * i:4 * i + (4, 1)[i], rot:].transpose(0, 1)
        assert torch.equal(out[0, ..., rot:].isnan(), want.isnan())
        assert torch.equal(out[0, ..., rot:].nan_to_num(), want.nan_to_num())
        assert torch.equal(out[0, ..., rot:].signbit(), want.signbit())
        # and the rotated ones what they are without the bad element
        turned = np64(out)[..., :rot]
        bound = _bound(ref[i], D, rot // 2, inter, dt, True)[..., :rot]
        assert (np.abs(turned - ref[i][..., :rot]) <= bound).all()


@pytest.mark.parametrize("D,rot,inter", LAYOUTS)
def test_unrotated_infinity_under_a_norm(ext, gpu, D, rot, inter):
    # the row's root is infinite: the element itself is NaN and every other one 0
    x, cos, sin, pos = _case(D, rot, torch.float32)
    x.view(40, 6, D)[5, 2, D - 1] = float("inf")
    w = torch.ones(D)
    args = _to(gpu, x, cos, sin, pos)
    q = ext.qk_norm_rope(args[0], 4, 1, *args[1:], q_weight=w.to(gpu), k_weight=w.to(gpu),
                         interleaved=inter)[0][0].cpu()
    with np.errstate(invalid="ignore"):
        ref = G.norm_rope(np64(x.view(40, 6, D)[5, 2]), cos[35].numpy(), sin[35].numpy(), w.numpy(),
                          1e-6, inter)
    assert np.isnan(ref[-1]) and (ref[:-1] == 0).all()
    assert torch.isnan(q[2, 5, -1]) and (q[2, 5, :-1] == 0).all()
    q[2, 5] = 0
    assert torch.isfinite(q).all()


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,rot,inter", LAYOUTS + [(64, 64, False), (128, 128, True), (80, 80, False)])
def test_quantized_rows_of_non_finite_heads(ext, gpu, D, rot, inter, dt, bad):
    # an infinity makes its row's scale infinite and every finite code 0, as the per-token
    # quantizer has it, byte for byte
    x, cos, sin, pos = _case(D, rot, dt)
    for t in range(6):
        x.view(40, 6, D)[6 * t + 1, t, (7 * t + D - 1) % D] = bad
    args = _to(gpu, x, cos, sin, pos)
    got = ext.qk_norm_rope(args[0], 4, 1, *args[1:], interleaved=inter)
    q = ext.qk_norm_rope_quantize(args[0], 4, 1, *args[1:], interleaved=inter)
    for i in range(3):
        c, s = ext.quantize_per_token(got[i])
        assert torch.equal(q[2 * i], c), "qkv"[i]
        assert torch.equal(q[2 * i + 1].isnan(), s.isnan())
        assert torch.equal(q[2 * i + 1].nan_to_num(), s.nan_to_num()), "qkv"[i]
