"""Attention over packed prompts and 4-bit decode carry their weights in two fp16 and everything
else in fp32: held to that, not to one fp16 a weight (GPU)."""
import numpy as np
import pytest
import torch

from grouped_helpers import assert_within, kv4_case, np64
from oracle import grouped_oracle as G
from test_kv4_gpu import _decode
from test_packed_gpu import _args, _case, _oracle

pytestmark = pytest.mark.gpu


def _bound(ref, mag, keys, vmax, smax):
    """Error of a row against float64, mag = sum p|v|, smax >= |score| log2 e.
    * A score is three fp32 roundings (two scales, the exponent's sum): smax * 3 * 2^-24 of p;
      exp2 and the product with the value scale 2^-22 together, in p's sum as in its product.
    * A weight in two fp16: 2^-22 of it, or half fp16's smallest step, 2^-25, beside a largest
      weight of 2^8 at least: 2^-33 of that, a key of code vmax.
    * fp32 sums: one rounding, 2^-24, per step of 16 keys, and 8 steps to join lanes, waves and
      splits, of O and of l; the quotient 2^-23.
    * One rounding to fp16: 2^-11, or half its smallest step."""
    f32 = 2 * (smax * 3 * 2.0 ** -24 + 2.0 ** -22) + 2 * (keys / 16 + 8) * 2.0 ** -24 + 2.0 ** -23
    inner = (f32 + 2.0 ** -22) * mag + keys * 2.0 ** -33 * vmax
    return inner + 2.0 ** -11 * (np.abs(ref) + inner) + 2.0 ** -25


def _smax(Q, sQ, K, sK, D):
    """|q . k| sQ sK / sqrt(D) log2 e is at most the product of the norms."""
    qn = (Q.double().norm(dim=-1) * sQ).max().item()
    kn = (K.double().norm(dim=-1) * sK).max().item()
    return qn * kn / D ** 0.5 * 1.4427


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,Hkv,D", [(12, 12, 64), (8, 2, 128), (4, 2, 256), (3, 3, 80)])
@pytest.mark.parametrize("lens", [[30, 70, 1, 0, 55], [257, 3, 700, 0, 33, 256], [2100]])
def test_packed_precision(ext, gpu, lens, H, Hkv, D, causal):
    c = _case(lens, H, Hkv, D, gpu, seed=17)
    out = ext.int8_attention_forward_packed(*_args(c), is_causal=causal)
    ref, mag = _oracle(c, causal)
    vmax = float((c["V"].float().abs().amax(-1) * c["sV"]).max())
    smax = _smax(c["Q"], c["sQ"], c["K"], c["sK"], D)
    assert_within(np64(out), ref, _bound(ref, mag, max(lens), vmax, smax), f"{lens} D{D}")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,H,Hkv,L", [(1, 8, 2, 1000), (7, 16, 4, 777), (2, 12, 12, 5000), (300, 8, 4, 400)])
def test_decode_precision(ext, gpu, B, H, Hkv, L, D):
    lens = [max(1, L - 3 * b) for b in range(B)]
    c = kv4_case(B + L, B, H, Hkv, D, 32, lens, gpu)
    out = _decode(ext, c)
    ref, mag = G.kv4_decode(*(c[k].cpu().numpy() for k in ("Q", "K", "V", "sQ", "sK", "sV", "tables", "lens")))
    vmax = float(7 * c["sV"].max())
    k = torch.from_numpy(G.kv4_unpack(c["K"].cpu().numpy()))
    smax = _smax(c["Q"], c["sQ"], k.to(gpu), c["sK"], D)
    assert_within(np64(out), ref, _bound(ref, mag, L, vmax, smax), f"B{B} D{D}")


@pytest.mark.parametrize("D", [64, 128])
def test_decode_under_other_plans(ext, gpu, D):
    # the plan, and with it the order of the sums, follows max_context and the batch; the result
    # stays within the bound of the one value
    c = kv4_case(21 + D, 3, 8, 2, D, 64, [5, 300, 411], gpu)
    ref, mag = G.kv4_decode(*(c[k].cpu().numpy() for k in ("Q", "K", "V", "sQ", "sK", "sV", "tables", "lens")))
    k = torch.from_numpy(G.kv4_unpack(c["K"].cpu().numpy()))
    bound = _bound(ref, mag, 411, float(7 * c["sV"].max()), _smax(c["Q"], c["sQ"], k.to(gpu), c["sK"], D))
    wide = torch.full((3, 1000), -1, dtype=torch.int32, device=gpu)
    wide[:, :c["tables"].shape[1]] = c["tables"]
    for top in (411, 1000, 4096, 64000):
        assert_within(np64(_decode(ext, dict(c, tables=wide, max_context=top))), ref, bound, f"max_context {top}")
    many = {n: c[n].repeat(*([100] + [1] * (c[n].dim() - 1))) for n in ("Q", "sQ", "tables", "lens")}
    out = np64(_decode(ext, dict(c, **many))).reshape(100, 3, 8, D)
    for i in range(100):
        assert_within(out[i], ref, bound, f"batch {i}")
