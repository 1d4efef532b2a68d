"""An infinite value scale: by the formula its key's contribution is p v sV, an infinity of v's
sign where v is not zero and a NaN where it is, in every row that sees the key (GPU)."""
import pytest
import torch

from grouped_helpers import kv4_case
from oracle import grouped_oracle as G
from test_kv4_gpu import _decode
from test_packed_gpu import _args, _case

pytestmark = pytest.mark.gpu


def _clamp(t):
    return t.double().nan_to_num(nan=0.0, posinf=1.0, neginf=-1.0)


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("at,causal", [(0, True), (70, True), (299, True), (70, False), (299, False)])
def test_packed(ext, gpu, at, causal, D, sign):
    c = _case([300, 40], 4, 2, D, gpu, seed=4)
    c["V"][:, at, ::5] = 0
    want = ext.int8_attention_forward_packed(*_args(c), is_causal=causal)
    c["sV"][:, at] = sign * float("inf")
    out = ext.int8_attention_forward_packed(*_args(c), is_causal=causal)
    first = at if causal else 0
    assert torch.equal(out[:, :first], want[:, :first]) and torch.equal(out[:, 300:], want[:, 300:])
    for h in range(4):
        v = c["V"][h // 2, at]
        rows = out[h, first:300]
        nan, inf = v == 0, sign * torch.sign(v.double())
        assert rows[:, nan].isnan().all()
        assert (_clamp(rows[:, ~nan]) == inf[~nan]).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,at", [(1, 0), (333, 0), (333, 40), (5000, 4999)])
def test_decode(ext, gpu, n, at, D):
    c = kv4_case(n + D, 2, 8, 2, D, 64, [n, 77], gpu)
    page, off = int(c["tables"][0, at // 64]), at % 64
    want = _decode(ext, c)
    c["sV"][page, :, off] = float("inf")
    out = _decode(ext, c)
    assert torch.equal(out[1], want[1])
    codes = torch.from_numpy(G.kv4_unpack(c["V"][page, :, off].cpu().numpy())).to(gpu)
    for h in range(8):
        v = codes[h // 4]
        nan = v == 0
        assert out[0, h, nan].isnan().all()
        assert (_clamp(out[0, h, ~nan]) == torch.sign(v[~nan].double())).all()
