"""An infinite value scale: by the formula its key's contribution is p v sV, an infinity of v's
sign where v is not zero and a NaN where it is, in every row that sees the key (GPU)."""
import pytest
import torch

from grouped_helpers import kv4_case
from oracle import grouped_oracle as G
from test_kv4_gpu import _decode

pytestmark = pytest.mark.gpu


def _clamp(t):
    return t.double().nan_to_num(nan=0.0, posinf=1.0, neginf=-1.0)


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
