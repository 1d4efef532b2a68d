"""Packed prompts whose sequence bounds leave the tokens or fall (GPU)."""
import pytest
import torch

import int8k_capi as capi
from test_packed_gpu import _args, _case, _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("cu,cut", [([0, 500], [0, 100]), ([-7, 30, 100], [0, 30, 100]),
                                    ([-9, -3, 40, 2 ** 31 - 1], [0, 0, 40, 100]),
                                    ([100, 400], [100, 100]), ([-2 ** 31, 100], [0, 100])])
def test_bounds_are_cut_to_the_tokens(ext, gpu, cu, cut, causal):
    c = _case([100], 4, 2, 64, gpu)
    c["cu"] = torch.tensor(cu, dtype=torch.int32, device=gpu)
    out = ext.int8_attention_forward_packed(*_args(c), is_causal=causal)
    c["cu"] = torch.tensor(cut, dtype=torch.int32, device=gpu)
    assert torch.equal(out, ext.int8_attention_forward_packed(*_args(c), is_causal=causal))
    _check(c, out, causal)


@pytest.mark.parametrize("zero_rest", [False, True])
@pytest.mark.parametrize("thd", [False, True])
@pytest.mark.parametrize("cu", [[0, 50, 20, 100], [90, 10], [100, 0, 100, 0, 100], [0, 300, -5, 70]])
def test_falling_bounds_write_nothing_outside(ext, gpu, cu, thd, zero_rest):
    c = _case([100], 4, 2, 64, gpu)
    c["cu"] = torch.tensor(cu, dtype=torch.int32, device=gpu)
    n = 100 * 4 * 64
    held = torch.full((3 * n,), 7.0, dtype=torch.float16, device=gpu)
    out = held[n:2 * n].view((100, 4, 64) if thd else (4, 100, 64))
    capi.attention_forward_packed(*_args(c), causal=True, out_thd=thd, zero_rest=zero_rest, out=out)
    assert (held[:n] == 7).all() and (held[2 * n:] == 7).all()
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("scale", [2.0 ** 14, float("inf"), float("nan")])
@pytest.mark.parametrize("at", [100, 129, 191, 260])
def test_later_value_scales_do_not_reach_earlier_queries(ext, gpu, at, scale, D):
    # neither as values nor as another order of rounding: bit for bit
    c = _case([300, 30], 4, 2, D, gpu, seed=3)
    want = ext.int8_attention_forward_packed(*_args(c), is_causal=True)
    c["sV"][:, at:at + 20] *= scale
    out = ext.int8_attention_forward_packed(*_args(c), is_causal=True)
    assert torch.equal(out[:, :at], want[:, :at])
    assert torch.equal(out[:, 300:], want[:, 300:])


def test_as_many_sequences_as_there_may_be(ext, gpu):
    # 65536 of them, most empty, one long; more bounds than tokens in the second call
    lens = torch.zeros(65536, dtype=torch.int32)
    lens[::9] = 1
    lens[5000] = 900
    for keep in (65536, 4000):
        part = lens.clone()
        part[keep:] = 0
        T = int(part.sum())
        c = _case([T], 2, 1, 16, gpu, seed=keep)
        c["cu"] = torch.cat((torch.zeros(1, dtype=torch.int32), part.cumsum(0).to(torch.int32))).to(gpu)
        out = ext.int8_attention_forward_packed(*_args(c), is_causal=True)
        _check(c, out, True, str(keep))
