"""Rows that one key dominates, with a long flat tail of small weights: where the dominant
key's value is zero the output is the tail's alone (GPU)."""
import math

import numpy as np
import pytest
import torch

from oracle import grouped_oracle as G

pytestmark = pytest.mark.gpu

GAPS = [24.6, 22.7, 20.3, 16.0, 8.0]  # log2 of the dominant weight over one of the tail's


def _expected(n, gap, tail_v):
    """The dims where the dominant value is 0 (and a key sees n tail keys)."""
    p = n * 2.0 ** -gap
    return p / (1 + p) * tail_v


def _bound(want, n, gap, tail_v, steps):
    # Scores reach 25 ln 2 < 2^5: three fp32 roundings each move a weight by 2^5 * 3 * 2^-24 <
    # 2^-17; exp2, the value scale and the weight's two fp16 stay below 2^-20 together; the sum
    # of the tail in `steps` fp32 additions loses steps * 2^-24 at most, beside a dominant
    # weight of 1 in l steps * 2^-24 of that.  A weight is off by half fp16's smallest step,
    # 2^-25, where the row's largest is 2^8 at least: 2^-33 of it a key.  One rounding to fp16.
    p = n * 2.0 ** -gap
    rel = 2.0 ** -16 + 2 * steps * 2.0 ** -24
    return rel * want + n * 2.0 ** -33 / (1 + p) * tail_v + 2.0 ** -11 * want + 2.0 ** -25


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,n", [(1, 8192), (1, 65536), (1024, 8192)])
@pytest.mark.parametrize("at", ["first", "middle", "last"])
def test_decode_flat_tail(ext, gpu, B, n, D, at):
    # one sequence is split over many waves, each with its own largest weight; a thousand (that
    # share their pages) leave a quarter of the tail to the dominant key's wave
    page, H = 64, 8
    NP = n // page
    codes = np.zeros((n, D), np.int8)
    where = {"first": 0, "middle": n // 2 + 5, "last": n - 1}[at]
    codes[where] = 7
    vals = np.ones((n, D), np.int8)
    vals[where] = 7
    vals[where, : D // 2] = 0
    to = lambda c: torch.from_numpy(G.kv4_pack(c)).view(NP, 1, page, D // 2).to(gpu)  # noqa: E731
    q = torch.full((B, H, D), 100, dtype=torch.int8, device=gpu)
    one = torch.ones(NP, 1, page, device=gpu)
    dot = 700 * D
    # head h's score of the dominant key lies gap_h log 2 above the tail's zeros
    gaps = (GAPS + GAPS)[:H]
    sq = torch.tensor([[g * math.log(2) * math.sqrt(D) / dot for g in gaps]], device=gpu)
    tables = torch.arange(NP, dtype=torch.int32, device=gpu).expand(B, NP).contiguous()
    out = ext.int8_decode_attention_forward_kv4_paged(
        q, to(codes), to(vals), sq.expand(B, H).contiguous(), one, one, tables,
        torch.full((B,), n, dtype=torch.int32, device=gpu), n)
    got = out[..., : D // 2].double().cpu()
    for h, gap in enumerate(gaps):
        want = _expected(n - 1, gap, 1.0)
        err = (got[:, h] - want).abs().max().item()
        assert err <= _bound(want, n, gap, 1.0, n // 32), (h, gap, got[0, h, 0].item(), want)


@pytest.mark.parametrize("D,n,causal", [(D, 8192, c) for D in (64, 128, 256) for c in (True, False)] + [(64, 65536, True)])
@pytest.mark.parametrize("at", ["first", "middle", "last"])
def test_packed_flat_tail(ext, gpu, n, D, causal, at):
    H = len(GAPS)
    where = {"first": 0, "middle": n // 2 + 5, "last": n - 40}[at]
    q = torch.zeros(H, n, D, dtype=torch.int8, device=gpu)
    q[:, -30:] = 100  # the queries that are looked at, all behind the dominant key
    k = torch.zeros(1, n, D, dtype=torch.int8, device=gpu)
    k[0, where] = 7
    v = torch.full((1, n, D), 10, dtype=torch.int8, device=gpu)
    v[0, where] = 70
    v[0, where, : D // 2] = 0
    sq = torch.tensor([g * math.log(2) * math.sqrt(D) / (700 * D) for g in GAPS], device=gpu)
    sq = sq.unsqueeze(1).expand(H, n).contiguous()
    one = torch.ones(1, n, device=gpu)
    out = ext.int8_attention_forward_packed(
        q, k, v, sq, one, one * 0.1, torch.tensor([0, n], dtype=torch.int32, device=gpu), is_causal=causal)
    got = out[:, -30:, : D // 2].double().cpu()
    for h, gap in enumerate(GAPS):
        for i in range(30):
            seen = n - 29 + i if causal else n
            want = _expected(seen - 1, gap, 1.0)
            err = (got[h, i] - want).abs().max().item()
            assert err <= _bound(want, n, gap, 1.0, n // 16) + 2.0 ** -22 * want, (h, i, gap, got[h, i, 0].item(), want)
