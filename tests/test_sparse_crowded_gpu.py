"""Selection where the scores crowd: one far score stretches the range, so that most of the others
share one of the 256 equal bins between the smallest and the largest (GPU)."""
import numpy as np
import pytest
import torch

from oracle import paged_oracle as P
from paged_helpers import sparse_case
from test_sparse_gpu import _check, _run

pytestmark = pytest.mark.gpu


def _crowd(c, b, h, n, top):
    """How many scores share the bin of the last block taken, and how many lie above it."""
    G = c["Q"].shape[1] // c["K"].shape[1]
    ids = c["tables"][b, :n].long().cpu().numpy()
    q, sq = (c[k][b, h * G:(h + 1) * G].cpu().numpy() for k in ("Q", "sQ"))
    score, nan = P.block_scores(q, sq, c["M"].cpu().numpy()[ids, h], c["sM"].cpu().numpy()[ids, h])
    score = score[:-1]
    assert not nan.any() and score.max() > score.min()
    bins = np.minimum((score - score.min()) * (256 / (score.max() - score.min())), 255).astype(int)
    last = np.sort(bins)[::-1][top - 2]
    return int((bins == last).sum()), int((bins > last).sum())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (8, 2)])
@pytest.mark.parametrize("n,top,far", [(1100, 300, 1), (2500, 1400, 1), (2500, 700, 3), (1500, 2, -1), (4000, 257, -1), (1025, 1024, 5)])
@pytest.mark.parametrize("ties", [False, True])
def test_most_scores_share_a_bin(ext, gpu, n, top, far, H, Hkv, D, ties):
    # far: so many scores far above the others; below them: one, so that the others share the top bin
    c = sparse_case(n + top + D, [16 * n - 3, 16 * (n // 2)], H, Hkv, D, 16, gpu, top)
    g = torch.Generator().manual_seed(n)
    ids = c["tables"][0, :n].long()
    if ties:  # few different means
        c["M"].copy_(c["M"][torch.randint(0, 7, (c["M"].shape[0],), generator=g).to(gpu)])
        c["sM"].fill_(0.01)
    if far < 0:
        c["Q"][0] = c["Q"][0, 0].clone()  # of the group's scores the largest counts: all far below
    for h in range(Hkv):
        q = c["Q"][0, h * (H // Hkv)].int()
        for i in torch.randperm(n - 1, generator=g)[:abs(far)].tolist():
            c["M"][ids[i], h] = (q if far > 0 else -q).clamp(-127, 127).to(torch.int8)
            c["sM"][ids[i], h] = 1e5
    for h in range(Hkv):
        crowd, above = _crowd(c, 0, h, n, top)
        assert crowd > 256 and (above > 0 or far < 0), (crowd, above)
    _check(c, _run(ext, c))


def test_crowds_inside_crowds(ext, gpu):
    # scores at five scales, so that the digits decide one after the other, and ties at the border
    n, top = 3000, 1111
    c = sparse_case(9, [16 * n], 1, 1, 64, 16, gpu, top)
    c["M"].copy_(c["M"][:1].expand_as(c["M"]).clone())
    c["Q"].copy_(c["M"][0, 0].expand_as(c["Q"]))
    g = torch.Generator().manual_seed(4)
    steps = torch.randint(0, 300, (c["sM"].numel(),), generator=g, dtype=torch.int32)
    scales = (torch.full((c["sM"].numel(),), 0.01).view(torch.int32) + steps).view(torch.float32)
    ids = c["tables"][0, :n].long().cpu()
    for k, x in enumerate((1e6, 1e4, 1e2, 1.0)):
        scales[ids[100 * k:100 * k + 40 * k + 1]] = x
    c["sM"].copy_(scales.view(c["sM"].shape))
    crowd, above = _crowd(c, 0, 0, n, top)
    assert crowd > 256 and above > 0
    _check(c, _run(ext, c))
