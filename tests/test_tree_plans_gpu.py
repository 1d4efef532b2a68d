"""Attention of drafted trees with every kernel that a plan picks from, whole sequences and cut ones,
at both head dims (GPU) against the 64-bit oracle."""
import pytest
import torch

import int8k_capi as capi
from paged_helpers import tree_case
from paged_plans import CASES
from test_tree_gpu import _check, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kernel,size", CASES)
def test_every_kernel(ext, gpu, kernel, size):
    D, (B, G, N, Hkv, top) = kernel[0], size
    g = torch.Generator().manual_seed(B + N + D)
    # one sequence of the whole length, an empty one, the others anything between
    lens = [top - N] + torch.randint(0, top - N, (B - 1,), generator=g).tolist()
    counts = [N] + torch.randint(0, N + 1, (B - 1,), generator=g).tolist()
    if B > 2:
        lens[-1] = 0
    c = tree_case(B + N + D, lens, N, G * Hkv, Hkv, D, 16 if top % 2 else 64, gpu, counts=counts, top=top)
    before = capi.paged_bad_ids()
    out = _run(ext, c)
    _check(c, out)
    assert capi.paged_bad_ids() == before
    assert torch.equal(_run(ext, c, True), out.transpose(1, 2))
    assert torch.equal(_run(ext, c), out)
