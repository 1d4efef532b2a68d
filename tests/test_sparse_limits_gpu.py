"""Sparse decode at the ends of its documented sizes (GPU)."""
import pytest
import torch

from paged_helpers import sparse_case
from test_sparse_gpu import _check, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("top", [2 ** 31 - 1, 2 ** 31 - 1024])
def test_more_blocks_asked_for_than_a_step_below_2_to_31(ext, gpu, top):
    # the entries behind the last block taken are filled by a loop whose index passes 2^31
    n = 37
    c = sparse_case(1, [16 * n], 4, 1, 64, 16, gpu, n)
    want = _run(ext, c)
    _check(c, want)
    c["top"] = top
    out, which = _run(ext, c)
    assert which.shape == (1, 1, top)
    assert torch.equal(out, want[0])
    assert (which[0, 0, :n].cpu() == torch.arange(n)).all()
    for at in range(n, top, 1 << 28):
        assert bool((which[0, 0, at:at + (1 << 28)] == -1).all())
