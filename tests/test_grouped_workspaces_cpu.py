"""Workspace sizes of the grouped-query serving entry points, without a GPU."""
import pytest

PACKED = 1


@pytest.mark.parametrize("K,N", [(4096, 28672), (4096, 128256), (8192, 28672)])
def test_linear_reads_wide_stored_weights_on_a_route_that_streams_them(capi, K, N):
    # One token against weights as stored: the tiles of 64 columns read 64 bytes a row and are
    # slower than the routes that stream whole lines or split K, which leave partials.
    assert capi.linear_workspace_bytes(1, K, N) >= N * 4
