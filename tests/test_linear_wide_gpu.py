"""int8_linear at the feed-forward and vocabulary sizes, against exact sums in float64 (GPU)."""
import pytest
import torch

from grouped_helpers import HALF, TINY

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("K,N", [(4096, 28672), (14336, 4096), (4096, 128256), (2048, 32000), (8192, 8256)])
@pytest.mark.parametrize("T,dt", [(1, torch.float16), (16, torch.bfloat16), (64, torch.float16), (200, torch.float32)])
def test_linear_wide(ext, gpu, T, K, N, packed, dt):
    g = torch.Generator(device=gpu).manual_seed(T + K + N)
    x = torch.randint(-128, 128, (T, K), dtype=torch.int8, device=gpu, generator=g)
    w = torch.randint(-128, 128, (N, K) if packed else (K, N), dtype=torch.int8, device=gpu, generator=g)
    sx, sw = (torch.rand(n, device=gpu, generator=g) * 0.01 + 1e-4 for n in (T, N))
    b = torch.randn(N, device=gpu, generator=g)
    y = ext.int8_linear(x, w, sx, sw, bias=b, prepacked=packed, dtype=dt)
    ref = torch.empty(T, N, dtype=torch.float64, device=gpu)
    for n0 in range(0, N, 16384):  # integer sums in float64 are exact
        n1 = min(N, n0 + 16384)
        part = w[n0:n1].double().t().contiguous() if packed else w[:, n0:n1].double()
        ref[:, n0:n1] = x.double() @ part
    ref = ref * sx.double().unsqueeze(1) * sw.double()
    # the sum's conversion, two products and the bias: 2^-24 each of what they round
    f32 = 4 * 2.0 ** -24 * (ref.abs() + b.double().abs())
    ref += b.double()
    over = (y.double() - ref).abs() - (f32 + HALF[dt] * (ref.abs() + f32) + TINY[dt])
    assert torch.isfinite(y).all() and over.max().item() <= 0


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("K,N", [(4096, 2048), (1040, 6000), (512, 16400)])
def test_rows_do_not_depend_on_the_route(ext, gpu, K, N, packed):
    # the sum is exact and its value one expression: a row's bits are those of a call of its own
    g = torch.Generator(device=gpu).manual_seed(K)
    T = 2500
    x = torch.randint(-128, 128, (T, K), dtype=torch.int8, device=gpu, generator=g)
    w = torch.randint(-128, 128, (N, K) if packed else (K, N), dtype=torch.int8, device=gpu, generator=g)
    sx, sw = (torch.rand(n, device=gpu, generator=g) * 0.01 for n in (T, N))
    b = torch.randn(N, device=gpu, generator=g)
    want = ext.int8_linear(x, w, sx, sw, bias=b, prepacked=packed, dtype=torch.float32)
    for n in (1, 20, 64, 130, 333, 512, 700, 1500):
        y = ext.int8_linear(x[-n:], w, sx[-n:], sw, bias=b, prepacked=packed, dtype=torch.float32)
        assert torch.equal(y, want[-n:]), n
