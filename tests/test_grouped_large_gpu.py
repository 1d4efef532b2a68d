"""The grouped-query operators on tensors whose offsets pass 32 bits (GPU): the last rows of a
large call equal those of a small one, bit for bit."""
import pytest
import torch

from grouped_helpers import quantize_rows, rows
from test_heads_gpu import _tables

pytestmark = pytest.mark.gpu


def test_linear_output_past_32_bits(ext, gpu):
    T, K, N = 300_000, 16, 16384  # 4.9 G outputs
    g = torch.Generator().manual_seed(1)
    x = torch.zeros(T, K, dtype=torch.int8, device=gpu)
    tail, sx = quantize_rows(rows(g, 70, K))
    x[-70:] = tail.to(gpu)
    scale = torch.ones(T, device=gpu)
    scale[-70:] = sx.to(gpu)
    w, sw = quantize_rows(torch.randn(N, K, generator=g))
    y = ext.int8_linear(x, w.to(gpu), scale, sw.to(gpu), prepacked=True)
    want = ext.int8_linear(x[-70:], w.to(gpu), scale[-70:], sw.to(gpu), prepacked=True)
    assert torch.equal(y[-70:], want)
    assert not y[:1000].any() and not y[T // 2:T // 2 + 1000].any()


@pytest.mark.parametrize("quantized", [False, True])
def test_heads_past_32_bits(ext, gpu, quantized):
    T, H, Hkv, D = 360_000, 32, 8, 128  # 2.2 G elements, 4.4 GB in
    g = torch.Generator().manual_seed(2)
    x = torch.zeros(T, (H + 2 * Hkv) * D, dtype=torch.bfloat16, device=gpu)
    x[-5:] = rows(g, 5, x.shape[1]).to(torch.bfloat16).to(gpu)
    cos, sin = (t.to(gpu) for t in _tables(D // 2))
    pos = (torch.arange(T, device=gpu) % 600).to(torch.int32)
    w = torch.rand(D, generator=g).to(gpu)
    f = ext.qk_norm_rope_quantize if quantized else ext.qk_norm_rope
    got = f(x, H, Hkv, cos, sin, pos, q_weight=w, k_weight=w)
    want = f(x[-5:].clone(), H, Hkv, cos, sin, pos[-5:].clone(), q_weight=w, k_weight=w)
    for a, b in zip(got, want):
        assert torch.equal(a[:, -5:], b)


def test_packed_past_32_bits(ext, gpu):
    n, L, H, D = 8000, 130, 36, 128  # queries of 4.8 GB, outputs of 9.6 GB
    T = n * L
    g = torch.Generator(device=gpu).manual_seed(3)
    Q = torch.zeros(H, T, D, dtype=torch.int8, device=gpu)
    Q[:, -2 * L:] = torch.randint(-127, 128, (H, 2 * L, D), dtype=torch.int8, device=gpu, generator=g)
    K, V = (torch.randint(-127, 128, (1, T, D), dtype=torch.int8, device=gpu, generator=g) for _ in range(2))
    sQ, sK, sV = (torch.rand(h, T, device=gpu, generator=g) * 0.02 + 0.001 for h in (H, 1, 1))
    cu = (torch.arange(n + 1, device=gpu) * L).to(torch.int32)
    out = ext.int8_attention_forward_packed(Q, K, V, sQ, sK, sV, cu, is_causal=True)
    tail = [t[:, -2 * L:].contiguous() for t in (Q, K, V, sQ, sK, sV)]
    want = ext.int8_attention_forward_packed(*tail, cu[:3].clone(), is_causal=True)
    assert torch.equal(out[:, -2 * L:], want)
