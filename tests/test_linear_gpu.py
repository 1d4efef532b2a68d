"""int8_linear against the 64-bit oracle (GPU): shapes around every tile and route edge, both
weight layouts, output types, scalar scales, bias; graph capture and streams."""
import numpy as np
import pytest
import torch

from grouped_helpers import HALF, TINY, assert_within, np64, quantize_rows, rows
from oracle import grouped_oracle as G

pytestmark = pytest.mark.gpu


def _case(T, K, N, seed=0):
    g = torch.Generator().manual_seed(seed + T + 3 * K + 7 * N)
    x, sx = quantize_rows(rows(g, T, K))
    wt, sw = quantize_rows(torch.randn(N, K, generator=g) * 0.02)
    return x, wt.t().contiguous(), sx, sw, torch.randn(N, generator=g)


def _bound(ref, mag, bias, dt):
    # fp32: conversion of the sum, two products, the bias sum (each 2^-24 of what it rounds)
    b = 0 if bias is None else np.abs(np64(bias))
    f32 = 4 * 2.0 ** -24 * (mag + b)
    return f32 + HALF[dt] * (np.abs(ref) + f32) + TINY[dt]


def _check(ext, gpu, T, K, N, dt, packed, bias, scalar=False, seed=0):
    x, w, sx, sw, b = _case(T, K, N, seed)
    if scalar:
        sx, sw = sx[:1].clone(), sw[:1].clone()
    b = b if bias else None
    W = w.t().contiguous() if packed else w
    y = ext.int8_linear(x.to(gpu), W.to(gpu), sx.to(gpu), sw.to(gpu),
                        bias=b.to(gpu) if bias else None, prepacked=packed, dtype=dt)
    torch.cuda.synchronize()
    assert y.shape == (T, N) and y.dtype == dt
    ref, mag = G.linear(x.numpy(), w.numpy(), sx.numpy(), sw.numpy(), b.numpy() if bias else None)
    assert_within(np64(y), ref, _bound(ref, mag, b, dt), f"T{T} K{K} N{N} {dt} packed={packed}")


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("T", [1, 2, 15, 31, 32, 33, 64, 127, 128, 129, 257, 512, 1000])
@pytest.mark.parametrize("K,N", [(16, 16), (512, 768), (1040, 528)])
def test_linear_shapes(ext, gpu, T, K, N, packed):
    _check(ext, gpu, T, K, N, torch.float16, packed, bias=T % 2 == 0)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("T,K,N", [(1, 4096, 2048), (40, 2048, 6144), (300, 2048, 1536),
                                   (2049, 1024, 1280), (1536, 2064, 4096), (4100, 512, 2320)])
def test_linear_types_and_routes(ext, gpu, T, K, N, packed, dt):
    _check(ext, gpu, T, K, N, dt, packed, bias=packed)


@pytest.mark.parametrize("T", [3, 200, 3000])
def test_linear_scalar_scales(ext, gpu, T):
    _check(ext, gpu, T, 1024, 1024, torch.bfloat16, True, bias=False, scalar=True)


@pytest.mark.parametrize("T,N", [(7, 512), (500, 512), (3000, 2048)])
def test_linear_extreme_codes(ext, gpu, T, N):
    # every product at its largest: the int32 sum of K = 131056 of 2^14 stays below 2^31
    K = 131056 if T < 10 else 16400
    x = torch.full((T, K), -128, dtype=torch.int8, device=gpu)
    w = torch.full((N, K), -128, dtype=torch.int8, device=gpu)
    one = torch.ones(1, device=gpu)
    y = ext.int8_linear(x, w, one, one, prepacked=True, dtype=torch.float32)
    assert torch.equal(y, torch.full((T, N), float(K * 16384), device=gpu))


def test_linear_leading_dims_and_views(ext, gpu):
    x, w, sx, sw, _ = _case(24, 512, 256)
    ref, mag = G.linear(x.numpy(), w.numpy(), sx.numpy(), sw.numpy())
    wide = torch.zeros(24, 1024, dtype=torch.int8)
    wide[:, 256:768] = x
    base = torch.zeros(24 * 512 + 3, dtype=torch.int8)
    base[3:] = x.reshape(-1)
    for view in (x.to(gpu).view(2, 3, 4, 512), wide.to(gpu)[:, 256:768],
                 base.to(gpu)[3:].view(24, 512)):
        y = ext.int8_linear(view, w.to(gpu), sx.to(gpu), sw.to(gpu))
        assert y.shape == view.shape[:-1] + (256,)
        assert_within(np64(y).reshape(24, 256), ref, _bound(ref, mag, None, torch.float16))


def test_linear_non_finite_scales_stay_in_their_rows(ext, gpu):
    x, w, sx, sw, _ = _case(300, 1024, 1024)
    sx[7], sx[8] = float("nan"), float("inf")
    y = ext.int8_linear(x.to(gpu), w.to(gpu), sx.to(gpu), sw.to(gpu)).cpu()
    assert torch.isnan(y[7]).all() and not torch.isfinite(y[8]).any()
    keep = torch.ones(300, dtype=torch.bool)
    keep[7:9] = False
    assert torch.isfinite(y[keep]).all()


@pytest.mark.parametrize("T", [1, 100, 700])
def test_linear_graph_replay_and_streams(ext, gpu, T):
    x, w, sx, sw, _ = (t.to(gpu) for t in _case(T, 1024, 512))
    want = ext.int8_linear(x, w, sx, sw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ext.int8_linear(x, w, sx, sw)
    side.synchronize()
    assert torch.equal(got, want)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        y1 = ext.int8_linear(x, w, sx, sw)
    with torch.cuda.graph(g2):
        y2 = ext.int8_linear(x, w, sx, sw)
    for i in range(3):
        x.copy_(x.flip(0))
        eager = ext.int8_linear(x, w, sx, sw)
        y1.zero_()
        y2.zero_()
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(y1, eager) and torch.equal(y2, eager), i


@pytest.mark.parametrize("T,K,N", [(2048, 2048, 6144), (1900, 1040, 6000), (2600, 1040, 3440)])
@pytest.mark.parametrize("dt", [torch.float16, torch.float32])
def test_linear_tiles_that_fill_the_last_round(ext, gpu, T, K, N, dt):
    # packed weights whose 256 x 192 tiles fit the CUs better than 256 x 256 ones, and ragged edges
    _check(ext, gpu, T, K, N, dt, packed=True, bias=True)


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("T,K,N", [(333, 2048, 2560), (300, 2064, 2576), (500, 4096, 2048), (130, 2176, 4112),
                                   (256, 3840, 4096)])
def test_linear_k_over_two_wave_groups(ext, gpu, T, K, N, packed):
    # at most 256 tiles of 64 x 64 and a long K: whole and ragged halves of it
    _check(ext, gpu, T, K, N, torch.bfloat16, packed, bias=True)
