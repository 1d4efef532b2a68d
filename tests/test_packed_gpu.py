"""Attention over packed prompts with grouped heads against the 64-bit oracle (GPU)."""
import numpy as np
import pytest
import torch

import int8k_capi as capi
from grouped_helpers import assert_within, attention_bound, np64, quantize_rows, rows
from oracle import grouped_oracle as G

pytestmark = pytest.mark.gpu


def _case(lens, H, Hkv, D, gpu, seed=0, tail=0, front=0):
    g = torch.Generator().manual_seed(seed + sum(lens) + D)
    T = front + sum(lens) + tail
    cu = torch.tensor([front] + [front + int(v) for v in np.cumsum(lens)], dtype=torch.int32)
    c = dict(cu=cu.to(gpu))
    for n, h in (("Q", H), ("K", Hkv), ("V", Hkv)):
        q, s = quantize_rows(rows(g, h, T, D))
        c[n], c["s" + n] = q.to(gpu), s.to(gpu)
    return c


def _args(c):
    return c["Q"], c["K"], c["V"], c["sQ"], c["sK"], c["sV"], c["cu"]


def _oracle(c, causal):
    return G.packed_attention(*(c[k].cpu().numpy() for k in ("Q", "K", "V", "sQ", "sK", "sV", "cu")),
                              causal)


def _check(c, out, causal, label=""):
    ref, mag = _oracle(c, causal)
    longest = int((c["cu"][1:] - c["cu"][:-1]).max())
    vmax = float((c["V"].float().abs().amax(-1) * c["sV"]).max())
    assert_within(np64(out), ref, attention_bound(ref, mag, longest, vmax), label)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,Hkv,D", [(12, 12, 64), (8, 2, 128), (6, 1, 64), (4, 2, 256), (3, 3, 80),
                                     (6, 2, 96), (2, 1, 16), (4, 4, 144)])
@pytest.mark.parametrize("lens", [[1], [0, 5, 0], [30, 70, 1, 0, 55], [64, 128, 65, 63],
                                  [257, 3, 700, 0, 33, 256]])
def test_packed(ext, gpu, lens, H, Hkv, D, causal):
    c = _case(lens, H, Hkv, D, gpu)
    out = ext.int8_attention_forward_packed(*_args(c), is_causal=causal)
    assert out.shape == c["Q"].shape and out.dtype == torch.float16
    _check(c, out, causal, f"{lens} H{H}/{Hkv} D{D} causal={causal}")
    thd = ext.int8_attention_forward_packed(*_args(c), is_causal=causal, out_thd=True)
    assert torch.equal(thd.transpose(0, 1), out)


@pytest.mark.parametrize("n", [1, 63, 64, 65, 130, 1000])
def test_packed_many_sequences(ext, gpu, n):
    rng = np.random.default_rng(n)
    lens = [int(v) for v in rng.integers(0, 40, n)]
    lens[-1] += 300
    c = _case(lens, 4, 2, 64, gpu, seed=n)
    _check(c, ext.int8_attention_forward_packed(*_args(c), is_causal=True), True)


def test_packed_one_long_among_short(ext, gpu):
    c = _case([40] * 20 + [3000] + [17] * 50, 2, 1, 128, gpu)
    _check(c, ext.int8_attention_forward_packed(*_args(c), is_causal=True), True)


def test_packed_equals_the_batched_kernel_on_equal_lengths(ext, gpu):
    c = _case([256] * 3, 4, 4, 128, gpu)
    out = ext.int8_attention_forward_packed(*_args(c), is_causal=True)
    b = [c[k].view(4, 3, 256, -1).transpose(0, 1).contiguous() for k in ("Q", "K", "V")]
    s = [c[k].view(4, 3, 256).transpose(0, 1).contiguous() for k in ("sQ", "sK", "sV")]
    ref = ext.int8_attention_forward(*b, *s, True).transpose(0, 1).reshape(4, 768, 128)
    # each side is within its bound of the oracle, so they are within twice that of each other
    exact, mag = _oracle(c, True)
    vmax = float((c["V"].float().abs().amax(-1) * c["sV"]).max())
    assert_within(np64(out), np64(ref), 2 * attention_bound(exact, mag, 256, vmax))


@pytest.mark.parametrize("front,tail", [(0, 1), (0, 300), (5, 0), (33, 700)])
def test_packed_rows_of_no_sequence(ext, gpu, front, tail):
    c = _case([100, 0, 20], 6, 3, 80, gpu, front=front, tail=tail)
    ref, mag = _oracle(c, True)
    out = ext.int8_attention_forward_packed(*_args(c), is_causal=True)
    _check(c, out, True)  # zeros outside, as the oracle has them
    end = front + 120
    for thd in (False, True):
        held = torch.full((c["Q"].shape[1], 6, 80) if thd else c["Q"].shape, 7.0,
                          dtype=torch.float16, device=gpu)
        capi.attention_forward_packed(*_args(c), causal=True, out_thd=thd, out=held)
        h = held.transpose(0, 1) if thd else held
        assert (h[:, :front] == 7).all() and (h[:, end:] == 7).all()
        assert torch.equal(h[:, front:end], out[:, front:end])


def test_packed_non_finite_scales_behind_the_sequences(ext, gpu):
    # rows of other sequences and of none never reach a sequence's outputs
    c = _case([70, 50], 4, 2, 64, gpu, tail=100)
    want = ext.int8_attention_forward_packed(*_args(c), is_causal=False)
    for k in ("sK", "sV", "sQ"):
        c[k][:, 70:] = float("nan")
    out = ext.int8_attention_forward_packed(*_args(c), is_causal=False)
    assert torch.equal(out[:, :70], want[:, :70])
    assert torch.isnan(out[:, 70:120]).all() and (out[:, 120:] == 0).all()


def test_packed_future_non_finite_keys_do_not_reach_causal_queries(ext, gpu):
    c = _case([150], 2, 1, 128, gpu)
    want = ext.int8_attention_forward_packed(*_args(c), is_causal=True)
    c["sK"][:, 100:] = float("nan")
    out = ext.int8_attention_forward_packed(*_args(c), is_causal=True)
    assert torch.equal(out[:, :100], want[:, :100])


@pytest.mark.parametrize("cu", [[0, 50, 20, 100], [0, 500], [-7, 30, 100], [90, 10]])
def test_packed_bounds_outside_the_tokens_are_cut(ext, gpu, cu):
    c = _case([100], 2, 2, 64, gpu)
    c["cu"] = torch.tensor(cu, dtype=torch.int32, device=gpu)
    out = ext.int8_attention_forward_packed(*_args(c), is_causal=True)
    torch.cuda.synchronize()
    assert out.shape == (2, 100, 64)


def test_packed_views_of_a_wider_tensor(ext, gpu):
    c = _case([40, 60], 4, 2, 64, gpu)
    want = ext.int8_attention_forward_packed(*_args(c), is_causal=True)
    for k in ("Q", "K", "V"):
        c[k] = c[k].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(ext.int8_attention_forward_packed(*_args(c), is_causal=True), want)


def test_packed_graph_replay_with_other_lengths(ext, gpu):
    c = _case([100, 28, 72], 4, 2, 64, gpu)
    run = lambda: ext.int8_attention_forward_packed(*_args(c), is_causal=True, out_thd=True)  # noqa: E731
    run()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = run()
    for cu in ([0, 100, 128, 200], [0, 1, 2, 3], [0, 0, 200, 200], [0, 60, 61, 150]):
        c["cu"].copy_(torch.tensor(cu, dtype=torch.int32))
        want = run()
        held.fill_(3)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want), cu
        _check(c, want.transpose(0, 1), True, str(cu))


def test_packed_rows_do_not_depend_on_their_neighbours(ext, gpu):
    # a query whose scores grow late sets its own reference; the others of its wave keep theirs
    c = _case([400], 2, 1, 128, gpu, seed=5)
    want = ext.int8_attention_forward_packed(*_args(c))
    assert torch.isfinite(want).all()
    q = torch.tensor([3, 40, 100, 255, 399], device=gpu)
    c["sQ"][:, q] *= 2.0 ** 10
    out = ext.int8_attention_forward_packed(*_args(c))
    rest = torch.ones(400, dtype=torch.bool, device=gpu)
    rest[q] = False
    assert torch.equal(out[:, rest], want[:, rest])
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("long_at", [0, 70, 149])
def test_packed_long_sequences_among_many(ext, gpu, long_at):
    # more than 64 sequences, some of them with 8 tiles and more, some empty
    lens = [(7 * k) % 60 for k in range(150)]
    lens[long_at], lens[(long_at + 64) % 150] = 1500, 1024
    c = _case(lens, 2, 1, 64, gpu, tail=5)
    _check(c, ext.int8_attention_forward_packed(*_args(c), is_causal=True), True)


def test_packed_prompts_of_one_token_round_only_their_output(ext, gpu):
    # one key, whose weight is exactly 1 in fp16: a few fp32 roundings (2^-20 together) and the
    # output's (2^-11)
    c = _case([1] * 40, 4, 2, 64, gpu, seed=9)
    ref, _ = _oracle(c, True)
    out = ext.int8_attention_forward_packed(*_args(c), is_causal=True)
    assert_within(np64(out), ref, (2.0 ** -11 + 2.0 ** -19) * np.abs(ref) + 2.0 ** -25)
