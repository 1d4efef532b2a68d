"""Inputs and error bounds shared by the tests of the grouped-query serving operators.

Bounds count roundings: a rounding to a type is off by at most half its epsilon relative to
the value (fp16 2^-11, bf16 2^-8, fp32 2^-24), or by half its smallest subnormal step.
"""
import numpy as np
import torch

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
# half the smallest subnormal step of the type
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}


def np64(t):
    return t.detach().double().cpu().numpy()


def quantize_rows(x):
    """Per-token int8 and fp32 scales, as the callers do."""
    s = x.float().abs().amax(-1).clamp(min=1e-8) / 127.0
    q = (x.float() / s.unsqueeze(-1)).round().clamp(-128, 127).to(torch.int8)
    return q, s


def rows(g, *shape):
    """N(0, 1) rows, one channel in 64 (at least one) x8."""
    x = torch.randn(*shape, generator=g)
    x[..., torch.randperm(shape[-1], generator=g)[:max(1, shape[-1] // 64)]] *= 8
    return x


def attention_bound(ref, mag, keys, vmax):
    """Error of an fp16 attention row against float64: the weights p are rounded to fp16 in the
    products and in their sum (2 * 2^-11 of sum p|v|), v * scale is rounded to fp16 (2^-11),
    scores of magnitude up to 2^7 in fp32 with three roundings move p by 2^7 * 3 * 2^-24 <
    2^-15, exp2 and the fp32 sums stay below 2^-15; weights below fp16's normal range (2^-14
    of the largest) are off by half a subnormal step 2^-25 each; the result is rounded once."""
    return (3 * 2.0 ** -11 + 2.0 ** -14) * mag + keys * 2.0 ** -25 * vmax + 2.0 ** -11 * np.abs(ref) + 2.0 ** -25


def assert_within(out, ref, bound, label=""):
    out = np.asarray(out, np.float64)
    assert out.shape == ref.shape, (out.shape, ref.shape)
    assert np.isfinite(out).all(), f"{label}: non-finite output"
    over = np.abs(out - ref) - bound
    i = np.unravel_index(np.argmax(over), over.shape)
    assert over[i] <= 0, f"{label}: at {i}: {out[i]} against {ref[i]}, bound {bound[i] if np.ndim(bound) else bound}"


def kv4_case(seed, B, H, Hkv, D, page, lens, device, spare=2):
    """A filled 4-bit cache with shuffled pages, and queries."""
    from oracle import grouped_oracle as G

    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    NP = sum(need) + spare
    cols = max(max(need), 1) + 1
    order = torch.randperm(NP, generator=g)
    tables = torch.full((B, cols), -1, dtype=torch.int32)  # padding is never read
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = order[at:at + n].to(torch.int32)
        at += n
    sides = []
    for _ in range(2):
        c, s = G.kv4_quantize(rows(g, NP, Hkv, page, D).numpy())
        sides.append((torch.from_numpy(G.kv4_pack(c)).to(device), torch.from_numpy(s).to(device)))
    q, sq = quantize_rows(torch.randn(B, H, D, generator=g))
    return dict(Q=q.to(device), sQ=sq.to(device), K=sides[0][0], sK=sides[0][1], V=sides[1][0],
                sV=sides[1][1], tables=tables.to(device),
                lens=torch.tensor(lens, dtype=torch.int32, device=device),
                max_context=max(max(lens), 1))
