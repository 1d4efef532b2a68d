"""Inputs and error bounds shared by the tests of the operators over the paged INT8 cache."""
import numpy as np
import torch

from grouped_helpers import quantize_rows, rows


def attention_bound(ref, mag, keys, vmax):
    """Error of an fp16 attention row against float64: weights p sV carry 22 bits (2^-22 of
    p|v|); scores of magnitude up to 2^7 in fp32 with three roundings move p by 2^7 * 3 * 2^-24
    < 2^-15, exp2 and the fp32 sums stay below another 2^-15; weights below fp16's normal range
    are off by 2^-25 beside a largest one of 2^9 or more, 2^-34 of it each; the result is
    rounded once."""
    return 2.0 ** -14 * mag + keys * 2.0 ** -34 * vmax + 2.0 ** -11 * np.abs(ref) + 2.0 ** -25


def tables_for(g, need, cols=None, spare=2):
    """Shuffled pages for sequences of need[b] pages; -1 behind them.  (tables, pages)."""
    NP = sum(need) + spare
    order = torch.randperm(NP, generator=g)
    tables = torch.full((len(need), cols or max(max(need), 1) + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = order[at:at + n].to(torch.int32)
        at += n
    return tables, NP


def words_of(sets, N):
    """int64 words [len(sets), ceil(N / 64)] of sets of node indices."""
    w = torch.zeros(len(sets), -(-N // 64), dtype=torch.int64)
    for i, s in enumerate(sets):
        for j in s:
            bit = 1 << (j % 64)
            w[i, j // 64] |= bit - (1 << 64) if bit == 1 << 63 else bit
    return w


def tree_words(g, N):
    """The ancestors of each node of a random tree, itself among them."""
    sets = []
    for i in range(N):
        parent = int(torch.randint(-1, i, (1,), generator=g)) if i else -1
        sets.append({i} | (sets[parent] if parent >= 0 else set()))
    return words_of(sets, N)


def tree_case(seed, lens, N, H, Hkv, D, page, device, counts=None, mask="each", top=None):
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    cn = counts or [N] * B
    tables, NP = tables_for(g, [-(-(max(n, 0) + c) // page) for n, c in zip(lens, cn)])
    k, sk = quantize_rows(rows(g, NP, Hkv, page, D))
    v, sv = quantize_rows(rows(g, NP, Hkv, page, D))
    q, sq = quantize_rows(torch.randn(B, H, N, D, generator=g))
    if mask == "each":
        m = torch.stack([tree_words(g, N) for _ in range(B)])
    else:
        m = tree_words(g, N) if mask == "shared" else None
    i32 = dict(dtype=torch.int32, device=device)
    return dict(Q=q.to(device), sQ=sq.to(device), K=k.to(device), sK=sk.to(device), V=v.to(device), sV=sv.to(device),
                tables=tables.to(device), lens=torch.tensor(lens, **i32),
                mask=None if m is None else m.to(device),
                counts=torch.tensor(counts, **i32) if counts else None,
                max_context=top or max(n + c for n, c in zip(lens, cn)) or 1)


def sparse_case(seed, lens, H, Hkv, D, page, device, top):
    from oracle import paged_oracle as P

    g = torch.Generator().manual_seed(seed)
    tables, NP = tables_for(g, [-(-n // page) for n in lens])
    k, sk = quantize_rows(rows(g, NP, Hkv, page, D) + torch.randn(NP, Hkv, 1, D, generator=g))
    v, sv = quantize_rows(rows(g, NP, Hkv, page, D))
    m, sm = P.page_means(k.numpy(), sk.numpy())
    q, sq = quantize_rows(torch.randn(len(lens), H, D, generator=g))
    d = dict(Q=q, sQ=sq, K=k, sK=sk, V=v, sV=sv, M=torch.from_numpy(m), sM=torch.from_numpy(sm), tables=tables,
             lens=torch.tensor(lens, dtype=torch.int32))
    return dict({n: t.to(device) for n, t in d.items()}, top=top, max_context=max(max(lens), 1))
