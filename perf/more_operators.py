"""Timed cases of the operators over a paged INT8 KV cache with grouped heads: its writer, its
readers for drafted trees and for selected blocks, and the two that keep it in order.

A case is a dict of plain values whose "op" names the operator:

    append   a fused QKV projection's rows: norms per head, rotation, queries as per-token INT8,
             keys and values into the cache
    tree     attention of a tree of drafted tokens: each sees the sequence and its ancestors
    move     the rows of an accepted path brought together in the cache
    means    the mean key of each page, which the block scores read
    sparse   one new token per sequence against the blocks with the highest scores

Inputs are seeded and synthetic: N(0, 1) activations with a few outlier channels (x8), quantized
symmetrically per row.  Codes and scales are returned as the values they stand for, in 16 bits.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}

# The largest listed work of each kind, which bounds the drawn cases.
MAX_APPEND_ELEMS = 8191 * 48 * 128
MAX_CACHE_ELEMS = 32 * 8 * 32768 * 128
MAX_TREE_ELEMS = 16 * 8 * 8192 * 128
MAX_TREE_SCORES = 4 * 32 * 64 * 16384
MAX_MOVE_ELEMS = 64 * 24 * 8 * 128
MAX_MEANS_ELEMS = 2048 * 8 * 64 * 128


def _ext():
    pkg = os.path.join(os.getcwd(), "int8-transformer-kernels_amd")
    if pkg not in sys.path:
        sys.path.insert(1, pkg)
    import int8_ext

    return int8_ext


def listed():
    return [
        # A decode step of 48 sequences, 32 query and 8 key heads of 128 with norms.
        dict(name="append_step", op="append", B=48, S=1, Hq=32, Hkv=8, D=128, rot=128, interleaved=False,
             norm=True, dtype="bf16", page=64),
        # A prompt with an odd number of tokens enters the cache.
        dict(name="append_prompt", op="append", B=1, S=8191, Hq=32, Hkv=8, D=128, rot=128,
             interleaved=False, norm=True, dtype="bf16", page=64),
        # One conversation of a thousand tokens, a chain of five drafted ones: latency.
        dict(name="tree_single", op="tree", B=1, N=5, Hq=32, Hkv=8, D=128, page=16, max_len=1000,
             shape="chain", shared=True, ragged=False, rows=False),
        # A batch of a small model with as many key heads as query heads, trees of different sizes.
        dict(name="tree_small_heads", op="tree", B=13, N=9, Hq=12, Hkv=12, D=64, page=32, max_len=3001,
             shape="tree", shared=False, ragged=True, rows=True),
        # The serving batch: 16 sequences of up to 8K tokens, one tree of 16 nodes for all.
        dict(name="tree_serving", op="tree", B=16, N=16, Hq=32, Hkv=8, D=128, page=64, max_len=8192,
             shape="tree", shared=True, ragged=False, rows=True),
        # Wide trees of 64 nodes over long contexts, 256 query rows for each key head.
        dict(name="tree_wide", op="tree", B=4, N=64, Hq=32, Hkv=8, D=128, page=64, max_len=16320,
             shape="tree", shared=False, ragged=False, rows=True),
        # The accepted path of one sequence: latency.
        dict(name="move_single", op="move", B=1, N=16, P=5, Hkv=8, D=128, page=16),
        # The accepted paths of a batch of 64.
        dict(name="move_batch", op="move", B=64, N=32, P=7, Hkv=8, D=128, page=16),
        # The pages that a decode step of 64 sequences fills.
        dict(name="means_step", op="means", n=4, Hkv=8, D=128, page=64),
        # The pages of a batch of prompts, 128K tokens.
        dict(name="means_prompt", op="means", n=2048, Hkv=8, D=128, page=64),
        # One conversation of 20000 tokens, 32 blocks of 64 read of it.
        dict(name="sparse_single", op="sparse", B=1, Hq=32, Hkv=8, D=128, page=64, max_len=20000, top=32),
        # The serving batch: 32 sequences of up to 32K tokens, 64 blocks of 64 each.
        dict(name="sparse_serving", op="sparse", B=32, Hq=32, Hkv=8, D=128, page=64, max_len=32768, top=64),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "append", "tree", "tree", "tree", "move", "means", "sparse", "sparse"])
    D, Hkv = rng.choice([64, 128, 128]), rng.choice([1, 2, 4, 8, 12])
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "append":
        G = rng.choice([1, 2, 4, 8])
        B, S = (_log_int(rng, 1, 128), rng.choice([1, 1, 5, 16])) if rng.random() < 0.5 else (rng.choice([1, 1, 2]), _log_int(rng, 16, 16384))
        S = max(1, min(S, MAX_APPEND_ELEMS // (B * (G + 2) * Hkv * D)))
        return dict(op=op, B=B, S=S, Hq=G * Hkv, Hkv=Hkv, D=D, rot=rng.choice([D, D, D // 2]),
                    interleaved=rng.random() < 0.3, norm=rng.random() < 0.6,
                    dtype=rng.choice(["fp16", "bf16", "bf16", "fp32"]), page=page)
    if op == "tree":
        G, B, N = rng.choice([1, 2, 3, 4, 6, 8]), _log_int(rng, 1, 32), _log_int(rng, 1, 100)
        L = _log_int(rng, 16, 32768)
        L = min(L, MAX_TREE_ELEMS // (B * Hkv * D), MAX_TREE_SCORES // (B * G * Hkv * N) - N)
        return dict(op=op, B=B, N=N, Hq=G * Hkv, Hkv=Hkv, D=D, page=page, max_len=max(L, 1),
                    shape=rng.choice(["tree", "tree", "chain"]), shared=rng.random() < 0.4,
                    ragged=rng.random() < 0.4, rows=rng.random() < 0.6)
    if op == "move":
        N = _log_int(rng, 8, 128)
        P = rng.randint(1, min(16, N // 2))
        B = max(1, min(_log_int(rng, 1, 64), MAX_MOVE_ELEMS // (P * Hkv * D)))
        return dict(op=op, B=B, N=N, P=P, Hkv=Hkv, D=D, page=rng.choice([16, 32, 64]))
    if op == "means":
        n = max(1, min(_log_int(rng, 1, 4096), MAX_MEANS_ELEMS // (Hkv * page * D)))
        return dict(op=op, n=n, Hkv=Hkv, D=D, page=page)
    G, B, L = rng.choice([1, 2, 3, 4, 8, 16]), _log_int(rng, 1, 64), _log_int(rng, 256, 65536)
    L = max(256, min(L, MAX_CACHE_ELEMS // (B * Hkv * D)))
    return dict(op=op, B=B, Hq=G * Hkv, Hkv=Hkv, D=D, page=page, max_len=L, top=_log_int(rng, 1, max(2, 4096 // page)))


# ------------------------------------------------------------------ inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _quantize_rows(x):
    s = x.float().abs().amax(dim=-1).clamp(min=1e-8) / 127.0
    q = (x.float() / s.unsqueeze(-1)).round_().clamp_(-128, 127).to(torch.int8)
    return q, s.contiguous()


def _rows(g, shape):
    """N(0, 1) rows of the last dimension, 1% of its channels (at least one) x8."""
    x = torch.randn(shape, generator=g, device=DEV)
    x[..., torch.randperm(shape[-1], generator=g, device=DEV)[:max(1, shape[-1] // 100)]] *= 8.0
    return x


def _pages(g, pages, H, page, D, centre=0.0):
    """A filled cache side, 2^24 elements at a time; the rows of a page about a mean of their own."""
    q = torch.empty((pages, H, page, D), dtype=torch.int8, device=DEV)
    s = torch.empty((pages, H, page), dtype=torch.float32, device=DEV)
    step = max(1, (1 << 24) // (H * page * D))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        x = _rows(g, (n, H, page, D))
        if centre:
            x += centre * torch.randn((n, H, 1, D), generator=g, device=DEV)
        q[p:p + n], s[p:p + n] = _quantize_rows(x)
    return q, s


def _tables(need, cpu):
    """Shuffled pages for sequences of `need` pages each, three more left free."""
    order = torch.randperm(int(need.sum()) + 3, generator=cpu)
    tables = torch.zeros((len(need), int(need.max())), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need.tolist()):
        tables[b, :n] = order[at:at + n].to(torch.int32)
        at += n
    return tables.to(DEV), len(order)


def _lens(c, cpu):
    top = c["max_len"]
    lens = torch.randint(max(1, top // 4), top + 1, (c["B"],), generator=cpu)
    lens[0] = top
    return lens


def _tree_words(c, cpu):
    """The ancestors of every node, itself among them, as bits of int64 words; random parents."""
    B, N = (1 if c["shared"] else c["B"]), c["N"]
    words = torch.zeros((B, N, -(-N // 64)), dtype=torch.int64)
    for b in range(B):
        sets = []
        for i in range(N):
            # a node's parent: the one before (chain), or one of the nodes so far, or the sequence
            parent = i - 1 if c["shape"] == "chain" else int(torch.randint(-1, i, (1,), generator=cpu)) if i else -1
            bits = (1 << i) | (sets[parent] if parent >= 0 else 0)
            sets.append(bits)
            for w in range(words.shape[2]):
                v = (bits >> (64 * w)) & (2 ** 64 - 1)
                words[b, i, w] = v - 2 ** 64 if v >= 2 ** 63 else v
    return (words[0] if c["shared"] else words).to(DEV)


def _page_means(k, sk):
    """Codes and scales of the mean rows of pages [n, H, P, D], summed in 64 bits."""
    q = torch.empty((k.shape[0], k.shape[1], k.shape[3]), dtype=torch.int8, device=k.device)
    s = torch.empty((k.shape[0], k.shape[1]), dtype=torch.float32, device=k.device)
    step = max(1, (1 << 25) // k[0].numel())
    for p in range(0, k.shape[0], step):
        x = k[p:p + step].double() * sk[p:p + step].double().unsqueeze(-1)
        q[p:p + step], s[p:p + step] = _quantize_rows((x.sum(2) / k.shape[2]).float())
    return q, s


def _inputs(c, seed):
    g, cpu = _gen(seed), torch.Generator().manual_seed(int(seed))
    H, D, page = c["Hkv"], c["D"], c["page"]
    if c["op"] == "append":
        B, S, R, T = c["B"], c["S"], c["rot"], c["B"] * c["S"]
        x = _rows(g, (B, S, (c["Hq"] + 2 * H) * D)).to(DTYPES[c["dtype"]])
        top = 32768  # the model's longest context, whose angles it keeps
        angle = torch.arange(top, dtype=torch.float64, device=DEV).unsqueeze(1) * (
            10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device=DEV) / R))
        first = torch.randint(0, top - S + 1, (B, 1), generator=g, device=DEV)
        pos = (first + torch.arange(S, device=DEV)).to(torch.int32).contiguous()
        w = [1 + 0.1 * torch.randn(D, generator=g, device=DEV) for _ in range(2)] if c["norm"] else [None, None]
        pages = -(-T // page)
        order = torch.randperm(pages, generator=cpu)
        t = torch.arange(T)
        slots = (order[t // page] * page + t % page).to(torch.int32).to(DEV)
        return dict(x=x, cos=angle.cos().float(), sin=angle.sin().float(), pos=pos, wq=w[0], wk=w[1], slots=slots,
                    K=torch.zeros((pages, H, page, D), dtype=torch.int8, device=DEV),
                    V=torch.zeros((pages, H, page, D), dtype=torch.int8, device=DEV),
                    sK=torch.zeros((pages, H, page), device=DEV), sV=torch.zeros((pages, H, page), device=DEV))
    if c["op"] == "move":
        # the pages with the drafted nodes; the nodes of the path lie behind its own length
        B, N, P = c["B"], c["N"], c["P"]
        per = -(-N // page) + 1
        k, sk = _pages(g, B * per, H, page, D)
        v, sv = _pages(g, B * per, H, page, D)
        order = torch.randperm(B * per, generator=cpu).view(B, per)
        first = torch.randint(0, page, (B, 1), generator=cpu)
        path = torch.stack([torch.randperm(N - P, generator=cpu)[:P].sort().values + P for _ in range(B)])

        def slots(node):
            at = first + node
            return (order.gather(1, at // page) * page + at % page).to(torch.int32).to(DEV)

        return dict(K=k, sK=sk, V=v, sV=sv, src=slots(path), dst=slots(torch.arange(P).expand(B, P)))
    if c["op"] == "means":
        k, sk = _pages(g, c["n"] + 3, H, page, D, centre=0.5)
        ids = torch.randperm(c["n"] + 3, generator=cpu)[:c["n"]].to(torch.int32).to(DEV)
        return dict(K=k, sK=sk, ids=ids, M=torch.zeros((c["n"] + 3, H, D), dtype=torch.int8, device=DEV),
                    sM=torch.zeros((c["n"] + 3, H), device=DEV))
    lens = _lens(c, cpu)
    if c["op"] == "tree":
        B, N = c["B"], c["N"]
        counts = torch.randint(max(1, N // 2), N + 1, (B,), generator=cpu) if c["ragged"] else torch.full((B,), N)
        tables, pages = _tables((lens + counts + page - 1) // page, cpu)
        k, sk = _pages(g, pages, H, page, D)
        v, sv = _pages(g, pages, H, page, D)
        q, sq = _quantize_rows(torch.randn((B, c["Hq"], N, D), generator=g, device=DEV).half())
        return dict(q=q, sq=sq, K=k, sK=sk, V=v, sV=sv, tables=tables, lens=lens.to(torch.int32).to(DEV),
                    words=_tree_words(c, cpu), counts=counts.to(torch.int32).to(DEV) if c["ragged"] else None)
    tables, pages = _tables((lens + page - 1) // page, cpu)
    k, sk = _pages(g, pages, H, page, D, centre=0.5)
    v, sv = _pages(g, pages, H, page, D)
    m, sm = _page_means(k, sk)
    q, sq = _quantize_rows(torch.randn((c["B"], c["Hq"], D), generator=g, device=DEV).half())
    return dict(q=q, sq=sq, K=k, sK=sk, V=v, sV=sv, M=m, sM=sm, tables=tables, lens=lens.to(torch.int32).to(DEV))


def prepare(case, seed):
    d = _inputs(case, seed)
    d["case"] = dict(case)
    return d


# -------------------------------------------------------------------- runs


def run(d):
    c = d["case"]
    if own:
        return _OWN[c["op"]](c, d, _ext())
    return _PLAIN[c["op"]](c, d)


def _own_append(c, d, ext):
    q, sq = ext.qk_norm_rope_append(d["x"], c["Hq"], c["Hkv"], d["cos"], d["sin"], d["pos"], d["K"], d["V"],
                                    d["sK"], d["sV"], d["slots"], q_weight=d["wq"], k_weight=d["wk"], eps=1e-6,
                                    interleaved=c["interleaved"])
    t = DTYPES["bf16"] if c["dtype"] == "bf16" else DTYPES["fp16"]
    return [ext.dequantize_per_token(*y, dtype=t) for y in ((q, sq), (d["K"], d["sK"]), (d["V"], d["sV"]))]


def _own_tree(c, d, ext):
    return ext.int8_tree_attention_forward_paged(
        d["q"], d["K"], d["V"], d["sq"], d["sK"], d["sV"], d["tables"], d["lens"], d["words"],
        min(c["max_len"] + c["N"], d["tables"].shape[1] * c["page"]), node_counts=d["counts"], out_bshd=c["rows"])


def _own_move(c, d, ext):
    ext.kv_cache_move_paged(d["K"], d["V"], d["sK"], d["sV"], d["src"], d["dst"])
    return [ext.dequantize_per_token(d["K"], d["sK"]), ext.dequantize_per_token(d["V"], d["sV"])]


def _own_means(c, d, ext):
    ext.kv_page_means(d["K"], d["sK"], d["ids"], d["M"], d["sM"])
    return ext.dequantize_per_token(d["M"], d["sM"])


def _own_sparse(c, d, ext):
    return ext.int8_decode_attention_forward_paged_sparse(
        d["q"], d["K"], d["V"], d["sq"], d["sK"], d["sV"], d["M"], d["sM"], d["tables"], d["lens"],
        c["max_len"], c["top"])


_OWN = dict(append=_own_append, tree=_own_tree, move=_own_move, means=_own_means, sparse=_own_sparse)


# ------------------------------------------------------------- plain forms


def _values(q, s, t=torch.float16):
    return (q.float() * s.unsqueeze(-1)).to(t)


def _plain_append(c, d):
    B, S, Hq, Hkv, D, R = (c[n] for n in ("B", "S", "Hq", "Hkv", "D", "rot"))
    dt, page, slots = DTYPES[c["dtype"]], c["page"], d["slots"].long()
    x = d["x"].view(B, S, Hq + 2 * Hkv, D).transpose(1, 2).float()
    pos = d["pos"].long()
    cos, sin = d["cos"][pos].unsqueeze(1), d["sin"][pos].unsqueeze(1)

    def rotated(y, w):
        if w is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w
        r = y[..., :R]
        if c["interleaved"]:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
        else:
            a, b = r[..., :R // 2], r[..., R // 2:]
            r = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
        return torch.cat((r, y[..., R:]), dim=-1).to(dt)

    def stored(y, pages, scales):
        q, s = _quantize_rows(y.transpose(1, 2).reshape(B * S, Hkv, D))
        pages[slots // page, :, slots % page] = q
        scales[slots // page, :, slots % page] = s

    q, sq = _quantize_rows(rotated(x[:, :Hq], d["wq"]))
    stored(rotated(x[:, Hq:Hq + Hkv], d["wk"]), d["K"], d["sK"])
    stored(x[:, Hq + Hkv:], d["V"], d["sV"])
    t = DTYPES["bf16"] if c["dtype"] == "bf16" else DTYPES["fp16"]
    return [_values(q, sq, t), _values(d["K"], d["sK"], t), _values(d["V"], d["sV"], t)]


def _attend(q, k, v, seen):
    """softmax(q k^T / sqrt(D)) v in 32 bits, q [B, Hkv, M, D], seen [B, 1 or Hkv, M, L]."""
    s = (q @ k.transpose(2, 3)).mul_(q.shape[-1] ** -0.5)
    s.masked_fill_(~seen, -math.inf)
    s.sub_(s.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    s.div_(s.sum(-1, keepdim=True).clamp_(min=1e-30))
    return s @ v


def _plain_tree(c, d):
    B, N, Hq, Hkv, D = c["B"], c["N"], c["Hq"], c["Hkv"], c["D"]
    t = d["tables"].long()

    def values(pages, scales):  # [B, Hkv, positions, D]
        return (pages[t].float() * scales[t].unsqueeze(-1)).transpose(1, 2).flatten(2, 3)

    k, v = values(d["K"], d["sK"]), values(d["V"], d["sV"])
    L = k.shape[2]
    i = torch.arange(N, device=DEV)
    words = d["words"] if d["words"].dim() == 3 else d["words"].unsqueeze(0).expand(B, -1, -1)
    sees = ((words[:, :, i // 64] >> (i % 64)) & 1).bool()  # [B, node, ancestor]
    count = d["counts"].view(B, 1) if d["counts"] is not None else torch.full((B, 1), N, device=DEV)
    node = torch.arange(L, device=DEV) - d["lens"].view(B, 1)  # [B, L]
    drafted = ((node >= 0) & (node < count)).unsqueeze(1)
    seen = (node < 0).unsqueeze(1) | (drafted & sees.gather(2, node.clamp(0, N - 1).unsqueeze(1).expand(B, N, L)))
    seen = seen & (i < count).unsqueeze(2)
    q = (d["q"].float() * d["sq"].unsqueeze(-1)).view(B, Hkv, Hq // Hkv * N, D)
    o = _attend(q, k, v, seen.repeat(1, Hq // Hkv, 1).unsqueeze(1)).view(B, Hq, N, D)
    o = o.masked_fill((i >= count).view(B, 1, N, 1), 0).to(torch.float16)
    return o.transpose(1, 2).contiguous() if c["rows"] else o


def _plain_move(c, d):
    page, src, dst = c["page"], d["src"].long(), d["dst"].long()
    for pages in (d["K"], d["V"], d["sK"], d["sV"]):
        pages[dst // page, :, dst % page] = pages[src // page, :, src % page]
    return [_values(d["K"], d["sK"]), _values(d["V"], d["sV"])]


def _plain_means(c, d):
    ids = d["ids"].long()
    d["M"][ids], d["sM"][ids] = _page_means(d["K"][ids], d["sK"][ids])
    return _values(d["M"], d["sM"])


def _plain_sparse(c, d):
    B, Hq, Hkv, D, page, top = (c[n] for n in ("B", "Hq", "Hkv", "D", "page", "top"))
    t, lens = d["tables"].long(), d["lens"].long()
    blocks = (lens + page - 1) // page
    # scores next to each other decide which block is read: 64 bits
    q = d["q"].view(B, Hkv, Hq // Hkv, D).double()
    m = d["M"][t].transpose(1, 2).double()  # [B, Hkv, blocks, D]
    s = (q.unsqueeze(3) * m.unsqueeze(2)).sum(-1) if q.numel() * m.shape[2] < 1 << 27 else q @ m.transpose(2, 3).contiguous()
    s = s * d["sM"][t].transpose(1, 2).unsqueeze(2) * d["sq"].view(B, Hkv, -1, 1)
    s = s.amax(2)
    i = torch.arange(t.shape[1], device=DEV)
    s = s.masked_fill(i == blocks.view(B, 1, 1) - 1, math.inf).masked_fill(i >= blocks.view(B, 1, 1), -math.inf)
    n = min(top, t.shape[1])
    taken = torch.sort(s, dim=-1, descending=True, stable=True).indices[..., :n].sort(dim=-1).values
    real = taken < blocks.view(B, 1, 1)
    ids = t.unsqueeze(1).expand(B, Hkv, -1).gather(2, taken)
    h = torch.arange(Hkv, device=DEV).view(1, Hkv, 1)

    def values(pages, scales):  # [B, Hkv, positions, D]
        return (pages[ids, h].float() * scales[ids, h].unsqueeze(-1)).flatten(2, 3)

    at = (taken.unsqueeze(-1) * page + torch.arange(page, device=DEV)).flatten(2)
    seen = (at < lens.view(B, 1, 1)).unsqueeze(2)
    o = _attend((d["q"].float() * d["sq"].unsqueeze(-1)).view(B, Hkv, -1, D), values(d["K"], d["sK"]),
                values(d["V"], d["sV"]), seen)
    which = torch.full((B, Hkv, top), -1, dtype=torch.int32, device=DEV)
    which[..., :n] = taken.masked_fill(~real, -1)
    return o.reshape(B, Hq, D).to(torch.float16), which


_PLAIN = dict(append=_plain_append, tree=_plain_tree, move=_plain_move, means=_plain_means, sparse=_plain_sparse)


# ------------------------------------------------------------------- work


def work(case):
    c = case
    D, H = c["D"], c["Hkv"]
    if c["op"] == "append":
        T, e = c["B"] * c["S"], DTYPES[c["dtype"]].itemsize
        rows = T * (c["Hq"] + 2 * H)
        stored = 2 * -(-T // c["page"]) * c["page"] * H
        # each row in once and out once as codes, angles of each position; the values of the queries
        # and of the pages in 16 bits
        return dict(bytes=rows * (D * e + D + 4) + T * (4 * c["rot"] + 8) + 2 * T * c["Hq"] * D + stored * 2 * D,
                    flops=8 * rows * D)
    if c["op"] == "tree":
        # lengths are uniform in [max_len / 4, max_len]
        mean = 0.625 if c["B"] > 1 else 1.0
        keys = int(c["B"] * (c["max_len"] * mean + c["N"]))
        rows = c["B"] * c["Hq"] * c["N"]
        return dict(bytes=2 * keys * H * (D + 4) + rows * (3 * D + 4), flops=4 * keys * c["Hq"] * c["N"] * D)
    if c["op"] == "move":
        pairs, rows = c["B"] * c["P"] * H, c["B"] * (-(-c["N"] // c["page"]) + 1) * c["page"] * H
        return dict(bytes=4 * pairs * (D + 4) + 2 * rows * (3 * D + 4), flops=2 * rows * D)
    if c["op"] == "means":
        rows = c["n"] * H * c["page"]
        return dict(bytes=rows * (D + 4) + c["n"] * H * (D + 4) + (c["n"] + 3) * H * 2 * D, flops=2 * rows * D)
    mean = 0.625 if c["B"] > 1 else 1.0
    blocks = int(c["B"] * c["max_len"] * mean / c["page"])
    keys = min(c["B"] * c["top"], blocks) * c["page"]
    return dict(bytes=blocks * H * (D + 4) + 2 * keys * H * (D + 4) + c["B"] * (c["Hq"] * (3 * D + 4) + 4 * H * c["top"]),
                flops=2 * blocks * c["Hq"] * D + 4 * keys * c["Hq"] * D)


# ------------------------------------------------------------------- 64 bits


def _softmax_rows(q, k, v, seen):
    """Rows of softmax(q k^T / sqrt(D)) v in float64; rows that see nothing are zeros."""
    s = torch.where(seen, (q @ k.t()) / math.sqrt(q.shape[1]), -math.inf)
    return torch.nan_to_num(torch.softmax(s, dim=-1), nan=0.0) @ v


def _sequence(d, m, pages, h):
    """Rows of one key head along a list of pages, in float64."""
    return (d[m][pages, h].double() * d["s" + m][pages, h].double().unsqueeze(-1)).flatten(0, 1)


def _exact_append(c, d):
    B, S, D, R, Hq, H = c["B"], c["S"], c["D"], c["rot"], c["Hq"], c["Hkv"]
    x = d["x"].double().reshape(B * S, Hq + 2 * H, D)
    turn = torch.complex(d["cos"].double(), d["sin"].double())[d["pos"].reshape(-1).long()].unsqueeze(1)

    def through_int8(y):
        y = y.to(DTYPES[c["dtype"]]).double()
        step = y.abs().amax(-1, keepdim=True).clamp(min=1e-8) / 127
        return (y / step).round() * step

    def turned(y, w):
        y = y.clone()
        if w is not None:
            y = y / (y.pow(2).sum(-1, keepdim=True) / D + 1e-6).sqrt() * w.double()
        first = slice(0, R, 2) if c["interleaved"] else slice(0, R // 2)
        second = slice(1, R, 2) if c["interleaved"] else slice(R // 2, R)
        z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn
        y[..., first], y[..., second] = z.real, z.imag
        return through_int8(y)

    def cached(y):
        out = torch.zeros(d["K"].shape[0] * c["page"], H, D, dtype=torch.float64, device=DEV)
        out[d["slots"].long()] = y
        return out.view(-1, c["page"], H, D).transpose(1, 2).contiguous()

    q = turned(x[:, :Hq], d["wq"]).reshape(B, S, Hq, D).transpose(1, 2).contiguous()
    return [q, cached(turned(x[:, Hq:Hq + H], d["wk"])), cached(through_int8(x[:, Hq + H:]))]


def _exact_tree(c, d):
    B, N, G, page = c["B"], c["N"], c["Hq"] // c["Hkv"], c["page"]
    out = torch.zeros((B, c["Hq"], N, c["D"]), dtype=torch.float64, device=DEV)
    host = d["words"].cpu().tolist()
    for b in range(B):
        n, count = int(d["lens"][b]), N if d["counts"] is None else int(d["counts"][b])
        masks = host if c["shared"] else host[b]
        bits = [sum((w % 2 ** 64) << (64 * k) for k, w in enumerate(row)) for row in masks]
        seen = torch.ones((count, n + count), dtype=torch.bool)
        seen[:, n:] = torch.tensor([[bool(bits[i] >> j & 1) for j in range(count)] for i in range(count)])
        pages = d["tables"][b, :-(-(n + count) // page)].long()
        seen = seen.to(DEV)
        for h in range(c["Hkv"]):
            k, v = (_sequence(d, m, pages, h)[:n + count] for m in "KV")
            for j in range(h * G, (h + 1) * G):
                q = d["q"][b, j, :count].double() * d["sq"][b, j, :count].double().unsqueeze(1)
                out[b, j, :count] = _softmax_rows(q, k, v, seen)
    return out.transpose(1, 2).contiguous() if c["rows"] else out


def _exact_means(c, d):
    ids = d["ids"].long()
    out = torch.zeros((d["K"].shape[0], c["Hkv"], c["D"]), dtype=torch.float64, device=DEV)
    for i in range(0, len(ids), 256):
        at = ids[i:i + 256]
        m = torch.einsum("nhpd,nhp->nhd", d["K"][at].double(), d["sK"][at].double()) / c["page"]
        step = m.abs().amax(-1, keepdim=True).clamp(min=1e-8) / 127
        out[at] = (m / step).round() * step
    return out


def _exact_sparse(c, d):
    B, Hkv, G, D, page, top = c["B"], c["Hkv"], c["Hq"] // c["Hkv"], c["D"], c["page"], c["top"]
    out = torch.empty((B, c["Hq"], D), dtype=torch.float64, device=DEV)
    which = torch.full((B, Hkv, top), -1, dtype=torch.int32)
    for b in range(B):
        n = int(d["lens"][b])
        t = d["tables"][b, :-(-n // page)].long()
        q = d["q"][b].double() * d["sq"][b].double().unsqueeze(1)
        for h in range(Hkv):
            m = d["M"][t, h].double() * d["sM"][t, h].double().unsqueeze(1)
            score = (m @ q[h * G:(h + 1) * G].t()).amax(1)[:-1].tolist()
            best = sorted(range(len(score)), key=lambda i: (-score[i], i))[:top - 1]
            taken = sorted(best + [len(t) - 1])
            which[b, h, :len(taken)] = torch.tensor(taken, dtype=torch.int32)
            pages = t[torch.tensor(taken, device=DEV)]
            last = (len(taken) - 1) * page + n - (len(t) - 1) * page
            k, v = (_sequence(d, s, pages, h)[:last] for s in "KV")
            out[b, h * G:(h + 1) * G] = _softmax_rows(q[h * G:(h + 1) * G], k, v, torch.ones(1, dtype=torch.bool, device=DEV))
    return out, which.to(DEV)


def _exact_move(c, d):
    out = []
    for m in "KV":
        x = (d[m].double() * d["s" + m].double().unsqueeze(-1)).transpose(1, 2).flatten(0, 1)  # by slot
        y = x.clone()
        for a, b in zip(d["src"].tolist(), d["dst"].tolist()):
            y[b] = x[a]
        out.append(y.view(-1, c["page"], c["Hkv"], c["D"]).transpose(1, 2).contiguous())
    return out


_EXACT = dict(append=_exact_append, tree=_exact_tree, move=_exact_move, means=_exact_means, sparse=_exact_sparse)


def exact(case, seed):
    return _EXACT[case["op"]](case, _inputs(case, seed))
