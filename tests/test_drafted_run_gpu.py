"""The operators over the paged INT8 cache as a drafted decoding step runs them (GPU): a prompt and
a tree of drafted tokens enter the cache, the tree attends, its accepted path is moved together, and
the next token decodes over selected blocks; every stage against the 64-bit oracle, eagerly and from
one captured graph."""
import numpy as np
import pytest
import torch

from grouped_helpers import assert_within, np64, quantize_rows
from oracle import paged_oracle as P
from paged_helpers import attention_bound, tables_for, words_of

pytestmark = pytest.mark.gpu


class Step:
    """One layer's buffers and the calls of a step."""

    def __init__(self, ext, gpu, H, Hkv, D, page, lens, N, top, seed):
        g = self.g = torch.Generator().manual_seed(seed)
        self.ext, self.H, self.Hkv, self.D, self.page, self.N, self.top = ext, H, Hkv, D, page, N, top
        self.B = len(lens)
        self.max_context = max(lens) + N + 1
        tables, NP = tables_for(g, [-(-(n + N + 1) // page) for n in lens])
        z = dict(device=gpu)
        self.tables, self.NP = tables.to(gpu), NP
        self.K, self.V = (torch.zeros(NP, Hkv, page, D, dtype=torch.int8, **z) for _ in range(2))
        self.sK, self.sV = torch.zeros(NP, Hkv, page, **z), torch.zeros(NP, Hkv, page, **z)
        self.M, self.sM = torch.zeros(NP, Hkv, D, dtype=torch.int8, **z), torch.zeros(NP, Hkv, **z)
        self.lens = torch.tensor(lens, dtype=torch.int32, **z)
        a = torch.rand(self.max_context, D // 2, generator=g) * 6.28
        self.cos, self.sin = a.cos().to(gpu), a.sin().to(gpu)
        self.wq, self.wk = ((1 + 0.1 * torch.randn(D, generator=g)).to(gpu) for _ in range(2))
        self.x = torch.zeros(self.B, N, (H + 2 * Hkv) * D, dtype=torch.bfloat16, **z)
        self.pos, self.slots = (torch.zeros(self.B, N, dtype=torch.int32, **z) for _ in range(2))
        self.mask = torch.zeros(self.B, N, -(-N // 64), dtype=torch.int64, **z)
        self.src, self.dst = (torch.full((self.B, N), -1, dtype=torch.int32, **z) for _ in range(2))
        self.full = torch.full((NP,), -1, dtype=torch.int32, **z)
        self.accepted = torch.zeros(self.B, dtype=torch.int32, **z)
        self.q1, s1 = quantize_rows(torch.randn(self.B, H, D, generator=g))
        self.q1, self.sq1 = self.q1.to(gpu), s1.to(gpu)

    def slot(self, b, pos):
        return int(self.tables[b, pos // self.page]) * self.page + pos % self.page

    def append(self, x, pos, slots):
        return self.ext.qk_norm_rope_append(x, self.H, self.Hkv, self.cos, self.sin, pos, self.K, self.V, self.sK, self.sV,
                                            slots, q_weight=self.wq, k_weight=self.wk)

    def prompts(self):
        width = self.x.shape[2]
        for b in range(self.B):
            n = int(self.lens[b])
            if n == 0:
                continue
            x = torch.randn(1, n, width, generator=self.g).to(torch.bfloat16).to(self.x.device)
            i32 = dict(dtype=torch.int32, device=x.device)
            self.append(x, torch.arange(n, **i32), torch.tensor([self.slot(b, j) for j in range(n)], **i32))
        self.full_pages()

    def full_pages(self):
        """Every full page of the sequences' committed positions is due."""
        ids = [int(self.tables[b, i]) for b in range(self.B) for i in range(int(self.lens[b] + self.accepted[b]) // self.page)]
        self.full.fill_(-1)
        self.full[:len(ids)] = torch.tensor(ids, dtype=torch.int32)
        return ids

    def draft(self):
        """A new tree for each sequence, an accepted path of it and where that goes."""
        for b in range(self.B):
            n, sets, depth = int(self.lens[b]), [], []
            for i in range(self.N):
                parent = int(torch.randint(-1, i, (1,), generator=self.g)) if i else -1
                sets.append({i} | (sets[parent] if parent >= 0 else set()))
                depth.append(depth[parent] + 1 if parent >= 0 else 0)
            self.mask[b] = words_of(sets, self.N)
            self.pos[b] = torch.tensor([n + d for d in depth], dtype=torch.int32)
            self.slots[b] = torch.tensor([self.slot(b, n + i) for i in range(self.N)], dtype=torch.int32)
            path = sorted(sets[int(torch.randint(0, self.N, (1,), generator=self.g))])
            self.src[b], self.dst[b] = -1, -1
            for k, i in enumerate(path):
                self.src[b, k], self.dst[b, k] = self.slot(b, n + i), self.slot(b, n + k)
            self.accepted[b] = len(path)
        self.x.copy_(torch.randn(self.x.shape, generator=self.g))

    def step(self):
        q, sq = self.append(self.x, self.pos, self.slots)
        y = self.ext.int8_tree_attention_forward_paged(q, self.K, self.V, sq, self.sK, self.sV, self.tables, self.lens,
                                                       self.mask, self.max_context, out_bshd=True)
        self.ext.kv_cache_move_paged(self.K, self.V, self.sK, self.sV, self.src, self.dst)
        self.ext.kv_page_means(self.K, self.sK, self.full, self.M, self.sM)
        out, which = self.ext.int8_decode_attention_forward_paged_sparse(
            self.q1, self.K, self.V, self.sq1, self.sK, self.sV, self.M, self.sM, self.tables, self.lens + self.accepted,
            self.max_context, self.top)
        return q, sq, y, out, which

    def cache(self):
        return [t.clone() for t in (self.K, self.V, self.sK, self.sV)]

    def check(self, before, got):
        """`got` of a step that began with the cache `before`, against the oracle stage by stage."""
        q, sq, y, out, which = (t.cpu().numpy() for t in got)
        K, V, sK, sV = (t.cpu().numpy().copy() for t in before)
        ref = [t.cpu().numpy() for t in self.ext.qk_norm_rope_quantize(self.x, self.H, self.Hkv, self.cos, self.sin, self.pos,
                                                                       self.wq, self.wk)]
        np.testing.assert_array_equal(q, ref[0])
        tables, lens = self.tables.cpu().numpy(), self.lens.cpu().numpy()
        slots = self.slots.cpu().numpy()
        for b in range(self.B):
            for i in range(self.N):
                p, o = slots[b, i] // self.page, slots[b, i] % self.page
                K[p, :, o], sK[p, :, o], V[p, :, o], sV[p, :, o] = (r[b, :, i] for r in ref[2:])
        want, mag = P.tree_attention(q, K, V, sq, sK, sV, tables, lens, self.mask.cpu().numpy(), None, self.max_context)
        vmax = float(127 * sV.max())
        bound = attention_bound(want, mag, self.max_context, vmax)
        assert_within(y, want.transpose(0, 2, 1, 3), bound.transpose(0, 2, 1, 3), "tree")
        for b in range(self.B):
            n, k = int(lens[b]), int(self.accepted[b])
            src = [int(s) for s in self.src[b].tolist()][:k]
            rows = [[t[s // self.page, :, s % self.page].copy() for s in src] for t in (K, V, sK, sV)]
            for j in range(k):
                d = self.slot(b, n + j)
                for t, r in zip((K, V, sK, sV), rows):
                    t[d // self.page, :, d % self.page] = r[j]
        for t, w in zip((self.K, self.V, self.sK, self.sV), (K, V, sK, sV)):
            np.testing.assert_array_equal(t.cpu().numpy(), w)
        M, sM = self.M.cpu().numpy(), self.sM.cpu().numpy()
        ids = [i for i in self.full.tolist() if i >= 0]
        m, sm = P.page_means(K[ids], sK[ids])
        np.testing.assert_array_equal(M[ids], m)
        np.testing.assert_array_equal(sM[ids], sm)
        want, mag, sel = P.sparse_decode(self.q1.cpu().numpy(), K, V, self.sq1.cpu().numpy(), sK, sV, M, sM, tables,
                                         lens + self.accepted.cpu().numpy(), self.max_context, self.top)
        np.testing.assert_array_equal(which, sel)
        assert_within(out, want, attention_bound(want, mag, self.top * self.page, vmax), "sparse")


@pytest.mark.parametrize("H,Hkv,D,page,lens,N,top", [
    (8, 2, 128, 16, [100, 0, 37, 333], 12, 5), (4, 4, 64, 32, [500, 31], 70, 4), (32, 8, 128, 64, [900], 16, 6)])
def test_drafted_steps(ext, gpu, H, Hkv, D, page, lens, N, top):
    s = Step(ext, gpu, H, Hkv, D, page, lens, N, top, seed=N + D)
    s.prompts()
    for _ in range(2):
        s.draft()
        s.full_pages()
        before = s.cache()
        s.check(before, s.step())
    # the same step from one graph, on new drafts, with the eager step between the replays
    graph = torch.cuda.CUDAGraph()
    s.draft()
    s.full_pages()
    with torch.cuda.graph(graph):
        captured = s.step()
    for _ in range(3):
        s.draft()
        s.full_pages()
        before = s.cache()
        graph.replay()
        torch.cuda.synchronize()
        got, after = [t.clone() for t in captured], s.cache()
        s.check(before, got)
        for t, b in zip((s.K, s.V, s.sK, s.sV), before):
            t.copy_(b)
        eager = s.step()
        for a, b in zip(got + after, list(eager) + s.cache()):
            assert torch.equal(a, b)
