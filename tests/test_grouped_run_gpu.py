"""The grouped-query serving operators as a model's layer runs them (GPU): prompts through
int8_linear, the heads, packed attention and the output projection while their keys and values
enter the 4-bit cache, then a decode step against it.  Every stage is checked against the
64-bit oracle on what the stage before handed it, and the whole run is captured and replayed."""
import numpy as np
import pytest
import torch

import int8k_capi as capi
from grouped_helpers import assert_within, attention_bound, np64, quantize_rows, rows
from oracle import grouped_oracle as G
from test_heads_gpu import _bound as heads_bound
from test_heads_gpu import _tables
from test_linear_gpu import _bound as linear_bound

pytestmark = pytest.mark.gpu

EPS = 1e-6


class Layer:
    """One attention layer with a 4-bit cache; every tensor a captured run reads keeps its place."""

    def __init__(self, ext, gpu, E, H, Hkv, D, rot, page, T, B, dt, inter):
        g = torch.Generator().manual_seed(E + D)
        self.ext, self.H, self.Hkv, self.D, self.dt, self.inter = ext, H, Hkv, D, dt, inter
        self.page, self.T, self.B, self.rot = page, T, B, rot
        self.w_in, self.s_in = quantize_rows(torch.randn((H + 2 * Hkv) * D, E, generator=g) * 0.05)
        self.w_out, self.s_out = quantize_rows(torch.randn(E, H * D, generator=g) * 0.05)
        self.bias = torch.randn((H + 2 * Hkv) * D, generator=g)
        self.cos, self.sin = _tables(rot // 2)
        self.wq, self.wk = torch.rand(D, generator=g) + 0.5, torch.rand(D, generator=g) + 0.5
        for n in ("w_in", "s_in", "w_out", "s_out", "bias", "cos", "sin", "wq", "wk"):
            setattr(self, n, getattr(self, n).to(gpu))
        self.cols = -(-(T + 1) // page)
        pages = B * self.cols + 1
        self.tables = torch.randperm(pages - 1, generator=g)[:B * self.cols].view(B, -1).to(torch.int32).to(gpu)
        self.K = torch.zeros(pages, Hkv, page, D // 2, dtype=torch.uint8, device=gpu)
        self.V = torch.zeros_like(self.K)
        self.sK = torch.zeros(pages, Hkv, page, device=gpu)
        self.sV = torch.zeros_like(self.sK)
        i32 = dict(dtype=torch.int32, device=gpu)
        self.x = torch.zeros(T, E, dtype=torch.float16, device=gpu)
        self.x1 = torch.zeros(B, E, dtype=torch.float16, device=gpu)
        self.cu, self.pos, self.slots = torch.zeros(B + 1, **i32), torch.zeros(T, **i32), torch.zeros(T, **i32)
        self.pos1, self.slots1, self.lens = (torch.zeros(B, **i32) for _ in range(3))

    def load(self, lens, seed):
        """New prompts of these lengths; tokens past the last one are padding."""
        g = torch.Generator().manual_seed(seed)
        cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        tables = self.tables.cpu().numpy()
        pos, slots = np.zeros(self.T, np.int32), np.full(self.T, -1, np.int32)
        for b, n in enumerate(lens):
            i = np.arange(n)
            pos[cu[b]:cu[b + 1]] = i
            slots[cu[b]:cu[b + 1]] = tables[b, i // self.page] * self.page + i % self.page
        n = np.array(lens)
        self.x.copy_(rows(g, *self.x.shape))
        self.x1.copy_(rows(g, *self.x1.shape))
        for t, v in ((self.cu, cu), (self.pos, pos), (self.slots, slots), (self.pos1, n), (self.lens, n + 1),
                     (self.slots1, tables[np.arange(self.B), n // self.page] * self.page + n % self.page)):
            t.copy_(torch.from_numpy(np.ascontiguousarray(v)).to(torch.int32))

    def clear(self):
        for t in (self.K, self.V, self.sK, self.sV):
            t.zero_()

    def project(self, x):
        q, s = self.ext.quantize_per_token(x)
        y = self.ext.int8_linear(q, self.w_in, s, self.s_in, bias=self.bias, prepacked=True, dtype=self.dt)
        return dict(xq=q, sx=s, y=y)

    def close(self, a, r):
        r["aq"], r["sa"] = self.ext.quantize_per_token(a.reshape(a.shape[0], -1))
        r["z"] = self.ext.int8_linear(r["aq"], self.w_out, r["sa"], self.s_out, prepacked=True, dtype=self.dt)
        return r

    def heads(self, y, pos, quantize):
        f = self.ext.qk_norm_rope_quantize if quantize else self.ext.qk_norm_rope
        return f(y, self.H, self.Hkv, self.cos, self.sin, pos, q_weight=self.wq, k_weight=self.wk, eps=EPS,
                 interleaved=self.inter)

    def prompts(self):
        r = self.project(self.x)
        r["heads"] = self.heads(r["y"], self.pos, False)
        r["q"], r["sq"], r["k"], r["sk"], r["v"], r["sv"] = self.heads(r["y"], self.pos, True)
        _, k, v = r["heads"]
        self.ext.kv4_cache_append(k.transpose(0, 1), v.transpose(0, 1), self.K, self.V, self.sK, self.sV, self.slots)
        r["a"] = self.ext.int8_attention_forward_packed(r["q"], r["k"], r["v"], r["sq"], r["sk"], r["sv"], self.cu,
                                                        True, True)
        return self.close(r["a"], r)

    def decode(self):
        r = self.project(self.x1)
        y = r["y"].view(self.B, 1, -1)
        pos = self.pos1.view(self.B, 1)
        r["heads"] = self.heads(y, pos, False)
        _, k, v = r["heads"]
        self.ext.kv4_cache_append(k[:, :, 0], v[:, :, 0], self.K, self.V, self.sK, self.sV, self.slots1)
        q, s = self.heads(y, pos, True)[:2]
        r["q"], r["sq"] = q[:, :, 0].contiguous(), s[:, :, 0].contiguous()
        r["a"] = self.ext.int8_decode_attention_forward_kv4_paged(
            r["q"], self.K, self.V, r["sq"], self.sK, self.sV, self.tables, self.lens, self.T + 1)
        return self.close(r["a"], r)

    # ---- checks

    def check_linear(self, q, s, w, sw, bias, y, label):
        ref, mag = G.linear(q.cpu().numpy(), w.t().cpu().numpy(), s.cpu().numpy(), sw.cpu().numpy(),
                            None if bias is None else bias.cpu().numpy())
        assert_within(np64(y), ref, linear_bound(ref, mag, bias, self.dt), label)

    def check_common(self, r, pos, label):
        self.check_linear(r["xq"], r["sx"], self.w_in, self.s_in, self.bias, r["y"], label + " qkv")
        self.check_linear(r["aq"], r["sa"], self.w_out, self.s_out, None, r["z"], label + " out")
        rows_ = r["y"].reshape(*pos.shape, -1)
        ref = G.qk_norm_rope(np64(rows_), self.H, self.Hkv, self.cos.cpu().numpy(), self.sin.cpu().numpy(),
                             pos.cpu().numpy(), self.wq.cpu().numpy(), self.wk.cpu().numpy(), EPS, self.inter)
        for i in range(3):
            assert_within(np64(r["heads"][i]).reshape(ref[i].shape), ref[i],
                          heads_bound(ref[i], self.D, self.rot // 2, self.inter, self.dt, i < 2), f"{label} {'qkv'[i]}")

    def check_prompts(self, r, lens):
        self.check_common(r, self.pos.view(1, -1), "prompts")
        c = [r[n].cpu().numpy() for n in ("q", "k", "v", "sq", "sk", "sv")]
        ref, mag = G.packed_attention(*c, self.cu.cpu().numpy(), True)
        vmax = float((r["v"].float().abs().amax(-1) * r["sv"]).max())
        assert_within(np64(r["a"]).transpose(1, 0, 2), ref, attention_bound(ref, mag, max(lens), vmax), "packed")
        assert not r["a"][sum(lens):].any()  # padding
        _, k, v = r["heads"]
        at = self.slots[:sum(lens)].cpu().numpy()
        for x, pages, scales in ((k, self.K, self.sK), (v, self.V, self.sV)):
            codes, s = G.kv4_quantize(x.float().transpose(0, 1)[:sum(lens)].cpu().numpy())
            np.testing.assert_array_equal(pages.cpu().numpy()[at // self.page, :, at % self.page], G.kv4_pack(codes))
            np.testing.assert_array_equal(scales.cpu().numpy()[at // self.page, :, at % self.page], s)

    def check_decode(self, r):
        self.check_common(r, self.pos1.view(self.B, 1), "decode")
        ref, mag = G.kv4_decode(*(t.cpu().numpy() for t in (r["q"], self.K, self.V, r["sq"], self.sK, self.sV,
                                                             self.tables, self.lens)))
        bound = attention_bound(ref, mag, int(self.lens.max()), float(7 * self.sV.max()))
        assert_within(np64(r["a"]), ref, bound, "decode attention")


CASES = [dict(E=512, H=8, Hkv=2, D=64, rot=64, page=16, T=190, dt=torch.float16, inter=False),
         dict(E=1024, H=12, Hkv=4, D=128, rot=64, page=64, T=450, dt=torch.bfloat16, inter=True)]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"D{c['D']}")
def test_layer_stage_by_stage(ext, gpu, case):
    layer = Layer(ext, gpu, B=4, **case)
    counts = capi.kv4_bad_ids(), capi.rope_bad_positions()
    for seed, lens in enumerate(([40, 1, 0, 133], [0, 0, 0, 3], [layer.page, 2 * layer.page, 17, 90])):
        layer.load(lens, seed)
        layer.check_prompts(layer.prompts(), lens)
        layer.check_decode(layer.decode())
    assert (capi.kv4_bad_ids(), capi.rope_bad_positions()) == counts


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"D{c['D']}")
def test_layer_captured_beside_another(ext, gpu, case):
    """Two layers, each captured on a stream of its own, replayed over each other with lengths
    and inputs that change between the replays."""
    layers = [Layer(ext, gpu, B=4, **case) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in layers]
    graphs, outs = [], []
    for k, layer in enumerate(layers):
        layer.load([20, 30, 5, 1], k)
        layer.prompts(), layer.decode()  # libraries and workspaces are up before the capture
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[k]):
            p, d = layer.prompts(), layer.decode()
        graphs.append(g)
        outs.append((p["a"], p["z"], d["a"], d["z"], layer.K, layer.sV))
    torch.cuda.synchronize()
    for seed, lens in enumerate(([40, 1, 0, 133], [0, 0, 0, 3], [64, 30, 17, 70])):
        want = []
        for k, layer in enumerate(layers):
            layer.load(lens[::1 - 2 * k], 10 * seed + k)
            layer.clear()
            p, d = layer.prompts(), layer.decode()
            want.append([t.clone() for t in (p["a"], p["z"], d["a"], d["z"], layer.K, layer.sV)])
            layer.clear()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for k in range(2):
            for i, (a, b) in enumerate(zip(outs[k], want[k])):
                assert torch.equal(a, b), (seed, k, i)
