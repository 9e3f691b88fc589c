"""GPU: the operators together, as a layer's step runs them: norm with the
residual, rotation of the queries, append with norm and rotation, attention
over the 4-bit cache, reading the cache back for a prompt's next chunk; under a
captured graph and on another stream; and PagedDSALayer with a 4-bit pool."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import dsa_oracle as O
from test_gpu_paged_layer import _Layer

pytestmark = pytest.mark.gpu


class _Step:
    """One decode step of B requests with fixed buffers."""

    def __init__(self, dev, B=3, H=16, ctx=500, hidden=1024, seed=1):
        from lagged_indexer_dsa_amd import formats as F
        from lagged_indexer_dsa_amd import ops
        from lagged_indexer_dsa_amd.rope import build_rope_table

        g = torch.Generator(device=dev).manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
        bf = torch.bfloat16
        self.B, self.H, self.npg = B, H, 10
        self.table = build_rope_table(1024, 64, device=dev)
        self.x, self.res = r(B, hidden).to(bf), r(B, hidden).to(bf)
        self.w, self.cw = (1 + 0.1 * r(hidden)).to(bf), (1 + 0.1 * r(512)).to(bf)
        self.wkv, self.wq = (r(hidden, 576) / hidden ** 0.5).to(bf), (r(hidden, H * 192) / hidden ** 0.5).to(bf)
        self.wik = (r(hidden, 128) / hidden ** 0.5).to(bf)
        self.uk = (r(128, 512) / 128 ** 0.5).to(bf)
        self.pt = torch.randperm(B * self.npg, generator=g, device=dev).int().reshape(B, self.npg)
        self.pool, self.index_k = F.new_latent_pool(B * self.npg, dev, bits=4), F.new_index_pool(B * self.npg, dev)
        self.rows = torch.arange(B, dtype=torch.int32, device=dev)
        # the cached prefix
        n = torch.tensor([ctx - 100 * b for b in range(B)], device=dev)
        pr = self.rows.repeat_interleave(n)
        pp = torch.cat([torch.arange(int(k), device=dev) for k in n]).int()
        ops.append_tokens(self.pt, pr, pp, kv_pool=self.pool, latent=r(len(pp), 576).to(bf), index_k=self.index_k,
                          keys=r(len(pp), 128).to(bf), cos_sin=self.table, norm_weight=self.cw, interleaved=True)
        self.pos = n.int()
        self.lens = n.int() + 1
        self.q = torch.zeros(B, H, 576, dtype=bf, device=dev)
        self.ws = ops.sparse_mla_workspace(B, H, 0, dev)
        self.out = torch.zeros(B, H, 512, dtype=bf, device=dev)
        self.start = (self.pos.clone(), self.lens.clone(), self.pool.clone(), self.index_k.clone(), self.res.clone())

    def reset(self):
        for t, s in zip((self.pos, self.lens, self.pool, self.index_k, self.res), self.start):
            t.copy_(s)

    def run(self):
        from lagged_indexer_dsa_amd import ops

        y, _ = ops.rms_norm(self.x, self.w, residual=self.res, out_residual=self.res)
        q = (y @ self.wq).view(self.B, self.H, 192)
        self.q[..., :512] = q[..., :128] @ self.uk
        ops.rotary(q[..., 128:], self.pos, self.table, interleaved=True, out=self.q[..., 512:])
        ops.append_tokens(self.pt, self.rows, self.pos, kv_pool=self.pool, latent=y @ self.wkv, index_k=self.index_k,
                          keys=y @ self.wik, cos_sin=self.table, norm_weight=self.cw, interleaved=True)
        ops.dense_mla_decode(self.q, self.pool, self.pt, self.lens, workspace=self.ws, out=self.out)
        self.pos += 1
        self.lens += 1
        return y


def test_a_step_against_the_oracle(dev):
    print("[layer ops] step", flush=True)
    s = _Step(dev)
    res0, pos0 = s.res.double().cpu().numpy(), s.pos.cpu().numpy()
    y = s.run()
    n = lambda t: t.double().cpu().numpy()  # noqa: E731
    yr, h = O.rms_norm(n(s.x), n(s.w), 1e-6, res0)
    assert np.all(np.abs(n(y) - yr) <= (2.0 ** -8 + 2.0 ** -18) * np.abs(yr))
    assert np.all(np.abs(n(s.res) - h) <= (2.0 ** -8 + 2.0 ** -23) * np.abs(h))
    t = n(s.table)[pos0]
    # the new rows, from the projections that were stored
    kv, ik = n(y @ s.wkv), n(y @ s.wik)
    pt = s.pt.cpu().numpy()
    slots = pt[np.arange(3), pos0 // 64] * 64 + pos0 % 64
    rows = s.pool.cpu().numpy()[slots]
    ref = O.pack_latent_rows_fp4(O.rms_norm(kv[:, :512], n(s.cw), 1e-6)[0].astype(np.float32), np.zeros((3, 64)))
    assert np.array_equal(rows[:, :272], ref[:, :272])
    rope = O.rotate(kv[:, 512:], t[:, :32], t[:, 32:], True)
    got = O.bf16_from_bits(rows[:, 272:].copy().view(np.uint16)).astype(np.float64)
    assert np.all(np.abs(got - rope) <= 2.0 ** -8 * np.abs(rope) + 2.0 ** -22 * np.abs(kv).max())
    kr = np.concatenate([O.rotate(ik[:, :64], t[:, :32], t[:, 32:], False), ik[:, 64:]], 1)
    pages = s.index_k.cpu().numpy()
    codes = pages[:, :8192].reshape(-1, 64, 128)[slots // 64, slots % 64]
    scale = pages[:, 8192:].copy().view(np.float32)[slots // 64, slots % 64][:, None].astype(np.float64)
    assert np.all(np.abs(O.e4m3_decode(codes) * scale - kr) <= 2.0 ** -4 * np.abs(kr) + 2.0 ** -9 * scale)
    # the attention over what the cache now holds
    kvs = O.dequant_latent_rows_fp4(s.pool.cpu().numpy())
    idx = np.full((3, 640), -1)
    for b in range(3):
        j = np.arange(pos0[b] + 1)
        idx[b, :len(j)] = pt[b, j // 64] * 64 + j % 64
    q = n(s.q)
    ref = O.mla_decode_values(q, kvs, idx, 576 ** -0.5)
    for b in range(3):
        k = kvs[idx[b][idx[b] >= 0]].astype(np.float64)
        p = np.exp(q[b] @ k.T * 576 ** -0.5)
        mag = p @ np.abs(k[:, :512]) / p.sum(-1, keepdims=True)
        assert np.all(np.abs(n(s.out)[b] - ref[b]) <= 2.0 ** -7 * np.abs(ref[b]) + 2.0 ** -8 * (1 + 2.0 ** -4) * mag)


def test_a_captured_step_replays_like_the_eager_one(dev):
    print("[layer ops] graph", flush=True)
    s = _Step(dev, seed=2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.run()                                             # warm up, on another stream than the current one
    torch.cuda.current_stream().wait_stream(side)
    want = []
    s.reset()
    for _ in range(4):
        s.run()
        want.append((s.out.clone(), s.res.clone(), s.pool.clone(), s.index_k.clone()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.run()
    s.reset()
    for k in range(4):
        graph.replay()
        torch.cuda.synchronize()
        noise = torch.randn(1 << 20, device=dev).sum()      # the program's own work between replays
        for got, ref in zip((s.out, s.res, s.pool, s.index_k), want[k]):
            assert torch.equal(got, ref), f"replay {k}"
        assert noise.isfinite()


def test_cache_read_back_for_a_prompt_chunk(dev):
    """A chunk of queries over cached 4-bit rows: read back, then the prefill
    attention against float64.  That op holds its keys in 8 bits and its
    probabilities in bf16 at least: the reference is over the 8-bit values, a
    probability off by 2^-8, the output rounded once."""
    from lagged_indexer_dsa_amd import attention_core as A
    from lagged_indexer_dsa_amd import ops

    print("[layer ops] read back", flush=True)
    s = _Step(dev, seed=3)
    T, S = 400, 24
    j = torch.arange(T, device=dev)
    kv = ops.read_latent_rows(s.pool, (s.pt[0].long()[j // 64] * 64 + j % 64).int())
    assert np.array_equal(kv.float().cpu().numpy(),
                          O.dequant_latent_rows_fp4(s.pool.cpu().numpy()[(s.pt[0].long()[j // 64] * 64 + j % 64).cpu().numpy()]))
    q = torch.randn(1, S, 16, 576, device=dev, generator=torch.Generator(device=dev).manual_seed(4)).to(torch.bfloat16)
    out = A.dense_mla_core(q, kv[None], 512)[0].double().cpu().numpy()
    kf = kv.float().cpu().numpy()
    kall = O.dequant_latent_rows(O.pack_latent_rows(kf[:, :512], kf[:, 512:])).astype(np.float64)
    for i in range(S):
        k = kall[:T - S + i + 1]
        p = np.exp(q[0, i].double().cpu().numpy() @ k.T * 576 ** -0.5)
        p /= p.sum(-1, keepdims=True)
        ref = p @ k[:, :512]
        assert np.all(np.abs(out[i] - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -8 * (p @ np.abs(k[:, :512])))


@pytest.mark.parametrize("batch", [1, 2])
def test_paged_layer_with_a_4bit_pool(dev, batch):
    from lagged_indexer_dsa_amd import _lib
    from lagged_indexer_dsa_amd.paged_layer import PagedDSALayer

    print("[layer ops] paged layer", flush=True)
    g = torch.Generator().manual_seed(7)
    layer = _Layer(g).to(dev)
    n0 = 3000
    xs = torch.randn(batch, n0, 256, generator=g).to(dev)
    steps = [torch.randn(batch, 1, 256, generator=g).to(dev) for _ in range(3)]
    with torch.no_grad():
        p4, p8 = (PagedDSALayer(layer, batch=batch, max_ctx=4096, device=dev, kv_bits=b) for b in (4, 8))
        for p in (p4, p8):
            p.append(xs, None)
        _lib.sync_timeouts(reset=True)
        att = None
        for i, x in enumerate(steps):
            h4, s4 = p4.fused_attention_and_indices(x, None, att, produce_indexer=i < 2)
            h8, s8 = p8.fused_attention_and_indices(x, None, att, produce_indexer=i < 2)
            assert torch.equal(p4.index_k, p8.index_k)       # the same keys, so the same selections
            if i < 2:
                assert torch.equal(s4, s8)
            else:
                assert s4 is None
            kv = O.dequant_latent_rows_fp4(p4.kv_pool.cpu().numpy())
            if att is None:
                idx = (np.arange(batch)[:, None] * p4.cap + np.arange(p4.length)[None]).astype(np.int64)
            else:
                idx = p4.attend.cpu().numpy()
            q = layer._mla_qkv(x, layer.q_latent(x), None)[0].reshape(batch, 16, 576).to(torch.bfloat16)
            ref = O.mla_decode_values(q.double().cpu().numpy(), kv, idx, 576 ** -0.5)
            assert np.abs(p4.out.double().cpu().numpy() - ref).max() <= 2.0 ** -7 * np.abs(ref).max()
            assert float((h4 - h8).norm() / h8.norm()) < 0.5
            att = s4
        assert _lib.sync_timeouts() == 0
        with pytest.raises(ValueError):
            PagedDSALayer(layer, batch=1, max_ctx=64, device=dev, kv_bits=5)


def test_paged_layers_keep_the_same_index_keys(dev):
    """Keys with a NaN or an infinity too: the index cache, and so the selection,
    is the same with latent rows of 8 and of 4 bits."""
    from lagged_indexer_dsa_amd.paged_layer import PagedDSALayer

    print("[layer ops] index keys with NaN", flush=True)
    layer = _Layer(torch.Generator().manual_seed(7)).to(dev)
    g = torch.Generator(device=dev).manual_seed(3)
    keys, kv = torch.randn(2, 70, 128, device=dev, generator=g), torch.randn(2, 70, 576, device=dev, generator=g)
    keys[0, 3, 17], keys[1, 69, 100], keys[1, 5, 0] = float("nan"), float("nan"), float("inf")
    keys[0, 64] = float("nan")
    p4, p8 = (PagedDSALayer(layer, batch=2, max_ctx=128, device=dev, kv_bits=b) for b in (4, 8))
    for p in (p4, p8):
        p._append(keys[:, :69], kv[:, :69])
        p._append(keys[:, 69:], kv[:, 69:])
    assert torch.equal(p4.index_k, p8.index_k) and bool(p4.index_k.any())
    back = O.dequant_latent_rows_fp4(p4.kv_pool.cpu().numpy())
    ref = O.pack_latent_rows_fp4(kv[:, :, :512].to(torch.bfloat16).float().cpu().numpy().reshape(140, 512),
                                 kv[:, :, 512:].float().cpu().numpy().reshape(140, 64))
    rows = np.r_[0:70, 128:198]
    assert np.array_equal(back[rows], O.dequant_latent_rows_fp4(ref))
