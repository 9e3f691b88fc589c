"""GPU: a chunk of tokens through PagedDSALayer, and the chunk and 8-bit
operators one after the other as a layer uses them.

The chunk is compared with the same rows taken one at a time by the decode path
(fused_attention_and_indices): both round queries and outputs to bf16 and the
probabilities to one or two bf16 terms, in other orders: 2e-2 of the largest
value, the decode path's own tolerance.  The selections are the exact top-k of
the chunk's own scores, bit for bit; the decode scan's 8-bit products are cut off
13 bits below the largest of 8, so keys next to the threshold may differ.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import dsa_oracle as O

from _cases import rel_err
from test_gpu_paged_layer import _Cfg, _Layer

pytestmark = pytest.mark.gpu


class _Small(_Cfg):
    index_topk = 192


def _layer(dev, seed):
    layer = _Layer(torch.Generator().manual_seed(seed))
    layer.config = _Small()
    return layer.to(dev)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("B,n0,S", [(1, 0, 1), (1, 70, 70), (2, 700, 5), (3, 130, 33)])
def test_chunk_is_its_rows(dev, bits, B, n0, S):
    from lagged_indexer_dsa_amd.paged_layer import PagedDSALayer

    print(f"[chunk layer] B={B} n0={n0} S={S} bits={bits}", flush=True)
    g = torch.Generator().manual_seed(17)
    prefix, x = torch.randn(B, n0, 256, generator=g).to(dev), torch.randn(B, S, 256, generator=g).to(dev)
    with torch.no_grad():
        first, second = _layer(dev, 1), _layer(dev, 2)
        sel = None
        for layer in (first, second):  # dense, then over the first layer's selections
            a = PagedDSALayer(layer, batch=B, max_ctx=n0 + S + 50, device=dev, kv_bits=bits)
            b = PagedDSALayer(layer, batch=B, max_ctx=n0 + S + 50, device=dev, kv_bits=bits)
            if n0:
                a.append(prefix, None)
                b.append(prefix, None)
            h, nxt = a.chunk_attention_and_indices(x, None, sel)
            assert h.shape == x.shape and nxt.shape == (B, S, 192) and nxt.dtype == torch.int64
            assert a.length == n0 + S
            k = 0
            for s in range(S):
                h1, nxt1 = b.fused_attention_and_indices(x[:, s:s + 1], None, None if sel is None else sel[:, s:s + 1])
                assert rel_err(h[:, s].cpu().numpy(), h1[:, 0].cpu().numpy()) < 2e-2, s
                for r in range(B):
                    mine = {p for p in nxt[r, s].tolist() if p < n0 + S}
                    theirs = {p for p in nxt1[r, 0].tolist() if p < n0 + s + 1}
                    assert len(mine) == len(theirs) == min(192, n0 + s + 1) and max(mine) <= n0 + s
                    k += len(mine - theirs)
            assert k <= 0.02 * B * S * 192
            # the caches are those of a plain append of the same rows (one row at a
            # time the projections' own products differ in the last bits)
            c = PagedDSALayer(layer, batch=B, max_ctx=n0 + S + 50, device=dev, kv_bits=bits)
            for part in (prefix, x) if n0 else (x,):
                c.append(part, None)
            assert torch.equal(a.kv_pool, c.kv_pool) and torch.equal(a.index_k, c.index_k)
            none = PagedDSALayer(layer, batch=B, max_ctx=n0 + S, device=dev, kv_bits=bits)
            if n0:
                none.append(prefix, None)
            h2, no = none.chunk_attention_and_indices(x, None, sel, produce_indexer=False)
            assert no is None and torch.equal(h2, h)
            sel = nxt


def test_selection_is_exact(dev):
    """The chunk's selection equals the oracle's top-k of the chunk's scores."""
    from lagged_indexer_dsa_amd import ops
    from lagged_indexer_dsa_amd.paged_layer import PagedDSALayer

    g = torch.Generator().manual_seed(3)
    n0, S = 1000, 40
    with torch.no_grad():
        layer = _layer(dev, 5)
        pl = PagedDSALayer(layer, batch=1, max_ctx=2048, device=dev)
        pl.append(torch.randn(1, n0, 256, generator=g).to(dev), None)
        x = torch.randn(1, S, 256, generator=g).to(dev)
        _, nxt = pl.chunk_attention_and_indices(x, None, None)
        iq, _, w = layer._indexer_qkw(x, layer.q_latent(x), None)
        q8, wf = ops.quantize_index_query(iq.reshape(S, 64, 128).to(torch.bfloat16).contiguous(),
                                          w.reshape(S, 64).float().contiguous())
        sc = ops.chunk_scan(q8, wf, pl.index_k, pl.page_table, torch.tensor([0, S], dtype=torch.int32, device=dev),
                            pl.seq_lens, 1088).cpu().numpy()
        want = O.topk_select(sc, np.arange(n0 + 1, n0 + S + 1), 192)
        for s in range(S):
            assert np.array_equal(nxt[0, s].cpu().numpy(), want[s])


def test_chunk_layer_refusals(dev):
    from lagged_indexer_dsa_amd.paged_layer import PagedDSALayer

    with torch.no_grad():
        pl = PagedDSALayer(_layer(dev, 5), batch=2, max_ctx=100, device=dev)
        x = torch.zeros(2, 3, 256, device=dev)
        for call in (lambda: pl.chunk_attention_and_indices(x[:1], None, None),
                     lambda: pl.chunk_attention_and_indices(x[:, :0], None, None),
                     lambda: pl.chunk_attention_and_indices(x, None, torch.zeros(2, 1, 192, dtype=torch.int64, device=dev)),
                     lambda: pl.chunk_attention_and_indices(torch.zeros(2, 129, 256, device=dev), None, None)):
            with pytest.raises(ValueError):
                call()
        assert pl.length == 0


@pytest.mark.parametrize("bits", [8, 4])
def test_a_layers_step_by_the_operators(dev, bits):
    """Norm and quantiser, the fused projection in 8 bits, rotation and append to
    both caches, scores, select, attention (dense and selected), output
    projection, then a mixture's gated experts: against the same steps in
    float64 on what each operator was given."""
    from lagged_indexer_dsa_amd import formats, ops, rope

    g = torch.Generator(device=dev).manual_seed(11)
    B, H, D = 2, 16, 512
    new, old = [37, 4], [300, 1000]
    n = sum(new)
    lens = [a + b for a, b in zip(new, old)]
    rnd = lambda *s, scale=1.0: torch.randn(*s, generator=g, device=dev) * scale  # noqa: E731
    table = rope.build_rope_table(2048, 64, device=dev)
    pages = sum(-(-m // 64) for m in lens) + 1
    pt = formats.random_page_table(lens, 32, pages, generator=torch.Generator().manual_seed(1)).to(dev)
    pool, index_k = formats.new_latent_pool(pages, dev, bits), formats.new_index_pool(pages, dev)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    # the cached prefixes
    for b in range(B):
        ops.append_tokens(pt, ints([b] * old[b]), ints(range(old[b])), kv_pool=pool, latent=rnd(old[b], 576), index_k=index_k,
                          keys=rnd(old[b], 128), cos_sin=table)
    # the step
    x = rnd(n, D).to(torch.bfloat16)
    wn = torch.ones(D, dtype=torch.bfloat16, device=dev)
    a, sa = ops.rms_norm_quant(x, wn)
    width = H * 576 + 576 + 64 * 128 + 128
    w8, ws = formats.quantize_weight(rnd(width, D, scale=D ** -0.5))
    y = ops.fp8_matmul(a, sa, w8, ws)
    deq = lambda c, s: c.view(torch.float8_e4m3fn).double() * s.double().repeat_interleave(128, -1)[..., :c.shape[-1]]  # noqa: E731
    wv = deq(w8, ws.repeat_interleave(128, 0)[:width])
    ref = deq(a, sa) @ wv.T
    assert float((y.double() - ref).abs().max()) <= (2.0 ** -9 + 2.0 ** -10) * float((deq(a, sa).abs() @ wv.abs().T).max())
    q, kv, iq, ik = y.split([H * 576, 576, 64 * 128, 128], dim=1)
    q = q.reshape(n, H, 576).contiguous()
    rows, pos = ints([b for b in range(B) for _ in range(new[b])]), ints([p for b in range(B) for p in range(old[b], lens[b])])
    ops.rotary(q[..., 512:], pos, table, out=q[..., 512:])
    ops.append_tokens(pt, rows, pos, kv_pool=pool, latent=kv, index_k=index_k, keys=ik, cos_sin=table)
    q8, wf = ops.quantize_index_query(iq.reshape(n, 64, 128).contiguous(), rnd(n, 64, scale=0.125))
    starts, seq = ints([0, new[0], n]), ints(lens)
    scores = ops.chunk_scan(q8, wf, index_k, pt, starts, seq, 2048)
    sel = ops.topk(scores, (pos + 1).to(torch.int32), 256)                      # positions, ascending
    dense = ops.chunk_attention(q, pool, pt, starts, seq)
    slots = torch.where(sel >= 0, pt[rows.long()].gather(1, sel.clamp_min(0).long() // 64) * 64 + sel % 64, -1).to(torch.int32)
    sparse = ops.sparse_mla_decode(q, pool, slots)
    vals = ops.read_latent_rows(pool, torch.arange(pool.shape[0], dtype=torch.int32, device=dev)).double()
    for i in (0, 1, 36, 37, 40):
        b, p = int(rows[i]), int(pos[i])
        everything = pt[b].long()[torch.arange(p + 1, device=dev) // 64] * 64 + torch.arange(p + 1, device=dev) % 64
        assert int((sel[i] >= 0).sum()) == min(256, p + 1) and int(sel[i].max()) <= p
        for got, at in ((dense[i], everything), (sparse[i], slots[i][slots[i] >= 0].long())):
            s = q[i].double() @ vals[at].T * 576 ** -0.5
            want = torch.softmax(s, -1) @ vals[at, :512]
            assert float((got.double() - want).abs().max()) <= 4 * 2.0 ** -9 * float(vals[at, :512].abs().max())
    # experts over the attention's output
    E, inner = 4, 384
    flat = dense.reshape(n, H * 512)[:, :D].contiguous()
    order = torch.randint(0, E, (n,), generator=g, device=dev).sort()[0]
    offsets = torch.searchsorted(order, torch.arange(E + 1, device=dev)).to(torch.int32)
    up8, ups = formats.quantize_weight(rnd(E, 2 * inner, D, scale=D ** -0.5))
    dn8, dns = formats.quantize_weight(rnd(E, D, inner, scale=inner ** -0.5))
    c, sc = ops.quantize_rows(flat)
    gu = ops.fp8_matmul_grouped(c, sc, up8, ups, offsets)
    c2, sc2 = ops.quantize_rows(gu[:, inner:], gate=gu[:, :inner])
    z = ops.fp8_matmul_grouped(c2, sc2, dn8, dns, offsets, dtype=torch.float32)
    for i in range(n):
        e = int(order[i])
        wv = deq(dn8[e], dns[e].repeat_interleave(128, 0)[:D])
        av = deq(c2[i:i + 1], sc2[i:i + 1])[0]
        want, S = wv @ av, wv.abs() @ av.abs()
        assert bool(((z[i].double() - want).abs() <= 270 * 2.0 ** -24 * S).all())
        up = deq(up8[e], ups[e].repeat_interleave(128, 0)[:2 * inner])
        xv = deq(c[i:i + 1], sc[i:i + 1])[0]
        err = (gu[i].double() - up @ xv).abs()
        assert bool((err <= 2.0 ** -9 * (up @ xv).abs() + (2.0 ** -10 + 2.0 ** -15) * (up.abs() @ xv.abs())).all())
