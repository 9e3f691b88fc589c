"""GPU: the chunk and 8-bit operators at ends of their ranges: gates whose
exponential passes fp32's range, outputs between 16-byte boundaries, long chunks
of a layer."""

from __future__ import annotations

import pytest
import torch

from test_gpu_fp8_matmul import _check_quant, _quant_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("group", [128, 0])
def test_gates_far_below_zero(dev, dtype, group):
    """x * g / (1 + e^-g) where the product with a large x is an ordinary number
    though g / (1 + e^-g) is below fp32's normal ones (g < -87.3) or e^-g above its
    largest (g < -88.7): a row a gate, each code with the product's sign."""
    from lagged_indexer_dsa_amd import ops

    g = torch.cat([-torch.arange(1, 84, device=dev), -torch.linspace(84, 100, 129, device=dev),
                   torch.tensor([101.0, 103.0, 105.0, 80.0, 5.0, -101.0, -103.0, -105.0], device=dev)]).to(dtype)
    silu = g.double() * torch.sigmoid(g.double())
    x = (1000 / silu.abs()).clamp_max(3e38).to(dtype)
    x[::2] *= -1
    x, g = x[:, None], g[:, None]
    got = ops.quantize_rows(x, gate=g, group=group)
    _check_quant(got, x, g, group)
    y, code = _quant_ref(x, g), got[0].view(torch.float8_e4m3fn).double()
    assert bool((y.abs() > 1e-6).all()) and bool((code.sign() == y.sign()).all())


def test_gates_below_every_product(dev):
    """Below -150 no x is large enough: codes of 0, the scale its floor's."""
    from lagged_indexer_dsa_amd import ops

    g = -torch.tensor([151.0, 200.0, 1000.0, 1e6, 1e30, 3e38], device=dev)[:, None]
    codes, scales = ops.quantize_rows(torch.full_like(g, 3e38), gate=g)
    assert not bool((codes & 0x7f).any())
    assert bool((scales == torch.tensor(1e-6, device=dev) / 448).all())


@pytest.mark.parametrize("new,lens,heads", [([3], [700], 16), ([2], [9000], 128), ([1], [9000], 16), ([40, 1, 300], [400, 5000, 300], 16)],
                         ids=lambda v: str(v))
def test_attention_into_an_output_between_boundaries(dev, new, lens, heads):
    """out on 8 bytes but not on 16: row tiles of few parts, of many, and whole ones."""
    from lagged_indexer_dsa_amd import ops
    from test_gpu_chunk_attention import _case, _check, _run

    c = _case(dev, 21, new, lens, heads, 8)
    want = _run(ops, c)
    _check(want, c, lens, ops)
    buf = torch.full((want.numel() + 12,), 3.0, dtype=torch.bfloat16, device=dev)
    out = buf[4:4 + want.numel()].view(want.shape)
    assert buf.data_ptr() % 16 == 0 and out.data_ptr() % 16 == 8
    _run(ops, c, out=out)
    assert torch.equal(out, want) and bool((buf[:4] == 3).all()) and bool((buf[-8:] == 3).all())
    with pytest.raises(RuntimeError, match="8-byte"):
        _run(ops, c, out=buf[1:1 + want.numel()].view(want.shape))


def _paged(dev, topk, batch, max_ctx, bits=8):
    from lagged_indexer_dsa_amd.paged_layer import PagedDSALayer
    from test_gpu_paged_layer import _Cfg, _Layer

    layer = _Layer(torch.Generator().manual_seed(6))
    layer.config = type("Small", (_Cfg,), dict(index_topk=topk))()
    return PagedDSALayer(layer.to(dev), batch=batch, max_ctx=max_ctx, device=dev, kv_bits=bits)


@pytest.mark.parametrize("bits", [8, 4])
def test_a_chunk_in_several_launches(dev, bits, monkeypatch):
    """Attention over selections and selection a few rows at a time: the selections
    of all rows at once, and the attention but for where its sums are cut (fp32 sums
    joined in another order, and the output's rounding to bf16: 2^-8 of the largest
    value, before a projection of 512 of them)."""
    from _cases import rel_err
    from lagged_indexer_dsa_amd import paged_layer

    g = torch.Generator().manual_seed(2)
    B, n0, S = 2, 300, 23
    prefix, x = torch.randn(B, n0, 256, generator=g).to(dev), torch.randn(B, S, 256, generator=g).to(dev)

    def step(sel):
        pl = _paged(dev, 64, B, n0 + S, bits)
        pl.append(prefix, None)
        return pl.chunk_attention_and_indices(x, None, sel)

    with torch.no_grad():
        _, sel = step(None)
        want = step(sel)
        for rows, scores in ((65535, 2 * 5 * 384), (9, 1 << 28), (1, 1)):
            monkeypatch.setattr(paged_layer, "MAX_ROWS", rows)
            monkeypatch.setattr(paged_layer, "MAX_SCORES", scores)
            got = step(sel)
            assert torch.equal(got[1], want[1]), (rows, scores)
            assert rel_err(got[0].cpu().numpy(), want[0].cpu().numpy()) < 2.0 ** -7, (rows, scores)


def test_a_chunk_of_more_rows_than_a_launch_takes(dev):
    """66000 tokens at once, dense and over selections: their selections are the
    exact ones of their own scores."""
    import numpy as np

    from lagged_indexer_dsa_amd import ops
    from oracle import dsa_oracle as O

    S, k = 66000, 64
    x = torch.randn(1, S, 256, generator=torch.Generator().manual_seed(4)).to(dev)
    sel = None
    with torch.no_grad():
        for i in range(2):
            print(f"[long chunk] pass {i}", flush=True)
            pl = _paged(dev, k, 1, S)
            h, sel = pl.chunk_attention_and_indices(x, None, sel)
            assert h.shape == x.shape and sel.shape == (1, S, k) and pl.length == S
        iq, _, w = pl.layer._indexer_qkw(x, pl.layer.q_latent(x), None)
        for r in (0, 5, 4063, 4064, 65534, 65535, 65999):
            q8, wf = ops.quantize_index_query(iq[:, r].to(torch.bfloat16).contiguous(), w[:, r].float().contiguous())
            sc = ops.chunk_scan(q8, wf, pl.index_k, pl.page_table, torch.tensor([0, 1], dtype=torch.int32, device=dev),
                                torch.tensor([r + 1], dtype=torch.int32, device=dev), pl.cap)
            want = O.topk_select(sc.cpu().numpy(), np.array([r + 1]), k)[0]
            want = np.where(want < 0, S, want)
            assert np.array_equal(np.sort(want), sel[0, r].cpu().numpy()), r
