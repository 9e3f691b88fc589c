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
