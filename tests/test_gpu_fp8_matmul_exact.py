"""GPU: ops.fp8_matmul and fp8_matmul_grouped on products whose every sum is a
whole number below 2^24, which fp32 and the 8-bit products (13 bits below the
largest of each 8) hold exactly: codes of 0, 1 and 2 of either sign, scales of 1
and 2 (at most 4 * 4 a product, 2^18 of them in K = 16384).  Each output is then
the exact number rounded once, bit for bit, in every type and by every kernel."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _whole(dev, g, *shape):
    v = torch.randint(-2, 3, shape, generator=g, device=dev).float()
    return v, v.to(torch.float8_e4m3fn)


def _scales(dev, g, *shape):
    return torch.randint(1, 3, shape, generator=g, device=dev).float()


def _spread(scale, K):
    return scale if scale.shape[-1] == 1 else scale.repeat_interleave(128, -1)[..., :K]


def _exact(a, sa, w, sw):
    N, K = w.shape
    x = (a * _spread(sa, K)).double() @ (w * _spread(sw.repeat_interleave(128, 0)[:N], K)).double().T
    assert float(x.abs().max()) < 2 ** 24
    return x


@pytest.mark.parametrize("rows", [1, 2, 16, 17, 32, 33, 64, 100, 128, 129, 300])
@pytest.mark.parametrize("N,K", [(1, 16), (130, 144), (128, 16384), (600, 4112), (2112, 7168), (33000, 256)])
def test_product_is_exact(dev, rows, N, K):
    from lagged_indexer_dsa_amd import ops

    print(f"[exact] rows={rows} N={N} K={K}", flush=True)
    g = torch.Generator(device=dev).manual_seed(rows * 7 + N)
    av, a = _whole(dev, g, rows, K)
    wv, w = _whole(dev, g, N, K)
    sw = _scales(dev, g, -(-N // 128), -(-K // 128))
    for groups in {1, -(-K // 128)}:
        sa = _scales(dev, g, rows, groups)
        want = _exact(av, sa, wv, sw)
        for dtype in TYPES:
            assert torch.equal(ops.fp8_matmul(a, sa, w, sw, dtype=dtype), want.float().to(dtype)), (groups, dtype)


@pytest.mark.parametrize("counts", [[5], [0, 3, 0, 1, 16, 17, 0], [64, 65, 0, 1], [130, 0, 257, 128, 1, 300], [0, 0, 900, 0],
                                    [2] * 70, [100] * 70, [31] + [1000] + [0] * 40, [1] + [0] * 100 + [300]],
                         ids=lambda c: f"{len(c)}x{max(c)}")
@pytest.mark.parametrize("N,K", [(300, 400), (129, 4096)])
def test_grouped_is_exact(dev, counts, N, K):
    from lagged_indexer_dsa_amd import ops

    print(f"[exact] {counts[:8]} N={N} K={K}", flush=True)
    g = torch.Generator(device=dev).manual_seed(len(counts) + N)
    E, rows = len(counts), sum(counts) + 3
    av, a = _whole(dev, g, rows, K)
    wv, w = _whole(dev, g, E, N, K)
    sa, sw = _scales(dev, g, rows, -(-K // 128)), _scales(dev, g, E, -(-N // 128), -(-K // 128))
    ends = [sum(counts[:e]) for e in range(E + 1)]
    want = torch.full((rows, N), 9.0, dtype=torch.float64, device=dev)
    for e, (i, j) in enumerate(zip(ends, ends[1:])):
        if j > i:
            want[i:j] = _exact(av[i:j], sa[i:j], wv[e], sw[e])
    off = torch.tensor(ends, dtype=torch.int32, device=dev)
    for dtype in TYPES:
        out = torch.full((rows, N), 9.0, dtype=dtype, device=dev)
        ops.fp8_matmul_grouped(a, sa, w, sw, off, out=out)
        assert torch.equal(out, want.float().to(dtype)), dtype
