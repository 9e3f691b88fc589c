"""GPU: ops.rms_norm, ops.rms_norm_quant and ops.rotary against float64.

Bounds.  A result is rounded once to its type (half a step: eps / 2 of the
value); before that, in fp32: the sum of squares is a chain of at most 32 terms
a lane and 10 levels of a tree (42 roundings, halved by the root), the root,
the quotient (2 steps each) and two products: under 32 * 2^-24 of the value.
A code is within half a step of value / scale (2^-4 of it, or 2^-10 scales).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import dsa_oracle as O

pytestmark = pytest.mark.gpu

F32 = 32 * 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _near(got: torch.Tensor, ref: np.ndarray, extra: float = F32) -> None:
    f = torch.finfo(got.dtype)
    err = np.abs(got.double().cpu().numpy() - ref)
    bound = (f.eps / 2 + extra) * np.abs(ref) + f.smallest_normal * f.eps
    assert np.all(err <= bound), (float((err / np.maximum(bound, 1e-300)).max()), np.argwhere(err > bound)[:3])


def _rand(dev, g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)


def _codes_near(codes, scales, y, group):
    """codes [n, D], scales [n, G] against y [n, D] float64."""
    n, D = y.shape
    group = group or D
    c = codes.view(torch.float8_e4m3fn).double().cpu().numpy()
    s = scales.double().cpu().numpy()
    for k, a in enumerate(range(0, D, group)):
        part = y[:, a:a + group]
        top = np.maximum(np.abs(part).max(1), 1e-6) / 448
        assert np.all(np.abs(s[:, k] - top) <= (F32 + 2.0 ** -22) * top), "scale"
        sk = s[:, k:k + 1]
        err = np.abs(c[:, a:a + group] * sk - part)
        assert np.all(err <= (2.0 ** -4 + F32) * np.abs(part) + 2.0 ** -10 * sk), "codes"


DIMS = [1, 2, 63, 64, 128, 130, 256, 512, 520, 1000, 1024, 1111, 1536, 2048, 2056, 4096, 5000, 7168, 8192, 8200, 12289,
        16384, 18432, 32768]


@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_norm_all_widths(dev, D, dtype):
    print(f"[norm] D={D} {dtype}", flush=True)
    from lagged_indexer_dsa_amd import ops

    g = torch.Generator(device=dev).manual_seed(D)
    for n in (1, 7):
        x, r = _rand(dev, g, n, D, dtype=dtype), _rand(dev, g, n, D, dtype=dtype, scale=3)
        w = 1 + _rand(dev, g, D, scale=0.3)
        for wt in (w, w.to(dtype)):
            y = ops.rms_norm(x, wt)
            ref, _ = O.rms_norm(x.double().cpu().numpy(), wt.double().cpu().numpy(), 1e-6)
            _near(y, ref)
        y, h = ops.rms_norm(x, wt, eps=1e-3, residual=r)
        ref, href = O.rms_norm(x.double().cpu().numpy(), wt.double().cpu().numpy(), 1e-3, r.double().cpu().numpy())
        # the fp32 sum x + r is off by 2^-24 of itself at most
        _near(y, ref, F32 + 2.0 ** -23)
        _near(h, href, 2.0 ** -24)
        for group in (128, 0):
            codes, scales, h2 = ops.rms_norm_quant(x, wt, eps=1e-3, residual=r, group=group)
            assert scales.shape == (n, -(-D // 128) if group else 1)
            assert torch.equal(h2, h)
            _codes_near(codes, scales, ref, group)


def test_norm_many_rows_and_strides(dev):
    from lagged_indexer_dsa_amd import ops

    print("[norm] strides", flush=True)
    g = torch.Generator(device=dev).manual_seed(3)
    wide = _rand(dev, g, 2, 1000, 2112, dtype=torch.bfloat16)
    w = _rand(dev, g, 1536, dtype=torch.bfloat16)
    for x in (wide[..., :1536], wide[..., 3:1539], wide[1, :, 576:], wide[:, ::2, :1536].reshape(-1, 1536),
              wide[0, ::3, 8:1544]):
        y = ops.rms_norm(x, w)
        ref, _ = O.rms_norm(x.double().cpu().numpy(), w.double().cpu().numpy(), 1e-6)
        assert y.shape == x.shape and y.is_contiguous()
        _near(y, ref)
    # a broadcast row, as input and as residual
    row = wide[0, :1, :1536].expand(5, 1536)
    x = wide[0, :5, 1:1537]
    y, h = ops.rms_norm(x, w, residual=row)
    ref, href = O.rms_norm(x.double().cpu().numpy(), w.double().cpu().numpy(), 1e-6, row.double().cpu().numpy())
    _near(y, ref, F32 + 2.0 ** -23)
    _near(h, href, 2.0 ** -24)
    # the residual updated in place, the given outputs used
    r = _rand(dev, g, 40, 512, dtype=torch.float16)
    x = _rand(dev, g, 40, 512, dtype=torch.float16)
    w = torch.ones(512, device=dev)
    y0, h0 = ops.rms_norm(x, w, residual=r)
    out = torch.empty_like(x)
    y1, h1 = ops.rms_norm(x, w, residual=r, out=out, out_residual=r)
    assert y1.data_ptr() == out.data_ptr() and h1.data_ptr() == r.data_ptr()
    assert torch.equal(y0, y1) and torch.equal(h0, r)
    # rows that are strided within a larger residual stream, the rest untouched
    stream = _rand(dev, g, 40, 600, dtype=torch.float16)
    keep = stream.clone()
    ops.rms_norm(x, w, residual=stream[:, 40:552], out_residual=stream[:, 40:552])
    assert torch.equal(stream[:, :40], keep[:, :40]) and torch.equal(stream[:, 552:], keep[:, 552:])
    assert torch.equal(stream[:, 40:552], (keep[:, 40:552].float() + x.float()).half())


@pytest.mark.parametrize("n,D", [(3, 9), (5000, 301), (70, 3001), (9, 9999)])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_norm_rows_between_boundaries(dev, n, D, dtype):
    """Rows, weights and outputs that begin anywhere: the same bits as from
    boundaries, in place too, and nothing beside them written."""
    from lagged_indexer_dsa_amd import ops

    print(f"[norm] between boundaries {(n, D, dtype)}", flush=True)
    g = torch.Generator(device=dev).manual_seed(n)
    E = -(-D // 8) * 8 + 16
    x, r = _rand(dev, g, n, D, dtype=dtype), _rand(dev, g, n, D, dtype=dtype)
    w = _rand(dev, g, D + 1, dtype=dtype)[1:]
    xa, ra, wa = torch.zeros(n, E, dtype=dtype, device=dev), torch.zeros(n, E, dtype=dtype, device=dev), w.clone()
    xa[:, :D], ra[:, :D] = x, r
    y, h = ops.rms_norm(xa[:, :D], wa, residual=ra[:, :D])           # rows on boundaries
    ref, _ = O.rms_norm(x.double().cpu().numpy(), w.double().cpu().numpy(), 1e-6, r.double().cpu().numpy())
    _near(y, ref, F32 + 2.0 ** -23)  # (the sum x + r is off by 2^-24 of itself)
    for off in (1, 3):
        wide = torch.full((n, D + 7), 5.0, dtype=dtype, device=dev)
        wide[:, off:off + D] = r
        big = torch.full((n * D + 16,), 5.0, dtype=dtype, device=dev)
        out = big[off:off + n * D].view(n, D)
        y2, h2 = ops.rms_norm(x, w, residual=wide[:, off:off + D], out=out, out_residual=wide[:, off:off + D])
        assert torch.equal(y2, y) and torch.equal(h2, h)
        assert (wide[:, :off] == 5).all() and (wide[:, off + D:] == 5).all()
        assert (big[:off] == 5).all() and (big[off + n * D:] == 5).all()
        for group in (128, 0):
            c0, s0, _ = ops.rms_norm_quant(xa[:, :D], wa, residual=ra[:, :D], group=group)
            cb = torch.full((n * D + 16,), 9, dtype=torch.uint8, device=dev)
            c1, s1, _ = ops.rms_norm_quant(x, w, residual=r, group=group, out_q=cb[off:off + n * D].view(n, D))
            assert torch.equal(c0, c1) and torch.equal(s0, s1)
            assert (cb[:off] == 9).all() and (cb[off + n * D:] == 9).all()


def test_norm_extremes(dev):
    from lagged_indexer_dsa_amd import ops

    print("[norm] extremes", flush=True)
    x = torch.zeros(6, 256, device=dev)
    x[1] = 1e-20
    x[2, 5] = float("nan")
    x[3, 5] = float("inf")
    x[4] = 1e15
    x[5, 200] = 3.0
    w = torch.ones(256, device=dev)
    y = ops.rms_norm(x, w).cpu()
    assert torch.equal(y[0], torch.zeros(256)) and y[2].isnan().all()
    assert y[3, 5].isnan() and torch.equal(y[3, :5], torch.zeros(5))
    assert torch.allclose(y[4], torch.ones(256), rtol=F32) and torch.allclose(y[1], torch.full((256,), 1e-17), rtol=F32)
    codes, scales = ops.rms_norm_quant(x, w)
    c, s = codes.cpu(), scales.cpu()
    assert (c[0] == 0).all() and (s[0] == torch.tensor(1e-6 / 448)).all()
    assert s[2].isnan().all() and ((c[2] & 0x7f) == 0x7f).all()
    assert s[3, 0].isnan() and not s[3, 1].isnan() and (c[3, 128:] == 0).all()
    assert ops.rms_norm(x[:0], w).shape == (0, 256)
    q, s = ops.rms_norm_quant(torch.zeros(3, 0, 256, device=dev), w)
    assert q.shape == (3, 0, 256) and s.shape == (3, 0, 2)


def test_norm_refusals(dev):
    from lagged_indexer_dsa_amd import ops

    print("[norm] refusals", flush=True)
    x, w = torch.zeros(4, 64, device=dev), torch.ones(64, device=dev)
    buf = torch.zeros(4, 128, device=dev)
    for call in (lambda: ops.rms_norm(x.double(), w), lambda: ops.rms_norm(x, w.half()), lambda: ops.rms_norm(x, w[:63]),
                 lambda: ops.rms_norm(x.t(), torch.ones(4, device=dev)), lambda: ops.rms_norm(x, w, residual=x.half()),
                 lambda: ops.rms_norm(x, w, residual=x[:2]), lambda: ops.rms_norm(x, w, out=x.half()),
                 lambda: ops.rms_norm(x, w, out_residual=x), lambda: ops.rms_norm(x, w, out=x),
                 lambda: ops.rms_norm(x, w, residual=buf[:, :64], out_residual=buf[:, 1:65]),
                 lambda: ops.rms_norm(x, w, residual=x.clone(), out_residual=x[:1].expand(4, 64)),
                 lambda: ops.rms_norm(x, w, residual=x.clone(), out_residual=x),
                 lambda: ops.rms_norm(torch.zeros(2, 32769, device=dev), torch.ones(32769, device=dev)),
                 lambda: ops.rms_norm_quant(x, w, group=64), lambda: ops.rms_norm_quant(x, w, out_q=x),
                 lambda: ops.rms_norm_quant(x, w, out_scale=torch.zeros(4, 2, device=dev)),
                 lambda: ops.rms_norm(torch.zeros(2, 3, 4, 64, device=dev).transpose(0, 1), w)):
        with pytest.raises(RuntimeError):
            call()


# ---- rotary ----

SHAPES = [(1, 1, 64, 64, 0), (3, 16, 192, 64, 128), (33, 5, 16, 10, 6), (17, 128, 64, 64, 0), (1000, 2, 576, 64, 512),
          (5, 3, 130, 128, 2), (9, 4, 96, 32, 40), (2, 1, 2, 2, 0), (4, 7, 200, 48, 72), (1, 300, 24, 16, 8)]


@pytest.mark.parametrize("n,H,D,R,start", SHAPES)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_rotary(dev, n, H, D, R, start, dtype):
    from lagged_indexer_dsa_amd import ops
    from lagged_indexer_dsa_amd.rope import build_rope_table

    print(f"[rotary] {(n, H, D, R, start)} {dtype}", flush=True)
    g = torch.Generator(device=dev).manual_seed(n * H + D)
    P = 5000
    table = build_rope_table(P, R, device=dev)
    pos = torch.randint(0, P, (n,), generator=g, device=dev)
    x = _rand(dev, g, n, H, D, dtype=dtype)
    tn = table[pos].double().cpu().numpy()[:, None]
    xn = x.double().cpu().numpy()
    for inter in (False, True):
        for inverse in (False, True):
            p = pos.int() if inverse else pos
            y = ops.rotary(x, p, table, interleaved=inter, start=start, inverse=inverse)
            part = xn[..., start:start + R]
            ref = O.rotate(part, tn[..., :R // 2], tn[..., R // 2:], inter, inverse)
            # two products and a sum in fp32 (or one of them fused), then one rounding
            f = torch.finfo(dtype)
            size = O.rotate(np.abs(part), np.abs(tn[..., :R // 2]), -np.abs(tn[..., R // 2:]), inter, False)
            size = np.maximum(size, O.rotate(np.abs(part), np.abs(tn[..., :R // 2]), np.abs(tn[..., R // 2:]), inter, False))
            bound = f.eps / 2 * (1 + 2.0 ** -22) * np.abs(ref) + 2 * 2.0 ** -24 * np.abs(size) + f.smallest_normal * f.eps
            got = y.double().cpu().numpy()
            assert np.all(np.abs(got[..., start:start + R] - ref) <= bound)
            rest = np.r_[0:start, start + R:D]
            assert np.array_equal(got[..., rest], xn[..., rest])
            # in place: the same bits
            z = x.clone()
            assert ops.rotary(z, p, table, interleaved=inter, start=start, inverse=inverse, out=z) is z
            assert torch.equal(z, y)
    # there and back, in fp32 to a few roundings of values at most |a| + |b|
    if dtype == torch.float32:
        back = ops.rotary(ops.rotary(x, pos, table, start=start), pos, table, start=start, inverse=True)
        assert float((back - x).abs().max()) <= 16 * 2.0 ** -24 * 2 * float(x.abs().max())


def test_rotary_slices_and_padding(dev):
    from lagged_indexer_dsa_amd import ops
    from lagged_indexer_dsa_amd.rope import build_rope_table

    print("[rotary] slices", flush=True)
    g = torch.Generator(device=dev).manual_seed(8)
    table = build_rope_table(300, 64, device=dev)
    q = _rand(dev, g, 21, 16, 192, dtype=torch.bfloat16)
    pos = torch.randint(0, 300, (21,), generator=g, device=dev, dtype=torch.int32)
    want = ops.rotary(q[..., 128:].contiguous(), pos, table, interleaved=True)
    # a slice of wider heads to a slice of others, the rest untouched
    att = torch.full((21, 16, 576), 7.0, dtype=torch.bfloat16, device=dev)
    ops.rotary(q[..., 128:], pos, table, interleaved=True, out=att[..., 512:])
    assert torch.equal(att[..., 512:], want) and bool((att[..., :512] == 7).all())
    # heads first
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(ops.rotary(qt[..., 128:], pos, table, interleaved=True), want)
    ot = torch.empty(16, 21, 64, dtype=torch.bfloat16, device=dev).transpose(0, 1)
    assert torch.equal(ops.rotary(q[..., 128:], pos, table, interleaved=True, out=ot), want)
    # off 16-byte boundaries
    assert torch.equal(ops.rotary(q[..., 127:], pos, table, interleaved=True, start=1)[..., 1:], want)
    # one key a token, shared by all heads (a broadcast input)
    k = _rand(dev, g, 21, 64)
    y = ops.rotary(k, pos, table)
    assert torch.equal(ops.rotary(k[:, None].expand(21, 4, 64), pos, table), y[:, None].expand(21, 4, 64))
    # padding tokens, and every second token of a tensor
    bad = pos.clone()
    bad[3], bad[7], bad[20] = -1, 300, 2 ** 31 - 1
    pad = torch.tensor([3, 7, 20], device=dev)
    part = q[..., 128:].clone()
    ops.rotary(part, bad, table, interleaved=True, out=part)
    got = ops.rotary(q[..., 128:], bad.long(), table, interleaved=True)
    ref = want.clone()
    ref[pad] = q[pad][..., 128:]
    assert torch.equal(part, ref) and torch.equal(got, ref)
    far = bad.long()
    far[3] = -(1 << 40)
    far[7] = 1 << 40
    assert torch.equal(ops.rotary(q[..., 128:], far, table, interleaved=True), ref)
    two = q[::2]
    assert torch.equal(ops.rotary(two[..., 128:], pos[::2].contiguous(), table, interleaved=True), want[::2])
    assert ops.rotary(q[:0], pos[:0], table).shape == (0, 16, 192)


def test_rotary_of_more_tokens_than_a_launch_holds(dev):
    """2^24 workgroups of 256 threads are more than a launch has."""
    from lagged_indexer_dsa_amd import ops

    print("[rotary] 2^24 + 5 tokens", flush=True)
    n, H = (1 << 24) + 5, 129                             # 129 pairs: a workgroup a token
    x = torch.ones(n, H, 2, dtype=torch.bfloat16, device=dev)
    table = torch.tensor([[0.5, 0.25], [2.0, 0.0], [0.0, 1.0]], device=dev)
    turned = torch.tensor([[0.25, 0.75], [2.0, 2.0], [-1.0, 1.0], [1.0, 1.0]], device=dev).to(torch.bfloat16)
    pos = (torch.arange(n, device=dev) % 4).int()         # (3: not in the table)
    assert ops.rotary(x, pos, table, out=x) is x
    for a in range(0, n, 1 << 21):
        assert torch.equal(x[a:a + (1 << 21)], turned[pos[a:a + (1 << 21)].long()][:, None].expand(-1, H, 2))


def test_rotary_refusals(dev):
    from lagged_indexer_dsa_amd import ops

    print("[rotary] refusals", flush=True)
    x = torch.zeros(4, 2, 64, device=dev)
    p = torch.zeros(4, dtype=torch.int32, device=dev)
    t = torch.zeros(8, 64, device=dev)
    buf = torch.zeros(4, 2, 128, device=dev)
    for call in (lambda: ops.rotary(x.double(), p, t), lambda: ops.rotary(x, p[:3], t), lambda: ops.rotary(x, p.float(), t),
                 lambda: ops.rotary(x, p, t.half()), lambda: ops.rotary(x, p, t, start=2),
                 lambda: ops.rotary(x, p, t[:, :63].contiguous()), lambda: ops.rotary(x[0, 0], p, t),
                 lambda: ops.rotary(x, p, t, out=x[:, :1].expand(4, 2, 64)), lambda: ops.rotary(x, p, t, out=x.half()),
                 lambda: ops.rotary(buf[..., :64], p, t, out=buf[..., 64:]),
                 lambda: ops.rotary(x[:1].expand(4, 2, 64), p, t, out=x),
                 lambda: ops.rotary(x, p, t, out=torch.zeros(4, 64, device=dev)[:, None].expand(4, 2, 64)),
                 lambda: ops.rotary(buf[..., ::2], p, t), lambda: ops.rotary(x, p, t[:0])):
        with pytest.raises(RuntimeError):
            call()
