"""GPU: ops.quantize_rows, ops.fp8_matmul and ops.fp8_matmul_grouped against
float64.

Bounds.  quantize_rows: silu's exponential, quotient and product are within 8
steps of fp32 (2^-24 each, the exponential's two and the quotient's two among
them), the scale's division half a step; a code is within half a step of value /
scale (2^-4 of it, or 2^-10 scales).
Products: a product of two e4m3 values is exact in fp32 and in the matrix unit's
bf16 products, which fp32 outputs take; a block's 128 are summed in an order and
with roundings of the matrix unit's own: 128 of a whole step (2^-23) at most, of
the sum S of the products' magnitudes; then a rounding of the scales' product,
and of one fma a block and 8 sums of the waves (2^-24 each): (256 + blocks + 10)
2^-24 S.  The result is rounded once (eps / 2).
bf16 and fp16 outputs take the 8-bit products: of each 8 of them, what lies more
than 13 bits below the largest's exponent is cut off (a 2^3 beside a 2^16 is
summed, a 2^2 is not), so a group of 8 is off by less than 8 * 2^-13 = 2^-10 of its
largest product, and all groups by less than 2^-10 S besides.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

F32 = 8 * 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _randn(dev, g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)


# ---- quantize_rows ----

def _quant_ref(x, gate):
    y = x.double()
    return y if gate is None else y * gate.double() * torch.sigmoid(gate.double())


def _check_quant(got, x, gate, group):
    codes, scales = got
    D = x.shape[-1]
    assert codes.dtype == torch.uint8 and codes.shape == x.shape
    y = _quant_ref(x, gate).reshape(-1, D)
    s = scales.double().reshape(y.shape[0], -1)
    c = codes.view(torch.float8_e4m3fn).double().reshape(-1, D)
    width = group or D
    assert s.shape[1] == -(-D // width)
    for k, a in enumerate(range(0, D, width)):
        part, sk = y[:, a:a + width], s[:, k:k + 1]
        top = part.abs().amax(1, keepdim=True).clamp_min(1e-6) / 448
        assert bool(((sk - top).abs() <= (F32 + 2.0 ** -23) * top).all()), "scale"
        err = (c[:, a:a + width] * sk - part).abs()
        assert bool((err <= (2.0 ** -4 + F32) * part.abs() + 2.0 ** -10 * sk).all()), "codes"


@pytest.mark.parametrize("D", [1, 7, 8, 64, 127, 128, 136, 500, 1000, 2048, 2056, 4097, 8192, 8200, 18432, 24576, 32761, 32768])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_quantize_all_widths(dev, D, dtype):
    from lagged_indexer_dsa_amd import ops

    print(f"[quant] D={D} {dtype}", flush=True)
    g = torch.Generator(device=dev).manual_seed(D)
    for n in (1, 5):
        gu = _randn(dev, g, n, 2 * D, dtype=dtype, scale=3)
        for group in (128, 0):
            _check_quant(ops.quantize_rows(gu[:, D:], group=group), gu[:, D:], None, group)
            _check_quant(ops.quantize_rows(gu[:, D:], gate=gu[:, :D], group=group), gu[:, D:], gu[:, :D], group)


def test_quantize_strides_and_given_outputs(dev):
    from lagged_indexer_dsa_amd import ops

    g = torch.Generator(device=dev).manual_seed(5)
    wide = _randn(dev, g, 3, 700, 2112, dtype=torch.bfloat16)
    row = wide[0, :1, :512].expand(9, 512)
    for x in (wide[..., :1536], wide[..., 3:1539], wide[1, ::2, 576:], row):
        a = ops.quantize_rows(x)
        _check_quant(a, x, None, 128)
        b = ops.quantize_rows(x.contiguous())
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    x = wide[0, :, :1536].contiguous()
    q, s = torch.empty(700, 1536, dtype=torch.uint8, device=dev), torch.empty(700, 12, device=dev)
    a = ops.quantize_rows(x, out_q=q, out_scale=s)
    assert a[0] is q and a[1] is s
    _check_quant(a, x, None, 128)
    # codes that begin between boundaries
    buf = torch.zeros(700 * 1536 + 3, dtype=torch.uint8, device=dev)
    odd = buf[3:].view(700, 1536)
    ops.quantize_rows(x, out_q=odd)
    assert torch.equal(odd, q) and not buf[:3].any()
    for shape in ((0, 128), (3, 0, 64)):
        codes, scales = ops.quantize_rows(torch.zeros(*shape, device=dev))
        assert codes.shape == shape and scales.shape == (*shape[:-1], 1)


def test_quantize_gates_at_their_ends(dev):
    """Gates from the most negative to the largest, infinities and NaN: torch's
    own 64-bit x * g * sigmoid(g), which is NaN for g = -inf."""
    from lagged_indexer_dsa_amd import ops

    g = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 5.0, -5.0, 17.5, -17.5, 60.0, -60.0, 87.9, -87.9, 88.9, -88.9, 103.0, -103.0,
                      150.0, -150.0, 1e4, -1e4, 1e30, -1e30], device=dev)
    x = torch.full_like(g, 1.5)[:, None]
    codes, scales = ops.quantize_rows(x, gate=g[:, None])       # a row a gate: its scale tells the value
    y = _quant_ref(x, g[:, None]).abs().clamp_min(1e-6)
    assert bool(((scales.double() * 448 - y).abs() <= (F32 + 2.0 ** -23) * y).all())
    for bad in (float("inf"), -float("inf"), float("nan")):
        gate = torch.ones(2, 256, device=dev)
        gate[1, 130] = bad
        codes, scales = ops.quantize_rows(torch.ones(2, 256, device=dev), gate=gate)
        c = codes.view(torch.float8_e4m3fn).float()
        assert torch.isfinite(scales[0]).all() and torch.isfinite(scales[1, 0]) and not torch.isfinite(scales[1, 1])
        assert torch.isnan(c[1, 130]) and not torch.isnan(c[0]).any() and not torch.isnan(c[1, :128]).any()
        if bad == float("inf"):  # every finite value over an infinite scale is 0
            assert torch.isinf(scales[1, 1]) and not c[1, 131:].any()
        else:
            assert torch.isnan(scales[1, 1]) and torch.isnan(c[1, 128:]).all()


def test_quantize_is_the_norms_rule(dev):
    """A norm with weight one and eps such that it divides by exactly 1."""
    from lagged_indexer_dsa_amd import ops

    g = torch.Generator(device=dev).manual_seed(9)
    x = torch.where(torch.rand(40, 512, generator=g, device=dev) < 0.5, -1.0, 1.0)
    a = ops.quantize_rows(x)
    b = ops.rms_norm_quant(x, torch.ones(512, device=dev), eps=0.0)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ---- products ----

def _values(codes, scale, rows):
    """float64 of codes [n, K] with scale [i, j] for `rows` rows and 128 columns."""
    n, K = codes.shape
    v = codes.view(torch.float8_e4m3fn).double()
    if scale.shape[1] == 1:
        return v * scale.double().repeat_interleave(rows, 0)[:n]
    return v * scale.double().repeat_interleave(rows, 0)[:n].repeat_interleave(128, 1)[:, :K]


def _near(got, a, w, blocks):
    ref, S = a @ w.T, a.abs() @ w.abs().T
    f = torch.finfo(got.dtype)
    bound = ((256 + blocks + 10) * 2.0 ** -24 + (0.0 if got.dtype == torch.float32 else 2.0 ** -10)) * S
    bound = bound + f.eps / 2 * (ref.abs() + bound) + f.smallest_normal * f.eps
    err = (got.double() - ref).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


def _operands(dev, g, rows, N, K, row_scale=False, lead=()):
    from lagged_indexer_dsa_amd import formats, ops

    x = _randn(dev, g, rows, K) * torch.exp(0.5 * _randn(dev, g, rows, 1))
    if K > 32768:  # above the quantiser's longest row: its groups as rows
        a, sa = ops.quantize_rows(x.view(-1, 128))
        a, sa = a.view(rows, K), sa.view(rows, K // 128)
    else:
        a, sa = ops.quantize_rows(x, group=0 if row_scale else 128)
    w, sw = formats.quantize_weight(_randn(dev, g, *lead, N, K, scale=0.05))
    return a, sa, w, sw


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 100, 127, 128, 129, 200, 257, 300])
@pytest.mark.parametrize("N,K", [(1, 16), (17, 144), (128, 128), (130, 1040), (576, 2048), (301, 7168)])
def test_product_all_sizes(dev, rows, N, K):
    from lagged_indexer_dsa_amd import ops

    print(f"[matmul] rows={rows} N={N} K={K}", flush=True)
    g = torch.Generator(device=dev).manual_seed(rows * 1000 + N)
    for row_scale in (False, True):
        a, sa, w, sw = _operands(dev, g, rows, N, K, row_scale)
        av, wv = _values(a, sa, 1), _values(w, sw, 128)
        for dtype in TYPES if not row_scale else TYPES[:1]:
            _near(ops.fp8_matmul(a, sa, w, sw, dtype=dtype), av, wv, -(-K // 128))


@pytest.mark.parametrize("rows,N,K", [(1, 2112, 7168), (32, 24576, 1536), (77, 128, 18432), (1000, 7168, 2048),
                                      (2049, 6144, 1536), (4097, 520, 512), (700, 24576, 528), (1, 64, 131072)])
def test_product_model_sizes(dev, rows, N, K):
    from lagged_indexer_dsa_amd import ops

    print(f"[matmul] rows={rows} N={N} K={K}", flush=True)
    g = torch.Generator(device=dev).manual_seed(rows + N)
    a, sa, w, sw = _operands(dev, g, rows, N, K)
    out = torch.full((rows, N), 7.0, dtype=torch.bfloat16, device=dev)
    got = ops.fp8_matmul(a, sa, w, sw, out=out)
    assert got is out
    _near(got, _values(a, sa, 1), _values(w, sw, 128), -(-K // 128))
    assert torch.equal(got, ops.fp8_matmul(a.view(torch.float8_e4m3fn), sa, w.view(torch.float8_e4m3fn), sw))


@pytest.mark.parametrize("rows", [3, 40, 300])
def test_product_edges(dev, rows):
    """Leading dimensions, no rows, outputs on odd addresses; NaN and infinite
    scales stay in their rows and outputs; a row's neighbours are untouched."""
    from lagged_indexer_dsa_amd import ops

    g = torch.Generator(device=dev).manual_seed(rows)
    N, K = 300, 400
    a, sa, w, sw = _operands(dev, g, rows, N, K)
    whole = ops.fp8_matmul(a, sa, w, sw)
    lead = ops.fp8_matmul(a.view(rows, 1, K), sa.view(rows, 1, 4), w, sw)
    assert lead.shape == (rows, 1, N) and torch.equal(lead[:, 0], whole)
    assert ops.fp8_matmul(a[:0], sa[:0], w, sw).shape == (0, N)
    assert ops.fp8_matmul(a, sa, w[:0], sw[:0]).shape == (rows, 0)
    buf = torch.full((rows * N + 9,), 3.0, dtype=torch.bfloat16, device=dev)
    ops.fp8_matmul(a, sa, w, sw, out=buf[1:1 + rows * N].view(rows, N))
    assert torch.equal(buf[1:1 + rows * N].view(rows, N), whole) and bool((buf[1 + rows * N:] == 3).all()) and buf[0] == 3
    a2, sa2, w2, sw2 = a.clone(), sa.clone(), w.clone(), sw.clone()
    a2[1, 399] = 0x7f                         # NaN code
    sa2[2, 3] = float("inf")
    w2[299, 0] = 0xff                         # NaN code
    sw2[1, 2] = float("nan")                  # outputs 128 .. 255
    got = ops.fp8_matmul(a2, sa2, w2, sw2)
    assert bool(got[1].isnan().all()) and bool(got[:, 299].isnan().all()) and bool(got[:, 128:256].isnan().all())
    assert not bool(got[2, :128].isfinite().any())
    keep = torch.ones(rows, dtype=torch.bool, device=dev)
    keep[1:3] = False
    assert torch.equal(got[keep][:, :128], whole[keep][:, :128]) and torch.equal(got[keep][:, 256:299], whole[keep][:, 256:299])


def _grouped_case(dev, counts, N, K, extra=0, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    rows = sum(counts) + extra
    a, sa, w, sw = _operands(dev, g, max(rows, 1), N, K, lead=(len(counts),))
    ends = [sum(counts[:e]) for e in range(len(counts) + 1)]
    return a[:rows], sa[:rows], w, sw, ends, torch.tensor(ends, dtype=torch.int32, device=dev)


def _check_grouped(got, a, sa, w, sw, ends, K):
    for e, (i, j) in enumerate(zip(ends, ends[1:])):
        if j > i:
            _near(got[i:j], _values(a[i:j], sa[i:j], 1), _values(w[e], sw[e], 128), -(-K // 128))


@pytest.mark.parametrize("counts", [[5], [0, 3, 0, 1, 16, 17, 0], [64, 65, 0, 1], [130, 0, 257, 128, 1, 300], [0, 0, 900, 0],
                                    [2] * 70, [100] * 70, [0, 0], [1] + [0] * 100 + [300]],
                         ids=lambda c: f"{len(c)}x{max(c)}")
@pytest.mark.parametrize("N,K", [(300, 400), (128, 1536)])
def test_grouped(dev, counts, N, K):
    from lagged_indexer_dsa_amd import ops

    print(f"[grouped] {counts[:8]} N={N} K={K}", flush=True)
    a, sa, w, sw, ends, offsets = _grouped_case(dev, counts, N, K, extra=3, seed=len(counts))
    out = torch.full((ends[-1] + 3, N), 5.0, dtype=torch.float32, device=dev)
    got = ops.fp8_matmul_grouped(a, sa, w, sw, offsets, out=out)
    assert got is out and bool((out[ends[-1]:] == 5).all())
    _check_grouped(got, a, sa, w, sw, ends, K)
    for dtype in TYPES[1:]:
        _check_grouped(ops.fp8_matmul_grouped(a, sa, w, sw, offsets, dtype=dtype), a, sa, w, sw, ends, K)


def test_grouped_offsets_need_not_begin_at_zero(dev):
    from lagged_indexer_dsa_amd import ops

    a, sa, w, sw, ends, offsets = _grouped_case(dev, [50, 20, 90], 256, 256)
    for lo in (0, 7):
        cut = torch.tensor([lo, 20, 20, 100], dtype=torch.int32, device=dev)
        out = torch.full((160, 256), 5.0, dtype=torch.bfloat16, device=dev)
        ops.fp8_matmul_grouped(a, sa, w, sw, cut, out=out)
        assert bool((out[:lo] == 5).all()) and bool((out[100:] == 5).all())
        _check_grouped(out, a, sa, w, sw, [lo, 20, 20, 100], 256)
    # offsets behind the rows end with them
    cut = torch.tensor([0, 150, 400, 900], dtype=torch.int32, device=dev)
    out = ops.fp8_matmul_grouped(a, sa, w, sw, cut)
    _check_grouped(out, a, sa, w, sw, [0, 150, 160, 160], 256)


def test_products_in_a_graph_and_on_a_stream(dev):
    """Quantiser and both products captured: replays read the inputs and offsets
    as they are then; every replay gives the eager call's bits."""
    from lagged_indexer_dsa_amd import ops

    a, sa, w, sw, ends, offsets = _grouped_case(dev, [30, 0, 200, 70], 512, 512, seed=3)
    x = torch.randn(300, 512, device=dev).to(torch.bfloat16)
    out = torch.zeros(300, 512, dtype=torch.bfloat16, device=dev)
    few = torch.zeros(20, 512, dtype=torch.bfloat16, device=dev)

    def step():
        q, s = ops.quantize_rows(x)
        ops.fp8_matmul_grouped(q, s, w, sw, offsets, out=out)
        ops.fp8_matmul(q[:20], s[:20], w[1], sw[1], out=few)

    side = torch.cuda.Stream(dev)
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        x.copy_(torch.randn(300, 512, device=dev))
        offsets.copy_(torch.tensor([0, 10 * i, 100, 100 + 50 * i, 300], dtype=torch.int32))
        step()
        torch.cuda.synchronize()
        want = out.clone(), few.clone()
        out.zero_()
        few.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(few, want[1])


def test_refusals(dev):
    from lagged_indexer_dsa_amd import ops

    a, w = torch.zeros(4, 256, dtype=torch.uint8, device=dev), torch.zeros(8, 256, dtype=torch.uint8, device=dev)
    sa, sw = torch.ones(4, 2, device=dev), torch.ones(1, 2, device=dev)
    off = torch.tensor([0, 4], dtype=torch.int32, device=dev)
    bad = [lambda: ops.fp8_matmul(a.float(), sa, w, sw), lambda: ops.fp8_matmul(a, sa.half(), w, sw),
           lambda: ops.fp8_matmul(a, sa[:, :1].expand(4, 2), w, sw), lambda: ops.fp8_matmul(a[:, :128], sa, w, sw),
           lambda: ops.fp8_matmul(a, sa, w[:, :128].contiguous(), sw), lambda: ops.fp8_matmul(a, sa, w, sw.T),
           lambda: ops.fp8_matmul(a, torch.ones(4, 3, device=dev), w, sw), lambda: ops.fp8_matmul(a, sa[:3], w, sw),
           lambda: ops.fp8_matmul(a[:, :100].contiguous(), sa[:, :1].contiguous(), w[:, :100].contiguous(), sw[:, :1].contiguous()),
           lambda: ops.fp8_matmul(a, sa, w, sw, dtype=torch.float64),
           lambda: ops.fp8_matmul(a, sa, w, sw, out=torch.zeros(4, 9, device=dev)),
           lambda: ops.fp8_matmul(a, sa, w, sw, out=a.view(torch.bfloat16)[:, :8]),
           lambda: ops.fp8_matmul(a, sa, w[None], sw[None]), lambda: ops.fp8_matmul(a, sa, w, sw.cpu()),
           lambda: ops.fp8_matmul_grouped(a, sa, w, sw, off), lambda: ops.fp8_matmul_grouped(a, sa, w[None], sw[None], off[:1]),
           lambda: ops.fp8_matmul_grouped(a, sa, w[None], sw[None], off.long()),
           lambda: ops.fp8_matmul_grouped(a, sa, w[None], sw[None], None),
           lambda: ops.fp8_matmul_grouped(a[None], sa[None], w[None], sw[None], off),
           lambda: ops.fp8_matmul(torch.zeros(4 * 256 + 8, dtype=torch.uint8, device=dev)[8:].view(4, 256), sa, w, sw),
           lambda: ops.quantize_rows(a), lambda: ops.quantize_rows(sa, group=64), lambda: ops.quantize_rows(sa, gate=sa[:3]),
           lambda: ops.quantize_rows(sa, gate=sa.half()), lambda: ops.quantize_rows(torch.zeros(2, 32769, device=dev)),
           lambda: ops.quantize_rows(torch.zeros(8, 4, device=dev).T), lambda: ops.quantize_rows(sa, out_q=a),
           lambda: ops.quantize_rows(a.view(torch.float32), out_q=a[:, :64]),
           lambda: ops.quantize_rows(a.view(torch.float32)[:, :8], out_q=a.view(-1)[:32].view(4, 8))]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was not refused")
