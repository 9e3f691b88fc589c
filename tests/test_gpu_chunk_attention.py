"""GPU: ops.chunk_attention against float64.

Bound of a row's output o, relative to the largest value a row can take, M = max
|kv| over the keys it sees.  The probabilities are rounded to bf16 once (2^-8 of
each) and their sum is of the rounded ones, so they move o by at most 2^-8 sum_j
w_j |v_j - o|, and values within +-M deviate from their mean o by at most M - o^2
/ M on average; the output's rounding adds 2^-8 |o|: together at most 2^-8 (M +
|o| - o^2 / M) <= 1.25 * 2^-8 M = 2.5 * 2^-9 M.  The scores' products (576 of a
whole step 2^-23, of the magnitudes' sum) move an exponent by d and o by at most
2 d M, here below 1.5 * 2^-9 M for |q| and |kv| of the cases: all within 4 * 2^-9
M.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _case(dev, seed, new, lens, heads, bits, extra=0, pt_stride=None, scale=1.0, spare=2):
    from lagged_indexer_dsa_amd import formats as F

    g = torch.Generator().manual_seed(seed)
    need = [-(-n // 64) for n in lens]
    pages = max(1, sum(need) + spare)
    pt = F.random_page_table(lens, pt_stride or max(1, max(need)), pages, generator=g)
    lat, rope = torch.randn(pages * 64, 512, generator=g), torch.randn(pages * 64, 64, generator=g)
    pack = F.pack_latent_rows if bits == 8 else F.pack_latent_rows_fp4
    n = sum(new) + extra
    starts = [sum(new[:b]) for b in range(len(new) + 1)]
    q = (scale * torch.randn(n, heads, 576, generator=g)).to(torch.bfloat16)
    return dict(q=q.to(dev), pool=pack(lat.to(dev), rope.to(dev)), pt=pt.to(dev), new=new, at=starts,
                starts=torch.tensor(starts, dtype=torch.int32, device=dev),
                lens=torch.tensor(lens, dtype=torch.int32, device=dev))


def _run(ops, c, **kw):
    return ops.chunk_attention(c["q"], c["pool"], c["pt"], c["starts"], c["lens"], **kw)


def _ref_row(c, values, b, i, p):
    """float64 output [H, 512] and M of row i of request b at position p."""
    H = c["q"].shape[1]
    seen = min(max(p + 1, 0), c["pt"].shape[1] * 64)
    g = torch.arange(seen, device=values.device)
    page = c["pt"][b].long()[g // 64]
    slots = page * 64 + g % 64
    slots = slots[(page >= 0) & (slots < len(values))]
    if not len(slots):
        return torch.zeros(H, 512, dtype=torch.float64, device=values.device), 0.0
    kv = values[slots]
    s = c["q"][c["at"][b] + i].double() @ kv.T * 576 ** -0.5
    return torch.softmax(s, dim=-1) @ kv[:, :512], float(kv[:, :512].abs().max())


def _check(got, c, lens, ops, rows=None):
    values = ops.read_latent_rows(c["pool"], torch.arange(len(c["pool"]), dtype=torch.int32, device=got.device)).double()
    for b, (t, n) in enumerate(zip(c["new"], lens)):
        pick = range(t) if t <= 12 else sorted({0, 1, t // 3, t // 2, t - 2, t - 1} | {r for r in rows or () if r < t})
        for i in pick:
            ref, M = _ref_row(c, values, b, i, n - t + i)
            err = float((got[c["at"][b] + i].double() - ref).abs().max())
            assert err <= 4 * 2.0 ** -9 * M, (b, i, err / (M or 1))


CASES = [([1], [1]), ([1], [64]), ([5], [5]), ([33], [33]), ([64], [64]), ([65], [130]), ([7], [513]), ([300], [1000]),
         ([1, 1, 1], [1, 63, 65]), ([4, 0, 3, 1], [2000, 50, 3, 511]), ([0, 9, 0], [0, 9, 0]), ([2] * 70, list(range(2, 72))),
         ([130, 1, 66], [700, 1025, 66]), ([1], [9000]), ([3, 2], [20000, 31])]


@pytest.mark.parametrize("new,lens", CASES, ids=lambda v: f"{len(v)}r{max(v)}")
@pytest.mark.parametrize("heads,bits", [(16, 8), (16, 4), (48, 8), (64, 4), (128, 8)])
def test_chunk_attention(dev, new, lens, heads, bits):
    from lagged_indexer_dsa_amd import ops

    print(f"[chunk attention] new={new[:6]} lens={lens[:6]} heads={heads} bits={bits}", flush=True)
    c = _case(dev, 11 + len(new), new, lens, heads, bits, extra=2)
    out = torch.full((sum(new) + 2, heads, 512), 7.0, dtype=torch.bfloat16, device=dev)
    got = _run(ops, c, out=out)
    assert got is out and bool((got[sum(new):] == 7).all())
    _check(got, c, lens, ops)
    again = _run(ops, c, workspace=ops.chunk_workspace(sum(new) + 9, heads, dev))
    assert torch.equal(again[:sum(new)], got[:sum(new)])


@pytest.mark.parametrize("bits", [8, 4])
def test_long_and_ragged(dev, bits):
    """Shares that begin and end inside row tiles of several requests."""
    from lagged_indexer_dsa_amd import ops

    print(f"[chunk attention] long, bits={bits}", flush=True)
    new, lens = [700, 1, 3, 0, 90, 1], [4000, 33000, 12345, 100, 90, 1]
    c = _case(dev, 3, new, lens, 32, bits)
    _check(_run(ops, c), c, lens, ops, rows=(31, 32, 127, 128, 500))


def test_one_row_a_request_is_dense_decode(dev):
    from lagged_indexer_dsa_amd import ops

    lens = [1, 64, 700, 3333]
    for bits in (8, 4):
        c = _case(dev, 7, [1] * 4, lens, 16, bits)
        a = _run(ops, c).double()
        b = ops.dense_mla_decode(c["q"], c["pool"], c["pt"], c["lens"]).double()
        assert float((a - b).abs().max()) <= 8 * 2.0 ** -9 * float(b.abs().max())
        _check(a.to(torch.bfloat16), c, lens, ops)


@pytest.mark.parametrize("bits", [8, 4])
def test_bad_pages_short_pools_and_rows_before_the_first_token(dev, bits):
    """Pages outside the pool, a pool that ends inside a page, lengths over the
    page table and below zero, more new tokens than cached ones."""
    from lagged_indexer_dsa_amd import ops

    print(f"[chunk attention] bad pages, bits={bits}", flush=True)
    c = _case(dev, 5, [9, 40, 6, 3], [9, 300, 200, 200], 16, bits)
    c["lens"].copy_(torch.tensor([5, 100000, -3, 200], dtype=torch.int32))
    last = c["pool"].shape[0] // 64 - 1
    c["pt"][1, 1] = -1
    c["pt"][1, 3] = 1 << 24
    c["pt"][3] = -7
    c["pt"][1, 4] = last
    c["pool"] = c["pool"][:last * 64 + 37].contiguous()
    got = _run(ops, c)
    _check(got, c, [5, 100000, 0, 200], ops)
    assert not bool(got[c["at"][2]:].any())
    # a pool of one row, of a row and a half tile, and of less than a tile at its end
    for rows in (1, 33, 64 + 45):
        c = _case(dev, 6, [20], [100], 16, bits)
        c["pt"].copy_(torch.tensor([[0, 1]], dtype=torch.int32))
        c["pool"] = c["pool"][:rows].contiguous()
        _check(_run(ops, c), c, [100], ops)


@pytest.mark.parametrize("bits", [8, 4])
def test_nan_and_infinity_behind_a_rows_position(dev, bits):
    """Keys of later tokens, and what the last page holds behind the request's
    end, do not reach a row; a row that sees a NaN is NaN."""
    from lagged_indexer_dsa_amd import ops

    c = _case(dev, 8, [40], [130], 16, bits)
    clean = _run(ops, c).clone()
    slot = lambda g: int(c["pt"][0, g // 64]) * 64 + g % 64  # noqa: E731
    dirty = c["pool"].clone()
    for g in range(130, 192):                            # behind the end: every byte a NaN's
        dirty[slot(g)] = 0xff
    assert torch.equal(_run(ops, dict(c, pool=dirty)), clean)
    for g in (110, 120):
        dirty[slot(g)] = 0xff
        dirty[slot(g), 272:] = 0 if bits == 4 else dirty[slot(g), 272:]
    got = _run(ops, dict(c, pool=dirty))
    seen = 110 - 90
    _check(got[:seen], dict(c, pool=c["pool"], new=[seen]), [110], ops)
    assert bool(got[seen:].isnan().all()) and not bool(got[:seen].isnan().any())


def test_one_key_outweighs_the_rest(dev):
    """Scores that rise by far more than 2^32 along the keys: the sums are redone
    about the true maximum, in whole tiles and in parts."""
    from lagged_indexer_dsa_amd import formats as F
    from lagged_indexer_dsa_amd import ops

    for new, n, heads in ((3, 700, 16), (200, 3000, 16), (2, 9000, 128)):
        c = _case(dev, 9, [new], [n], heads, 8)
        kv = torch.randn(len(c["pool"]), 576, device=dev)
        kv[:, :64] = 0.25
        grow = torch.zeros(len(kv), device=dev)
        g = torch.arange(n, device=dev)
        slots = c["pt"][0].long()[g // 64] * 64 + g % 64
        grow[slots] = g / n
        kv[:, 0] = 40 * grow                             # scores climb with the position
        kv[slots[n // 2], 1] = 60.0                      # and one key stands out
        c["pool"] = F.pack_latent_rows(kv[:, :512], kv[:, 512:])
        c["q"] = torch.zeros_like(c["q"])
        c["q"][..., 0], c["q"][..., 1] = 60.0, 200.0
        _check(_run(ops, c), c, [n], ops)


@pytest.mark.parametrize("n", (600, 4000))
@pytest.mark.parametrize("low,peak,rest", ((0, 140, 135), (-120, 20, 12), (0, 140, 140), (100, 100, -60)))
def test_parts_with_far_reference_points(dev, n, low, peak, rest):
    """One share's scores rise by 140 in log2 behind its first keys, while the
    others begin near that height: every part counts by where its weight is."""
    from lagged_indexer_dsa_amd import formats as F
    from lagged_indexer_dsa_amd import ops

    c = _case(dev, 13, [1], [n], 16, 8)
    kv = torch.randn(len(c["pool"]), 576, device=dev)
    kv[:, 512:] = 0
    g = torch.arange(n, device=dev)
    slots = c["pt"][0].long()[g // 64] * 64 + g % 64
    level = torch.full((n,), float(rest), device=dev)
    level[:100] = low
    level[100] = peak
    kv[slots, 512] = level
    c["pool"] = F.pack_latent_rows(kv[:, :512], kv[:, 512:])
    c["q"][..., 512:] = 0
    c["q"][..., :512] *= 0.05
    c["q"][..., 512] = 16.625  # 16.625 / 24 log2(e) = 0.9994
    _check(_run(ops, c), c, [n], ops)


def test_graph_streams_and_shared_workspace(dev):
    """Captured and replayed with other lengths and starts; two calls of one
    workspace in turn; every replay the eager call's bits."""
    from lagged_indexer_dsa_amd import ops

    c = _case(dev, 10, [60, 2, 9], [900, 4000, 9], 32, 8, pt_stride=80)
    d = _case(dev, 12, [5], [600], 16, 4)
    ws = ops.chunk_workspace(71, 32, dev)
    out, out2 = torch.zeros(71, 32, 512, dtype=torch.bfloat16, device=dev), torch.zeros(5, 16, 512, dtype=torch.bfloat16, device=dev)

    def step():
        _run(ops, c, workspace=ws, out=out)
        _run(ops, d, workspace=ws, out=out2)

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for starts, lens in (([0, 60, 62, 71], [900, 4000, 9]), ([0, 1, 70, 71], [300, 4000, 5]), ([0, 0, 0, 71], [0, 0, 71]),
                         ([0, 60, 62, 71], [61, 4000, 9])):
        c["starts"].copy_(torch.tensor(starts, dtype=torch.int32))
        c["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        out.zero_()
        out2.zero_()
        step()
        torch.cuda.synchronize()
        want = out.clone(), out2.clone()
        _check(out, dict(c, at=starts, new=[b - a for a, b in zip(starts, starts[1:])]), lens, ops)
        out.zero_()
        out2.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(out2, want[1])


def test_chunk_attention_refusals(dev):
    from lagged_indexer_dsa_amd import ops

    c = _case(dev, 3, [2, 3], [70, 90], 16, 8)
    q, pool, pt, s, n = c["q"], c["pool"], c["pt"], c["starts"], c["lens"]
    call = ops.chunk_attention
    bad = [lambda: call(q[..., :512].contiguous(), pool, pt, s, n), lambda: call(q.float(), pool, pt, s, n),
           lambda: call(q[:, :8].contiguous(), pool, pt, s, n), lambda: call(q[:, ::2], pool, pt, s, n),
           lambda: call(q, pool[:, :600].contiguous(), pt, s, n), lambda: call(q, pool[:0], pt, s, n),
           lambda: call(q, pool, pt.long(), s, n), lambda: call(q, pool, pt[:1], s, n), lambda: call(q, pool, pt, s[1:], n),
           lambda: call(q, pool, pt, s.long(), n), lambda: call(q, pool, pt, s, n[:1]), lambda: call(q, pool, pt, s, n.cpu()),
           lambda: call(q, pool, pt, s, n, out=torch.zeros(5, 16, 576, dtype=torch.bfloat16, device=dev)),
           lambda: call(q, pool, pt, s, n, workspace=ops.chunk_workspace(4, 16, dev)),
           lambda: call(q, pool, pt, s, n, workspace=ops.chunk_workspace(5, 16, "cpu")),
           lambda: ops.chunk_workspace(4, 24, dev), lambda: ops.chunk_workspace(0, 16, dev)]
    for i, f in enumerate(bad):
        with pytest.raises(RuntimeError):
            f()
            pytest.fail(f"call {i} was not refused")
    empty = call(q[:0], pool, pt, torch.zeros_like(s), n)
    assert empty.shape == (0, 16, 512)


def test_refuses_outputs_over_inputs(dev):
    """out may share no byte with what the call reads, its workspace among them."""
    from lagged_indexer_dsa_amd import ops

    c = _case(dev, 14, [2], [70], 16, 8)
    nbytes = 2 * 16 * 512 * 2
    ws = ops.chunk_workspace(2, 16, dev)
    for buf in (c["q"].view(torch.uint8).flatten(), c["pool"].flatten(), ws):
        out = buf[:nbytes].view(torch.bfloat16).view(2, 16, 512)
        with pytest.raises(RuntimeError, match="overlaps"):
            _run(ops, c, workspace=ws, out=out)
    index_k = torch.zeros(2, 8448, dtype=torch.uint8, device=dev)
    q8, w = torch.zeros(2, 64, 128, dtype=torch.uint8, device=dev), torch.ones(2, 64, device=dev)
    for buf in (q8.flatten(), index_k.flatten()):
        with pytest.raises(RuntimeError, match="overlaps"):
            ops.chunk_scan(q8, w, index_k, c["pt"], c["starts"], c["lens"], 128,
                           out=buf[:2 * 128 * 4].view(torch.float32).view(2, 128))
