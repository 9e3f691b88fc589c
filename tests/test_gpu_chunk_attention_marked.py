"""GPU: ops.chunk_attention over keys that mark their tiles (_marked.py): every
output element of every row, so that a key tile or a part of a split row that is
left out, repeated or taken from a neighbour shows, however long the row."""

from __future__ import annotations

import pytest
import torch

from _marked import marks, shares, worst

pytestmark = pytest.mark.gpu


def _case(dev, seed, new, lens, heads, bits):
    from lagged_indexer_dsa_amd import formats as F

    g = torch.Generator(device=dev).manual_seed(seed)
    pages = sum(-(-n // 64) for n in lens) + 2
    pt = F.random_page_table(lens, max(1, max(-(-n // 64) for n in lens)), pages, generator=torch.Generator().manual_seed(seed))
    lat, rope = torch.zeros(pages * 64, 512, device=dev), torch.randn(pages * 64, 64, generator=g, device=dev)
    slots = []
    for b, n in enumerate(lens):
        at = torch.arange(n, device=dev)
        slots.append(pt[b].to(dev).long()[at // 64] * 64 + at % 64)
        lat[slots[-1], marks(n, dev)] = 1.0
    pool = (F.pack_latent_rows if bits == 8 else F.pack_latent_rows_fp4)(lat, rope)
    q = torch.zeros(sum(new), heads, 576, dtype=torch.bfloat16, device=dev)
    q[..., 512:] = 2 * torch.randn(sum(new), heads, 64, generator=g, device=dev)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    starts = [sum(new[:b]) for b in range(len(new) + 1)]
    return q, pool, pt.to(dev), ints(starts), ints(lens), slots, starts


def _check(out, q, pool, slots, starts, new, lens):
    from lagged_indexer_dsa_amd import ops

    H = q.shape[1]
    for b, (t, n) in enumerate(zip(new, lens)):
        if not t:
            continue
        kv = ops.read_latent_rows(pool, slots[b].to(torch.int32))
        assert bool((kv[:, :512].sum(-1) == 1).all())
        step = max(1, (1 << 27) // (n * H))
        for i in range(0, t, step):
            rows = slice(starts[b] + i, starts[b] + min(t, i + step))
            pos = torch.arange(n - t + i, n - t + min(t, i + step), device=q.device).repeat_interleave(H)
            ref = shares(q[rows, :, 512:].reshape(-1, 64), kv[:, 512:], pos)
            assert worst(out[rows].reshape(-1, 512), ref) <= 1, (b, i)


@pytest.mark.parametrize("new,lens", [([1], [1]), ([33], [33]), ([65], [130]), ([300], [1000]), ([1], [9000]), ([7], [9001]),
                                      ([1], [33000]), ([1], [131072]), ([3, 2], [20000, 31]), ([4, 0, 3, 1], [2000, 50, 3, 511]),
                                      ([130, 1, 66], [700, 1025, 66]), ([2] * 70, list(range(2, 72))), ([1] * 20, [4097] * 20),
                                      ([700, 1, 3, 0, 90, 1], [4000, 33000, 12345, 100, 90, 1])],
                         ids=lambda v: f"{len(v)}r{max(v)}")
@pytest.mark.parametrize("heads,bits", [(16, 8), (16, 4), (48, 8), (64, 4), (128, 8)])
def test_every_tile_once(dev, new, lens, heads, bits):
    from lagged_indexer_dsa_amd import ops

    print(f"[marked] new={new[:6]} lens={lens[:6]} heads={heads} bits={bits}", flush=True)
    q, pool, pt, s, n, slots, starts = _case(dev, 31 + len(new), new, lens, heads, bits)
    out = ops.chunk_attention(q, pool, pt, s, n)
    _check(out, q, pool, slots, starts, new, lens)


def test_every_tile_once_where_shares_differ(dev):
    """The same requests cut otherwise by what is beside them."""
    from lagged_indexer_dsa_amd import ops

    for k in range(1, 12):
        new, lens = [3, 40, 1] + [k] * k, [5000 + 97 * k, 1500, 7000 - 31 * k] + [100 * k] * k
        print(f"[marked] {k}", flush=True)
        q, pool, pt, s, n, slots, starts = _case(dev, 50 + k, new, lens, 16, 8)
        _check(ops.chunk_attention(q, pool, pt, s, n), q, pool, slots, starts, new, lens)


@pytest.mark.parametrize("new,lens,heads", [([1], [5000], 1024), ([5, 2], [300, 77], 1024), ([1] * 3000, [65] * 3000, 16),
                                            ([0] * 500 + [3] + [0] * 500 + [2] + [0] * 63, [9] * 500 + [4000] + [9] * 500 + [2] + [0] * 63, 32)],
                         ids=("h1024", "h1024two", "3000r", "empties"))
def test_most_heads_and_many_requests(dev, new, lens, heads):
    from lagged_indexer_dsa_amd import ops

    print(f"[marked] {len(new)} requests, heads={heads}", flush=True)
    q, pool, pt, s, n, slots, starts = _case(dev, 9, new, lens, heads, 8)
    _check(ops.chunk_attention(q, pool, pt, s, n), q, pool, slots, starts, new, lens)


def test_two_calls_at_once(dev):
    """On two streams, each with its own workspace, beside each other: the bits of
    each alone."""
    from lagged_indexer_dsa_amd import ops

    cases = [_case(dev, 3, [600, 3], [5000, 30000], 32, 8), _case(dev, 4, [4] * 16, [3000 + 700 * i for i in range(16)], 16, 4)]
    want = [ops.chunk_attention(*c[:5]) for c in cases]
    outs = [[torch.zeros_like(w) for _ in range(6)] for w in want]
    ws = [ops.chunk_workspace(c[0].shape[0], c[0].shape[1], dev) for c in cases]
    streams = [torch.cuda.Stream(dev) for _ in cases]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for i in range(6):
        for c, o, w, st in zip(cases, outs, ws, streams):
            with torch.cuda.stream(st):
                ops.chunk_attention(*c[:5], workspace=w, out=o[i])
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert all(torch.equal(x, w) for x in o)


@pytest.mark.parametrize("e", [-30, -56, 40])
def test_small_and_large_latents(dev, e):
    """Latent values of 2^-56 (far below any that the library's packers write) and
    2^40 come out as those of 1 do, but for a step of the output (2^-7) where what a
    sum of products of 2^-136 loses turns its rounding."""
    from lagged_indexer_dsa_amd import ops

    q, pool, pt, s, n, slots, starts = _case(dev, 8, [5, 1], [700, 9000], 16, 8)
    want = ops.chunk_attention(q, pool, pt, s, n)
    pool = pool.clone()
    scales = pool[:, 512:528].contiguous().view(torch.float32) * 2.0 ** e
    pool[:, 512:528] = scales.view(torch.uint8)
    got = ops.chunk_attention(q, pool, pt, s, n)
    err = (got.double() * 2.0 ** -e - want.double()).abs()
    assert float((err / want.double().clamp_min(1e-30)).max()) <= 2.0 ** -7
    _check((got.float() * 2.0 ** -e).to(torch.bfloat16), q, _unscaled(pool, e), slots, starts, [5, 1], [700, 9000])


def _unscaled(pool, e):
    pool = pool.clone()
    pool[:, 512:528] = (pool[:, 512:528].contiguous().view(torch.float32) * 2.0 ** -e).view(torch.uint8)
    return pool
