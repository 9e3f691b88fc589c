"""GPU: ops.chunk_scan against float64 and against ops.indexer_scan.

Bound: a key's 128 products are summed with roundings of the matrix unit's own
(128 of a whole step 2^-23 of the products' magnitudes at most), the heads by one
fma and sum each (up to 64 + 4), then the key's scale: (256 + 72) 2^-24 of the sum
of the magnitudes.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from _cases import index_case, to_dev
from oracle import dsa_oracle as O

pytestmark = pytest.mark.gpu


def _case(dev, seed, new, lens, heads, extra=0, pt_stride=None):
    """Paged keys of requests of lens tokens, queries of their last new[b]."""
    c = to_dev(index_case(seed, lens, heads, pt_stride=pt_stride), dev)
    n = sum(new) + extra
    rng = np.random.default_rng(seed + 1)
    qc, sq = O.quantize_rowwise(rng.standard_normal((n, heads, 128)).astype(np.float32))
    w = (rng.standard_normal((n, heads)).astype(np.float32) * sq / np.sqrt(heads)).astype(np.float32)
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    return dict(q=torch.from_numpy(qc).to(dev), w=torch.from_numpy(w).to(dev), pages=c["pages"], pt=c["pt"],
                starts=torch.from_numpy(starts).to(dev), lens=c["lens"], new=new, at=starts)


def _run(ops, c, slab, out=None):
    return ops.chunk_scan(c["q"], c["w"], c["pages"], c["pt"], c["starts"], c["lens"], slab, out=out)


def _check(got, c, lens, slab):
    kv = c["pages"][:, :8192].view(torch.float8_e4m3fn).double().reshape(-1, 128)
    ks = c["pages"].view(torch.float32)[:, 2048:].reshape(-1).double()
    for b, (t, n) in enumerate(zip(c["new"], lens)):
        for i in range(t):
            p, row = n - t + i, got[c["at"][b] + i]
            seen = min(max(p + 1, 0), c["pt"].shape[1] * 64, slab)
            assert bool((row[seen:] == float("-inf")).all()), (b, i)
            if not seen:
                continue
            g = torch.arange(seen, device=row.device)
            page = c["pt"][b].long()[g // 64]
            ok = (page >= 0) & (page < c["pages"].shape[0])
            slots = page.clamp(0, c["pages"].shape[0] - 1) * 64 + g % 64
            q = c["q"][c["at"][b] + i].view(torch.float8_e4m3fn).double()
            w = c["w"][c["at"][b] + i].double()
            ref = (w @ (q @ kv[slots].T).clamp_min(0)) * ks[slots]
            S = (w.abs() @ (q.abs() @ kv[slots].abs().T)) * ks[slots].abs()
            err = (row[:seen].double() - ref).abs()
            assert bool((err[ok] <= 328 * 2.0 ** -24 * S[ok]).all()), (b, i, float((err / S)[ok].max()))
            assert bool((row[:seen][~ok] == float("-inf")).all())


CASES = [([1], [1]), ([1], [64]), ([5], [5]), ([64], [64]), ([65], [130]), ([7], [513]), ([300], [1000]), ([1, 1, 1], [1, 63, 65]),
         ([4, 0, 3, 1], [2000, 50, 3, 511]), ([0, 9, 0], [0, 9, 0]), ([2] * 70, list(range(2, 72))), ([130, 1, 66], [700, 1025, 66])]


@pytest.mark.parametrize("new,lens", CASES, ids=lambda v: f"{len(v)}r{max(v)}")
@pytest.mark.parametrize("heads", [16, 32, 48, 64])
def test_chunk_scan(dev, new, lens, heads):
    from lagged_indexer_dsa_amd import ops

    print(f"[chunk scan] new={new[:6]} lens={lens[:6]} heads={heads}", flush=True)
    c = _case(dev, 11 + len(new), new, lens, heads, extra=2)
    slab = c["pt"].shape[1] * 64
    for s in {slab, max(1, slab - 37), slab + 700}:
        out = torch.full((sum(new) + 2, s), 7.0, device=dev)
        got = _run(ops, c, s, out)
        assert got is out and bool((got[sum(new):] == 7).all())
        _check(got, c, lens, s)


def test_rows_before_the_first_token_and_bad_pages(dev):
    """More new tokens than cached ones: the first rows see nothing.  Pages
    outside the cache, lengths over the page table and below zero."""
    from lagged_indexer_dsa_amd import ops

    c = _case(dev, 5, [9, 4, 6], [9, 300, 200], 64)
    c["lens"].copy_(torch.tensor([5, 100000, -3], dtype=torch.int32))
    c["pt"][1, 1] = -1
    c["pt"][1, 3] = c["pages"].shape[0]
    slab = c["pt"].shape[1] * 64
    _check(_run(ops, c, slab), c, [5, 100000, 0], slab)


def test_a_row_alone_and_in_a_chunk(dev):
    """A row's scores do not depend on the rows beside it, bit for bit; the
    decode scan's are the same but for its 8-bit products (of each 8, cut off 13
    bits below the largest: 2^-10 of the magnitudes' sum)."""
    from lagged_indexer_dsa_amd import ops

    c = _case(dev, 8, [513], [9000], 64)
    slab = c["pt"].shape[1] * 64
    got = _run(ops, c, slab)
    for i in (0, 1, 255, 512):
        n = 9000 - 512 + i
        one = dict(c, q=c["q"][i:i + 1].contiguous(), w=c["w"][i:i + 1].contiguous(),
                   starts=torch.tensor([0, 1], dtype=torch.int32, device=dev),
                   lens=torch.tensor([n], dtype=torch.int32, device=dev))
        assert torch.equal(got[i], _run(ops, one, slab)[0])
        dec = ops.indexer_scan(one["q"], one["w"], c["pages"], c["pt"], one["lens"], slab)[0]
        g = torch.arange(n, device=dev)
        slots = c["pt"][0].long()[g // 64] * 64 + g % 64
        k = c["pages"][:, :8192].view(torch.float8_e4m3fn).double().reshape(-1, 128)[slots]
        ks = c["pages"].view(torch.float32)[:, 2048:].reshape(-1).double()[slots]
        S = (one["w"][0].double().abs() @ (one["q"][0].view(torch.float8_e4m3fn).double().abs() @ k.abs().T)) * ks
        assert bool(((dec[:n].double() - got[i, :n].double()).abs() <= (2.0 ** -10 + 2 * 328 * 2.0 ** -24) * S).all())
        assert bool((dec[n:] == got[i, n:]).all())


def test_chunk_scan_refusals(dev):
    from lagged_indexer_dsa_amd import ops

    c = _case(dev, 3, [2, 3], [70, 90], 32)
    bad = [lambda: ops.chunk_scan(c["q"][..., :64], c["w"], c["pages"], c["pt"], c["starts"], c["lens"], 128),
           lambda: ops.chunk_scan(c["q"], c["w"][:, :16], c["pages"], c["pt"], c["starts"], c["lens"], 128),
           lambda: ops.chunk_scan(c["q"], c["w"], c["pages"][:, :8192], c["pt"], c["starts"], c["lens"], 128),
           lambda: ops.chunk_scan(c["q"], c["w"], c["pages"], c["pt"].long(), c["starts"], c["lens"], 128),
           lambda: ops.chunk_scan(c["q"], c["w"], c["pages"], c["pt"], c["starts"][:2], c["lens"], 128),
           lambda: ops.chunk_scan(c["q"], c["w"], c["pages"], c["pt"], c["starts"], c["lens"].long(), 128),
           lambda: ops.chunk_scan(c["q"], c["w"], c["pages"], c["pt"], c["starts"], c["lens"], 0),
           lambda: ops.chunk_scan(c["q"][:, :8].contiguous(), c["w"][:, :8].contiguous(), c["pages"], c["pt"], c["starts"],
                                  c["lens"], 128),
           lambda: ops.chunk_scan(c["q"], c["w"], c["pages"], c["pt"], c["starts"], c["lens"].cpu(), 128),
           lambda: ops.chunk_scan(c["q"], c["w"], c["pages"], c["pt"], c["starts"], c["lens"], 128,
                                  out=torch.zeros(5, 64, device=dev))]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was not refused")
