"""GPU: decode attention over 400-byte latent rows against float64.

Bound.  The keys' values are exact.  A score is off by fp32's sums of 576
products: under 2^-14 for these inputs (36 chained sums a lane at 2^-24 of at
most 60); each probability then by 2^-14, and it is rounded to bf16 (2^-8 of
it).  The output is divided by the sum of the rounded probabilities (2^-8 of
it) and rounded to bf16 (2^-8 of it).  With some fp32 roundings: 2^-7 of the
output and 2^-8 (1 + 2^-4) of sum p |v|.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import dsa_oracle as O

pytestmark = pytest.mark.gpu

SM = 576 ** -0.5


def _pool(seed, n):
    rng = np.random.default_rng(seed)
    lat = rng.standard_normal((n, 512)).astype(np.float32) * np.exp(0.5 * rng.standard_normal((n, 1))).astype(np.float32)
    return O.pack_latent_rows_fp4(lat, rng.standard_normal((n, 64)).astype(np.float32))


def _q(seed, B, H, scale=1.0):
    rng = np.random.default_rng(seed + 77)
    return O.bf16_rn((rng.standard_normal((B, H, 576)) * scale).astype(np.float32))


def _dev(a, dev, bf16=False):
    if bf16:
        return torch.from_numpy(O.bf16_bits(a).view(np.int16)).view(torch.bfloat16).to(dev)
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def _check(out, q, kv, idx, sm=SM):
    ref = O.mla_decode_values(q, kv, idx, sm)
    got = out.double().cpu().numpy()
    for b in range(len(q)):
        sel = idx[b][(idx[b] >= 0) & (idx[b] < len(kv))]
        if not sel.size:
            assert not got[b].any(), f"row {b} has no key"
            continue
        k = kv[sel].astype(np.float64)
        s = q[b].astype(np.float64) @ k.T * sm
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        bound = 2.0 ** -7 * np.abs(ref[b]) + 2.0 ** -8 * (1 + 2.0 ** -4) * (p @ np.abs(k[:, :512]))
        err = np.abs(got[b] - ref[b])
        assert np.all(err <= bound), f"row {b}: {float((err / bound).max())} of the bound"


SPARSE = [(1, 16, 1, 64, 0), (1, 16, 2048, 5000, 0), (3, 32, 777, 3000, 0), (2, 128, 130, 400, 0), (1, 16, 2048, 5000, 1),
          (2, 48, 300, 1000, 5), (300, 16, 65, 500, 0), (1, 1024, 40, 64, 0), (5, 16, 1000, 1200, 128), (260, 16, 200, 512, 3)]


@pytest.mark.parametrize("B,H,topk,n,nsplit", SPARSE)
def test_sparse(dev, B, H, topk, n, nsplit):
    from lagged_indexer_dsa_amd import ops

    print(f"[fp4 sparse] {(B, H, topk, n, nsplit)}", flush=True)
    rng = np.random.default_rng(B + topk)
    rows = _pool(n, n)
    q = _q(n, B, H)
    idx = np.stack([rng.permutation(n)[:topk] if topk <= n else np.r_[rng.permutation(n), np.full(topk - n, -1)]
                    for _ in range(B)]).astype(np.int32)
    drop = rng.random(idx.shape)
    idx[drop < 0.02] = -1
    idx[(drop > 0.98)] = n + 5
    if B > 2:
        idx[1] = -1                                       # a row that attends nothing
        idx[2, 1:] = -1                                   # a row of one key, first place
        idx[2, 0] = n - 1
    qd, pool, id_ = _dev(q, dev, True), _dev(rows, dev), _dev(idx, dev)
    out = ops.sparse_mla_decode(qd, pool, id_, nsplit=nsplit)
    _check(out, q, O.dequant_latent_rows_fp4(rows), idx)
    # the same call, the same bits; with a workspace full of anything, too
    ws = ops.sparse_mla_workspace(B, H, nsplit, dev)
    ws.view(torch.uint8)[ops._lib.load().dsa_sparse_mla_barrier_bytes(B, H, 0):].fill_(0xFF)
    again = ops.sparse_mla_decode(qd, pool, id_, nsplit=nsplit, workspace=ws, out=torch.full_like(out, 3.0))
    assert torch.equal(again, out)


DENSE = [(1, 16, [1], 0), (1, 16, [4097], 0), (3, 64, [777, 0, 5000], 0), (2, 128, [130, 2000], 0), (8, 32, [64] * 8, 0),
         (4, 16, [0, 0, 0, 0], 0), (5, 16, [1, 63, 64, 65, 9000], 7), (1, 16, [20000], 128), (70, 16, None, 0),
         (300, 16, None, 0), (2, 1024, [100, 257], 0), (257, 16, None, 2), (130, 32, None, 4)]


@pytest.mark.parametrize("B,H,lens,nsplit", DENSE)
def test_dense(dev, B, H, lens, nsplit):
    from lagged_indexer_dsa_amd import ops

    print(f"[fp4 dense] {(B, H, lens, nsplit)}", flush=True)
    rng = np.random.default_rng(B * H)
    lens = np.array(lens if lens is not None else rng.integers(0, 400, B), dtype=np.int32)
    pts = max(1, int(lens.max()) // 64 + 2)
    need = -(-lens // 64)
    pages = int(need.sum()) + 1
    perm = rng.permutation(pages)
    pt = np.full((B, pts), -1, dtype=np.int32)
    at = 0
    for b in range(B):
        pt[b, :need[b]] = perm[at:at + need[b]]
        at += need[b]
    rows = _pool(B, pages * 64)
    q = _q(B, B, H)
    idx = np.full((B, max(1, int(lens.max()))), -1, dtype=np.int64)
    for b in range(B):
        j = np.arange(lens[b])
        idx[b, :lens[b]] = pt[b, j // 64] * 64 + j % 64
    args = [_dev(q, dev, True), _dev(rows, dev), _dev(pt, dev), _dev(lens, dev)]
    out = ops.dense_mla_decode(*args, nsplit=nsplit)
    _check(out, q, O.dequant_latent_rows_fp4(rows), idx)
    again = ops.dense_mla_decode(*args, nsplit=nsplit, workspace=ops.sparse_mla_workspace(B, H, nsplit, dev),
                                 out=torch.full_like(out, 3.0))
    assert torch.equal(again, out)
    if B == 3:  # lengths past the table are cut to it; pages that are not there are not attended
        over = _dev(np.array([pts * 64 + 999, -4, 5000], dtype=np.int32), dev)
        cut = np.full((3, pts * 64), -1, dtype=np.int64)
        for b, n in ((0, pts * 64), (2, 5000)):
            j = np.arange(n)
            cut[b, :n] = np.where(pt[b, j // 64] >= 0, pt[b, j // 64] * 64 + j % 64, -1)
        _check(ops.dense_mla_decode(*args[:3], over), q, O.dequant_latent_rows_fp4(rows), cut)


@pytest.mark.parametrize("H,nsplit", [(16, 1), (48, 1), (32, 2)])
def test_every_count_of_tiles(dev, H, nsplit):
    """Chunks of one to nine tiles (128 keys) and their borders: the first three
    tiles are on their way from the start, later ones follow a tile behind."""
    from lagged_indexer_dsa_amd import ops

    print(f"[fp4 tiles] {(H, nsplit)}", flush=True)
    lens = np.array([n * 128 + d for n in range(1, 9) for d in (-1, 0, 1)], dtype=np.int32)
    B, pts = len(lens), 17
    rng = np.random.default_rng(H)
    pt = rng.permutation(B * pts).reshape(B, pts).astype(np.int32)
    rows, q = _pool(H, B * pts * 64), _q(3, B, H)
    idx = np.full((B, int(lens.max())), -1, dtype=np.int64)
    for b in range(B):
        j = np.arange(lens[b])
        idx[b, :lens[b]] = pt[b, j // 64] * 64 + j % 64
    out = ops.dense_mla_decode(_dev(q, dev, True), _dev(rows, dev), _dev(pt, dev), _dev(lens, dev), nsplit=nsplit)
    _check(out, q, O.dequant_latent_rows_fp4(rows), idx)
    # the same keys as selections
    out = ops.sparse_mla_decode(_dev(q, dev, True), _dev(rows, dev), _dev(idx.astype(np.int32), dev), nsplit=nsplit)
    _check(out, q, O.dequant_latent_rows_fp4(rows), idx)


@pytest.mark.parametrize("nsplit", [1, 0, 3])
@pytest.mark.parametrize("H", [16, 48])
def test_one_key_at_every_border(dev, H, nsplit):
    """Rows whose queries look like one key, which then holds nearly all of the
    weight (a score of about 24 where others are near 1): the output is that key's
    value, so the loss of any one at a border of a tile (128 keys), of a wave's
    part (32), of a page (64) or of a row's end shows in every dim."""
    from lagged_indexer_dsa_amd import ops

    print(f"[fp4 borders] {(H, nsplit)}", flush=True)
    n = 2500
    at = np.unique(np.clip([128 * k + d for k in range(20) for d in (-1, 0)] + [31, 32, 33, 63, 64, 65, 95, 96, 2495, 2499], 0, n - 1))
    B, pts = len(at), -(-n // 64)
    rng = np.random.default_rng(H + nsplit)
    rows = O.pack_latent_rows_fp4(rng.standard_normal((pts * 64, 512)).astype(np.float32),
                                  rng.standard_normal((pts * 64, 64)).astype(np.float32))
    kv = O.dequant_latent_rows_fp4(rows)
    pt = rng.permutation(pts).astype(np.int32)
    j = np.arange(n)
    slots = pt[j // 64].astype(np.int64) * 64 + j % 64
    q = O.bf16_rn(kv[slots[at]][:, None] * np.linspace(0.9, 1.1, H, dtype=np.float32)[None, :, None])
    idx = np.repeat(slots[None], B, 0)
    weight = np.exp(np.einsum("bhd,bd->bh", q.astype(np.float64), kv[slots[at]].astype(np.float64)) * SM)
    assert weight.min() > 100 * n * np.exp(2.0)                    # the key outweighs the rest
    qd, pool, ptd = _dev(q, dev, True), _dev(rows, dev), _dev(np.repeat(pt[None], B, 0), dev)
    _check(ops.sparse_mla_decode(qd, pool, _dev(idx.astype(np.int32), dev), nsplit=nsplit), q, kv, idx)
    # dense: the whole row; rows that end with the key; rows that end just before it
    for lens in (np.full(B, n), at + 1, at):
        cut = np.where(j[None] < lens[:, None], idx, -1)
        _check(ops.dense_mla_decode(qd, pool, ptd, _dev(lens.astype(np.int32), dev), nsplit=nsplit), q, kv, cut)


@pytest.mark.parametrize("B,nsplit,least", [(8, 128, 64), (3, 128, 128), (200, 4, 2)])
def test_long_selections_in_as_many_chunks_as_there_may_be(dev, B, nsplit, least):
    """512 chunks for all rows together: a larger split count gives the bits of the
    one that reaches them."""
    from lagged_indexer_dsa_amd import _lib, ops

    topk = 16384 if B < 100 else 700
    print(f"[fp4 chunks] {(B, topk, nsplit)}", flush=True)
    rng = np.random.default_rng(B)
    rows, q = _pool(33, topk + 1000), _q(33, B, 16)
    idx = np.stack([rng.permutation(topk + 1000)[:topk] for _ in range(B)]).astype(np.int32)
    idx[rng.random(idx.shape) < 0.01] = -1
    args = _dev(q, dev, True), _dev(rows, dev), _dev(idx, dev)
    out = ops.sparse_mla_decode(*args, nsplit=nsplit)
    _check(out, q, O.dequant_latent_rows_fp4(rows), idx)
    assert torch.equal(out, ops.sparse_mla_decode(*args, nsplit=least))
    size = _lib.load().dsa_mla_fp4_workspace_bytes
    # (partials of a chunk and 16 heads; 25 lines of 64 words a barrier; a row's plan)
    assert size(B, 16, nsplit) == min(512, B * nsplit) * 16 * 514 * 4 + B * (25 * 64 * 4 + 8)


@pytest.mark.parametrize("sm", [0.0, -SM, 0.02])
def test_other_scales(dev, sm):
    """A scale that is not positive is applied before the maximum is taken.
    (None is larger than the default, so the bound above holds.)"""
    from lagged_indexer_dsa_amd import ops

    print(f"[fp4 scale] {sm}", flush=True)
    rng = np.random.default_rng(8)
    rows, q = _pool(21, 900), _q(21, 2, 32)
    idx = np.stack([rng.permutation(900)[:700] for _ in range(2)]).astype(np.int32)
    idx[0, rng.random(700) < 0.3] = -1
    idx[1, 300:] = -1
    for nsplit in (1, 0):
        out = ops.sparse_mla_decode(_dev(q, dev, True), _dev(rows, dev), _dev(idx, dev), sm_scale=sm, nsplit=nsplit)
        _check(out, q, O.dequant_latent_rows_fp4(rows), idx, sm)


@pytest.mark.parametrize("nsplit", [1, 2, 0])
def test_tiles_without_a_key(dev, nsplit):
    """Tiles, waves' parts of one and whole chunks whose keys are masked, first, in
    the middle and last, with NaN and infinities in the rows they would name and in
    row 0 (which is read in their place): the keys that are there, alone."""
    from lagged_indexer_dsa_amd import ops

    print(f"[fp4 masked tiles] {nsplit}", flush=True)
    n = 1300
    rows, q = _pool(41, 1344), _q(41, 9, 32)
    rows[0, 256:272], rows[0, 272:400:2] = 255, 0xff
    rows[1, 272:274] = np.array([0xff80], np.uint16).view(np.uint8)            # rope: minus infinity
    idx = np.repeat(np.arange(20, 20 + n)[None], 9, 0)
    idx[0, :300] = -1                                  # the first two tiles and a part of the third
    idx[1, :n - 1] = -1                                # the last key alone
    idx[2, 1:] = -1                                    # the first alone
    idx[3, 128:1280] = 1 << 30                         # all but the first tile and what follows the tenth
    idx[4, :] = -5                                     # none
    idx[5, :] = np.where(np.arange(n) // 32 % 2, idx[5], -1)                   # every second wave's part
    idx[6, :] = np.where(np.arange(n) // 128 % 2, idx[6], 1344)                # every second tile
    idx[7, 96:] = -1
    idx[8, :640] = -1                                  # with two chunks, nearly the first
    out = ops.sparse_mla_decode(_dev(q, dev, True), _dev(rows, dev), _dev(idx.astype(np.int32), dev), nsplit=nsplit)
    clean = rows.copy()
    clean[:2] = 0
    kv = O.dequant_latent_rows_fp4(clean)
    _check(out, q, kv, idx)
    # pages that are not there, in a table of 21
    pt = np.repeat(np.arange(21, dtype=np.int32)[None], 9, 0)
    pt[:, 0] = -1                                      # (the page of rows 0 and 1)
    pt[0, :6], pt[1, :20], pt[2, 2:], pt[3, 2:19] = -1, 21, -1, 1 << 25
    pt[4], pt[5, ::2], pt[6, 4:12], pt[7, 1:20] = -7, -1, -1, -1
    lens = np.array([1344, 1344, 1300, 1344, 1344, 1343, 1281, 1344, 70], dtype=np.int32)
    j = np.arange(1344)
    page = pt[:, j // 64].astype(np.int64)
    cut = np.where((page >= 0) & (page < 21) & (j[None] < lens[:, None]), page * 64 + j % 64, -1)
    out = ops.dense_mla_decode(_dev(q, dev, True), _dev(rows, dev), _dev(pt, dev), _dev(lens, dev), nsplit=nsplit)
    _check(out, q, kv, cut)


def test_sharp_and_growing_scores(dev):
    """Scores whose maximum rises along the row by far more than the sums'
    slack, and rows where one key outweighs the others."""
    from lagged_indexer_dsa_amd import ops

    print("[fp4] growing scores", flush=True)
    n = 3000
    rng = np.random.default_rng(4)
    lat = rng.standard_normal((n, 512)).astype(np.float32)
    lat *= np.linspace(0.05, 40, n, dtype=np.float32)[:, None]
    rows = O.pack_latent_rows_fp4(lat, np.zeros((n, 64), np.float32))
    kv = O.dequant_latent_rows_fp4(rows)
    idx = np.stack([np.arange(n), np.arange(n)[::-1], rng.permutation(n)]).astype(np.int32)
    q = _q(9, 3, 16, 0.3)
    for nsplit in (1, 4, 0):
        out = ops.sparse_mla_decode(_dev(q, dev, True), _dev(rows, dev), _dev(idx, dev), nsplit=nsplit)
        ref = O.mla_decode_values(q, kv, idx, SM)
        # scores to about 300: an fp32 sum's error there (2^-24 * 36 * 5000)
        # moves a probability by 2^-6 of itself at most, its rounding by 2^-8
        for b in range(3):
            s = q[b].astype(np.float64) @ kv[idx[b]].T.astype(np.float64) * SM
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            bound = 2.0 ** -7 * np.abs(ref[b]) + (2.0 ** -6 + 2.0 ** -8) * (p @ np.abs(kv[idx[b], :512].astype(np.float64)))
            assert np.all(np.abs(out[b].double().cpu().numpy() - ref[b]) <= bound)


def test_nan_stays_where_it_is(dev):
    """A NaN group in a row that is not attended reaches nothing; attended, it
    makes its dims (through the score, all of them) NaN for that request only."""
    from lagged_indexer_dsa_amd import ops

    print("[fp4] NaN", flush=True)
    rows = _pool(1, 640)
    rows[100, 256 + 3] = 255
    rows[101, 272:274] = np.array([0x7f80], np.uint16).view(np.uint8)     # rope infinity
    q = _q(1, 3, 16)
    idx = np.stack([np.r_[np.arange(100), np.arange(102, 302)], np.r_[np.arange(200, 499), 100], np.arange(300, 600)])
    out = ops.sparse_mla_decode(_dev(q, dev, True), _dev(rows, dev), _dev(idx.astype(np.int32), dev)).cpu()
    kv = O.dequant_latent_rows_fp4(rows)
    assert out[1].isnan().all() and not out[[0, 2]].isnan().any()
    clean = kv.copy()
    clean[100:102] = 0
    _check(out[[0, 2]], q[[0, 2]], clean, idx[[0, 2]])
    lens = torch.tensor([100, 0], dtype=torch.int32, device=dev)
    pt = torch.arange(10, dtype=torch.int32, device=dev).repeat(2, 1)
    d = ops.dense_mla_decode(_dev(q[:2], dev, True), _dev(rows, dev), pt, lens).cpu()
    assert d.isfinite().all() and not d[1].any()


def test_far_slots(dev):
    from lagged_indexer_dsa_amd import ops

    print("[fp4] far slots", flush=True)
    n = ((1 << 32) // 400 + 4096) // 64 * 64
    pool = torch.zeros(n, 400, dtype=torch.uint8, device=dev)
    rows = _pool(6, 256)
    pool[n - 256:] = _dev(rows, dev)
    q = _q(6, 1, 16)
    idx = (n - 256 + np.arange(256)).astype(np.int32)[None]
    out = ops.sparse_mla_decode(_dev(q, dev, True), pool, _dev(idx, dev))
    _check(out, q, O.dequant_latent_rows_fp4(rows), np.arange(256)[None])
    pt = _dev((n // 64 - 4 + np.arange(4)).astype(np.int32)[None], dev)
    out = ops.dense_mla_decode(_dev(q, dev, True), pool, pt, torch.tensor([256], dtype=torch.int32, device=dev))
    _check(out, q, O.dequant_latent_rows_fp4(rows), np.arange(256)[None])


def test_one_workspace_for_both_formats(dev):
    """Calls over 8- and 4-bit rows take turns with a workspace."""
    from lagged_indexer_dsa_amd import _lib, formats as F, ops

    print("[fp4] shared workspace", flush=True)
    g = torch.Generator(device=dev).manual_seed(2)
    lat, rope = torch.randn(4096, 512, device=dev, generator=g), torch.randn(4096, 64, device=dev, generator=g)
    p8, p4 = F.pack_latent_rows(lat, rope), F.pack_latent_rows_fp4(lat, rope)
    q = torch.randn(2, 16, 576, device=dev, generator=g).to(torch.bfloat16)
    idx = torch.stack([torch.randperm(4096, generator=g, device=dev)[:2048] for _ in range(2)]).int()
    ref8, ref4 = ops.sparse_mla_decode(q, p8, idx), ops.sparse_mla_decode(q, p4, idx)
    assert float((ref8.float() - ref4.float()).norm() / ref8.float().norm()) < 0.5   # the same rows, coarser
    ws = ops.sparse_mla_workspace(2, 16, 0, dev)
    _lib.sync_timeouts(reset=True)
    for _ in range(3):
        assert torch.equal(ops.sparse_mla_decode(q, p4, idx, workspace=ws), ref4)
        got8 = ops.sparse_mla_decode(q, p8, idx, workspace=ws)
        assert float((got8.float() - ref8.float()).abs().max()) <= 2.0 ** -6 * float(ref8.float().abs().max())
    assert _lib.sync_timeouts() == 0


@pytest.mark.parametrize("captured", [False, True])
def test_calls_of_other_batches_on_one_workspace(dev, captured):
    """A workspace for the largest batch: 4-bit calls of fewer rows (whose partial
    sums would begin where the larger batch has barriers) between 8-bit calls of
    all of them, each like the call with a workspace of its own."""
    from lagged_indexer_dsa_amd import _lib, formats as F, ops

    print(f"[fp4] other batches on one workspace, captured {captured}", flush=True)
    g = torch.Generator(device=dev).manual_seed(12)
    lat, rope = torch.randn(4096, 512, device=dev, generator=g), torch.randn(4096, 64, device=dev, generator=g)
    p8, p4 = F.pack_latent_rows(lat, rope), F.pack_latent_rows_fp4(lat, rope)
    q = torch.randn(8, 32, 576, device=dev, generator=g).to(torch.bfloat16)
    idx = torch.stack([torch.randperm(4096, generator=g, device=dev)[:2048] for _ in range(8)]).int()
    pt = torch.arange(64, device=dev, dtype=torch.int32).reshape(8, 8)
    lens = torch.tensor([512, 3, 500, 0, 129, 64, 400, 1], dtype=torch.int32, device=dev)
    ws = ops.sparse_mla_workspace(8, 32, 0, dev)
    outs = [torch.zeros(b, h, 512, dtype=torch.bfloat16, device=dev) for b, h in ((8, 32), (1, 16), (8, 32), (3, 32), (8, 16))]
    q1, q5 = q[:1, :16].contiguous(), q[:, :16].contiguous()
    calls = [lambda w, o: ops.sparse_mla_decode(q, p8, idx, nsplit=4, workspace=w, out=o),
             lambda w, o: ops.sparse_mla_decode(q1, p4, idx[:1], workspace=w, out=o),
             lambda w, o: ops.dense_mla_decode(q, p8, pt, lens, nsplit=3, workspace=w, out=o),
             lambda w, o: ops.dense_mla_decode(q[:3], p4, pt[:3], lens[:3], nsplit=6, workspace=w, out=o),
             lambda w, o: ops.sparse_mla_decode(q5, p4, idx, nsplit=16, workspace=w, out=o)]
    _lib.sync_timeouts(reset=True)
    want = [f(ops.sparse_mla_workspace(8, 32, 0, dev), None).clone() for f in calls]
    run = [lambda f=f, o=o: f(ws, o) for f, o in zip(calls, outs)]
    if captured:
        for k, f in enumerate(run):
            f()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                f()
            run[k] = graph.replay
    for turn in range(3):
        for o in outs:
            o.zero_()
        for k in (1, 0, 3, 2, 4, 0, 1, 2):
            run[k]()
        torch.cuda.synchronize()
        for k, (o, w) in enumerate(zip(outs, want)):
            assert torch.equal(o, w), f"turn {turn}, call {k}"
    assert _lib.sync_timeouts() == 0


def test_graphs_on_one_workspace_and_calls_at_once(dev):
    """Two captured calls of other sizes and formats share a workspace and are
    replayed in turn; calls on two streams with a workspace each run together."""
    from lagged_indexer_dsa_amd import formats as F, ops

    print("[fp4] graphs", flush=True)
    g = torch.Generator(device=dev).manual_seed(5)
    lat, rope = torch.randn(4096, 512, device=dev, generator=g), torch.randn(4096, 64, device=dev, generator=g)
    p4, p8 = F.pack_latent_rows_fp4(lat, rope), F.pack_latent_rows(lat, rope)
    q = torch.randn(2, 32, 576, device=dev, generator=g).to(torch.bfloat16)
    idx = torch.stack([torch.randperm(4096, generator=g, device=dev)[:2048] for _ in range(2)]).int()
    pt = torch.arange(64, device=dev, dtype=torch.int32).reshape(2, 32)
    lens = torch.tensor([2048, 700], dtype=torch.int32, device=dev)
    ws = ops.sparse_mla_workspace(2, 32, 0, dev)
    outs = [torch.zeros(2, 32, 512, dtype=torch.bfloat16, device=dev) for _ in range(3)]
    calls = [lambda: ops.sparse_mla_decode(q, p4, idx, workspace=ws, out=outs[0]),
             lambda: ops.dense_mla_decode(q, p4, pt, lens, nsplit=5, workspace=ws, out=outs[1]),
             lambda: ops.sparse_mla_decode(q, p8, idx, nsplit=8, workspace=ws, out=outs[2])]
    want = [f().clone() for f in calls]
    graphs = []
    for f in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            f()
    for turn in range(4):
        for o in outs:
            o.zero_()
        for k in (turn % 3, (turn + 1) % 3, (turn + 2) % 3):
            graphs[k].replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w), f"turn {turn}"
    streams = [torch.cuda.Stream() for _ in range(2)]
    spaces = [ops.sparse_mla_workspace(2, 32, 0, dev) for _ in streams]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(5):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(ops.sparse_mla_decode(q, p4, idx, workspace=spaces[k]) if k else
                              ops.dense_mla_decode(q, p4, pt, lens, nsplit=5, workspace=spaces[k]))
    torch.cuda.synchronize()
    for o in got[0]:
        assert torch.equal(o, want[1])
    for o in got[1]:
        assert torch.equal(o, want[0])


def test_refusals(dev):
    from lagged_indexer_dsa_amd import ops

    print("[fp4] refusals", flush=True)
    q = torch.zeros(2, 16, 576, dtype=torch.bfloat16, device=dev)
    pool = torch.zeros(128, 400, dtype=torch.uint8, device=dev)
    idx = torch.zeros(2, 64, dtype=torch.int32, device=dev)
    pt, lens = idx[:, :2].contiguous(), idx[:, 0].contiguous()
    s, d = ops.sparse_mla_decode, ops.dense_mla_decode
    for f in (lambda: s(q.float(), pool, idx), lambda: s(q[..., :512].contiguous(), pool, idx),
              lambda: s(q, pool.view(torch.int8), idx), lambda: s(q, pool, idx.long()), lambda: s(q, pool, idx[:1]),
              lambda: s(q[:, :8].contiguous(), pool, idx), lambda: s(q, pool, idx, nsplit=129),
              lambda: s(q, pool, idx, nsplit=16, workspace=torch.zeros(64, device=dev)),
              lambda: s(q, pool, idx, out=torch.zeros(2, 16, 512, device=dev)), lambda: s(q, pool[:0], idx),
              lambda: s(q, pool, idx[:, :0].contiguous()), lambda: s(q, pool, idx[:, ::2]),
              lambda: d(q, pool, pt.long(), lens), lambda: d(q, pool, pt, lens[:1]), lambda: d(q, pool, pt[:1], lens),
              lambda: d(q, pool, pt, lens.long()), lambda: d(q, pool, pt[:, :0].contiguous(), lens)):
        with pytest.raises(RuntimeError):
            f()
