"""GPU: ops.append_tokens and ops.read_latent_rows against the oracle.

Without a rotation every stored byte is the oracle's (a norm is computed in
fp64, so that its fp32 value is the rounded one).  A turned value is off by two
fp32 roundings of its products before its own rounding; its codes are held to
half a code step of that.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import dsa_oracle as O
from test_layer_ops_host import fp4_edge_rows

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _case(dev, seed, n, B, npg, dtype, lens=400, scale=1.0):
    rng = np.random.default_rng(seed)
    pt = np.full((B, npg), -1, dtype=np.int32)
    need = -(-lens // 64)
    pt[:, :need] = rng.permutation(B * need).reshape(B, need)
    flat = rng.permutation(B * lens)[:n]
    rows, pos = (flat // lens).astype(np.int32), (flat % lens).astype(np.int32)
    g = torch.Generator(device=dev).manual_seed(seed)
    lat = (torch.randn(n, 576, generator=g, device=dev) * scale).to(dtype)
    keys = (torch.randn(n, 128, generator=g, device=dev) * scale).to(dtype)
    t = lambda a: torch.from_numpy(a).to(dev)  # noqa: E731
    return dict(pt=t(pt), rows=t(rows), pos=t(pos), lat=lat, keys=keys, pages=B * need,
                slots=pt[rows, pos // 64].astype(np.int64) * 64 + pos % 64)


def _np(t):
    return t.double().cpu().numpy()


def _pack(bits, lat, rope):
    f = O.pack_latent_rows if bits == 8 else O.pack_latent_rows_fp4
    return f(lat.astype(np.float32), rope.astype(np.float32))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,norm", [(1, True), (37, False), (333, True)])
def test_append_without_rotation_is_the_oracles_bytes(dev, bits, dtype, n, norm):
    from lagged_indexer_dsa_amd import ops

    print(f"[append] {bits} bits {dtype} n={n} norm={norm}", flush=True)
    c = _case(dev, n + bits, n, 3, 9, dtype)
    row = 656 if bits == 8 else 400
    pool = torch.full((c["pages"] * 64, row), 0xA5, dtype=torch.uint8, device=dev)
    idx = torch.full((c["pages"], 8448), 0x5A, dtype=torch.uint8, device=dev)
    w = (1 + 0.3 * torch.randn(512, device=dev, generator=torch.Generator(device=dev).manual_seed(1))).to(dtype)
    ops.append_tokens(c["pt"], c["rows"], c["pos"], kv_pool=pool, latent=c["lat"], index_k=idx, keys=c["keys"],
                      norm_weight=w if norm else None, eps=1e-5)
    x = _np(c["lat"])
    lat = O.rms_norm(x[:, :512], _np(w), 1e-5)[0] if norm else x[:, :512]
    ref = np.full(tuple(pool.shape), 0xA5, dtype=np.uint8)
    ref[c["slots"]] = _pack(bits, lat, x[:, 512:])
    assert np.array_equal(pool.cpu().numpy(), ref)
    codes, scale = O.quantize_rowwise(_np(c["keys"]))
    refi = np.full(tuple(idx.shape), 0x5A, dtype=np.uint8)
    for i, s in enumerate(c["slots"]):
        p, k = divmod(int(s), 64)
        refi[p, 128 * k:128 * k + 128] = codes[i]
        refi[p, 8192 + 4 * k:8196 + 4 * k] = scale[i:i + 1].view(np.uint8)
    assert np.array_equal(idx.cpu().numpy(), refi)
    # read back: what the attention sees
    got = ops.read_latent_rows(pool, torch.from_numpy(c["slots"].astype(np.int32)).to(dev))
    vals = (O.dequant_latent_rows if bits == 8 else O.dequant_latent_rows_fp4)(ref[c["slots"]])
    assert np.array_equal(got.float().cpu().numpy(), vals)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_append_with_rotation(dev, inter, dtype):
    from lagged_indexer_dsa_amd import ops
    from lagged_indexer_dsa_amd.rope import RopeScaling, build_rope_table

    print(f"[append] rotation {inter} {dtype}", flush=True)
    c = _case(dev, 5, 200, 2, 7, dtype)
    table = build_rope_table(400, 64, scaling=RopeScaling("yarn", 4.0), device=dev)
    pool = torch.zeros(c["pages"] * 64, 656, dtype=torch.uint8, device=dev)
    idx = torch.zeros(c["pages"], 8448, dtype=torch.uint8, device=dev)
    # inputs as slices of a wider projection
    both = torch.cat([c["lat"].new_zeros(200, 8), c["lat"], c["keys"]], dim=1)
    ops.append_tokens(c["pt"], c["rows"], c["pos"], kv_pool=pool, latent=both[:, 8:584], index_k=idx, keys=both[:, 584:],
                      cos_sin=table, interleaved=inter, index_interleaved=not inter)
    t = _np(table)[c["pos"].cpu().numpy()]
    x, k = _np(c["lat"]), _np(c["keys"])
    rows = pool.cpu().numpy()[c["slots"]]
    assert np.array_equal(rows[:, :528], O.pack_latent_rows(x[:, :512].astype(np.float32), np.zeros((200, 64)))[:, :528])
    ref = O.rotate(x[:, 512:], t[:, :32], t[:, 32:], inter)
    size = 2 * np.abs(x[:, 512:]).max() * np.abs(t).max()
    got = O.bf16_from_bits(rows[:, 528:].copy().view(np.uint16)).astype(np.float64)
    assert np.all(np.abs(got - ref) <= 2.0 ** -8 * np.abs(ref) + 2 * 2.0 ** -24 * size)
    kr = np.concatenate([O.rotate(k[:, :64], t[:, :32], t[:, 32:], not inter), k[:, 64:]], axis=1)
    pages = idx.cpu().numpy()
    p, s = c["slots"] // 64, c["slots"] % 64
    codes = pages[:, :8192].reshape(-1, 64, 128)[p, s]
    scale = pages[:, 8192:].copy().view(np.float32)[p, s].astype(np.float64)[:, None]
    top = np.abs(kr).max(1, keepdims=True) / 448
    assert np.all(np.abs(scale - top) <= 2.0 ** -22 * top + 2.0 ** -23 * size / 448)
    err = np.abs(O.e4m3_decode(codes) * scale - kr)
    assert np.all(err <= (2.0 ** -4 + 2.0 ** -20) * np.abs(kr) + 2.0 ** -10 * scale + 2.0 ** -23 * size)


def test_append_equals_the_older_ops(dev):
    """Without norm and rotation: the bytes that append_latent_rows and
    append_index_keys store."""
    from lagged_indexer_dsa_amd import ops

    print("[append] older ops", flush=True)
    c = _case(dev, 11, 700, 4, 8, torch.bfloat16, scale=9.0)
    a = [torch.zeros(c["pages"] * 64, 656, dtype=torch.uint8, device=dev) for _ in range(2)]
    b = [torch.zeros(c["pages"], 8448, dtype=torch.uint8, device=dev) for _ in range(2)]
    ops.append_tokens(c["pt"], c["rows"], c["pos"], kv_pool=a[0], latent=c["lat"])
    ops.append_tokens(c["pt"], c["rows"], c["pos"], index_k=b[0], keys=c["keys"])
    ops.append_latent_rows(a[1], torch.from_numpy(c["slots"].astype(np.int32)).to(dev), c["lat"])
    ops.append_index_keys(b[1], c["pt"], c["rows"], c["pos"], c["keys"])
    assert torch.equal(*a) and torch.equal(*b)


def test_fp4_edges(dev):
    """Every code, midpoint and scale border, non-finite groups, unaligned rows."""
    from lagged_indexer_dsa_amd import ops

    print("[append] 4-bit edges", flush=True)
    lat = fp4_edge_rows()
    n = len(lat)
    x = torch.zeros(n, 577, device=dev)
    x[:, 1:513] = torch.from_numpy(lat).to(dev)
    pt = torch.arange(-(-n // 64), dtype=torch.int32, device=dev)[None]
    pos = torch.arange(n, dtype=torch.int32, device=dev)
    ref = O.pack_latent_rows_fp4(lat, np.zeros((n, 64), np.float32))
    finite = np.repeat(np.isfinite(lat).reshape(n, 16, 32).all(-1), 16, axis=1)
    for src in (x[:, 1:], x[:, 1:].contiguous()):
        pool = torch.zeros(pt.shape[1] * 64, 400, dtype=torch.uint8, device=dev)
        ops.append_tokens(pt, torch.zeros_like(pos), pos, kv_pool=pool, latent=src)
        got = pool[:n].cpu().numpy()
        assert np.array_equal(got[:, 256:], ref[:, 256:])
        assert np.array_equal(got[:, :256][finite], ref[:, :256][finite])
        back = ops.read_latent_rows(pool, pos).float().cpu().numpy()
        assert np.array_equal(back, O.dequant_latent_rows_fp4(ref), equal_nan=True)


def test_nan_reaches_the_cache(dev):
    from lagged_indexer_dsa_amd import ops

    print("[append] NaN", flush=True)
    c = _case(dev, 3, 4, 1, 2, torch.float32, lens=64)
    c["lat"][1, 130] = float("nan")
    c["lat"][2, 520] = float("inf")
    c["keys"][1, 100] = float("nan")
    pool = torch.zeros(64, 656, dtype=torch.uint8, device=dev)
    idx = torch.zeros(1, 8448, dtype=torch.uint8, device=dev)
    ops.append_tokens(c["pt"], c["rows"], c["pos"], kv_pool=pool, latent=c["lat"], index_k=idx, keys=c["keys"])
    v = ops.read_latent_rows(pool, torch.from_numpy(c["slots"].astype(np.int32)).to(dev)).float().cpu()
    assert v[1, 128:256].isnan().all() and not v[1, :128].isnan().any() and not v[1, 256:].isnan().any()
    assert v[2, 520].isinf() and v[[0, 3]].isfinite().all()
    scale = idx[0, 8192:].view(torch.float32).cpu()
    assert scale[int(c["slots"][1])].isnan() and scale[int(c["slots"][0])].isfinite()
    ops.append_tokens(c["pt"], c["rows"], c["pos"], kv_pool=pool, latent=c["lat"], norm_weight=torch.ones(512, device=dev))
    v = ops.read_latent_rows(pool, torch.from_numpy(c["slots"].astype(np.int32)).to(dev)).float().cpu()
    assert v[1, :512].isnan().all()


@pytest.mark.parametrize("bits", [8, 4])
def test_tokens_without_a_place_are_skipped(dev, bits):
    from lagged_indexer_dsa_amd import ops
    from lagged_indexer_dsa_amd.rope import build_rope_table

    print(f"[append] skipped tokens {bits}", flush=True)
    row = 656 if bits == 8 else 400
    pt = torch.tensor([[2, -1, 900, 1, 5]], dtype=torch.int32, device=dev)
    rows = torch.tensor([0, 0, 0, 0, 0, 1, -1, 0, 0, 0], dtype=torch.int32, device=dev)
    pos = torch.tensor([3, 64, 130, 320, -1, 0, 0, 200, 2 ** 31 - 1, 300], dtype=torch.int32, device=dev)
    # 3: stored; 64, 130: no page; 320, -1, 2^31-1: outside the table; rows 1, -1:
    # none; 200: page 1; 300: page 5, not in the pools
    n = len(rows)
    lat = torch.randn(n, 576, device=dev)
    keys = torch.randn(n, 128, device=dev)
    pool = torch.full((5 * 64 - 1, row), 0x11, dtype=torch.uint8, device=dev)
    idx = torch.full((5, 8448), 0x22, dtype=torch.uint8, device=dev)
    ops.append_tokens(pt, rows, pos, kv_pool=pool, latent=lat, index_k=idx, keys=keys)
    touched = (pool != 0x11).any(1).nonzero().flatten().tolist()
    assert touched == [64 + 200 % 64, 2 * 64 + 3]
    assert (idx != 0x22).any(1).nonzero().flatten().tolist() == [1, 2]
    # a table that ends before position 200
    pool.fill_(0x11)
    ops.append_tokens(pt, rows, pos, kv_pool=pool, latent=lat, cos_sin=build_rope_table(200, 64, device=dev))
    assert (pool != 0x11).any(1).nonzero().flatten().tolist() == [2 * 64 + 3]
    slots = torch.tensor([-1, 0, 5 * 64 - 1, 5 * 64 - 2, 2 ** 31 - 1], dtype=torch.int32, device=dev)
    v = ops.read_latent_rows(pool, slots)
    assert bool((v[[0, 2, 4]] == 0).all()) and bool((v[[1, 3]] != 0).any(1).all())
    assert ops.read_latent_rows(pool, slots[:0]).shape == (0, 576)
    ops.append_tokens(pt, rows[:0], pos[:0], kv_pool=pool, latent=lat[:0])


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("kv_rows,pages", [(128, 4), (256, 2), (150, 3)])
def test_a_token_is_in_both_caches_or_in_none(dev, bits, kv_rows, pages):
    """Caches of other capacities: what one has no place for, the other does not
    hold either; a call for one of them goes by that one's capacity."""
    from lagged_indexer_dsa_amd import ops

    print(f"[append] caches of other capacities {(bits, kv_rows, pages)}", flush=True)
    row = 656 if bits == 8 else 400
    pt = torch.tensor([[3, 1, 2, 0]], dtype=torch.int32, device=dev)
    pos = torch.arange(5, 256, 10, dtype=torch.int32, device=dev)
    rows = torch.zeros_like(pos)
    g = torch.Generator(device=dev).manual_seed(5)
    lat, keys = torch.randn(len(pos), 576, device=dev, generator=g), torch.randn(len(pos), 128, device=dev, generator=g)
    slots = pt[0].long()[pos.long() // 64] * 64 + pos.long() % 64
    in_kv, in_idx = slots < kv_rows, slots // 64 < pages
    assert bool((in_kv & in_idx).any()) and bool((~(in_kv & in_idx)).any())

    def held(**kw):
        pool = torch.full((kv_rows, row), 0x11, dtype=torch.uint8, device=dev)
        idx = torch.full((pages, 8448), 0x22, dtype=torch.uint8, device=dev)
        both = dict(kv_pool=pool, latent=lat, index_k=idx, keys=keys)
        ops.append_tokens(pt, rows, pos, **{k: v for k, v in both.items() if k in kw["of"]})
        a = (pool != 0x11).any(1).nonzero().flatten()
        codes, scales = idx[:, :8192].reshape(pages * 64, 128), idx[:, 8192:].reshape(pages * 64, 4)
        b, s = (codes != 0x22).any(1).nonzero().flatten(), (scales != 0x22).any(1).nonzero().flatten()
        assert torch.equal(b, s)
        return a.tolist(), b.tolist()
    want = lambda m: sorted(slots[m].tolist())  # noqa: E731
    assert held(of=("kv_pool", "latent", "index_k", "keys")) == (want(in_kv & in_idx), want(in_kv & in_idx))
    assert held(of=("kv_pool", "latent")) == (want(in_kv), [])
    assert held(of=("index_k", "keys")) == ([], want(in_idx))


@pytest.mark.parametrize("bits", [8, 4])
def test_slots_past_2_31_bytes(dev, bits):
    from lagged_indexer_dsa_amd import ops

    print(f"[append] far slots {bits}", flush=True)
    row = 656 if bits == 8 else 400
    pages = (1 << 32) // (row * 64) + 10
    pool = torch.zeros(pages * 64, row, dtype=torch.uint8, device=dev)
    pt = torch.tensor([[pages - 1, 0]], dtype=torch.int32, device=dev)
    rows = torch.zeros(2, dtype=torch.int32, device=dev)
    pos = torch.tensor([63, 64], dtype=torch.int32, device=dev)
    lat = torch.randn(2, 576, device=dev, generator=torch.Generator(device=dev).manual_seed(9))
    ops.append_tokens(pt, rows, pos, kv_pool=pool, latent=lat)
    slots = torch.tensor([pages * 64 - 1, 0], dtype=torch.int32, device=dev)
    x = lat.cpu().numpy()
    ref = _pack(bits, x[:, :512], x[:, 512:])
    assert np.array_equal(pool[slots.long()].cpu().numpy(), ref)
    vals = (O.dequant_latent_rows if bits == 8 else O.dequant_latent_rows_fp4)(ref)
    assert np.array_equal(ops.read_latent_rows(pool, slots).float().cpu().numpy(), vals)


def test_append_of_more_tokens_than_a_launch_holds(dev):
    """A wave a token: 2^26 are more than a launch has.  Nearly all are padding;
    those with a place are at the borders of the launches it takes."""
    from lagged_indexer_dsa_amd import ops

    print("[append] 2^26 + 9 tokens", flush=True)
    n = (1 << 26) + 9
    at = torch.tensor([0, 1, (1 << 25) - 1, 1 << 25, (1 << 25) + 3, (1 << 26) - 1, 1 << 26, n - 2, n - 1], device=dev)
    rows = torch.full((n,), -1, dtype=torch.int32, device=dev)
    pos = torch.zeros(n, dtype=torch.int32, device=dev)
    rows[at] = 0
    pos[at] = 7 * torch.arange(len(at), device=dev, dtype=torch.int32)
    g = torch.Generator(device=dev).manual_seed(4)
    lat, keys = torch.randn(1, 576, device=dev, generator=g), torch.randn(1, 128, device=dev, generator=g)
    pt = torch.tensor([[1]], dtype=torch.int32, device=dev)
    pool, idx = torch.zeros(128, 400, dtype=torch.uint8, device=dev), torch.zeros(2, 8448, dtype=torch.uint8, device=dev)
    ops.append_tokens(pt, rows, pos, kv_pool=pool, latent=lat.expand(n, 576), index_k=idx, keys=keys.expand(n, 128))
    slots = [64 + 7 * k for k in range(len(at))]
    assert pool.any(1).nonzero().flatten().tolist() == slots
    assert idx[:, :8192].reshape(128, 128).any(1).nonzero().flatten().tolist() == slots
    x = lat.cpu().numpy()
    assert np.array_equal(pool[slots].cpu().numpy(), np.repeat(_pack(4, x[:, :512], x[:, 512:]), len(at), 0))


@pytest.mark.parametrize("bits", [8, 4])
def test_read_in_more_than_one_launch(dev, bits):
    """2^26 rows a launch; 77 GB of values."""
    from lagged_indexer_dsa_amd import ops

    n = (1 << 26) + 9
    if torch.cuda.mem_get_info(dev)[0] < 90 << 30:
        torch.cuda.empty_cache()
    if torch.cuda.mem_get_info(dev)[0] < 90 << 30:
        pytest.skip("needs 90 GB of device memory")
    print(f"[read] 2^26 + 9 rows {bits}", flush=True)
    rng = np.random.default_rng(bits)
    rows = _pack(bits, rng.standard_normal((3, 512)), rng.standard_normal((3, 64)))
    f = O.dequant_latent_rows if bits == 8 else O.dequant_latent_rows_fp4
    vals = torch.cat([torch.from_numpy(f(rows)), torch.zeros(1, 576)]).to(dev).to(torch.bfloat16)
    slots = (torch.arange(n, device=dev) % 4).int()       # (3: outside the pool, zeros)
    out = ops.read_latent_rows(torch.from_numpy(rows).to(dev), slots)
    for a in range(0, n, 1 << 22):
        assert torch.equal(out[a:a + (1 << 22)], vals[slots[a:a + (1 << 22)].long()])
    del out
    torch.cuda.empty_cache()


def test_append_and_read_refusals(dev):
    from lagged_indexer_dsa_amd import ops

    print("[append] refusals", flush=True)
    c = _case(dev, 2, 4, 1, 2, torch.bfloat16, lens=64)
    pool = torch.zeros(64, 400, dtype=torch.uint8, device=dev)
    idx = torch.zeros(1, 8448, dtype=torch.uint8, device=dev)
    ok = dict(kv_pool=pool, latent=c["lat"], index_k=idx, keys=c["keys"])
    t = torch.zeros(64, 64, device=dev)

    def call(pt=c["pt"], rows=c["rows"], pos=c["pos"], **kw):
        return lambda: ops.append_tokens(pt, rows, pos, **{**ok, **kw})
    for f in (call(kv_pool=None), call(latent=None), call(index_k=None), call(keys=c["keys"].float()),
              call(latent=c["lat"][:3]), call(latent=c["lat"].t().contiguous().t()), call(kv_pool=pool[:, :300]),
              call(kv_pool=pool.float()), call(index_k=idx[:, :8000]), call(cos_sin=t[:, :32].contiguous()),
              call(cos_sin=t.half()), call(norm_weight=torch.ones(576, device=dev)), call(rows=c["rows"].long()),
              call(pos=c["pos"][:3]), call(pt=c["pt"].long()), call(latent=None, kv_pool=None, index_k=None, keys=None),
              call(latent=None, kv_pool=None, norm_weight=torch.ones(512, device=dev)), call(kv_pool=pool[:0]),
              call(norm_weight=torch.ones(512, device=dev).half()),
              lambda: ops.read_latent_rows(pool[:, :300].contiguous(), c["rows"]),
              lambda: ops.read_latent_rows(pool, c["rows"].long()),
              lambda: ops.read_latent_rows(pool, c["rows"], out=torch.zeros(3, 576, dtype=torch.bfloat16, device=dev)),
              lambda: ops.append_latent_rows(pool, c["rows"], c["lat"])):
        with pytest.raises(RuntimeError):
            f()
