"""CPU: contracts of the operators around the cached attention (no launch):
rope tables against their formulas, the 4-bit row format's builder against the
oracle's exhaustive one, refusals of CPU tensors, and the C ABI's argument
checks, which answer before anything is launched."""

from __future__ import annotations

import math
import shutil
import subprocess
import sys

import numpy as np
import pytest
import torch

from oracle import dsa_oracle as O


@pytest.fixture(scope="module")
def lib():
    from lagged_indexer_dsa_amd import _lib

    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built (run __graft_entry__.build())")
    return _lib.load()


# ---- rope tables ----

def test_plain_table_is_the_formula():
    from lagged_indexer_dsa_amd.rope import build_rope_table

    t = build_rope_table(70001, 64).double().numpy()
    p, i = np.arange(70001)[:, None], np.arange(32)[None, :]
    a = p * 10000.0 ** (-2 * i / 64)
    # one rounding to fp32 of values at most 1; the angle's float64 error is
    # under 70000 * 2^-52, below a tenth of an fp32 half step
    assert np.abs(t[:, :32] - np.cos(a)).max() <= 2.0 ** -24
    assert np.abs(t[:, 32:] - np.sin(a)).max() <= 2.0 ** -24


def test_scaled_frequencies():
    from lagged_indexer_dsa_amd.rope import RopeScaling, build_rope_table, rope_frequencies

    f = rope_frequencies(64, 10000.0)
    lin = rope_frequencies(64, 10000.0, RopeScaling("linear", 8.0))
    assert torch.allclose(lin * 8, f, rtol=1e-15)
    ntk = rope_frequencies(64, 10000.0, RopeScaling("ntk", 8.0))
    assert ntk[0] == f[0] and math.isclose(float(ntk[-1]), float(f[-1]) / 8, rel_tol=1e-12)
    yarn = rope_frequencies(64, 10000.0, RopeScaling("yarn", 40.0))
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(yarn[turns > 40], f[turns > 40])                # fast pairs stay
    slow = turns < 0.7
    assert torch.allclose(yarn[slow], f[slow] / 40, rtol=1e-15)        # slow ones are stretched
    assert bool(((yarn <= f) & (yarn >= f / 40 * (1 - 1e-12))).all()) and bool((yarn[:-1] > yarn[1:]).all())
    t = build_rope_table(4, 64, scaling=RopeScaling("yarn", 40.0))
    assert math.isclose(float(t[0, 0]), 0.1 * math.log(40.0) + 1, rel_tol=1e-7)
    t = build_rope_table(4, 64, scaling=RopeScaling("yarn", 40.0, mscale_all_dim=1.0))
    assert float(t[0, 0]) == 1.0


def test_yarn_where_no_pair_turns_often():
    """A trained context in which even the fastest pair turns less than beta_slow
    times: every pair is slowed by the factor, the first too; one in which the
    slowest turns more than beta_fast times: none is."""
    from lagged_indexer_dsa_amd.rope import RopeScaling, rope_frequencies

    f = rope_frequencies(64, 10000.0)
    for kw in (dict(original_max_pos=6), dict(original_max_pos=1), dict(original_max_pos=100, beta_slow=20.0),
               dict(original_max_pos=4, beta_fast=1.0)):
        assert 0.5 * kw["original_max_pos"] / math.pi < kw.get("beta_slow", 1.0)       # pair 0's turns
        assert torch.allclose(rope_frequencies(64, 10000.0, RopeScaling("yarn", 8.0, **kw)), f / 8, rtol=1e-15), kw
    assert torch.equal(rope_frequencies(64, 10000.0, RopeScaling("yarn", 8.0, original_max_pos=1 << 24)), f)
    # at the first pair's own count of turns the ramp begins with it
    y = rope_frequencies(64, 10000.0, RopeScaling("yarn", 8.0, original_max_pos=200, beta_slow=1.0, beta_fast=40.0))
    assert y[0] == f[0] and torch.allclose(y[-1], f[-1] / 8, rtol=1e-15)


def test_rope_refusals():
    from lagged_indexer_dsa_amd.rope import RopeScaling, build_rope_table

    for kw in (dict(max_pos=0), dict(max_pos=4, dim=63), dict(max_pos=4, dim=0), dict(max_pos=4, theta=1.0),
               dict(max_pos=4, dim=2, scaling=RopeScaling("ntk", 2.0))):
        with pytest.raises(ValueError):
            build_rope_table(**kw)
    for a in (("cubic", 2.0), ("linear", 0.5), ("linear", float("nan")), ("yarn", float("inf"))):
        with pytest.raises(ValueError):
            RopeScaling(*a)
    with pytest.raises(ValueError):
        RopeScaling("yarn", 2.0, beta_fast=1.0, beta_slow=2.0)


# ---- the 4-bit row ----

def fp4_edge_rows() -> np.ndarray:
    """Rows of 512 whose groups hold every code, every midpoint and its
    neighbours, at several scales; zero, tiny, huge and non-finite groups."""
    mags = np.array([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6], np.float32)
    near = np.concatenate([mags, np.nextafter(mags, np.float32(9)), np.nextafter(mags, np.float32(-9))])
    vals = np.concatenate([near, -near]).astype(np.float32)
    groups = []
    for k in (-20, -3, 0, 1, 90, 120):
        for i in range(0, len(vals), 31):
            part = vals[i:i + 31]
            part = part[np.abs(part) <= 6]
            g = np.zeros(32, np.float32)
            g[:len(part)], g[31] = part, 6.0
            groups.append(g * np.float32(2.0 ** k))
    groups.append(np.zeros(32, np.float32))
    groups.append(np.full(32, 1e-9, np.float32))
    groups.append(np.full(32, -1e-40, np.float32))
    groups.append(np.linspace(-3e38, 3.4e38, 32, dtype=np.float32))
    for bad in (np.nan, np.inf, -np.inf):
        g = np.linspace(-2, 2, 32, dtype=np.float32)
        g[7] = bad
        groups.append(g)
    for top in (6.0, np.nextafter(np.float32(6), np.float32(7)), 3.0, 7.9, 8.0, 1e-6, 1.2e-6):
        g = np.linspace(-1, 1, 32, dtype=np.float32) * np.float32(top)
        groups.append(g)
    while len(groups) % 16:
        groups.append(np.zeros(32, np.float32))
    return np.stack(groups).reshape(-1, 512)


def test_fp4_builder_equals_oracle():
    from lagged_indexer_dsa_amd import formats as F

    rng = np.random.default_rng(3)
    lat = np.concatenate([fp4_edge_rows(), rng.standard_normal((40, 512)).astype(np.float32) * 7])
    rope = rng.standard_normal((len(lat), 64)).astype(np.float32)
    ref = O.pack_latent_rows_fp4(lat, rope)
    got = F.pack_latent_rows_fp4(torch.from_numpy(lat), torch.from_numpy(rope)).numpy()
    finite = np.isfinite(lat).reshape(len(lat), 16, 32).all(-1)
    assert np.array_equal(got[:, 256:], ref[:, 256:])
    codes = np.repeat(finite, 16, axis=1)                      # the codes of a NaN group mean nothing
    assert np.array_equal(got[:, :256][codes], ref[:, :256][codes])
    # what they read back as: within half a code step of the value, none saturated
    # (3.4e38 lies nearest to 4 * 2^126 = 2^128, which bf16 holds as infinity)
    back = O.dequant_latent_rows_fp4(ref)[:, :512].reshape(-1, 32)
    x, ok = lat.reshape(-1, 32).astype(np.float64), finite.reshape(-1)
    s = 2.0 ** (ref[:, 256:272].reshape(-1).astype(np.float64) - 127)[:, None]
    half = np.where(np.abs(x) < 2 * s, 0.25, np.where(np.abs(x) < 4 * s, 0.5, 1.0)) * s
    over = np.abs(x) >= 3.5 * 2.0 ** 126
    assert (over & ok[:, None]).any() and np.isinf(back[over & ok[:, None]]).all()
    assert np.all((np.abs(back - x) <= half)[ok & ~over.any(1)]) and np.all((np.abs(back - x) <= half)[~over & ok[:, None]])
    assert np.isnan(back[~ok]).all() and (~ok).sum() == 3


def test_new_latent_pool_formats():
    from lagged_indexer_dsa_amd import formats as F

    assert F.new_latent_pool(2, "cpu").shape == (128, 656)
    assert F.new_latent_pool(2, "cpu", bits=4).shape == (128, 400)
    with pytest.raises(ValueError):
        F.new_latent_pool(2, "cpu", bits=6)


# ---- refusals ----

def test_ops_refuse_cpu_tensors():
    from lagged_indexer_dsa_amd import ops

    x, w = torch.zeros(2, 64), torch.ones(64)
    i = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: ops.rms_norm(x, w), lambda: ops.rms_norm_quant(x, w), lambda: ops.rotary(x, i, torch.zeros(4, 64)),
                 lambda: ops.append_tokens(i[None], i, i, index_k=torch.zeros(1, 8448, dtype=torch.uint8),
                                           keys=torch.zeros(2, 128)),
                 lambda: ops.read_latent_rows(torch.zeros(4, 400, dtype=torch.uint8), i),
                 lambda: ops.sparse_mla_decode(torch.zeros(1, 16, 576, dtype=torch.bfloat16),
                                               torch.zeros(4, 400, dtype=torch.uint8), i[None])):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_import_on_a_torch_without_a_gpu_backend():
    """Such a torch has none of the device functions that a call looks up: the
    package imports, and its ops refuse CPU tensors with their own message."""
    from conftest import PKG_ROOT

    code = f"""
import sys, torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda_")]:
    delattr(torch._C, name)
sys.path.insert(0, {str(PKG_ROOT)!r})
from lagged_indexer_dsa_amd import ops
i = torch.zeros(2, dtype=torch.int32)
for call in (lambda: ops.rms_norm(torch.zeros(2, 64), torch.ones(64)),
             lambda: ops.read_latent_rows(torch.zeros(4, 400, dtype=torch.uint8), i),
             lambda: ops.sparse_mla_decode(torch.zeros(1, 16, 576, dtype=torch.bfloat16),
                                           torch.zeros(4, 656, dtype=torch.uint8), i[None])):
    try:
        call()
        sys.exit("no refusal")
    except RuntimeError as e:
        assert "no CPU path" in str(e), e
"""
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-2000:]


def test_decode_layer_refuses_4bit_pool():
    from lagged_indexer_dsa_amd.decode import DecodeLayer

    with pytest.raises(RuntimeError, match="656"):
        DecodeLayer(q_fp8=None, w=None, index_k=None, q_bf16=torch.zeros(1, 16, 576, dtype=torch.bfloat16),
                    kv_pool=torch.zeros(64, 400, dtype=torch.uint8), page_table=torch.zeros(1, 1, dtype=torch.int32),
                    seq_lens=torch.zeros(1, dtype=torch.int32), slab_stride=64)


def test_packed_arguments_are_the_headers_structures(tmp_path):
    """The Python side packs the argument structures field by field: their
    sizes and last fields' places as a C compiler lays out the header."""
    from conftest import REPO
    from lagged_indexer_dsa_amd._lib import APPEND_ARGS, NORM_ARGS, ROTARY_ARGS

    cc = shutil.which("gcc") or shutil.which("cc")
    if not cc:
        pytest.skip("no C compiler")
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include "dsa_mli.h"\n' + "".join(
        f'_Static_assert(sizeof({t}) == {p.size} && offsetof({t}, {f}) == {at}, "{t}");\n'
        for t, p, f, at in (("dsa_norm_args", NORM_ARGS, "group", 104), ("dsa_rotary_args", ROTARY_ARGS, "inverse", 104),
                            ("dsa_append_args", APPEND_ARGS, "index_interleaved", 148))))
    subprocess.run([cc, "-std=c11", "-fsyntax-only", f"-I{REPO / 'include'}", str(src)], check=True)


def test_norm_contract(lib):
    from lagged_indexer_dsa_amd._lib import NORM_ARGS, DSA_ERR_INVALID_ARG, DSA_ERR_UNSUPPORTED, DSA_OK

    def call(x=16, dt=1, xs=64, r=None, rs=0, w=16, wd=1, y=16, c=None, s=None, g=0, h=None, hs=0, n=2, D=64):
        p = [v or 0 for v in (x, r, w, y, c, s, h)]
        return lib.dsa_rms_norm(NORM_ARGS.pack(*p, xs, rs, hs, 1e-6, n, D, dt, wd, g), None)
    assert lib.dsa_rms_norm(None, None) == DSA_ERR_INVALID_ARG
    assert call(n=0, x=None) == DSA_OK
    for kw in (dict(n=-1), dict(x=None), dict(w=None), dict(y=None), dict(c=16), dict(y=None, c=16), dict(dt=3),
               dict(wd=2), dict(h=16), dict(r=16, rs=64, h=16, hs=63), dict(xs=-64)):
        assert call(**kw) == DSA_ERR_INVALID_ARG, kw
    for kw in (dict(D=0), dict(D=32769), dict(y=None, c=16, s=16, g=64)):
        assert call(**kw) == DSA_ERR_UNSUPPORTED, kw
    assert b"dsa_rms_norm" in lib.dsa_last_error()


def test_rotary_contract(lib):
    from lagged_indexer_dsa_amd._lib import ROTARY_ARGS, DSA_ERR_INVALID_ARG, DSA_ERR_UNSUPPORTED, DSA_OK

    def call(x=16, dt=1, pos=16, pb=4, t=16, P=8, o=16, n=2, H=2, D=64, R=64, start=0):
        p = [v or 0 for v in (x, pos, t, o)]
        return lib.dsa_rotary(ROTARY_ARGS.pack(*p, H * D, D, H * D, D, P, n, H, D, R, start, dt, pb, 0, 0), None)
    assert lib.dsa_rotary(None, None) == DSA_ERR_INVALID_ARG
    assert call(n=0, x=None) == DSA_OK
    for kw in (dict(n=-1), dict(x=None), dict(pos=None), dict(t=None), dict(o=None), dict(dt=5), dict(pb=2), dict(P=0),
               dict(R=0), dict(R=63), dict(R=66), dict(start=2), dict(start=-2, R=32), dict(D=65538),
               dict(start=2 ** 31 - 2, R=4), dict(start=4, R=2 ** 31 - 2)):
        assert call(**kw) == DSA_ERR_INVALID_ARG, kw
    assert call(H=1 << 26) == DSA_ERR_UNSUPPORTED
    assert b"dsa_rotary" in lib.dsa_last_error()


def test_append_and_read_contract(lib):
    from lagged_indexer_dsa_amd._lib import APPEND_ARGS, DSA_ERR_INVALID_ARG, DSA_ERR_UNSUPPORTED, DSA_OK

    def call(rows=16, pos=16, n=2, pt=16, B=1, pts=4, cs=16, cr=8, dt=1, lat=16, ls=576, w=None, wd=0, pool=16, kv=64,
             rb=656, k=16, ks=128, idx=16, pages=1):
        p = [v or 0 for v in (rows, pos, pt, cs, lat, w, pool, k, idx)]
        return lib.dsa_append_tokens(APPEND_ARGS.pack(*p, cr, ls, kv, ks, pages, 1e-6, n, B, pts, dt, wd, rb, 0, 0), None)
    assert lib.dsa_append_tokens(None, None) == DSA_ERR_INVALID_ARG
    assert call(n=0, rows=None) == DSA_OK
    for kw in (dict(n=-1), dict(rows=None), dict(pos=None), dict(pt=None), dict(lat=None, k=None), dict(B=0), dict(pts=0),
               dict(cr=0), dict(dt=3), dict(w=16, wd=2), dict(pool=None), dict(kv=0), dict(pool=24), dict(idx=None),
               dict(pages=0), dict(idx=24), dict(ls=-1)):
        assert call(**kw) == DSA_ERR_INVALID_ARG, kw
    assert call(rb=512) == DSA_ERR_UNSUPPORTED
    r = lib.dsa_read_latent_rows
    assert r(None, 4, 656, None, 0, None, None) == DSA_OK
    assert r(16, 4, 656, 16, -1, 16, None) == DSA_ERR_INVALID_ARG
    assert r(16, 0, 656, 16, 2, 16, None) == DSA_ERR_INVALID_ARG
    assert r(16, 4, 656, None, 2, 16, None) == DSA_ERR_INVALID_ARG
    assert r(24, 4, 656, 16, 2, 16, None) == DSA_ERR_INVALID_ARG
    assert r(16, 4, 600, 16, 2, 16, None) == DSA_ERR_UNSUPPORTED


def test_fp4_mla_contract(lib):
    from lagged_indexer_dsa_amd._lib import DSA_ERR_INVALID_ARG, DSA_ERR_UNSUPPORTED

    f, d, ws = lib.dsa_sparse_mla_decode_fp4, lib.dsa_dense_mla_decode_fp4, lib.dsa_mla_fp4_workspace_bytes
    assert f(16, 16, 10, 16, 16, 16, 1, 24, 2048, 0, 0.04, None) == DSA_ERR_UNSUPPORTED
    assert f(16, 16, 10, 16, 16, 16, 1, 16, 2048, 129, 0.04, None) == DSA_ERR_UNSUPPORTED
    assert f(16, 16, 10, None, 16, 16, 1, 16, 2048, 0, 0.04, None) == DSA_ERR_INVALID_ARG
    assert f(16, 16, 0, 16, 16, 16, 1, 16, 2048, 0, 0.04, None) == DSA_ERR_INVALID_ARG
    assert f(16, 24, 10, 16, 16, 16, 1, 16, 2048, 0, 0.04, None) == DSA_ERR_INVALID_ARG
    assert d(16, 16, 10, None, 4, 16, 16, 16, 1, 16, 0, 0.04, None) == DSA_ERR_INVALID_ARG
    assert d(16, 16, 10, 16, 0, 16, 16, 16, 1, 16, 0, 0.04, None) == DSA_ERR_INVALID_ARG
    assert d(16, 16, 10, 16, (1 << 24) + 1, 16, 16, 16, 1, 16, 0, 0.04, None) == DSA_ERR_UNSUPPORTED
    assert d(16, 16, 10, 16, 4, 16, None, 16, 1, 16, 0, 0.04, None) == DSA_ERR_INVALID_ARG
    assert ws(1, 15, 8) == 0 and ws(0, 16, 8) == 0 and ws(1, 16, 129) == 0
    barriers = 25 * 64 * 4
    assert ws(1, 16, 8) == barriers + 8 * 16 * 514 * 4 + 8       # partial sums, and a plan of 8 bytes a row
    assert ws(3, 32, 8) == 3 * 2 * barriers + 24 * 32 * 514 * 4 + 3 * 8
    assert ws(2, 16, 128) >= ws(2, 16, 64) and ws(7, 16, 1) == 16


def test_workspace_for_any_split_count(lib):
    """The workspace of nsplit 0 holds every split count, of either format."""
    from lagged_indexer_dsa_amd import ops

    for B, H in ((1, 16), (4, 48), (5, 16), (3, 128), (6, 80)):
        nbytes = ops.sparse_mla_workspace(B, H, 0, "cpu").numel() * 4
        for n in range(0, 129):
            assert nbytes >= lib.dsa_mla_fp4_workspace_bytes(B, H, n), (B, H, n)
            assert nbytes >= lib.dsa_sparse_mla_workspace_bytes(B, H, n), (B, H, n)


def _barriers(B, H):
    return B * (H // 16) * 25 * 64 * 4


@pytest.mark.parametrize("B,H,nsplit", [(8, 16, 0), (32, 16, 8), (8, 128, 0), (1, 16, 0), (2, 16, 8), (3, 48, 1),
                                        (100, 64, 2), (300, 16, 3), (64, 128, 0)])
def test_4bit_partials_are_clear_of_every_barrier(lib, B, H, nsplit):
    """One workspace, 8-bit calls of any rows and heads that it is enough for (a
    barrier a row and 16 heads, at its start), 4-bit calls likewise: where the
    4-bit ones write lies behind all of those barriers and inside the workspace."""
    total = lib.dsa_mla_shared_workspace_bytes(B, H, nsplit)
    shapes = [(b, h, n) for b in (1, 2, 3, 5, 8, 31, 32, 33, 100, 256, 257, 300) for h in (16, 32, 48, 64, 128, 1024)
              for n in (0, 1, 2, 3, 8, 64, 65, 128)] + [(B, H, n) for n in range(129)]
    # (what an 8-bit call needs is least for one split)
    last = max(_barriers(b, h) for b, h, _ in shapes if lib.dsa_sparse_mla_workspace_bytes(b, h, 1) <= total)
    assert last >= _barriers(B, H)
    took = refused = 0
    for b, h, n in shapes:
        at, need = lib.dsa_mla_fp4_workspace_in(total, b, h, n), lib.dsa_mla_fp4_workspace_bytes(b, h, n)
        if at < 0:
            refused += 1
        elif need > 16:                                      # (16: nothing is read or written)
            took += 1
            assert last <= at + _barriers(b, h) and at + need <= total and at % 16 == 0, (b, h, n)
    assert took and refused
    if nsplit == 0:  # sized for every count of splits, and for fewer rows
        assert all(lib.dsa_mla_fp4_workspace_in(total, b, H, n) >= 0 for b in range(1, B + 1) for n in range(129))
    else:
        assert lib.dsa_mla_fp4_workspace_in(total, B, H, nsplit) >= 0
    # the partials begin where those of an 8-bit call of these rows and heads would, counted from there
    assert lib.dsa_sparse_mla_barrier_bytes(B, H, 0) == _barriers(B, H)


def test_shared_workspace_contract(lib):
    assert lib.dsa_mla_shared_workspace_bytes(1, 15, 8) == 0 and lib.dsa_mla_shared_workspace_bytes(0, 16, 8) == 0
    assert lib.dsa_mla_shared_workspace_bytes(1, 16, 129) == 0
    f = lib.dsa_mla_fp4_workspace_in
    assert f(1 << 30, 1, 15, 8) == -1 and f(1 << 30, 1, 16, -1) == -1 and f(0, 1, 16, 8) == -1
    assert f(16, 7, 16, 1) == 0 and f(15, 7, 16, 1) == -1    # unsplit rows read none
    from lagged_indexer_dsa_amd import ops

    for B, H, n in ((1, 16, 8), (5, 32, 1), (4, 16, 0)):
        assert ops.sparse_mla_workspace(B, H, n, "cpu").nbytes == lib.dsa_mla_shared_workspace_bytes(B, H, n)
    with pytest.raises(RuntimeError):
        ops.sparse_mla_workspace(1, 24, 8, "cpu")


def test_workspace_of_8bit_layers(lib):
    """A layer over 656-byte rows holds what its calls need and no 4-bit partials."""
    from lagged_indexer_dsa_amd import ops
    from lagged_indexer_dsa_amd.decode import DecodeLayer

    for B, H, n in ((1, 16, 0), (3, 32, 8), (100, 16, 0)):
        want = lib.dsa_sparse_mla_workspace_bytes(B, H, n)
        assert ops.sparse_mla_workspace(B, H, n, "cpu", kv_bits=8).nbytes == want
        for bits in (None, 4):
            assert ops.sparse_mla_workspace(B, H, n, "cpu", kv_bits=bits).nbytes == lib.dsa_mla_shared_workspace_bytes(B, H, n)
        layer = DecodeLayer(q_fp8=None, w=None, index_k=None, q_bf16=torch.zeros(B, H, 576, dtype=torch.bfloat16),
                            kv_pool=torch.zeros(64, 656, dtype=torch.uint8),
                            page_table=torch.zeros(B, 1, dtype=torch.int32), seq_lens=torch.zeros(B, dtype=torch.int32),
                            slab_stride=64, nsplit=n)
        assert layer.workspace.nbytes == want
    with pytest.raises(ValueError):
        ops.sparse_mla_workspace(1, 16, 0, "cpu", kv_bits=6)
