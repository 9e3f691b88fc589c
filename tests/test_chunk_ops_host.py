"""CPU: contracts of the chunk and 8-bit product operators (no launch): the C
ABI's argument checks, which answer before anything is launched, the packed
structures against the header, the weight builder against a plain loop, and
refusals of CPU tensors."""

from __future__ import annotations

import shutil
import subprocess

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


def test_packed_arguments_are_the_headers_structures(tmp_path):
    from conftest import REPO
    from lagged_indexer_dsa_amd._lib import MATMUL_ARGS, QUANT_ARGS

    cc = shutil.which("gcc") or shutil.which("cc")
    if not cc:
        pytest.skip("no C compiler")
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include "dsa_mli.h"\n' + "".join(
        f'_Static_assert(sizeof({t}) == {p.size} && offsetof({t}, {f}) == {at}, "{t}");\n'
        for t, p, f, at in (("dsa_quant_args", QUANT_ARGS, "group", 60), ("dsa_matmul_args", MATMUL_ARGS, "out_dtype", 68))))
    subprocess.run([cc, "-std=c11", "-fsyntax-only", f"-I{REPO / 'include'}", str(src)], check=True)


def test_quantize_rows_contract(lib):
    from lagged_indexer_dsa_amd._lib import DSA_ERR_INVALID_ARG, DSA_ERR_UNSUPPORTED, DSA_OK, QUANT_ARGS

    def call(x=16, g=0, c=16, s=16, xs=64, gs=0, n=2, D=64, dt=1, group=128):
        return lib.dsa_quantize_rows(QUANT_ARGS.pack(x, g, c, s, xs, gs, n, D, dt, group), None)
    assert lib.dsa_quantize_rows(None, None) == DSA_ERR_INVALID_ARG
    assert call(n=0, x=0) == DSA_OK
    for kw in (dict(n=-1), dict(x=0), dict(c=0), dict(s=0), dict(dt=3), dict(dt=-1), dict(xs=-1), dict(g=16, gs=-2)):
        assert call(**kw) == DSA_ERR_INVALID_ARG, kw
    for kw in (dict(D=0), dict(D=32769), dict(group=64)):
        assert call(**kw) == DSA_ERR_UNSUPPORTED, kw
    assert b"dsa_quantize_rows" in lib.dsa_last_error()


def test_fp8_matmul_contract(lib):
    from lagged_indexer_dsa_amd._lib import DSA_ERR_INVALID_ARG, DSA_ERR_UNSUPPORTED, DSA_OK, MATMUL_ARGS

    def call(a=16, sa=16, w=16, sw=16, off=0, out=16, rows=2, N=8, K=256, E=1, groups=2, dt=1):
        return lib.dsa_fp8_matmul(MATMUL_ARGS.pack(a, sa, w, sw, off, out, rows, N, K, E, groups, dt), None)
    assert lib.dsa_fp8_matmul(None, None) == DSA_ERR_INVALID_ARG
    assert call(rows=0, a=0) == DSA_OK and call(N=0, w=0) == DSA_OK
    for kw in (dict(rows=-1), dict(N=-1), dict(a=0), dict(sa=0), dict(w=0), dict(sw=0), dict(out=0), dict(E=0), dict(E=2),
               dict(groups=3), dict(groups=0), dict(dt=3), dict(a=24), dict(w=24)):
        assert call(**kw) == DSA_ERR_INVALID_ARG, kw
    for kw in (dict(K=0), dict(K=100), dict(K=131088), dict(rows=2 ** 31 - 1, N=2 ** 20), dict(off=16, E=2 ** 20, N=1024)):
        assert call(**{"groups": 1, **kw}) == DSA_ERR_UNSUPPORTED, kw
    assert b"dsa_fp8_matmul" in lib.dsa_last_error()


def test_chunk_contracts(lib):
    from lagged_indexer_dsa_amd._lib import DSA_ERR_INVALID_ARG, DSA_ERR_UNSUPPORTED, DSA_OK

    def scan(q=16, w=16, k=16, pages=4, pt=16, st=16, seq=16, out=16, n=3, B=2, H=64, pts=4, slab=256):
        return lib.dsa_chunk_scan(q, w, k, pages, pt, st, seq, out, n, B, H, pts, slab, None)
    assert scan(n=0, q=None) == DSA_OK and scan(B=0, pt=None) == DSA_OK
    for kw in (dict(n=-1), dict(B=-1), dict(q=None), dict(w=None), dict(k=None), dict(pt=None), dict(st=None), dict(seq=None),
               dict(out=None), dict(pages=0), dict(pts=0), dict(slab=0), dict(q=24), dict(k=24), dict(w=24)):
        assert scan(**kw) == DSA_ERR_INVALID_ARG, kw
    for kw in (dict(H=24), dict(H=80), dict(slab=(1 << 28) + 1), dict(pts=(1 << 22) + 1)):
        assert scan(**kw) == DSA_ERR_UNSUPPORTED, kw

    def attend(q=16, kv=16, rows=64, rb=656, pt=16, st=16, seq=16, ws=16, out=16, n=3, B=2, H=16, pts=4):
        return lib.dsa_chunk_attention(q, kv, rows, rb, pt, st, seq, ws, out, n, B, H, pts, 0.04, None)
    assert attend(n=0, q=None) == DSA_OK and attend(B=0, pt=None) == DSA_OK
    for kw in (dict(n=-1), dict(B=-1), dict(q=None), dict(kv=None), dict(pt=None), dict(st=None), dict(seq=None),
               dict(ws=None), dict(out=None), dict(rows=0), dict(q=24), dict(kv=24), dict(ws=24), dict(out=20)):
        assert attend(**kw) == DSA_ERR_INVALID_ARG, kw
    for kw in (dict(H=24), dict(H=0), dict(H=1040), dict(rb=600), dict(pts=0), dict(pts=(1 << 22) + 1), dict(n=2 ** 27)):
        assert attend(**kw) == DSA_ERR_UNSUPPORTED, kw
    size = lib.dsa_chunk_attention_workspace_bytes
    assert size(0, 16) == 0 and size(1, 24) == 0 and size(2 ** 27, 16) == 0
    sizes = [size(n, 16) for n in (1, 2, 7, 8, 9, 1000, 100000)]
    assert sizes == sorted(sizes) and sizes[-1] == size(8, 16) and sizes[0] < sizes[2] and sizes[-1] < 135 * 2 ** 20
    assert size(3, 128) == size(1, 128) == size(8, 16)                          # a tile's 128 rows are the most


@pytest.mark.parametrize("N,K", [(1, 16), (128, 128), (130, 300), (300, 1040)])
def test_quantize_weight_is_blocks_of_the_rowwise_rule(N, K):
    from lagged_indexer_dsa_amd import formats

    w = torch.randn(2, N, K, generator=torch.Generator().manual_seed(N))
    codes, scale = formats.quantize_weight(w)
    assert codes.shape == (2, N, K) and codes.dtype == torch.uint8
    assert scale.shape == (2, -(-N // 128), -(-K // 128)) and scale.dtype == torch.float32
    for e in range(2):
        for i in range(0, N, 128):
            for j in range(0, K, 128):
                block = w[e, i:i + 128, j:j + 128].numpy()
                want, s = O.quantize_rowwise(block.reshape(1, -1))
                assert np.array_equal(codes[e, i:i + 128, j:j + 128].numpy().reshape(1, -1), want)
                assert scale[e, i // 128, j // 128] == s[0]


def test_ops_refuse_cpu_tensors():
    from lagged_indexer_dsa_amd import ops

    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)  # noqa: E731
    i = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    one = torch.ones(2, 1)
    for call in (lambda: ops.quantize_rows(torch.zeros(2, 64)), lambda: ops.fp8_matmul(u8(2, 64), one, u8(4, 64), torch.ones(1, 1)),
                 lambda: ops.fp8_matmul_grouped(u8(2, 64), one, u8(1, 4, 64), torch.ones(1, 1, 1), i(0, 2)),
                 lambda: ops.chunk_scan(u8(1, 16, 128), torch.ones(1, 16), u8(1, 8448), i(0)[None], i(0, 1), i(1), 64),
                 lambda: ops.chunk_attention(torch.zeros(1, 16, 576, dtype=torch.bfloat16), u8(64, 656), i(0)[None], i(0, 1), i(1))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
