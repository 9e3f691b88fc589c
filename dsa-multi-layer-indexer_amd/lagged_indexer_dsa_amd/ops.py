"""torch-tensor entry points onto the C ABI (one launch sequence each).

Every op requires device (HIP) tensors and runs on torch's current stream;
there is no CPU path.  Shapes/dtypes are checked here; the library re-checks
its own contract and raises :class:`DsaError` (a RuntimeError) on violation.
"""

from __future__ import annotations

import torch

from . import _lib
from ._lib import (
    DSA_TOPK_POSITION_ORDER,
    DSA_TOPK_SORTED,
    FP4_ROW_BYTES,
    INDEX_DIM,
    INDEX_PAGE_BYTES,
    LATENT_DIM,
    LATENT_ROW_BYTES,
    MATMUL_MAX_K,
    NORM_MAX_DIM,
    PAGE_TOKENS,
    QK_DIM,
    ROPE_DIM,
)


def _dev(*tensors: torch.Tensor) -> None:
    for t in tensors:
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise RuntimeError("lagged_indexer_dsa_amd ops need GPU (HIP) tensors; there is no CPU path")
        if not t.is_contiguous():
            raise RuntimeError("lagged_indexer_dsa_amd ops need contiguous tensors")


def _current_device() -> int:
    # (looked up in the call: a torch without a GPU backend has no such function)
    return torch._C._cuda_getDevice()


def _stream() -> int:
    # torch.cuda.current_stream().cuda_stream without building the two objects
    # around it (0.2 us against 2.7, a fifth of a small call)
    return torch._C._cuda_getCurrentRawStream(_current_device())


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _nbytes(t: torch.Tensor) -> int:
    return t.nbytes


def _need_bytes(name: str, t: torch.Tensor, nbytes: int) -> None:
    """The C ABI takes raw pointers: a caller buffer smaller than the
    library's size function says would be overrun on the device."""
    if _nbytes(t) < nbytes:
        raise RuntimeError(f"{name} holds {_nbytes(t)} bytes, the call needs {nbytes}")


def _need_shape(name: str, t: torch.Tensor, shape: tuple, dtype) -> None:
    if t.shape != shape or t.dtype != dtype or not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous {dtype} {tuple(shape)}, got {t.dtype} {tuple(t.shape)}")


def indexer_scan(q_fp8: torch.Tensor, w: torch.Tensor, index_k: torch.Tensor,
                 page_table: torch.Tensor, seq_lens: torch.Tensor, slab_stride: int,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """fp8 lightning-indexer scores over the paged index-K cache.

    q_fp8 [B,Hidx,128] uint8 (e4m3 codes) or float8_e4m3fn; w [B,Hidx] f32
    (q-scale folded in); index_k [P,8448] uint8; page_table [B,pt] int32;
    seq_lens [B] int32  ->  scores [B, slab_stride] f32 (-inf past seq_len).
    Reference: K:2990-2992 ref_indexer_logits_fp8; attention_core.py:27-49.
    """
    q_fp8 = q_fp8.view(torch.uint8) if q_fp8.dtype == torch.float8_e4m3fn else q_fp8
    _dev(q_fp8, w, index_k, page_table, seq_lens)
    B, Hidx, D = q_fp8.shape
    if D != INDEX_DIM or q_fp8.dtype != torch.uint8:
        raise RuntimeError("q_fp8 must be [B, Hidx, 128] e4m3 bytes")
    if w.shape != (B, Hidx) or w.dtype != torch.float32:
        raise RuntimeError("w must be [B, Hidx] float32")
    if index_k.dim() != 2 or index_k.shape[1] != INDEX_PAGE_BYTES or index_k.dtype != torch.uint8:
        raise RuntimeError("index_k must be [pages, 8448] uint8")
    if page_table.dim() != 2 or page_table.shape[0] != B or page_table.dtype != torch.int32:
        raise RuntimeError("page_table must be [B, pt_stride] int32")
    if seq_lens.shape != (B,) or seq_lens.dtype != torch.int32:
        raise RuntimeError("seq_lens must be [B] int32")
    if out is None:
        out = torch.empty(B, slab_stride, dtype=torch.float32, device=q_fp8.device)
    _dev(out)
    if out.shape != (B, slab_stride) or out.dtype != torch.float32:
        raise RuntimeError("out must be [B, slab_stride] float32")
    _lib.call("dsa_indexer_scan", q_fp8.data_ptr(), w.data_ptr(), index_k.data_ptr(),
              index_k.shape[0], page_table.data_ptr(), seq_lens.data_ptr(), out.data_ptr(),
              B, Hidx, page_table.shape[1], slab_stride, _stream())
    return out


def topk_scratch(B: int, slab: int, device) -> torch.Tensor:
    """Zero-filled scratch for :func:`topk` (each call leaves it zeroed)."""
    nbytes = _lib.load().dsa_topk_scratch_bytes(B, slab)
    if nbytes == 0:
        raise RuntimeError(f"bad top-k scratch shape B={B} slab={slab}")
    return torch.zeros(nbytes // 4, dtype=torch.int32, device=device)


def topk(scores: torch.Tensor, seq_lens: torch.Tensor, k: int, sorted: bool = False,
         pad_value: int = -1, page_table: torch.Tensor | None = None,
         out: torch.Tensor | None = None, scratch: torch.Tensor | None = None) -> torch.Tensor:
    """Exact top-k per row (score desc, ties -> lower index), int32 [B, k].

    sorted=False: ascending positions (or KV slots through page_table), pads
    last.  sorted=True: torch.topk order with the lower-index tie rule.
    Non-finite selections and missing slots are ``pad_value``.
    Reference: attention_core.py:66-91 select_topk.
    """
    _dev(scores, seq_lens)
    if scores.dim() != 2 or scores.dtype != torch.float32:
        raise RuntimeError("scores must be [B, slab] float32")
    B, slab = scores.shape
    if seq_lens.shape != (B,) or seq_lens.dtype != torch.int32:
        raise RuntimeError("seq_lens must be [B] int32")
    if page_table is not None:
        _dev(page_table)
    if out is None:
        out = torch.empty(B, k, dtype=torch.int32, device=scores.device)
    if scratch is None:
        scratch = topk_scratch(B, slab, scores.device)
    _dev(out, scratch)
    _need_shape("out", out, (B, k), torch.int32)
    _need_bytes("top-k scratch", scratch, _lib.load().dsa_topk_scratch_bytes(B, slab))
    _lib.call("dsa_topk", scores.data_ptr(), seq_lens.data_ptr(), _ptr(page_table),
              0 if page_table is None else page_table.shape[1], scratch.data_ptr(),
              out.data_ptr(), B, slab, k,
              DSA_TOPK_SORTED if sorted else DSA_TOPK_POSITION_ORDER, pad_value, _stream())
    return out


def select_rows(scores: torch.Tensor, k: int, pad_value: int) -> torch.Tensor | None:
    """:func:`topk` with sorted=True over whole rows, as int64 and in one
    launch; None for the shapes the row kernel does not take."""
    _dev(scores)
    shape = scores.shape
    if len(shape) != 2 or scores.dtype != torch.float32:
        raise RuntimeError("scores must be [B, slab] float32")
    B, slab = shape
    if not _lib.load().dsa_select_rows_supported(B, slab, k):
        return None
    out = torch.empty(B, k, dtype=torch.int64, device=scores.device)
    _lib.call("dsa_select_rows", scores.data_ptr(), None, out.data_ptr(), B, slab, k, pad_value, _stream())
    return out


def sparse_mla_workspace(B: int, H: int, nsplit: int, device, kv_bits: int | None = None) -> torch.Tensor:
    """Zero-filled workspace (split partials + the splits' barriers; every
    call leaves the barriers ready), for pools of either row format.  nsplit=0
    sizes it for any split count; kv_bits=8 for pools of 656-byte rows only (for
    a few rows less than half the bytes).

    Calls over 400-byte rows of any B and H that it is enough for may use it, in
    turn with calls over 656-byte rows.  Those must all be of one B * H: their
    partials begin behind as many barriers as the call itself has.
    """
    lib = _lib.load()
    if kv_bits not in (None, 4, 8):
        raise ValueError(f"latent rows are kept in 8 or 4 bits, got {kv_bits}")
    size = lib.dsa_sparse_mla_workspace_bytes if kv_bits == 8 else lib.dsa_mla_shared_workspace_bytes
    nbytes = size(B, H, nsplit)
    if nbytes == 0:
        raise RuntimeError(f"bad sparse MLA workspace shape B={B} H={H} nsplit={nsplit}")
    return torch.zeros(nbytes // 4, dtype=torch.float32, device=device)


def _call_workspace(B: int, H: int, nsplit: int, device) -> torch.Tensor:
    """Workspace of one call at a known split count: the barriers zeroed, the
    partials (overwritten before they are read) not.  Many unsplit rows read
    neither."""
    lib = _lib.load()
    nbytes = lib.dsa_sparse_mla_workspace_bytes(B, H, nsplit)
    if nbytes == 0:
        raise RuntimeError(f"bad sparse MLA workspace shape B={B} H={H} nsplit={nsplit}")
    barriers = lib.dsa_sparse_mla_barrier_bytes(B, H, nsplit)
    ws = torch.empty(nbytes // 4 if barriers else 4, dtype=torch.float32, device=device)
    ws[:barriers // 4].zero_()
    return ws


def _resolve_nsplit(nsplit: int, B: int, H: int, keys: int) -> int:
    """The split count a call takes (nsplit = 0: the library's choice)."""
    return nsplit or max(1, _lib.load().dsa_sparse_mla_auto_nsplit(B, H, keys))


def _here(dev: int, *tensors: torch.Tensor | None) -> None:
    """All on device `dev`, the one the call's kernels go to."""
    for t in tensors:
        if t is not None and t.get_device() != dev:
            if dev < 0 or t.get_device() < 0:
                raise RuntimeError("lagged_indexer_dsa_amd ops need GPU (HIP) tensors; there is no CPU path")
            raise RuntimeError(f"tensors on different devices: cuda:{dev} and {t.device}")
    if dev < 0:
        raise RuntimeError("lagged_indexer_dsa_amd ops need GPU (HIP) tensors; there is no CPU path")
    if dev != _current_device():
        raise RuntimeError(f"tensors are on cuda:{dev}, the current device is cuda:{_current_device()}")


def _fp4_call(q, kv_pool, sm_scale, nsplit: int, workspace, out, *others):
    """What a decode call over 400-byte rows checks besides its keys; ws: the
    address in the workspace that the call gets."""
    qs = q.shape
    if len(qs) != 3 or qs[2] != QK_DIM or q.dtype != torch.bfloat16:
        raise RuntimeError("q must be [B, H, 576] bfloat16")
    if kv_pool.dtype != torch.uint8:
        raise RuntimeError("kv_pool must be [rows, 400] uint8")
    B, H, _ = qs
    _here(q.get_device(), kv_pool, workspace, out, *others)
    lib = _lib.load()
    if workspace is None:
        workspace = torch.empty(lib.dsa_mla_fp4_workspace_bytes(B, H, nsplit), dtype=torch.uint8, device=q.device)
        ws = workspace.data_ptr()
    else:  # behind the barriers that calls over 656-byte rows may have in it
        at = lib.dsa_mla_fp4_workspace_in(_nbytes(workspace), B, H, nsplit)
        if at < 0:
            raise RuntimeError(f"the 4-bit MLA workspace of {_nbytes(workspace)} bytes is not enough for B={B} H={H} "
                               f"nsplit={nsplit} (ops.sparse_mla_workspace: "
                               f"{lib.dsa_mla_shared_workspace_bytes(B, H, nsplit)} bytes)")
        if not workspace.is_contiguous():
            raise RuntimeError("the 4-bit MLA workspace must be contiguous")
        ws = workspace.data_ptr() + at
    if out is None:
        out = torch.empty(B, H, LATENT_DIM, dtype=torch.bfloat16, device=q.device)
    else:
        _need_shape("out", out, (B, H, LATENT_DIM), torch.bfloat16)
    return B, H, QK_DIM ** -0.5 if sm_scale is None else float(sm_scale), workspace, ws, out


def sparse_mla_decode(q: torch.Tensor, kv_pool: torch.Tensor, idx: torch.Tensor,
                      sm_scale: float | None = None, nsplit: int = 0,
                      workspace: torch.Tensor | None = None,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """Split-K sparse MLA over the latent pool, in 656-byte fp8 rows or in
    400-byte 4-bit ones.

    q [B,H,576] bf16; kv_pool [rows,656] or [rows,400] uint8; idx [B,topk]
    int32 KV slots (out-of-range = masked)  ->  out [B,H,512] bf16.
    Reference: attention_core.py:121-146 sparse_mla_core; K:2950-2966.
    """
    _dev(q, kv_pool, idx)
    if kv_pool.dim() == 2 and kv_pool.shape[1] == FP4_ROW_BYTES:
        B, H, sm_scale, workspace, ws, out = _fp4_call(q, kv_pool, sm_scale, nsplit, workspace, out, idx)
        if idx.dim() != 2 or idx.shape[0] != B or idx.dtype != torch.int32:
            raise RuntimeError("idx must be [B, topk] int32")
        _lib.call("dsa_sparse_mla_decode_fp4", q.data_ptr(), kv_pool.data_ptr(), kv_pool.shape[0], idx.data_ptr(), ws,
                  out.data_ptr(), B, H, idx.shape[1], nsplit, sm_scale, _stream())
        return out
    if q.dim() != 3 or q.shape[2] != QK_DIM or q.dtype != torch.bfloat16:
        raise RuntimeError("q must be [B, H, 576] bfloat16")
    B, H, _ = q.shape
    if kv_pool.dim() != 2 or kv_pool.shape[1] != LATENT_ROW_BYTES or kv_pool.dtype != torch.uint8:
        raise RuntimeError("kv_pool must be [rows, 656] uint8")
    if idx.dim() != 2 or idx.shape[0] != B or idx.dtype != torch.int32:
        raise RuntimeError("idx must be [B, topk] int32")
    if sm_scale is None:
        sm_scale = QK_DIM ** -0.5
    if workspace is None:
        nsplit = _resolve_nsplit(nsplit, B, H, idx.shape[1])
        workspace = _call_workspace(B, H, nsplit, q.device)
    else:  # sized for this nsplit (nsplit=0, the library's choice: the largest size)
        _dev(workspace)
        _need_bytes("sparse MLA workspace", workspace, _lib.load().dsa_sparse_mla_workspace_bytes(B, H, nsplit))
    if out is None:
        out = torch.empty(B, H, LATENT_DIM, dtype=torch.bfloat16, device=q.device)
    _dev(out)
    _need_shape("out", out, (B, H, LATENT_DIM), torch.bfloat16)
    _lib.call("dsa_sparse_mla_decode", q.data_ptr(), kv_pool.data_ptr(), kv_pool.shape[0],
              idx.data_ptr(), workspace.data_ptr(), out.data_ptr(), B, H, idx.shape[1], nsplit,
              float(sm_scale), _stream())
    return out


def dense_mla_decode(q: torch.Tensor, kv_pool: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                     sm_scale: float | None = None, nsplit: int = 0,
                     workspace: torch.Tensor | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Dense MLA of each decode row over its first seq_lens[b] tokens, their
    latent rows found through the page table (64-token pages).

    q [B,H,576] bf16; kv_pool [rows,656] or [rows,400] uint8; page_table
    [B,pt] int32; seq_lens [B] int32  ->  out [B,H,512] bf16.
    Reference: attention_core.py:142-160 dense_mla_core; model.py:104-114.
    """
    _dev(q, kv_pool, page_table, seq_lens)
    if kv_pool.dim() == 2 and kv_pool.shape[1] == FP4_ROW_BYTES:
        B, H, sm_scale, workspace, ws, out = _fp4_call(q, kv_pool, sm_scale, nsplit, workspace, out, page_table, seq_lens)
        if page_table.dim() != 2 or page_table.shape[0] != B or page_table.dtype != torch.int32:
            raise RuntimeError("page_table must be [B, pt_stride] int32")
        _need_shape("seq_lens", seq_lens, (B,), torch.int32)
        _lib.call("dsa_dense_mla_decode_fp4", q.data_ptr(), kv_pool.data_ptr(), kv_pool.shape[0],
                  page_table.data_ptr(), page_table.shape[1], seq_lens.data_ptr(), ws, out.data_ptr(), B, H, nsplit,
                  sm_scale, _stream())
        return out
    if q.dim() != 3 or q.shape[2] != QK_DIM or q.dtype != torch.bfloat16:
        raise RuntimeError("q must be [B, H, 576] bfloat16")
    B, H, _ = q.shape
    if kv_pool.dim() != 2 or kv_pool.shape[1] != LATENT_ROW_BYTES or kv_pool.dtype != torch.uint8:
        raise RuntimeError("kv_pool must be [rows, 656] uint8")
    if page_table.dim() != 2 or page_table.shape[0] != B or page_table.dtype != torch.int32:
        raise RuntimeError("page_table must be [B, pt_stride] int32")
    _need_shape("seq_lens", seq_lens, (B,), torch.int32)
    if sm_scale is None:
        sm_scale = QK_DIM ** -0.5
    if workspace is None:
        nsplit = _resolve_nsplit(nsplit, B, H, page_table.shape[1] * PAGE_TOKENS)
        workspace = _call_workspace(B, H, nsplit, q.device)
    else:  # sized for this nsplit (nsplit=0, the library's choice: the largest size)
        _dev(workspace)
        _need_bytes("sparse MLA workspace", workspace, _lib.load().dsa_sparse_mla_workspace_bytes(B, H, nsplit))
    if out is None:
        out = torch.empty(B, H, LATENT_DIM, dtype=torch.bfloat16, device=q.device)
    _dev(out)
    _need_shape("out", out, (B, H, LATENT_DIM), torch.bfloat16)
    _lib.call("dsa_dense_mla_decode", q.data_ptr(), kv_pool.data_ptr(), kv_pool.shape[0], page_table.data_ptr(),
              page_table.shape[1], seq_lens.data_ptr(), workspace.data_ptr(), out.data_ptr(), B, H, nsplit,
              float(sm_scale), _stream())
    return out


# ---- prefill attention (many query rows against the same keys) ----

_PACK_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _kernel_input(x: torch.Tensor) -> torch.Tensor:
    """x as the prefill kernels read it: fp32, bf16 or fp16, contiguous,
    16-byte aligned."""
    x = (x if x.dtype in _PACK_DTYPES else x.float()).contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _need_kv(kv: torch.Tensor) -> None:
    shape = kv.shape
    if len(shape) != 3 or shape[2] != QK_DIM:
        raise RuntimeError(f"kv must be [B, T, 576], got {tuple(shape)}")


def _pack_source(kv: torch.Tensor) -> torch.Tensor:
    """kv [B, T, 576] as the pack kernels read it (rope rounded to bf16 once)."""
    if kv.dtype not in _PACK_DTYPES:
        x = kv.float()
        x[..., LATENT_DIM:] = kv[..., LATENT_DIM:].to(torch.bfloat16)
        kv = x
    return _kernel_input(kv)


def prefill_logits(q: torch.Tensor, k: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """Indexer scores [B, S, T] fp32 of q [B, S, H, 128] and w [B, S, H] over
    k [B, T, 128], quantised per row inside.  Reference: attention_core.py:27-49."""
    q, k, w = _kernel_input(q), _kernel_input(k), _kernel_input(w)
    _dev(q, k, w)
    qs, ks = q.shape, k.shape  # (each read of a shape builds it anew)
    if len(qs) != 4 or qs[3] != INDEX_DIM:
        raise RuntimeError(f"q must be [B, S, H, 128], got {tuple(qs)}")
    B, S, H, _ = qs
    if len(ks) != 3 or ks[0] != B or ks[2] != INDEX_DIM:
        raise RuntimeError(f"k must be [{B}, T, 128], got {tuple(ks)}")
    if w.shape != qs[:3]:
        raise RuntimeError(f"w must be {(B, S, H)}, got {tuple(w.shape)}")
    T = ks[1]
    ws = torch.empty(_lib.load().dsa_prefill_logits_workspace_bytes(B, S, H, T), dtype=torch.uint8, device=q.device)
    out = torch.empty(B, S, T, dtype=torch.float32, device=q.device)
    _lib.call("dsa_prefill_logits", q.data_ptr(), _PACK_DTYPES[q.dtype], k.data_ptr(), _PACK_DTYPES[k.dtype],
              w.data_ptr(), _PACK_DTYPES[w.dtype], ws.data_ptr(), out.data_ptr(), B, S, H, T, _stream())
    return out


def pack_latent_rows(kv: torch.Tensor, row_stride: int) -> torch.Tensor:
    """kv [B, T, 576] -> 656-byte fp8 rows [B * row_stride, 656] (rows past T
    of a request zero)."""
    _need_kv(kv)
    kv = _pack_source(kv)
    _dev(kv)
    B, T, _ = kv.shape
    if row_stride < T:
        raise RuntimeError(f"row_stride {row_stride} below the {T} rows of a request")
    rows = torch.empty(B * row_stride, LATENT_ROW_BYTES, dtype=torch.uint8, device=kv.device)
    _lib.call("dsa_pack_latent_rows", kv.data_ptr(), _PACK_DTYPES[kv.dtype], B, T, row_stride, rows.data_ptr(),
              _stream())
    return rows


def selection_set(idx: torch.Tensor, T: int, as_bits: bool) -> torch.Tensor:
    """Selections idx [B, S, n] (int32 or int64 positions) as sets over the
    row's causal keys (query row s of S sees keys 0 .. T - S + s): a bitmap per
    row, or the KV slots b * T + position ascending, then -1 [B * S, n]."""
    idx = idx.contiguous()
    _dev(idx)
    shape = idx.shape
    if len(shape) != 3 or idx.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"idx must be [B, S, n] int32 or int64, got {idx.dtype} {tuple(shape)}")
    B, S, n = shape
    lib = _lib.load()
    if as_bits:
        out = torch.empty(lib.dsa_selection_bits_bytes(B * S, T) // 4, dtype=torch.int32, device=idx.device)
    else:
        out = torch.empty(B * S, n, dtype=torch.int32, device=idx.device)
    _lib.call("dsa_selection_set", idx.data_ptr(), idx.element_size(), B, S, n, T,
              out.data_ptr() if as_bits else None, None if as_bits else out.data_ptr(), _stream())
    return out


def prefill_attention(q: torch.Tensor, kv: torch.Tensor, bits: torch.Tensor | None = None,
                      sm_scale: float | None = None) -> torch.Tensor:
    """q [B, S, H, 576] bf16 over kv [B, T, 576]: query row s of S attends keys
    0 .. T - S + s, or those of its bitmap (:func:`selection_set`) ->
    [B, S, H, 512] bf16.  Reference: attention_core.py:121-160."""
    _need_kv(kv)
    kv = _pack_source(kv)
    _dev(q, kv)
    qs = q.shape
    if len(qs) != 4 or qs[3] != QK_DIM or q.dtype != torch.bfloat16:
        raise RuntimeError("q must be [B, S, H, 576] bfloat16")
    B, S, H, _ = qs
    requests, T, _ = kv.shape
    if requests != B:
        raise RuntimeError(f"kv holds {requests} requests, q {B}")
    lib = _lib.load()
    keys = torch.empty(lib.dsa_prefill_keys_bytes(B, T), dtype=torch.uint8, device=q.device)
    ws = torch.empty(lib.dsa_prefill_workspace_bytes(B, S, H, T), dtype=torch.uint8, device=q.device)
    out = torch.empty(B, S, H, LATENT_DIM, dtype=torch.bfloat16, device=q.device)
    if bits is not None:
        _dev(bits)
        if bits.dtype != torch.int32:
            raise RuntimeError("bits must be int32")
        _need_bytes("bits", bits, lib.dsa_selection_bits_bytes(B * S, T))
    st = _stream()
    _lib.call("dsa_pack_prefill_keys", kv.data_ptr(), _PACK_DTYPES[kv.dtype], B, T, keys.data_ptr(), st)
    _lib.call("dsa_prefill_attention", q.data_ptr(), keys.data_ptr(), _ptr(bits), ws.data_ptr(), out.data_ptr(),
              B, S, H, T, float(QK_DIM ** -0.5 if sm_scale is None else sm_scale), st)
    return out


# ---- decode-step operand preparation (the inputs the decode layer reads) ----

def quantize_index_query(q: torch.Tensor, w: torch.Tensor, out_q: torch.Tensor | None = None,
                         out_w: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Indexer query [B, Hidx, 128] bf16 and head weights [B, Hidx] fp32 ->
    (e4m3 codes uint8 [B, Hidx, 128], folded weights w * scale fp32).
    Per (token, head): scale = max(amax, 1e-6) / 448 (K:2969-2974, K:2984-2985)."""
    _dev(q, w)
    if q.dim() != 3 or q.shape[2] != INDEX_DIM or q.dtype != torch.bfloat16:
        raise RuntimeError("q must be [B, Hidx, 128] bfloat16")
    B, H, _ = q.shape
    _need_shape("w", w, (B, H), torch.float32)
    if out_q is None:
        out_q = torch.empty(B, H, INDEX_DIM, dtype=torch.uint8, device=q.device)
    if out_w is None:
        out_w = torch.empty(B, H, dtype=torch.float32, device=q.device)
    _dev(out_q, out_w)
    _need_shape("out_q", out_q, (B, H, INDEX_DIM), torch.uint8)
    _need_shape("out_w", out_w, (B, H), torch.float32)
    _lib.call("dsa_quantize_index_query", q.data_ptr(), w.data_ptr(), out_q.data_ptr(), out_w.data_ptr(),
              B, H, _stream())
    return out_q, out_w


def append_index_keys(index_k: torch.Tensor, page_table: torch.Tensor, rows: torch.Tensor,
                      pos: torch.Tensor, keys: torch.Tensor) -> None:
    """Quantize keys [n, 128] bf16 (per token, e4m3 + fp32 scale) into the
    paged index cache at token positions pos[i] of rows rows[i] (P:339-342)."""
    _dev(index_k, page_table, rows, pos, keys)
    n = keys.shape[0]
    if keys.dim() != 2 or keys.shape[1] != INDEX_DIM or keys.dtype != torch.bfloat16:
        raise RuntimeError("keys must be [n, 128] bfloat16")
    if index_k.dim() != 2 or index_k.shape[1] != INDEX_PAGE_BYTES or index_k.dtype != torch.uint8:
        raise RuntimeError("index_k must be [pages, 8448] uint8")
    if page_table.dim() != 2 or page_table.dtype != torch.int32:
        raise RuntimeError("page_table must be [B, pt_stride] int32")
    _need_shape("rows", rows, (n,), torch.int32)
    _need_shape("pos", pos, (n,), torch.int32)
    _lib.call("dsa_append_index_keys", keys.data_ptr(), rows.data_ptr(), pos.data_ptr(), n,
              page_table.data_ptr(), page_table.shape[1], index_k.data_ptr(), index_k.shape[0], _stream())


def append_latent_rows(kv_pool: torch.Tensor, slots: torch.Tensor, latent: torch.Tensor) -> None:
    """Pack latent [n, 576] bf16 (512 latent | 64 rope) into 656-byte fp8 rows
    at KV slots slots[i] (per-128 e4m3 + fp32 scales, bf16 rope; K:1114)."""
    _dev(kv_pool, slots, latent)
    n = latent.shape[0]
    if latent.dim() != 2 or latent.shape[1] != QK_DIM or latent.dtype != torch.bfloat16:
        raise RuntimeError("latent must be [n, 576] bfloat16")
    if kv_pool.dim() != 2 or kv_pool.shape[1] != LATENT_ROW_BYTES or kv_pool.dtype != torch.uint8:
        raise RuntimeError("kv_pool must be [rows, 656] uint8")
    _need_shape("slots", slots, (n,), torch.int32)
    _lib.call("dsa_append_latent_rows", latent.data_ptr(), slots.data_ptr(), n, kv_pool.data_ptr(),
              kv_pool.shape[0], _stream())


# ---- around the cached attention: norm, rotation, cache appends and reads ----

def _row_stride(name: str, x: torch.Tensor, n: int, D: int) -> int:
    """The stride between the n rows of x [..., D]; refuses what has none."""
    if x.is_contiguous():
        return D
    st = x.stride()
    if D > 1 and st[-1] != 1:
        raise RuntimeError(f"{name}'s last dimension must be contiguous")
    if n <= 1:
        return D
    dims = [(k, t) for k, t in zip(x.shape[:-1], st[:-1]) if k > 1]
    for (k, t), (_, outer) in zip(dims[1:], dims[:-1]):
        if outer != k * t:
            raise RuntimeError(f"{name}'s leading dimensions must be one stride apart, got strides {st}")
    return dims[-1][1]


def _new(x: torch.Tensor, shape, dtype) -> torch.Tensor:
    """A contiguous tensor on x's device.  (Of x's own shape and type 1.2 us;
    from single sizes 1.4, from a shape 2.4.)"""
    if dtype == x.dtype and shape == x.shape and x.is_contiguous():
        return torch.empty_like(x)
    return torch.empty(*shape, dtype=dtype, device=x.device)


def _span(t: torch.Tensor) -> tuple[int, int]:
    """The bytes a non-empty tensor lies in."""
    at = t.data_ptr()
    if t.is_contiguous():
        return at, at + t.nbytes
    end = 1
    for n, st in zip(t.shape, t.stride()):
        end += (n - 1) * st
    return at, at + end * t.element_size()


def _need_apart(name: str, out: torch.Tensor, *inputs: torch.Tensor | None) -> None:
    """An output's bytes hold none of the inputs'."""
    lo, hi = _span(out)
    for t in inputs:
        if t is not None:
            a, b = _span(t)
            if a < hi and lo < b:
                raise RuntimeError(f"{name} overlaps an input")


def _norm(x, weight, eps, residual, outs, group, out_residual):
    """Checks and launch of a norm; outs: its output and, quantised, the
    scales, as the caller gave them (None: new ones).  Returns all outputs."""
    shape, dt = x.shape, x.dtype
    dtype = _PACK_DTYPES.get(dt)
    if dtype is None:
        raise RuntimeError(f"x must be float32, bfloat16 or float16, got {dt}")
    dev = x.get_device()
    D = shape[-1] if shape else 0
    if not 1 <= D <= NORM_MAX_DIM:
        raise RuntimeError(f"x must be [..., D] with D from 1 to {NORM_MAX_DIM}, got {tuple(shape)}")
    _here(dev, weight, residual, out_residual, *outs)
    n = x.numel() // D
    wt = weight.dtype
    if weight.shape != (D,) or (wt != dt and wt != torch.float32) or not weight.is_contiguous():
        raise RuntimeError(f"weight must be [{D}] of x's type or float32, got {wt} {tuple(weight.shape)}")
    quant = len(outs) == 2
    if quant:
        sshape = (*shape[:-1], -(-D // 128) if group else 1)
        kinds = (("out_q", shape, torch.uint8), ("out_scale", sshape, torch.float32))
    else:
        kinds = (("out", shape, dt),)
    res = []
    for t, (name, want, kind) in zip(outs, kinds):
        if t is None:
            t = _new(x, want, kind)
        else:
            _need_shape(name, t, want, kind)
            if n:
                _need_apart(name, t, x, residual, weight, out_residual, *res)
        res.append(t)
    xs, rs, hs, rp, hp = _row_stride("x", x, n, D), 0, 0, 0, 0
    if residual is not None:
        if residual.dtype != dt or residual.shape != shape:
            raise RuntimeError(f"residual must be {dt} {tuple(shape)}, got {residual.dtype} {tuple(residual.shape)}")
        rs, rp = _row_stride("residual", residual, n, D), residual.data_ptr()
        if out_residual is None:
            h = _new(x, shape, dt)
            hs = D
        else:
            h = out_residual
            if h.dtype != dt or h.shape != shape:
                raise RuntimeError(f"out_residual must be {dt} {tuple(shape)}, got {h.dtype} {tuple(h.shape)}")
            hs = _row_stride("out_residual", h, n, D)
            if n > 1 and hs < D:
                raise RuntimeError("out_residual's rows overlap")
            if n:
                same = h is residual or (h.data_ptr() == rp and hs == rs)
                _need_apart("out_residual", h, x, weight, None if same else residual)
        hp = h.data_ptr()
        res.append(h)
    elif out_residual is not None:
        raise RuntimeError("out_residual without a residual")
    if n:
        y = res[0].data_ptr()
        a = _lib.NORM_ARGS.pack(x.data_ptr(), rp, weight.data_ptr(), 0 if quant else y, y if quant else 0,
                                res[1].data_ptr() if quant else 0, hp, xs, rs, hs, eps, n, D, dtype, _PACK_DTYPES[wt],
                                group)
        _lib.call("dsa_rms_norm", a, torch._C._cuda_getCurrentRawStream(dev))
    return res


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: torch.Tensor | None = None,
             out: torch.Tensor | None = None, out_residual: torch.Tensor | None = None):
    """h = x + residual (or x); h / sqrt(mean(h^2) + eps) * weight over the last
    dim, in fp32 -> out, of x's type; with a residual (out, h).

    x [..., D] fp32, bf16 or fp16 (rows any one stride apart, D up to 32768),
    residual of the same shape and type, weight [D] of x's type or fp32.
    out_residual may be residual itself; otherwise outputs must not overlap
    inputs (a tensor reaches from its first element to its last, so an output
    between an input's rows is refused too).  h is rounded to x's type only as it is stored.
    Reference: dsa_layer.py:32-52 RMSNorm.
    """
    res = _norm(x, weight, eps, residual, (out,), 0, out_residual)
    return res[0] if residual is None else tuple(res)


def rms_norm_quant(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: torch.Tensor | None = None,
                   group: int = 128, out_q: torch.Tensor | None = None, out_scale: torch.Tensor | None = None,
                   out_residual: torch.Tensor | None = None):
    """:func:`rms_norm` with its output in e4m3: (codes uint8 [..., D], scales
    fp32 [..., groups]) and, with a residual, h.

    group 128: a scale per 128 values (the last group may be short); group 0:
    one per row.  scale = max(amax, 1e-6) / 448; a NaN makes its group's scale
    and codes NaN.  Reference: dsa_layer.py:32-52 and the act_quant before an
    fp8 product (inference/modeling/kernels.py:35-117).
    """
    if group not in (0, 128):
        raise RuntimeError(f"group must be 128 or 0, got {group}")
    return tuple(_norm(x, weight, eps, residual, (out_q, out_scale), group, out_residual))


def rotary(x: torch.Tensor, pos: torch.Tensor, cos_sin: torch.Tensor, interleaved: bool = False, start: int = 0,
           inverse: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """Values start .. start + R - 1 of every head turned by its token's
    position: (a, b) -> (a cos - b sin, b cos + a sin), in fp32.

    x [n, H, D] or [n, D] fp32, bf16 or fp16, any strides but a contiguous last
    dim (a slice of wider heads); pos [n] int32 or int64; cos_sin [positions, R]
    fp32 (``rope.build_rope_table``).  Pairs are i and i + R/2 or, interleaved,
    2i and 2i + 1; inverse turns back (and is the gradient's direction).  out:
    x itself (only the turned values are touched), a tensor that does not
    overlap it (from first element to last: not the gaps between x's heads), or
    None for a new one; the other values are copied then.  A
    token whose position is not in the table (padding, say -1) is not turned.
    Reference: rope.py:25-84 apply_rotary.
    """
    shape, dt, st, pt = x.shape, x.dtype, x.stride(), pos.dtype
    dev = x.get_device()
    _here(dev, pos, cos_sin, out)
    if len(shape) == 3:
        n, H, D = shape
        xn, xh, xd = st
    elif len(shape) == 2:
        (n, D), H = shape, 1
        (xn, xd), xh = st, 0
    else:
        raise RuntimeError(f"x must be [n, H, D] or [n, D], got {tuple(shape)}")
    dtype = _PACK_DTYPES.get(dt)
    if dtype is None:
        raise RuntimeError(f"x must be float32, bfloat16 or float16, got {dt}")
    if pos.shape != (n,) or (pt != torch.int32 and pt != torch.int64) or not pos.is_contiguous():
        raise RuntimeError(f"pos must be contiguous [{n}] int32 or int64, got {pt} {tuple(pos.shape)}")
    table = cos_sin.shape
    if len(table) != 2 or cos_sin.dtype != torch.float32 or not cos_sin.is_contiguous():
        raise RuntimeError("cos_sin must be contiguous [positions, R] float32")
    P, R = table
    if R < 2 or R % 2 or start < 0 or start + R > D or P < 1:
        raise RuntimeError(f"a table of {P} positions and {R} values does not fit values {start} on of {D}")
    if xd != 1 and D > 1:
        raise RuntimeError("x's last dimension must be contiguous")
    xp = x.data_ptr()
    if out is None:
        out = _new(x, shape, dt)
        on, oh = H * D, D
    else:
        if out.shape != shape or out.dtype != dt:
            raise RuntimeError(f"out must be {dt} {tuple(shape)}, got {out.dtype} {tuple(out.shape)}")
        ot = out.stride()
        if ot[-1] != 1 and D > 1:
            raise RuntimeError("out's last dimension must be contiguous")
        on, oh = (ot[0], ot[1]) if len(shape) == 3 else (ot[0], 0)
        # no two heads of out at one place: the larger stride steps over the others
        (small, ns), (large, nl) = ((on, n), (oh, H)) if on < oh else ((oh, H), (on, n))
        if (ns > 1 and small < D) or (nl > 1 and large < (ns - 1) * small + D):
            raise RuntimeError(f"out's heads overlap (strides {ot})")
        if n and H:
            same = out.data_ptr() == xp
            if same and (on, oh) != (xn, xh):
                raise RuntimeError("out is x with other strides")
            _need_apart("out", out, pos, cos_sin, None if same else x)
    if n and H:
        a = _lib.ROTARY_ARGS.pack(xp, pos.data_ptr(), cos_sin.data_ptr(), out.data_ptr(), xn, xh, on, oh, P, n, H, D, R,
                                  start, dtype, 4 if pt == torch.int32 else 8, interleaved, inverse)
        _lib.call("dsa_rotary", a, torch._C._cuda_getCurrentRawStream(dev))
    return out


def append_tokens(page_table: torch.Tensor, rows: torch.Tensor, pos: torch.Tensor,
                  kv_pool: torch.Tensor | None = None, latent: torch.Tensor | None = None,
                  index_k: torch.Tensor | None = None, keys: torch.Tensor | None = None,
                  cos_sin: torch.Tensor | None = None, norm_weight: torch.Tensor | None = None, eps: float = 1e-6,
                  interleaved: bool = False, index_interleaved: bool = False) -> None:
    """New tokens into the paged caches, in one launch: token i belongs to
    request rows[i] at position pos[i], its page in page_table [B, pt_stride]
    int32.

    latent [n, 576] (512 latent | 64 rope): the latent part normed when
    norm_weight [512] is given, the rope part turned when cos_sin [positions, 64]
    is given (:func:`rotary`'s pairs and table), into kv_pool: [rows, 656]
    uint8 (e4m3, a scale per 128) or [rows, 400] (4-bit e2m1, a power-of-two
    scale per 32).  keys [n, 128]: the first 64 turned, into index_k [pages,
    8448].  A NaN makes its 128 values' (4 bits: 32 values') scale NaN, where
    :func:`append_index_keys` and :func:`append_latent_rows` pass it over.  Either
    pair may be left out.  latent and keys are fp32, bf16 or
    fp16, rows any one stride apart; norm_weight of the same type or fp32.  A
    token without a request, page, slot or table row is skipped, in both caches
    where one of them has no place for it; two tokens of one slot must hold the
    same values.
    Reference: sglang overlay P:252-363, P:789; dsa_layer.py:92-143.
    """
    dev = rows.get_device()
    _here(dev, page_table, pos, kv_pool, latent, index_k, keys, cos_sin, norm_weight)
    pts = page_table.shape
    if len(pts) != 2 or 0 in pts or page_table.dtype != torch.int32 or not page_table.is_contiguous():
        raise RuntimeError("page_table must be contiguous [B, pt_stride] int32")
    n = rows.numel()
    if rows.shape != (n,) or rows.dtype != torch.int32 or not rows.is_contiguous():
        raise RuntimeError("rows must be contiguous [n] int32")
    if pos.shape != (n,) or pos.dtype != torch.int32 or not pos.is_contiguous():
        raise RuntimeError(f"pos must be contiguous [{n}] int32")
    if (latent is None) != (kv_pool is None) or (keys is None) != (index_k is None) or (latent is None and keys is None):
        raise RuntimeError("latent goes with kv_pool, keys with index_k, and one of them is needed")
    dt = (keys if latent is None else latent).dtype
    dtype = _PACK_DTYPES.get(dt)
    if dtype is None:
        raise RuntimeError(f"latent and keys must be float32, bfloat16 or float16, got {dt}")
    lp = ls = wp = wt = pp = kv_rows = row_bytes = kp = ks = ip = pages = tp = table_rows = 0
    if latent is not None:
        ls, lp = _append_rows("latent", latent, n, QK_DIM, dt), latent.data_ptr()
        pool = kv_pool.shape
        kv_rows, row_bytes = pool if len(pool) == 2 else (0, 0)
        if (row_bytes != LATENT_ROW_BYTES and row_bytes != FP4_ROW_BYTES) or not kv_rows or kv_pool.dtype != torch.uint8 \
                or not kv_pool.is_contiguous():
            raise RuntimeError("kv_pool must be contiguous [rows, 656] or [rows, 400] uint8")
        pp = kv_pool.data_ptr()
        if norm_weight is not None:
            nt = norm_weight.dtype
            if norm_weight.shape != (LATENT_DIM,) or (nt != dt and nt != torch.float32) or not norm_weight.is_contiguous():
                raise RuntimeError("norm_weight must be [512] of the latent's type or float32")
            wp, wt = norm_weight.data_ptr(), _PACK_DTYPES[nt]
    elif norm_weight is not None:
        raise RuntimeError("norm_weight without a latent")
    if keys is not None:
        ks, kp = _append_rows("keys", keys, n, INDEX_DIM, dt), keys.data_ptr()
        idx = index_k.shape
        if len(idx) != 2 or idx[1] != INDEX_PAGE_BYTES or not idx[0] or index_k.dtype != torch.uint8 \
                or not index_k.is_contiguous():
            raise RuntimeError("index_k must be contiguous [pages, 8448] uint8")
        ip, pages = index_k.data_ptr(), idx[0]
    if cos_sin is not None:
        table = cos_sin.shape
        if len(table) != 2 or table[1] != ROPE_DIM or not table[0] or cos_sin.dtype != torch.float32 \
                or not cos_sin.is_contiguous():
            raise RuntimeError("cos_sin must be contiguous [positions, 64] float32")
        tp, table_rows = cos_sin.data_ptr(), table[0]
    a = _lib.APPEND_ARGS.pack(rows.data_ptr(), pos.data_ptr(), page_table.data_ptr(), tp, lp, wp, pp, kp, ip, table_rows,
                              ls, kv_rows, ks, pages, eps, n, pts[0], pts[1], dtype, wt, row_bytes, interleaved,
                              index_interleaved)
    _lib.call("dsa_append_tokens", a, torch._C._cuda_getCurrentRawStream(dev))


def _append_rows(name: str, x: torch.Tensor, n: int, width: int, dtype) -> int:
    """The row stride of an append's input."""
    st = x.stride()
    if x.shape != (n, width) or x.dtype != dtype or st[1] != 1:
        raise RuntimeError(f"{name} must be {dtype} [{n}, {width}] with a contiguous last dimension, got {x.dtype} "
                           f"{tuple(x.shape)}")
    return st[0]


def read_latent_rows(kv_pool: torch.Tensor, slots: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """The values of cached latent rows, bf16 [n, 576] (512 latent | 64 rope):
    what the attention reads of KV slots slots [n] int32 of a pool of 656- or
    400-byte rows.  With them the prefill ops attend a cached prefix.  A slot
    outside the pool gives zeros.  Reference: P:789 dequantize_k_cache.
    """
    dev = kv_pool.get_device()
    _here(dev, slots, out)
    pool = kv_pool.shape
    kv_rows, row_bytes = pool if len(pool) == 2 else (0, 0)
    if (row_bytes != LATENT_ROW_BYTES and row_bytes != FP4_ROW_BYTES) or not kv_rows or kv_pool.dtype != torch.uint8 \
            or not kv_pool.is_contiguous():
        raise RuntimeError("kv_pool must be contiguous [rows, 656] or [rows, 400] uint8")
    n = slots.numel()
    if slots.shape != (n,) or slots.dtype != torch.int32 or not slots.is_contiguous():
        raise RuntimeError("slots must be contiguous [n] int32")
    if out is None:
        out = torch.empty(n, QK_DIM, dtype=torch.bfloat16, device=kv_pool.device)
    else:
        _need_shape("out", out, (n, QK_DIM), torch.bfloat16)
    _lib.call("dsa_read_latent_rows", kv_pool.data_ptr(), kv_rows, row_bytes, slots.data_ptr(), n, out.data_ptr(),
              torch._C._cuda_getCurrentRawStream(dev))
    return out


# ---- 8-bit products: row quantiser, products with block scales ----

def quantize_rows(x: torch.Tensor, gate: torch.Tensor | None = None, group: int = 128,
                  out_q: torch.Tensor | None = None, out_scale: torch.Tensor | None = None):
    """x, or x * silu(gate), in e4m3: (codes uint8 [..., D], scales fp32
    [..., groups]), by :func:`rms_norm_quant`'s rule.

    x [..., D] fp32, bf16 or fp16 (rows any one stride apart, D up to 32768),
    gate of the same shape and type (the two halves of one projection).  group
    128: a scale per 128 values (the last group may be short); group 0: one per
    row.  scale = max(amax, 1e-6) / 448; a NaN makes its group's scale and codes
    NaN.  Outputs must not overlap inputs.
    Reference: inference/modeling/kernels.py:35-117.
    """
    if group not in (0, 128):
        raise RuntimeError(f"group must be 128 or 0, got {group}")
    shape, dt = x.shape, x.dtype
    dtype = _PACK_DTYPES.get(dt)
    if dtype is None:
        raise RuntimeError(f"x must be float32, bfloat16 or float16, got {dt}")
    dev = x.get_device()
    D = shape[-1] if shape else 0
    if not 1 <= D <= NORM_MAX_DIM:
        raise RuntimeError(f"x must be [..., D] with D from 1 to {NORM_MAX_DIM}, got {tuple(shape)}")
    _here(dev, gate, out_q, out_scale)
    n = x.numel() // D
    xs, gs, gp = _row_stride("x", x, n, D), 0, 0
    if gate is not None:
        if gate.dtype != dt or gate.shape != shape:
            raise RuntimeError(f"gate must be {dt} {tuple(shape)}, got {gate.dtype} {tuple(gate.shape)}")
        gs, gp = _row_stride("gate", gate, n, D), gate.data_ptr()
    sshape = (*shape[:-1], -(-D // 128) if group else 1)
    if out_q is None:
        out_q = torch.empty(shape, dtype=torch.uint8, device=x.device)
    else:
        _need_shape("out_q", out_q, shape, torch.uint8)
        if n:
            _need_apart("out_q", out_q, x, gate)
    if out_scale is None:
        out_scale = torch.empty(sshape, dtype=torch.float32, device=x.device)
    else:
        _need_shape("out_scale", out_scale, sshape, torch.float32)
        if n:
            _need_apart("out_scale", out_scale, x, gate, out_q)
    if n:
        a = _lib.QUANT_ARGS.pack(x.data_ptr(), gp, out_q.data_ptr(), out_scale.data_ptr(), xs, gs, n, D, dtype, group)
        _lib.call("dsa_quantize_rows", a, torch._C._cuda_getCurrentRawStream(dev))
    return out_q, out_scale


def _matmul(a, a_scale, w, w_scale, offsets, dtype, out):
    """Checks and launch of a product; w [experts, N, K] or [N, K]."""
    for name, t in (("a", a), ("w", w)):
        if t.dtype != torch.uint8 and t.dtype != torch.float8_e4m3fn:
            raise RuntimeError(f"{name} must hold e4m3 codes (uint8 or float8_e4m3fn), got {t.dtype}")
        if not t.is_contiguous():
            raise RuntimeError(f"{name} must be contiguous")
    dev = a.get_device()
    _here(dev, a_scale, w, w_scale, offsets, out)
    ash, wsh = a.shape, w.shape
    if len(wsh) != (2 if offsets is None else 3) or not ash or ash[-1] != wsh[-1]:
        raise RuntimeError(f"a must be [..., K] and w {'[N, K]' if offsets is None else '[experts, N, K]'}, got "
                           f"{tuple(ash)} and {tuple(wsh)}")
    K, N = wsh[-1], wsh[-2]
    if not 16 <= K <= MATMUL_MAX_K or K % 16:
        raise RuntimeError(f"K must be a multiple of 16 up to {MATMUL_MAX_K}, got {K}")
    n = a.numel() // K
    groups = -(-K // 128)
    ss = a_scale.shape
    if a_scale.dtype != torch.float32 or not a_scale.is_contiguous() or ss[:-1] != ash[:-1] or len(ss) != len(ash) or \
            ss[-1] not in (1, groups):
        raise RuntimeError(f"a_scale must be contiguous float32 {(*ash[:-1], groups)}, or 1 a row, got {a_scale.dtype} "
                           f"{tuple(ss)}")
    _need_shape("w_scale", w_scale, (*wsh[:-2], -(-N // 128), groups), torch.float32)
    experts = 1
    if offsets is not None:
        experts = wsh[0]
        _need_shape("offsets", offsets, (experts + 1,), torch.int32)
    if out is None:
        if dtype not in _PACK_DTYPES:
            raise RuntimeError(f"the output must be float32, bfloat16 or float16, got {dtype}")
        out = torch.empty(*ash[:-1], N, dtype=dtype, device=a.device)
    else:
        dtype = out.dtype
        if dtype not in _PACK_DTYPES:
            raise RuntimeError(f"out must be float32, bfloat16 or float16, got {dtype}")
        _need_shape("out", out, (*ash[:-1], N), dtype)
        if n and N:
            _need_apart("out", out, a, a_scale, w if w.numel() else None, w_scale if w.numel() else None, offsets)
    if n and N and experts:
        p = _lib.MATMUL_ARGS.pack(a.data_ptr(), a_scale.data_ptr(), w.data_ptr(), w_scale.data_ptr(),
                                  0 if offsets is None else offsets.data_ptr(), out.data_ptr(), n, N, K, experts, ss[-1],
                                  _PACK_DTYPES[dtype])
        _lib.call("dsa_fp8_matmul", p, torch._C._cuda_getCurrentRawStream(dev))
    return out


def fp8_matmul(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
               dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rows a [..., K] times weights w [N, K]^T, both e4m3 codes, summed in fp32
    -> [..., N] of ``dtype`` (fp32, bf16 or fp16), or of out's type.

    a_scale [..., ceil(K/128)] fp32, or [..., 1] for one scale a row: what
    :func:`rms_norm_quant` and :func:`quantize_rows` give; w_scale [ceil(N/128),
    ceil(K/128)] fp32, a scale per 128 x 128 block (``formats.quantize_weight``).
    K a multiple of 16; everything contiguous.  Which kernel runs, and the order
    of its sum, depends on the number of rows: a row alone and among others may
    differ in the last bits.
    Reference: inference/modeling/kernels.py:120-221.
    """
    return _matmul(a, a_scale, w, w_scale, None, dtype, out)


def fp8_matmul_grouped(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
                       offsets: torch.Tensor, dtype: torch.dtype = torch.bfloat16,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`fp8_matmul` with the weights of experts: rows offsets[e] ..
    offsets[e + 1] - 1 of a [n, K] times w[e] of w [experts, N, K].

    offsets [experts + 1] int32 on the device, not falling, from 0 or later to
    at most n; w_scale [experts, ceil(N/128), ceil(K/128)].  An expert may have
    no row; rows outside all of them are left as they are (new outputs: undefined).
    """
    if a.dim() != 2:
        raise RuntimeError(f"a must be [n, K], got {tuple(a.shape)}")
    if offsets is None:
        raise RuntimeError("offsets are needed")
    return _matmul(a, a_scale, w, w_scale, offsets, dtype, out)


# ---- a chunk of new tokens over the paged caches ----

def _chunk(page_table, q_start, seq_lens) -> int:
    """What the chunk ops check of their requests; returns how many there are."""
    pts = page_table.shape
    if len(pts) != 2 or 0 in pts or page_table.dtype != torch.int32 or not page_table.is_contiguous():
        raise RuntimeError("page_table must be contiguous [B, pt_stride] int32")
    B = pts[0]
    _need_shape("q_start", q_start, (B + 1,), torch.int32)
    _need_shape("seq_lens", seq_lens, (B,), torch.int32)
    return B


def chunk_scan(q_fp8: torch.Tensor, w: torch.Tensor, index_k: torch.Tensor, page_table: torch.Tensor,
               q_start: torch.Tensor, seq_lens: torch.Tensor, slab_stride: int,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`indexer_scan` for more than one row a request: rows q_start[b] ..
    q_start[b + 1] - 1 are the last tokens of request b, whose index keys (theirs
    too) are the first seq_lens[b] of the paged cache; a row's scores end at its
    own position.

    q_fp8 [n,Hidx,128] e4m3 codes; w [n,Hidx] f32 (q-scale folded in); index_k
    [P,8448] uint8; page_table [B,pt] int32; q_start [B+1] int32, not falling;
    seq_lens [B] int32  ->  scores [n, slab_stride] f32 (-inf behind the row's
    position, and all of them for a row before position 0).  Rows of no request
    are left as they are (new scores: undefined).
    Reference: attention_core.py:27-63 indexer_logits, apply_causal_mask.
    """
    q_fp8 = q_fp8.view(torch.uint8) if q_fp8.dtype == torch.float8_e4m3fn else q_fp8
    _here(q_fp8.get_device(), w, index_k, page_table, q_start, seq_lens, out)
    qs = q_fp8.shape
    if len(qs) != 3 or qs[2] != INDEX_DIM or q_fp8.dtype != torch.uint8 or not q_fp8.is_contiguous():
        raise RuntimeError("q_fp8 must be contiguous [n, Hidx, 128] e4m3 bytes")
    n, Hidx, _ = qs
    _need_shape("w", w, (n, Hidx), torch.float32)
    ks = index_k.shape
    if len(ks) != 2 or ks[1] != INDEX_PAGE_BYTES or index_k.dtype != torch.uint8 or not index_k.is_contiguous():
        raise RuntimeError("index_k must be contiguous [pages, 8448] uint8")
    B = _chunk(page_table, q_start, seq_lens)
    if out is None:
        out = torch.empty(n, slab_stride, dtype=torch.float32, device=q_fp8.device)
    else:
        _need_shape("out", out, (n, slab_stride), torch.float32)
        if n:
            _need_apart("out", out, q_fp8, w, index_k, page_table, q_start, seq_lens)
    if n:
        _lib.call("dsa_chunk_scan", q_fp8.data_ptr(), w.data_ptr(), index_k.data_ptr(), ks[0], page_table.data_ptr(),
                  q_start.data_ptr(), seq_lens.data_ptr(), out.data_ptr(), n, B, Hidx, page_table.shape[1], slab_stride,
                  _stream())
    return out


def chunk_workspace(n: int, H: int, device) -> torch.Tensor:
    """Workspace of :func:`chunk_attention` calls of up to n rows of up to H
    heads (no initialisation needed; at most 135 MB)."""
    nbytes = _lib.load().dsa_chunk_attention_workspace_bytes(n, H)
    if nbytes == 0:
        raise RuntimeError(f"bad chunk attention shape n={n} H={H}")
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def chunk_attention(q: torch.Tensor, kv_pool: torch.Tensor, page_table: torch.Tensor, q_start: torch.Tensor,
                    seq_lens: torch.Tensor, sm_scale: float | None = None, workspace: torch.Tensor | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`dense_mla_decode` for more than one row a request: rows q_start[b]
    .. q_start[b + 1] - 1 are the last tokens of request b, whose latent rows
    (theirs too) are the first seq_lens[b] of the paged cache; each attends the
    tokens up to its own.

    q [n,H,576] bf16; kv_pool [rows,656] or [rows,400] uint8; page_table [B,pt]
    int32; q_start [B+1] int32, not falling; seq_lens [B] int32  ->  out
    [n,H,512] bf16 (0 for a row before position 0).  Rows of no request are left
    as they are (a new out: undefined).  Probabilities are rounded to bf16;
    latent values below 2^-56, which no packer here writes, lose bits.  workspace:
    :func:`chunk_workspace` of at least this n and H; calls that overlap in time
    must not share one.  For a sparse layer's chunk each row is a row of
    :func:`sparse_mla_decode`.
    Reference: attention_core.py:142-160 dense_mla_core.
    """
    qs, ps = q.shape, kv_pool.shape
    dev = q.get_device()
    _here(dev, kv_pool, page_table, q_start, seq_lens, workspace, out)
    if len(qs) != 3 or qs[2] != QK_DIM or q.dtype != torch.bfloat16 or not q.is_contiguous():
        raise RuntimeError("q must be contiguous [n, H, 576] bfloat16")
    n, H, _ = qs
    if len(ps) != 2 or (ps[1] != LATENT_ROW_BYTES and ps[1] != FP4_ROW_BYTES) or not ps[0] or \
            kv_pool.dtype != torch.uint8 or not kv_pool.is_contiguous():
        raise RuntimeError("kv_pool must be contiguous [rows, 656] or [rows, 400] uint8")
    B = _chunk(page_table, q_start, seq_lens)
    if out is None:
        out = torch.empty(n, H, LATENT_DIM, dtype=torch.bfloat16, device=q.device)
    else:
        _need_shape("out", out, (n, H, LATENT_DIM), torch.bfloat16)
        if n:
            _need_apart("out", out, q, kv_pool, page_table, q_start, seq_lens, workspace)
    if n:
        if workspace is None:
            workspace = chunk_workspace(n, H, q.device)
        else:
            if not workspace.is_contiguous():
                raise RuntimeError("the chunk attention workspace must be contiguous")
            _need_bytes("chunk attention workspace", workspace, _lib.load().dsa_chunk_attention_workspace_bytes(n, H))
        _lib.call("dsa_chunk_attention", q.data_ptr(), kv_pool.data_ptr(), ps[0], ps[1], page_table.data_ptr(),
                  q_start.data_ptr(), seq_lens.data_ptr(), workspace.data_ptr(), out.data_ptr(), n, B, H,
                  page_table.shape[1], QK_DIM ** -0.5 if sm_scale is None else float(sm_scale),
                  torch._C._cuda_getCurrentRawStream(dev))
    return out
