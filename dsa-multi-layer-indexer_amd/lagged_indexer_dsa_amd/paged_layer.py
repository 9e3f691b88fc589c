"""Decode-time adapter of a ``DSALayer``: persistent paged fp8 caches and the
fused layer launch.

The reference's ``DSALayer.fused_attention_and_indices`` (dsa_layer.py:173-192)
recomputes the whole key set on every call.  At decode time the keys of the
prefix never change, so :class:`PagedDSALayer` keeps them where the serving
path keeps them -- the paged index-K cache and the 656-byte fp8 latent pool
of one layer -- appends each new token once (the HIP quantizers of
``ops.append_index_keys`` / ``ops.append_latent_rows``), and answers a decode
row with ONE ``dsa_decode_layer`` launch: the attention over the given
(lagged) selection and this layer's indexer scan and top-k side by side.

It wraps any module with the reference layer's projection methods
(``q_latent``, ``_mla_qkv``, ``_indexer_qkw``, ``_project_output`` and a
``config`` with ``index_topk``); the projections stay in torch, outside the
timed hot path.  Shapes the kernels accept: kv_lora_rank 512, rope 64
(576-wide absorbed queries), index_head_dim 128, index_n_heads 16/32/48/64,
attention heads a multiple of 16.

With ``kv_bits=4`` the latent pool holds 400-byte rows (39 % less cache); the
latent rows of new tokens are then stored by ``ops.append_tokens``, the index
keys as with 8 bits (the selections do not depend on kv_bits, for keys with a
NaN either), and the attention is a launch of its own ahead of the layer's scan
and top-k.

A chunk of new tokens (a part of a prompt after a cached prefix, or drafted
tokens) goes through ``chunk_attention_and_indices``: appended together, then
the dense attention of ``ops.chunk_attention`` or the rows' selections by
``ops.sparse_mla_decode``, and the indexer's scores by ``ops.chunk_scan`` with
one select over all rows.

Index convention: selections cross this API as token positions, int64
``[B, 1, topk]`` like ``select_topk`` returns them, with the sentinel
``S_kv`` (the row length) for unused entries.  They come back in ascending
position order -- the decode kernels' order -- where ``select_topk`` orders by
score; both are the same set, which is all ``sparse_mla_core`` reads.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib, ops
from ._lib import INDEX_DIM, LATENT_DIM, PAGE_TOKENS, QK_DIM, LayerArgs
from .formats import new_latent_pool

# What a chunk's sparse attention and selection take at a time: the rows of the
# decode and select launches, and scores in memory (2^28: 1 GiB).  A longer chunk
# goes through in several.
MAX_ROWS = 65535
MAX_SCORES = 1 << 28


class PagedDSALayer:
    """Paged caches of one layer for ``batch`` rows of up to ``max_ctx``
    tokens each (identity paging: row b owns pages [b*npg, (b+1)*npg))."""

    def __init__(self, layer, batch: int, max_ctx: int, device=None, nsplit: int = 0,
                 kv_bits: int = 8) -> None:
        cfg = layer.config
        if cfg.kv_lora_rank + cfg.qk_rope_head_dim != QK_DIM or cfg.kv_lora_rank != LATENT_DIM:
            raise ValueError("the fp8 latent format needs kv_lora_rank 512 and qk_rope_head_dim 64")
        if cfg.index_head_dim != INDEX_DIM or cfg.index_n_heads not in (16, 32, 48, 64):
            raise ValueError("the fp8 indexer needs index_head_dim 128 and 16/32/48/64 index heads")
        if cfg.num_attention_heads % 16:
            raise ValueError("the attention heads must be a multiple of 16")
        dev = torch.device(device) if device is not None else next(layer.parameters()).device
        self.layer, self.B, self.topk = layer, int(batch), int(cfg.index_topk)
        self.H, self.Hidx = cfg.num_attention_heads, cfg.index_n_heads
        self.npg = max(1, -(-int(max_ctx) // PAGE_TOKENS))
        self.cap = self.npg * PAGE_TOKENS
        B = self.B
        self.page_table = (torch.arange(B, dtype=torch.int32, device=dev)[:, None] * self.npg
                           + torch.arange(self.npg, dtype=torch.int32, device=dev)[None, :]).contiguous()
        self.index_k = torch.zeros(B * self.npg, _lib.INDEX_PAGE_BYTES, dtype=torch.uint8, device=dev)
        self.kv_bits = int(kv_bits)
        self.kv_pool = new_latent_pool(B * self.npg, dev, self.kv_bits)
        self.seq_lens = torch.zeros(B, dtype=torch.int32, device=dev)
        self.length = 0
        self.scores = torch.empty(B, self.cap, dtype=torch.float32, device=dev)
        self.topk_scratch = ops.topk_scratch(B, self.cap, dev)
        self.next_idx = torch.full((B, self.topk), -1, dtype=torch.int32, device=dev)
        self.attend = torch.full((B, self.topk), -1, dtype=torch.int32, device=dev)
        self.nsplit = int(nsplit)
        self.workspace = ops.sparse_mla_workspace(B, self.H, self.nsplit, dev, kv_bits=self.kv_bits)
        self.out = torch.zeros(B, self.H, LATENT_DIM, dtype=torch.bfloat16, device=dev)
        self.q_fp8 = torch.empty(B, self.Hidx, INDEX_DIM, dtype=torch.uint8, device=dev)
        self.w = torch.empty(B, self.Hidx, dtype=torch.float32, device=dev)
        self._rows = torch.arange(B, dtype=torch.int32, device=dev)
        self._base = (torch.arange(B, dtype=torch.int64, device=dev) * self.cap)[:, None]
        self._starts = torch.arange(B + 1, dtype=torch.int32, device=dev)

    # ---- cache maintenance ----
    def _append(self, index_k: torch.Tensor, kv: torch.Tensor) -> None:
        """Store keys [B,S,128] and latent rows [B,S,576] of the next S tokens."""
        B, S = kv.shape[0], kv.shape[1]
        if self.length + S > self.cap:
            raise ValueError(f"context {self.length + S} above the cache's {self.cap} tokens")
        pos = torch.arange(self.length, self.length + S, dtype=torch.int32, device=kv.device)
        rows = self._rows.repeat_interleave(S)
        posb = pos.repeat(B)
        keys = index_k.reshape(B * S, INDEX_DIM).to(torch.bfloat16).contiguous()
        latent = kv.reshape(B * S, QK_DIM).to(torch.bfloat16).contiguous()
        # (append_tokens has another rule for a key with a NaN: its scale is NaN)
        ops.append_index_keys(self.index_k, self.page_table, rows, posb, keys)
        if self.kv_bits == 4:
            ops.append_tokens(self.page_table, rows, posb, kv_pool=self.kv_pool, latent=latent)
        else:
            slots = (rows.long() * self.cap + posb.long()).to(torch.int32)
            ops.append_latent_rows(self.kv_pool, slots, latent)
        self.length += S
        self.seq_lens.fill_(self.length)

    def append(self, x_norm: torch.Tensor, rope) -> None:
        """Project and store the keys of S new tokens ([B, S, hidden], rope
        caches for their positions) without attending (prompt prefill)."""
        c_q = self.layer.q_latent(x_norm)
        _, kv = self.layer._mla_qkv(x_norm, c_q, rope)
        _, index_k, _ = self.layer._indexer_qkw(x_norm, c_q, rope)
        self._append(index_k, kv)

    # ---- index conventions ----
    def _to_slots(self, indices: torch.Tensor) -> torch.Tensor:
        """[B,1,topk] positions (sentinel / negatives unused) -> int32 KV slots."""
        idx = indices.reshape(self.B, -1).long()
        if idx.shape[1] != self.topk:
            raise ValueError(f"indices must be [B, 1, {self.topk}], got {tuple(indices.shape)}")
        ok = (idx >= 0) & (idx < self.length)
        return torch.where(ok, idx + self._base, torch.full_like(idx, -1)).to(torch.int32)

    def _to_positions(self, slots: torch.Tensor) -> torch.Tensor:
        s = slots.long()
        return torch.where(s >= 0, s - self._base, torch.full_like(s, self.length)).reshape(self.B, 1, self.topk)

    # ---- the decode row ----
    def fused_attention_and_indices(self, x_norm: torch.Tensor, rope, attn_indices: torch.Tensor | None,
                                    produce_indexer: bool = True):
        """The decode row at position ``length`` ([B, 1, hidden], rope caches
        for that position): its key and latent row are appended first (a row
        attends itself), then one launch attends ``attn_indices`` (dense when
        None) and, if asked, runs this layer's indexer.  Returns (attention
        hidden output [B, 1, hidden], next indices [B, 1, topk] or None)
        (dsa_layer.py:173-192)."""
        if x_norm.dim() != 3 or x_norm.shape[:2] != (self.B, 1):
            raise ValueError(f"x_norm must be [{self.B}, 1, hidden] (one decode row per request)")
        lay = self.layer
        c_q = lay.q_latent(x_norm)
        q, kv = lay._mla_qkv(x_norm, c_q, rope)
        index_q = index_k = weights = None
        if produce_indexer:
            index_q, index_k, weights = lay._indexer_qkw(x_norm, c_q, rope)
        else:
            _, index_k, _ = lay._indexer_qkw(x_norm, c_q, rope)
        self._append(index_k, kv)
        q_bf16 = q.reshape(self.B, self.H, QK_DIM).to(torch.bfloat16).contiguous()
        if produce_indexer:
            ops.quantize_index_query(index_q.reshape(self.B, self.Hidx, INDEX_DIM).to(torch.bfloat16).contiguous(),
                                     weights.reshape(self.B, self.Hidx).float().contiguous(),
                                     out_q=self.q_fp8, out_w=self.w)
        a = LayerArgs()
        if produce_indexer:
            a.q_fp8, a.w = self.q_fp8.data_ptr(), self.w.data_ptr()
            a.index_k, a.num_idx_pages = self.index_k.data_ptr(), self.index_k.shape[0]
            a.Hidx = self.Hidx
        a.scores, a.topk_scratch, a.next_idx = (self.scores.data_ptr(), self.topk_scratch.data_ptr(),
                                                self.next_idx.data_ptr())
        if attn_indices is not None:
            self.attend.copy_(self._to_slots(attn_indices))
        if self.kv_bits == 4:
            if attn_indices is None:
                ops.dense_mla_decode(q_bf16, self.kv_pool, self.page_table, self.seq_lens, nsplit=self.nsplit,
                                     workspace=self.workspace, out=self.out)
            else:
                ops.sparse_mla_decode(q_bf16, self.kv_pool, self.attend, nsplit=self.nsplit, workspace=self.workspace,
                                      out=self.out)
        else:
            a.q_bf16, a.kv_pool, a.kv_rows = q_bf16.data_ptr(), self.kv_pool.data_ptr(), self.kv_pool.shape[0]
            a.workspace, a.out_bf16 = self.workspace.data_ptr(), self.out.data_ptr()
            if attn_indices is None:
                a.dense = 1
            else:
                a.attend_idx = self.attend.data_ptr()
        a.page_table, a.seq_lens = self.page_table.data_ptr(), self.seq_lens.data_ptr()
        a.B, a.H, a.topk, a.nsplit = self.B, self.H, self.topk, self.nsplit
        a.pt_stride, a.slab_stride = self.npg, self.cap
        a.sm_scale = QK_DIM ** -0.5
        if produce_indexer or self.kv_bits == 8:
            _lib.call("dsa_decode_layer", ctypes.byref(a), torch.cuda.current_stream().cuda_stream)
        o_latent = self.out.float().reshape(self.B, 1, self.H, LATENT_DIM).to(x_norm.dtype)
        hidden = lay._project_output(o_latent)
        nxt = self._to_positions(self.next_idx) if produce_indexer else None
        return hidden, nxt

    # ---- a chunk of rows ----
    def chunk_attention_and_indices(self, x_norm: torch.Tensor, rope, attn_indices: torch.Tensor | None,
                                    produce_indexer: bool = True):
        """The S rows at positions ``length`` .. ``length + S - 1`` ([B, S,
        hidden], rope caches for those positions): their keys and latent rows are
        appended first, then each row attends ``attn_indices`` [B, S, topk] (those
        up to its own position) or, when None, every token up to its own, and, if
        asked, this layer's indexer selects among the same tokens.  Returns
        (attention hidden output [B, S, hidden], next indices [B, S, topk] or
        None) (dsa_layer.py:145-192 over a cached prefix)."""
        if x_norm.dim() != 3 or x_norm.shape[0] != self.B or x_norm.shape[1] < 1:
            raise ValueError(f"x_norm must be [{self.B}, S, hidden], got {tuple(x_norm.shape)}")
        S = x_norm.shape[1]
        n = self.B * S
        if attn_indices is not None and attn_indices.shape != (self.B, S, self.topk):
            raise ValueError(f"indices must be [{self.B}, {S}, {self.topk}], got {tuple(attn_indices.shape)}")
        lay = self.layer
        c_q = lay.q_latent(x_norm)
        q, kv = lay._mla_qkv(x_norm, c_q, rope)
        index_q, index_k, weights = lay._indexer_qkw(x_norm, c_q, rope)
        pos = torch.arange(self.length, self.length + S, device=x_norm.device)
        self._append(index_k, kv)
        q_bf16 = q.reshape(n, self.H, QK_DIM).to(torch.bfloat16).contiguous()
        if attn_indices is None:
            out = ops.chunk_attention(q_bf16, self.kv_pool, self.page_table, self._starts * S, self.seq_lens)
        else:
            idx = attn_indices.long()
            seen = (idx >= 0) & (idx <= pos[None, :, None])
            slots = torch.where(seen, idx + self._base[:, None], torch.full_like(idx, -1))
            slots = slots.reshape(n, self.topk).to(torch.int32)
            out = torch.empty(n, self.H, LATENT_DIM, dtype=torch.bfloat16, device=q_bf16.device)
            for i in range(0, n, MAX_ROWS):
                ops.sparse_mla_decode(q_bf16[i:i + MAX_ROWS], self.kv_pool, slots[i:i + MAX_ROWS], out=out[i:i + MAX_ROWS])
        hidden = lay._project_output(out.float().reshape(self.B, S, self.H, LATENT_DIM).to(x_norm.dtype))
        if not produce_indexer:
            return hidden, None
        q_fp8, w = ops.quantize_index_query(index_q.reshape(n, self.Hidx, INDEX_DIM).to(torch.bfloat16).contiguous(),
                                            weights.reshape(n, self.Hidx).float().contiguous())
        q_fp8, w = q_fp8.reshape(self.B, S, self.Hidx, INDEX_DIM), w.reshape(self.B, S, self.Hidx)
        slab = max(-(-self.length // PAGE_TOKENS) * PAGE_TOKENS, self.topk)
        step = max(1, min(MAX_ROWS, MAX_SCORES // slab) // self.B)  # tokens of each request at a time
        if step >= S:
            return hidden, self._select_chunk(q_fp8, w, self.seq_lens, slab)
        return hidden, torch.cat([self._select_chunk(q_fp8[:, i:i + step].contiguous(), w[:, i:i + step].contiguous(),
                                                     self.seq_lens - max(0, S - i - step), slab)
                                  for i in range(0, S, step)], dim=1)

    def _select_chunk(self, q_fp8: torch.Tensor, w: torch.Tensor, seq_lens: torch.Tensor, slab: int) -> torch.Tensor:
        """Selections [B, s, topk] of the queries [B, s, Hidx, 128], each
        request's the last of its first seq_lens[b] tokens."""
        s = q_fp8.shape[1]
        n = self.B * s
        scores = ops.chunk_scan(q_fp8.reshape(n, self.Hidx, INDEX_DIM), w.reshape(n, self.Hidx), self.index_k,
                                self.page_table, self._starts * s, seq_lens, slab)
        # the scores behind a row's position are -inf, which the select pads
        nxt = ops.select_rows(scores, self.topk, self.length)
        if nxt is None:
            lens = torch.full((n,), slab, dtype=torch.int32, device=scores.device)
            nxt = ops.topk(scores, lens, self.topk, pad_value=self.length).long()
        return nxt.reshape(self.B, s, self.topk).sort(dim=-1)[0]  # ascending, the sentinel behind
