"""Latent attention: a paged cache whose keys and values are one shared row a
token (a latent and a rotated key), absorbed attention over it for new tokens,
and expanded attention for prompt chunks.  The reference's caches are per head
(src/inference/forward.rs:16-19); it has no counterpart."""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from ._lib import BF16, call, check, lib
from .kv import _check, _grad_on, _ID_TORCH, _on, _Pages, _raw_stream, _refuse_gradient, _written, Rotary, torch_dtype_id

__all__ = ["LatentKvCache", "latent_prefill"]


def _heads(t: torch.Tensor, name: str, index: int, n: int, heads: int, dim: int) -> Tuple[int, int, int]:
    """Address and token and head strides of a [n, heads, dim] tensor on device
    `index` whose rows are each contiguous."""
    if t.shape != (n, heads, dim):
        raise ValueError(f"{name} must be [{n}, {heads}, {dim}], not {list(t.shape)}")
    if t.get_device() != index:
        raise ValueError(f"{name}: tensor on cuda:{index} expected")
    token, head, element = t.stride()
    if element != 1 and dim != 1 and t.numel():
        raise ValueError(f"{name}: rows must be contiguous")
    return t.data_ptr(), token, head


class LatentKvCache(_Pages):
    """A paged cache of latent rows (it_kv_cache_wrap_latent), [num_blocks]
    pages of block_size rows of latent_dim + rope_dim elements (F32, F16 or
    BF16): the latent that all heads' keys and values are projected from, then
    the rotated key that all heads share.

    n_layers > 1 holds every layer of a model, as PagedKvCache does: evict /
    copy_blocks / move / sync_tables act on the whole cache; append, gather and
    decode go through `layer(l)`."""

    _LAYER_FIELDS = _Pages._LAYER_FIELDS + ("latent_dim", "rope_dim")

    def __init__(self, num_blocks: int, block_size: int, latent_dim: int, rope_dim: int, dtype: int = BF16, device: int = 0,
                 n_layers: int = 1):
        page = lib.it_kv_page_bytes(block_size, latent_dim + rope_dim, dtype)
        if page <= 0 or dtype not in _ID_TORCH:
            raise ValueError("unsupported cache shape")
        dev = torch.device("cuda", device)
        self.k_pool = torch.zeros(n_layers * num_blocks * page, dtype=torch.uint8, device=dev)
        self.v_pool = None
        h = C.c_void_p()
        check(lib.it_kv_cache_wrap_latent(device, n_layers, self.k_pool.data_ptr(), num_blocks, block_size, latent_dim, rope_dim,
                                          dtype, C.byref(h)))
        self._adopt(h, device)
        self.num_blocks, self.block_size, self.n_kv_heads = num_blocks, block_size, 1
        self.latent_dim, self.rope_dim, self.head_dim = latent_dim, rope_dim, latent_dim + rope_dim
        self.dtype = dtype
        self.page_bytes = page
        self.device = dev
        self.n_layers = n_layers
        self._parent = None

    def view(self) -> torch.Tensor:
        """Typed view [num_blocks, block_size, latent_dim + rope_dim] of a layer."""
        self._one_layer()
        return self.k_pool.view(_ID_TORCH[self.dtype]).view(self.num_blocks, self.block_size, self.head_dim)

    # ---- data movement ----------------------------------------------------
    def append(self, kv: torch.Tensor, slot_mapping: torch.Tensor, rotary: Optional[Rotary] = None,
               positions: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
               q_rope: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None,
               q_out_dtype: Optional[torch.dtype] = None, rows_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """Latent rows into their slots (it_latent_append): kv [n_tokens,
        latent_dim + rope_dim] (rows contiguous, any token stride), its latent
        part normalised by its root mean square and multiplied by weight
        [latent_dim] (None: as it is), its rope part turned to int32 positions
        by rotary (None: as it is).  q_rope [n_tokens, n_heads, rope_dim] (any
        token and head strides: the rope part of the heads' projection) is
        turned with it: returned as q_out (q_rope itself is allowed, inside a
        projection that holds kv too), or a new tensor of q's dtype or
        q_out_dtype.  rows_out [n_tokens, latent_dim + rope_dim] of the cache's
        dtype gets the stored rows too.  Carries no gradient: tensors that
        require one are refused, unless gradients are off."""
        if _grad_on() and (kv.requires_grad or (weight is not None and weight.requires_grad) or
                           (q_rope is not None and q_rope.requires_grad) or (q_out is not None and q_out.requires_grad) or
                           (rows_out is not None and rows_out.requires_grad)):
            _refuse_gradient("append")
        if slot_mapping.dtype != torch.int64:
            raise TypeError("slot_mapping must be int64")
        n, index = slot_mapping.numel(), self._index
        if kv.shape != (n, self.head_dim):
            raise ValueError(f"kv must be [n_tokens, {self.head_dim}], with a slot per token")
        if kv.get_device() != index:
            raise ValueError(f"kv: tensor on cuda:{index} expected")
        token, element = kv.stride()
        if element != 1 and kv.numel():
            raise ValueError("kv: rows must be contiguous")
        if (rotary is None) != (positions is None):
            raise TypeError("rotary and positions go together")
        pa = wa = qa = oa = ra = given = None
        qs = qh = os = oh = heads = out_id = weight_id = 0
        if positions is not None:
            if positions.dtype != torch.int32 or positions.numel() != n:
                raise TypeError("positions must be int32, one per token")
            pa = _on(positions, index)
        if weight is not None:
            if weight.numel() != self.latent_dim:
                raise ValueError("weight must be [latent_dim]")
            wa, weight_id = _on(weight, index), torch_dtype_id(weight.dtype)
        if q_rope is not None:
            if q_rope.dtype != kv.dtype:
                raise TypeError("q_rope and kv must have one dtype")
            heads = q_rope.shape[1] if q_rope.dim() == 3 else 0
            qa, qs, qh = _heads(q_rope, "q_rope", index, n, heads, self.rope_dim)
            given = q_out
            if q_out is None:
                q_out = torch.empty((n, heads, self.rope_dim), dtype=q_out_dtype or q_rope.dtype, device=self.device)
            oa, os, oh = _heads(q_out, "q_out", index, n, heads, self.rope_dim)
            out_id = torch_dtype_id(q_out.dtype)
        elif q_out is not None:
            raise ValueError("q_out without q_rope")
        if rows_out is not None:
            if rows_out.shape != kv.shape or rows_out.dtype != _ID_TORCH[self.dtype]:
                raise TypeError("rows_out must have kv's shape and the cache's dtype")
            ra = _on(rows_out, index)
        _check(call.it_latent_append(self._at, None if rotary is None else rotary._at, kv.data_ptr(), torch_dtype_id(kv.dtype),
                                     token, wa, weight_id, float(eps), qa, qs, qh, heads, oa, out_id, os, oh, ra,
                                     _on(slot_mapping, index), pa, n, _raw_stream(index)))
        if given is not None:
            _written(given)
        if rows_out is not None:
            _written(rows_out)
        return q_out

    def gather(self, block_tables: torch.Tensor, ctx_lens: torch.Tensor, start_pos: Optional[torch.Tensor], cu_out: torch.Tensor,
               max_tokens: int, out: torch.Tensor) -> None:
        """Rows of each sequence's tokens start .. ctx in order (it_kv_gather),
        sequence b from row cu_out[b] of out [rows, latent_dim + rope_dim]:
        what the projection up of a chunk after a cached prefix reads."""
        if out.dtype != _ID_TORCH[self.dtype] or out.dim() != 2 or out.shape[1] != self.head_dim:
            raise TypeError("out must be [rows, latent_dim + rope_dim] of the cache's dtype")
        at = self._index
        for t, dt, name in ((block_tables, torch.int32, "block_tables"), (ctx_lens, torch.int32, "ctx_lens"),
                            (start_pos, torch.int32, "start_pos"), (cu_out, torch.int64, "cu_out")):
            if t is not None and t.dtype != dt:
                raise TypeError(f"{name} must be {dt}")
        _check(call.it_kv_gather(self._at, _on(block_tables, at), block_tables.shape[1], _on(ctx_lens, at),
                                 None if start_pos is None else _on(start_pos, at), _on(cu_out, at), ctx_lens.numel(), max_tokens,
                                 _on(out, at), None, _raw_stream(at)))

    # ---- attention --------------------------------------------------------
    def decode_workspace(self, n_seqs: int, n_heads: int, max_tokens: int, q_len: int = 1) -> torch.Tensor:
        """A workspace for `decode` (calls that overlap in time need one each)."""
        nbytes = call.it_latent_decode_workspace(self._at, n_seqs, q_len, n_heads, max_tokens)
        return torch.empty(nbytes, dtype=torch.uint8, device=self.device)

    def decode(self, q_latent: torch.Tensor, q_rope: torch.Tensor, block_tables: torch.Tensor, ctx_lens: torch.Tensor,
               max_tokens: int, scale: float, start_pos: Optional[torch.Tensor] = None, q_len: int = 1,
               out: Optional[torch.Tensor] = None, ws: Optional[torch.Tensor] = None,
               out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """Absorbed attention of the last q_len tokens of each sequence, whose
        rows are already appended (it_latent_decode): q_latent [n_seqs * q_len,
        n_heads, latent_dim] (each head's query through its key projection,
        transposed) and q_rope [.., rope_dim], of the cache's dtype, parts of
        one tensor or of two; scale the expanded form's, 1 / sqrt(its key
        width).  max_tokens bounds the contexts (with start_pos: what is seen of
        them and up to 31 more).  Returns [n_seqs * q_len, n_heads, latent_dim], which the
        caller projects up to each head's value, without a gradient: queries
        that require one are refused, unless gradients are off."""
        if _grad_on() and (q_latent.requires_grad or q_rope.requires_grad or (out is not None and out.requires_grad)):
            _refuse_gradient("decode")
        index, n_seqs = self._index, ctx_lens.numel()
        if q_latent.dim() != 3 or q_latent.dtype != q_rope.dtype:
            raise ValueError("q_latent and q_rope must be [n_seqs * q_len, n_heads, ..] of one dtype")
        n, heads = n_seqs * q_len, q_latent.shape[1]
        la, ls, lh = _heads(q_latent, "q_latent", index, n, heads, self.latent_dim)
        ra, rs, rh = _heads(q_rope, "q_rope", index, n, heads, self.rope_dim)
        if block_tables.dtype != torch.int32 or ctx_lens.dtype != torch.int32 or block_tables.dim() != 2 or block_tables.shape[0] != n_seqs:
            raise TypeError("block_tables must be int32 [n_seqs, max_blocks], ctx_lens int32 [n_seqs]")
        if start_pos is not None and (start_pos.dtype != torch.int32 or start_pos.numel() != n_seqs):
            raise TypeError("start_pos must be int32 [n_seqs]")
        given = out
        if out is None:
            out = torch.empty((n, heads, self.latent_dim), dtype=out_dtype or q_latent.dtype, device=self.device)
        elif out.shape != q_latent.shape:
            raise ValueError("out must have q_latent's shape")
        if ws is None:
            ws = self.decode_workspace(n_seqs, heads, max_tokens, q_len)
        _check(call.it_latent_decode(self._at, la, ra, torch_dtype_id(q_latent.dtype), ls, lh, rs, rh, heads, q_len,
                                     _on(block_tables, index), block_tables.shape[1], _on(ctx_lens, index),
                                     None if start_pos is None else _on(start_pos, index), n_seqs, max_tokens, float(scale),
                                     _on(ws, index), ws.nbytes, _on(out, index), torch_dtype_id(out.dtype), _raw_stream(index)))
        if given is not None:
            _written(given)
        return out


def latent_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_rope: torch.Tensor, cu_q: torch.Tensor, cu_k: torch.Tensor,
                   max_q_len: int, max_k_len: int, scale: float, causal: bool = True, out: Optional[torch.Tensor] = None,
                   out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Expanded attention over contiguous keys and values (it_latent_prefill):
    q [total_q, n_heads, nope + rope], k [total_k, n_heads, nope] and v [total_k,
    n_heads, v_dim] projected up from the latents (parts of one tensor too),
    k_rope [total_k, rope] shared by all heads (a part of the gathered rows);
    int32 cu_q, cu_k [n_seqs + 1], and bounds of the sequences' lengths, past
    which a sequence is not computed.  With causal, query i of a sequence sees
    its keys 0 .. k_len - q_len + i.  Returns [total_q, n_heads, v_dim], without
    a gradient: tensors that require one are refused, unless gradients are off."""
    if _grad_on() and (q.requires_grad or k.requires_grad or v.requires_grad or k_rope.requires_grad or
                       (out is not None and out.requires_grad)):
        _refuse_gradient("latent_prefill")
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3 or k_rope.dim() != 2:
        raise ValueError("q, k, v must be [tokens, n_heads, dim], k_rope [tokens, rope_dim]")
    index = q.get_device()
    if index < 0:
        raise ValueError("device tensor expected")
    (total_q, heads, width), (total_k, _, nope), rope = q.shape, k.shape, k_rope.shape[1]
    if nope + rope != width:
        raise ValueError(f"q holds {width} elements a head, k and k_rope {nope} + {rope}")
    if k.dtype != q.dtype or v.dtype != q.dtype or k_rope.dtype != q.dtype:
        raise TypeError("q, k, v and k_rope must have one dtype")
    if cu_q.dtype != torch.int32 or cu_k.dtype != torch.int32 or cu_q.numel() != cu_k.numel() or cu_q.numel() < 1:
        raise TypeError("cu_q and cu_k must be int32 [n_seqs + 1]")
    qa, qs, qh = _heads(q, "q", index, total_q, heads, width)
    ka, ks, kh = _heads(k, "k", index, total_k, heads, nope)
    va, vs, vh = _heads(v, "v", index, total_k, heads, v.shape[2])
    if k_rope.shape[0] != total_k or k_rope.get_device() != index or (k_rope.stride(1) != 1 and rope != 1 and k_rope.numel()):
        raise ValueError(f"k_rope must be [{total_k}, rope_dim] on cuda:{index}, rows contiguous")
    shape, given = (total_q, heads, v.shape[2]), out
    if out is None:
        out = torch.empty(shape, dtype=out_dtype or q.dtype, device=q.device)
    elif out.shape != shape:
        raise ValueError("out must be [total_q, n_heads, v_dim]")
    args = (qa, ka, va, k_rope.data_ptr(), torch_dtype_id(q.dtype), qs, qh, ks, kh, vs, vh, k_rope.stride(0), heads, nope, rope,
            v.shape[2], _on(cu_q, index), _on(cu_k, index), cu_q.numel() - 1, total_q, total_k, max_q_len, max_k_len, float(scale),
            int(bool(causal)), _on(out, index), torch_dtype_id(out.dtype), _raw_stream(index))
    if torch._C._cuda_getDevice() == index:
        _check(call.it_latent_prefill(*args))
    else:
        with torch.cuda.device(index):
            _check(call.it_latent_prefill(*args))
    if given is not None:
        _written(given)
    return out
