"""Attention of new tokens over the quantised paged cache (libqlinear).

The reference's decode attention reads one new token per sequence through a
block table (src/kernels/paged_attention_triton.py:23-193).  Here a request
brings one token, a chain, or a tree of drafted tokens (speculative decoding),
all of them attending in one call to the 8- or 4-bit cache in place.
"""
from __future__ import annotations

import torch

from .. import _lib
from ._launch import activation_code, call, current_raw_stream, call_flags, on_device, scratch
from .kv_cache import QuantizedKVCache


_workspace_bytes: dict[int, int] = {}


def _workspace(device: torch.device) -> torch.Tensor:
    nbytes = _workspace_bytes.get(device.index)
    if nbytes is None:
        with on_device(device):                      # what the largest head needs, so that no call outgrows it
            nbytes = max(_lib.load().ql_tree_attention_workspace_size(d) for d in (64, 128, 256))
        _workspace_bytes[device.index] = nbytes
    return scratch(device, current_raw_stream(device.index), nbytes)


def pack_tree_mask(visible: torch.Tensor) -> torch.Tensor:
    """Boolean (..., tokens, tokens), true where the row's token sees the
    column's, as 64-bit words (..., tokens, words): bit d % 64 of word d // 64
    for new token d."""
    n = visible.shape[-1]
    words = max(1, -(-n // 64))
    bits = torch.zeros(*visible.shape[:-1], words * 64, dtype=torch.int64, device=visible.device)
    bits[..., :n] = visible
    return (bits.unflatten(-1, (words, 64)) << torch.arange(64, device=visible.device)).sum(-1)


def tree_mask_from_parents(parents) -> torch.Tensor:
    """The packed mask of one tree on the CPU: token i sees itself and its
    ancestors; parents[i] < i is its parent, or -1 for a root."""
    n = len(parents)
    visible = torch.eye(n, dtype=torch.bool)
    for i, parent in enumerate(parents):
        assert -1 <= parent < i, f"token {i}'s parent must come before it, got {parent}"
        if parent >= 0:
            visible[i] |= visible[parent]
    return pack_tree_mask(visible)


def tree_attention(q: torch.Tensor, cache: QuantizedKVCache, page_table: torch.Tensor, kv_lens: torch.Tensor,
                   cu_q: torch.Tensor = None, mask: torch.Tensor = None, max_q: int = None, max_kv: int = None,
                   scale: float = None, out: torch.Tensor = None, return_lse: bool = False):
    """Attention of the new tokens q (total_q, q_heads, head_dim) fp16 / bf16
    over their requests' cached rows, the new tokens' own (already appended)
    included.

    * page_table int32 (batch, pages): position j of request b is in page
      ``page_table[b, j // page_size]``;
    * kv_lens int32 (batch,): cached positions, new tokens included (they are
      the last ones);
    * cu_q int32 (batch + 1,): request b's rows are cu_q[b] .. cu_q[b+1] - 1
      (rows that it does not cover are left as they are: not written); None gives each total_q / batch rows (one token each in plain decoding);
    * mask int64 (total_q, words): which of its request's new tokens a row
      sees (``pack_tree_mask``); None: those up to itself.  Every row sees all
      positions before the new tokens.  A row that sees nothing gives zeros;
    * max_q, max_kv: the most rows and positions of any request, where the
      caller knows them; they only help to choose the launch;
    * scale: on the scores, 1 / sqrt(head_dim) by default.

    Returns (total_q, q_heads, head_dim) in q's dtype, and with
    ``return_lse`` the rows' log-sums (total_q, q_heads) fp32 (minus infinity
    where nothing is seen).  Gradients are not recorded: both are detached."""
    shape, dev, dtype = q.shape, cache.device, q.dtype
    assert q.is_cuda and len(shape) == 3, f"q must be a CUDA tensor (total_q, q_heads, head_dim), got {tuple(shape)}"
    total_q, q_heads, head_dim = shape
    code = activation_code(dtype, "tree_attention: q")
    assert q.device == dev and head_dim == cache.head_dim, \
        f"q must be (total_q, q_heads, {cache.head_dim}) on {dev}, got {tuple(shape)} on {q.device}"
    assert q_heads % cache.kv_heads == 0, f"q_heads {q_heads} must be a multiple of kv_heads {cache.kv_heads}"
    if page_table.dtype != torch.int32 or kv_lens.dtype != torch.int32:
        raise TypeError(f"page_table and kv_lens must be int32, got {page_table.dtype} and {kv_lens.dtype}")
    table_shape, lens_shape = page_table.shape, kv_lens.shape
    assert len(lens_shape) == 1 and kv_lens.device == dev, f"kv_lens must be (batch,) on {dev}"
    batch = lens_shape[0]
    assert len(table_shape) == 2 and table_shape[0] == batch and page_table.device == dev, \
        f"page_table must be ({batch}, pages) on {dev}, got {tuple(table_shape)} on {page_table.device}"
    if not kv_lens.is_contiguous():
        kv_lens = kv_lens.contiguous()
    cu_ptr, mask_ptr, words = 0, 0, 0
    if cu_q is not None:
        if cu_q.dtype != torch.int32:
            raise TypeError(f"cu_q must be int32, got {cu_q.dtype}")
        assert cu_q.shape == (batch + 1,) and cu_q.device == dev, f"cu_q must be ({batch + 1},) on {dev}"
        if not cu_q.is_contiguous():
            cu_q = cu_q.contiguous()
        cu_ptr = cu_q.data_ptr()
        if max_q is None:
            max_q = total_q
    elif total_q > 0:
        assert batch > 0, "q has rows but there is no request"
        assert total_q % batch == 0, f"{total_q} rows do not divide among {batch} requests: pass cu_q"
        max_q = total_q // batch
    if mask is not None:
        if mask.dtype != torch.int64:
            raise TypeError(f"mask must be int64, got {mask.dtype}")
        assert mask.dim() == 2 and mask.shape[0] == total_q and mask.device == dev, \
            f"mask must be ({total_q}, words) on {dev}, got {tuple(mask.shape)} on {mask.device}"
        words = mask.shape[1]
        assert 1 <= words <= 1024, f"mask must have 1 to 1024 words a row, got {words}"
        mask = mask.contiguous()
        mask_ptr = mask.data_ptr()
    if out is None:
        out = q.new_empty(shape)
    else:
        assert out.shape == shape and out.dtype == dtype and out.device == dev and out.is_contiguous(), \
            f"out must be contiguous {tuple(shape)} {dtype} on {dev}"
    lse = torch.empty((total_q, q_heads), dtype=torch.float32, device=dev) if return_lse else None
    if total_q > 0 and batch > 0:
        qs, ts, width = q.stride(), page_table.stride(), table_shape[1]
        if qs[2] != 1:
            q = q.contiguous()
            qs = q.stride()
        if ts[1] != 1 or ts[0] < width and batch > 1:        # also one row for all (expanded), or rows that overlap
            page_table = page_table.contiguous()
            ts = page_table.stride()
        if max_kv is None:
            max_kv = width * cache.page_size
        ws = _workspace(dev)
        packed = _lib.TREE_ATTENTION_ARGS.pack(
            *cache.fields, q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0, page_table.data_ptr(),
            kv_lens.data_ptr(), cu_ptr, mask_ptr, batch, total_q, q_heads, qs[0], qs[1], width,
            ts[0] if batch > 1 else width, words, max_q, max_kv, code,
            head_dim ** -0.5 if scale is None else scale, ws.data_ptr(), ws.numel(), call_flags())
        call(_lib.load().ql_tree_attention, packed, dev)
    return (out, lse) if return_lse else out


__all__ = ["tree_attention", "pack_tree_mask", "tree_mask_from_parents"]
