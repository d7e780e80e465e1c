"""Attention of requests that share long prefixes, over the quantised paged
cache (libqlinear).

Requests of a batch that begin alike (a system prompt, many answers to one
question, many questions about one document) share the pages of that beginning.
``tree_attention`` reads them once for every request; here each group's prefix
is read once for all its rows, and what a request has of its own as before.
"""
from __future__ import annotations

import torch

from .. import _lib
from ._launch import activation_code, call, call_flags
from .kv_cache import QuantizedKVCache
from .tree_attention import _workspace


def parts_size(total_q: int, q_heads: int, head_dim: int) -> int:
    """ql_shared_attention_parts_size, without the call: the rows' sums up to a multiple of 16 bytes, then their outputs."""
    rows = total_q * q_heads
    return (8 * rows + 15 & -16) + 4 * rows * head_dim


def _index(t: torch.Tensor, shape: tuple, device: torch.device, what: str) -> torch.Tensor:
    if t.dtype != torch.int32:
        raise TypeError(f"{what} must be int32, got {t.dtype}")
    assert t.shape == shape and t.device == device, \
        f"{what} must be {shape} on {device}, got {tuple(t.shape)} on {t.device}"
    return t if t.is_contiguous() else t.contiguous()


def _table(t: torch.Tensor, rows: int, device: torch.device, what: str):
    """The table, its entries between rows and its width."""
    if t.dtype != torch.int32:
        raise TypeError(f"{what} must be int32, got {t.dtype}")
    assert t.dim() == 2 and t.shape[0] == rows and t.device == device, \
        f"{what} must be ({rows}, pages) on {device}, got {tuple(t.shape)} on {t.device}"
    stride, width = t.stride(), t.shape[1]
    if stride[1] != 1 or stride[0] < width and rows > 1:
        t = t.contiguous()
        stride = t.stride()
    return t, stride[0] if rows > 1 else width, width


def shared_prefix_attention(q: torch.Tensor, cache: QuantizedKVCache, prefix_table: torch.Tensor,
                            prefix_lens: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor,
                            cu_group: torch.Tensor = None, cu_q: torch.Tensor = None, mask: torch.Tensor = None,
                            max_q: int = None, max_prefix: int = None, max_kv: int = None, scale: float = None,
                            out: torch.Tensor = None, return_lse: bool = False):
    """Attention of the new tokens q (total_q, q_heads, head_dim) fp16 / bf16:
    of each over its group's prefix, all of it, and its request's own cached
    rows, as ``tree_attention`` sees these.

    * prefix_table int32 (groups, pages), prefix_lens int32 (groups,): the
      pages and lengths of the prefixes;
    * cu_group int32 (groups + 1,): group g's requests are cu_group[g] ..
      cu_group[g+1] - 1 (not decreasing; requests outside have no prefix); None:
      one group of all requests;
    * page_table int32 (batch, pages), kv_lens int32 (batch,): the requests' own
      positions behind the prefix, new tokens included; they begin a page;
    * cu_q, mask, max_q, scale: as in ``tree_attention``; the mask is over the
      new tokens, and rows of q behind the last request's are left as they are
      in the output (not written: pass ``out`` to say what they hold);
    * max_prefix, max_kv: the most positions of any prefix, and of any request's
      own, where the caller knows them; they only help to choose the launch.

    Returns what ``tree_attention`` returns, of the softmax over both."""
    shape, dev, dtype = q.shape, cache.device, q.dtype
    assert q.is_cuda and len(shape) == 3, f"q must be a CUDA tensor (total_q, q_heads, head_dim), got {tuple(shape)}"
    total_q, q_heads, head_dim = shape
    code = activation_code(dtype, "shared_prefix_attention: q")
    assert q.device == dev and head_dim == cache.head_dim, \
        f"q must be (total_q, q_heads, {cache.head_dim}) on {dev}, got {tuple(shape)} on {q.device}"
    assert q_heads % cache.kv_heads == 0, f"q_heads {q_heads} must be a multiple of kv_heads {cache.kv_heads}"
    assert kv_lens.dim() == 1 and prefix_lens.dim() == 1, "kv_lens must be (batch,) and prefix_lens (groups,)"
    batch, groups = kv_lens.shape[0], prefix_lens.shape[0]
    kv_lens, prefix_lens = _index(kv_lens, (batch,), dev, "kv_lens"), _index(prefix_lens, (groups,), dev, "prefix_lens")
    page_table, stride, width = _table(page_table, batch, dev, "page_table")
    prefix_table, prefix_stride, prefix_width = _table(prefix_table, groups, dev, "prefix_table")
    group_ptr, cu_ptr, mask_ptr, words = 0, 0, 0, 0
    if cu_group is not None:
        cu_group = _index(cu_group, (groups + 1,), dev, "cu_group")
        group_ptr = cu_group.data_ptr()
    else:
        assert groups == 1, f"{groups} prefixes: pass cu_group"
    if cu_q is not None:
        cu_q = _index(cu_q, (batch + 1,), dev, "cu_q")
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
        qs = q.stride()
        if qs[2] != 1:
            q = q.contiguous()
            qs = q.stride()
        lib, ws = _lib.load(), _workspace(dev)
        # of this call alone: the allocator hands it on only to what the stream runs later
        nbytes = parts_size(total_q, q_heads, head_dim)
        parts = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        packed = _lib.SHARED_ATTENTION_ARGS.pack(
            *cache.fields, q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0, page_table.data_ptr(),
            kv_lens.data_ptr(), cu_ptr, mask_ptr, batch, total_q, q_heads, qs[0], qs[1], width, stride, words, max_q,
            width * cache.page_size if max_kv is None else max_kv, code, head_dim ** -0.5 if scale is None else scale,
            ws.data_ptr(), ws.numel(), call_flags(), prefix_table.data_ptr(), prefix_lens.data_ptr(), group_ptr,
            parts.data_ptr(), groups, prefix_width, prefix_stride,
            prefix_width * cache.page_size if max_prefix is None else max_prefix, nbytes)
        call(lib.ql_shared_attention, packed, dev)
    return (out, lse) if return_lse else out


__all__ = ["shared_prefix_attention"]
