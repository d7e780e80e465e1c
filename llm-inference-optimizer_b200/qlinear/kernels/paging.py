"""Page tables of a serving batch, kept and advanced on the GPU (libqlinear).

The reference's block manager hands out pages on the host, one Python call per
sequence and step (src/kv_cache/block_manager.py:25-198).  Here the page table,
the requests' lengths and the stack of free pages are tensors, and one launch a
step gives refused tokens' pages back, takes the pages of the new tokens and
writes what ``append_kv`` and ``tree_attention`` need: slots, positions, the
tokens' division among the requests, lengths.  A captured graph replays it step
after step.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _lib
from ._launch import call, call_flags


class StepPlan(NamedTuple):
    """A step's new tokens.  ``cu_q`` int32 (batch + 1,): request b's are rows
    cu_q[b] .. cu_q[b + 1] - 1; ``slots`` int64 and ``positions`` int32
    (max_tokens,), -1 and 0 behind the last row; ``kv_lens`` int32 (batch,) is
    the page tables' own ``lens``, the new tokens included; ``refused`` int32
    (1,): requests that asked for tokens and got none."""
    cu_q: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor
    kv_lens: torch.Tensor
    refused: torch.Tensor


class PageTables:
    """Which pages of a pool each request of a batch holds, and which are free.

    * page_table int32 (batch, width): the first ceil(lens[b] / page_size)
      entries of row b are its pages (further ones mean nothing);
    * lens int32 (batch,): its cached tokens; a row of 0 is a free place;
    * free_pages int32 (num_pages,) and free_count int32 (1,): the first
      free_count entries are the free pages, the last of them taken first.

    The tensors are the object's for its life, and calls change them: calls that
    share some (two tables over one stack of free pages, say) must follow one
    another, as they do on one stream."""

    page_table = property(lambda self: self._tensors[0])
    lens = property(lambda self: self._tensors[1])
    free_pages = property(lambda self: self._tensors[2])
    free_count = property(lambda self: self._tensors[3])

    def __init__(self, page_table: torch.Tensor, lens: torch.Tensor, free_pages: torch.Tensor,
                 free_count: torch.Tensor, page_size: int):
        for name, t in (("page_table", page_table), ("lens", lens), ("free_pages", free_pages),
                        ("free_count", free_count)):
            if t.dtype != torch.int32:
                raise TypeError(f"{name} must be int32, got {t.dtype}")
            assert t.device == lens.device, f"{name} is on {t.device}, lens on {lens.device}"
        assert page_table.dim() == 2 and lens.shape == page_table.shape[:1] and lens.is_contiguous(), \
            f"page_table must be (batch, width) and lens (batch,), got {tuple(page_table.shape)} and {tuple(lens.shape)}"
        self.batch, self.width = page_table.shape
        if self.batch > 8192:
            raise ValueError(f"a batch has at most 8192 requests, got {self.batch}")
        assert self.batch * self.width < 2 ** 31, f"page_table has too many entries: {tuple(page_table.shape)}"
        stride = page_table.stride(0) if self.batch > 1 else self.width
        assert (page_table.stride(1) == 1 or self.width <= 1) and stride >= self.width, \
            "page_table's rows must be contiguous and apart from one another"
        assert free_pages.dim() == 1 and free_pages.is_contiguous(), "free_pages must be (num_pages,), contiguous"
        assert free_count.numel() == 1, f"free_count must hold one number, got {tuple(free_count.shape)}"
        if page_size < 1 or page_size > 65536 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two up to 65536, got {page_size}")
        self.num_pages, self.page_size, self.device = free_pages.shape[0], page_size, lens.device
        self._tensors = (page_table, lens, free_pages, free_count)
        self._state = (page_table.data_ptr(), lens.data_ptr(), free_pages.data_ptr(), free_count.data_ptr())
        self._sizes = (self.batch, self.width, stride, self.num_pages, page_size)

    @classmethod
    def empty(cls, batch: int, width: int, num_pages: int, page_size: int, device="cuda") -> "PageTables":
        """No tokens, all of the pool's pages free, page 0 taken first."""
        table = torch.zeros(batch, width, dtype=torch.int32, device=device)
        free = torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=device)
        return cls(table, torch.zeros(batch, dtype=torch.int32, device=device), free,
                   torch.full((1,), num_pages, dtype=torch.int32, device=device), page_size)

    def step_buffers(self, max_tokens: int) -> StepPlan:
        """Room for a step's plan, to be passed as ``out`` step after step."""
        dev, i32 = self.device, torch.int32
        return StepPlan(torch.empty(self.batch + 1, dtype=i32, device=dev),
                        torch.empty(max_tokens, dtype=torch.int64, device=dev),
                        torch.empty(max_tokens, dtype=i32, device=dev), self._tensors[1],
                        torch.empty(1, dtype=i32, device=dev))


def plan_step(pages: PageTables, new_tokens: torch.Tensor, max_tokens: int, keep: torch.Tensor = None,
              out: StepPlan = None) -> StepPlan:
    """Cuts every request to its first keep (batch,) int32 tokens (None: all),
    returns the pages behind them, grows it by new_tokens (batch,) int32 and
    gives the pages and slots of those.  Page tables and lengths are updated
    in place.

    A finished request is cut to 0; rejected drafts are cut off with the length
    that was accepted.  Requests are served in order: one whose pages do not fit
    its row of the table, whose tokens do not fit ``max_tokens`` behind those
    before it, or that needs pages which are not free behind what requests
    before it need, is only cut, and counts in ``refused``."""
    dev, batch = pages.device, pages.batch
    assert dev.type == "cuda", f"plan_step: the page tables are on {dev}"
    if new_tokens.dtype != torch.int32:
        raise TypeError(f"new_tokens must be int32, got {new_tokens.dtype}")
    assert new_tokens.shape == (batch,) and new_tokens.device == dev, \
        f"new_tokens must be ({batch},) on {dev}, got {tuple(new_tokens.shape)} on {new_tokens.device}"
    if not new_tokens.is_contiguous():
        new_tokens = new_tokens.contiguous()
    keep_ptr = 0
    if keep is not None:
        if keep.dtype != torch.int32:
            raise TypeError(f"keep must be int32, got {keep.dtype}")
        assert keep.shape == (batch,) and keep.device == dev, \
            f"keep must be ({batch},) on {dev}, got {tuple(keep.shape)} on {keep.device}"
        if not keep.is_contiguous():
            keep = keep.contiguous()
        keep_ptr = keep.data_ptr()
    if max_tokens < 0 or max_tokens >= 2 ** 31 - 1:
        raise ValueError(f"max_tokens must be from 0 to 2^31 - 2, got {max_tokens}")
    if out is None:
        out = pages.step_buffers(max_tokens)
        cu_q, slots, positions, _, refused = out
    else:
        cu_q, slots, positions, lens, refused = out
        if (slots.dtype, positions.dtype, cu_q.dtype, refused.dtype) != (torch.int64, torch.int32, torch.int32, torch.int32):
            raise TypeError("out must hold cu_q, positions and refused in int32 and slots in int64")
        assert cu_q.shape == (batch + 1,) and slots.shape == positions.shape == (max_tokens,) and refused.shape == (1,) \
            and lens is pages.lens, f"out does not fit {batch} requests and {max_tokens} tokens"
        for t in (cu_q, slots, positions, refused):
            assert t.device == dev and t.is_contiguous(), f"out must be contiguous on {dev}"
    packed = _lib.PLAN_STEP_ARGS.pack(*pages._state, keep_ptr, new_tokens.data_ptr(), cu_q.data_ptr(), slots.data_ptr(),
                                      positions.data_ptr(), refused.data_ptr(), *pages._sizes, max_tokens, call_flags())
    call(_lib.load().ql_plan_step, packed, dev)
    return out


__all__ = ["PageTables", "StepPlan", "plan_step"]
