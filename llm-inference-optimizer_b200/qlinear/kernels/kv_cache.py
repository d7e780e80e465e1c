"""Quantised paged key/value cache (libqlinear).

The reference keeps fp16 pools of pages with a block table per sequence
(src/kv_cache/block_manager.py:25-198).  Here a cached row (one token of one
key/value head) is held in 8 or 4 bits: integer codes and a bf16 scale, per
row at 8 bits (head_dim + 2 bytes) and per 64 elements at 4 bits.

``append_kv`` quantises new keys and values into their slots, turning k (and
q) by rotary positions in the same launch; ``read_kv`` reads rows back;
``tree_attention`` attends over the cache in place.  A slot is
``page * page_size + offset``.
"""
from __future__ import annotations

import torch

from .. import _lib
from ._launch import activation_code, call, call_flags, index_bytes
from .rotary import RotaryTable

GROUP4 = 64                     # elements that share a scale at 4 bits


class QuantizedKVCache:
    """One layer's pool: codes (num_pages, kv_heads, page_size, row bytes),
    int8 at 8 bits and uint8 at 4, and scales bf16 (num_pages, kv_heads,
    page_size, groups).  Pages may be strided views (a slice of a pool for
    all layers); within a page the tensors are contiguous.  The tensors are
    the cache's for its life: to grow a pool, make another cache."""

    # calls pass on the addresses that `fields` holds, so none may be exchanged for another tensor
    k_codes = property(lambda self: self._tensors[0])
    k_scales = property(lambda self: self._tensors[1])
    v_codes = property(lambda self: self._tensors[2])
    v_scales = property(lambda self: self._tensors[3])

    def __init__(self, k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor,
                 v_scales: torch.Tensor):
        if k_codes.dtype not in (torch.int8, torch.uint8):
            raise TypeError(f"codes must be int8 (8 bits) or uint8 (4 bits), got {k_codes.dtype}")
        self.bits = 8 if k_codes.dtype == torch.int8 else 4
        assert k_codes.dim() == 4, f"codes must have 4 dimensions, got {tuple(k_codes.shape)}"
        self.num_pages, self.kv_heads, self.page_size, row = k_codes.shape
        self.head_dim = row * 8 // self.bits
        self.groups = 1 if self.bits == 8 else self.head_dim // GROUP4
        if self.head_dim not in (64, 128, 256):
            raise ValueError(f"head_dim must be 64, 128 or 256, got {self.head_dim}")
        if self.page_size < 16 or self.page_size > 65536 or self.page_size & (self.page_size - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 65536, got {self.page_size}")
        assert self.num_pages > 0 and self.kv_heads > 0, "the pool is empty"
        assert v_codes.shape == k_codes.shape and v_codes.dtype == k_codes.dtype, "k and v codes differ in form"
        for t in (k_scales, v_scales):
            assert t.shape == (*k_codes.shape[:3], self.groups), f"scales shape {tuple(t.shape)}"
            if t.dtype != torch.bfloat16:
                raise TypeError(f"scales must be bf16, got {t.dtype}")
        self.device = k_codes.device
        for t in (k_codes, k_scales, v_codes, v_scales):
            assert t.device == self.device, "codes and scales must be on one device"
            assert t[0].is_contiguous(), "codes and scales must be contiguous within a page"
        self._tensors = (k_codes, k_scales, v_codes, v_scales)
        ts = (k_codes, v_codes, k_scales, v_scales)
        strides = [t.stride(0) if self.num_pages > 1 else t[0].numel() for t in ts]
        # the C structure's fields, which stay as they are for the cache's life
        self.fields = (k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(), v_scales.data_ptr(),
                       self.num_pages, self.page_size, self.kv_heads, self.head_dim, self.bits, *strides)

    @classmethod
    def empty(cls, num_pages: int, page_size: int, kv_heads: int, head_dim: int, bits: int = 8,
              device="cuda") -> "QuantizedKVCache":
        """A pool of zero rows."""
        if bits not in (8, 4):
            raise ValueError(f"bits must be 8 or 4, got {bits}")
        row, groups = (head_dim, 1) if bits == 8 else (head_dim // 2, max(1, head_dim // GROUP4))
        ts = []
        for _ in range(2):
            codes = torch.zeros(num_pages, kv_heads, page_size, row, device=device,
                                dtype=torch.int8 if bits == 8 else torch.uint8)
            ts += [codes if bits == 8 else codes.fill_(0x88),
                   torch.zeros(num_pages, kv_heads, page_size, groups, dtype=torch.bfloat16, device=device)]
        return cls(*ts)

    def num_bytes(self) -> int:
        """Bytes held on the device: codes and scales of keys and values."""
        return sum(t.numel() * t.element_size()
                   for t in (self.k_codes, self.k_scales, self.v_codes, self.v_scales))

    def move(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Copies the rows at slots `src` (rows,) to `dst` (all read before any
        is written): the rows of accepted drafted tokens close up behind the
        context.  Codes move as they are, so nothing is rounded again.  A pair
        with a negative slot is skipped, and one with a slot past the pool,
        which is recorded as elsewhere."""
        index_bytes(src, "src"), index_bytes(dst, "dst")
        assert src.dim() == 1 and src.shape == dst.shape, \
            f"src and dst must be (rows,) alike, got {tuple(src.shape)} and {tuple(dst.shape)}"
        assert src.device == self.device and dst.device == self.device, f"src and dst must be on {self.device}"
        if src.shape[0] == 0:
            return
        end, pairs = self.num_pages * self.page_size, torch.stack((src.long(), dst.long()))
        inside = pairs < end
        if self.device.type == "cuda":
            read_kv(self, torch.where(inside, -1, pairs).view(-1))     # records what is past the pool
        # no size may depend on the slots: a skipped pair repeats one that is kept, or moves row 0 to itself if none is
        kept = (inside & (pairs >= 0)).all(0)
        pairs = torch.where(kept, pairs, (pairs * kept).index_select(1, kept.byte().argmax(0, keepdim=True)))
        (page, to_page), (at, to_at) = (pairs >> self.page_size.bit_length() - 1).unbind(), \
            (pairs & self.page_size - 1).unbind()
        for t in (self.k_codes, self.k_scales, self.v_codes, self.v_scales):
            rows = t.transpose(1, 2)
            rows.index_put_((to_page, to_at), rows[page, at])


def append_kv(cache: QuantizedKVCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
              q: torch.Tensor = None, positions: torch.Tensor = None, rotary: RotaryTable = None,
              q_out: torch.Tensor = None) -> torch.Tensor | None:
    """Quantises k, v (tokens, kv_heads, head_dim) fp16 / bf16 into `slots`
    (tokens,); a negative slot writes nothing.  With `rotary` and `positions`,
    k is turned first, in fp32; with q (tokens, q_heads, head_dim) too, q is
    turned by the same angles and returned (in `q_out`, which may be q).
    Tensors may have any strides with unit stride along head_dim, such as
    the column slices of a fused projection's output.  Gradients are not
    recorded: the result is detached."""
    shape, dev = k.shape, cache.device
    tokens = shape[0]
    assert k.device == dev and k.is_cuda, f"k is on {k.device}, the cache on {dev}"
    assert shape == (tokens, cache.kv_heads, cache.head_dim), \
        f"k must be (tokens, {cache.kv_heads}, {cache.head_dim}), got {tuple(shape)}"
    dtype = k.dtype
    code = activation_code(dtype, "append_kv: k")
    assert v.shape == shape and v.dtype == dtype and v.device == dev, f"v must be {tuple(shape)} {dtype} on {dev}"
    assert slots.shape == (tokens,) and slots.device == dev, \
        f"slots must be ({tokens},) on {dev}, got {tuple(slots.shape)} on {slots.device}"
    ks, vs = k.stride(), v.stride()
    if ks[2] != 1:
        k = k.contiguous()
        ks = k.stride()
    if vs[2] != 1:
        v = v.contiguous()
        vs = v.stride()
    if not slots.is_contiguous():
        slots = slots.contiguous()
    table, position_ptr, turn = 0, 0, (0, 0, 0, 8)
    if rotary is not None:
        assert positions is not None, "rotary and positions go together"
        assert rotary.device == dev, f"the rotary table is on {rotary.device}, k on {dev}"
        assert rotary.rotary_dim <= cache.head_dim, f"rotary_dim {rotary.rotary_dim} > head_dim {cache.head_dim}"
        assert positions.shape == (tokens,) and positions.device == dev, \
            f"positions must be ({tokens},) on {dev}, got {tuple(positions.shape)} on {positions.device}"
        if not positions.is_contiguous():
            positions = positions.contiguous()
        table, position_ptr = rotary.ptr, positions.data_ptr()
        turn = (rotary.rotary_dim, rotary.max_positions, rotary.layout_code, index_bytes(positions, "positions"))
    else:
        assert positions is None, "rotary and positions go together"
    q_heads, q_ptr, q_out_ptr, qs, os_ = 0, 0, 0, (0, 0), (0, 0)
    if q is not None:
        assert rotary is not None, "q is taken to be turned: pass rotary and positions"
        q_shape = q.shape
        assert len(q_shape) == 3 and q_shape[0] == tokens and q_shape[2] == shape[2] and q.dtype == dtype \
            and q.device == dev, f"q must be ({tokens}, q_heads, {shape[2]}) {dtype} on {dev}"
        if q_out is None:
            q_out = q.new_empty(q_shape)
        else:
            assert q_out.shape == q_shape and q_out.dtype == dtype and q_out.device == dev \
                and q_out.stride(-1) == 1, f"q_out must be {tuple(q_shape)} {dtype} with unit inner stride"
        qs, os_ = q.stride(), q_out.stride()
        if qs[2] != 1:
            q = q.contiguous()
            qs = q.stride()
        q_heads, q_ptr, q_out_ptr = q_shape[1], q.data_ptr(), q_out.data_ptr()
    else:
        assert q_out is None, "q_out without q"
    if tokens == 0:
        return q_out
    packed = _lib.KV_APPEND_ARGS.pack(
        *cache.fields, k.data_ptr(), v.data_ptr(), q_ptr, q_out_ptr, slots.data_ptr(), table, position_ptr, tokens,
        q_heads, ks[0], ks[1], vs[0], vs[1], qs[0], qs[1], os_[0], os_[1], code, index_bytes(slots, "slots"),
        *turn, call_flags())
    call(_lib.load().ql_kv_append, packed, dev)
    return q_out


def read_kv(cache: QuantizedKVCache, slots: torch.Tensor,
            dtype: torch.dtype = torch.float16) -> tuple[torch.Tensor, torch.Tensor]:
    """The rows at `slots` (tokens,) as k, v (tokens, kv_heads, head_dim) in
    fp16 or bf16, one rounding; zeros where a slot is negative."""
    dev = cache.device
    assert slots.dim() == 1 and slots.device == dev, f"slots must be (tokens,) on {dev}"
    code = activation_code(dtype, "read_kv: dtype")
    tokens = slots.shape[0]
    k, v = torch.empty((2, tokens, cache.kv_heads, cache.head_dim), dtype=dtype, device=dev).unbind(0)
    if tokens == 0:
        return k, v
    if not slots.is_contiguous():
        slots = slots.contiguous()
    packed = _lib.KV_READ_ARGS.pack(*cache.fields, slots.data_ptr(), k.data_ptr(), v.data_ptr(), tokens, code,
                                    index_bytes(slots, "slots"), call_flags())
    call(_lib.load().ql_kv_read, packed, dev)
    return k, v


__all__ = ["QuantizedKVCache", "append_kv", "read_kv", "GROUP4"]
