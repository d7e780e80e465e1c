"""Rotary positions for query and key heads (libqlinear).

The reference's engines rotate q and k between the projections and the
attention with the model's cos / sin tensors (src/engine/paged_engine.py:98-126).
``RotaryTable`` holds those angles for every position once, with any scaling
for long contexts folded in; ``apply_rotary`` turns heads by them in one
launch, reading the column slices of a fused projection's output as they are.
Turning q and k while k is written to a cache is ``kv_cache.append_kv``.
"""
from __future__ import annotations

import math

import torch

from .. import _lib
from ._launch import activation_code, call, call_flags, index_bytes

# What a model's configuration says of its rotary positions.  (mrope: the three positions of a token of text are one.)
_KEYS = {"rope_type", "type", "rope_theta", "partial_rotary_factor", "factor", "original_max_position_embeddings",
         "max_position_embeddings", "low_freq_factor", "high_freq_factor", "beta_fast", "beta_slow", "attention_factor",
         "truncate", "mscale", "mscale_all_dim", "finetuned", "mrope_section", "mrope_interleaved"}
LAYOUTS = {"half": _lib.QL_ROTARY_HALF, "interleaved": _lib.QL_ROTARY_INTERLEAVED}


def _kind(scaling: dict) -> str:
    """The scaling's name, under its older key too."""
    return scaling.get("rope_type") or scaling.get("type") or "default"


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: dict | None = None,
                       max_positions: int | None = None) -> tuple[torch.Tensor, float]:
    """Radians per position of each pair (float64 [rotary_dim / 2]) and the
    factor on cos and sin.  `scaling` follows the model configurations:
    ``{"rope_type": name, ...}`` with

    * ``default``: base ** (-2i / rotary_dim);
    * ``linear``: all of them divided by ``factor``;
    * ``dynamic``: the base grown so that ``max_positions`` positions span what
      ``original_max_position_embeddings`` did (times ``factor``);
    * ``llama3``: wavelengths longer than original / low_freq_factor divided by
      ``factor``, shorter than original / high_freq_factor kept, and a linear
      step in original / wavelength between;
    * ``yarn``: pairs that turn less than ``beta_slow`` times over the original
      length divided by ``factor``, more than ``beta_fast`` times kept, a ramp
      over the pair index between (its ends whole pairs, unless ``truncate``
      is false), and cos / sin times ``attention_factor``; that is unless given
      m(1) with m(x) = 0.1 x ln(factor) + 1, or m(mscale) / m(mscale_all_dim)
      where both are.

    Keys that it does not know are refused, since they may change the angles
    (parameters by kind of layer among them: pass one kind's).
    """
    s = {name: value for name, value in (scaling or {}).items() if value is not None}
    unknown = sorted(set(s) - _KEYS)
    if unknown:
        raise ValueError(f"rotary scaling has keys that are not known: {', '.join(map(repr, unknown))}")
    kind = _kind(s)
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)

    def need(name):
        if s.get(name) is None:
            raise ValueError(f"rotary scaling {kind!r} needs {name!r}")
        return float(s[name])

    if kind == "dynamic":
        old, factor = need("original_max_position_embeddings"), need("factor")
        if max_positions is not None and max_positions > old:
            base = base * (factor * max_positions / old - (factor - 1.0)) ** (rotary_dim / (rotary_dim - 2.0))
    f = float(base) ** (-2.0 * i / rotary_dim)
    if kind in ("default", "dynamic"):
        return f, 1.0
    if kind == "linear":
        return f / need("factor"), 1.0
    if kind == "llama3":
        old, low, high = (need("original_max_position_embeddings"), need("low_freq_factor"),
                          need("high_freq_factor"))
        kept = ((old * f / (2.0 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        return f * (kept + (1.0 - kept) / need("factor")), 1.0
    if kind == "yarn":
        old, factor = need("original_max_position_embeddings"), need("factor")

        def pair_with(turns):            # the (fractional) pair that turns so often over the original length
            return rotary_dim * math.log(old / (2.0 * math.pi * turns)) / (2.0 * math.log(base))

        fast, slow = s.get("beta_fast") or 32.0, s.get("beta_slow") or 1.0
        lo, hi = pair_with(fast), pair_with(slow)
        if s.get("truncate", True):
            lo, hi = math.floor(lo), math.ceil(hi)
        lo, hi = max(lo, 0), min(hi, rotary_dim - 1)
        kept = 1.0 - ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        factor_on = s.get("attention_factor")
        if factor_on is None:
            one, both = float(s.get("mscale") or 0.0), float(s.get("mscale_all_dim") or 0.0)
            if both and not one or one not in (0.0, 1.0) and not both:
                raise ValueError("rotary scaling 'yarn': mscale and mscale_all_dim go together")

            def m(x):
                return 0.1 * x * math.log(factor) + 1.0 if factor > 1.0 else 1.0

            factor_on = m(one) / m(both) if both else m(1.0)
        return f * (kept + (1.0 - kept) / factor), float(factor_on)
    raise ValueError(f"unknown rotary scaling {kind!r}")


class RotaryTable:
    """cos and sin of every position: fp32 [max_positions, rotary_dim / 2, 2].
    The tensor is the table's for its life: calls pass on its address."""

    table = property(lambda self: self._table)

    def __init__(self, table: torch.Tensor, layout: str = "half"):
        if layout not in LAYOUTS:
            raise ValueError(f"layout must be one of {sorted(LAYOUTS)}, got {layout!r}")
        if table.dtype != torch.float32 or table.dim() != 3 or table.shape[2] != 2:
            raise TypeError(f"table must be fp32 [max_positions, rotary_dim / 2, 2], got {table.dtype} "
                            f"{tuple(table.shape)}")
        if table.shape[0] == 0 or table.shape[1] == 0 or table.shape[1] % 4 != 0:
            raise ValueError(f"rotary_dim must be a positive multiple of 8 and the table not empty, got "
                             f"{tuple(table.shape)}")
        self._table = table.contiguous()
        self.layout = layout
        self.device, self.ptr, self.layout_code = self.table.device, self.table.data_ptr(), LAYOUTS[layout]
        self.rotary_dim = 2 * table.shape[1]
        self.max_positions = table.shape[0]

    @classmethod
    def build(cls, rotary_dim: int, max_positions: int, base: float = 10000.0, layout: str = "half",
              scaling: dict | None = None, device="cuda") -> "RotaryTable":
        """The table of `rotary_frequencies`, computed in float64 and rounded once."""
        f, factor = rotary_frequencies(rotary_dim, base, scaling, max_positions)
        angles = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * f.to(device)
        return cls((torch.stack([angles.cos(), angles.sin()], dim=-1) * factor).float(), layout)

    @classmethod
    def from_config(cls, config, max_positions: int | None = None, layout: str = "half",
                    device="cuda") -> "RotaryTable":
        """From a decoder model's configuration (``rope_parameters``, or
        ``rope_theta`` and ``rope_scaling``)."""
        s = dict(getattr(config, "rope_parameters", None) or getattr(config, "rope_scaling", None) or {})
        base = s.get("rope_theta") or getattr(config, "rope_theta", None) or 10000.0
        if _kind(s) not in ("default", "linear") and s.get("original_max_position_embeddings") is None:
            s["original_max_position_embeddings"] = config.max_position_embeddings
        head_dim = getattr(config, "head_dim", None) or config.hidden_size // config.num_attention_heads
        part = s.get("partial_rotary_factor") or getattr(config, "partial_rotary_factor", None) or 1.0
        return cls.build(int(head_dim * part), max_positions or config.max_position_embeddings, base, layout, s,
                         device)


def apply_rotary(x: torch.Tensor, positions: torch.Tensor, rotary: RotaryTable, out: torch.Tensor = None,
                 inverse: bool = False) -> torch.Tensor:
    """Turns x (tokens, heads, head_dim) fp16 / bf16 by the angles of
    positions (tokens,): the first ``rotary.rotary_dim`` elements of each head
    in ``rotary.layout``'s pairs, the rest unchanged, one rounding.  x and
    `out` may have any strides with unit stride along head_dim; ``out=x``
    turns in place.  ``inverse=True`` turns by the negative angles: it maps the
    gradient of the call's result to that of x, and undoes the call where the
    table has no factor on its cosines and sines (with one, as yarn's, there and
    back is its square times x).  Gradients are not recorded: the result is
    detached, whatever x is."""
    shape, dev = x.shape, x.device
    assert x.is_cuda and len(shape) == 3, f"x must be a CUDA tensor (tokens, heads, head_dim), got {tuple(shape)}"
    tokens, heads, head_dim = shape
    dtype = activation_code(x.dtype, "apply_rotary: x")
    assert positions.shape == (tokens,) and positions.device == dev, \
        f"positions must be ({tokens},) on {dev}, got {tuple(positions.shape)} on {positions.device}"
    assert rotary.device == dev, f"the rotary table is on {rotary.device}, x on {dev}"
    assert rotary.rotary_dim <= head_dim and head_dim % 8 == 0, \
        f"head_dim {head_dim} must be a multiple of 8 and at least rotary_dim {rotary.rotary_dim}"
    if out is None:
        out = x.new_empty(shape)
    else:
        assert out.shape == shape and out.dtype == x.dtype and out.device == dev, \
            f"out must be {tuple(shape)} {x.dtype} on {dev}"
        assert out.stride(-1) == 1, "out must have unit stride along head_dim"
    if tokens == 0 or heads == 0:
        return out
    xs, os_ = x.stride(), out.stride()
    if xs[2] != 1:
        x = x.contiguous()
        xs = x.stride()
    if not positions.is_contiguous():
        positions = positions.contiguous()
    packed = _lib.ROTARY_ARGS.pack(
        x.data_ptr(), out.data_ptr(), rotary.ptr, positions.data_ptr(), tokens, heads, head_dim, rotary.rotary_dim,
        rotary.max_positions, xs[0], xs[1], os_[0], os_[1], dtype, rotary.layout_code,
        index_bytes(positions, "positions"), 1 if inverse else 0, call_flags())
    call(_lib.load().ql_rotary, packed, dev)
    return out


__all__ = ["RotaryTable", "apply_rotary", "rotary_frequencies"]
